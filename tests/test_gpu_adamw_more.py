"""AdamW between other work: calls from a stream that is not the last step's, and tensors that are pieces of larger buffers."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _busy(stream):
    """Some milliseconds of work on a stream."""
    import torch
    with torch.cuda.stream(stream):
        work = torch.ones(8192, 8192, device="cuda")
        for _ in range(4):
            work = work @ work * 1e-4
    return work


def _made(n=5000):
    import torch
    from nerf_amd import AdamW
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    p, g = [torch.randn(n, generator=gen, device="cuda")], [torch.randn(n, generator=gen, device="cuda")]
    opt = AdamW(p, g, lr=1e-2)
    opt.step()
    torch.cuda.synchronize()
    return p, g, opt


def test_the_count_of_a_step_on_another_stream():
    """state_dict() from the default stream while a step waits behind work on another one: count and tensors are those after the step."""
    import torch
    p, g, opt = _made()
    q, h, alone = _made()
    alone.step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    _busy(s)
    with torch.cuda.stream(s):
        opt.step()
    saved = opt.state_dict()
    copies = {k: [t.clone() for t in v] for k, v in saved.items() if isinstance(v, list)}
    torch.cuda.synchronize()
    assert saved["step"] == 2 and opt.get_step() == 2
    for k, v in copies.items():
        assert torch.equal(v[0], alone.state[k][0]), k
    assert torch.equal(p[0], q[0])


def test_the_count_set_behind_a_step_on_another_stream():
    """set_step() from the default stream while a step waits on another one: the step is done with before, and the count is the one set."""
    import torch
    p, g, opt = _made()
    s = torch.cuda.Stream()
    _busy(s)
    with torch.cuda.stream(s):
        opt.step()
    opt.set_step(10)
    torch.cuda.synchronize()
    assert opt.get_step() == 10
    opt.step()
    assert opt.get_step() == 11


def test_the_count_of_a_step_on_a_fixed_stream():
    import torch
    p, g, opt = _made()
    s = torch.cuda.Stream()
    opt.set_stream(s.cuda_stream)
    _busy(s)
    opt.step()
    opt.set_stream(None)
    assert opt.get_step() == 2
    opt.set_stream(s.cuda_stream)
    _busy(s)
    opt.step()
    assert opt.get_step() == 3


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_lies_between_tensors(dtype, bits):
    """Tensors that start at multiples of 256 in shared buffers whose gaps hold NaN: norm, step and read_state neither read nor change the gaps."""
    import torch
    from nerf_amd import AdamW
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    sizes = [1, 3, 128, 257, 4097, 300]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // 256) * 256
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)

    def make(gap):
        flat = torch.full((at,), gap, dtype=t, device="cuda")
        return flat, [flat[a:a + n] for a, n in zip(starts, sizes)]

    outcome = []
    values = [[torch.randn(n, generator=gen, device="cuda").to(t) for n in sizes] for _ in range(2)]
    for gap in (0.0, float("nan")):
        (fp, p), (fg, g) = make(gap), make(gap)
        for x, y in ((p, values[0]), (g, values[1])):
            for a, b in zip(x, y):
                a.copy_(b)
        opt = AdamW(p, g, lr=1e-2, state_bits=bits)
        norm = opt.grad_norm(max_norm=0.5)
        opt.step(grad_scale=norm[1:])
        outcome.append([norm, *opt.read_state(), *[x.clone() for x in p]])
        inside = torch.zeros(at, dtype=torch.bool, device="cuda")
        for a, n in zip(starts, sizes):
            inside[a:a + n] = True
        for flat in (fp, fg):
            assert (torch.isnan(flat[~inside]).all() if math.isnan(gap) else (flat[~inside] == 0).all()) and torch.isfinite(flat[inside]).all()
    exact = math.sqrt(sum((x.double() ** 2).sum().item() for x in values[1]))
    assert abs(outcome[1][0][0].item() - exact) <= 2.0 ** -23 * exact
    assert all(torch.equal(a, b) for a, b in zip(*outcome))
