"""The forward pass where pre-activations are near the type's largest number: finite wherever the formula's result is."""
import math

import pytest

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


def _act(g, kind):
    import torch
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return g * 0.5 * torch.erfc(-g / math.sqrt(2.0))
    if kind == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return torch.clamp(g, min=0)


# few rows, tiles, and the gate in parts
@pytest.mark.parametrize("rows,n", [(1, 48), (20, 48), (100, 48), (3000, 64), (100, 1024)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
def test_values_near_the_largest(act, dtype, rows, n):
    """g from the largest number down, u = 1/2: h and y are half of g where it is positive and zero else.  Roundings: h and y half a step each, the
    activation 1e-6 of its size, and 1e-6 where that is small."""
    import torch
    from nerf_amd import GatedFFN
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    top = torch.finfo(t).max
    g = top * torch.linspace(1.0, 0.25, n // 2, dtype=torch.float64)
    x = torch.cat([g, -g]).to(t).cuda().repeat(rows, 1)
    assert torch.isfinite(x).all()
    eye, zero = torch.eye(n, device="cuda").to(t), torch.zeros(n, device="cuda").to(t)
    half = torch.full((n,), 0.5, device="cuda").to(t)
    blk = GatedFFN(n, n, dtype=dtype, activation=act, bias=True)
    y = blk.forward(x, eye, torch.zeros_like(eye), eye, zero, half, zero)
    want = _act(x.double(), act) * 0.5
    assert torch.isfinite(want).all() and torch.isfinite(y).all()
    assert ((y.double() - want).abs() <= (torch.finfo(t).eps + 1e-6) * want.abs() + 1e-6).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_forward_over_the_whole_range(act, dtype):
    """Magnitudes from 1e-30 to 2.5e38 of either sign, on the few-row path and in tiles, with the same bounds."""
    import torch
    from nerf_amd import GatedFFN
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    n = 256
    x = torch.cat([s * torch.logspace(-30, 38.4, n // 2, dtype=torch.float64) for s in (1, -1)]).to(t).cuda().repeat(70, 1)
    eye, zero = torch.eye(n, device="cuda").to(t), torch.zeros(n, device="cuda").to(t)
    half = torch.full((n,), 0.5, device="cuda").to(t)
    blk = GatedFFN(n, n, dtype=dtype, activation=act, bias=True)
    want = 0.5 * _act(x.double(), act)
    for rows in (70, 3):
        y = blk.forward(x[:rows], eye, torch.zeros_like(eye), eye, zero, half, zero)
        assert torch.isfinite(y).all()
        assert ((y.double() - want[:rows]).abs() <= (torch.finfo(t).eps + 1e-6) * want[:rows].abs() + 1e-6).all()
