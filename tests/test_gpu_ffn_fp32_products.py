"""The feed-forward block's products of fp32 pieces, one term at a time: operands with one value in each row or column, so that every output is
one product of numbers with 24 bits, and a piece that is missing, misplaced or badly rounded shows in it.

Bound of one product, in units of u = 2^-24 of it.  An operand is three bf16 pieces, each rounded to nearest: |x1| <= 2^-8 and |x2| <= 2^-17 of
the power of two below |x|, so that the products left out, x1 w2 + x2 w1 + x2 w2, are at most 2^-24 + 2^-34: 1.01 u, or nothing where one operand is
a power of two (its second and third piece are zero).  The six others are exact in fp32 and added one after the other, smallest first: only
the last sum is as large as the product, the five before it are below 2^-6 of it.  A sum that is cut off instead of rounded loses 2 u of itself: 2 (1 +
5 / 64) < 2.2 u.  Products that follow one another add up; relu, factors of one and powers of two round nothing."""
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND, CUT = 2.2 * U, 1.01 * U


def _mantissas(shape, gen):
    """24-bit numbers in [1, 2) of either sign: random ones, and every other one just below 1 + 2^-7, whose lower pieces are large if cut off."""
    import torch
    m = 1 + torch.randint(0, 1 << 23, shape, generator=gen, device="cuda").double() * 2.0 ** -23
    near = 1 + 2.0 ** -7 - torch.randint(1, 64, shape, generator=gen, device="cuda").double() * 2.0 ** -23
    pick = torch.randint(0, 2, shape, generator=gen, device="cuda") == 0
    return torch.where(pick, near, m).float()


def _powers(shape, gen):
    import torch
    return torch.ldexp(torch.ones(shape, device="cuda"), torch.randint(-3, 4, shape, generator=gen, device="cuda"))


def _scattered(n, values, gen):
    """[n][n] with one value in each row and in each column."""
    import torch
    w = torch.zeros(n, n, device="cuda")
    w[torch.arange(n, device="cuda"), torch.randperm(n, generator=gen, device="cuda")] = values
    return w


def _case(rows, n, path, full, seed):
    """path: the weight that the values go through, w_gate with u = 1 or w_up with g = 1; full: whether that one or w_down has 24 bits, the
    other one has powers of two."""
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    w = _scattered(n, _mantissas((n,), gen) if full == "first" else _powers((n,), gen), gen)
    wd = _scattered(n, _mantissas((n,), gen) if full == "down" else _powers((n,), gen), gen)
    zero, one = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    a = {"x": _mantissas((rows, n), gen), "dy": _mantissas((rows, n), gen), "w_down": wd, "b_down": zero}
    if path == "gate":
        a.update(w_gate=w, w_up=torch.zeros_like(w), b_gate=zero, b_up=one)
    else:
        a.update(w_gate=torch.zeros_like(w), w_up=w, b_gate=one, b_up=zero)
    return a, w


def _block(n):
    from nerf_amd import GatedFFN
    return GatedFFN(n, n, dtype="f32", activation="relu", bias=True)


def _backward(blk, a, **kw):
    return blk.backward(a["x"], a["w_gate"], a["w_up"], a["w_down"], a["dy"], a["b_gate"], a["b_up"], **kw)


def _close(got, want, rel, name):
    off = (got.double() - want).abs()
    worst = (off / want.abs().clamp(min=1e-300)).max().item() / U
    assert (off <= rel * want.abs()).all(), f"{name}: {worst:.3g} units of 2^-24, {rel / U:.3g} allowed"


# 64 x 128, 128 x 128 and 256 x 256 tiles; the gate, dh and the weight gradients whole and in parts; sizes that end inside a tile
SIZES = [(65, 64), (100, 1024), (300, 264), (1000, 72), (2048, 2048), (16384, 512), (9000, 257), (524, 549), (34000, 256)]


@pytest.mark.parametrize("full", ["first", "down"])
@pytest.mark.parametrize("path", ["gate", "up"])
@pytest.mark.parametrize("rows,n", SIZES)
def test_forward_and_dx(rows, n, path, full):
    a, w = _case(rows, n, path, full, rows + n)
    if path == "gate":
        a["x"] = a["x"].abs()
        w.abs_()
    blk = _block(n)
    x, dy, wide, wd = a["x"].double(), a["dy"].double(), w.double(), a["w_down"].double()
    both = CUT + 2 * ROUND                    # of the two products one has two operands of 24 bits
    y = blk.forward(a["x"], a["w_gate"], a["w_up"], a["w_down"], a["b_gate"], a["b_up"], a["b_down"])
    _close(y, (x @ wide.t()) @ wd.t(), both * (1 + U), "y")
    dx = _backward(blk, a, need_weights=False)["dx"]
    _close(dx, (dy @ wd) @ wide, both * (1 + U), "dx")


@pytest.mark.parametrize("path", ["gate", "up"])
@pytest.mark.parametrize("rows,n", SIZES)
def test_weight_gradients(rows, n, path):
    """dy has one value in each column: one row of x and h meets each of its values."""
    import torch
    a, w = _case(rows, n, path, "neither", 3 * rows + n)
    if path == "gate":
        a["x"] = a["x"].abs()
        w.abs_()
    cols = torch.arange(n, device="cuda")
    dense, a["dy"] = a["dy"], torch.zeros_like(a["dy"])
    at = cols * 37 % rows
    a["dy"][at, cols] = dense[at, cols]
    x, dy, wide, wd = a["x"].double(), a["dy"].double(), w.double(), a["w_down"].double()
    g = _backward(_block(n), a, need_dx=False)
    dh = dy @ wd                              # powers of two: no bits are cut
    name = "dw_gate" if path == "gate" else "dw_up"
    _close(g[name], dh.t() @ x, (CUT + 2 * ROUND) * (1 + U), name)
    _close(g["dw_down"], dy.t() @ (x @ wide.t()), (CUT + 2 * ROUND) * (1 + U), "dw_down")


def _bits(values):
    import torch
    return torch.tensor(values, dtype=torch.int64, device="cuda").to(torch.int32).view(torch.float32)


@pytest.mark.parametrize("rows", [70, 4096])
def test_the_largest_and_the_smallest_numbers(rows):
    """Values next to fp32's largest, which round to an infinite bf16, and its smallest normal ones, of which what is below 2^-133 may be
    dropped."""
    import torch
    top = [0x7f7fffff, 0x7f7f8000, 0x7f7f7fff, 0x7f7f8001, 0x7f7f0000, 0x7f7effff, 0x7f000000, 0x7effffff]
    low = [0x00800000, 0x00800001, 0x00ffffff, 0x00c08081, 0x01008001, 0x02ffffff, 0x00807fff, 0x00808000]
    big = _bits(top + [t | 0x80000000 for t in top])
    small = _bits(low + [t | 0x80000000 for t in low])
    n = 16
    for values, factor in ((big, 2.0 ** -20), (small, 2.0 ** 40)):
        eye = torch.eye(n, device="cuda")
        zero, one = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
        x = values.repeat(rows, 1)
        blk = _block(n)
        y = blk.forward(x, torch.zeros_like(eye), factor * eye, eye, one, zero, zero)
        want = x.double() * factor
        assert ((y.double() - want).abs() <= 2 * ROUND * (1 + U) * want.abs() + 2.0 ** -133 * factor).all()
        # dy takes them through dh and du = dh; x = 1, so that dg = dh u stays in fp32's range as well
        dx = blk.backward(torch.ones_like(x), torch.zeros_like(eye), factor * eye, eye, x, one, zero, need_weights=False)["dx"]
        assert ((dx.double() - want).abs() <= 2 * ROUND * (1 + U) * want.abs() + 2.0 ** -133 * factor).all()


@pytest.mark.parametrize("rows", [70, 4096])
@pytest.mark.parametrize("bits", [0x7f800000, 0xff800000, 0x7fc00000, 0xffc00000, 0x7fffffff, 0xffffffff, 0x7f800001, 0x7f80ffff, 0xff808000, 0x7fffff80])
def test_every_infinity_and_nan_shows(rows, bits):
    """Whatever the bits of a NaN, and for both infinities: NaN in its own row of y and dx, and in the weight gradients it meets."""
    import torch
    n = 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    w = [make(n, n), make(n, n), make(n, n)]
    b = [make(n), make(n), make(n)]
    x, dy = make(rows, n), make(rows, n)
    x.view(torch.int32)[5, 7] = bits if bits < 1 << 31 else bits - (1 << 32)
    from nerf_amd import GatedFFN
    blk = GatedFFN(n, n, dtype="f32", activation="silu", bias=True)
    y = blk.forward(x, *w, *b)
    g = blk.backward(x, *w, dy, b[0], b[1])
    rest = [r for r in range(rows) if r != 5]
    for t in (y, g["dx"]):
        assert torch.isnan(t[5]).all() and torch.isfinite(t[rest]).all()
    assert torch.isnan(g["dw_gate"]).all() and torch.isnan(g["dw_up"]).all() and torch.isnan(g["dw_down"]).all()
