"""The norm with the residual's addition on the GPU against the oracle in 64 bits.

float32 results: 1e-5 of the tensor's largest value.  bfloat16 results: half a step, 2^-8 of their own value, more.  The
backward reads the sum as it was stored; where that is bfloat16, the normalised row it uses is off by up to half a step of
itself, and the gradients' formula carries that on (spelled out in _backward_tolerance).  e4m3 values: half a step, 2^-4 of
the value, or half of the smallest step, 2^-10, in units of the row's scale."""
import pytest
import torch

from oracle import selective
from residual_norm import residual_rms_norm, residual_rms_norm_e4m3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = torch.finfo(torch.bfloat16).eps / 2
TYPES = [("f32", torch.float32, torch.float32), ("bf16", torch.bfloat16, torch.bfloat16), ("bf16_f32", torch.bfloat16, torch.float32),
         ("f32_none", torch.float32, None), ("bf16_none", torch.bfloat16, None)]
SIZES = [(1, 1), (3, 2), (5, 7), (1, 16), (17, 64), (9, 100), (4, 255), (6, 1024), (3, 1028), (2, 2048), (2, 2049), (3, 4096),
         (2, 5001), (2, 8192), (2, 8196), (1, 16384), (1, 20001)]


def inputs(rows, D, xt, rt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, D, generator=g).to(xt)
    r = None if rt is None else (torch.randn(rows, D, generator=g) * 3).to(rt)
    w = 1 + 0.3 * torch.randn(D, generator=g)
    return x, r, w, torch.randn(rows, D, generator=g).to(xt), None if rt is None else torch.randn(rows, D, generator=g).to(rt)


def check(got, want, name, extra=0.0):
    got64, want = got.detach().cpu().double(), want.detach()
    tol = 1e-5 * float(want.abs().max()) + 1e-30 + extra + (HALF * want.abs() if got.dtype == torch.bfloat16 else 0)
    worst = float(((got64 - want).abs() - tol).max())
    assert worst <= 0, f"{name}: over the tolerance by {worst:.3g}"


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("xt,rt", [t[1:] for t in TYPES], ids=[t[0] for t in TYPES])
def test_norm_and_gradients(size, xt, rt):
    x, r, w, go, gt = inputs(*size, xt, rt)
    xd, rd, wd = x.double().requires_grad_(), None if r is None else r.double().requires_grad_(), w.double().requires_grad_()
    out, total = selective.rms_norm(xd, rd, wd, 1e-5)
    leaves = [t for t in (xd, rd, wd) if t is not None]
    loss = (out * go.double()).sum() + (0 if gt is None else (total * gt.double()).sum())
    grads = torch.autograd.grad(loss, leaves)
    on = lambda t: None if t is None else t.to(DEV)
    if size[1] > 16384:
        o, s = residual_rms_norm(on(x), on(r), on(w))
        check(o, out, "out")
        check(s, total, "sum")
        return
    gx, gr, gw = on(x).requires_grad_(), None if r is None else on(r).requires_grad_(), on(w).requires_grad_()
    o, s = residual_rms_norm(gx, gr, gw)
    check(o, out, "out")
    check(s, total, "sum")
    with torch.no_grad():
        o2, s2 = residual_rms_norm(gx, gr, gw)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    got = torch.autograd.grad((o, s) if gt is not None else o, [t for t in (gx, gr, gw) if t is not None],
                              (on(go), on(gt)) if gt is not None else on(go))
    ex, ew = _backward_tolerance(total.detach(), w.double(), go.double(), s.dtype == torch.bfloat16 and r is not None)
    check(got[0], grads[0], "g_x", ex)
    if r is not None:
        check(got[1], grads[1], "g_residual", ex)
    check(got[-1], grads[-1], "g_weight", ew)


def _backward_tolerance(total, w, go, rounded):
    """g_x = rstd (g w - hat m) is a difference, and for D = 1 of two numbers that agree to 1e-5 of themselves (hat = 1 up to
    eps): float32 holds the bar of 1e-5 for the two terms, not for what is left of them, so their size is what it is taken
    of.  A sum stored in bfloat16 adds: hat is off by HALF |hat|, so hat m by HALF (|hat m| + |hat| mean|g w hat|) and g hat,
    summed over the rows, by HALF sum|g hat|."""
    rstd = 1 / torch.sqrt((total * total).mean(-1, keepdim=True) + 1e-5)
    hat, gw = total * rstd, go * w
    m = (gw * hat).mean(-1, keepdim=True)
    terms = 1e-5 * rstd * (gw.abs() + (hat * m).abs())
    if not rounded:
        return terms, 0.0
    ex = HALF * rstd * ((hat * m).abs() + hat.abs() * (gw * hat).abs().mean(-1, keepdim=True)) * (1 + HALF)
    return ex + terms, HALF * (go * hat).abs().sum(0)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("xt,rt", [t[1:] for t in TYPES], ids=[t[0] for t in TYPES])
def test_norm_in_8_bits(size, xt, rt):
    x, r, w, _, _ = inputs(*size, xt, rt, seed=3)
    out, total = selective.rms_norm(x.double(), None if r is None else r.double(), w.double(), 1e-5)
    on = lambda t: None if t is None else t.to(DEV)
    o, scale, s = residual_rms_norm_e4m3(on(x), on(r), on(w))
    assert o.dtype == torch.float8_e4m3fn and scale.shape == (size[0], 1)
    check(s, total, "sum")
    want = out.abs().amax(-1, keepdim=True) / 448
    check(scale, want, "scale")
    q = o.cpu().double()
    assert float(q.abs().amax(-1).min()) == 448.0                     # the largest value of each row is the type's largest
    step = torch.maximum(out.abs() * 2.0 ** -4, want * 2.0 ** -10)
    # 1e-5: the float32 arithmetic in front of the rounding
    assert float(((q * scale.cpu().double() - out).abs() - step * (1 + 1e-5) - 1e-5 * out.abs()).max()) <= 0


def test_norm_rows_of_zeros_nan_and_infinities():
    x = torch.randn(5, 100)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 7] = float("inf")
    out, total = residual_rms_norm(x.to(DEV), None, torch.ones(100, device=DEV))
    out = out.cpu()
    assert not out[1].any() and torch.isnan(out[2]).all() and torch.isnan(out[3, 7]) and torch.isfinite(out[[0, 4]]).all()
    o, scale, _ = residual_rms_norm_e4m3(x.to(DEV), None, torch.ones(100, device=DEV))
    o, scale = o.cpu().float(), scale.cpu()
    assert float(scale[1]) == 1.0 and not o[1].any() and torch.isnan(o[2]).all()
    assert torch.isfinite(o[[0, 4]]).all() and float(o[0].abs().max()) == 448.0


def test_norm_of_many_rows_and_leading_axes():
    g = torch.Generator().manual_seed(4)
    x, r = torch.randn(7, 311, 48, generator=g), torch.randn(7, 311, 48, generator=g)
    w = torch.rand(48, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (x.transpose(0, 1), r.transpose(0, 1), w)]
    out, total = residual_rms_norm(*leaves)
    wd = [t.double().requires_grad_() for t in (x.transpose(0, 1), r.transpose(0, 1), w)]
    o, t = selective.rms_norm(*wd, 1e-5)
    check(out, o, "out")
    go = torch.randn(o.shape, generator=g)
    got = torch.autograd.grad(out, leaves, go.to(DEV))
    for a, b, n in zip(got, torch.autograd.grad(o, wd, go.double()), ("x", "residual", "weight")):
        check(a, b, n)
    again = torch.autograd.grad(residual_rms_norm(*leaves)[0], leaves, go.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("size", [1e-20, 1e-36, 1e-40, 3e-44])
def test_eight_bit_rows_of_tiny_numbers(size):
    """Values down to the smallest numbers of float32 still fill the type's range; nothing turns into infinity or NaN."""
    x = torch.zeros(2, 64)
    x[0] = torch.linspace(-1, 1, 64) * size * 1e-3
    x[1] = torch.linspace(-1, 1, 64)
    w = torch.full((64,), 1.0)
    o, scale, _ = residual_rms_norm_e4m3(x.to(DEV), None, w.to(DEV))
    o, scale = o.cpu().float(), scale.cpu()
    assert torch.isfinite(o).all() and torch.isfinite(scale).all() and float(scale.min()) > 0
    assert float(o[1].abs().max()) == 448.0
    y = x[0].double() / (1e-5 ** 0.5)                           # the row's mean square vanishes next to eps
    assert float((o[0].double() * scale[0].double() - y).abs().max()) <= float(y.abs().max()) * 2.0 ** -4 + 2 * 1.4e-45


@pytest.mark.parametrize("xt,rt", [t[1:] for t in TYPES], ids=[t[0] for t in TYPES])
@pytest.mark.parametrize("D", [100, 1024, 2051, 9000])
def test_eight_bit_values_are_the_quotients(D, xt, rt):
    """Rows of ones with eps = 0 have a norm of exactly 1, so that a row's results are the weight's values and the quotients
    by the row's scale are known to the last bit: many lie on a border of two e4m3 values, or a rounding beside one, and
    have to fall to the side that the division gives them."""
    g = torch.Generator().manual_seed(D)
    x = torch.ones(3, D).to(xt)
    r = None if rt is None else torch.zeros(3, D).to(rt)
    for k in range(8):
        top = 448 * float(1 + torch.rand((), generator=g))               # the scale, between 1 and 2
        scale = torch.tensor(top, dtype=torch.float32) / 448
        grid = torch.randint(0, 126, (D,), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
        step = torch.where(grid < 2.0 ** -6, 2.0 ** -9, torch.exp2(torch.frexp(grid).exponent - 4.0))
        border = grid + step / 2                                        # exact: e4m3 values have four bits
        w = (border * scale) * torch.where(torch.rand(D, generator=g) < 0.5, -1.0, 1.0)
        w[int(torch.randint(0, D, (), generator=g))] = top
        assert float(w.abs().max()) == float(torch.tensor(top, dtype=torch.float32))
        o, s, _ = residual_rms_norm_e4m3(x.to(DEV), None if r is None else r.to(DEV), w.to(DEV), 0.0)
        assert torch.equal(s.cpu(), scale.expand(3, 1))
        want = (w / scale).to(torch.float8_e4m3fn).float()
        assert torch.equal(o.cpu().float(), want.expand(3, D)), f"{int((o.cpu().float() != want).sum())} of {3 * D} differ"


def test_eight_bit_scales_among_the_smallest_numbers():
    """A row's largest value is a few hundred times float32's smallest number, where max / 448 is off by up to half of
    itself: the scale is then the next number above it, so that no quotient passes the type's largest value."""
    tops = list(range(1, 1200, 7)) + [449, 465, 600, 671, 672, 673, 1119, 1120, 5000, 6271, 6272, 6273]
    x, least = torch.ones(1, 64, device=DEV), 2.0 ** -149
    for k in tops:
        w = (torch.arange(64) * k // 63).double() * least * torch.where(torch.arange(64) % 2 == 0, 1.0, -1.0)
        o, scale, _ = residual_rms_norm_e4m3(x, None, w.float().to(DEV), 0.0)
        o, scale = o.cpu().double(), float(scale)
        assert torch.isfinite(o).all(), k
        assert scale == -(-k // 448) * least, (k, scale / least)
        # half a step of the type: 2^-4 of the value, or 2^-10 of the scale; the quotient is rounded once before, by 2^-24
        bound = torch.maximum(w.abs() * 2.0 ** -4, torch.tensor(scale * 2.0 ** -10, dtype=torch.float64)) * (1 + 2.0 ** -20)
        assert float(((o * scale - w).abs() - bound).max()) <= 0, k
