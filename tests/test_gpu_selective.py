"""Selective scan, short causal convolution and their single-token forms on the GPU against the oracle in 64 bits.

Tolerances, relative to the largest value of the tensor: 1e-5 with float32 inputs (the bar of the other operators: a
result here is a sum of at most some thousand products whose factors carry a few roundings of 2^-24 each).  With bfloat16
inputs the oracle sees the same rounded inputs and a bfloat16 result is off by at most half a step more, 2^-8 of its own
value; the float32 results (states, gradients of parameters) keep the first bar."""
import pytest
import torch

from oracle import selective
from residual_norm import residual_rms_norm
from selective_scan import causal_conv, causal_conv_step, selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2


def check(got, want, name):
    want = want.detach()
    got64 = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got64).all() or not torch.isfinite(want).all(), name
    top = float(want.abs().max()) if want.numel() else 0.0
    tol = 1e-5 * top + 1e-30 + (HALF_STEP * want.abs() if got.dtype == torch.bfloat16 else 0)
    worst = float(((got64 - want).abs() - tol).max()) if want.numel() else 0.0
    assert worst <= 0, f"{name}: over the tolerance by {worst:.3g} (largest value {top:.3g})"


def rows(g, N, H, L, E, dtype, order):
    """(N, H, L, E): dense; the view of step-major storage; or that of a wider row that starts at an odd element."""
    if order == "dense":
        t = torch.randn(N, H, L, E, generator=g)
    elif order == "steps":
        t = torch.randn(L, N, H, E, generator=g).permute(1, 2, 0, 3)
    else:
        t = torch.randn(L, N, H, 2 * E + 3, generator=g)[..., 1:E + 1].permute(1, 2, 0, 3)
    return t.to(dtype)


def place(t, like=None):
    """On the GPU with the strides of the CPU tensor."""
    base = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
    return base.copy_(t)


def scan_case(N, H, L, E, S, G, dtype=torch.float32, order="steps", gate=True, D=True, bias=True, state=True, keep=False,
              lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = dict(u=rows(g, N, H, L, E, dtype, order), delta=rows(g, N, H, L, E, dtype, order),
             A=-torch.exp(torch.randn(H, E, S, generator=g) * 0.7), B=rows(g, N, G, L, S, dtype, order),
             C=rows(g, N, G, L, S, dtype, order), D=torch.randn(H, E, generator=g) if D else None,
             z=rows(g, N, H, L, E, dtype, order) if gate else None,
             delta_bias=torch.randn(H, E, generator=g) - 1 if bias else None,
             state=torch.randn(N, H, E, S, generator=g) if state else None)
    m = dict(keep=(torch.rand(N, L, generator=g) > 0.15).float() if keep else None,
             lengths=torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None)
    go = rows(g, N, H, L, E, dtype, order)
    return a, m, go, torch.randn(N, H, E, S, generator=g)


def run_scan(a, m, go, gl, softplus=True):
    """(got, want): dicts of the outputs and of every gradient."""
    want_in = {k: None if v is None else v.double().requires_grad_() for k, v in a.items()}
    out, last = selective.scan(**want_in, **m, softplus=softplus)
    leaves = [k for k in a if a[k] is not None]
    grads = torch.autograd.grad((out * go.double()).sum() + (last * gl.double()).sum(), [want_in[k] for k in leaves],
                                allow_unused=True)
    want = dict(out=out, last=last, **{"g_" + k: torch.zeros_like(want_in[k]) if v is None else v for k, v in zip(leaves, grads)})
    got_in = {k: None if v is None else place(v).requires_grad_() for k, v in a.items()}
    md = {k: None if v is None else v.to(DEV) for k, v in m.items()}
    out, last = selective_scan(**got_in, **md, softplus=softplus)
    grads = torch.autograd.grad((out, last), [got_in[k] for k in leaves], (place(go), gl.to(DEV)))
    got = dict(out=out, last=last, **{"g_" + k: v for k, v in zip(leaves, grads)})
    with torch.no_grad():      # the path without the saved states gives the same bits
        o2, l2 = selective_scan(**got_in, **md, softplus=softplus)
    assert torch.equal(o2, out) and torch.equal(l2, last)
    return got, want


SHAPES = [(1, 1, 1, 1, 16, 1), (2, 3, 17, 5, 16, 3), (1, 6, 33, 20, 8, 2), (3, 2, 50, 32, 12, 1), (2, 1, 40, 130, 32, 1),
          (1, 2, 20, 9, 64, 2), (1, 1, 16, 64, 4, 1), (2, 8, 31, 32, 16, 8), (1, 1, 2, 3, 1, 1), (1, 2, 19, 7, 37, 1)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_scan_and_gradients(shape, dtype):
    got, want = run_scan(*scan_case(*shape, dtype=dtype))
    for k in want:
        check(got[k], want[k], k)


@pytest.mark.parametrize("options", [
    dict(gate=False), dict(D=False), dict(bias=False), dict(state=False), dict(gate=False, D=False, bias=False, state=False),
    dict(keep=True), dict(lengths=[23, 0, 1]), dict(keep=True, lengths=[23, 16, 17]), dict(lengths=[40, -3, 5]),
    dict(order="dense"), dict(order="offset"), dict(order="offset", keep=True, gate=False)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_scan_options(options, dtype):
    got, want = run_scan(*scan_case(3, 2, 23, 13, 16, 2, dtype=dtype, **options))
    for k in want:
        check(got[k], want[k], k)


def test_scan_without_softplus_and_with_growing_states():
    a, m, go, gl = scan_case(2, 2, 20, 6, 16, 1, bias=False)
    a["delta"] = a["delta"].abs() * 0.1
    a["A"] = -a["A"]                                       # a decay above one is allowed
    got, want = run_scan(a, m, go, gl, softplus=False)
    for k in want:
        check(got[k], want[k], k)


def test_scan_step_sizes_from_tiny_to_large():
    """softplus over its whole range: for large negative arguments the step is exp of them, to full relative precision."""
    L = 24
    a, m, go, gl = scan_case(1, 1, L, 8, 16, 1, bias=False, gate=False, D=False, state=False)
    a["delta"] = torch.linspace(-60, 40, L)[None, None, :, None].expand(1, 1, L, 8).contiguous()
    a["u"] = torch.randn(1, 1, L, 8, generator=torch.Generator().manual_seed(2)) * torch.exp(-a["delta"].clamp(max=0))
    got, want = run_scan(a, m, go, gl)
    for k in ("out", "last", "g_u", "g_B", "g_C", "g_A"):
        check(got[k], want[k], k)
    ratio = got["g_delta"].cpu().double() / want["g_delta"]
    assert float((ratio[:, :, :14] - 1).abs().max()) < 1e-4    # tiny steps: the gradient is relative to themselves


@pytest.mark.parametrize("N,H,L,E,S,G", [(1, 1, 700, 96, 16, 1), (2, 2, 333, 40, 8, 1), (1, 2, 401, 9, 33, 2), (1, 1, 1500, 3, 16, 1)])
@pytest.mark.parametrize("keep", [False, True])
def test_scan_long_rows(N, H, L, E, S, G, keep):
    """Rows that are cut into segments, with and without resets, one of them ending inside a segment in the middle."""
    got, want = run_scan(*scan_case(N, H, L, E, S, G, keep=keep, lengths=[L, L - 100][:N]))
    for k in want:
        check(got[k], want[k], k)


@pytest.mark.parametrize("N,H,L,E,S,G", [(1, 1, 700, 96, 16, 1), (2, 2, 333, 40, 8, 1), (1, 2, 401, 9, 33, 2)])
def test_scan_long_rows_in_16_bits(N, H, L, E, S, G):
    got, want = run_scan(*scan_case(N, H, L, E, S, G, dtype=torch.bfloat16, keep=True, lengths=[L, L - 100][:N]))
    for k in want:
        check(got[k], want[k], k)


# calls that fill a quarter of the device and more: few segments, tiles of channels that end inside a group
WIDE = [(2, 1, 37, 2048, 16, 1), (4, 2, 50, 600, 20, 2), (3, 1, 33, 1500, 32, 1), (9, 8, 20, 40, 64, 4), (16, 1, 97, 203, 9, 1)]


@pytest.mark.parametrize("shape", WIDE, ids=str)
@pytest.mark.parametrize("options", [dict(), dict(keep=True, gate=False, state=False), dict(ragged=True, keep=True, order="offset"),
                                     dict(D=False, bias=False, order="dense")], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_scan_of_many_channels(shape, options, dtype):
    options = dict(options)
    N, L = shape[0], shape[2]
    if options.pop("ragged", False):
        options["lengths"] = [L, 0, 1, 17, L - 1, 16][:N] + [L] * (N - 6)
    got, want = run_scan(*scan_case(*shape, dtype=dtype, **options))
    for k in want:
        check(got[k], want[k], k)


@pytest.mark.parametrize("lengths", [[700, 10, 0], [0, 0, 0], [3, 700, 699], [1, 1, 700], [512, 33, 32]], ids=str)
def test_segments_of_rows_of_different_lengths(lengths):
    """The segments are shared out over all rows: long ones get more of them, short and empty ones one."""
    got, want = run_scan(*scan_case(3, 1, 700, 5, 16, 1, lengths=lengths, keep=True))
    for k in want:
        check(got[k], want[k], k)


def test_segments_of_many_rows_of_different_lengths():
    g = torch.Generator().manual_seed(12)
    lengths = torch.randint(0, 150, (70,), generator=g).tolist()
    got, want = run_scan(*scan_case(70, 1, 150, 3, 16, 1, lengths=lengths))
    for k in want:
        check(got[k], want[k], k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N,L,lengths", [(70, 900, {3: 900, 64: 40}), (5, 2100, {1: 2100, 4: 17}), (4, 700, {})], ids=str)
def test_one_long_row_among_short_ones(N, L, lengths, dtype):
    """Most of the segments go to one row, and most of what is filled with zeros belongs to the others."""
    lengths = [lengths.get(n, n % 3) for n in range(N)]
    a, m, go, gl = scan_case(N, 1, L, 5, 16, 1, lengths=lengths, dtype=dtype)
    got, want = run_scan(a, m, go, gl)
    for k in want:
        check(got[k], want[k], k)
    for k in ("out", "g_u", "g_delta", "g_z", "g_B", "g_C"):
        for n, end in enumerate(lengths):
            assert not got[k][n, :, end:].any(), (k, n)


def scan_time(N, L, lengths, backward):
    """us of a scan of 64 channels x 16 states, the best of five."""
    r = lambda *s: torch.randn(*s, device=DEV)
    d = dict(u=r(N, 1, L, 64), delta=r(N, 1, L, 64), A=-torch.rand(1, 64, 16, device=DEV), B=r(N, 1, L, 16), C=r(N, 1, L, 16))
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    if backward:
        d = {k: v.requires_grad_() for k, v in d.items()}
        g = r(N, 1, L, 64)
    best = float("inf")
    for _ in range(6):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        out = selective_scan(**d, lengths=lengths)[0]
        if backward:
            torch.autograd.grad(out, list(d.values()), g)
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end) * 1e3)
    return best


@pytest.mark.parametrize("backward", [False, True])
def test_segments_of_a_long_row_are_bounded(backward):
    """A segment joins those in front of it one after the other: a row of 12001 steps beside 31 of 64 is cut into about as many as
    alone (measured: 141 and 344 us with up to 751 of them, 54 and 190 now, and 43 and 106 alone, where the padded rows' zeros
    take 20 and 60 us)."""
    alone = scan_time(1, 12001, None, backward)
    pad = torch.empty(4 if backward else 1, 32, 12001, 64, device=DEV)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(3):
        start.record()
        pad.zero_()
        end.record()
        torch.cuda.synchronize()
    assert scan_time(32, 12001, [12001] + [64] * 31, backward) < 1.7 * (alone + start.elapsed_time(end) * 1e3)


@pytest.mark.parametrize("backward", [False, True])
def test_padding_behind_short_rows_costs_what_it_is(backward):
    """Zeros behind short rows are filled by all workgroups: a row of 100000 steps beside three of one step takes at most three
    times what it takes alone (measured: ten times where each row's own workgroups filled them, 1.7 times now)."""
    assert scan_time(4, 100000, [100000, 1, 1, 1], backward) < 3 * scan_time(1, 100000, None, backward)


def test_masked_places_may_hold_anything():
    """NaN behind a row's length and in a state that a reset drops change nothing and reach no result."""
    a, m, go, gl = scan_case(2, 2, 21, 6, 16, 1, lengths=[21, 9])
    m["keep"] = torch.ones(2, 21)
    m["keep"][:, 0] = 0
    m["keep"][0, 11] = 0
    base, _ = run_scan(a, m, go, gl)
    bad = {k: None if v is None else v.clone(memory_format=torch.preserve_format) for k, v in a.items()}
    for k in ("u", "delta", "z", "B", "C"):
        bad[k][1, :, 9:] = float("nan")
    bad["state"][:] = float("inf")
    gob = go.clone(memory_format=torch.preserve_format)
    gob[1, :, 9:] = float("nan")
    leaves = {k: place(v).requires_grad_() for k, v in bad.items()}
    out, last = selective_scan(**leaves, keep=m["keep"].to(DEV), lengths=m["lengths"].to(DEV))
    grads = torch.autograd.grad((out, last), list(leaves.values()), (place(gob), gl.to(DEV)))
    assert torch.equal(out, base["out"]) and torch.equal(last, base["last"])
    for k, v in zip(leaves, grads):
        assert torch.equal(v, base["g_" + k]), k


def test_nan_passes_where_it_is_not_masked():
    a, m, _, _ = scan_case(1, 1, 8, 4, 16, 1)
    a = {k: v if v is None else place(v) for k, v in a.items()}
    a["delta"][0, 0, 3, 2] = float("nan")
    out, last = selective_scan(**a)
    nan = torch.isnan(out[0, 0])
    assert nan[3:, 2].all() and not nan[:, [0, 1, 3]].any() and not nan[:3].any() and torch.isnan(last[0, 0, 2]).all()


def test_infinite_decays_and_overflowing_products():
    """A = -inf forgets at once, in rows of any length; a state of zero stays zero where the decays' product overflows."""
    L = 75
    a, m, go, gl = scan_case(2, 1, L, 4, 16, 1, state=True, lengths=[L, 37])
    a["A"][:, 1] = float("-inf")
    fast = {**a, "A": torch.where(torch.isinf(a["A"]), torch.full_like(a["A"], -1e30), a["A"])}
    got = selective_scan(**{k: place(v) for k, v in a.items()}, lengths=m["lengths"].to(DEV))
    want = selective.scan(**{k: v.double() for k, v in fast.items()}, lengths=m["lengths"])
    check(got[0], want[0], "out")
    check(got[1], want[1], "last")
    u = torch.zeros(1, 1, 4000, 4, device=DEV)
    B = torch.ones(1, 1, 4000, 16, device=DEV)
    out, last = selective_scan(u, torch.ones_like(u), torch.ones(1, 4, 16, device=DEV), B, B)     # decays of e a step
    assert not out.any() and not last.any()


@pytest.mark.parametrize("sign", [1.0, -1.0], ids=["growing", "shrinking"])
@pytest.mark.parametrize("L,at", [(2048, (3, 10, 17, 30)), (700, (5, 300, 301, 699))], ids=str)
def test_states_whose_decays_multiply_beyond_float32(sign, L, at):
    """A state of e^-69 that grows by e^92 (or of e^69 that shrinks by it), and the same for its gradient: the steps' product leaves
    float32's range, the state does not, in rows that are cut into segments as in short ones.  Tolerance: the exponent of 92 is
    rounded three times (the decay, its product with the step size or their sum, log2 e), by 2^-24 of itself each, 1.7e-5 in all;
    the exponentials and products add a few roundings of 2^-24."""
    a, m, go, gl = scan_case(1, 1, L, 4, 16, 1, gate=False, D=False, bias=False)
    a["delta"] = torch.zeros(1, 1, L, 4)
    a["delta"][:, :, list(at)] = 23.0
    a["A"] = torch.full_like(a["A"], sign)
    small = 1e-30 if sign > 0 else 1e30
    a["u"], a["state"], gl = torch.zeros_like(a["u"]), a["state"] * small, gl * small
    go = torch.zeros_like(go)
    got, want = run_scan(a, m, go, gl, softplus=False)
    for k in ("out", "last", "g_state", "g_A"):
        top = float(want[k].detach().abs().max())
        assert torch.isfinite(got[k]).all(), k
        assert float((got[k].detach().cpu().double() - want[k].detach()).abs().max()) <= 2e-5 * top, k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_packed_rows_equal_single_sequences(dtype):
    a, _, _, _ = scan_case(1, 2, 45, 24, 16, 1, dtype=dtype, state=False)
    a = {k: v if v is None else place(v) for k, v in a.items()}
    cuts = [0, 7, 8, 30, 45]
    keep = torch.ones(1, 45, device=DEV)
    keep[0, cuts[:-1]] = 0
    out, last = selective_scan(**a, keep=keep)
    parts = [selective_scan(**{k: (v[:, :, lo:hi] if v is not None and v.dim() == 4 else v) for k, v in a.items()})
             for lo, hi in zip(cuts, cuts[1:])]
    want = torch.cat([p[0] for p in parts], 2).cpu().double()
    check(out, want, "out")
    check(last, parts[-1][1].cpu().double(), "last")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_step(shape, dtype):
    N, H, _, E, S, G = shape
    a, m, _, _ = scan_case(N, H, 3, E, S, G, dtype=dtype, keep=True)
    m["keep"][0, 1] = 0
    out, last = selective.scan(**{k: v if v is None else v.double() for k, v in a.items()}, **m)
    d = {k: v if v is None else place(v) for k, v in a.items()}
    state, kd = d["state"], m["keep"].to(DEV)
    for t in range(3):
        o = selective_scan_step(d["u"][:, :, t], d["delta"][:, :, t], state, d["A"], d["B"][:, :, t], d["C"][:, :, t], d["D"],
                                d["z"][:, :, t], d["delta_bias"], kd[:, t])
        check(o, out[:, :, t], f"out {t}")
    check(state, last, "state")


def test_step_overwrites_a_strided_state():
    a, _, _, _ = scan_case(2, 1, 1, 8, 16, 1)
    d = {k: place(v) for k, v in a.items()}
    pool = torch.zeros(2, 1, 8, 2, 16, device=DEV)
    pool[:, :, :, 1] = d["state"]
    one = {k: v[:, :, 0] if v.dim() == 4 and k != "state" else v for k, v in d.items()}
    ref = d["state"].clone()
    o1 = selective_scan_step(**{**one, "state": ref})
    o2 = selective_scan_step(**{**one, "state": pool[:, :, :, 1]})
    assert torch.equal(o1, o2) and torch.equal(pool[:, :, :, 1], ref) and not pool[:, :, :, 0].any()


# ---- convolution
def conv_case(N, H, L, E, W, dtype=torch.float32, order="steps", bias=True, state=True, keep=False, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = dict(x=rows(g, N, H, L, E, dtype, order), weight=torch.randn(H, E, W, generator=g),
             bias=torch.randn(H, E, generator=g) if bias else None,
             state=torch.randn(N, H, W - 1, E, generator=g).to(dtype) if state else None)
    m = dict(keep=(torch.rand(N, L, generator=g) > 0.25).float() if keep else None,
             lengths=torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None)
    return a, m, rows(g, N, H, L, E, dtype, order), torch.randn(N, H, W - 1, E, generator=g).to(dtype)


def run_conv(a, m, go, gl, silu=True):
    w = {k: None if v is None else v.double().requires_grad_() for k, v in a.items()}
    out, last = selective.conv(**w, **m, silu=silu)
    leaves = [k for k in a if a[k] is not None]
    grads = torch.autograd.grad((out * go.double()).sum() + (last * gl.double()).sum(), [w[k] for k in leaves], allow_unused=True)
    want = dict(out=out, last=last, **{"g_" + k: torch.zeros_like(w[k]) if v is None else v for k, v in zip(leaves, grads)})
    d = {k: None if v is None else place(v).requires_grad_() for k, v in a.items()}
    md = {k: None if v is None else v.to(DEV) for k, v in m.items()}
    out, last = causal_conv(**d, **md, silu=silu)
    grads = torch.autograd.grad((out, last), [d[k] for k in leaves], (place(go), gl.to(DEV)))
    got = dict(out=out, last=last, **{"g_" + k: v for k, v in zip(leaves, grads)})
    for k in want:
        check(got[k], want[k], k)


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 3, 2, 5), (1, 2, 17, 16), (2, 1, 150, 40), (3, 2, 33, 7), (1, 4, 15, 64)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_conv_and_gradients(shape, W, dtype):
    run_conv(*conv_case(*shape, W, dtype=dtype))


@pytest.mark.parametrize("options", [
    dict(bias=False), dict(state=False), dict(keep=True), dict(lengths=[37, 0, 1]), dict(keep=True, lengths=[37, 16, 18]),
    dict(lengths=[99, -1, 33]), dict(order="dense"), dict(order="offset"), dict(silu=False), dict(keep=True, lengths=[2, 3, 17])], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_conv_options(options, dtype):
    options = dict(options)
    silu = options.pop("silu", True)
    run_conv(*conv_case(3, 2, 37, 24, 4, dtype=dtype, **options), silu=silu)


@pytest.mark.parametrize("E,W,order,dtype", [(2752, 4, "steps", torch.float32), (2752, 2, "dense", torch.bfloat16),
                                             (2753, 3, "offset", torch.bfloat16)], ids=str)
@pytest.mark.parametrize("masks", [dict(), dict(keep=True, lengths=[650, 0, 17, 128])], ids=["plain", "masked"])
def test_conv_of_many_steps_and_channels(E, W, order, dtype, masks):
    """Calls that fill the device, whose backward walks runs of 16 steps."""
    run_conv(*conv_case(4, 1, 650, E, W, dtype=dtype, order=order, **masks))


def test_conv_masked_places_may_hold_anything():
    a, m, go, gl = conv_case(2, 1, 20, 8, 4, lengths=[20, 6])
    m["keep"] = torch.ones(2, 20)
    m["keep"][:, 0] = 0
    d = {k: place(v).requires_grad_() for k, v in a.items()}
    md = {k: v.to(DEV) for k, v in m.items()}
    out, last = causal_conv(**d, **md)
    grads = torch.autograd.grad((out, last), list(d.values()), (place(go), gl.to(DEV)))
    bad = {k: place(v) for k, v in a.items()}
    bad["x"][1, :, 6:] = float("nan")
    bad["state"][:] = float("nan")
    gob = place(go)
    gob[1, :, 6:] = float("nan")
    bad = {k: v.requires_grad_() for k, v in bad.items()}
    out2, last2 = causal_conv(**bad, **md)
    grads2 = torch.autograd.grad((out2, last2), list(bad.values()), (gob, gl.to(DEV)))
    assert torch.equal(out, out2) and torch.equal(last, last2)
    for x, y in zip(grads, grads2):
        assert torch.equal(x, y)


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("E", [1, 7, 24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_conv_step(E, W, dtype):
    a, m, _, _ = conv_case(3, 2, 5, E, W, dtype=dtype, keep=True)
    m["keep"][1, 2] = 0
    out, last = selective.conv(**{k: v.double() for k, v in a.items()}, **m)
    d = {k: place(v) for k, v in a.items()}
    kd = m["keep"].to(DEV)
    for t in range(5):
        check(causal_conv_step(d["x"][:, :, t], d["state"], d["weight"], d["bias"], kd[:, t]), out[:, :, t], f"out {t}")
    check(d["state"], last, "state")


# ---- together, and under a caller's conditions
def _layer(d, h, state, keep=None, lengths=None):
    """norm -> convolution -> scan on (N, H, L, E) rows, as a layer runs them."""
    conv_state, scan_state = state
    N, H, L, E = h.shape
    y, _ = residual_rms_norm(h.permute(2, 0, 1, 3).reshape(L, N, H * E), None, d["norm"])
    x, conv_state = causal_conv(y.reshape(L, N, H, E).permute(1, 2, 0, 3), d["weight"], d["bias"], conv_state, keep, lengths)
    out, scan_state = selective_scan(x, x * 0.5, d["A"], d["B"][:, :, :L], d["C"][:, :, :L], d["D"], h, d["delta_bias"], scan_state,
                                     keep, lengths)
    return out, (conv_state, scan_state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_prompt_then_tokens_equals_the_whole_sequence(dtype):
    """A prompt of 13 steps and then 6 single tokens on the carried states, against all 19 steps at once."""
    N, H, L, E, S = 2, 2, 19, 12, 16
    a, _, _, _ = scan_case(N, H, L, E, S, 1, dtype=dtype, state=False)
    g = torch.Generator().manual_seed(9)
    d = {k: v if v is None else place(v) for k, v in a.items()}
    d.update(weight=torch.randn(H, E, 4, generator=g).to(DEV), bias=torch.randn(H, E, generator=g).to(DEV),
             norm=torch.rand(H * E, generator=g).to(DEV) + 0.5)
    h = d["u"]
    with torch.no_grad():
        whole, (cs, ss) = _layer(d, h, (None, None))
        out, (c, s) = _layer(d, h[:, :, :13], (None, None))
        outs = [out]
        for t in range(13, L):
            y, _ = residual_rms_norm(h[:, :, t].reshape(N, H * E), None, d["norm"])
            x = causal_conv_step(y.reshape(N, H, E), c, d["weight"], d["bias"])
            outs.append(selective_scan_step(x, x * 0.5, s, d["A"], d["B"][:, :, t], d["C"][:, :, t], d["D"], h[:, :, t],
                                            d["delta_bias"])[:, :, None])
    check(torch.cat(outs, 2), whole.cpu().double(), "out")
    check(c, cs.cpu().double(), "conv state")
    check(s, ss.cpu().double(), "scan state")


def test_another_stream_and_repeated_calls_give_the_same_bits():
    a, m, go, gl = scan_case(3, 2, 70, 40, 16, 1, dtype=torch.bfloat16, keep=True, lengths=[70, 33, 5])
    d = {k: place(v).requires_grad_() for k, v in a.items()}
    md = {k: v.to(DEV) for k, v in m.items()}
    gd = (place(go), gl.to(DEV))

    def once():
        out, last = selective_scan(**d, **md)
        return [out, last, *torch.autograd.grad((out, last), list(d.values()), gd)]
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(first, second, once()):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_replays_from_a_captured_graph():
    """Forward and backward of convolution and scan, captured once and replayed on new inputs in place."""
    N, H, L, E, S = 2, 2, 50, 24, 16
    a, m, go, gl = scan_case(N, H, L, E, S, 1, lengths=[50, 20])
    ca, _, _, _ = conv_case(N, H, L, E, 4)
    d = {k: place(v) for k, v in a.items()}
    c = {k: place(v) for k, v in ca.items()}
    ln, god, gld = m["lengths"].to(DEV), place(go), gl.to(DEV)

    def step():
        leaves = {k: v.detach().requires_grad_() for k, v in d.items() if k != "u"}
        cl = {k: v.detach().requires_grad_() for k, v in c.items()}
        x, _ = causal_conv(cl["x"], cl["weight"], cl["bias"], cl["state"], None, ln)
        out, last = selective_scan(x, leaves["delta"], leaves["A"], leaves["B"], leaves["C"], leaves["D"], leaves["z"],
                                   leaves["delta_bias"], leaves["state"], None, ln)
        return [out, last, *torch.autograd.grad((out, last), [*leaves.values(), *cl.values()], (god, gld))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    g = torch.Generator().manual_seed(11)
    for k in range(3):
        c["x"].copy_(torch.randn(c["x"].shape, generator=g))
        d["state"].copy_(torch.randn(d["state"].shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in res]
        for x, y in zip(got, step()):
            assert torch.equal(x, y), k


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_is_refused_while_an_eager_graph_holds_the_leaves():
    """A backward captured then would end the process; the forward raises in front of any launch, and with the eager graph
    gone the same leaves can be captured."""
    a, _, go, _ = scan_case(2, 2, 20, 8, 16, 1)
    d = {k: place(v) for k, v in a.items()}
    w, b = torch.randn(2, 8, 4, device=DEV), torch.randn(16, device=DEV)
    calls = {"selective_scan": (lambda t: selective_scan(**{**d, "A": t})[0], d["A"]),
             "causal_conv": (lambda t: causal_conv(d["u"], t)[0], w),
             "residual_rms_norm": (lambda t: residual_rms_norm(d["B"], d["C"], t)[0], b)}
    for name, (call, t) in calls.items():
        leaf = t.detach().requires_grad_()
        held = call(leaf)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=name + ": a stream is being captured"):
            with torch.cuda.graph(graph):
                call(leaf)
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):     # without gradients there is nothing to join
            still = call(leaf)
        graph.replay()
        assert torch.equal(still, held), name
        g = torch.randn_like(held)
        want, = torch.autograd.grad(held, leaf, g)
        del held
        side = torch.cuda.Stream()                         # warm-up, as usual in front of a capture
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call(leaf), leaf, g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(call(leaf), leaf, g)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


def test_second_derivatives_are_refused():
    """With a graph of the gradients recorded they have the same values, and a derivative of them raises."""
    a, _, go, _ = scan_case(1, 2, 20, 8, 16, 1)
    d = {k: place(v) for k, v in a.items()}
    w, b = torch.randn(2, 8, 4, device=DEV), torch.randn(16, device=DEV)
    calls = {"selective_scan": (lambda t: selective_scan(**{**d, "u": t})[0], d["u"]),
             "causal_conv": (lambda t: causal_conv(t, w)[0], d["u"]),
             "residual_rms_norm": (lambda t: residual_rms_norm(t, t, b)[0], torch.randn(5, 16, device=DEV))}
    for name, (call, t) in calls.items():
        leaf = t.detach().requires_grad_()
        out = call(leaf)
        first, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        plain, = torch.autograd.grad(call(leaf), leaf, 2 * out.detach())
        assert torch.equal(first.detach(), plain), name
        with pytest.raises(RuntimeError, match=name + " has no second derivative"):
            (call(leaf).sum() + first.square().sum()).backward()       # a penalty on the gradient next to a loss


def test_second_derivatives_of_chosen_tensors_are_refused():
    """Asked for the derivative of a gradient by some tensors only, autograd follows the paths to them: there is one to every
    tensor that the gradient was computed from."""
    a, _, _, _ = scan_case(1, 2, 20, 8, 16, 1)
    d = {k: place(v) for k, v in a.items()}
    conv = dict(x=d["u"], weight=torch.randn(2, 8, 4, device=DEV), bias=torch.randn(2, 8, device=DEV))
    norm = dict(x=torch.randn(5, 16, device=DEV), residual=torch.randn(5, 16, device=DEV), weight=torch.randn(16, device=DEV))
    for op, args in ((selective_scan, d), (causal_conv, conv), (residual_rms_norm, norm),
                     (residual_rms_norm, {**norm, "residual": None})):
        leaves = {k: v.detach().requires_grad_() for k, v in args.items() if v is not None}
        out = op(**{**args, **leaves})[0]
        g = torch.randn_like(out).requires_grad_()
        for k, by in leaves.items():
            first, = torch.autograd.grad(out, by, g, create_graph=True)
            for second in [*leaves.values(), g]:
                with pytest.raises(RuntimeError, match=op.__name__ + " has no second derivative"):
                    torch.autograd.grad(first.sum(), second, allow_unused=True, retain_graph=True)
    w = norm["weight"]
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.functional.hessian(lambda t: residual_rms_norm(t, None, w)[0].sum(), norm["x"])


def test_gradients_with_tangents_are_refused():
    """Forward mode over the backward: a gradient that comes in with a tangent raises instead of losing it."""
    import torch.autograd.forward_ad as forward_ad
    a, _, go, _ = scan_case(1, 2, 20, 8, 16, 1)
    d = {k: place(v) for k, v in a.items()}
    w, b = torch.randn(2, 8, 4, device=DEV), torch.randn(16, device=DEV)
    calls = {"selective_scan": (lambda t: selective_scan(**{**d, "u": t})[0], d["u"]),
             "causal_conv": (lambda t: causal_conv(t, w)[0], d["u"]),
             "residual_rms_norm": (lambda t: residual_rms_norm(t, t, b)[0], torch.randn(5, 16, device=DEV))}
    for name, (call, t) in calls.items():
        leaf = t.detach().requires_grad_()
        out = call(leaf)
        g = torch.randn_like(out)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match=name + " has no derivative in forward mode"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(g, g))


def test_offsets_past_32_bits():
    """Rows whose elements lie further than 2^32 bytes (and 2^31 elements) apart."""
    H, E, S, L = 1, 16, 16, 5
    far = (1 << 31) // 4 + 64                                  # elements between two steps: 4 of them pass 2^31
    store = torch.empty(far * (L - 1) + E, device=DEV, dtype=torch.bfloat16)
    u = store.as_strided((1, H, L, E), (1, E, far, 1))
    a, m, go, gl = scan_case(1, H, L, E, S, 1, dtype=torch.bfloat16)
    u.copy_(a["u"])
    d = {k: place(v) for k, v in a.items()}
    near = selective_scan(**d)
    wide = selective_scan(**{**d, "u": u})
    assert torch.equal(near[0], wide[0]) and torch.equal(near[1], wide[1])
    ca, _, _, _ = conv_case(1, H, L, E, 4, dtype=torch.bfloat16)
    c = {k: place(v) for k, v in ca.items()}
    u.copy_(c["x"])
    assert torch.equal(causal_conv(**c)[0], causal_conv(**{**c, "x": u})[0])


@pytest.mark.parametrize("gate", [True, False])
def test_gradients_of_rows_past_32_bits(gate):
    """The backward on rows whose 16 steps span 2 GiB and more, of different lengths, with resets, cut into segments whose last
    blocks are partial: the same bits as on compact rows."""
    N, H, L, E, S, W = 2, 1, 70, 16, 16, 4
    far = (1 << 26) + 64                                       # elements between two steps: 16 of them pass 2^31 bytes
    store = torch.empty(far * (L - 1) + 8 * E * N, device=DEV, dtype=torch.bfloat16)
    views = iter(store.as_strided((N, H, L, E), (E, E, far, 1), k * E * N) for k in range(8))

    def spread(t):
        v = next(views)
        v.copy_(t)
        return v
    a, m, go, gl = scan_case(N, H, L, E, S, 1, dtype=torch.bfloat16, gate=gate, keep=True, lengths=[L, 45])
    near = {k: place(v) for k, v in a.items() if v is not None}
    wide = {k: spread(v) if k in ("u", "delta", "z") else v for k, v in near.items()}
    mask = {k: v.to(DEV) for k, v in m.items()}
    results = []
    for d, g in ((near, place(go)), (wide, spread(go))):
        leaves = {k: v.detach().requires_grad_() for k, v in d.items()}
        out, last = selective_scan(**leaves, **mask)
        results.append((out, last, *torch.autograd.grad((out, last), list(leaves.values()), (g, gl.to(DEV)))))
    assert all(torch.equal(x, y) for x, y in zip(*results))
    a, m, go, gl = conv_case(N, H, L, E, W, dtype=torch.bfloat16, keep=True, lengths=[L, 45])
    near = {k: place(v) for k, v in a.items()}
    wide = {**near, "x": spread(near["x"])}
    mask = {k: v.to(DEV) for k, v in m.items()}
    results = []
    for d, g in ((near, place(go)), (wide, spread(go))):
        leaves = {k: v.detach().requires_grad_() for k, v in d.items()}
        out, last = causal_conv(**leaves, **mask)
        results.append((out, last, *torch.autograd.grad((out, last), list(leaves.values()), (g, gl.to(DEV)))))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_scan_refuses_a_forward_that_no_backward_could_follow():
    """N G L S beyond 2^30, with gradients recorded; the long axes are broadcast ones."""
    wide = lambda *s: torch.ones(*s, device=DEV)
    u, b = wide(32, 1, 1, 1).expand(32, 1, 1 << 20, 1), wide(32, 1, 1, 64).expand(32, 1, 1 << 20, 64)
    A = -wide(1, 1, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="sizes beyond what the kernels take"):
        selective_scan(u, u, A, b, b)


def test_conv_of_more_workgroups_than_a_row_of_the_grid():
    """2^23 rows of one step and 128 channels: what the forward takes, the backward takes.  All numbers are whole and below 2^24,
    so that the sums are exact."""
    N, E, W = 1 << 23, 128, 2
    x = torch.arange(E, device=DEV).remainder(2).to(torch.bfloat16).view(1, 1, 1, E).expand(N, 1, 1, E).requires_grad_()
    w = torch.tensor([3.0, 2.0], device=DEV).expand(1, E, W).contiguous().requires_grad_()
    bias = torch.ones(1, E, device=DEV).requires_grad_()
    out, last = causal_conv(x, w, bias, silu=False)
    g = torch.ones(1, 1, 1, E, device=DEV, dtype=torch.bfloat16).expand(N, 1, 1, E)
    with torch.no_grad():
        first = x[0, 0, 0].float()
        assert bool((out == (1 + 2 * first)).all()) and bool((last == first).all())
        del last
    gx, gw, gb = torch.autograd.grad(out, (x, w, bias), g)
    assert bool((gx == 2).all())
    assert torch.equal(gw[0, :, 1], N * first) and not gw[0, :, 0].any() and bool((gb == N).all())


def test_empty_calls():
    z = lambda *s: torch.zeros(*s, device=DEV)
    state = torch.randn(2, 1, 4, 16, device=DEV)
    out, last = selective_scan(z(2, 1, 0, 4), z(2, 1, 0, 4), z(1, 4, 16), z(2, 1, 0, 16), z(2, 1, 0, 16), state=state)
    assert out.shape == (2, 1, 0, 4) and torch.equal(last, state)
    leaf = state.clone().requires_grad_()
    _, last = selective_scan(z(2, 1, 0, 4), z(2, 1, 0, 4), z(1, 4, 16), z(2, 1, 0, 16), z(2, 1, 0, 16), state=leaf)
    g = torch.randn_like(state)
    assert torch.equal(torch.autograd.grad(last, leaf, g)[0], g)
    cs = torch.randn(2, 1, 3, 4, device=DEV)
    out, last = causal_conv(z(2, 1, 0, 4), z(1, 4, 4), state=cs)
    assert out.shape == (2, 1, 0, 4) and torch.equal(last, cs)
    assert selective_scan(z(0, 1, 3, 4), z(0, 1, 3, 4), z(1, 4, 16), z(0, 1, 3, 16), z(0, 1, 3, 16))[0].shape == (0, 1, 3, 4)
