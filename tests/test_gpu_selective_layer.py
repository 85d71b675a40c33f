"""The selective state-space layers on the GPU: against the same layer written from the oracle's operators in 64 bits, and
their forms (segments, unrolls, single tokens, padded batches, 8-bit projection) against each other.

Tolerance of the float32 layers: each of the seven operators in a row (norm, four projections, convolution, scan) holds
1e-5 of its largest value, so a result and its gradients hold 1e-4."""
import copy

import pytest
import torch
import torch.nn.functional as F

from layer import SelectiveLayer, SelectiveStack
from oracle import selective

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 1e-4


def close(got, want, name, tol=TOL):
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    err = float((got - want).abs().max()) / max(float(want.abs().max()), 1e-30)
    assert got.shape == want.shape and err < tol, f"{name}: {err:.3g}"


def plain_mix(p, layer, h, residual, keep=None, lengths=None):
    """mix() in float64 from parameters p (name -> tensor)."""
    L, B, _ = h.shape
    H, d, S, G, r = layer.num_head, layer.dim_head, layer.d_state, layer.groups, layer.dt_rank
    heads = lambda t: t.reshape(L, B, H, d).permute(1, 2, 0, 3)
    rows = lambda t: t.permute(2, 0, 1, 3).reshape(L, B, H * d)
    y, total = selective.rms_norm(h, residual, p["norm_weight"], layer.eps)
    xz = F.linear(y, p["in_linear.weight"])
    x, z = heads(xz[..., :H * d]), heads(xz[..., H * d:])
    x, _ = selective.conv(x, p["conv_weight"], p["conv_bias"], None, keep, lengths)
    q = F.linear(rows(x), p["x_linear.weight"])
    dt = heads(F.linear(q[..., :r], p["dt_linear.weight"]))
    Bm, Cm = (t.reshape(L, B, G, S).permute(1, 2, 0, 3) for t in (q[..., r:r + G * S], q[..., r + G * S:]))
    out, _ = selective.scan(x, dt, -torch.exp(p["A_log"]), Bm, Cm, p["D"], z, p["dt_bias"], None, keep, lengths)
    return F.linear(rows(out), p["out_linear.weight"]), total


def make(seed=0, **kw):
    torch.manual_seed(seed)
    layer = SelectiveLayer(4, 8, 24, 0.0, **kw).to(DEV)
    with torch.no_grad():
        for q in (layer.A_log, layer.D, layer.norm_weight, layer.conv_bias):
            q.add_(0.1 * torch.randn_like(q))
    return layer


@pytest.mark.parametrize("kw", [dict(), dict(groups=2, d_state=8, d_conv=3), dict(groups=4, d_state=20, d_conv=2, dt_rank=3)], ids=str)
def test_layer_and_gradients_against_the_oracle(kw):
    layer = make(**kw)
    g = torch.Generator().manual_seed(1)
    h = torch.randn(19, 3, 24, generator=g)
    go = torch.randn(19, 3, 24, generator=g)
    lengths = torch.tensor([19, 7, 1], dtype=torch.int32)
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in layer.named_parameters()}
    hd = h.double().requires_grad_()
    want = hd + plain_mix(p, layer, hd, None, None, lengths)[0]
    grads = torch.autograd.grad(want, [hd, *p.values()], go.double())
    hg = h.to(DEV).requires_grad_()
    out = layer(hg, lengths=lengths.to(DEV))
    close(out, want, "out")
    got = torch.autograd.grad(out, [hg, *layer.parameters()], go.to(DEV))
    for k, a, b in zip(["h", *p], got, grads):
        close(a, b, "g_" + k)


def test_stack_and_gradients_against_the_oracle():
    torch.manual_seed(3)
    stack = SelectiveStack(2, 2, 8, 16, 0.0).to(DEV)
    g = torch.Generator().manual_seed(4)
    h, go = torch.randn(11, 2, 16, generator=g), torch.randn(11, 2, 16, generator=g)
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in stack.named_parameters()}
    x, residual = h.double().requires_grad_(), torch.zeros(11, 2, 16, dtype=torch.float64)
    h0 = x
    for i, layer in enumerate(stack.layers):
        mine = {k.split(".", 2)[2]: v for k, v in p.items() if k.startswith(f"layers.{i}.")}
        x, residual = plain_mix(mine, layer, x, residual)
    want = selective.rms_norm(x, residual, p["norm_weight"], stack.eps)[0]
    hg = h.to(DEV).requires_grad_()
    out, _ = stack(hg)
    close(out, want, "out")
    grads = torch.autograd.grad(want, [h0, *p.values()], go.double())
    got = torch.autograd.grad(out, [hg, *stack.parameters()], go.to(DEV))
    for k, a, b in zip(["h", *p], got, grads):
        close(a, b, "g_" + k)


def test_segments_unrolls_and_tokens_agree():
    """One call, two calls with the state carried, an unroll with resets, and single tokens on the same rows."""
    layer = make(2)
    h = torch.randn(21, 3, 24, generator=torch.Generator().manual_seed(5)).to(DEV)
    notdone = torch.ones(21, 3, device=DEV)
    notdone[0] = notdone[8, 1] = notdone[20, 2] = 0
    with torch.no_grad():
        whole, end = layer(h, get_state=True)
        first, state = layer(h[:9], get_state=True)
        second, state = layer(h[9:], state, get_state=True)
        close(torch.cat((first, second)), whole, "segments")
        close(state[1], end[1], "scan state")
        assert torch.equal(state[0], end[0])
        unroll, ustate = layer.forward_steps(h, notdone, tuple(torch.randn_like(s) for s in end))
        state = layer.start(3, DEV)
        tokens = [layer.step(h[t], state, notdone[t].contiguous()) for t in range(21)]
        close(torch.stack(tokens), unroll, "tokens")
        close(state[1], ustate[1], "scan state of the tokens")
    close(unroll[:8], whole[:8], "rows in front of the first reset")
    lengths = torch.tensor([21, 4, 0], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        padded, pstate = layer(h, get_state=True, lengths=lengths)
        short, sstate = layer(h[:4, 1:2], get_state=True)
    close(padded[:4, 1:2], short, "padded row")
    close(pstate[1][1:2], sstate[1], "state of the padded row")
    assert torch.equal(padded[4:, 1], h[4:, 1])            # behind a row's end the layer adds nothing


def test_bf16_layer_runs_and_is_near_the_float32_one():
    layer = make(6)
    h = torch.randn(33, 2, 24, generator=torch.Generator().manual_seed(7)).to(DEV)
    with torch.no_grad():
        want = layer(h)
    low = make(6).to(torch.bfloat16)
    x = h.bfloat16().requires_grad_()
    out = low(x)
    # seven roundings to bfloat16 in a row, half a step of 2^-8 of the largest value each
    close(out, want, "out", 7 * 2.0 ** -8)
    out.float().square().sum().backward()
    assert all(torch.isfinite(q.grad).all() for q in low.parameters()) and torch.isfinite(x.grad).all()


def test_eight_bit_projection():
    """The rows of the norm and the weight are rounded to e4m3: each factor of the projection is off by at most half a step,
    2^-4 of itself, so a product by 2 * 2^-4 (and their product), and a projected value by that share of the sum of its
    terms' sizes; float32 accumulation and the bfloat16 result (2^-8) add to it."""
    torch.manual_seed(8)
    layer = SelectiveLayer(4, 16, 32, 0.0).to(DEV).to(torch.bfloat16).serve_e4m3()
    for rows in (1, 3, 16, 100):
        h = torch.randn(rows, 2, 32, generator=torch.Generator().manual_seed(rows)).to(DEV).bfloat16()
        with torch.no_grad():
            got, total = layer._project_in(h, None)
            y, _ = selective.rms_norm(h.cpu().double(), None, layer.norm_weight.detach().cpu().double(), layer.eps)
            w = layer.in_linear.weight.detach().cpu().double()
            want, size = F.linear(y, w), F.linear(y.abs(), w.abs())
            bound = size * (2 * 2.0 ** -4 + 2.0 ** -8 + 1e-3) + want.abs() * 2.0 ** -8
            # values below the smallest normal number of e4m3 are off by 2^-10 of the row's scale at most
            bound = bound + 2.0 ** -10 / 448 * (F.linear(y.abs().amax(-1, keepdim=True).expand_as(y), w.abs())
                                                + F.linear(y.abs(), w.abs().amax(1, keepdim=True).expand_as(w)))
            assert torch.equal(total, h)
            assert float(((got.cpu().double() - want).abs() - bound).max()) <= 0
            assert layer(h).shape == h.shape
            state = layer.start(2, DEV, torch.bfloat16)
            assert torch.isfinite(layer.step(h[0], state)).all()
    out = layer(h)                                         # with gradients recorded the 16-bit projection runs
    assert out.requires_grad
    with pytest.raises(ValueError, match="divisible"):
        SelectiveLayer(1, 4, 24, 0.0).serve_e4m3()


def test_eight_bit_projection_follows_its_weight():
    """A weight that is stepped, loaded, replaced, converted or copied is not served from its old 8-bit form."""
    fresh = lambda layer: SelectiveLayer(2, 16, 32, 0.0).to(DEV).to(layer.in_linear.weight.dtype)
    h = torch.randn(5, 2, 32, generator=torch.Generator().manual_seed(3)).to(DEV)

    @torch.no_grad()
    def served_as_it_is(layer, name):
        x = h.to(layer.in_linear.weight.dtype)
        other = fresh(layer)
        other.load_state_dict(layer.state_dict())
        assert torch.equal(layer(x), other.serve_e4m3()(x)), name
    torch.manual_seed(12)
    layer = SelectiveLayer(2, 16, 32, 0.0).to(DEV).serve_e4m3()
    served_as_it_is(layer, "as made")
    opt = torch.optim.SGD(layer.parameters(), lr=0.1)
    layer(h).square().sum().backward()
    opt.step()
    served_as_it_is(layer, "stepped")
    layer.load_state_dict(fresh(layer).state_dict())
    served_as_it_is(layer, "loaded")
    layer.in_linear.weight = torch.nn.Parameter(torch.randn_like(layer.in_linear.weight))
    served_as_it_is(layer, "replaced")
    twin = copy.deepcopy(layer)
    with torch.no_grad():
        twin.in_linear.weight.mul_(-0.5)
    served_as_it_is(twin, "copied and changed")
    served_as_it_is(layer, "the copy's origin")
    served_as_it_is(layer.to(torch.bfloat16), "converted")
    served_as_it_is(SelectiveLayer(2, 16, 32, 0.0).serve_e4m3().to(DEV), "moved")


def test_stack_steps_equal_the_stack():
    torch.manual_seed(9)
    stack = SelectiveStack(2, 2, 16, 32, 0.0).to(DEV)
    h = torch.randn(9, 3, 32, generator=torch.Generator().manual_seed(10)).to(DEV)
    with torch.no_grad():
        whole, _ = stack(h)
        states = [layer.start(3, DEV) for layer in stack.layers]
        steps = torch.stack([stack.step(h[t], states) for t in range(9)])
    close(steps, whole, "steps")


def test_replays_follow_the_8_bit_weight():
    """A graph captured with the 8-bit projection gives what the layer gives, also once the weight was stepped, loaded or
    replaced and the layer called (or serve_e4m3) in between."""
    torch.manual_seed(14)
    layer = SelectiveLayer(2, 16, 32, 0.0).to(DEV).to(torch.bfloat16).serve_e4m3()
    h = torch.randn(5, 3, 32, generator=torch.Generator().manual_seed(15)).to(DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        layer(h)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = layer(h)

    def load():
        layer.load_state_dict({**layer.state_dict(), "in_linear.weight": torch.randn_like(layer.in_linear.weight)})

    def step():
        with torch.no_grad():
            layer.in_linear.weight.mul_(-1.5)

    def replace():
        layer.in_linear.weight = torch.nn.Parameter(torch.randn_like(layer.in_linear.weight))
    for change in (lambda: None, step, load, replace, step):
        change()
        with torch.no_grad():
            want = layer(h)
        junk = [torch.full((64, 32), 1e4, device=DEV).to(torch.float8_e4m3fn) for _ in range(4)]   # where a freed weight lay
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del junk
    step()
    layer.serve_e4m3()
    graph.replay()
    with torch.no_grad():
        assert torch.equal(out, layer(h))


def test_the_8_bit_weight_is_not_converted_in_a_capture():
    """Recorded into a graph, the conversion would not have run when the next eager call takes the weight for converted."""
    h = torch.randn(5, 3, 32, generator=torch.Generator().manual_seed(16)).to(DEV).bfloat16()
    torch.manual_seed(17)
    layer = SelectiveLayer(2, 16, 32, 0.0).to(DEV).to(torch.bfloat16).serve_e4m3()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        layer(h)
    torch.cuda.current_stream().wait_stream(side)
    twin = copy.deepcopy(layer)                            # has no 8-bit weight yet
    with torch.no_grad():
        layer.in_linear.weight.mul_(-0.5)
        twin.in_linear.weight.mul_(-0.5)
    for each in (layer, twin):
        for call in (lambda: each(h), each.serve_e4m3):
            with pytest.raises(RuntimeError, match="while a stream is being captured"):
                with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
                    call()
        with torch.no_grad():
            want = each(h)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = each(h)
            for _ in range(3):
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want)


def test_the_8_bit_weight_is_ready_for_other_streams():
    """Converted on a stream that is busy, then used on another one without a wait between them."""
    torch.manual_seed(18)
    layer = SelectiveLayer(2, 16, 32, 0.0).to(DEV).to(torch.bfloat16).serve_e4m3()
    h = torch.randn(5, 3, 32, generator=torch.Generator().manual_seed(19)).to(DEV).bfloat16()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.no_grad():
            layer(h)
            layer.in_linear.weight.copy_(torch.randn_like(layer.in_linear.weight))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            layer.serve_e4m3()
        with torch.no_grad():
            got = layer(h)
            side.synchronize()
            want = SelectiveLayer(2, 16, 32, 0.0).to(DEV).to(torch.bfloat16)
            want.load_state_dict(layer.state_dict())
            assert torch.equal(got, want.serve_e4m3()(h))


@pytest.mark.parametrize("rows,weights", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)], ids=str)
def test_eight_bit_projection_with_rows_of_another_type(rows, weights):
    """The projection's result has the type of the layer's weights, in 8 bits as in 16 or 32: the same calls run, and their
    states have the same types."""
    torch.manual_seed(20)
    layer = SelectiveLayer(2, 16, 32, 0.0).to(DEV).to(weights)
    stack = SelectiveStack(2, 2, 16, 32, 0.0).to(DEV).to(weights)
    h = torch.randn(9, 3, 32, generator=torch.Generator().manual_seed(21)).to(DEV).to(rows)
    with torch.no_grad():
        want, state = layer(h, get_state=True)
        swant, sstates = stack(h)
        layer.serve_e4m3(), stack.serve_e4m3()
        got, state8 = layer(h, get_state=True)
        sgot, sstates8 = stack(h)
        assert torch.isfinite(layer.step(h[0], layer.start(3, DEV, weights))).all()
        assert torch.isfinite(stack.step(h[0], [each.start(3, DEV, weights) for each in stack.layers])).all()
    for a, b in [(got, want), (sgot, swant), *zip(state8, state), *((x, y) for p, q in zip(sstates8, sstates) for x, y in zip(p, q))]:
        assert a.dtype == b.dtype and a.shape == b.shape and torch.isfinite(a).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_capture_is_refused_while_an_eager_graph_holds_a_parameter(dtype):
    """The layer hands its parameters to the operators converted, or to its projections: they are found behind the inputs."""
    layer = make(22).to(dtype)
    stack = SelectiveStack(2, 2, 16, 32, 0.0).to(DEV).to(dtype)
    h = torch.randn(7, 2, 24, generator=torch.Generator().manual_seed(23)).to(DEV).to(dtype)
    hs = torch.randn(7, 2, 32, generator=torch.Generator().manual_seed(24)).to(DEV).to(dtype)
    for model, x in ((layer, h), (stack, hs)):
        side = torch.cuda.Stream()                         # warm-up: the projections' library makes its handles
        side.wait_stream(torch.cuda.current_stream())
        with torch.no_grad(), torch.cuda.stream(side):
            model(x)
        torch.cuda.current_stream().wait_stream(side)
        for held in model.parameters():                    # each of them alone
            eager = held * 2
            with pytest.raises(RuntimeError, match="a stream is being captured"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    model(x)
            with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
                model(x)
            del eager
        side = torch.cuda.Stream()                         # held by a graph of a side stream: may be joined
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = model(x)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            model(x)
        del eager


def test_capture_is_refused_for_leaves_behind_the_inputs():
    """A leaf that reaches an operator through other operations counts as its leaf."""
    from residual_norm import residual_rms_norm
    leaf, w = torch.randn(4, 16, device=DEV).requires_grad_(), torch.randn(16, device=DEV)
    eager = leaf.exp()
    with pytest.raises(RuntimeError, match="residual_rms_norm: a stream is being captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            residual_rms_norm(-torch.exp(leaf.double().float()), None, w)
    del eager
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        residual_rms_norm(-torch.exp(leaf.double().float()), None, w)


def test_stack_with_resets_equals_its_parts():
    """keep is (batch, steps): a row with a reset is the two sequences in front of it and behind it."""
    torch.manual_seed(25)
    stack = SelectiveStack(2, 2, 16, 32, 0.0).to(DEV)
    h = torch.randn(9, 3, 32, generator=torch.Generator().manual_seed(26)).to(DEV)
    keep = torch.ones(3, 9, device=DEV)
    keep[1, 4] = 0
    with torch.no_grad():
        out, states = stack(h, keep=keep)
        plain, plain_states = stack(h)
        front, _ = stack(h[:4])
        back, back_states = stack(h[4:])
        step_states = [layer.start(3, DEV) for layer in stack.layers]
        steps = torch.stack([stack.step(h[t], step_states, keep[:, t].contiguous()) for t in range(9)])
    close(out[:, [0, 2]], plain[:, [0, 2]], "rows without a reset")
    close(out[:4, 1], front[:, 1], "in front of the reset")
    close(out[4:, 1], back[:, 1], "behind the reset")
    close(steps, out, "single tokens")
    for a, b, c, d in zip(states, back_states, plain_states, step_states):
        for k in range(2):
            close(a[k][1], b[k][1], "state behind the reset")
            close(a[k][0], c[k][0], "state without a reset")
            close(d[k], a[k], "state of the single tokens")
    with pytest.raises(ValueError, match="keep"):
        stack(h, keep=keep.t())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_training_step_replays_from_a_captured_graph(dtype):
    layer = make(27).to(dtype)
    g = torch.Generator().manual_seed(28)
    h, go = (torch.randn(33, 2, 24, generator=g).to(DEV).to(dtype) for _ in range(2))
    leaves = list(layer.parameters())

    def step():
        out = layer(h)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        with torch.no_grad():
            h.copy_(torch.randn(33, 2, 24, generator=g))
        for t in got:
            t.zero_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for name, a, b in zip(["out", *(n for n, _ in layer.named_parameters())], got, want):
            assert torch.equal(a, b), (k, name)
        del want
