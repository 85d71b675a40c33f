"""What the selective-scan, convolution and norm operators refuse, checked without a GPU: the C entry points reject bad
arguments before they touch the device (placeholder pointers are never dereferenced), the host layer before it calls them."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

P = ctypes.c_void_p
I3 = ctypes.c_int64 * 3


def fake():
    return P(0x1000)


def test_scan_argument_validation():
    import srwm_hip
    L = srwm_hip.lib()
    N, H, T, E, S, G = 2, 4, 8, 16, 16, 2
    ok, okb = I3(H * T * E, T * E, E), I3(G * T * S, T * S, S)

    def forward(u=fake(), us=ok, z=P(None), zs=None, A=fake(), os=ok, last=fake(), n=N, h=H, s=S, g=G, flags=0, fn=None):
        fn = fn or L.selective_scan_forward_f32
        return fn(u, us, fake(), ok, z, zs, fake(), okb, fake(), okb, A, fake(), fake(), fake(), P(None), P(None), fake(), os,
                  last, P(None), P(None), n, h, T, E, s, g, flags, P(None))
    for fn in (L.selective_scan_forward_f32, L.selective_scan_forward_bf16):
        assert forward(u=P(None), fn=fn) == -1
        assert forward(us=None, fn=fn) == -1
        assert forward(z=fake(), fn=fn) == -1                       # a gate comes with its strides
        assert forward(last=P(None), fn=fn) == -1
        assert forward(n=0, fn=fn) == -1
        assert forward(h=3, fn=fn) == -1                            # 3 heads in 2 groups
        assert forward(g=0, fn=fn) == -1
        assert forward(s=0, fn=fn) == -1
        assert forward(flags=16, fn=fn) == -1
        assert forward(s=65, fn=fn) == -2
        assert forward(n=(1 << 23) + 1, fn=fn) == -2                    # more workgroups than a launch takes
        assert forward(us=I3(1 << 41, E, E), fn=fn) == -3
        assert forward(os=I3(0, T * E, E), fn=fn) == -3             # rows of out on top of each other
        assert forward(A=P(0x1004), fn=fn) == -3                    # not 16-byte aligned

    def backward(saved=fake(), go=fake(), z=P(None), zs=None, gz=P(None), gus=ok, work=fake(), flags=0):
        return L.selective_scan_backward_bf16(fake(), ok, fake(), ok, z, zs, fake(), okb, fake(), okb, fake(), fake(), fake(),
                                              P(None), P(None), saved, go, ok, P(None), fake(), gus, fake(), ok, gz, zs, fake(),
                                              okb, fake(), okb, fake(), fake(), fake(), fake(), work, N, H, T, E, S, G, flags,
                                              P(None))
    assert backward(saved=P(None)) == -1
    assert backward(go=P(None)) == -1
    assert backward(z=fake(), zs=ok) == -1                          # the gate's gradient is not optional
    assert backward(work=P(None)) == -1
    assert backward(flags=srwm_hip.FLAG_SILU) == -1
    assert backward(gus=I3(H * T * E, T * E, 0)) == -3
    step = lambda state, s=S: L.selective_scan_step_f32(fake(), ok, fake(), ok, P(None), None, fake(), okb, fake(), okb, fake(),
                                                        P(None), P(None), P(None), state, fake(), ok, N, H, E, s, G, 0, P(None))
    assert step(P(None)) == -1 and step(P(0x1008)) == -3 and step(fake(), 65) == -2
    n = (ctypes.c_int64 * 1)()
    assert L.selective_scan_workspace(n, N, H, T, E, S, G, 1) == 0 and n[0] >= N * G * T * 2 * S
    assert L.selective_scan_workspace(None, N, H, T, E, S, G, 1) == -1 and L.selective_scan_workspace(n, N, H, T, E, 65, G, 1) == -2


def test_conv_and_norm_argument_validation():
    import srwm_hip
    L = srwm_hip.lib()
    N, H, T, E = 2, 4, 8, 16
    ok = I3(H * T * E, T * E, E)
    conv = lambda x=fake(), os=ok, w=4, last=fake(), flags=0, n=N: L.causal_conv_forward_bf16(
        x, ok, fake(), P(None), P(None), P(None), P(None), fake(), os, last, n, H, T, E, w, flags, P(None))
    assert conv(x=P(None)) == -1 and conv(last=P(None)) == -1 and conv(flags=1) == -1 and conv(w=0) == -1 and conv(n=0) == -1
    assert conv(w=1) == -2 and conv(w=5) == -2
    assert conv(os=I3(H * T * E, T * E, 1)) == -3
    back = lambda go=fake(), work=fake(): L.causal_conv_backward_f32(
        fake(), ok, fake(), P(None), P(None), P(None), P(None), go, ok, P(None), fake(), ok, fake(), P(None), P(None), work,
        N, H, T, E, 4, 0, P(None))
    assert back(go=P(None)) == -1 and back(work=P(None)) == -1
    assert L.causal_conv_step_f32(fake(), ok, fake(), P(None), P(None), P(None), fake(), ok, N, H, E, 4, 0, P(None)) == -1
    eps = (ctypes.c_float * 1)(1e-5)
    norm = lambda x=fake(), s=fake(), e=eps, rows=4, D=8, flags=0: L.residual_rms_norm_forward_bf16(
        x, fake(), fake(), fake(), s, P(None), e, rows, D, flags, P(None))
    assert norm(x=P(None)) == -1 and norm(s=P(None)) == -1 and norm(e=None) == -1 and norm(rows=0) == -1 and norm(D=0) == -1
    assert norm(flags=2) == -1 and norm(rows=(1 << 25) + 1) == -2 and norm(rows=(1 << 23) + 1, D=2049) == -2
    assert L.residual_rms_norm_e4m3_f32(fake(), P(None), fake(), fake(), P(None), P(None), eps, 4, 8, 0, P(None)) == -1
    nb = lambda D: L.residual_rms_norm_backward_f32(fake(), fake(), fake(), fake(), P(None), fake(), P(None), fake(), fake(), 4, D,
                                                    1, P(None))
    assert nb(8) == -1                                             # an unknown flag
    n = (ctypes.c_int64 * 1)()
    assert L.causal_conv_workspace(n, N, H, T, E, 4) == 0 and n[0] > 0
    assert L.residual_rms_norm_workspace(n, 4, 8) == 0 and n[0] > 0 and L.residual_rms_norm_workspace(n, 0, 8) == -1


def test_host_layer_refusals():
    from residual_norm import residual_rms_norm, residual_rms_norm_e4m3
    from selective_scan import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    z = torch.zeros
    with pytest.raises(RuntimeError, match="no CPU path"):
        selective_scan(z(1, 1, 2, 4), z(1, 1, 2, 4), z(1, 4, 16), z(1, 1, 2, 16), z(1, 1, 2, 16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        causal_conv(z(1, 1, 2, 4), z(1, 4, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        residual_rms_norm(z(2, 4), None, z(4))
    with pytest.raises(ValueError, match="groups"):
        selective_scan(z(1, 3, 2, 4), z(1, 3, 2, 4), z(3, 4, 16), z(1, 2, 2, 16), z(1, 2, 2, 16))
    with pytest.raises(ValueError, match="at least one state"):    # its output would be D u silu(z), not zeros
        selective_scan(z(1, 1, 2, 4), z(1, 1, 2, 4), z(1, 4, 0), z(1, 1, 2, 0), z(1, 1, 2, 0))
    with pytest.raises(ValueError, match="at least one state"):
        selective_scan_step(z(1, 1, 4), z(1, 1, 4), z(1, 1, 4, 0), z(1, 4, 0), z(1, 1, 0), z(1, 1, 0))
    with pytest.raises(ValueError, match="N, H, L, E"):
        selective_scan(z(1, 2, 4), z(1, 2, 4), z(1, 4, 16), z(1, 2, 16), z(1, 2, 16))
    with pytest.raises(TypeError, match="float32 or torch.bfloat16"):
        selective_scan(z(1, 1, 2, 4).half(), z(1, 1, 2, 4), z(1, 4, 16), z(1, 1, 2, 16), z(1, 1, 2, 16))
    with pytest.raises(TypeError):
        causal_conv(None, z(1, 4, 4))
    # the single-token forms and the 8-bit norm have no backward, and say so
    w = z(1, 4, 4).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        causal_conv_step(z(1, 1, 4), z(1, 1, 3, 4), w)
    with pytest.raises(RuntimeError, match="no backward"):
        selective_scan_step(z(1, 1, 4), z(1, 1, 4), z(1, 1, 4, 16), z(1, 4, 16).requires_grad_(), z(1, 1, 16), z(1, 1, 16))
    with pytest.raises(RuntimeError, match="no backward"):
        residual_rms_norm_e4m3(z(2, 4), None, z(4).requires_grad_())
    with pytest.raises(ValueError, match="no backward for rows longer"):
        residual_rms_norm(z(1, 16385), None, z(16385).requires_grad_())


def every_operator():
    """(operator, its arguments) for each one, on the CPU."""
    from residual_norm import residual_rms_norm, residual_rms_norm_e4m3
    from selective_scan import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    z = torch.zeros
    scan = dict(u=z(1, 1, 2, 4), delta=z(1, 1, 2, 4), A=z(1, 4, 16), B=z(1, 1, 2, 16), C=z(1, 1, 2, 16), D=z(1, 4), z=z(1, 1, 2, 4),
                delta_bias=z(1, 4), state=z(1, 1, 4, 16))
    step = dict(scan, **{k: scan[k][:, :, 0] for k in ("u", "delta", "B", "C", "z")})
    conv = dict(x=z(1, 1, 2, 4), weight=z(1, 4, 4), bias=z(1, 4), state=z(1, 1, 3, 4))
    norm = dict(x=z(2, 4), residual=z(2, 4), weight=z(4))
    return [(selective_scan, scan), (selective_scan_step, step), (causal_conv, conv),
             (causal_conv_step, dict(conv, x=z(1, 1, 4))), (residual_rms_norm, norm), (residual_rms_norm_e4m3, norm)]


def test_derivatives_in_forward_mode_are_refused():
    """A dual tensor asks for no gradient by itself: every operator raises for it, with and without gradients recorded."""
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level():
        for fn, args in every_operator():
            for k in args:
                dual = dict(args, **{k: forward_ad.make_dual(args[k], torch.ones_like(args[k]))})
                for recorded in (True, False):
                    with torch.set_grad_enabled(recorded):
                        with pytest.raises(RuntimeError, match=fn.__name__ + " has no derivative in forward mode"):
                            fn(**dual)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tracing_is_refused():
    """A trace would hold the call's allocations without its kernels."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    for fn, args in every_operator():
        error = pytest.raises(RuntimeError, match=fn.__name__ + " cannot be traced")
        call = lambda *t: fn(**dict(zip(args, t)))
        for recorded in (True, False):
            with torch.set_grad_enabled(recorded):
                with error:
                    torch.jit.trace(call, tuple(args.values()), check_trace=False)
                for mode in ("real", "fake"):
                    with error:
                        make_fx(call, tracing_mode=mode)(*args.values())
                with FakeTensorMode(allow_non_fake_inputs=True), error:
                    call(*args.values())


def test_output_rows_follow_the_input():
    import srwm_hip
    srwm_hip = srwm_hip.binding()
    x = torch.zeros(5, 3, 2 * 2 * 4).view(5, 3, 2, 2, 4)[:, :, 1].permute(1, 2, 0, 3)     # the second half of wider rows
    out = srwm_hip.rows_like(x)
    assert out.shape == (3, 2, 5, 4) and out.stride(-1) == 1
    assert out.permute(2, 0, 1, 3).is_contiguous()                                     # step-major, dense
    assert srwm_hip.rows_like(torch.zeros(3, 2, 5, 8)[..., ::2]).stride(-1) == 1
    assert srwm_hip.rows_like(torch.zeros(3, 2, 4, 5).transpose(2, 3)).stride(-1) == 1


def test_binding_is_loaded_at_the_first_call():
    """Importing the layers asks for no library: a missing binding raises where one of its operators is called."""
    code = ("import sys; sys.path.insert(0, 'modern-srwm_amd'); import srwm_hip; srwm_hip.BINDING_PATH = '/nonexistent.so'\n"
            "import torch, layer, residual_norm\n"
            "try: residual_norm.residual_rms_norm(torch.zeros(2, 4), None, torch.zeros(4))\n"
            "except RuntimeError as e: assert 'is missing' in str(e), e\n"
            "else: raise AssertionError('no error')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True, timeout=100)


def test_scan_limit_of_the_backward_is_known_in_front():
    """N G L S beyond 2^30: the forward runs, the backward's workspace cannot be asked for."""
    import srwm_hip
    n = (ctypes.c_int64 * 1)()
    size = lambda backward: srwm_hip.lib().selective_scan_workspace(n, 32, 1, 1 << 20, 1, 64, 1, backward)
    assert size(0) == 0 and size(1) == -2
