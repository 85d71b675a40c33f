"""Host side of libsrwm_hip.so: loads the C-ABI library with ctypes and exposes the four
extension-level functions with the positional tensor lists of the reference's pybind
modules (supervised_learning/self_ref_v0/self_ref_v0.cu:1344-1356,
supervised_learning/fast_weight/fast_weight_cuda.cu:667-679):

    self_ref_forward(x, W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff, beta_diff, out)
    self_ref_backward(x, q, k, beta, y_diff, q_diff, k_diff, beta_diff, grad_out,
                      W_y, W_q, W_k, w_b, grad_x, grad_W_y, grad_W_q, grad_W_k, grad_w_b)
    fast_weight_forward(q, k, v, beta, v_old, v_insert, kv, out)
    fast_weight_backward(q, k, v, beta, v_old, v_insert, grad_out, kv,
                         grad_q, grad_k, grad_v, grad_beta)

PyTorch is used for device memory and streams only.  There is no CPU path: a missing
library, a CPU tensor or a non-float32 tensor raises.
"""
import ctypes
import functools
import os
import subprocess

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_PKG = os.path.dirname(_HERE)
LIB_PATH = os.path.join(_PKG, "lib", "libsrwm_hip.so")
CSRC = os.path.join(_PKG, "csrc")

# flags of include/srwm_hip.h
GRAD_STATE_ZERO = 0
GRAD_STATE_IN = 1
GRAD_STATE_ACCUM = 2
FLAG_GENERIC = 16
FLAG_NO_FALLBACK = 8192    # raise where the register-resident kernels do not take the call instead of running the LDS-resident ones
FLAG_CHUNKWISE = 32     # delta forward: chunkwise MFMA kernel (E == M in {64, 128})
FLAG_EXACT_PRODUCTS = 512   # chunkwise kernels with bf16 inputs: every product from hi + lo operand pairs
FLAG_BF16_GRADS = 1024      # chunkwise delta backward with bf16 inputs: grad_q, grad_k, grad_v written as bf16 by the library
FLAG_SPARSE_V_OLD = 4096    # chunkwise delta forward: v_old only for steps with |beta| < 2^-24 (all a chunkwise backward reads of it)
FLAG_NORM_EPS = 2048        # delta_layer_prologue: 1e-5 added to the normalisers of q and k
FLAG_SOFTPLUS = 16384       # selective_scan: dt = softplus(delta + delta_bias)
FLAG_SILU = 32768           # causal_conv: silu behind the convolution
FLAG_RESIDUAL_F32 = 65536   # residual_rms_norm with bfloat16 rows: the residual and the sum are float32
FLAG_STATE_SHIFT = 64      # layer entry points: the state tensors hold W minus the shared weights
FLAG_FRESH_STATE = 128     # layer forward: start from the shared weights
FLAG_SOFTMAX_INPUT = 256   # layer entry points: x is given before its softmax

ABI_VERSION = 18

# True: a call that the register-resident kernels do not take (head size without an instantiation, misaligned
# base or strides) raises instead of running on the several times slower LDS-resident kernels
NO_FALLBACK = False

_lib = None

_F = ctypes.c_void_p      # device float*
_S = ctypes.POINTER(ctypes.c_int64)
_I = ctypes.c_int
_U = ctypes.c_uint

_SIGNATURES = {
    "srwm_forward_f32": [_F, _S] + [_F] * 12 + [_I] * 4 + [_U, ctypes.c_void_p],
    "srwm_forward_bf16": [_F, _S] + [_F] * 12 + [_I] * 4 + [_U, ctypes.c_void_p],
    "srwm_backward_bf16": [_F, _S] + [_F] * 7 + [_F, _S] + [_F] * 9 + [_I] * 4 + [_U, ctypes.c_void_p],
    "srwm_forward_wide_f32": [_F, _S] + [_F] * 12 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_backward_wide_f32": [_F, _S] + [_F] * 7 + [_F, _S] + [_F] * 9 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_layer_forward_f32": [_F, _S] + [_F] * 17 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_layer_backward_f32": [_F, _S] + [_F] * 7 + [_F, _S] + [_F] * 9 + [_S] + [_F] * 8 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_layer_backward_noalloc_f32": [_F, _S] + [_F] * 7 + [_F, _S] + [_F] * 9 + [_S] + [_F] * 4 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_layer_forward_bf16": [_F, _S] + [_F] * 17 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_layer_backward_bf16": [_F, _S] + [_F] * 7 + [_F, _S] + [_F] * 9 + [_S] + [_F] * 8 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_forward_steps_f32": [_F, _S] + [_F] * 17 + [_I] * 4 + [_U, ctypes.c_void_p],
    "srwm_readout_grad_wide_f32": [_F] * 5 + [_F, _S] + [_F] * 2 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_layer_readout_grad_f32": [_F, _S] + [_F] * 5 + [_F, _S] + [_F, _F, _S] + [_F] * 2 + [_I] * 5 + [_U, ctypes.c_void_p],
    "srwm_readout_grad_f32": [_F] * 5 + [_F, _S] + [_F] * 2 + [_I] * 4 + [_U, ctypes.c_void_p],
    "srwm_backward_f32": [_F, _S] + [_F] * 7 + [_F, _S] + [_F] * 9 + [_I] * 4 + [_U, ctypes.c_void_p],
    "delta_forward_steps_f32": [_F, _S] * 4 + [_F] * 5 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_readout_replay_f32": [_F, _S] + [_F, _F] + [_F, _S] + [_F, _F] + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_steps_backward_f32": [_F, _S] * 4 + [_F] * 3 + [_F, _S] + [_F] * 5 + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_forward_f32": [_F, _S] * 4 + [_F] * 4 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_backward_f32": [_F, _S] * 4 + [_F, _F] + [_F, _S] + [_F] * 6 + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_forward_bf16": [_F, _S] * 4 + [_F] * 4 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_backward_bf16": [_F, _S] * 4 + [_F, _F] + [_F, _S] + [_F] * 6 + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_layer_prologue_f32": [_F] * 6 + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_layer_prologue_grad_f32": [_F, _S] * 4 + [_F] * 5 + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_layer_prologue_bf16": [_F] * 6 + [_I] * 5 + [_U, ctypes.c_void_p],
    "delta_layer_prologue_grad_bf16": [_F, _S] * 4 + [_F] * 5 + [_I] * 5 + [_U, ctypes.c_void_p],
    "selective_scan_forward_f32": [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 7 + [_S] + [_F] * 3 + [_I] * 6 + [_U, ctypes.c_void_p],
    "selective_scan_forward_bf16": [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 7 + [_S] + [_F] * 3 + [_I] * 6 + [_U, ctypes.c_void_p],
    "selective_scan_backward_f32": [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 7 + [_S] + [_F] * 2 + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 5 + [_I] * 6 + [_U, ctypes.c_void_p],
    "selective_scan_backward_bf16": [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 7 + [_S] + [_F] * 2 + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 5 + [_I] * 6 + [_U, ctypes.c_void_p],
    "selective_scan_step_f32": [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 6 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "selective_scan_step_bf16": [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] + [_S] + [_F] * 6 + [_S] + [_I] * 5 + [_U, ctypes.c_void_p],
    "causal_conv_forward_f32": [_F] + [_S] + [_F] * 6 + [_S] + [_F] + [_I] * 5 + [_U, ctypes.c_void_p],
    "causal_conv_forward_bf16": [_F] + [_S] + [_F] * 6 + [_S] + [_F] + [_I] * 5 + [_U, ctypes.c_void_p],
    "causal_conv_backward_f32": [_F] + [_S] + [_F] * 6 + [_S] + [_F] * 2 + [_S] + [_F] * 4 + [_I] * 5 + [_U, ctypes.c_void_p],
    "causal_conv_backward_bf16": [_F] + [_S] + [_F] * 6 + [_S] + [_F] * 2 + [_S] + [_F] * 4 + [_I] * 5 + [_U, ctypes.c_void_p],
    "causal_conv_step_f32": [_F] + [_S] + [_F] * 5 + [_S] + [_I] * 4 + [_U, ctypes.c_void_p],
    "causal_conv_step_bf16": [_F] + [_S] + [_F] * 5 + [_S] + [_I] * 4 + [_U, ctypes.c_void_p],
    "residual_rms_norm_forward_f32": [_F] * 7 + [_I] * 2 + [_U, ctypes.c_void_p],
    "residual_rms_norm_forward_bf16": [_F] * 7 + [_I] * 2 + [_U, ctypes.c_void_p],
    "residual_rms_norm_e4m3_f32": [_F] * 7 + [_I] * 2 + [_U, ctypes.c_void_p],
    "residual_rms_norm_e4m3_bf16": [_F] * 7 + [_I] * 2 + [_U, ctypes.c_void_p],
    "residual_rms_norm_backward_f32": [_F] * 9 + [_I] * 2 + [_U, ctypes.c_void_p],
    "residual_rms_norm_backward_bf16": [_F] * 9 + [_I] * 2 + [_U, ctypes.c_void_p],
    "selective_scan_workspace": [_S] + [_I] * 7,
    "causal_conv_workspace": [_S] + [_I] * 5,
    "residual_rms_norm_workspace": [_S] + [_I] * 2,
}


def build(verbose=False):
    """Compile libsrwm_hip.so for gfx950 with hipcc (always recompiles)."""
    out = None if verbose else subprocess.DEVNULL
    subprocess.check_call(["make", "-C", CSRC, "-B", "-j8"], stdout=out, stderr=out)
    return LIB_PATH


def lib():
    """The loaded library.  Raises if it has not been built -- there is no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C {CSRC}` "
                "(or __graft_entry__.build()); the HIP kernels have no CPU/PyTorch fallback")
        L = ctypes.CDLL(LIB_PATH)
        L.srwm_hip_abi_version.restype = _I
        if L.srwm_hip_abi_version() != ABI_VERSION:
            raise RuntimeError("libsrwm_hip.so ABI version mismatch; rebuild the library")
        for name, args in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = _I
        L.srwm_hip_strerror.restype = ctypes.c_char_p
        L.srwm_hip_strerror.argtypes = [_I]
        L.srwm_hip_limits.argtypes = [ctypes.POINTER(_I)] * 3
        L.srwm_hip_limits.restype = _I
        L.srwm_hip_scratch_bytes.restype = ctypes.c_size_t
        L.srwm_hip_scratch_bytes.argtypes = []
        L.srwm_hip_fallback_calls.restype = ctypes.c_uint64
        L.srwm_hip_fallback_calls.argtypes = []
        _lib = L
    return _lib


def fallback_calls():
    """Calls since the library was loaded that the register-resident kernels did not take (head size, alignment) and the
    several times slower LDS-resident kernels served; calls that asked for those with FLAG_GENERIC are not counted."""
    return int(lib().srwm_hip_fallback_calls())


def limits(device=None):
    """(max E of SRWM forward, max E of SRWM backward, max E == M of the delta rule)."""
    a, b, c = _I(), _I(), _I()
    with torch.cuda.device(device):
        lib().srwm_hip_limits(ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
    return a.value, b.value, c.value


def _check(code, what):
    if code != 0:
        msg = lib().srwm_hip_strerror(code).decode()
        raise RuntimeError(f"{what} failed with code {code}: {msg}")


def _require(t, name, shape=None, dtype=torch.float32):
    # runs some twenty times per operator call, on a path that is host-bound for single-step calls:
    # only attribute reads and identity / tuple comparisons on the success path
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU (got {t.device}); there is no CPU path")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _fam(flags):
    return flags | FLAG_NO_FALLBACK if NO_FALLBACK and not flags & FLAG_GENERIC else flags


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def _rows_ok(t):
    """Can the kernels address this tensor through (n, h, l) strides: last axis contiguous, rows
    aligned to four elements."""
    ok = t.stride(-1) == 1 or t.shape[-1] == 1
    if ok and t.shape[-1] % 4 == 0:
        ok = t.data_ptr() % (4 * t.element_size()) == 0 and all(s % 4 == 0 for s in t.stride()[:3])
    return ok


def _strided(t):
    """A tensor the kernels can read through (n, h, l) strides.  Anything else is copied."""
    if not _rows_ok(t):
        t = t.contiguous()
    return t, (ctypes.c_int64 * 3)(*t.stride()[:3])


class _Dense:
    """Context for tensors the kernels address densely: contiguous ones pass through; others
    are staged through a contiguous copy that is written back on exit when `writeback`."""

    def __init__(self, tensors, writeback):
        self.orig = list(tensors)
        self.writeback = writeback
        self.work = [t if t.is_contiguous() else t.contiguous() for t in self.orig]

    def __enter__(self):
        return self.work

    def __exit__(self, *exc):
        if self.writeback and exc[0] is None:
            for o, w in zip(self.orig, self.work):
                if o is not w:
                    o.copy_(w)
        return False


def _has_bf16_kernel(E, M):
    return E == M and E in (8, 16, 32, 64, 128)


# torch's own fast path to the current stream's handle (what its compiled-code launchers use); the
# public Stream object costs several microseconds to build per call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    if _raw_stream is not None and device.index is not None:
        return ctypes.c_void_p(_raw_stream(device.index))
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def self_ref_forward(x, W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff, beta_diff, out,
                     flags=0):
    """SRWM forward over the whole sequence.  W_y, W_q, W_k, w_b are overwritten with the
    final state; q ... out are overwritten with the per-step vectors.  W_y is (N, H, E, Y):
    Y = E for the plain operator, any other width (3E+1 in the reference's second variant)
    makes out and y_diff (N, H, L, Y).  x and out may both be bfloat16; everything else stays
    float32."""
    io = x.dtype if isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 else torch.float32
    _require(x, "x", None, io)
    N, H, L, E = x.shape
    _require(W_y, "W_y")
    Y = W_y.shape[-1]
    _require(W_y, "W_y", (N, H, E, Y))
    for t, nm in ((W_q, "W_q"), (W_k, "W_k")):
        _require(t, nm, (N, H, E, E))
    _require(w_b, "w_b", (N, H, E, 4))
    for t, nm in ((q, "q"), (k, "k"), (q_diff, "q_diff"), (k_diff, "k_diff")):
        _require(t, nm, (N, H, L, E))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(out, "out", (N, H, L, Y), io)
    _require(beta, "beta", (N, H, L, 4))
    _require(beta_diff, "beta_diff", (N, H, L, 4))
    if x.numel() == 0 or Y == 0:
        return
    xs, xstr = _strided(x)
    null = ctypes.c_void_p(None)
    with torch.cuda.device(x.device), \
            _Dense([W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff, beta_diff, out], True) as d:
        if io == torch.bfloat16 and Y == E:
            name = "srwm_forward_bf16"
            code = lib().srwm_forward_bf16(_ptr(xs), xstr, *[_ptr(t) for t in d], N, H, L, E, _fam(flags),
                                           _stream(x.device))
        elif io == torch.bfloat16:   # wide output block: the layer entry point without any of its extras
            name = "srwm_layer_forward_bf16"
            code = lib().srwm_layer_forward_bf16(_ptr(xs), xstr, null, null, null, null, null,
                                                 *[_ptr(t) for t in d], None, N, H, L, E, Y, _fam(flags), _stream(x.device))
        elif Y == E:
            name = "srwm_forward_f32"
            code = lib().srwm_forward_f32(_ptr(xs), xstr, *[_ptr(t) for t in d], N, H, L, E, _fam(flags),
                                          _stream(x.device))
        else:
            name = "srwm_forward_wide_f32"
            code = lib().srwm_forward_wide_f32(_ptr(xs), xstr, *[_ptr(t) for t in d], N, H, L, E, Y,
                                               _fam(flags), _stream(x.device))
    _check(code, name)


def self_ref_forward_steps(x, keep, slow, W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff,
                           beta_diff, out, flags=0):
    """SRWM forward over all steps of an unroll with per-step resets: where keep[n, t] == 0 the
    state of batch row n is replaced, before step t, by the shared weights `slow` = (W_y, W_q,
    W_k: (1 or no batch axis, H, E, E), w_b: (..., H, E, 4)).  keep: (N, L) float32 or None.
    Otherwise as self_ref_forward.  A W_y of another width (N, H, E, Y) selects the wide-output form."""
    _require(x, "x")
    N, H, L, E = x.shape
    if isinstance(W_y, torch.Tensor) and W_y.dim() == 4 and W_y.shape[-1] != E:
        return self_ref_layer_forward(x, keep, slow, W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff,
                                      beta_diff, out, flags=flags)
    for t, nm in ((W_y, "W_y"), (W_q, "W_q"), (W_k, "W_k")):
        _require(t, nm, (N, H, E, E))
    _require(w_b, "w_b", (N, H, E, 4))
    for t, nm in ((q, "q"), (k, "k"), (y_diff, "y_diff"), (q_diff, "q_diff"), (k_diff, "k_diff"),
                  (out, "out")):
        _require(t, nm, (N, H, L, E))
    _require(beta, "beta", (N, H, L, 4))
    _require(beta_diff, "beta_diff", (N, H, L, 4))
    null = ctypes.c_void_p(None)
    sl = [null] * 4
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
        shapes = ((H, E, E),) * 3 + ((H, E, 4),)
        sl = []
        for t, shp, nm in zip(slow, shapes, ("slow W_y", "slow W_q", "slow W_k", "slow w_b")):
            t = t.detach().reshape(shp) if isinstance(t, torch.Tensor) and t.numel() == H * E * shp[-1] else t
            _require(t, nm, shp)
            sl.append(t.contiguous())
    if x.numel() == 0:
        return
    xs, xstr = _strided(x)
    with torch.cuda.device(x.device), \
            _Dense([W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff, beta_diff, out], True) as d:
        code = lib().srwm_forward_steps_f32(
            _ptr(xs), xstr, _ptr(keep) if keep is not None else null,
            *[(_ptr(t) if keep is not None else t) for t in sl],
            *[_ptr(t) for t in d], N, H, L, E, _fam(flags), _stream(x.device))
    _check(code, "srwm_forward_steps_f32")


def self_ref_readout_grad(k, beta, y_diff, keep, slow_W_y, grad_out, W_y_entry, grad_x, flags=0):
    """grad_x[n, h, t] = W_y,t-1 grad_out[n, h, t] for an unroll whose carried state is detached
    between steps; W_y_entry is the (N, H, E, E) y block as it was before self_ref_forward_steps.
    flags: FLAG_GENERIC forces the LDS-resident kernel."""
    _require(k, "k")
    N, H, L, E = k.shape
    _require(y_diff, "y_diff")
    Y = y_diff.shape[-1]                      # width of the output block (E, or 3E+1 for the wide variant)
    _require(beta, "beta", (N, H, L, 4))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(grad_out, "grad_out", (N, H, L, Y))
    _require(W_y_entry, "W_y_entry", (N, H, E, Y))
    _require(grad_x, "grad_x", (N, H, L, E))
    null = ctypes.c_void_p(None)
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
        slow_W_y = slow_W_y.detach().reshape(H, E, Y).contiguous()
        _require(slow_W_y, "slow W_y", (H, E, Y))
    if k.numel() == 0:
        return
    gos, gstr = _strided(grad_out)
    with torch.cuda.device(k.device), _Dense([k, beta, y_diff, W_y_entry], False) as sv, \
            _Dense([grad_x], True) as gr:
        code = lib().srwm_readout_grad_wide_f32(
            _ptr(sv[0]), _ptr(sv[1]), _ptr(sv[2]), _ptr(keep) if keep is not None else null,
            _ptr(slow_W_y) if keep is not None else null, _ptr(gos), gstr, _ptr(sv[3]), _ptr(gr[0]),
            N, H, L, E, Y, _fam(flags), _stream(k.device))
    _check(code, "srwm_readout_grad_wide_f32")


def self_ref_layer_readout_grad(x, k, beta, y_diff, keep, slow_W_y, grad_out, W_y_entry, grad_x, grad_W_y,
                                grad_slow_W_y, flags=0):
    """self_ref_readout_grad plus the gradient of the shared W_y, for a layer's whole unroll:
    grad_x[n, h, t] = W_y,t-1 grad_out[n, h, t]; grad_W_y[n, h] = sum_t x_t (x) grad_out_t
    ((N, H, E, Y), written); grad_slow_W_y (H, E, Y) = its sum over the batch.  x: the operator's
    input (soft-maxed if the layer soft-maxes it), any strides.  flags: FLAG_STATE_SHIFT (W_y_entry
    is the carried shift from the shared weights), FLAG_GENERIC."""
    _require(k, "k")
    N, H, L, E = k.shape
    _require(y_diff, "y_diff")
    Y = y_diff.shape[-1]
    _require(x, "x", (N, H, L, E))
    _require(beta, "beta", (N, H, L, 4))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(grad_out, "grad_out", (N, H, L, Y))
    _require(W_y_entry, "W_y_entry", (N, H, E, Y))
    _require(grad_x, "grad_x", (N, H, L, E))
    _require(grad_W_y, "grad_W_y", (N, H, E, Y))
    _require(grad_slow_W_y, "grad_slow_W_y", (H, E, Y))
    if not (grad_W_y.is_contiguous() and grad_slow_W_y.is_contiguous()):
        raise ValueError("grad_W_y and grad_slow_W_y must be contiguous")
    slow_W_y = slow_W_y.detach().reshape(H, E, Y).contiguous()
    _require(slow_W_y, "slow W_y", (H, E, Y))
    null = ctypes.c_void_p(None)
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
    if k.numel() == 0:
        grad_W_y.zero_()
        grad_slow_W_y.zero_()
        return
    xs, xstr = _strided(x)
    gos, gstr = _strided(grad_out)
    with torch.cuda.device(k.device), _Dense([k, beta, y_diff, W_y_entry], False) as sv, \
            _Dense([] if grad_x.stride(-1) == 1 else [grad_x], True) as gr:
        gxt = gr[0] if gr else grad_x   # rows at any strides: a permuted buffer is written in place
        code = lib().srwm_layer_readout_grad_f32(
            _ptr(xs), xstr, _ptr(sv[0]), _ptr(sv[1]), _ptr(sv[2]), _ptr(keep) if keep is not None else null,
            _ptr(slow_W_y), _ptr(gos), gstr, _ptr(sv[3]), _ptr(gxt), (ctypes.c_int64 * 3)(*gxt.stride()[:3]),
            _ptr(grad_W_y), _ptr(grad_slow_W_y), N, H, L, E, Y, _fam(flags), _stream(k.device))
    _check(code, "srwm_layer_readout_grad_f32")


def self_ref_backward(x, q, k, beta, y_diff, q_diff, k_diff, beta_diff, grad_out,
                      W_y, W_q, W_k, w_b, grad_x, grad_W_y, grad_W_q, grad_W_k, grad_w_b,
                      flags=GRAD_STATE_ACCUM):
    """SRWM backward.  W_* must hold the final state the forward left behind.  By default
    behaves like the reference extension function: the grad_W buffers are read as the
    gradient w.r.t. the final state and the result is added to them (identical to a plain
    overwrite when they arrive zero-filled, which is how SelfRefv0.backward calls it).
    W_y (N, H, E, Y) fixes the width of y_diff, grad_out and grad_W_y.  x and grad_out may both be
    bfloat16; grad_x and everything else stay float32."""
    io = x.dtype if isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 else torch.float32
    _require(x, "x", None, io)
    N, H, L, E = x.shape
    _require(W_y, "W_y")
    Y = W_y.shape[-1]
    for t, nm in ((q, "q"), (k, "k"), (q_diff, "q_diff"), (k_diff, "k_diff"), (grad_x, "grad_x")):
        _require(t, nm, (N, H, L, E))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(grad_out, "grad_out", (N, H, L, Y), io)
    _require(beta, "beta", (N, H, L, 4))
    _require(beta_diff, "beta_diff", (N, H, L, 4))
    for t, nm in ((W_y, "W_y"), (grad_W_y, "grad_W_y")):
        _require(t, nm, (N, H, E, Y))
    for t, nm in ((W_q, "W_q"), (W_k, "W_k"), (grad_W_q, "grad_W_q"), (grad_W_k, "grad_W_k")):
        _require(t, nm, (N, H, E, E))
    _require(w_b, "w_b", (N, H, E, 4))
    _require(grad_w_b, "grad_w_b", (N, H, E, 4))
    if x.numel() == 0 or Y == 0:
        # no steps: the state gradient passes through unchanged (zero when none came in)
        if (flags & 3) == GRAD_STATE_ZERO:
            for g in (grad_W_y, grad_W_q, grad_W_k, grad_w_b):
                g.zero_()
        return
    xs, xstr = _strided(x)
    gos, gstr = _strided(grad_out)
    with torch.cuda.device(x.device), \
            _Dense([q, k, beta, y_diff, q_diff, k_diff, beta_diff], False) as sv, \
            _Dense([W_y, W_q, W_k, w_b], False) as st, \
            _Dense([grad_x, grad_W_y, grad_W_q, grad_W_k, grad_w_b], True) as gr:
        if io == torch.bfloat16 and Y == E:
            name = "srwm_backward_bf16"
            code = lib().srwm_backward_bf16(_ptr(xs), xstr, *[_ptr(t) for t in sv], _ptr(gos), gstr,
                                            *[_ptr(t) for t in st], *[_ptr(t) for t in gr],
                                            N, H, L, E, _fam(flags), _stream(x.device))
        elif io == torch.bfloat16:
            null = ctypes.c_void_p(None)
            name = "srwm_layer_backward_bf16"
            code = lib().srwm_layer_backward_bf16(_ptr(xs), xstr, *[_ptr(t) for t in sv], _ptr(gos), gstr,
                                                  null, null, null, null, *[_ptr(t) for t in st],
                                                  _ptr(gr[0]), None, *[_ptr(t) for t in gr[1:]], null, null, null, null,
                                                  N, H, L, E, Y, _fam(flags), _stream(x.device))
        elif Y == E:
            name = "srwm_backward_f32"
            code = lib().srwm_backward_f32(_ptr(xs), xstr, *[_ptr(t) for t in sv], _ptr(gos), gstr,
                                           *[_ptr(t) for t in st], *[_ptr(t) for t in gr],
                                           N, H, L, E, _fam(flags), _stream(x.device))
        else:
            name = "srwm_backward_wide_f32"
            code = lib().srwm_backward_wide_f32(_ptr(xs), xstr, *[_ptr(t) for t in sv], _ptr(gos), gstr,
                                                *[_ptr(t) for t in st], *[_ptr(t) for t in gr],
                                                N, H, L, E, Y, _fam(flags), _stream(x.device))
    _check(code, name)


def _shared(slow, H, E, Y):
    """The layer's parameters as dense (H, E, .) tensors; a leading batch axis of 1 is dropped."""
    shapes = ((H, E, Y), (H, E, E), (H, E, E), (H, E, 4))
    out = []
    for t, shp, nm in zip(slow, shapes, ("shared W_y", "shared W_q", "shared W_k", "shared w_b")):
        _require(t, nm)
        if t.dim() == 4 and t.shape[0] == 1:
            t = t[0]
        _require(t, nm, shp)
        out.append(t if t.is_contiguous() else t.detach().contiguous())   # only its address is used
    return out


def self_ref_layer_forward(x, keep, slow, W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff,
                           beta_diff, out, flags=0):
    """SRWM forward with the layers' prologue and epilogue inside the kernel: `slow` = the shared
    weights (W_y: (1, H, E, Y) or (H, E, Y), ...), read without a repeat(); flags FLAG_FRESH_STATE
    (start from them, W_* are outputs), FLAG_STATE_SHIFT (W_* hold the state minus the shared
    weights, in and out), FLAG_SOFTMAX_INPUT (x is soft-maxed by the kernel); keep as in
    self_ref_forward_steps.  x and out may both be bfloat16."""
    io = x.dtype if isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 else torch.float32
    _require(x, "x", None, io)
    N, H, L, E = x.shape
    _require(W_y, "W_y")
    Y = W_y.shape[-1]
    _require(W_y, "W_y", (N, H, E, Y))
    for t, nm in ((W_q, "W_q"), (W_k, "W_k")):
        _require(t, nm, (N, H, E, E))
    _require(w_b, "w_b", (N, H, E, 4))
    for t, nm in ((q, "q"), (k, "k"), (q_diff, "q_diff"), (k_diff, "k_diff")):
        _require(t, nm, (N, H, L, E))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(out, "out", (N, H, L, Y), io)
    _require(beta, "beta", (N, H, L, 4))
    _require(beta_diff, "beta_diff", (N, H, L, 4))
    sl = _shared(slow, H, E, Y)
    null = ctypes.c_void_p(None)
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
    if x.numel() == 0:
        if flags & FLAG_FRESH_STATE:   # no steps: the state is the shared weights (a zero shift)
            for w, sw in zip((W_y, W_q, W_k, w_b), sl):
                if flags & FLAG_STATE_SHIFT:
                    w.zero_()
                else:
                    w.copy_(sw.unsqueeze(0).expand_as(w))
        return
    xs, xstr = _strided(x)
    by_strides = _rows_ok(out)   # a permuted buffer is written in place
    with torch.cuda.device(x.device), \
            _Dense([W_y, W_q, W_k, w_b, q, k, beta, y_diff, q_diff, k_diff, beta_diff], True) as d, \
            _Dense([] if by_strides else [out], True) as o:
        ot = out if by_strides else o[0]
        name = "srwm_layer_forward_bf16" if io == torch.bfloat16 else "srwm_layer_forward_f32"
        code = getattr(lib(), name)(
            _ptr(xs), xstr, _ptr(keep) if keep is not None else null, *[_ptr(t) for t in sl],
            *[_ptr(t) for t in d], _ptr(ot), (ctypes.c_int64 * 3)(*ot.stride()[:3]), N, H, L, E, Y, _fam(flags),
            _stream(x.device))
    _check(code, name)


def self_ref_layer_backward(x, q, k, beta, y_diff, q_diff, k_diff, beta_diff, grad_out, slow,
                            W_y, W_q, W_k, w_b, grad_x, grad_W, grad_slow, flags=GRAD_STATE_ZERO):
    """Backward of self_ref_layer_forward (without resets).  W_*: the final state as the forward
    left it; grad_W: four (N, H, E, .) tensors (SRWM_GRAD_STATE_* semantics, per batch row);
    grad_slow: four (H, E, .) tensors receiving the sum of grad_W over the batch, or None.
    x and grad_out may both be bfloat16; every gradient comes back in float32."""
    io = x.dtype if isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 else torch.float32
    _require(x, "x", None, io)
    N, H, L, E = x.shape
    _require(W_y, "W_y")
    Y = W_y.shape[-1]
    for t, nm in ((q, "q"), (k, "k"), (q_diff, "q_diff"), (k_diff, "k_diff"), (grad_x, "grad_x")):
        _require(t, nm, (N, H, L, E))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(grad_out, "grad_out", (N, H, L, Y), io)
    _require(beta, "beta", (N, H, L, 4))
    _require(beta_diff, "beta_diff", (N, H, L, 4))
    shapes = ((N, H, E, Y), (N, H, E, E), (N, H, E, E), (N, H, E, 4))
    for t, g, shp in zip((W_y, W_q, W_k, w_b), grad_W, shapes):
        _require(t, "state", shp)
        _require(g, "grad_W", shp)
        if not g.is_contiguous():
            raise ValueError("grad_W tensors must be contiguous")
    sl = _shared(slow, H, E, Y)
    null = ctypes.c_void_p(None)
    gsl = [null] * 4
    if grad_slow is not None:
        for g, shp in zip(grad_slow, ((H, E, Y), (H, E, E), (H, E, E), (H, E, 4))):
            _require(g, "grad_slow", shp)
            if not g.is_contiguous():
                raise ValueError("grad_slow tensors must be contiguous")
        gsl = [_ptr(g) for g in grad_slow]
    if x.numel() == 0:
        if (flags & 3) == GRAD_STATE_ZERO:
            for g in grad_W:
                g.zero_()
        if grad_slow is not None:
            for gs_, g in zip(grad_slow, grad_W):
                gs_.copy_(g.sum(0))
        return
    xs, xstr = _strided(x)
    gos, gstr = _strided(grad_out)
    with torch.cuda.device(x.device), \
            _Dense([q, k, beta, y_diff, q_diff, k_diff, beta_diff], False) as sv, \
            _Dense([W_y, W_q, W_k, w_b], False) as st, \
            _Dense([] if grad_x.stride(-1) == 1 else [grad_x], True) as gx:
        gxt = gx[0] if gx else grad_x   # any row strides: the kernels store grad_x element by element
        name = "srwm_layer_backward_bf16" if io == torch.bfloat16 else "srwm_layer_backward_f32"
        code = getattr(lib(), name)(
            _ptr(xs), xstr, *[_ptr(t) for t in sv], _ptr(gos), gstr, *[_ptr(t) for t in sl],
            *[_ptr(t) for t in st], _ptr(gxt), (ctypes.c_int64 * 3)(*gxt.stride()[:3]), *[_ptr(g) for g in grad_W], *gsl,
            N, H, L, E, Y, _fam(flags), _stream(x.device))
    _check(code, name)


def scratch_bytes():
    """Size of the static device array behind self_ref_layer_backward_noalloc."""
    return int(lib().srwm_hip_scratch_bytes())


def self_ref_layer_backward_noalloc(x, q, k, beta, y_diff, q_diff, k_diff, beta_diff, grad_out, slow,
                                    W_y, W_q, W_k, w_b, grad_x, grad_slow, flags=0):
    """self_ref_layer_backward without the per-row gradient tensors: they live in a static device
    array inside the library, so the call allocates nothing (every tensor must already be dense where
    the kernels need it dense; nothing is copied here).  grad_slow: four (H, E, .) tensors, required.
    Raises when N*H*E*(Y+2E+4) floats exceed scratch_bytes().  Calls that overlap on one GPU share the
    array and race; calls on one stream are ordered."""
    _require(x, "x")
    N, H, L, E = x.shape
    _require(W_y, "W_y")
    Y = W_y.shape[-1]
    for t, nm in ((q, "q"), (k, "k"), (q_diff, "q_diff"), (k_diff, "k_diff"), (grad_x, "grad_x")):
        _require(t, nm, (N, H, L, E))
    _require(y_diff, "y_diff", (N, H, L, Y))
    _require(grad_out, "grad_out", (N, H, L, Y))
    _require(beta, "beta", (N, H, L, 4))
    _require(beta_diff, "beta_diff", (N, H, L, 4))
    for t, shp in zip((W_y, W_q, W_k, w_b), ((N, H, E, Y), (N, H, E, E), (N, H, E, E), (N, H, E, 4))):
        _require(t, "state", shp)
    if not all(isinstance(t, torch.Tensor) and t.is_contiguous() for t in slow):
        raise ValueError("self_ref_layer_backward_noalloc copies nothing: the shared weights must be contiguous")
    sl = _shared(slow, H, E, Y)
    for g, shp in zip(grad_slow, ((H, E, Y), (H, E, E), (H, E, E), (H, E, 4))):
        _require(g, "grad_slow", shp)
    dense = [q, k, beta, y_diff, q_diff, k_diff, beta_diff, W_y, W_q, W_k, w_b, grad_x, *grad_slow]
    if not all(t.is_contiguous() for t in dense):
        raise ValueError("self_ref_layer_backward_noalloc copies nothing: saved vectors, state and gradients "
                         "must be contiguous")
    (xs, xstr), (gos, gstr) = _strided(x), _strided(grad_out)
    if xs is not x or gos is not grad_out:
        raise ValueError("self_ref_layer_backward_noalloc copies nothing: x and grad_out need a contiguous, "
                         "16-byte aligned last axis")
    with torch.cuda.device(x.device):
        code = lib().srwm_layer_backward_noalloc_f32(
            _ptr(x), xstr, *[_ptr(t) for t in (q, k, beta, y_diff, q_diff, k_diff, beta_diff)], _ptr(grad_out), gstr,
            *[_ptr(t) for t in sl], *[_ptr(t) for t in (W_y, W_q, W_k, w_b)], _ptr(grad_x), None,
            *[_ptr(g) for g in grad_slow], N, H, L, E, Y, _fam(flags), _stream(x.device))
    _check(code, "srwm_layer_backward_noalloc_f32")


# names of the extension functions of the reference's wide-output variant
# (reinforcement_learning/torchbeast/self_ref_v1/__init__.py:31-32): same call, W_y is (N,H,E,3E+1)
self_ref_forward_v1 = self_ref_forward
self_ref_backward_v1 = self_ref_backward


def fast_weight_forward(q, k, v, beta, v_old, v_insert, kv, out, flags=0):
    """Delta-rule forward.  kv ([N,H,E,M], fp32) is overwritten with the final memory.
    q, k, v, beta and out are all float32 or all bfloat16; v_old, v_insert and kv are float32.
    out may have any strides with a contiguous last axis (a permuted buffer is written in place)."""
    io = q.dtype if isinstance(q, torch.Tensor) and q.dtype == torch.bfloat16 else torch.float32
    _require(q, "q", None, io)
    N, H, L, E = q.shape
    _require(k, "k", (N, H, L, E), io)
    _require(v, "v", None, io)
    M = v.shape[-1]
    _require(v, "v", (N, H, L, M), io)
    _require(beta, "beta", (N, H, L, 1), io)
    _require(out, "out", (N, H, L, M), io)
    for t, nm in ((v_old, "v_old"), (v_insert, "v_insert")):
        _require(t, nm, (N, H, L, M))
    _require(kv, "kv", (N, H, E, M))
    if q.numel() == 0 or v.numel() == 0:
        return
    if io == torch.bfloat16 and not _has_bf16_kernel(E, M):
        # no bf16 kernel for this size: widen, run the fp32 kernels, round the output
        o32 = torch.empty(out.shape, device=out.device, dtype=torch.float32)
        fast_weight_forward(q.float(), k.float(), v.float(), beta.float(), v_old, v_insert, kv, o32, flags)
        out.copy_(o32)
        return
    fn = lib().delta_forward_bf16 if io == torch.bfloat16 else lib().delta_forward_f32
    (qs, qstr), (ks, kstr), (vs, vstr), (bs, bstr) = (_strided(t) for t in (q, k, v, beta))
    by_strides = _rows_ok(out)
    with torch.cuda.device(q.device), _Dense([v_old, v_insert, kv], True) as d, _Dense([] if by_strides else [out], True) as o:
        ot = out if by_strides else o[0]
        code = fn(_ptr(qs), qstr, _ptr(ks), kstr, _ptr(vs), vstr, _ptr(bs), bstr,
                  *[_ptr(t) for t in d], _ptr(ot), (ctypes.c_int64 * 3)(*ot.stride()[:3]), N, H, L, E, M, _fam(flags),
                  _stream(q.device))
    _check(code, fn.__name__)


def fast_weight_forward_steps(q, k, v, beta, keep, v_old, v_insert, kv, out, flags=0):
    """Delta-rule forward over all steps of an unroll; the memory is zeroed before step t of batch
    row n where keep[n, t] == 0 (keep: (N, L) float32 or None).  float32 only."""
    _require(q, "q")
    N, H, L, E = q.shape
    _require(k, "k", (N, H, L, E))
    _require(v, "v")
    M = v.shape[-1]
    _require(v, "v", (N, H, L, M))
    _require(beta, "beta", (N, H, L, 1))
    for t, nm in ((v_old, "v_old"), (v_insert, "v_insert"), (out, "out")):
        _require(t, nm, (N, H, L, M))
    _require(kv, "kv", (N, H, E, M))
    null = ctypes.c_void_p(None)
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
    if q.numel() == 0 or v.numel() == 0:
        return
    (qs, qstr), (ks, kstr), (vs, vstr), (bs, bstr) = (_strided(t) for t in (q, k, v, beta))
    by_strides = _rows_ok(out)
    with torch.cuda.device(q.device), _Dense([v_old, v_insert, kv], True) as d, _Dense([] if by_strides else [out], True) as o:
        ot = out if by_strides else o[0]
        code = lib().delta_forward_steps_f32(_ptr(qs), qstr, _ptr(ks), kstr, _ptr(vs), vstr, _ptr(bs), bstr,
                                             _ptr(keep) if keep is not None else null,
                                             *[_ptr(t) for t in d], _ptr(ot), (ctypes.c_int64 * 3)(*ot.stride()[:3]),
                                             N, H, L, E, M, _fam(flags), _stream(q.device))
    _check(code, "delta_forward_steps_f32")


def fast_weight_readout_replay(k, v_insert, keep, grad_out, kv_entry, u, flags=0):
    """u[n, h, t] = W_{t-1} grad_out[n, h, t] for an unroll whose memory carries no gradient;
    kv_entry is the (N, H, E, M) memory as it was before fast_weight_forward_steps.
    flags: FLAG_GENERIC forces the LDS-resident kernel."""
    _require(k, "k")
    N, H, L, E = k.shape
    _require(v_insert, "v_insert")
    M = v_insert.shape[-1]
    _require(v_insert, "v_insert", (N, H, L, M))
    _require(grad_out, "grad_out", (N, H, L, M))
    _require(kv_entry, "kv_entry", (N, H, E, M))
    _require(u, "u", (N, H, L, E))
    null = ctypes.c_void_p(None)
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
    if k.numel() == 0:
        return
    (ks, kstr), (gos, gstr) = _strided(k), _strided(grad_out)
    with torch.cuda.device(k.device), _Dense([v_insert, kv_entry], False) as sv, _Dense([u], True) as d:
        code = lib().delta_readout_replay_f32(_ptr(ks), kstr, _ptr(sv[0]), _ptr(keep) if keep is not None else null,
                                              _ptr(gos), gstr, _ptr(sv[1]), _ptr(d[0]), N, H, L, E, M, _fam(flags),
                                              _stream(k.device))
    _check(code, "delta_readout_replay_f32")


def fast_weight_steps_backward(q, k, v, beta, keep, v_old, v_insert, grad_out, kv_entry, grad_q, grad_k, grad_v,
                               grad_beta, flags=0):
    """The whole backward of fast_weight_forward_steps (the memory carries no gradient): the replay
    of fast_weight_readout_replay and the per-step formulas, two launches.  grad_q, grad_k: (N, H, L, E);
    grad_v: (N, H, L, M); grad_beta: (N, H, L, 1); all overwritten."""
    _require(q, "q")
    N, H, L, E = q.shape
    _require(v, "v")
    M = v.shape[-1]
    _require(k, "k", (N, H, L, E))
    _require(v, "v", (N, H, L, M))
    _require(beta, "beta", (N, H, L, 1))
    for t, nm in ((v_old, "v_old"), (v_insert, "v_insert"), (grad_out, "grad_out"), (grad_v, "grad_v")):
        _require(t, nm, (N, H, L, M))
    _require(kv_entry, "kv_entry", (N, H, E, M))
    _require(grad_q, "grad_q", (N, H, L, E))
    _require(grad_k, "grad_k", (N, H, L, E))
    _require(grad_beta, "grad_beta", (N, H, L, 1))
    null = ctypes.c_void_p(None)
    if keep is not None:
        _require(keep, "keep", (N, L))
        keep = keep.contiguous()
    if q.numel() == 0:
        return
    (qs, qstr), (ks, kstr), (vs, vstr), (bs, bstr), (gos, gstr) = (_strided(t) for t in (q, k, v, beta, grad_out))
    with torch.cuda.device(q.device), _Dense([v_old, v_insert, kv_entry], False) as sv, \
            _Dense([grad_q, grad_k, grad_v, grad_beta], True) as d:
        code = lib().delta_steps_backward_f32(
            _ptr(qs), qstr, _ptr(ks), kstr, _ptr(vs), vstr, _ptr(bs), bstr, _ptr(keep) if keep is not None else null,
            _ptr(sv[0]), _ptr(sv[1]), _ptr(gos), gstr, _ptr(sv[2]), *[_ptr(t) for t in d], N, H, L, E, M, _fam(flags),
            _stream(q.device))
    _check(code, "delta_steps_backward_f32")


def delta_layer_prologue(rows, E, M, eps=False):
    """rows: (L, N, H, 2E+M+1) float32 or bfloat16, contiguous -- the delta-rule layers' projection [q~ | k~ | v | b~].
    Returns q, k: (L, N, H, E) normalised (elu + 1 over its sum, plus 1e-5 when `eps`), v: (L, N, H, M),
    beta: (L, N, H) = sigmoid, in the type of `rows`, and sums: (L, N, H, 2) float32; all freshly allocated and
    contiguous, from one launch."""
    io = rows.dtype if isinstance(rows, torch.Tensor) and rows.dtype == torch.bfloat16 else torch.float32
    _require(rows, "rows", None, io)
    L, N, H, W = rows.shape
    if W != 2 * E + M + 1 or not rows.is_contiguous():
        raise ValueError(f"rows must be contiguous with last axis 2E+M+1 = {2 * E + M + 1} (got {tuple(rows.shape)})")
    new = lambda *sh: torch.empty(sh, device=rows.device, dtype=io)
    q, k, v, beta = new(L, N, H, E), new(L, N, H, E), new(L, N, H, M), new(L, N, H)
    sums = torch.empty((L, N, H, 2), device=rows.device, dtype=torch.float32)
    if rows.numel():
        fn = lib().delta_layer_prologue_bf16 if io == torch.bfloat16 else lib().delta_layer_prologue_f32
        with torch.cuda.device(rows.device):
            code = fn(_ptr(rows), _ptr(q), _ptr(k), _ptr(v), _ptr(beta), _ptr(sums),
                      N, H, L, E, M, FLAG_NORM_EPS if eps else 0, _stream(rows.device))
        _check(code, fn.__name__)
    return q, k, v, beta, sums


def delta_layer_prologue_grad(grad_q, grad_k, grad_v, grad_beta, q, k, beta, sums):
    """Backward of delta_layer_prologue.  grad_q, grad_k: (N, H, L, E), grad_v: (N, H, L, M), grad_beta:
    (N, H, L, 1), any strides with a contiguous last axis (the operator's gradients as they are);
    q, k, beta, sums as delta_layer_prologue returned them.  Returns the gradient of `rows`, (L, N, H, 2E+M+1)."""
    L, N, H, E = q.shape
    M = grad_v.shape[-1]
    io = q.dtype if isinstance(q, torch.Tensor) and q.dtype == torch.bfloat16 else torch.float32
    _require(q, "q", None, io)
    _require(k, "k", (L, N, H, E), io)
    _require(beta, "beta", (L, N, H), io)
    _require(sums, "sums", (L, N, H, 2))
    gs = []
    for t, nm, w in ((grad_q, "grad_q", E), (grad_k, "grad_k", E), (grad_v, "grad_v", M), (grad_beta, "grad_beta", 1)):
        _require(t, nm, (N, H, L, w), io)
        if w > 1 and t.stride(-1) != 1:
            t = t.contiguous()
        gs.append((t, (ctypes.c_int64 * 3)(*t.stride()[:3])))
    q, k, beta, sums = (t.contiguous() for t in (q, k, beta, sums))
    grad_rows = torch.empty((L, N, H, 2 * E + M + 1), device=q.device, dtype=io)
    if grad_rows.numel():
        fn = lib().delta_layer_prologue_grad_bf16 if io == torch.bfloat16 else lib().delta_layer_prologue_grad_f32
        with torch.cuda.device(q.device):
            code = fn(*[a for t, st in gs for a in (_ptr(t), st)], _ptr(q), _ptr(k), _ptr(beta), _ptr(sums),
                      _ptr(grad_rows), N, H, L, E, M, 0, _stream(q.device))
        _check(code, fn.__name__)
    return grad_rows


def fast_weight_backward(q, k, v, beta, v_old, v_insert, grad_out, kv, grad_q, grad_k, grad_v,
                         grad_beta, grad_kv=None, flags=GRAD_STATE_ZERO):
    """Delta-rule backward.  kv must hold the final memory and is reverted to the initial
    one.  grad_kv (optional, beyond the reference's list): gradient of the memory, see
    the SRWM_GRAD_STATE_* flags."""
    io = q.dtype if isinstance(q, torch.Tensor) and q.dtype == torch.bfloat16 else torch.float32
    _require(q, "q", None, io)
    N, H, L, E = q.shape
    _require(k, "k", (N, H, L, E), io)
    _require(v, "v", None, io)
    M = v.shape[-1]
    _require(beta, "beta", (N, H, L, 1), io)
    for t, nm in ((v_old, "v_old"), (v_insert, "v_insert")):
        _require(t, nm, (N, H, L, M))
    _require(grad_out, "grad_out", (N, H, L, M), io)
    _require(kv, "kv", (N, H, E, M))
    # the library writes fp32 gradients; with bf16 inputs the caller may pass fp32 tensors
    # (used as they are) or bf16 ones (filled through an fp32 temporary)
    gdt = lambda t: torch.float32 if (isinstance(t, torch.Tensor) and t.dtype == torch.float32) else io
    _require(grad_q, "grad_q", (N, H, L, E), gdt(grad_q))
    _require(grad_k, "grad_k", (N, H, L, E), gdt(grad_k))
    _require(grad_v, "grad_v", (N, H, L, M), gdt(grad_v))
    _require(grad_beta, "grad_beta", (N, H, L, 1), gdt(grad_beta))
    if grad_kv is not None:
        _require(grad_kv, "grad_kv", (N, H, E, M))
    if q.numel() == 0 or v.numel() == 0:
        if grad_kv is not None and (flags & 3) == GRAD_STATE_ZERO:
            grad_kv.zero_()
        return
    if io == torch.bfloat16 and not _has_bf16_kernel(E, M):
        g32 = [torch.empty(t.shape, device=t.device, dtype=torch.float32)
               for t in (grad_q, grad_k, grad_v, grad_beta)]
        fast_weight_backward(q.float(), k.float(), v.float(), beta.float(), v_old, v_insert,
                             grad_out.float(), kv, *g32, grad_kv=grad_kv, flags=flags)
        for dst, src in zip((grad_q, grad_k, grad_v, grad_beta), g32):
            dst.copy_(src)
        return
    fn = lib().delta_backward_bf16 if io == torch.bfloat16 else lib().delta_backward_f32
    (qs, qstr), (ks, kstr), (vs, vstr), (bs, bstr), (gos, gstr) = (
        _strided(t) for t in (q, k, v, beta, grad_out))
    if io == torch.bfloat16:
        bf_outs = (grad_q, grad_k, grad_v, grad_beta)
        # The chunkwise kernels round grad_q, grad_k, grad_v themselves when all three are bf16, no
        # gradient of the memory is asked for and single products are allowed; grad_beta is fp32 there.
        native = (bool(flags & FLAG_CHUNKWISE) and not flags & FLAG_EXACT_PRODUCTS and grad_kv is None and
                  all(t.dtype == torch.bfloat16 for t in bf_outs[:3]))
        if native:
            flags |= FLAG_BF16_GRADS
        # otherwise the library returns every gradient in fp32 and bf16 destinations are rounded here
        grad_q, grad_k, grad_v, grad_beta = (
            t if t.dtype == torch.float32 or (native and i < 3)
            else torch.empty(t.shape, device=t.device, dtype=torch.float32)
            for i, t in enumerate(bf_outs))
    outs = [kv, grad_q, grad_k, grad_v, grad_beta] + ([grad_kv] if grad_kv is not None else [])
    with torch.cuda.device(q.device), _Dense([v_old, v_insert], False) as sv, _Dense(outs, True) as d:
        gkv = _ptr(d[5]) if grad_kv is not None else ctypes.c_void_p(None)
        code = fn(_ptr(qs), qstr, _ptr(ks), kstr, _ptr(vs), vstr, _ptr(bs), bstr,
                  _ptr(sv[0]), _ptr(sv[1]), _ptr(gos), gstr,
                  *[_ptr(t) for t in d[:5]], gkv, N, H, L, E, M, _fam(flags), _stream(q.device))
    _check(code, fn.__name__)
    if io == torch.bfloat16:
        for dst, src in zip(bf_outs, (grad_q, grad_k, grad_v, grad_beta)):
            if dst is not src:
                dst.copy_(src)


# ---- selective scan, short causal convolution, norm -------------------------------------------------------------------
# These functions allocate what they return.  Optional tensors may be None.

_I3 = ctypes.c_int64 * 3


def _io_dtype(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not torch.float32 and t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be torch.float32 or torch.bfloat16 (got {t.dtype})")
    return t.dtype


def _gpu(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU (got {t.device}); there is no CPU path")
    return t.device


def _on(t, name, shape, dtype, device):
    """_require, and on the device of the call's other tensors.  `device` is a GPU's (_gpu has seen to that).  The success path is three comparisons: single-token calls are bound by this side."""
    try:
        if t.dtype is dtype and t.shape == shape and t.device == device:
            return
    except AttributeError:
        pass
    _require(t, name, shape, dtype)
    raise RuntimeError(f"{name} lives on {t.device}, the call's other tensors on {device}")


def _rows_in(t, name, shape, dtype, device):
    """A (N, H, L, E) tensor, or the (N, H, E) rows of one step, as the kernels read it: any strides with a contiguous
    last axis (other layouts are copied).  Returns the tensor, which the caller keeps until the launch, and its strides."""
    _on(t, name, shape, dtype, device)
    st = t.stride()
    if st[-1] != 1 and shape[-1] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, _I3(st[0], st[1], st[2] if len(st) == 4 else 0)


def _dense_in(t, name, shape, dtype, device):
    """A dense tensor that starts at a multiple of 16 bytes (copied where it is not), or None."""
    if t is None:
        return None
    _on(t, name, shape, dtype, device)
    if not t.is_contiguous():
        t = t.contiguous()
    if t.data_ptr() & 15:
        t = t.clone()
    return t


class _Here:
    """Stands for torch.cuda.device() where the tensors' device is the current one already (the context itself costs
    more than a microsecond)."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE_ALREADY = _Here()


def _device(device):
    return _HERE_ALREADY if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _strides3(t):
    a, b, c, _ = t.stride()
    return _I3(a, b, c)


def _overwritten(t):
    """A tensor that a kernel overwrites: itself where it is dense and 16-byte aligned, else a copy to write back from."""
    return t if t.is_contiguous() and t.data_ptr() & 15 == 0 else t.clone(memory_format=torch.contiguous_format)


def _p(t):
    return None if t is None else t.data_ptr()


def rows_like(t):
    """An empty tensor of t's shape and type in the memory order of t's rows, its last axis contiguous."""
    out = torch.empty_like(t)
    if out.stride(-1) != 1 and out.shape[-1] != 1:
        out = torch.empty(t.shape, device=t.device, dtype=t.dtype)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_floats(name, *dims):
    n = (ctypes.c_int64 * 1)()
    _check(getattr(lib(), name)(n, *dims), name)
    return n[0]


def _workspace(name, device, *dims):
    """What an entry point asks for at these sizes, or None."""
    n = _workspace_floats(name, *dims)
    return torch.empty(n, device=device, dtype=torch.float32) if n else None


def _masks(keep, lengths, N, L, device):
    return _dense_in(keep, "keep", (N, L), torch.float32, device), _dense_in(lengths, "lengths", (N,), torch.int32, device)


def _scan_sizes(u, A, B):
    if u.dim() != 4 or A.dim() != 3 or B.dim() != 4:
        raise ValueError("u must be (N, H, L, E), A (H, E, S), B and C (N, G, L, S)")
    N, H, L, E = u.shape
    G, S = B.shape[1], A.shape[-1]
    if G == 0 or H % G:
        raise ValueError(f"the {H} heads must divide into the {G} groups of B and C")
    return N, H, L, E, S, G


def selective_scan_forward(u, delta, A, B, C, D, z, delta_bias, state, keep, lengths, softplus, save):
    """The scan over whole sequences.  Returns out (in the memory order of u's rows), last (N, H, E, S) and, with `save`,
    the states that selective_scan_backward starts from (else None)."""
    io = _io_dtype(u, "u")
    for t, nm in ((A, "A"), (B, "B")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{nm} must be a torch.Tensor")
    N, H, L, E, S, G = _scan_sizes(u, A, B)
    dev = _gpu(u, "u")
    us, ustr = _rows_in(u, "u", (N, H, L, E), io, dev)
    ds, dstr = _rows_in(delta, "delta", (N, H, L, E), io, dev)
    zs, zstr = (None, None) if z is None else _rows_in(z, "z", (N, H, L, E), io, dev)
    Bs, bstr = _rows_in(B, "B", (N, G, L, S), io, dev)
    Cs, cstr = _rows_in(C, "C", (N, G, L, S), io, dev)
    A = _dense_in(A, "A", (H, E, S), torch.float32, dev)
    D = _dense_in(D, "D", (H, E), torch.float32, dev)
    bias = _dense_in(delta_bias, "delta_bias", (H, E), torch.float32, dev)
    state = _dense_in(state, "state", (N, H, E, S), torch.float32, dev)
    keep, lengths = _masks(keep, lengths, N, L, dev)
    out = rows_like(u)
    last = torch.empty((N, H, E, S), device=dev, dtype=torch.float32)
    saved = torch.empty((N, (L + 15) // 16, H * E, S), device=dev, dtype=torch.float32) if save else None
    if u.numel() == 0 or S == 0:
        out.zero_()
        last.zero_() if state is None else last.copy_(state)
        return out, last, saved
    work = _workspace("selective_scan_workspace", dev, N, H, L, E, S, G, 0)
    fn = lib().selective_scan_forward_bf16 if io is torch.bfloat16 else lib().selective_scan_forward_f32
    with _device(dev):
        code = fn(_p(us), ustr, _p(ds), dstr, _p(zs), zstr, _p(Bs), bstr, _p(Cs), cstr, _p(A), _p(D), _p(bias), _p(state),
                  _p(keep), _p(lengths), _p(out), _strides3(out), _p(last), _p(saved), _p(work), N, H, L, E,
                  S, G, FLAG_SOFTPLUS if softplus else 0, _stream(dev))
    _check(code, fn.__name__)
    return out, last, saved


def selective_scan_backward(u, delta, A, B, C, D, z, delta_bias, keep, lengths, saved, grad_out, grad_last, softplus,
                            with_state):
    """Gradients of selective_scan_forward, from the states it saved.  grad_last may be None.  Returns those of u, delta,
    A, B, C, D, z, delta_bias and (with `with_state`) state; None for what was None."""
    io = _io_dtype(u, "u")
    N, H, L, E, S, G = _scan_sizes(u, A, B)
    dev = _gpu(u, "u")
    us, ustr = _rows_in(u, "u", (N, H, L, E), io, dev)
    ds, dstr = _rows_in(delta, "delta", (N, H, L, E), io, dev)
    zs, zstr = (None, None) if z is None else _rows_in(z, "z", (N, H, L, E), io, dev)
    Bs, bstr = _rows_in(B, "B", (N, G, L, S), io, dev)
    Cs, cstr = _rows_in(C, "C", (N, G, L, S), io, dev)
    A = _dense_in(A, "A", (H, E, S), torch.float32, dev)
    Dd = _dense_in(D, "D", (H, E), torch.float32, dev)
    bias = _dense_in(delta_bias, "delta_bias", (H, E), torch.float32, dev)
    keep, lengths = _masks(keep, lengths, N, L, dev)
    saved = _dense_in(saved, "saved", (N, (L + 15) // 16, H * E, S), torch.float32, dev)
    gos, gostr = _rows_in(grad_out, "grad_out", (N, H, L, E), io, dev)
    glast = _dense_in(grad_last, "grad_last", (N, H, E, S), torch.float32, dev)
    gu, gdelta, gz = rows_like(u), rows_like(delta), None if z is None else rows_like(z)
    gB, gC = rows_like(B), rows_like(C)
    gA = torch.empty_like(A)
    gD, gbias = None if D is None else torch.empty_like(Dd), None if bias is None else torch.empty_like(bias)
    gstate = torch.empty((N, H, E, S), device=dev, dtype=torch.float32) if with_state else None
    if u.numel() == 0 or S == 0:
        for t in (gu, gdelta, gz, gB, gC, gA, gD, gbias):
            if t is not None:
                t.zero_()
        if gstate is not None:
            gstate.zero_() if glast is None else gstate.copy_(glast)
        return gu, gdelta, gA, gB, gC, gD, gz, gbias, gstate
    fn = lib().selective_scan_backward_bf16 if io is torch.bfloat16 else lib().selective_scan_backward_f32
    work = _workspace("selective_scan_workspace", dev, N, H, L, E, S, G, 1)
    st = _strides3
    with _device(dev):
        code = fn(_p(us), ustr, _p(ds), dstr, _p(zs), zstr, _p(Bs), bstr, _p(Cs), cstr, _p(A), _p(Dd), _p(bias), _p(keep),
                  _p(lengths), _p(saved), _p(gos), gostr, _p(glast), _p(gu), st(gu), _p(gdelta), st(gdelta), _p(gz),
                  None if gz is None else st(gz), _p(gB), st(gB), _p(gC), st(gC), _p(gA), _p(gD), _p(gbias), _p(gstate),
                  _p(work), N, H, L, E, S, G, FLAG_SOFTPLUS if softplus else 0, _stream(dev))
    _check(code, fn.__name__)
    return gu, gdelta, gA, gB, gC, gD, gz, gbias, gstate


def selective_scan_step(u, delta, state, A, B, C, D, z, delta_bias, keep, softplus):
    """One token: u, delta, z (N, H, E), B, C (N, G, S), keep (N,); state (N, H, E, S) is overwritten.  Returns out."""
    io = _io_dtype(u, "u")
    if u.dim() != 3 or not isinstance(A, torch.Tensor) or A.dim() != 3 or not isinstance(B, torch.Tensor) or B.dim() != 3:
        raise ValueError("u must be (N, H, E), A (H, E, S), B and C (N, G, S)")
    N, H, E = u.shape
    G, S = B.shape[1], A.shape[-1]
    if G == 0 or H % G:
        raise ValueError(f"the {H} heads must divide into the {G} groups of B and C")
    dev = _gpu(u, "u")
    us, ustr = _rows_in(u, "u", (N, H, E), io, dev)
    ds, dstr = _rows_in(delta, "delta", (N, H, E), io, dev)
    zs, zstr = (None, None) if z is None else _rows_in(z, "z", (N, H, E), io, dev)
    Bs, bstr = _rows_in(B, "B", (N, G, S), io, dev)
    Cs, cstr = _rows_in(C, "C", (N, G, S), io, dev)
    A = _dense_in(A, "A", (H, E, S), torch.float32, dev)
    D = _dense_in(D, "D", (H, E), torch.float32, dev)
    bias = _dense_in(delta_bias, "delta_bias", (H, E), torch.float32, dev)
    keep = _dense_in(keep, "keep", (N,), torch.float32, dev)
    _on(state, "state", (N, H, E, S), torch.float32, dev)
    out = u.new_empty((N, H, E))
    if u.numel() == 0 or S == 0:
        return out.zero_()
    fn = lib().selective_scan_step_bf16 if io is torch.bfloat16 else lib().selective_scan_step_f32
    h = _overwritten(state)
    with _device(dev):
        code = fn(_p(us), ustr, _p(ds), dstr, _p(zs), zstr, _p(Bs), bstr, _p(Cs), cstr, _p(A), _p(D), _p(bias), _p(keep),
                  _p(h), _p(out), _I3(H * E, E, 0), N, H, E, S, G, FLAG_SOFTPLUS if softplus else 0, _stream(dev))
    _check(code, fn.__name__)
    if h is not state:
        state.copy_(h)
    return out


def causal_conv_forward(x, weight, bias, state, keep, lengths, silu):
    """Short causal depthwise convolution.  Returns out (in the memory order of x's rows) and last (N, H, W-1, E)."""
    io = _io_dtype(x, "x")
    if x.dim() != 4 or not isinstance(weight, torch.Tensor) or weight.dim() != 3:
        raise ValueError("x must be (N, H, L, E), weight (H, E, W)")
    N, H, L, E = x.shape
    W = weight.shape[-1]
    dev = _gpu(x, "x")
    xs, xstr = _rows_in(x, "x", (N, H, L, E), io, dev)
    weight = _dense_in(weight, "weight", (H, E, W), torch.float32, dev)
    bias = _dense_in(bias, "bias", (H, E), torch.float32, dev)
    if not 2 <= W <= 4:
        raise ValueError(f"the convolution has 2 to 4 taps (got {W})")
    state = _dense_in(state, "state", (N, H, W - 1, E), io, dev)
    keep, lengths = _masks(keep, lengths, N, L, dev)
    out = rows_like(x)
    last = torch.empty((N, H, W - 1, E), device=dev, dtype=io)
    if x.numel() == 0:
        last.zero_() if state is None else last.copy_(state)
        return out, last
    fn = lib().causal_conv_forward_bf16 if io is torch.bfloat16 else lib().causal_conv_forward_f32
    with _device(dev):
        code = fn(_p(xs), xstr, _p(weight), _p(bias), _p(state), _p(keep), _p(lengths), _p(out), _strides3(out),
                  _p(last), N, H, L, E, W, FLAG_SILU if silu else 0, _stream(dev))
    _check(code, fn.__name__)
    return out, last


def causal_conv_backward(x, weight, bias, state, keep, lengths, grad_out, grad_last, silu):
    """Gradients of causal_conv_forward: x, weight, bias, state (None for what was None).  grad_last may be None."""
    io = _io_dtype(x, "x")
    N, H, L, E = x.shape
    W = weight.shape[-1]
    dev = _gpu(x, "x")
    xs, xstr = _rows_in(x, "x", (N, H, L, E), io, dev)
    weight = _dense_in(weight, "weight", (H, E, W), torch.float32, dev)
    bias = _dense_in(bias, "bias", (H, E), torch.float32, dev)
    state = _dense_in(state, "state", (N, H, W - 1, E), io, dev)
    keep, lengths = _masks(keep, lengths, N, L, dev)
    gos, gostr = _rows_in(grad_out, "grad_out", (N, H, L, E), io, dev)
    glast = _dense_in(grad_last, "grad_last", (N, H, W - 1, E), io, dev)
    gx, gw = rows_like(x), torch.empty_like(weight)
    gb = None if bias is None else torch.empty_like(bias)
    gstate = None if state is None else torch.empty_like(state)
    if x.numel() == 0:
        gw.zero_()
        if gb is not None:
            gb.zero_()
        if gstate is not None:
            gstate.zero_() if glast is None else gstate.copy_(glast)
        return gx, gw, gb, gstate
    fn = lib().causal_conv_backward_bf16 if io is torch.bfloat16 else lib().causal_conv_backward_f32
    work = _workspace("causal_conv_workspace", dev, N, H, L, E, W)
    with _device(dev):
        code = fn(_p(xs), xstr, _p(weight), _p(bias), _p(state), _p(keep), _p(lengths), _p(gos), gostr, _p(glast), _p(gx),
                  _strides3(gx), _p(gw), _p(gb), _p(gstate), _p(work), N, H, L, E, W, FLAG_SILU if silu else 0,
                  _stream(dev))
    _check(code, fn.__name__)
    return gx, gw, gb, gstate


def causal_conv_step(x, state, weight, bias, keep, silu):
    """One token: x (N, H, E), keep (N,); state (N, H, W-1, E) is overwritten.  Returns out."""
    io = _io_dtype(x, "x")
    if x.dim() != 3 or not isinstance(weight, torch.Tensor) or weight.dim() != 3:
        raise ValueError("x must be (N, H, E), weight (H, E, W)")
    N, H, E = x.shape
    W = weight.shape[-1]
    dev = _gpu(x, "x")
    xs, xstr = _rows_in(x, "x", (N, H, E), io, dev)
    weight = _dense_in(weight, "weight", (H, E, W), torch.float32, dev)
    bias = _dense_in(bias, "bias", (H, E), torch.float32, dev)
    if not 2 <= W <= 4:
        raise ValueError(f"the convolution has 2 to 4 taps (got {W})")
    keep = _dense_in(keep, "keep", (N,), torch.float32, dev)
    _on(state, "state", (N, H, W - 1, E), io, dev)
    out = x.new_empty((N, H, E))
    if x.numel() == 0:
        return out
    fn = lib().causal_conv_step_bf16 if io is torch.bfloat16 else lib().causal_conv_step_f32
    h = _overwritten(state)
    with _device(dev):
        code = fn(_p(xs), xstr, _p(weight), _p(bias), _p(keep), _p(h), _p(out), _I3(H * E, E, 0), N, H, E, W,
                  FLAG_SILU if silu else 0, _stream(dev))
    _check(code, fn.__name__)
    if h is not state:
        state.copy_(h)
    return out


def _norm_rows(x, residual, weight):
    io = _io_dtype(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have a last axis to normalise over")
    D, dev = x.shape[-1], _gpu(x, "x")
    xs = _dense_in(x, "x", x.shape, io, dev)
    rdt = io
    if residual is not None:
        rdt = _io_dtype(residual, "residual")
        if io is torch.float32 and rdt is not torch.float32:
            raise TypeError("a float32 x takes a float32 residual")
        residual = _dense_in(residual, "residual", x.shape, rdt, dev)
    weight = _dense_in(weight, "weight", (D,), torch.float32, dev)
    if D == 0:
        raise ValueError("the norm's rows are empty")
    flags = FLAG_RESIDUAL_F32 if io is torch.bfloat16 and rdt is torch.float32 else 0
    return xs, residual, weight, io, rdt, x.numel() // D, D, dev, flags


def residual_rms_norm_forward(x, residual, weight, eps, save):
    """Root-mean-square norm of x + residual over the last axis.  Returns out (like x), the sum (like residual; x itself
    without one) and, with `save`, the rows' reciprocal norms for the backward (else None)."""
    xs, residual, weight, io, rdt, rows, D, dev, flags = _norm_rows(x, residual, weight)
    out = torch.empty(x.shape, device=dev, dtype=io)
    total = xs if residual is None else torch.empty(x.shape, device=dev, dtype=rdt)
    rstd = torch.empty(rows, device=dev, dtype=torch.float32) if save else None
    if rows:
        fn = lib().residual_rms_norm_forward_bf16 if io is torch.bfloat16 else lib().residual_rms_norm_forward_f32
        with _device(dev):
            code = fn(_p(xs), _p(residual), _p(weight), _p(out), None if residual is None else _p(total), _p(rstd),
                      (ctypes.c_float * 1)(eps), rows, D, flags, _stream(dev))
        _check(code, fn.__name__)
    return out, total, rstd


def residual_rms_norm_e4m3(x, residual, weight, eps):
    """The same with out in torch.float8_e4m3fn.  Returns out, scale (the rows' scales, last axis 1), sum."""
    xs, residual, weight, io, rdt, rows, D, dev, flags = _norm_rows(x, residual, weight)
    out = torch.empty(x.shape, device=dev, dtype=torch.float8_e4m3fn)
    scale = torch.empty((*x.shape[:-1], 1), device=dev, dtype=torch.float32)
    total = xs if residual is None else torch.empty(x.shape, device=dev, dtype=rdt)
    if rows:
        fn = lib().residual_rms_norm_e4m3_bf16 if io is torch.bfloat16 else lib().residual_rms_norm_e4m3_f32
        with _device(dev):
            code = fn(_p(xs), _p(residual), _p(weight), _p(out), _p(scale), None if residual is None else _p(total),
                      (ctypes.c_float * 1)(eps), rows, D, flags, _stream(dev))
        _check(code, fn.__name__)
    return out, scale, total


def residual_rms_norm_backward(total, weight, rstd, grad_out, grad_total, with_residual):
    """Gradients of residual_rms_norm_forward from the sum it returned: x (like grad_out), residual (like the sum; None
    without `with_residual`), weight.  grad_total may be None."""
    io, rdt, D, dev = _io_dtype(grad_out, "grad_out"), _io_dtype(total, "total"), total.shape[-1], _gpu(total, "total")
    total = _dense_in(total, "total", total.shape, rdt, dev)
    weight = _dense_in(weight, "weight", (D,), torch.float32, dev)
    go = _dense_in(grad_out, "grad_out", total.shape, io, dev)
    gt = _dense_in(grad_total, "grad_total", total.shape, rdt, dev)
    rows = total.numel() // D
    gx = torch.empty(total.shape, device=dev, dtype=io)
    gr = torch.empty(total.shape, device=dev, dtype=rdt) if with_residual else None
    gw = torch.empty_like(weight)
    if not rows:
        return gx, gr, gw.zero_()
    fn = lib().residual_rms_norm_backward_bf16 if io is torch.bfloat16 else lib().residual_rms_norm_backward_f32
    work = _workspace("residual_rms_norm_workspace", dev, rows, D)
    flags = FLAG_RESIDUAL_F32 if io is torch.bfloat16 and rdt is torch.float32 else 0
    with _device(dev):
        code = fn(_p(total), _p(weight), _p(rstd), _p(go), _p(gt), _p(gx), _p(gr), _p(gw), _p(work), rows, D, flags,
                  _stream(dev))
    _check(code, fn.__name__)
    return gx, gr, gw
