"""Root-mean-square norm with the residual's addition in one pass, backed by libsrwm_hip.so.

    out, total = residual_rms_norm(x, residual, weight, eps)
    out, scale, total = residual_rms_norm_e4m3(x, residual, weight, eps)

total = x + residual,  out = total / sqrt(mean(total^2) + eps) * weight over the last axis.

x: (..., D) float32 or bfloat16; residual: the same shape, float32, or bfloat16 with a bfloat16 x (None: total is x
itself); weight: (D,) float32.  out has the type of x and total that of residual; the norm is taken of the sum before it is
rounded to that type.  The second form serves layers whose projection runs in 8 bits: out is torch.float8_e4m3fn,
each row divided by scale = max|row| / 448 (1 for a row of zeros) and rounded to nearest even, so that out * scale is the
norm's result; it has no backward.  Rows longer than 16384 have no backward either.
There are no second derivatives and none in forward mode, and a call cannot be traced (torch.jit.trace, make_fx): such calls
raise.
"""
import srwm_hip


def residual_rms_norm(x, residual, weight, eps=1e-5):
    """(out, total); see the module's text."""
    return srwm_hip.binding().residual_rms_norm(x, residual, weight, eps)


def residual_rms_norm_e4m3(x, residual, weight, eps=1e-5):
    """(out, scale, total) with out in torch.float8_e4m3fn and one scale per row; see the module's text.  No backward."""
    return srwm_hip.binding().residual_rms_norm_e4m3(x, residual, weight, eps)
