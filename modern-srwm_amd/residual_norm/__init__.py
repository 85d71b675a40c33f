"""Root-mean-square norm with the residual's addition in one pass, backed by libsrwm_hip.so.

    out, total = residual_rms_norm(x, residual, weight, eps)
    out, scale, total = residual_rms_norm_e4m3(x, residual, weight, eps)

total = x + residual,  out = total / sqrt(mean(total^2) + eps) * weight over the last axis.

x: (..., D) float32 or bfloat16; residual: the same shape, float32, or bfloat16 with a bfloat16 x (None: total is x
itself); weight: (D,) float32.  out has the type of x and total that of residual; the norm is taken of the sum before it is
rounded to that type.  The second form serves layers whose projection runs in 8 bits: out is torch.float8_e4m3fn,
each row divided by scale = max|row| / 448 (1 for a row of zeros) and rounded to nearest even, so that out * scale is the
norm's result; it has no backward.  Rows longer than 16384 have no backward either.
"""
import torch

import srwm_hip

MAX_BACKWARD = 16384


class ResidualRMSNorm(torch.autograd.Function):
    """residual_rms_norm with its backward."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        out, total, rstd = srwm_hip.residual_rms_norm_forward(x, residual, weight, eps, True)
        ctx.set_materialize_grads(False)
        ctx.has_residual = residual is not None
        ctx.save_for_backward(total, weight, rstd)
        ctx.io = x.dtype
        return (out, total) if ctx.has_residual else out

    @staticmethod
    def backward(ctx, grad_out, grad_total=None):
        total, weight, rstd = ctx.saved_tensors
        if grad_out is None:
            grad_out = torch.zeros(total.shape, device=total.device, dtype=ctx.io)
        gx, gr, gw = srwm_hip.residual_rms_norm_backward(total, weight, rstd, grad_out, grad_total, ctx.has_residual)
        return gx, gr, gw, None


def residual_rms_norm(x, residual, weight, eps=1e-5):
    """(out, total); see the module's text."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        if x.shape[-1] > MAX_BACKWARD:
            raise ValueError(f"residual_rms_norm has no backward for rows longer than {MAX_BACKWARD}")
        if residual is None:
            return ResidualRMSNorm.apply(x, None, weight, eps), x
        return ResidualRMSNorm.apply(x, residual, weight, eps)
    out, total, _ = srwm_hip.residual_rms_norm_forward(x, residual, weight, eps, False)
    return out, x if residual is None else total


def residual_rms_norm_e4m3(x, residual, weight, eps=1e-5):
    """(out, scale, total) with out in torch.float8_e4m3fn and one scale per row; see the module's text.  No backward."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError("residual_rms_norm_e4m3 has no backward: call it under torch.no_grad()")
    out, scale, total = srwm_hip.residual_rms_norm_e4m3(x, residual, weight, eps)
    return out, scale, x if residual is None else total
