"""Selective scan, short causal convolution and root-mean-square norm, written from their definitions as loops over
single steps in float64 (or whatever type comes in); gradients come from autograd.  Test infrastructure only."""
import torch


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, keep=None, lengths=None, softplus=True):
    """u, delta, z (N,H,L,E), A (H,E,S), B, C (N,G,L,S), D, delta_bias (H,E), state (N,H,E,S) -> out, last."""
    N, H, L, E = u.shape
    S, G = A.shape[-1], B.shape[1]
    rows_out, rows_last = [], []
    for n in range(N):
        end = L if lengths is None else min(max(int(lengths[n]), 0), L)
        h = torch.zeros(H, E, S, dtype=u.dtype) if state is None else state[n]
        out = []
        for t in range(L):
            if t >= end:
                out.append(torch.zeros(H, E, dtype=u.dtype))
                continue
            dt = delta[n, :, t] if delta_bias is None else delta[n, :, t] + delta_bias
            if softplus:
                dt = torch.logaddexp(dt, torch.zeros_like(dt))
            b = B[n, :, t].repeat_interleave(H // G, 0)[:, None]      # (H, 1, S)
            c = C[n, :, t].repeat_interleave(H // G, 0)[:, None]
            if keep is not None and float(keep[n, t]) == 0:
                h = torch.zeros(H, E, S, dtype=u.dtype)
            h = torch.exp(dt[..., None] * A) * h + (dt * u[n, :, t])[..., None] * b
            y = (h * c).sum(-1)
            if D is not None:
                y = y + D * u[n, :, t]
            if z is not None:
                y = y * z[n, :, t] * torch.sigmoid(z[n, :, t])
            out.append(y)
        rows_out.append(torch.stack(out, 1) if out else u[n])
        rows_last.append(h)
    return torch.stack(rows_out), torch.stack(rows_last)


def conv(x, weight, bias=None, state=None, keep=None, lengths=None, silu=True):
    """x (N,H,L,E), weight (H,E,W), bias (H,E), state (N,H,W-1,E) -> out, last."""
    N, H, L, E = x.shape
    W = weight.shape[-1]
    rows_out, rows_last = [], []
    zero = torch.zeros(H, E, dtype=x.dtype)
    for n in range(N):
        end = L if lengths is None else min(max(int(lengths[n]), 0), L)
        seen = [zero] * (W - 1) if state is None else [state[n, :, j] for j in range(W - 1)]
        out = []
        for t in range(L):
            if t >= end:
                out.append(zero)
                continue
            if keep is not None and float(keep[n, t]) == 0:
                seen = [zero] * (W - 1)
            seen = seen[-(W - 1):] + [x[n, :, t]]
            y = sum(weight[..., j] * seen[j] for j in range(W))
            if bias is not None:
                y = y + bias
            out.append(y * torch.sigmoid(y) if silu else y)
        rows_out.append(torch.stack(out, 1) if out else x[n])
        rows_last.append(torch.stack(seen[-(W - 1):], 1))
    return torch.stack(rows_out), torch.stack(rows_last)


def rms_norm(x, residual, weight, eps):
    total = x if residual is None else x + residual
    return total / torch.sqrt((total * total).mean(-1, keepdim=True) + eps) * weight, total
