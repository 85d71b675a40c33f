"""Selective state-space operators, backed by libsrwm_hip.so: the scan, the short causal convolution in front of it, and
their single-token forms.  The recurrence is a sibling of the delta rule's: a state of fixed size per channel, overwritten
at every step, whose decay depends on the step instead of its correction.

    out, last = selective_scan(u, delta, A, B, C, D, z, delta_bias, state, keep, lengths)
    out, last = causal_conv(x, weight, bias, state, keep, lengths)
    out = selective_scan_step(u, delta, state, A, B, C, D, z, delta_bias, keep)      # state overwritten
    out = causal_conv_step(x, state, weight, bias, keep)                             # state overwritten

With dt = softplus(delta + delta_bias), per channel and state

    h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,      out_t = (C_t . h_t + D u_t) * silu(z_t)

u, delta, z: (N, H, L, E) float32 or bfloat16, any strides with a contiguous last axis (the permuted views of step-major
storage are read in place); A: (H, E, S), S <= 64; D, delta_bias: (H, E); B, C: (N, G, L, S) in the type of u, each
group of H / G heads sharing one (G = 1: shared by all channels); D, z, delta_bias, state may be None.  A, D, delta_bias
and the states (N, H, E, S) are float32, and so is all arithmetic.

    out_t = silu(bias + sum_j weight[j] x_{t-W+1+j})

x: (N, H, L, E); weight: (H, E, W) float32 with W = 2, 3 or 4; bias: (H, E) or None; the carried rows, state and last,
are the W - 1 newest inputs, (N, H, W-1, E) in the type of x.

state (None: zeros) comes before the first step, `last` is what is carried on.  keep: (N, L) float32 or None, 0 where the
state is zeroed before the step, as in the step mode of the other operators; sequences packed one behind the other into a
row get a 0 at their first steps.  lengths: (N,) int32 or None, the steps of each row of a padded batch: steps behind them
are not read, their rows of out and of the gradients are zeros, and `last` is the state at the row's end.

Gradients go to every float tensor, through `last` and into `state` as well; keep and lengths get none.  There are no second
derivatives and none in forward mode, and a call cannot be traced (torch.jit.trace, make_fx): such calls raise.
"""
import srwm_hip


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, keep=None, lengths=None, softplus=True):
    """The scan over whole sequences: (out, last).  See the module's text.  softplus=False: dt = delta + delta_bias."""
    return srwm_hip.binding().selective_scan(u, delta, A, B, C, D, z, delta_bias, state, keep, lengths, softplus)


def selective_scan_step(u, delta, state, A, B, C, D=None, z=None, delta_bias=None, keep=None, softplus=True):
    """One token: u, delta, z (N, H, E), B and C (N, G, S), keep (N,).  state is OVERWRITTEN; returns out (N, H, E).
    There is no backward: the call raises where a gradient would be asked of it."""
    return srwm_hip.binding().selective_scan_step(u, delta, state, A, B, C, D, z, delta_bias, keep, softplus)


def causal_conv(x, weight, bias=None, state=None, keep=None, lengths=None, silu=True):
    """Short causal depthwise convolution over whole sequences: (out, last).  silu=False: no activation behind it."""
    return srwm_hip.binding().causal_conv(x, weight, bias, state, keep, lengths, silu)


def causal_conv_step(x, state, weight, bias=None, keep=None, silu=True):
    """One token: x (N, H, E), keep (N,).  state (N, H, W-1, E) is OVERWRITTEN; returns out (N, H, E).  No backward: the
    call raises where a gradient would be asked of it."""
    return srwm_hip.binding().causal_conv_step(x, state, weight, bias, keep, silu)
