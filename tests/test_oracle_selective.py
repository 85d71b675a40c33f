"""The oracle of the selective state-space operators: its gradients against differences, closed forms, and the layouts
(packed sequences, padded batches) that have to be equal to single sequences.  CPU only."""
import torch

from oracle import selective


def _scan_inputs(N, H, L, E, S, G, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    return dict(u=r(N, H, L, E), delta=r(N, H, L, E), A=-torch.exp(r(H, E, S) * 0.5), B=r(N, G, L, S), C=r(N, G, L, S),
                D=r(H, E), z=r(N, H, L, E), delta_bias=r(H, E), state=r(N, H, E, S))


def test_scan_gradients_against_differences():
    a = _scan_inputs(2, 2, 4, 2, 3, 1)
    keep = torch.tensor([[1., 1, 0, 1], [0, 1, 1, 1]])
    lengths = torch.tensor([4, 3])
    names = list(a)
    f = lambda *v: selective.scan(**dict(zip(names, v)), keep=keep, lengths=lengths)
    assert torch.autograd.gradcheck(f, [a[k].requires_grad_() for k in names], eps=1e-6, atol=1e-7)


def test_conv_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    keep = torch.tensor([[1., 1, 0, 1, 1], [1, 1, 1, 1, 0]])
    lengths = torch.tensor([5, 2])
    for W in (2, 3, 4):
        ins = (r(2, 2, 5, 2), r(2, 2, W), r(2, 2), r(2, 2, W - 1, 2))
        assert torch.autograd.gradcheck(lambda *v: selective.conv(*v, keep, lengths), ins, eps=1e-6, atol=1e-7)


def test_scan_without_decay_is_a_cumulative_sum():
    a = _scan_inputs(1, 1, 9, 3, 2, 1, seed=3)
    a.update(A=torch.zeros(1, 3, 2, dtype=torch.float64), D=None, z=None, delta_bias=None, state=None)
    out, last = selective.scan(**a, softplus=False)
    w = (a["delta"] * a["u"])[..., None] * a["B"][:, :, :, None]          # (1, 1, L, E, S)
    h = w.cumsum(2)
    assert torch.allclose(out, (h * a["C"][:, :, :, None]).sum(-1), atol=1e-12)
    assert torch.allclose(last, h[:, :, -1], atol=1e-12)


def test_packed_and_padded_rows_are_single_sequences():
    a = _scan_inputs(1, 2, 10, 3, 4, 2, seed=4)
    a["state"] = None
    keep = torch.ones(1, 10)
    keep[0, 0] = keep[0, 6] = 0
    out, last = selective.scan(**a, keep=keep)
    cut = lambda lo, hi: {k: (v[:, :, lo:hi] if v is not None and v.dim() == 4 else v) for k, v in a.items()}
    first, second = selective.scan(**cut(0, 6)), selective.scan(**cut(6, 10))
    assert torch.equal(out, torch.cat((first[0], second[0]), 2)) and torch.equal(last, second[1])
    out, last = selective.scan(**a, lengths=torch.tensor([6]))
    assert torch.equal(out[:, :, :6], first[0]) and torch.equal(last, first[1]) and not out[:, :, 6:].any()


def test_conv_is_a_grouped_convolution():
    g = torch.Generator().manual_seed(5)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 3, 11, 4), (3, 4, 4), (3, 4)))
    out, last = selective.conv(x, w, b, silu=False)
    flat = x.permute(0, 1, 3, 2).reshape(2, 12, 11)
    ref = torch.nn.functional.conv1d(torch.nn.functional.pad(flat, (3, 0)), w.reshape(12, 1, 4), b.reshape(12), groups=12)
    assert torch.allclose(out, ref.reshape(2, 3, 4, 11).permute(0, 1, 3, 2), atol=1e-12)
    assert torch.equal(last, x[:, :, -3:])
