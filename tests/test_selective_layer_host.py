"""What the selective state-space layers do without the GPU: the 8-bit form of the input projection's weight."""
import torch

from layer import SelectiveLayer


def test_the_8_bit_weight_is_overwritten_where_it_lies():
    """A captured graph holds its address: a changed weight is converted into the same memory."""
    torch.manual_seed(1)
    layer = SelectiveLayer(2, 16, 32, 0.0).serve_e4m3()
    first = layer._weight_e4m3()
    at = [t.data_ptr() for t in first]
    for change in (lambda w: w.mul_(-3.0), lambda w: w.copy_(torch.randn_like(w))):
        with torch.no_grad():
            change(layer.in_linear.weight)
        now = layer._weight_e4m3()
        assert [t.data_ptr() for t in now] == at
        back = now[0].float() * now[1].t()
        # half a step of e4m3: 2^-4 of the value, or 2^-10 of the row's scale; two roundings of 2^-24 in front
        bound = torch.maximum(layer.in_linear.weight.abs() * 2.0 ** -4, now[1].t() * 2.0 ** -10) * (1 + 1e-5)
        assert ((back - layer.in_linear.weight).abs() <= bound).all()
    layer.in_linear.weight = torch.nn.Parameter(torch.randn_like(layer.in_linear.weight))
    assert [t.data_ptr() for t in layer._weight_e4m3()] == at
    with torch.inference_mode():                        # converted there, overwritten outside and the other way round
        other = SelectiveLayer(2, 16, 32, 0.0).serve_e4m3()
        at = other._weight_e4m3()[0].data_ptr()
    with torch.no_grad():
        assert other.serve_e4m3()._weight_e4m3()[0].data_ptr() == at
    with torch.inference_mode():
        assert other.serve_e4m3()._weight_e4m3()[0].data_ptr() == at


def test_the_8_bit_weight_follows_conversions_and_back():
    """Rounded to 16 bits and widened again, the weight has the same type, device and version as before."""
    torch.manual_seed(2)
    layer = SelectiveLayer(2, 16, 32, 0.0).serve_e4m3()
    at = layer._weight_e4m3()[0].data_ptr()
    layer.to(torch.bfloat16).to(torch.float32)
    fresh = SelectiveLayer(2, 16, 32, 0.0)
    fresh.load_state_dict(layer.state_dict())
    for a, b in zip(layer._weight_e4m3(), fresh.serve_e4m3()._weight_e4m3()):
        assert torch.equal(a.float(), b.float())
    assert layer._weight_e4m3()[0].data_ptr() == at
    assert SelectiveLayer(2, 16, 32, 0.0).to(torch.bfloat16)._eight is None
