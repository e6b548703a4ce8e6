"""The e4m3 weights of an fp8_experts layer after a write that leaves no trace."""
import pytest
import torch

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


@needs_cuda
def test_quantize_weights_renews_them():
    from test_moe_weights import _buffer, _layer, _write, _x
    buf = _buffer()
    layer, x = _layer(buf, fp8_experts=True), _x()
    with torch.no_grad():
        old = layer(x)
        _write(layer, 'data')
        layer.quantize_weights()
        fresh = _layer(buf, fp8_experts=True)
        fresh.load_state_dict(layer.state_dict())
        y = layer(x)
        assert torch.equal(y, fresh(x)) and not torch.equal(y, old)
    buf.check()
    buf.destroy()
