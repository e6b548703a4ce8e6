"""The kept copy of the quantised weights, made in inference mode and renewed outside of it."""
import pytest
import torch

from deepep_trn_b200.models.moe import MoELayer
from test_moe_weights import Group, _equal, _ptrs, _write


@pytest.mark.parametrize('first,then', [(True, False), (False, True), (True, True)])
def test_copy_is_renewed_in_and_out_of_inference_mode(first, then):
    layer = MoELayer(Group(), 256, 128, 4, 2, fp8_block=True)
    with torch.inference_mode(first):
        layer.quantize_weights()
        kept = layer._block_weights(False)
        assert _equal(kept, layer)
    _write(layer, 'no_grad')
    with torch.inference_mode(then):
        layer.quantize_weights()
        assert _ptrs(layer._block_weights(False)) == _ptrs(kept) and _equal(kept, layer)
