"""Sizes of the gated block and of the packed gradient that are no whole numbers: no device is needed."""
import pytest
import torch

from eoq_quantization_b200 import gated

CODES, SCALES = torch.zeros(64, 64, dtype=torch.uint8), torch.ones(64, dtype=torch.float16)
X = torch.zeros(2, 128, dtype=torch.float16)


@pytest.mark.parametrize("sizes,error", [((64.0, 128, 4, 128), TypeError), ((64, None, 4, 128), TypeError), ((64, 128, "4", 128), TypeError),
                                         ((64, 128, 4, 128.0), TypeError), ((2 ** 70, 128, 4, 128), OverflowError)])
def test_sizes(sizes, error):
    with pytest.raises(error):
        gated.gated_packed(CODES, SCALES, CODES, SCALES, *sizes, X)
    with pytest.raises(error):
        gated.packed_input_grad(CODES, SCALES, *sizes, X[:, :64])
