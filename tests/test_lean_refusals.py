"""Arguments that the memory-lean operators refuse by their own checks."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import act8_unpack
from vodascheduler_amd.ops.linear_xent import linear_cross_entropy


def test_a_number_is_no_checkpoint():
    z = torch.zeros(())
    with pytest.raises(ValueError):
        act8_unpack(z.to(torch.float8_e4m3fn), z.to(torch.uint8).view(torch.float8_e8m0fnu), 1)


@pytest.mark.parametrize("dtype", [torch.complex64, torch.float32, torch.bool])
def test_labels_are_integers(dtype):
    with pytest.raises(TypeError):
        linear_cross_entropy(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=dtype))
