"""Arguments that the memory-lean operators refuse by their own checks."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import act8_unpack


def test_a_number_is_no_checkpoint():
    z = torch.zeros(())
    with pytest.raises(ValueError):
        act8_unpack(z.to(torch.float8_e4m3fn), z.to(torch.uint8).view(torch.float8_e8m0fnu), 1)
