"""More of what the 4-bit operators and the scored router refuse before anything is launched: no GPU."""
import pytest
import torch

from supersonic_b200.csrc import ops
from supersonic_b200.csrc.ops import KernelError
from test_fp4_refusals import OnDevice, current_device, z  # noqa: F401


def route(logits, e, w):
    ops.route_scored(logits, 8, e, w)


@pytest.mark.parametrize("logits, e, w", [
    (z(8), z(3, 2, dtype=torch.int32), z(3, 2)), (z(), z(3, 2, dtype=torch.int32), z(3, 2)), (z(3, 8), z(dtype=torch.int32), z()),
    (z(3, 8), z(3, dtype=torch.int32), z(3)), (z(2, 3, 8), z(3, 2, dtype=torch.int32), z(3, 2)), (z(3, 8), z(1, 3, 2, dtype=torch.int32), z(1, 3, 2)),
])
def test_route_refuses_tensors_of_other_dimensions(logits, e, w):
    with pytest.raises(KernelError):
        route(logits, e, w)
