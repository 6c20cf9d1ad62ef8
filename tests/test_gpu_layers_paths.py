"""Layer operators on sizes that take paths of their own: groups of several whole waves side by side, packed sequences in fp16."""
import pytest
import torch

from . import test_gpu_gated as gated
from . import test_gpu_group_norm as norm

pytestmark = pytest.mark.gpu


# (columns of a group are multiples of 64 slots of 16 bytes, several groups to a workgroup)
@pytest.mark.parametrize("dtype,shape,groups", [(torch.float32, (4, 2, 1024), 4), (torch.float32, (3, 7, 1536), 3), (torch.bfloat16, (4, 2, 2048), 4),
                                                (torch.float16, (5, 3, 3584), 7), (torch.float32, (600, 2, 512), 2), (torch.bfloat16, (300, 5, 1024), 2)])
def test_groups_of_whole_waves(shape, groups, dtype):
    x, d_y, weight, bias = norm.make(shape, dtype, seed=sum(shape))
    norm.check(x, d_y, weight, bias, groups, "silu")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("bounds", gated.BOUNDS, ids=lambda b: "-".join(map(str, b)))
def test_packed_sequences_in_half_precision(bounds, reverse):
    gated.check(gated.make((bounds[-1], 67), torch.float16, seed=len(bounds), sequences=len(bounds) - 1), torch.float16, reverse, bounds)
