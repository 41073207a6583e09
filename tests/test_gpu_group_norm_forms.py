"""Group norm in the forms that only large inputs take, against the definition in 64 bits (y, dx, dw, db), with the tolerances of test_gpu_group_norm.py."""
import pytest
import torch

from test_gpu_group_norm import check, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,B", [(torch.float32, 2), (torch.bfloat16, 3)])
def test_as_many_groups_as_there_may_be_channels(ops, dtype, B):
    """2^22 groups of one channel: a wave has 64 of them, so the rows' backward has 65536 sets of groups, one more than a launch's y takes."""
    check(ops, (B, 1 << 22), 1 << 22, dtype, act="silu")
