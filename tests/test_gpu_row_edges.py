"""group_rows where its workgroups' memory passes a border."""
import pytest
import torch

from sfnx_amd import moe
from tests.rows_util import *  # noqa: F401,F403
from tests.test_gpu_rows import check_groups

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [0, 700])
@pytest.mark.parametrize("G", [2190, 2191, 2335, 2336, 2338, 2340, 2341])
def test_groups_about_64_kb(G, n):
    """28 bytes a group and 144 more pass 64 KB from 2336 groups on, without them from 2341 on"""
    ids = torch.randint(-1, G, (n,), generator=gen(G), dtype=torch.int32)
    g = moe.RowGroups(n, G)
    moe.group_rows(ids.cuda(), g)
    check_groups(ids.tolist(), g)
