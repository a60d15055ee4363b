"""How long a list kvq_page_copy_launch takes, without a GPU: what it refuses and
what gets past its checks (to the device's, which there is none of)."""
import pytest
import torch

from test_pages_cpu import INVALID, launch
from test_share_cpu import copy


@pytest.mark.parametrize("kw", [dict(copies=1 << 24, num_pages=1 << 26), dict(copies=1 << 20, num_pages=(1 << 20) - 1, layers=16),
                                dict(copies=1 << 19, num_pages=1 << 19, layers=1 << 12), dict(copies=(1 << 24) - 1, layers=65535)])
def test_refused(kw):
    assert launch("kvq_page_copy_launch", copy(**kw)) == INVALID


@pytest.mark.skipif(torch.cuda.is_available(), reason="stand-in pointers are not for a device")
@pytest.mark.parametrize("kw", [dict(copies=1 << 19, num_pages=1 << 19, layers=32), dict(copies=1 << 18, num_pages=1 << 18, layers=64),
                                dict(copies=(1 << 24) - 1, num_pages=1 << 26, layers=100), dict(copies=1 << 20, num_pages=9, layers=15)])
def test_taken(kw):
    assert launch("kvq_page_copy_launch", copy(**kw)) not in (0, INVALID)
