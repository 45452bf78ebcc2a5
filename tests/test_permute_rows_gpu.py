"""Rows of sorted_src behind the last routed one, which dropped entries leave over."""

import pytest
import torch

from src import _lib, router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_permute_leaves_readable_rows_behind_the_last():
    """gather_rows takes every row of sorted_src, dropped entries or not."""
    junk = [torch.full((4096,), 2 ** 30, dtype=torch.int32, device=DEV) for _ in range(8)]
    del junk                                                       # memory with far indexes in it, to be reused
    ids = torch.full((1000, 4), -1, dtype=torch.int32, device=DEV)
    ids[:10] = torch.arange(4, dtype=torch.int32, device=DEV)
    gs, src, inv = router.permute(ids, 8)
    torch.cuda.synchronize()
    assert torch.all(src[int(gs.sum()):] == 0)
    _lib.device_status(reset=True)
