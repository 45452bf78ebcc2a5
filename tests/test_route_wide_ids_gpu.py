"""Given experts in every integer type: an id that 32 bits would wrap is out of range, not another expert."""

import pytest
import torch

from src import router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16,
                                   torch.uint32, torch.uint64])
def test_given_ids_of_any_integer_type(dtype):
    x = torch.randn((6, 8), device=DEV)
    ids = torch.tensor([[0, 1], [2, 3], [7, 0], [5, 5], [6, 2], [1, 4]])
    want = router.route_forward_train(x, 2, ids=ids.to(DEV))
    info = torch.iinfo(dtype)
    wide = ids.clone()
    far = [(0, 1, info.max)] if info.bits < 64 else [(0, 1, 2 ** 32 + 3), (2, 0, 2 ** 40 + 7)]
    for t, j, v in far:
        wide[t, j] = v
    got = router.route_forward_train(x, 2, ids=wide.to(dtype).to(DEV))
    drop = torch.zeros((6, 2), dtype=torch.bool)
    for t, j, _ in far:
        drop[t, j] = True
    assert torch.equal(got.ids.cpu(), torch.where(drop, -1, want.ids.cpu()))
