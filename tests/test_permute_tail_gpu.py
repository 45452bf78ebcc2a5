"""moe_permute writes every row of sorted_src itself: through the C entry points
(route -> permute -> gather over all rows, as only the device knows how many
are routed), and without a launch of its own for the rows behind the last."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import moe_oracle as orc
from src import _lib, router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("T,k,E,drop", [(1, 1, 1, 1.0), (1, 3, 4, 0.0), (300, 4, 8, 0.5), (512, 1, 2, 0.002), (700, 3, 1024, 1.0),
                                        (5000, 8, 64, 0.3), (4096, 1, 7, 0.0), (100_000, 2, 256, 0.9)])
def test_every_row_is_written(T, k, E, drop):
    rng = np.random.default_rng(T + E)
    N = T * k
    ids = rng.integers(0, E, size=(T, k)).astype(np.int32)
    bad = rng.random((T, k)) < drop
    ids[bad] = rng.choice([-1, E, 2 ** 31 - 1, -2 ** 31], size=int(bad.sum())).astype(np.int32)
    L = _lib.lib()
    vp = ctypes.c_void_p
    dev_ids = torch.from_numpy(ids).to(DEV)
    gs = torch.full((E,), -5, dtype=torch.int32, device=DEV)
    src = torch.full((N,), max(0, N - 1), dtype=torch.int32, device=DEV)       # rows that could be read, but not 0
    inv = torch.full((N,), -9, dtype=torch.int32, device=DEV)
    need = int(L.moe_permute_workspace_size(N, E))
    ws = torch.full((need + 64,), 0x7e, dtype=torch.uint8, device=DEV)
    stream = vp(torch.cuda.current_stream().cuda_stream)
    assert L.moe_permute(vp(dev_ids.data_ptr()), N, E, vp(gs.data_ptr()), vp(src.data_ptr()), vp(inv.data_ptr()),
                         vp(ws.data_ptr()), need, stream) == 0
    x = torch.randn((T, 8), device=DEV)
    xs = torch.zeros((N, 8), device=DEV)
    assert L.moe_gather_rows(vp(x.data_ptr()), vp(src.data_ptr()), N, k, 32, vp(xs.data_ptr()), stream) == 0
    torch.cuda.synchronize()
    rgs, rsrc, rinv = orc.permute_by_expert(ids, E)
    n = int(rgs.sum())
    assert np.array_equal(gs.cpu().numpy(), rgs) and np.array_equal(inv.cpu().numpy(), np.asarray(rinv).reshape(-1))
    assert np.array_equal(src.cpu().numpy(), np.concatenate([rsrc, np.zeros(N - n, rsrc.dtype)]))
    assert torch.equal(xs, x[src.long() // k]) and torch.all(ws[need:] == 0x7e)
    if drop:
        _lib.device_status(reset=True)


def test_three_launches_and_no_fill():
    from torch.profiler import ProfilerActivity, profile
    ids = torch.randint(0, 8, (500, 2), dtype=torch.int32, device=DEV)
    router.permute(ids, 8)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        router.permute(ids, 8)
        torch.cuda.synchronize()
    events = [e for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA]
    if not events:
        pytest.skip("the profiler recorded no GPU activity on this box")
    assert len(events) == 3 and all("perm_" in e.name for e in events), [e.name for e in events]
