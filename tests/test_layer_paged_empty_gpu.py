"""A layer call whose rows belong to no sequence is refused: there is no attention output for what follows to read."""
import pytest
import torch

from test_layer_paged_gpu import setup

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_layer_without_sequences_is_refused(pkg):
    T, D, HQ, HKV, DH, HID = 32, 256, 4, 2, 64, 512
    L, layout, cache, table, drv, g = setup(pkg, T, D, HQ, HKV, DH, HID, True, False, 16, torch.float16, 1)
    i32 = dict(dtype=torch.int32, device=DEV)
    batch = pkg.PagedBatch(torch.zeros(0, 4, **i32), torch.zeros(1, **i32), torch.zeros(0, **i32))
    tokens, cos = torch.ones(T, D, device=DEV), torch.ones(T, DH // 2, device=DEV)
    out = torch.full_like(tokens, 7.0)
    with pytest.raises(pkg.W8A8Error, match="of 0 sequences"):
        drv.forward_paged(drv.pack(L), tokens, cos, cos, cache, batch, out=out)
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())
    drv.close()
