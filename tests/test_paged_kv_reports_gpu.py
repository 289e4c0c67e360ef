"""What the report of a kernel says names what the caller has to look at."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_position_outside_the_rotation_tables_is_named(pkg):
    """A token at position 20 with tables of 20 rows: not appended, reported once; position 19 is appended."""
    i32 = dict(dtype=torch.int32, device=DEV)
    x, tables = torch.ones(1, 1, 64, device=DEV).half(), torch.ones(20, 32, device=DEV)
    kw = dict(rope_cos=tables, rope_sin=tables, rope_order=pkg.ROPE_HALVES, rope_by_position=True)
    pages = [torch.zeros(2, 1, 16, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
    cache = pkg.PagedKVCache(*pages)
    batches = [pkg.PagedBatch(torch.tensor([[0, 1]], **i32), torch.tensor([0, 1], **i32), torch.tensor([n], **i32)) for n in (20, 21)]
    pkg.kv_append(cache, batches[1], x, x, **kw)
    torch.cuda.synchronize()
    with pytest.raises(pkg.W8A8Error, match="outside its rotation tables"):
        pkg.kv_append(cache, batches[0], x, x, **kw)
    assert not bool(pages[1].any())
    pkg.kv_append(cache, batches[0], x, x, **kw)
    torch.cuda.synchronize()
    assert pkg.poll_status() == 0
    assert bool((pages[1][1, 0, 3] == 1).all()) and int(pages[1].count_nonzero()) == 64
