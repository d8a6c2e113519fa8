"""How exact attention of one token over pages is, where looser bounds would not show a part of the arithmetic that is missing or cut off, against the same
mathematics in 64 bits."""
import pytest
import torch
from test_gpu_paged import Pool, decode_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", ["u8", "u4"])
def test_heads_of_a_group_of_very_different_queries(gpu, store, D):
    """Codes: heads share a KV head's rows and nothing else. What a head's queries are rounded by goes by that head: beside one 2^40 times as large (more than fp16
    spans), and beside one of zeros, the others keep the bounds of a head alone, and give the bits that they give there."""
    print("queries", store, D, flush=True)
    pool = Pool(gpu, store, [300, 33, 1], 2, D, 16, seed=D)
    q = torch.randn(3, 16, D, generator=pool.gen)
    factor = 2.0 ** torch.tensor([0, 20, -20, 0, 40, -30, 0, -200])
    factor[3] = 0.0
    q = (q * factor.repeat(2)[:, None]).to(pool.dtype)
    _, out, lse = decode_and_check(pool, gpu, 16, q=q)
    alone = q.clone()
    alone[:, [1, 4, 9, 12]] = 0.0
    got, got_lse = pool.buffers.decode(alone.to(gpu), pool.table_gpu, pool.lens_gpu, return_lse=True)
    keep = [0, 2, 3, 5, 6, 7, 8, 10, 11, 13, 14, 15]
    assert torch.equal(got[:, keep], out[:, keep]) and torch.equal(got_lse[:, keep], lse[:, keep])
