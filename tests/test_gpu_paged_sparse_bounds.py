"""What the bounds of a page say about its keys' products with a query, page for page: scores that count the keys as the store's 16-bit type rounds them.

Slack, relative to a key's sum of |q[d] k[d]|: the two sums of the reference, in 64 bits, are each off by D * 2^-53 of it at most. Rows of codes are products of 32 bits (2^-24 of a value) that
are rounded to 16 bits, half a step: 2^-8 of a bfloat16 value, 2^-11 of a float16 one, or 2^-25 where that is more (float16 below 2^-14)."""
import pytest
import torch

from test_gpu_paged import HALF_STEP, STORES, Pool
from test_gpu_paged_sparse import bounds_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("store", STORES)
def test_products_of_every_pages_keys(gpu, store, D):
    """Plain rows: none exceeds its own page's score. Rows of codes, which attention takes unrounded: some do, in pages of one token about every second, by no more than the
    rounding."""
    print("products", store, D, flush=True)
    Hkv, group, page = 2, 3, 16
    pool = Pool(gpu, store, [700] + [page * i + 1 for i in range(40)], Hkv, D, page, seed=D)
    bounds = bounds_of(pool, gpu).double()
    above = 0
    for b, n in enumerate(pool.lens):
        q = torch.randn(Hkv, group, D, generator=pool.gen).to(pool.dtype).double()
        for i in range(-(-n // page)):
            low, high = bounds[int(pool.table[b, i])].unbind(1)  # (Hkv, D)
            score = torch.maximum(q * low[:, None], q * high[:, None]).sum(-1)  # (Hkv, group)
            keys = pool.rows[0][b][:, i * page : (i + 1) * page].transpose(1, 2)
            product, size = q @ keys, q.abs() @ keys.abs()
            slack = 2 * D * 2.0**-53 * size
            if pool.bits:
                slack = slack + (HALF_STEP[pool.dtype] * (1 + 2.0**-23) + 2.0**-24) * size
                if pool.dtype == torch.float16:
                    slack = slack + 2.0**-25 * q.abs().sum(-1, keepdim=True)
            assert (product <= score[..., None] + slack).all()
            above += int((product > score[..., None] + 2 * D * 2.0**-53 * size).any())
    assert above > 0 if pool.bits else above == 0
