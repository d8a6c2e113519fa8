"""Calls of the paged cache at the sizes where one launch ends."""
import pytest
import torch

from keys_values_amd.kvcache.paged import PagedKVCacheBuffers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hkv,bits", [(4100, 16, None), (65535, 2, None), (33000, 3, 8)])
def test_read_of_many_sequences(gpu, B, Hkv, bits):
    """More (sequence, head) pairs than a grid has rows. Rows of a sequence are those of its one page, of which there are a few."""
    print("read", B, Hkv, bits, flush=True)
    gen = torch.Generator().manual_seed(B)
    buffers = PagedKVCacheBuffers(50, 16, Hkv, 64, torch.bfloat16, bits, gpu)
    key, value = (torch.randn(800, Hkv, 64, generator=gen).to(torch.bfloat16).to(gpu) for _ in range(2))
    buffers.write(key, value, torch.arange(800, device=gpu))
    table = torch.randint(-1, 51, (B, 2), generator=gen, dtype=torch.int32).to(gpu)
    lens = torch.randint(0, 20, (B,), generator=gen, dtype=torch.int32).to(gpu)
    length = 5
    k, v = buffers.read(table, lens, length)
    pages = torch.arange(50, dtype=torch.int32, device=gpu)[:, None]
    whole = buffers.read(pages, torch.full((50,), 16, dtype=torch.int32, device=gpu), length)  # every page as a sequence
    there = ((table[:, :1] >= 0) & (table[:, :1] < 50) & (torch.arange(length, device=gpu) < lens[:, None]))[:, None, :, None]
    for got, pages_of in zip((k, v), whole):
        want = torch.where(there, pages_of[table[:, 0].clamp(0, 49).long()], 0.0)
        assert torch.equal(got, want)
