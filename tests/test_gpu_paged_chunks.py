"""Later chunks of the prompts of a ragged batch over a paged cache: rotated and written together, attended to one sequence a call."""
import pytest
import torch

from keys_values_amd.attention import ops
from keys_values_amd.kvcache.paged import PagedKVCacheBuffers
from keys_values_amd.longctx import ops as rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,dtype,D", [(None, torch.bfloat16, 128), (None, torch.float16, 64), (8, torch.bfloat16, 64), (4, torch.bfloat16, 128)])
def test_chunks_of_a_ragged_batch(gpu, bits, dtype, D):
    """Earlier tokens and chunks of different lengths, one prompt beginning; every chunk sees the rows before it and itself, causally. In 64 bits over the rows that
    the cache hands back; a weight and the output are rounded to the type, once each, and logits are off by (D + 8) 2^-24 sum |q k|."""
    Hq, Hkv, page = 8, 2, 16
    earlier, chunk = [130, 0, 37, 5], [40, 33, 1, 70]
    gen = torch.Generator().manual_seed(D)
    u = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-11
    cos, sin = rows.rope_tables(300, D, 1e6, gpu, rotary_dim=D)
    buffers = PagedKVCacheBuffers(60, page, Hkv, D, dtype, bits, gpu)
    table = torch.randperm(60, generator=gen)[:52].view(4, 13).to(torch.int32).to(gpu)
    lens = torch.zeros(4, dtype=torch.int32, device=gpu)
    for part, attend in ((earlier, False), (chunk, True)):
        packed = torch.randn(sum(part), (Hq + 2 * Hkv) * D, generator=gen).to(dtype).to(gpu)
        seq = torch.repeat_interleave(torch.arange(4), torch.tensor(part)).to(gpu)
        first = (torch.tensor(part).cumsum(0) - torch.tensor(part)).to(gpu)
        positions = torch.arange(sum(part), device=gpu) - first[seq] + lens[seq]
        rows.rotary_(packed, Hq, Hkv, D, None, None, 0.0, cos, sin, positions.to(torch.int32))
        heads = packed.view(-1, Hq + 2 * Hkv, D)
        slots = table[seq, positions // page].long() * page + positions % page
        buffers.write(heads[:, Hq : Hq + Hkv], heads[:, Hq + Hkv :], slots)
        lens += torch.tensor(part, dtype=torch.int32, device=gpu)
    host = lens.tolist()
    assert host == [a + b for a, b in zip(earlier, chunk)]
    k_all, v_all = buffers.read(table, lens, max(host))
    for b, (before, n) in enumerate(zip(earlier, chunk)):
        k, v = buffers.read(table[b : b + 1], lens[b : b + 1], host[b])
        assert torch.equal(k[0], k_all[b, :, : host[b]]) and torch.equal(v[0], v_all[b, :, : host[b]])
        assert (k_all[b, :, host[b] :] == 0).all()
        q = heads[int(first[b]) : int(first[b]) + n, :Hq].transpose(0, 1)[None]
        out = ops.prefill_core(q, k, v, D**-0.5, before)[0]
        q64, k64, v64 = q[0].double().cpu(), *(x[0].double().cpu().repeat_interleave(Hq // Hkv, 0) for x in (k, v))
        hidden = torch.arange(host[b])[None] > before + torch.arange(n)[:, None]
        p = torch.softmax((q64 @ k64.transpose(1, 2) * D**-0.5).masked_fill(hidden, -torch.inf), -1)
        want, size = p @ v64, p @ v64.abs()
        moved = 2 * (D + 8) * 2.0**-24 * (q64.abs() @ k64.abs().transpose(1, 2)).amax(-1, keepdim=True) * D**-0.5
        tol = u * want.abs() + (u + moved + 2.0**-16) * size * (1 + u) + 2.0**-24
        err = (out[0].transpose(0, 1).double().cpu() - want).abs()
        assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} tolerances"
