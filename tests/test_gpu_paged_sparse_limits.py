"""The sparse paged operators at the sizes where one launch, one window of sequences or one kernel ends; references on the device, in 64 bits where numbers are computed."""
import math

import pytest
import torch

from keys_values_amd.attention import ops
from keys_values_amd.kvcache.paged import PagedKVCacheBuffers, paged_bounds
from keys_values_amd.longctx import ops as rows

from test_gpu_paged import check_decode
from test_gpu_paged_sparse import append_both_ways, bits_of, check_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hkv,D,page", [(65535, 1, 64, 16), (300, 3, 128, 32), (64, 2, 64, 256), (65, 2, 256, 64), (129, 1, 64, 1024)])
@pytest.mark.parametrize("tokens", [None, 1, 20])
def test_bounds_of_many_sequences(gpu, B, Hkv, D, page, tokens):
    """A page or two of every sequence, in tables with room for more."""
    print("bounds", B, Hkv, D, page, tokens, flush=True)
    gen = torch.Generator(device=gpu).manual_seed(B)
    k = torch.randn(2 * B, Hkv, page, D, generator=gen, dtype=torch.float16, device=gpu)
    lens = torch.randint(0, 2 * page + 1, (B,), generator=gen, dtype=torch.int32, device=gpu)
    lens[B // 2], lens[-1] = 2 * page, 1
    table = torch.full((B, 7), -1, dtype=torch.int32, device=gpu)
    table[:, :2] = torch.randperm(2 * B, generator=gen, device=gpu).view(B, 2)
    bounds = torch.full((2 * B, Hkv, 2, D), 9.5, dtype=torch.float16, device=gpu)
    paged_bounds(k, bounds, table, lens, tokens)
    want = torch.full_like(bounds, 9.5)
    for i in range(2):
        looked = (lens > i * page) & ((i + 1) * page > lens - (10**9 if tokens is None else tokens))
        at, n = table[looked, i].long(), lens[looked]
        behind = (torch.arange(page, device=gpu)[None] + i * page >= n[:, None])[:, None, :, None]
        for side, fill in ((0, math.inf), (1, -math.inf)):
            x = k[at].masked_fill(behind, fill)
            want[at, :, side] = x.amin(2) if side == 0 else x.amax(2)
    assert torch.equal(bounds, want)


@pytest.mark.parametrize("B,Hkv,group,width", [(65535, 2, 1, 3), (20000, 2, 4, 130), (9000, 5, 2, 128), (70, 1, 16, 600), (1100, 2, 1, 1001), (600, 2, 2, 2048), (300, 2, 2, 4095),
                                               (270, 1, 1, 8192), (300, 1, 4, 8200), (140, 1, 1, 16383), (70, 1, 2, 32767)])
def test_select_of_many_sequences(gpu, B, Hkv, group, width):
    """Any sequences over a pool of few pages."""
    print("select", B, Hkv, group, width, flush=True)
    gen = torch.Generator(device=gpu).manual_seed(width)
    P, D, page, count, first, last = 50, 64, 16, min(20, width), 1, 1
    bounds = torch.randn(P, Hkv, 2, D, generator=gen, dtype=torch.float32, device=gpu).sort(2).values.to(torch.bfloat16)
    q = torch.randn(B, Hkv * group, D, generator=gen, dtype=torch.float32, device=gpu).to(torch.bfloat16)
    table = torch.randint(-1, P + 1, (B, width), generator=gen, dtype=torch.int32, device=gpu)
    lens = torch.randint(-3, width * page + 40, (B,), generator=gen, dtype=torch.int32, device=gpu)
    got = ops.paged_select(q, bounds, table, lens, page, count, first, last)
    q64, b64 = q.double().view(B, Hkv, group, D), bounds.double()
    score = torch.full((B, Hkv, P), -math.inf, device=gpu)
    for h in range(Hkv):
        s = q64[:, h].clamp(min=0).flatten(0, 1) @ b64[:, h, 1].T + q64[:, h].clamp(max=0).flatten(0, 1) @ b64[:, h, 0].T
        score[:, h] = s.float().view(B, group, P).amax(1)
    n = ((lens.clamp(min=0) + page - 1) // page).clamp(max=width)[:, None]
    i = torch.arange(width, device=gpu)
    there = (table >= 0) & (table < P) & (i < n)
    rank = score.gather(2, table.clamp(0, P - 1).long()[:, None].expand(B, Hkv, width))
    rank = torch.where(((i < first) | (i >= n - last))[:, None], math.inf, rank).masked_fill(~there[:, None], -math.inf)
    best = rank.sort(dim=-1, descending=True, stable=True)
    want = torch.where(best.values == -math.inf, width, best.indices)[..., :count].sort(-1).values
    assert torch.equal(got, torch.where(want == width, -1, want).to(torch.int32))


@pytest.mark.parametrize("B,Hkv,bits,count", [(65535, 2, None, 2), (33000, 3, 8, 3), (20000, 1, 4, 40)])
def test_chosen_of_many_sequences(gpu, B, Hkv, bits, count):
    """Sequences over a pool of few pages, a sample of them against 64 bits."""
    print("chosen", B, Hkv, bits, flush=True)
    gen = torch.Generator().manual_seed(B)
    buffers = PagedKVCacheBuffers(50, 16, Hkv, 64, torch.bfloat16, bits, gpu)
    key, value = (torch.randn(800, Hkv, 64, generator=gen).to(torch.bfloat16).to(gpu) for _ in range(2))
    buffers.write(key, value, torch.arange(800, device=gpu))
    width = 2 * count
    table = torch.randint(0, 50, (B, width), generator=gen, dtype=torch.int32).to(gpu)
    lens = torch.randint(0, width * 16 + 1, (B,), generator=gen, dtype=torch.int32).to(gpu)
    chosen = torch.argsort(torch.rand(B, Hkv, width, generator=gen), -1)[..., :count].to(torch.int32)
    q = torch.randn(B, 2 * Hkv, 64, generator=gen).to(torch.bfloat16)
    out, lse = buffers.decode(q.to(gpu), table, lens, return_lse=True, chosen=chosen.to(gpu))
    pages = torch.arange(50, dtype=torch.int32, device=gpu)[:, None]
    k, v = (x.double().cpu() for x in buffers.read(pages, torch.full((50,), 16, dtype=torch.int32, device=gpu), 16))
    spans = None if bits is None else (buffers.quant.v_scale.cpu() * (1 << bits))
    for b in (0, 1, B // 3, B // 2, B - 2, B - 1):
        n = int(lens[b])
        for h in range(Hkv):
            P = -(-n // 16)
            at = [(int(table[b, i]), t) for i in chosen[b, h, :P].tolist() if i < P for t in range(min(16, n - 16 * i))]
            p, t = (torch.tensor([x[j] for x in at], dtype=torch.long) for j in (0, 1))
            mine = slice(2 * h, 2 * h + 2)
            if bits is None:
                check_decode(out[b, mine].cpu(), lse[b, mine].cpu(), q[b, mine], k[p, h, t][None], v[p, h, t][None], 0.125, torch.bfloat16)
            elif n:
                stored = [(x.cpu()[p, h, t]) for x in (buffers.k, buffers.v)]
                if bits == 4:
                    stored = [torch.cat((x >> 4, x & 15), -1) for x in stored]
                r = [(x.long() - buffers.quant[2 * j + 1].cpu()[p, h, t][:, None]).double() * buffers.quant[2 * j].cpu()[p, h, t].double()[:, None] for j, x in enumerate(stored)]
                if len(p):
                    check_decode(out[b, mine].cpu(), lse[b, mine].cpu(), q[b, mine], r[0][None], r[1][None], 0.125, torch.bfloat16, spans[p, h, t][None])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("store", ["bf16", "u8"])
def test_append_around_the_split_of_tokens(gpu, store):
    """Where a token's rows move from several workgroups to one, for heads that fill one, two, three rows a lane and more."""
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    for tokens in (2 * cus, 2 * cus + 1):
        for Hq, Hkv, D in ((1, 1, 64), (12, 2, 128), (30, 5, 128), (28, 4, 256), (96, 8, 128), (128, 2, 256)):
            qkv, got, want, _ = append_both_ways(gpu, store, tokens, Hq, Hkv, D, 16, D, False, True, seed=Hq)
            check_append(qkv, got, want, Hq, D)


def test_heads_of_zeros_do_not_change_their_neighbours(gpu):
    """Without an epsilon a head of zeros is divided by zero; the heads beside it are normalised as they are elsewhere, in one call and in two."""
    gen = torch.Generator().manual_seed(5)
    tokens, Hq, Hkv, D, page = 40, 6, 2, 64, 16
    cos, sin = rows.rope_tables(100, D, 1e4, gpu)
    w = (1 + 0.2 * torch.randn(D, generator=gen)).to(gpu)
    x = torch.randn(tokens, Hq + 2 * Hkv, D, generator=gen).to(torch.bfloat16)
    zeros = torch.rand(tokens, Hq + Hkv, generator=gen) < 0.2
    y = x.clone()
    y[:, : Hq + Hkv][zeros] = 0.0
    y[::3, -Hkv:] = 0.0  # value heads are not normalised
    positions = torch.randint(0, 100, (tokens,), generator=gen, dtype=torch.int32).to(gpu)
    slots = torch.randperm(3 * page, generator=gen)[:tokens].to(gpu)
    alone, beside, one = x.flatten(1).to(gpu), y.flatten(1).to(gpu), y.flatten(1).to(gpu)
    for t in (alone, beside):
        rows.rotary_(t, Hq, Hkv, D, w, w, 0.0, cos, sin, positions)
    a, b = (t.view(tokens, -1, D)[:, : Hq + Hkv].cpu() for t in (alone, beside))
    assert torch.equal(a[~zeros], b[~zeros]) and torch.isnan(b[zeros]).all()
    pool = PagedKVCacheBuffers(3, page, Hkv, D, device=gpu)
    pool.append(one, Hq, w, w, 0.0, cos, sin, positions, slots)
    assert torch.equal(bits_of(one[:, : Hq * D]), bits_of(beside[:, : Hq * D]))
    assert torch.equal(bits_of(pool.k[slots // page, :, slots % page]), bits_of(beside.view(tokens, -1, D)[:, Hq:-Hkv]))
    assert torch.equal(pool.v[slots // page, :, slots % page], beside.view(tokens, -1, D)[:, -Hkv:])
