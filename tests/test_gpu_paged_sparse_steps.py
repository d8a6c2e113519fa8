"""Steps of sparse attention as a server makes them: captured ones replayed over tables that have changed, several new tokens of a sequence at once."""
import math

import pytest
import torch

from test_gpu_paged import STORES, check_decode, stored_rows, stored_spans
from test_gpu_paged_sparse import SparseLayer, want_chosen

pytestmark = pytest.mark.gpu


def relocate(layer, gen):
    """All of the pool's pages to other places, with their state and bounds, and two sequences to each other's rows of the table: in place, as a captured step reads them."""
    b = layer.buffers
    to = torch.randperm(b.num_pages, generator=gen).to(layer.table.device)
    for t in (b.k, b.v, *(b.quant or ()), b.bounds):
        moved = torch.empty_like(t)
        moved[to] = t
        t.copy_(moved)
    rows = to[layer.table.long()].to(torch.int32)
    lens = layer.lens.clone()
    order = torch.randperm(layer.B, generator=gen).to(rows.device)
    layer.table.copy_(rows[order])
    layer.lens.copy_(lens[order])


@pytest.mark.parametrize("store", ["bf16", "u8", "u4_fp16"])
def test_captured_steps_over_other_tables(gpu, store):
    """Replays over pages that have moved and sequences that have changed places, each checked against 64 bits and the eager calls."""
    layer = SparseLayer(gpu, store, [130, 0, 2000, 1], 8, 2, 128, 16, 40, count=40)
    gen = torch.Generator().manual_seed(41)
    layer.next()
    layer.step()  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    layer.next()
    with torch.cuda.graph(graph):
        chosen, out, lse = layer.step()
    before = layer.table.clone()
    for _ in range(4):
        relocate(layer, gen)
        assert not torch.equal(layer.table, before)
        before = layer.table.clone()
        layer.next()
        graph.replay()
        torch.cuda.synchronize()
        layer.check(chosen, out, lse)
        q = layer.qkv.view(layer.B, -1, 128)[:, :8]
        again = layer.buffers.select(q, layer.table, layer.lens, 40)
        assert torch.equal(again, chosen)
        eager = layer.buffers.decode(q, layer.table, layer.lens, return_lse=True, chosen=again)
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)


@pytest.mark.parametrize("new", [2, 5, 20])
@pytest.mark.parametrize("store", STORES)
def test_several_new_tokens_of_a_sequence(gpu, store, new):
    """Appended in one call, bounds brought up to date once with all of them, then a row of the table and a length for each token: every token chooses for itself and attends
    to what is in front of it and to itself. Bounds of a page that later tokens lie in too allow more than its earlier keys do."""
    print("several", store, new, flush=True)
    Hq, Hkv, D, page, count = 6, 2, 128, 16, 9
    layer = SparseLayer(gpu, store, [14, 300, 1, 47], Hq, Hkv, D, page, 42, count=count)
    B, b, dtype = layer.B, layer.buffers, layer.buffers.dtype
    positions = (layer.lens[:, None] + torch.arange(new, device=gpu)).to(torch.int32)  # (B, new)
    qkv = torch.randn(B, new, (Hq + 2 * Hkv) * D, generator=layer.gen).to(dtype).to(gpu)
    b.append(qkv, Hq, layer.qw, layer.kw, 1e-6, layer.cos, layer.sin, positions, b.slots(layer.table, positions))
    b.update_bounds(layer.table, layer.lens + new, tokens=new)
    q = qkv.view(B * new, -1, D)[:, :Hq]
    table, lens = layer.table.repeat_interleave(new, 0), (positions + 1).flatten()
    chosen = b.select(q, table, lens, count, 1, 2)
    out, lse = b.decode(q, table, lens, return_lse=True, chosen=chosen)
    assert torch.equal(chosen.cpu(), want_chosen(q, b.bounds, table, lens, page, count, 1, 2))
    G = Hq // Hkv
    for i, n in enumerate(lens.tolist()):
        pages = table[i].cpu()
        k, v = (stored_rows(b, j, pages, n) for j in (0, 1))
        spans = stored_spans(b, pages, n)
        for h in range(Hkv):
            some = [u for u in chosen[i, h].tolist() if u >= 0]
            assert -(-n // page) - 1 in some  # the page of the token itself
            at = torch.cat([torch.arange(u * page, min(n, (u + 1) * page)) for u in some])
            mine = slice(h * G, h * G + G)
            check_decode(out[i, mine].cpu(), lse[i, mine].cpu(), q[i, mine].cpu(), k[h : h + 1, at], v[h : h + 1, at], D**-0.5, dtype, None if spans is None else spans[h : h + 1, at])
    for i, n in enumerate((layer.lens + new).tolist()):
        k = stored_rows(b, 0, layer.table[i].cpu(), n)
        for u in range(-(-n // page)):
            mine = k[:, u * page : (u + 1) * page]
            assert torch.equal(b.bounds[int(layer.table[i, u])].cpu(), torch.stack((mine.amin(1), mine.amax(1)), 1).to(dtype))
    assert math.isfinite(lse.sum().item())
