"""Steps of sparse attention as a server makes them: captured ones replayed over tables that have changed."""
import pytest
import torch

from test_gpu_paged_sparse import SparseLayer

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
