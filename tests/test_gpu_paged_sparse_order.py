"""The sums behind the choice of pages: the same for a page wherever it lies and however the work is split, also where another order of summation would give others.

A sum of products in 64 bits is off by D * 2^-53 of its sum of magnitudes, and its rounding to 32 bits sees 2^-24 of what is left: where large terms cancel, two orders round differently."""
import pytest
import torch

from keys_values_amd.attention import ops

pytestmark = pytest.mark.gpu


def cancelling(kinds, Hkv, group, D, dtype, gen, gpu):
    """(q, bounds of `kinds` pages) with pairs of terms of 2^40 that cancel beside terms of 1 and less."""
    q = torch.randn(1, Hkv * group, D, generator=gen)
    keys = torch.randn(kinds, Hkv, D, generator=gen)
    size = 2.0**20 if dtype == torch.bfloat16 else 2.0**14  # of either factor
    at = torch.randperm(D, generator=gen)[: D // 4]
    q[..., at] *= size
    keys[..., at] *= size
    half = at[: D // 8], at[D // 8 :]
    q[..., half[1]] = q[..., half[0]]
    keys[..., half[1]] = -keys[..., half[0]]
    return q.to(dtype).to(gpu), torch.stack((keys, keys), 2).to(dtype).to(gpu)


@pytest.mark.parametrize("group", [1, 4, 5, 16])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16), (256, torch.bfloat16)])
def test_pages_alike_tie_wherever_they_lie(gpu, D, dtype, group):
    """Pages of a few kinds all over the table: of a kind the front ones are chosen, and one kind at most is chosen in part. The kernel for few pages chooses as the kernels for
    many do, and a sequence alone as in a batch."""
    print("order", D, dtype, group, flush=True)
    gen = torch.Generator().manual_seed(D + group)
    Hkv, kinds, page = 2, 9, 16
    q, bounds = cancelling(kinds, Hkv, group, D, dtype, gen, gpu)
    products = q.view(Hkv, group, 1, D).double().cpu() * bounds[:, :, 0].transpose(0, 1)[:, None].double().cpu()  # there sums go one by one
    forward, backward = products.cumsum(-1)[..., -1].float(), products.flip(-1).cumsum(-1)[..., -1].float()
    assert (forward != backward).any()  # the order is seen
    for pages in (100, 128, 1000, 3001, 9000):
        table = torch.randint(0, kinds, (1, pages), generator=gen, dtype=torch.int32).to(gpu)
        lens = torch.tensor([pages * page], dtype=torch.int32, device=gpu)
        for count in (1, pages // 7, pages // 2):
            chosen = ops.paged_select(q, bounds, table, lens, page, count, 0, 0)
            for h in range(Hkv):
                mine = chosen[0, h].long()
                assert (mine >= 0).all()
                parts = 0
                for kind in range(kinds):
                    all_of = torch.nonzero(table[0] == kind)[:, 0]
                    some = mine[table[0, mine] == kind]
                    assert torch.equal(some, all_of[: len(some)])
                    parts += 0 < len(some) < len(all_of)
                assert parts <= 1
            # a wider table of more sequences, of which this one is the last
            wide = torch.randint(0, kinds, (7, pages + 200), generator=gen, dtype=torch.int32).to(gpu)
            wide[-1, :pages] = table[0]
            more = torch.randint(1, (pages + 200) * page, (7,), generator=gen, dtype=torch.int32).to(gpu)
            more[-1] = lens[0]
            assert torch.equal(ops.paged_select(q.expand(7, -1, -1), bounds, wide, more, page, count, 0, 0)[-1], chosen[0])


def test_bounds_the_wrong_way_round(gpu):
    """Where a lowest value exceeds the highest, positive queries meet the second and negative ones the first all the same."""
    gen = torch.Generator().manual_seed(3)
    Hkv, group, D, pages, page = 2, 3, 64, 300, 16
    q, bounds = torch.randn(1, Hkv * group, D, generator=gen).to(torch.bfloat16), torch.randn(pages, Hkv, 2, D, generator=gen).to(torch.bfloat16)
    heads = q.double().view(Hkv, group, 1, D)
    low, high = (bounds[:, :, i].transpose(0, 1)[:, None].double() for i in (0, 1))
    score = (heads.clamp(min=0) * high + heads.clamp(max=0) * low).sum(-1).float().amax(1)
    for n in (100, pages):
        table, lens = torch.arange(n, dtype=torch.int32)[None].to(gpu), torch.tensor([n * page], dtype=torch.int32, device=gpu)
        got = ops.paged_select(q.to(gpu), bounds.to(gpu), table, lens, page, 20, 0, 0)
        assert torch.equal(got[0].cpu().long(), score[:, :n].sort(dim=-1, descending=True, stable=True).indices[:, :20].sort(-1).values)
