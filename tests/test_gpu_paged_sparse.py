"""Sparse attention over a paged cache on the device: append with rotation, bounds of pages, the choice of pages, attention over them, and a layer's step of the four.

Tolerances: attention over chosen pages is held to those of attention over all of a sequence's (test_gpu_paged.py), with the chosen rows as its rows. What an append
stores is, bit for bit, what rotary_ and paged_write store, which have tests of their own against 64 bits. Bounds and choices are exact: a minimum is one of the values
that paged_read gives, and scores are sums, in 64 bits, of products that 32 bits hold exactly (16-bit factors): over 512 of them two orders of summation differ
by 2^-53 * 512 of the sum of magnitudes at most, 2^-20 of what rounding to 32 bits is. Inputs whose scores come nearer than that to a border of
two 32-bit numbers would be a coincidence of one in a million, and the inputs are fixed."""
import math

import pytest
import torch

from keys_values_amd.attention import ops
from keys_values_amd.kvcache.paged import PagedKVCacheBuffers, paged_append, paged_bounds, paged_write
from keys_values_amd.longctx import ops as rows

from test_gpu_paged import STORES, Layer, Pool, check_decode, check_rotary, stored_rows, stored_spans

pytestmark = pytest.mark.gpu


def bits_of(t):
    return t.contiguous().view(torch.uint8)


# ---- append ---------------------------------------------------------------------------------------------------------


def append_both_ways(gpu, store, tokens, Hq, Hkv, D, page, part, interleaved, norm, seed=0, context=3000, odd=True, spread=True):
    """(qkv, pool) after the one call and after the two, from the same start."""
    dtype, bits = STORES[store]
    gen = torch.Generator().manual_seed(seed + tokens + D)
    pages = 2 * -(-tokens // page) + 1
    pools = [PagedKVCacheBuffers(pages, page, Hkv, D, dtype, bits, gpu) for _ in range(2)]
    for pool in pools:
        for t in (pool.k, pool.v):
            t.view(torch.uint8).fill_(0x5A)
    x = torch.randn(tokens, Hq + 2 * Hkv, D, generator=gen)
    if spread:
        x *= 2.0 ** torch.randint(-12, 8, (tokens, Hq + 2 * Hkv, 1), generator=gen)
    x[0, 0] = 0.25
    if tokens > 5:
        x[3, -1, 7], x[4, Hq] = math.nan, 0.0
    qkv = x.flatten(1).to(dtype).to(gpu)
    cos, sin = rows.rope_tables(context, D, 1e4, gpu, rotary_dim=part)
    positions = torch.randint(0, context, (tokens,), generator=gen, dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    if odd and tokens > 20:
        positions[2], positions[3], positions[5], positions[-1] = -1, context, 2**31 - 1, -(2**31)
        slots[5], slots[9], slots[10], slots[11], slots[12] = -1, -1, pages * page, -(2**62), 2**62
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=gen)).to(gpu) for _ in range(2)) if norm else (None, None)
    angles = (qw, kw, 1e-5, cos, sin, positions.to(gpu))
    one, two = qkv.clone(), qkv.clone()
    pools[0].append(one, Hq, *angles, slots.to(gpu), interleaved)
    rows.rotary_(two, Hq, Hkv, D, *angles, interleaved)
    heads = two.view(tokens, -1, D)
    there = (positions >= 0) & (positions < context)
    pools[1].write(heads[:, Hq:-Hkv], heads[:, -Hkv:], torch.where(there, slots, -1).to(gpu))
    return qkv, (one, pools[0]), (two, pools[1]), (angles, slots)


def check_append(qkv, got, want, Hq, D):
    (one, pool), (two, other) = got, want
    assert torch.equal(bits_of(one[:, : Hq * D]), bits_of(two[:, : Hq * D]))
    assert torch.equal(bits_of(one[:, Hq * D :]), bits_of(qkv[:, Hq * D :]))  # keys and values stay
    for a, b in zip((pool.k, pool.v, *(pool.quant or ())), (other.k, other.v, *(other.quant or ()))):
        assert torch.equal(bits_of(a), bits_of(b))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("D,part", [(64, 64), (64, 16), (128, 128), (128, 48), (256, 256), (256, 32)])
def test_append(gpu, D, part, store, interleaved, norm):
    print("append", D, part, store, interleaved, norm, flush=True)
    for tokens, Hq, Hkv, page in ((1, 1, 1, 16), (37, 7, 1, 16), (70, 9, 3, 64), (5, 64, 8, 1024)):
        qkv, got, want, _ = append_both_ways(gpu, store, tokens, Hq, Hkv, D, page, part, interleaved, norm)
        check_append(qkv, got, want, Hq, D)


@pytest.mark.parametrize("store,tokens,Hq,Hkv,D,page", [("bf16", 9000, 32, 8, 128, 64), ("u8", 5001, 28, 4, 128, 16), ("u4_fp16", 7000, 8, 2, 64, 32), ("fp16", 3000, 24, 8, 256, 128)])
def test_append_of_many_tokens(gpu, store, tokens, Hq, Hkv, D, page):
    print("append", store, tokens, flush=True)
    qkv, got, want, _ = append_both_ways(gpu, store, tokens, Hq, Hkv, D, page, D, False, True, spread=False)
    check_append(qkv, got, want, Hq, D)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("store,norm", [("bf16", True), ("fp16", False)])
def test_append_against_64_bits(gpu, store, norm, interleaved):
    """Queries where they were and keys where their slots say, against the rotation in 64 bits; values as they are."""
    tokens, Hq, Hkv, D, page = 50, 5, 2, 128, 16
    qkv, (one, pool), _, (angles, slots) = append_both_ways(gpu, store, tokens, Hq, Hkv, D, page, 64, interleaved, norm, odd=False, spread=False)
    heads = one.view(tokens, -1, D).clone()
    for i, pages in ((0, pool.k), (1, pool.v)):
        heads[:, Hq + i * Hkv : Hq + (i + 1) * Hkv] = pages[slots // page, :, slots % page]
    fine = torch.ones(tokens, dtype=torch.bool)
    fine[3] = False  # has a NaN among its values
    qw, kw, eps, cos, sin, positions = angles
    check_rotary(qkv[fine], heads.flatten(1)[fine], Hq, Hkv, D, qw, kw, eps, cos, sin, positions[fine.to(positions.device)], interleaved)


def test_append_of_views_and_batches(gpu):
    """Tokens in rows of a wider tensor, of two axes, pages whose heads lie behind their places."""
    gen = torch.Generator().manual_seed(4)
    B, n, Hq, Hkv, D, page = 3, 5, 4, 2, 128, 16
    wide = torch.randn(B, n, (Hq + 2 * Hkv) * D + 64, generator=gen).to(torch.bfloat16).to(gpu)
    before = wide.clone()
    qkv = wide[..., :-64]
    cos, sin = rows.rope_tables(100, D, 1e6, gpu)
    positions = torch.randint(-1, 100, (B, n), generator=gen, dtype=torch.int32).to(gpu)
    both = torch.zeros(9, page, 2, Hkv, D, dtype=torch.bfloat16, device=gpu)
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    slots = torch.randperm(9 * page, generator=gen)[: B * n].to(gpu)
    paged_append(qkv, Hq, Hkv, D, None, None, 0.0, cos, sin, positions, k, v, slots.view(B, n))
    want = before[..., :-64].contiguous()
    rows.rotary_(want, Hq, Hkv, D, None, None, 0.0, cos, sin, positions)
    assert torch.equal(wide[..., : Hq * D], want[..., : Hq * D]) and torch.equal(wide[..., Hq * D :], before[..., Hq * D :])
    stored = torch.zeros_like(both)
    heads = want.view(B * n, -1, D)
    paged_write(heads[:, Hq:-Hkv], heads[:, -Hkv:], stored[:, :, 0].transpose(1, 2), stored[:, :, 1].transpose(1, 2), torch.where(positions.flatten() >= 0, slots, -1))
    assert torch.equal(both, stored)
    none = torch.empty(0, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=gpu)
    paged_append(none, Hq, Hkv, D, None, None, 0.0, cos, sin, torch.empty(0, dtype=torch.int32, device=gpu), k, v, slots[:0])
    assert torch.equal(both, stored)


# ---- bounds ---------------------------------------------------------------------------------------------------------

MARK = 7.5


def bounds_of(pool, gpu, **kwargs):
    got = torch.full((pool.num_pages, pool.Hkv, 2, pool.D), MARK, dtype=pool.dtype, device=gpu)
    paged_bounds(pool.buffers.k, got, pool.table_gpu, pool.lens_gpu, quant=pool.buffers.quant, **kwargs)
    return got.cpu()


def want_bounds(pool, tokens=None):
    """Minimum and maximum of the rows in 64 bits, rounded: rounding keeps the order."""
    want = torch.full((pool.num_pages, pool.Hkv, 2, pool.D), MARK, dtype=torch.float64)
    for b, n in enumerate(pool.lens):
        for i in range(0 if tokens is None else max(0, n - tokens) // pool.page, -(-n // pool.page) if tokens != 0 else 0):
            x = pool.rows[0][b][:, i * pool.page : (i + 1) * pool.page]
            if 0 <= int(pool.table_gpu[b, i]) < pool.num_pages:
                want[int(pool.table_gpu[b, i])] = torch.stack((x.amin(1), x.amax(1)), 1)
    return want.to(pool.dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", STORES)
def test_bounds_of_every_store(gpu, store, D):
    print("bounds", store, D, flush=True)
    for page in (16, 64, 512):
        pool = Pool(gpu, store, [0, 1, 15, 16, 17, 100, 515, 1300], 3, D, page, seed=D + page)
        for tokens in (None, 0, 1, 2, 17, 300, 5000):
            assert torch.equal(bounds_of(pool, gpu, tokens=tokens), want_bounds(pool, tokens)), tokens


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
def test_bounds_of_page_sizes(gpu, page):
    for store in ("bf16", "u4_fp16"):
        pool = Pool(gpu, store, [page - 1, page, page + 1, 3 * page, 1], 1, 64, page, seed=page)
        for tokens in (None, 1, page):
            assert torch.equal(bounds_of(pool, gpu, tokens=tokens), want_bounds(pool, tokens))


def test_bounds_of_pages_that_are_not_there(gpu):
    """Entries outside the pool, lengths behind the table's last page, negative lengths."""
    pool = Pool(gpu, "bf16", [100, 64, 40], 2, 64, 16, seed=3, width=7)
    for b, i, bad in ((0, 2, -1), (0, 3, pool.num_pages), (1, 3, 2**31 - 1), (2, 0, -(2**31))):
        pool.table_gpu[b, i] = bad
    pool.lens_gpu[2] = -5
    pool.lens[2] = 0
    for tokens in (None, 1, 40):
        assert torch.equal(bounds_of(pool, gpu, tokens=tokens), want_bounds(pool, tokens))
    whole = Pool(gpu, "u8", [160], 2, 64, 16, seed=4)
    whole.table_gpu = whole.table_gpu[:, :10]
    whole.lens_gpu[0] = 2**31 - 1  # taken as the table's 160
    for tokens in (None, 1, 33):
        assert torch.equal(bounds_of(whole, gpu, tokens=tokens), want_bounds(whole, tokens))
    none = torch.full((pool.num_pages, 2, 2, 64), MARK, dtype=torch.bfloat16, device=gpu)
    paged_bounds(pool.buffers.k, none, pool.table_gpu[:0], pool.lens_gpu[:0])
    assert (none == MARK).all()


@pytest.mark.parametrize("store", STORES)
def test_bounds_of_what_is_not_finite(gpu, store):
    """A NaN makes its value's bounds NaN; infinities are bounds like others; of codes, a row's scale is all of its values'."""
    pool = Pool(gpu, store, [100], 2, 128, 32, seed=8)
    p, q = int(pool.table[0, 1]), int(pool.table[0, 2])
    if pool.bits is None:
        pool.buffers.k[p, 1, 5, 9], pool.buffers.k[q, 0, 31, 2], pool.buffers.k[q, 0, 30, 3] = math.nan, math.inf, -math.inf
    else:
        pool.buffers.quant.k_scale[p, 1, 5] = math.nan
    got, want = bounds_of(pool, gpu), want_bounds(pool)
    if pool.bits is None:
        want[p, 1, :, 9], want[q, 0, 1, 2], want[q, 0, 0, 3] = math.nan, math.inf, -math.inf
    else:
        want[p, 1] = math.nan
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


def test_bounds_in_views(gpu):
    pool = Pool(gpu, "u8_fp16", [50, 333, 16], 2, 128, 32, seed=9)
    wide = torch.full((pool.num_pages, 2, 3, 3, 128), MARK, dtype=torch.float16, device=gpu)
    bounds = wide[:, :, :2, 1].transpose(1, 2)  # sides before heads
    paged_bounds(pool.buffers.k, bounds, pool.table_gpu, pool.lens_gpu, quant=tuple(pool.buffers.quant))
    assert torch.equal(bounds.cpu(), want_bounds(pool))
    assert (wide[:, :, 2] == MARK).all() and (wide[..., 0, :] == MARK).all() and (wide[..., 2, :] == MARK).all()


def test_shared_pages_have_the_bounds_of_whole_pages(gpu):
    """A common prompt's pages in two sequences."""
    pool = Pool(gpu, "bf16", [64, 100], 2, 64, 16, seed=10)
    pool.table_gpu[1, :3] = pool.table_gpu[0, :3]
    pool.rows[0][1][:, :48] = pool.rows[0][0][:, :48]
    assert torch.equal(bounds_of(pool, gpu), want_bounds(pool))


# ---- the choice -----------------------------------------------------------------------------------------------------


def want_chosen(q, bounds, table, lens, page, count, first, last):
    """(B, Hkv, count) by the definition in 64 bits, on the CPU."""
    q, bounds, num_pages = q.double().cpu(), bounds.double().cpu(), bounds.shape[0]
    table, lens = table.cpu(), lens.cpu().tolist()
    (B, Hq, D), Hkv = q.shape, bounds.shape[1]
    out = torch.full((B, Hkv, count), -1, dtype=torch.int32)
    for b in range(B):
        P = min(-(-max(lens[b], 0) // page), table.shape[1])
        at = table[b, :P].long()
        there = (at >= 0) & (at < num_pages)
        mine = bounds[at.where(there, torch.zeros_like(at))]  # (P, Hkv, 2, D)
        i = torch.arange(P)
        for h in range(Hkv):
            heads = q[b].view(Hkv, -1, 1, D)[h]
            products = torch.maximum(heads * mine[None, :, h, 0], heads * mine[None, :, h, 1])
            score = products.sum(-1).float()  # (group, P)
            odd = ~torch.isfinite(score) | ~torch.isfinite(mine[None, :, h]).all(-1).all(-1)
            score = torch.where(odd, math.inf, score).amax(0).double()
            rank = torch.where((i < first) | (i >= P - last), 1e300, torch.where(score == math.inf, 1e200, score))
            rank = torch.where(there, rank, -math.inf)
            best = rank.sort(dim=0, descending=True, stable=True).indices[:count]
            best = best[there[best]].sort().values
            out[b, h, : len(best)] = best.to(torch.int32)
    return out


def a_choice(gpu, lens, Hq, Hkv, D, page, dtype=torch.bfloat16, seed=0, width=None):
    gen = torch.Generator().manual_seed(seed)
    P = max([-(-max(n, 0) // page) for n in lens] + [1])
    width, used = width or P + 2, sum(-(-max(n, 0) // page) for n in lens)
    order, table = torch.randperm(used + 3, generator=gen).to(torch.int32), torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        m = -(-max(n, 0) // page)
        table[b, :m], order = order[:m], order[m:]
    middle, reach = torch.randn(used + 3, Hkv, D, generator=gen), torch.rand(used + 3, Hkv, D, generator=gen)
    bounds = torch.stack((middle - reach, middle + reach), 2).to(dtype)
    q = torch.randn(len(lens), Hq, D, generator=gen).to(dtype)
    return q.to(gpu), bounds.to(gpu), table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)


def choose_and_check(q, bounds, table, lens, page, count, first=1, last=1):
    got = ops.paged_select(q, bounds, table, lens, page, count, first, last)
    assert got.dtype == torch.int32 and got.is_contiguous()
    assert torch.equal(got.cpu(), want_chosen(q, bounds, table, lens, page, count, first, last))
    return got


CHOICES = [0, 1, 15, 16, 17, 100, 255, 256, 257, 1000, 4000, 16385]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_select(gpu, D, dtype):
    print("select", D, dtype, flush=True)
    args = a_choice(gpu, CHOICES, 8, 2, D, 16, dtype, seed=D)
    for count, first, last in ((1, 0, 0), (1, 1, 0), (2, 1, 1), (16, 1, 1), (16, 0, 1), (63, 3, 7), (64, 0, 0), (65, 30, 35), (1000, 1, 1), (1030, 1, 2), (5000, 0, 0)):
        choose_and_check(*args, 16, count, first, last)


@pytest.mark.parametrize("group", range(1, 17))
def test_select_of_head_layouts(gpu, group):
    for D, dtype, Hkv in ((64, torch.float16, 5), (128, torch.bfloat16, 1), (256, torch.bfloat16, 2)):
        choose_and_check(*a_choice(gpu, [700, 0, 3000, 40], Hkv * group, Hkv, D, 16, dtype, seed=group), 16, 20)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
def test_select_of_page_sizes(gpu, page):
    choose_and_check(*a_choice(gpu, [page - 1, page, page + 1, 40 * page + 5, 200 * page], 4, 2, 128, page, seed=page), page, 12, 1, 2)


@pytest.mark.parametrize("B,Hkv,low,high", [(70, 2, 1, 700), (300, 1, 0, 300), (130, 7, 0, 2000), (2, 1, 200000, 600001), (1, 8, 131072, 131072)])
def test_select_of_batches(gpu, B, Hkv, low, high):
    print("select", B, Hkv, flush=True)
    gen = torch.Generator().manual_seed(B)
    lens = [high] + torch.randint(low, high + 1, (B - 1,), generator=gen).tolist()
    args = a_choice(gpu, lens, 4 * Hkv, Hkv, 64, 16, seed=B)
    for count, first, last in ((24, 1, 2), (500, 1, 2), (24, 4, 20), (20, 20, 0), (3, 1, 1)):
        choose_and_check(*args, 16, count, first, last)


@pytest.mark.parametrize("width", [1, 2, 16, 17, 127, 128, 129, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769])
def test_select_of_table_widths(gpu, width):
    """Where one kernel's pages end and the next one's begin."""
    print("select", width, flush=True)
    for Hq, Hkv, D, dtype in ((8, 2, 128, torch.bfloat16), (5, 1, 64, torch.float16), (32, 2, 256, torch.bfloat16)):
        if D == 256 and width > 2049:
            continue
        args = a_choice(gpu, [16 * width, 0, 16 * width - 5, 8 * width + 3, 1], Hq, Hkv, D, 16, dtype, seed=width, width=width)
        for count, first, last in ((1, 0, 1), (min(40, width + 3), 1, 0), (max(2, width // 2), 1, 1), (width, 0, 0)):
            choose_and_check(*args, 16, count, first, last)


def test_select_of_very_long_sequences(gpu):
    """More pages than a workgroup holds: 70000 of 16 tokens."""
    args = a_choice(gpu, [1120000, 5, 530000], 2, 1, 64, 16, seed=2)
    for count in (64, 40000):
        choose_and_check(*args, 16, count)


@pytest.mark.parametrize("pages", [100, 128])
@pytest.mark.parametrize("group", [1, 5, 16])
def test_select_of_few_pages(gpu, group, pages):
    """Tables that one workgroup has whole: ties, what is not finite, pages that are not there."""
    q, bounds, table, lens = a_choice(gpu, [16 * pages, 500, 7, 1024], 2 * group, 2, 128, 16, seed=group, width=pages)
    choose_and_check(q, bounds, table, lens, 16, 20, 1, 2)
    bounds[int(table[0, 40]), 1, 0, 3] = math.nan
    bounds[int(table[0, 41]), :, 1, 3] = math.inf
    table[0, ::3], table[1, 5], table[3, :] = -1, bounds.shape[0], -7
    got = choose_and_check(q, bounds, table, lens, 16, 12, 2, 3)
    assert 40 in got[0, 1].tolist() and 41 in got[0, 0].tolist() and (got[3] == -1).all()
    q[1, 0, 0] = math.inf
    choose_and_check(q, bounds, table, lens, 16, 60, 0, 0)
    bounds[:] = bounds[3:4].clone()
    choose_and_check(q, bounds, table, lens, 16, 9, 0, 1)
    choose_and_check(torch.zeros_like(q), bounds, table, lens, 16, 50, 0, 0)


@pytest.mark.parametrize("group", [1, 4, 7, 16])
def test_select_of_equal_scores(gpu, group):
    """Ties go to the page in front: all pages alike, many alike, of two values."""
    q, bounds, table, lens = a_choice(gpu, [3000, 500, 16384], 2 * group, 2, 128, 16, seed=11)
    bounds[:] = bounds[:1]
    for count in (1, 10, 200, 1023, 1024, 1025):
        got = choose_and_check(q, bounds, table, lens, 16, count, 0, 0)
        assert got[2, 0].tolist() == [i if i < 1024 else -1 for i in range(count)]
    bounds[::3] += 1.0
    for count in (10, 200, 400):
        choose_and_check(q, bounds, table, lens, 16, count, 1, 3)


def test_select_of_zeros_and_signs(gpu):
    """Queries of zeros tie all pages (of either zero); scores below zero; denormal products."""
    q, bounds, table, lens = a_choice(gpu, [2000, 333], 4, 2, 64, 16, torch.float16, seed=12)
    q[0] = 0.0
    q[1] *= -0.0
    got = choose_and_check(q, bounds, table, lens, 16, 10, 0, 0)
    assert got[0, 0].tolist() == list(range(10))
    q, bounds, table, lens = a_choice(gpu, [2000, 333], 4, 2, 64, 16, torch.bfloat16, seed=13)
    bounds[:, :, 0], bounds[:, :, 1] = -3.0 - torch.rand(bounds.shape[0], 2, 64, device=gpu), -2.5
    q.abs_()
    choose_and_check(q, bounds, table, lens, 16, 10, 0, 0)
    choose_and_check(q * 2.0**-100, bounds, table, lens, 16, 10, 0, 0)
    choose_and_check(q * 2.0**-124, bounds * 2.0**-10, table, lens, 16, 10, 0, 0)  # scores among the denormal numbers
    choose_and_check(q * 2.0**110, bounds * 2.0**14, table, lens, 16, 10, 0, 0)    # and some that 32 bits do not hold


def test_select_of_what_is_not_finite(gpu):
    """Pages with bounds that are not finite come before others; a query that is not finite ties all pages."""
    q, bounds, table, lens = a_choice(gpu, [3000, 3000, 3000], 4, 2, 64, 16, seed=14)
    for b, i, value in ((0, 100, math.nan), (0, 7, math.inf), (1, 180, -math.inf), (1, 181, math.nan)):
        bounds[int(table[b, i]), :, i % 2, 5] = value
    q[2, 1, 3] = math.nan
    got = choose_and_check(q, bounds, table, lens, 16, 8, 1, 1)
    assert {7, 100} <= set(got[0, 1].tolist()) and {180, 181} <= set(got[1, 0].tolist())
    assert got[2, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 187]


def test_select_leaves_out_pages_that_are_not_there(gpu):
    q, bounds, table, lens = a_choice(gpu, [1000, 160, 48], 4, 2, 64, 16, seed=15)
    table[0, ::2] = -1
    table[0, 1], table[1, 9], table[2, :3] = bounds.shape[0], 2**31 - 1, -(2**31)
    for count in (4, 31, 40, 70):
        got = choose_and_check(q, bounds, table, lens, 16, count, 1, 1)
        assert (got[2] == -1).all()
    lens[1], lens[2] = 2**31 - 1, -3  # the table's last page is the last; none
    choose_and_check(q, bounds, table[:, :10], lens, 16, 9, 1, 1)
    assert ops.paged_select(q[:0], bounds, table[:0], lens[:0], 16, 5).shape == (0, 2, 5)


def test_select_of_views(gpu):
    q, bounds, table, lens = a_choice(gpu, [900, 40, 5000], 6, 2, 128, 32, seed=16)
    qkv = torch.randn(3, 10, 128, device=gpu).to(q.dtype)
    qkv[:, :6] = q
    wide = torch.zeros(bounds.shape[0], 2, 3, 2, 128, dtype=q.dtype, device=gpu)
    wide[:, :, 1] = bounds.transpose(1, 2)
    t = torch.full((3, table.shape[1] + 9), -5, dtype=torch.int32, device=gpu)[:, 4 : 4 + table.shape[1]]
    t.copy_(table)
    assert torch.equal(choose_and_check(qkv[:, :6], wide[:, :, 1].transpose(1, 2), t, lens, 32, 30), ops.paged_select(q, bounds, table, lens, 32, 30))


@pytest.mark.parametrize("store", STORES)
def test_scores_bound_what_is_attended_to(gpu, store):
    """With one page to choose, none of the other pages' keys has a larger product with a query than the bounds of the chosen one allow."""
    pool = Pool(gpu, store, [3000, 700], 2, 64, 16, seed=17)
    bounds = torch.zeros(pool.num_pages, 2, 2, 64, dtype=pool.dtype, device=gpu)
    paged_bounds(pool.buffers.k, bounds, pool.table_gpu, pool.lens_gpu, quant=pool.buffers.quant)
    q = torch.randn(2, 6, 64, generator=pool.gen).to(pool.dtype)
    got = choose_and_check(q.to(gpu), bounds, pool.table_gpu, pool.lens_gpu, 16, 1, 0, 0).cpu()
    for b in range(2):
        for h in range(2):
            heads, page = q[b].view(2, 3, 64)[h].double(), int(pool.table[b, got[b, h, 0]])
            most = torch.maximum(heads * bounds[page, h, 0].double().cpu(), heads * bounds[page, h, 1].double().cpu()).sum(-1).max()
            # rows of codes are bounded as rounded to 16 bits
            slack = 2.0**-7 * (heads.abs() @ pool.rows[0][b][h].abs().T).max() if pool.bits else 2.0**-22 * most.abs()
            assert (heads @ pool.rows[0][b][h].T).max() <= most + slack


def test_select_gives_the_same_every_time_and_on_two_streams(gpu):
    args = [a_choice(gpu, [40000, 9, 3000], 8, 2, 128, 16, seed=18 + i) for i in range(2)]
    want = [choose_and_check(*a, 16, 50) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                got.append(ops.paged_select(*a, 16, 50))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---- attention over chosen pages ------------------------------------------------------------------------------------


def some_pages(pool, count, seed=0, shuffled=False):
    """Lists of any pages, the last (which may not be full) among them; -1 behind."""
    gen = torch.Generator().manual_seed(seed)
    chosen = torch.full((len(pool.lens), pool.Hkv, count), -1, dtype=torch.int32)
    for b, n in enumerate(pool.lens):
        P = -(-n // pool.page)
        for h in range(pool.Hkv):
            some = torch.randperm(P, generator=gen)[:count]
            if P and P - 1 not in some.tolist():
                some[-1] = P - 1
            chosen[b, h, : len(some)] = (some if shuffled else some.sort().values).to(torch.int32)
    return chosen


def check_chosen(pool, out, lse, q, chosen, scale):
    """Against the rows that the lists name; entries behind the number of the sequence's pages do not count."""
    Hq, G = q.shape[1], q.shape[1] // pool.Hkv
    for b, n in enumerate(pool.lens):
        P = -(-n // pool.page)
        for h in range(pool.Hkv):
            at = [i * pool.page + t for i in chosen[b, h, :P].tolist() if 0 <= i < P for t in range(min(pool.page, n - i * pool.page))]
            at = [t for t in at if 0 <= int(pool.table_gpu[b, t // pool.page]) < pool.num_pages]
            mine = slice(h * G, h * G + G)
            r = [x[b][h : h + 1, at] for x in pool.rows]
            check_decode(out[b, mine].cpu(), lse[b, mine].cpu(), q[b, mine], *r, scale, pool.dtype, pool.spans[b][h : h + 1, at] if pool.bits else None)


def attend_and_check(pool, gpu, Hq, chosen, scale=None, q=None):
    scale = pool.D**-0.5 if scale is None else scale
    if q is None:
        q = torch.randn(len(pool.lens), Hq, pool.D, generator=pool.gen).to(pool.dtype)
    out, lse = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu, scale, return_lse=True, chosen=chosen.to(gpu))
    assert out.dtype == pool.dtype and lse.dtype == torch.float32 and lse.shape == q.shape[:2]
    check_chosen(pool, out, lse, q, chosen, scale)
    return q, out, lse


LENS = [0, 1, 15, 16, 17, 33, 129, 300, 515, 1000, 2600]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", STORES)
def test_chosen_of_every_store(gpu, store, D):
    print("chosen", store, D, flush=True)
    pool = Pool(gpu, store, LENS, 2, D, 16, seed=D)
    for count in (1, 7, 40, 200):
        attend_and_check(pool, gpu, 8, some_pages(pool, count, seed=count))


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 12, 16])
@pytest.mark.parametrize("store,D", [("bf16", 128), ("u8", 64), ("u4_fp16", 128), ("fp16", 256)])
def test_chosen_of_head_layouts(gpu, store, D, group):
    pool = Pool(gpu, store, [900, 0, 77], 5, D, 32, seed=group)
    attend_and_check(pool, gpu, 5 * group, some_pages(pool, 6, seed=group))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("store", ["bf16", "u8", "u4"])
def test_chosen_of_page_sizes(gpu, store, page):
    pool = Pool(gpu, store, [1, page - 1, page, page + 1, 5 * page + 17], 2, 128, page, seed=page)
    for count in (1, 3, 9):
        attend_and_check(pool, gpu, 4, some_pages(pool, count, seed=page))


@pytest.mark.parametrize("store", STORES)
def test_chosen_in_any_order_with_gaps_and_twice(gpu, store):
    """The last page, not full, in the middle of a list; entries that name nothing; pages named twice; entries behind the sequence's number of pages."""
    pool = Pool(gpu, store, [1003, 200, 33, 16, 700], 2, 64, 16, seed=21)
    chosen = some_pages(pool, 50, seed=3, shuffled=True)
    chosen[0, 0, 5], chosen[0, 0, 6], chosen[0, 1, 30], chosen[0, 1, 2] = -1, 63, 2**31 - 1, -(2**31)
    chosen[0, 1, 10:20] = chosen[0, 1, 9]
    chosen[1, 0, :13] = 12
    chosen[1, 1, 13:] = 0  # a sequence of 13 pages: not read
    chosen[2, 0, :3] = -1  # nothing is left
    chosen[3, 0, 0] = 1    # no such page
    chosen[4, 1, :] = torch.arange(49, -1, -1, dtype=torch.int32)
    _, out, lse = attend_and_check(pool, gpu, 6, chosen)
    assert (out[2, :3] == 0).all() and (lse[2, :3] == -math.inf).all() and (out[3, :3] == 0).all()


@pytest.mark.parametrize("store", STORES)
def test_chosen_leaves_out_pages_that_are_not_there(gpu, store):
    pool = Pool(gpu, store, [800, 100, 64], 2, 128, 16, seed=22)
    chosen = some_pages(pool, 30, seed=5)
    for b, i, bad in ((0, 49, -1), (0, 8, pool.num_pages), (1, 0, 2**31 - 1), (2, 3, -(2**31))):
        pool.table_gpu[b, i] = bad
    attend_and_check(pool, gpu, 4, chosen)
    whole = Pool(gpu, store, [160], 2, 128, 16, seed=6)
    whole.table_gpu = whole.table_gpu[:, :10]
    whole.lens_gpu[0] = 2**31 - 1  # taken as the table's 160
    attend_and_check(whole, gpu, 4, torch.tensor([[[9, 0, 4], [8, 10, 1]]], dtype=torch.int32))
    whole.lens_gpu[0] = -8
    out, lse = whole.buffers.decode(torch.randn(1, 4, 128).to(whole.dtype).to(gpu), whole.table_gpu, whole.lens_gpu, return_lse=True, chosen=torch.zeros(1, 2, 3, dtype=torch.int32, device=gpu))
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("store,B,Hq,Hkv,D,page,low,high,count", [
    ("bf16", 1, 8, 2, 128, 16, 20000, 20000, 1000),  # one long list over all workgroups
    ("u8", 3, 4, 1, 64, 64, 1, 30001, 300),
    ("u4", 2, 16, 1, 128, 32, 9000, 12345, 350),
    ("fp16", 2, 2, 1, 256, 128, 5000, 9999, 40),
    ("bf16", 70, 4, 2, 64, 16, 1, 1700, 40),          # more than 64 sequences
    ("u8_fp16", 300, 2, 1, 64, 16, 0, 900, 33),       # more than 256
    ("u4_fp16", 130, 7, 7, 64, 16, 0, 800, 36),       # more pairs than workgroups
    ("bf16", 1, 1, 1, 64, 16, 1, 1, 1),
])
def test_chosen_of_batches(gpu, store, B, Hq, Hkv, D, page, low, high, count):
    print("chosen", store, B, Hq, Hkv, D, flush=True)
    gen = torch.Generator().manual_seed(B)
    lens = [high] + torch.randint(low, high + 1, (B - 1,), generator=gen).tolist()
    pool = Pool(gpu, store, lens, Hkv, D, page, seed=B + 1, width=-(-high // page) + 20)
    attend_and_check(pool, gpu, Hq, some_pages(pool, count, seed=B))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("D,page,count", [(128, 16, 64), (64, 64, 9), (256, 128, 16)])
def test_chosen_of_many_lists(gpu, store, D, page, count):
    """Lists enough to keep all units busy, each a workgroup's; of 512 tokens more and to 2048, full and not."""
    gen = torch.Generator().manual_seed(D)
    lens = torch.randint(0, 70, (140,), generator=gen).tolist()
    lens[3], lens[5], lens[17], lens[70], lens[138], lens[139] = 0, count * page + 1, count * page, 1, count * page // 2 + 9, 2 * count * page
    pool = Pool(gpu, store, lens, 4, D, page, seed=count)
    attend_and_check(pool, gpu, 8, some_pages(pool, count, seed=count))


@pytest.mark.parametrize("store,D,page", [("bf16", 64, 16), ("u8_fp16", 128, 64), ("u4", 64, 32), ("u4_fp16", 256, 16)])
def test_chosen_of_shares_of_many_pages(gpu, store, D, page):
    """More than 4096 keys of a list a workgroup, over the ends of pairs; sequences of the same pages in orders of their own."""
    B, Hkv, n = 48, 2, 24576
    dtype, bits = STORES[store]
    gen = torch.Generator().manual_seed(D + page)
    one = Pool(gpu, store, [n], Hkv, D, page, seed=D)
    pages = n // page
    order = torch.stack([torch.randperm(pages, generator=gen) for _ in range(B)])
    lens = torch.randint(n - 4000, n + 1, (B,), generator=gen).tolist()
    lens[3], lens[40] = 0, 5
    count = pages - pages // 20
    chosen = torch.full((B, Hkv, count), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(Hkv):
            some = torch.randperm(-(-lens[b] // page), generator=gen)[:count]
            chosen[b, h, : len(some)] = some.to(torch.int32)
    q = torch.randn(B, 2 * Hkv, D, generator=gen).to(dtype)
    out, lse = one.buffers.decode(q.to(gpu), one.table[0, :pages][order].to(torch.int32).to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), return_lse=True, chosen=chosen.to(gpu))
    for b in (0, 3, 17, 40, 41, 47):
        for h in range(Hkv):
            at = (chosen[b, h].long()[:, None] * page + torch.arange(page)).flatten()
            at = at[(at >= 0) & (at < lens[b])]
            at = order[b][at // page] * page + at % page
            r = [x[0][h : h + 1, at] for x in one.rows]
            mine = slice(2 * h, 2 * h + 2)
            check_decode(out[b, mine].cpu(), lse[b, mine].cpu(), q[b, mine], *r, D**-0.5, dtype, one.spans[0][h : h + 1, at] if bits else None)


def test_lists_in_views(gpu):
    """One list for all heads or sequences, lists in rows of a wider tensor."""
    pool = Pool(gpu, "bf16", [300, 300, 300], 2, 64, 16, seed=23)
    q = torch.randn(3, 4, 64, generator=pool.gen).to(pool.dtype).to(gpu)
    one = torch.tensor([3, 18, 7], dtype=torch.int32, device=gpu)
    for chosen in (one.expand(3, 2, 3), torch.stack((one, one + 0))[None].expand(3, 2, 3), torch.nn.functional.pad(one.expand(3, 2, 3), (2, 4), value=1)[..., 2:5]):
        out, lse = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu, return_lse=True, chosen=chosen)
        check_chosen(pool, out, lse, q.cpu(), one.cpu().expand(3, 2, 3), 0.125)


@pytest.mark.parametrize("store", STORES)
def test_all_pages_chosen_is_attention_over_all(gpu, store):
    """Bit for bit, where the work is split alike: whole pages, as many entries as the table has."""
    pool = Pool(gpu, store, [1008, 0, 48, 2048], 2, 128, 16, seed=24, width=128)
    q = torch.randn(4, 8, 128, generator=pool.gen).to(pool.dtype).to(gpu)
    want = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu, return_lse=True)
    got = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu, return_lse=True, chosen=torch.arange(128, dtype=torch.int32, device=gpu).expand(4, 2, 128))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_chosen(pool, *got, q.cpu(), torch.arange(128, dtype=torch.int32).expand(4, 2, 128), 128**-0.5)


def test_chosen_gives_the_same_bits_and_runs_on_two_streams(gpu):
    pools = [Pool(gpu, s, [3000, 900, 41], 2, 128, 16, seed=25 + i) for i, s in enumerate(("bf16", "u8"))]
    lists = [some_pages(p, 60, seed=i) for i, p in enumerate(pools)]
    want = [attend_and_check(p, gpu, 8, c) for p, c in zip(pools, lists)]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for p, s, c, (q, _, _) in zip(pools, streams, lists, want):
            with torch.cuda.stream(s):
                got.append(p.buffers.decode(q.to(gpu), p.table_gpu, p.lens_gpu, return_lse=True, chosen=c.to(gpu)))
        torch.cuda.synchronize()
        for (out, lse), (_, o, x) in zip(got, want):
            assert torch.equal(out, o) and torch.equal(lse, x)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_chosen_hands_on_what_is_not_finite(gpu, value):
    """In a chosen page's row; not in pages that are not chosen, nor behind the last token."""
    pool = Pool(gpu, "bf16", [1000, 1000], 1, 64, 16, seed=27)
    chosen = torch.tensor([[[62, 3, 9]], [[62, 4, 9]]], dtype=torch.int32)
    q = torch.randn(2, 4, 64, generator=pool.gen).to(pool.dtype)
    pool.buffers.v[int(pool.table[0, 3]), 0, 2, 5] = value
    pool.buffers.v[int(pool.table[1, 3]), 0, 2, 5] = value
    out, lse = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu, return_lse=True, chosen=chosen.to(gpu))
    pool.rows[1][0][0, 3 * 16 + 2, 5] = 0.0
    other = [d for d in range(64) if d != 5]
    if math.isnan(value):
        assert torch.isnan(out[0, :, 5]).all()
    else:
        assert (out[0, :, 5] == value).all()
    assert torch.isfinite(out[0, :, other]).all() and torch.isfinite(out[1]).all() and torch.isfinite(lse).all()
    at = [62 * 16 + t for t in range(8)] + list(range(64, 80)) + list(range(144, 160))
    check_decode(out[1].cpu(), lse[1].cpu(), q[1], *(x[1][:, at] for x in pool.rows), 0.125, pool.dtype)


def test_pages_beyond_32_bits(gpu):
    """A pool of more than 4 GiB a tensor: rows appended at both ends, their bounds, attention over them."""
    page, Hq, Hkv, D, pages = 256, 16, 8, 128, 9000
    k, v = (torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    bounds = torch.zeros(pages, Hkv, 2, D, dtype=torch.bfloat16, device=gpu)
    gen = torch.Generator().manual_seed(2)
    n = 1000
    table = torch.tensor([[pages - 1, 0, 8500, pages - 2]], dtype=torch.int32)
    at = torch.arange(n)
    qkv = torch.randn(n, (Hq + 2 * Hkv) * D, generator=gen).to(torch.bfloat16).to(gpu)
    cos, sin = rows.rope_tables(n, D, 1e6, gpu)
    rotated = rows.rotary_(qkv.clone(), Hq, Hkv, D, None, None, 0.0, cos, sin, at.to(torch.int32).to(gpu)).view(n, -1, D)
    paged_append(qkv, Hq, Hkv, D, None, None, 0.0, cos, sin, at.to(torch.int32).to(gpu), k, v, (table[0].long()[at // page] * page + at % page).to(gpu))
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    paged_bounds(k, bounds, table.to(gpu), lens)
    key, value = rotated[:, Hq:-Hkv].transpose(0, 1), rotated[:, -Hkv:].transpose(0, 1)
    for i, p in enumerate(table[0].tolist()):
        mine = key[:, i * page : min(n, (i + 1) * page)]
        assert torch.equal(k[p, :, : mine.shape[1]], mine)
        assert torch.equal(bounds[p, :, 0], mine.amin(1)) and torch.equal(bounds[p, :, 1], mine.amax(1))
    q = rotated[-1:, :Hq].contiguous()
    chosen = ops.paged_select(q, bounds, table.to(gpu), lens, page, 3)
    assert torch.equal(chosen.cpu(), want_chosen(q, bounds, table, lens, page, 3, 1, 1))
    out, lse = ops.paged_decode_chosen(q, k, v, table.to(gpu), lens, chosen, D**-0.5, True)
    for h in range(Hkv):
        at = torch.cat([torch.arange(i * page, min(n, (i + 1) * page)) for i in chosen[0, h].tolist()])
        check_decode(out[0, 2 * h : 2 * h + 2].cpu(), lse[0, 2 * h : 2 * h + 2].cpu(), q[0, 2 * h : 2 * h + 2].cpu(), key[h : h + 1, at].double().cpu(), value[h : h + 1, at].double().cpu(),
                     D**-0.5, torch.bfloat16)


# ---- refusals -------------------------------------------------------------------------------------------------------


def test_what_is_refused(gpu):
    pool = Pool(gpu, "bf16", [100, 40], 2, 64, 16, seed=30)
    b, table, lens = pool.buffers, pool.table_gpu, pool.lens_gpu
    bounds = torch.zeros(pool.num_pages, 2, 2, 64, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=gpu)
    chosen = torch.zeros(2, 2, 3, dtype=torch.int32, device=gpu)
    select = lambda **k: ops.paged_select(**{**dict(query=q, bounds=bounds, block_table=table, lens=lens, page_size=16, count=4), **k})  # noqa: E731
    attend = lambda **k: ops.paged_decode_chosen(**{**dict(query=q, key_pages=b.k, value_pages=b.v, block_table=table, lens=lens, chosen=chosen, scale=0.1), **k})  # noqa: E731
    bound = lambda **k: paged_bounds(**{**dict(key_pages=b.k, bounds=bounds, block_table=table, lens=lens), **k})  # noqa: E731
    cos, sin = rows.rope_tables(200, 64, 1e4, gpu)
    qkv, pos, slots = torch.zeros(5, 8 * 64, dtype=torch.bfloat16, device=gpu), torch.zeros(5, dtype=torch.int32, device=gpu), torch.arange(5, device=gpu)
    append = lambda **k: paged_append(**{**dict(qkv=qkv, n_head=4, n_query_groups=2, head_size=64, q_weight=None, k_weight=None, eps=0.0, cos=cos, sin=sin, positions=pos,  # noqa: E731
                                                key_pages=b.k, value_pages=b.v, slots=slots), **k})
    select(), attend(), bound(), append()
    for call, kwargs in (
        (select, dict(count=0)), (select, dict(first=3, last=2)), (select, dict(count=-1)), (select, dict(first=-1)), (select, dict(count=2**40)), (select, dict(query=q[:1])),
        (select, dict(query=q[:, :3])), (select, dict(query=q[..., :32])), (select, dict(bounds=bounds[:, :, :1])), (select, dict(bounds=bounds[0])), (select, dict(lens=lens.long())),
        (select, dict(block_table=table.long())), (attend, dict(chosen=chosen.long())), (attend, dict(chosen=chosen[:, :1])), (attend, dict(chosen=chosen[:1])),
        (attend, dict(chosen=chosen[..., :0])), (attend, dict(chosen=chosen[0])), (attend, dict(chosen=torch.zeros(2, 2, 6, dtype=torch.int32, device=gpu)[..., ::2])),
        (attend, dict(scale=0.0)), (bound, dict(tokens=-1)), (bound, dict(bounds=bounds[:-1])), (bound, dict(bounds=bounds[:, :1])), (bound, dict(lens=lens[:1])),
        (append, dict(slots=slots[:4])), (append, dict(slots=slots.int())), (append, dict(positions=pos.long())), (append, dict(n_head=6, n_query_groups=1)), (append, dict(qkv=qkv[:, :-64])),
        (append, dict(k_weight=torch.ones(64, device=gpu))), (append, dict(key_pages=b.k[:, :1], value_pages=b.v[:, :1])),
    ):
        with pytest.raises(ValueError):
            call(**kwargs)
    for call, kwargs in (
        (select, dict(page_size=24)), (select, dict(query=q.half())), (select, dict(query=q.float())), (select, dict(bounds=bounds.float())),
        (select, dict(query=torch.zeros(2, 34, 64, dtype=torch.bfloat16, device=gpu))), (attend, dict(query=torch.zeros(2, 34, 64, dtype=torch.bfloat16, device=gpu))),
        (bound, dict(bounds=bounds.half())), (append, dict(qkv=qkv.half())), (append, dict(qkv=qkv.float())),
    ):
        with pytest.raises(NotImplementedError):
            call(**kwargs)
    with pytest.raises(RuntimeError):
        attend(chosen=chosen.cpu())
    for call in (select, attend, bound):
        with pytest.raises(TypeError):
            call(lens=None)


# ---- together -------------------------------------------------------------------------------------------------------


class SparseLayer(Layer):
    """A layer's step of generation with a choice of pages: append, bounds, select, attention, on buffers that stay in place."""

    def __init__(self, gpu, store, lens, Hq, Hkv, D, page, seed, count, first=1, last=1):
        super().__init__(gpu, store, lens, Hq, Hkv, D, page, seed)
        self.buffers.bounds = torch.zeros(self.buffers.num_pages, Hkv, 2, D, dtype=self.buffers.dtype, device=gpu)
        self.count, self.first, self.last = count, first, last
        self.buffers.update_bounds(self.table, self.lens)

    def step(self):
        self.buffers.append(self.qkv, self.Hq, self.qw, self.kw, 1e-6, self.cos, self.sin, self.positions, self.slots)
        self.buffers.update_bounds(self.table, self.lens, tokens=1)
        q = self.qkv.view(self.B, -1, self.D)[:, : self.Hq]
        chosen = self.buffers.select(q, self.table, self.lens, self.count, self.first, self.last)
        return (chosen, *self.buffers.decode(q, self.table, self.lens, return_lse=True, chosen=chosen))

    def check(self, chosen, out, lse):
        heads, D, G = self.before.view(self.B, -1, self.D), self.D, self.Hq // self.Hkv
        want = rows.rotary_(self.before.clone(), self.Hq, self.Hkv, D, self.qw, self.kw, 1e-6, self.cos, self.sin, self.positions).view(self.B, -1, D)
        now = self.qkv.view(self.B, -1, D)
        assert torch.equal(now[:, : self.Hq], want[:, : self.Hq]) and torch.equal(now[:, self.Hq :], heads[:, self.Hq :])
        table, q = self.table.cpu(), now[:, : self.Hq].cpu()
        for b, n in enumerate(self.lens.tolist()):
            if n == 0:
                assert (chosen[b] == -1).all() and (out[b] == 0).all() and (lse[b] == -math.inf).all()
                continue
            k, v = (stored_rows(self.buffers, i, table[b], n) for i in (0, 1))
            spans = stored_spans(self.buffers, table[b], n)
            if self.buffers.num_bits is None:
                assert torch.equal(k[:, -1], want[b, self.Hq : -self.Hkv].double().cpu()) and torch.equal(v[:, -1], heads[b, -self.Hkv :].double().cpu())
            for i in range(-(-n // self.page)):  # bounds of earlier steps hold too
                mine = k[:, i * self.page : (i + 1) * self.page]
                assert torch.equal(self.buffers.bounds[int(table[b, i])].cpu(), torch.stack((mine.amin(1), mine.amax(1)), 1).to(q.dtype))
            for h in range(self.Hkv):
                at = torch.cat([torch.arange(i * self.page, min(n, (i + 1) * self.page)) for i in chosen[b, h].tolist() if i >= 0])
                mine = slice(h * G, h * G + G)
                check_decode(out[b, mine].cpu(), lse[b, mine].cpu(), q[b, mine], k[h : h + 1, at], v[h : h + 1, at], D**-0.5, q.dtype, None if spans is None else spans[h : h + 1, at])
        assert torch.equal(chosen.cpu(), want_chosen(q, self.buffers.bounds, table, self.lens, self.page, self.count, self.first, self.last))


@pytest.mark.parametrize("store", STORES)
def test_steps_of_generation(gpu, store):
    layer = SparseLayer(gpu, store, [15, 0, 900, 31], 8, 2, 128, 16, 31, count=12, last=2)
    for _ in range(3):
        layer.next()
        layer.check(*layer.step())


@pytest.mark.parametrize("store", ["bf16", "u8", "u4_fp16"])
def test_captured_steps(gpu, store):
    """A captured step, replayed over growing lengths, with eager steps of another layer between the replays."""
    layer = SparseLayer(gpu, store, [130, 0, 2000, 1], 8, 2, 128, 16, 32, count=40)
    other = SparseLayer(gpu, store, [40, 300], 8, 2, 128, 16, 33, count=4)
    layer.next()
    layer.step()  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    layer.next()
    with torch.cuda.graph(graph):
        chosen, out, lse = layer.step()
    for _ in range(4):
        layer.next()
        graph.replay()
        other.next()
        got = other.step()
        torch.cuda.synchronize()
        other.check(*got)
        layer.check(chosen, out, lse)
        q = layer.qkv.view(layer.B, -1, 128)[:, :8]
        again = layer.buffers.decode(q, layer.table, layer.lens, return_lse=True, chosen=layer.buffers.select(q, layer.table, layer.lens, 40))
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)  # the eager result


@pytest.mark.parametrize("shared", [False, True])
def test_two_captured_steps_in_turn(gpu, shared):
    """Two graphs, each replayed before the other's results are looked at; of one memory pool in the order of their capture only, as torch asks for."""
    layers = [SparseLayer(gpu, store, lens, 6, 2, 64, 32, 34 + i, count=10) for i, (store, lens) in enumerate((("fp16", [900, 33, 0]), ("u4", [5, 1500])))]
    graphs, results, pool = [], [], None
    for layer in layers:
        layer.next()
        layer.step()
        torch.cuda.synchronize()
        layer.next()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            results.append(layer.step())
        pool = graphs[0].pool() if shared else None
    stream = torch.cuda.Stream()
    for order in ((0, 1),) * 4 if shared else ((0, 1), (1, 0), (0, 1), (1, 0)):
        for i in order:
            layers[i].next()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i in order:
                graphs[i].replay()
        torch.cuda.synchronize()
        for layer, got in zip(layers, results):
            if not shared or layer is layers[-1]:
                layer.check(*got)


def test_all_pages_chosen_step_is_a_dense_step(gpu):
    """With room for all pages, a step gives what rotary, write and attention over the whole sequences give, to the roundings of either."""
    layer = SparseLayer(gpu, "bf16", [200, 17], 4, 2, 64, 16, 36, count=64)
    layer.next()
    chosen, out, lse = layer.step()
    layer.check(chosen, out, lse)
    dense, dense_lse = layer.buffers.decode(layer.qkv.view(2, -1, 64)[:, :4], layer.table, layer.lens, return_lse=True)
    for b, n in enumerate(layer.lens.tolist()):
        k, v = (stored_rows(layer.buffers, i, layer.table[b].cpu(), n) for i in (0, 1))
        for got in ((out, lse), (dense, dense_lse)):
            check_decode(got[0][b].cpu(), got[1][b].cpu(), layer.qkv.view(2, -1, 64)[b, :4].cpu(), k, v, 0.125, torch.bfloat16)
