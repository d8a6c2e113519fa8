"""Operators of a paged cache on the device: page write and read-back, attention of one token over pages, rotary positions of ragged batches, and a
layer's step of the three, each against the same mathematics in 64 bits.

Tolerances: u is half a step of the outputs' type (relative to the value: bf16 2^-8, fp16 2^-11). An attention output is rounded once
(u |o|); a weight is rounded to the operands' 16-bit type before it meets V, at most w_u = 2^-8 for bf16 rows, 2^-11 for fp16 rows and for codes, which
moves the output by w_u (sum p |v|) at most. A row of codes is met from its middle code: half its span (scale times number of codes) stands for |v|. A
logit, D products added in fp32, is off by at most (D + 8) 2^-24 sum |q k|, which moves weights by that, relatively, above and below the
fraction. fp32 sums and exponentials behind it are allowed 2^-16 (sum p |v|). Weights underflow: exp2 gives 0 for what is below 2^-126 of the
largest, and a weight that is held in fp16, in units in which the largest is 2^7 at least, is rounded by 2^-25 at most where it is not a normal
number, 2^-32 of the largest. Over n rows of bf16 that is at most 2^-126 n max |v|, of fp16 2^-32 n max |v|, and of codes, whose scale is part
of the weight (in units of a power of two, at most twice the largest), 2^-32 n times the largest span."""
import math

import pytest
import torch

from keys_values_amd.attention import ops
from keys_values_amd.kvcache.paged import PagedKVCacheBuffers, paged_read, paged_write
from keys_values_amd.kvcache.quantize import RowQuantizer
from keys_values_amd.longctx import ops as rows

pytestmark = pytest.mark.gpu

STORES = {"bf16": (torch.bfloat16, None), "fp16": (torch.float16, None), "u8": (torch.bfloat16, 8), "u8_fp16": (torch.float16, 8), "u4": (torch.bfloat16, 4),
          "u4_fp16": (torch.float16, 4)}
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 300, 515, 1000]


class Pool:
    """A pool filled by hand: every row NaN (plain) or of NaN scale (codes) unless a sequence has it."""

    def __init__(self, gpu, store, lens, Hkv, D, page, seed=0, width=None, num_pages=None):
        dtype, bits = STORES[store]
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.D, self.Hkv, self.page, self.dtype, self.bits, self.gen = lens, D, Hkv, page, dtype, bits, gen
        used = [-(-n // page) for n in lens]
        self.num_pages = num_pages or sum(used) + 3
        self.width = width or max(max(used), 1) + 1
        self.buffers = PagedKVCacheBuffers(self.num_pages, page, Hkv, D, dtype, bits, gpu)
        order = torch.randperm(self.num_pages, generator=gen).tolist()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        for b, n in enumerate(used):
            for i in range(n):
                self.table[b, i] = order.pop()
        # rows as the 64-bit reference takes them, (B, Hkv, T, D) each
        self.rows, self.spans = [[], []], []
        for i, pages in enumerate((self.buffers.k, self.buffers.v)):
            shape = (self.num_pages, Hkv, page)
            if bits is None:
                host = torch.full((*shape, D), math.nan, dtype=dtype)
                values = torch.randn(*shape, D, generator=gen).to(dtype)
            else:
                host = torch.randint(0, 256, (*shape, D // 2 if bits == 4 else D), generator=gen, dtype=torch.int32).to(torch.uint8)
                scale, zp = torch.full(shape, math.nan), torch.full(shape, 2**30, dtype=torch.int32)
                scales = (4.0 + 4.0 * torch.rand(shape, generator=gen)) / (1 << bits)
                zps = torch.randint(0, 1 << bits, shape, generator=gen, dtype=torch.int32)
            for b, n in enumerate(lens):
                got, spans = torch.zeros(Hkv, n, D, dtype=torch.float64), torch.zeros(Hkv, n)
                for t in range(0, n, page):
                    p, m = int(self.table[b, t // page]), min(page, n - t)
                    if bits is None:
                        host[p, :, :m] = values[p, :, :m]
                        got[:, t : t + m] = values[p, :, :m].double()
                    else:
                        scale[p, :, :m], zp[p, :, :m] = scales[p, :, :m], zps[p, :, :m]
                        spans[:, t : t + m] = scales[p, :, :m] * (1 << bits)
                        c = host[p, :, :m].long()
                        c = torch.cat((c >> 4, c & 15), -1) if bits == 4 else c
                        got[:, t : t + m] = (c - zp[p, :, :m, None]).double() * scale[p, :, :m, None].double()
                self.rows[i].append(got)
                if i == 1:
                    self.spans.append(spans if bits else None)
            pages.copy_(host)
            if bits is not None:
                self.buffers.quant[2 * i].copy_(scale)
                self.buffers.quant[2 * i + 1].copy_(zp)
        self.table_gpu = self.table.to(gpu)
        self.lens_gpu = torch.tensor(lens, dtype=torch.int32, device=gpu)


def check_decode(out, lse, q, keys, values, scale, dtype, spans=None):
    """out (Hq, D), lse (Hq) of one sequence against q (Hq, D) and rows (Hkv, n, D) in 64 bits; spans (Hkv, n): of V rows of codes."""
    Hq, D = q.shape
    Hkv, n, _ = keys.shape
    assert out.dtype == dtype and out.shape == q.shape
    if n == 0:
        assert (out == 0).all() and (lse == -math.inf).all()
        return
    q64 = q.double().view(Hkv, Hq // Hkv, D)
    logits = q64 @ keys.transpose(1, 2) * scale
    p = torch.softmax(logits, -1)
    ref, ref_lse = p @ values, torch.logsumexp(logits, -1)
    size = p @ values.abs()
    moved = 2 * (D + 8) * 2.0**-24 * (q64.abs() @ keys.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale  # of a weight, relatively
    u = HALF_STEP[dtype]
    w_u = 2.0**-11 if spans is not None or dtype == torch.float16 else 2.0**-8
    if spans is not None:
        met, lost = p @ (spans.double()[..., None] / 2), 2.0**-32 * spans.max().item()
    else:
        met, lost = size, (2.0**-32 if dtype == torch.float16 else 2.0**-126) * values.abs().max().item()
    tol = u * ref.abs() + (w_u * met + (moved + 2.0**-16) * size) * (1 + u) + n * lost + (2.0**-24 if dtype == torch.float16 else 0.0)
    err = (out.double().cpu().view(ref.shape) - ref).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} tolerances"
    tol_lse = (moved[..., 0] + (n / 16 + 64) * 2.0**-24) / math.log(2) + ref_lse.abs() / math.log(2) * 2.0**-22
    err = (lse.double().cpu().view(ref_lse.shape) - ref_lse / math.log(2)).abs()
    assert (err <= tol_lse).all(), f"lse off by {(err / tol_lse).max().item():.2f} tolerances"


def decode_and_check(pool, gpu, Hq, scale=None, q=None):
    D = pool.D
    scale = D**-0.5 if scale is None else scale
    if q is None:
        q = torch.randn(len(pool.lens), Hq, D, generator=pool.gen).to(pool.dtype)
    out, lse = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu, scale, return_lse=True)
    assert lse.dtype == torch.float32 and lse.shape == q.shape[:2]
    for b in range(len(pool.lens)):
        check_decode(out[b].cpu(), lse[b].cpu(), q[b], pool.rows[0][b], pool.rows[1][b], scale, pool.dtype, pool.spans[b])
    return q, out, lse


# ---- decode ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", STORES)
def test_decode_of_every_store(gpu, store, D):
    print("decode", store, D, flush=True)
    pool = Pool(gpu, store, LENS, 2, D, 16, seed=D)
    decode_and_check(pool, gpu, 8)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 12, 16])
@pytest.mark.parametrize("store,D", [("bf16", 128), ("u8", 64), ("u4_fp16", 128), ("fp16", 256)])
def test_decode_of_head_layouts(gpu, store, D, group):
    print("decode heads", store, D, group, flush=True)
    pool = Pool(gpu, store, [200, 0, 77], 3, D, 32, seed=group)
    decode_and_check(pool, gpu, 3 * group)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("store", ["bf16", "u8", "u4"])
def test_decode_of_page_sizes(gpu, store, page):
    print("decode pages", store, page, flush=True)
    pool = Pool(gpu, store, [1, page - 1, page, page + 1, 2 * page + 17], 2, 128, page, seed=page)
    decode_and_check(pool, gpu, 4)


@pytest.mark.parametrize("store,B,Hq,Hkv,D,page,low,high", [
    ("bf16", 1, 8, 2, 128, 16, 20000, 20000),   # one long sequence over all workgroups
    ("u8", 3, 4, 1, 64, 64, 1, 30001),
    ("u4", 2, 16, 1, 128, 32, 9000, 12345),
    ("fp16", 2, 2, 1, 256, 128, 5000, 9999),
    ("bf16", 70, 4, 2, 64, 16, 1, 700),         # more than 64 sequences
    ("u8_fp16", 300, 2, 1, 64, 16, 0, 90),      # more than 256
    ("bf16", 1, 1, 1, 64, 16, 1, 1),
])
def test_decode_of_batches(gpu, store, B, Hq, Hkv, D, page, low, high):
    print("decode batch", store, B, Hq, Hkv, D, flush=True)
    gen = torch.Generator().manual_seed(B)
    lens = [high] + torch.randint(low, high + 1, (B - 1,), generator=gen).tolist()
    pool = Pool(gpu, store, lens, Hkv, D, page, seed=B + 1, width=-(-high // page) + 200)
    decode_and_check(pool, gpu, Hq)


@pytest.mark.parametrize("store,B,Hq,Hkv,D,low,high", [
    ("bf16", 500, 2, 2, 64, 0, 150),    # more pairs than workgroups
    ("u4", 260, 8, 4, 64, 1, 100),
    ("fp16", 130, 7, 7, 128, 1, 9),
    ("u8", 300, 3, 3, 256, 0, 60),
])
def test_decode_of_more_pairs_than_workgroups(gpu, store, B, Hq, Hkv, D, low, high):
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(low, high + 1, (B,), generator=gen).tolist()
    lens[B // 2], lens[-1] = 3000, 700
    pool = Pool(gpu, store, lens, Hkv, D, 32, seed=B)
    decode_and_check(pool, gpu, Hq)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("page,width", [(16, 32), (512, 1), (16, 33), (128, 4), (1024, 1)])
def test_decode_of_tables_around_512_tokens(gpu, store, page, width):
    """Up to 512 tokens, nothing is joined."""
    lens = [512, 511, 1, 0, 385, 129]
    pool = Pool(gpu, store, lens, 2, 64, page, seed=page + width, width=width)
    decode_and_check(pool, gpu, 6)


@pytest.mark.parametrize("store,D,page", [("bf16", 64, 16), ("u8_fp16", 128, 64), ("u4", 64, 32), ("fp16", 128, 1024), ("u4_fp16", 256, 16)])
def test_decode_of_shares_of_many_pages(gpu, store, D, page):
    """Sequences of the same pages in orders of their own: more than 4096 keys a workgroup, over the ends of pairs."""
    B, Hkv, n = 48, 2, 24576
    dtype, bits = STORES[store]
    gen = torch.Generator().manual_seed(D + page)
    one = Pool(gpu, store, [n], Hkv, D, page, seed=D)
    pages = n // page
    assert n % page == 0
    order = torch.stack([torch.randperm(pages, generator=gen) for _ in range(B)])
    lens = torch.randint(n - 4000, n + 1, (B,), generator=gen).tolist()
    lens[3], lens[40] = 0, 5
    table = one.table[0, :pages][order].to(torch.int32).to(gpu)
    q = torch.randn(B, 2 * Hkv, D, generator=gen).to(dtype)
    out, lse = one.buffers.decode(q.to(gpu), table, torch.tensor(lens, dtype=torch.int32, device=gpu), return_lse=True)
    for b in (0, 3, 17, 40, 41, 47):
        at = (order[b][:, None] * page + torch.arange(page)).flatten()[: lens[b]]
        check_decode(out[b].cpu(), lse[b].cpu(), q[b], one.rows[0][0][:, at], one.rows[1][0][:, at], D**-0.5, dtype, one.spans[0][:, at] if bits else None)


@pytest.mark.parametrize("store", ["u8", "u8_fp16", "u4", "u4_fp16"])
def test_decode_of_scales_of_either_sign(gpu, store):
    """(code - zero point) * scale holds for negative scales too."""
    pool = Pool(gpu, store, [300, 70, 1], 2, 128, 16, seed=51)
    for i in (0, 2):
        sign = torch.randint(0, 2, pool.buffers.quant[i].shape, generator=pool.gen) * 2.0 - 1.0
        if i == 2:
            sign[int(pool.table[1, 0])] = -1.0  # a sequence begins with them
            sign[int(pool.table[2, 0])] = -1.0
        pool.buffers.quant[i].mul_(sign.to(gpu))
        for b, n in enumerate(pool.lens):
            for t in range(0, n, 16):
                pool.rows[i // 2][b][:, t : t + 16] *= sign[int(pool.table[b, t // 16])][:, : min(16, n - t), None].double()
    decode_and_check(pool, gpu, 8)


def test_decode_without_tokens(gpu):
    pool = Pool(gpu, "bf16", [0, 0, 0], 2, 64, 16)
    pool.lens_gpu[1] = -7  # no length
    q = torch.randn(3, 4, 64, generator=pool.gen).to(torch.bfloat16).to(gpu)
    out, lse = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = pool.buffers.decode(q[:0], pool.table_gpu[:0], pool.lens_gpu[:0], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.parametrize("store", STORES)
def test_decode_leaves_out_pages_that_are_not_there(gpu, store):
    """Table entries outside the pool: their tokens are left out; lengths end at the table's last page."""
    lens, page = [100, 64, 40, 3000], 16
    pool = Pool(gpu, store, lens, 2, 128, page, seed=5)
    gone = {0: [2, 6], 1: [0, 1, 2, 3], 2: [1], 3: list(range(8, 20))}
    for b, pages in gone.items():
        for i, at in enumerate(pages):
            pool.table_gpu[b, at] = (-1, pool.num_pages, -(2**31), 2**31 - 1)[i % 4]
        keep = torch.tensor([t // page not in pages for t in range(lens[b])])
        for r in (*pool.rows, *([pool.spans] if pool.bits else [])):
            r[b] = r[b][:, keep]
    wide = -(-3000 // page)
    pool.table_gpu = pool.table_gpu[:, :wide]
    pool.lens_gpu[3] = 2**31 - 1
    last = pool.width * page  # rows of the last page behind 3000 are NaN: give the table's end whole pages
    assert last > 3000 and 3000 % page == 8
    pool.lens_gpu[3] = 3000
    decode_and_check(pool, gpu, 4)
    whole = Pool(gpu, store, [160], 2, 128, page, seed=6)
    whole.table_gpu = whole.table_gpu[:, :10]
    whole.lens_gpu[0] = 2**31 - 1  # taken as the table's 160
    decode_and_check(whole, gpu, 4)


@pytest.mark.parametrize("store", ["bf16", "u8"])
def test_decode_of_views(gpu, store):
    """K and V in one tensor, heads behind places, tables and queries that are parts of larger ones."""
    pool = Pool(gpu, store, [50, 333, 16], 2, 128, 32, seed=9)
    b = pool.buffers
    both = torch.empty(b.num_pages, 32, 2, 2, b.k.shape[-1], dtype=b.k.dtype, device=gpu)  # page, place, K or V, head, value
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    k.copy_(b.k)
    v.copy_(b.v)
    quant = None
    if b.quant is not None:
        state = torch.empty(b.num_pages, 3, 4, 32, dtype=torch.float32, device=gpu)  # four arrays that share strides, a head more than there are
        quant = []
        for i, t in enumerate(b.quant):
            part = state[:, :2, i] if t.dtype == torch.float32 else state.view(torch.int32)[:, :2, i]
            part.copy_(t)
            quant.append(part)
    table = torch.full((3, pool.width + 5), -3, dtype=torch.int32, device=gpu)[:, 2 : 2 + pool.width]
    table.copy_(pool.table_gpu)
    qkv = torch.randn(3, 8 + 4, 128, generator=pool.gen).to(pool.dtype).to(gpu)
    q = qkv[:, :8]
    out, lse = ops.paged_decode(q, k, v, table, pool.lens_gpu, 0.07, True, quant if quant is None else ops.QuantState(*quant))
    for i in range(3):
        check_decode(out[i].cpu(), lse[i].cpu(), q[i].cpu(), pool.rows[0][i], pool.rows[1][i], 0.07, pool.dtype, pool.spans[i])
    got = paged_read(k, v, table, pool.lens_gpu, 333, 128, pool.dtype, None if quant is None else tuple(quant))
    want = b.read(pool.table_gpu, pool.lens_gpu, 333)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("factor", [1.0e-3, 30.0])
def test_decode_of_flat_and_of_sharp_weights(gpu, store, factor):
    pool = Pool(gpu, store, [400, 3, 129], 2, 64, 16, seed=3)
    q = (factor * torch.randn(3, 8, 64, generator=pool.gen)).to(pool.dtype)
    decode_and_check(pool, gpu, 8, q=q)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("store", STORES)
def test_decode_of_logits_in_order(gpu, store, rising):
    """Keys along the query, so that the running maximum moves with every block, or never again; spans of 2^60 and more between the weights."""
    dtype, bits = STORES[store]
    n, D = 700, 64
    buffers = PagedKVCacheBuffers(50, 16, 1, D, dtype, bits, gpu)
    gen = torch.Generator().manual_seed(1)
    table = torch.randperm(50, generator=gen).to(torch.int32)[None, :44]
    direction = torch.sign(torch.randn(D, generator=gen))
    t = torch.linspace(-1, 1, n) * (1 if rising else -1)
    key = (t[:, None] * direction * 0.5).to(dtype)[:, None]
    value = torch.randn(n, 1, D, generator=gen).to(dtype)
    slots = buffers.slots(table.to(gpu), torch.arange(n, device=gpu)[None])
    buffers.write(key.to(gpu), value.to(gpu), slots)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    q = (torch.stack([direction * f for f in (0.5, 2.0, 6.0, -6.0)])[None]).to(dtype)
    out, lse = buffers.decode(q.to(gpu), table.to(gpu), lens, 1.0, True)
    rows64 = [stored_rows(buffers, i, table[0], n) for i in (0, 1)]
    check_decode(out[0].cpu(), lse[0].cpu(), q[0], *rows64, 1.0, dtype, stored_spans(buffers, table[0], n))


def stored_rows(buffers, i, pages, n):
    """K (0) or V (1) rows in 64 bits of a sequence, (Hkv, n, D), from what the pool holds."""
    x = (buffers.k, buffers.v)[i].cpu()[pages.long()]
    if buffers.num_bits == 4:
        x = torch.cat((x >> 4, x & 15), -1)
    if buffers.num_bits:
        x = (x.long() - buffers.quant[2 * i + 1].cpu()[pages.long()][..., None]).double() * buffers.quant[2 * i].cpu()[pages.long()].double()[..., None]
    return x.double().permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[-1])[:, :n]


def stored_spans(buffers, pages, n):
    if buffers.num_bits is None:
        return None
    return (buffers.quant.v_scale.cpu()[pages.long()] * (1 << buffers.num_bits)).transpose(0, 1).flatten(1)[:, :n]


@pytest.mark.parametrize("bits", [8, 4])
def test_decode_of_rows_whose_scales_differ(gpu, bits):
    """Scales from 2^-20 to 2^10 side by side, rows far from zero (zero points of thousands) and constant ones (scale 2^-23, zero points of millions)."""
    D, n = 128, 300
    buffers = PagedKVCacheBuffers(40, 16, 2, D, torch.bfloat16, bits, gpu)
    gen = torch.Generator().manual_seed(4)
    table = torch.randperm(40, generator=gen).to(torch.int32)[None, :19]
    key = torch.randn(n, 2, D, generator=gen)
    value = torch.randn(n, 2, D, generator=gen) * 2.0 ** torch.randint(-20, 11, (n, 2, 1), generator=gen)
    value[5::7] = 50.0 + 0.01 * value[5::7].clamp(-3, 3)
    value[3::11] = 0.75
    key[4::13] = 0.5
    key, value = key.to(torch.bfloat16), value.to(torch.bfloat16)
    buffers.write(key.to(gpu), value.to(gpu), buffers.slots(table.to(gpu), torch.arange(n, device=gpu)[None]))
    rows64 = [stored_rows(buffers, i, table[0], n) for i in (0, 1)]
    q = torch.randn(1, 8, D, generator=gen).to(torch.bfloat16)
    for m in (n, 4, 12):
        out, lse = buffers.decode(q.to(gpu), table.to(gpu), torch.tensor([m], dtype=torch.int32, device=gpu), return_lse=True)
        check_decode(out[0].cpu(), lse[0].cpu(), q[0], rows64[0][:, :m], rows64[1][:, :m], D**-0.5, torch.bfloat16, stored_spans(buffers, table[0], m))


@pytest.mark.parametrize("store", STORES)
def test_decode_hands_on_what_is_not_finite(gpu, store):
    """A NaN among a sequence's rows, or in its query, is the sequence's own."""
    pool = Pool(gpu, store, [100, 100, 60], 1, 64, 16, seed=8)
    q = torch.randn(3, 4, 64, generator=pool.gen).to(pool.dtype)
    p = int(pool.table[1, 3])
    if pool.bits is None:
        pool.buffers.v[p, 0, 2, 5] = math.nan
    else:
        pool.buffers.quant.v_scale[p, 0, 2] = math.nan
    q[2, 1] = math.nan
    out, lse = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu, return_lse=True)
    check_decode(out[0].cpu(), lse[0].cpu(), q[0], pool.rows[0][0], pool.rows[1][0], 0.125, pool.dtype, pool.spans[0])
    bad = torch.isnan(out[1].cpu())
    assert bad.all() if pool.bits else (bad[:, 5].all() and bad.sum() == 4)
    assert torch.isnan(out[2, 1].cpu()).all() and torch.isnan(lse[2, 1].cpu())
    for h in (0, 2, 3):
        assert torch.isfinite(out[2, h].cpu()).all()


def test_decode_of_pages_beyond_32_bits(gpu):
    """A pool of more than 4 GiB a tensor; the sequence's pages lie at both ends."""
    page, Hkv, D, n = 256, 8, 128, 1000
    pages = 9000  # 4.7 GB of K
    k, v = (torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    gen = torch.Generator().manual_seed(2)
    table = torch.tensor([[pages - 1, 0, 8500, pages - 2]], dtype=torch.int32)
    key, value = (torch.randn(n, Hkv, D, generator=gen).to(torch.bfloat16) for _ in range(2))
    at = torch.arange(n)
    slots = table[0].long()[at // page] * page + at % page
    paged_write(key.to(gpu), value.to(gpu), k, v, slots.to(gpu))
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    got = paged_read(k, v, table.to(gpu), lens, n)
    assert torch.equal(got[0][0].cpu(), key.transpose(0, 1)) and torch.equal(got[1][0].cpu(), value.transpose(0, 1))
    q = torch.randn(1, 16, D, generator=gen).to(torch.bfloat16)
    out, lse = ops.paged_decode(q.to(gpu), k, v, table.to(gpu), lens, D**-0.5, True)
    check_decode(out[0].cpu(), lse[0].cpu(), q[0], key.double().transpose(0, 1), value.double().transpose(0, 1), D**-0.5, torch.bfloat16)


def test_decode_gives_the_same_bits_every_time(gpu):
    pool = Pool(gpu, "bf16", [5000, 1, 700, 0, 2222], 2, 128, 16, seed=11)
    q, out, lse = decode_and_check(pool, gpu, 8)
    for _ in range(5):
        again = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu, 128**-0.5, True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_decode_on_two_streams(gpu):
    pools = [Pool(gpu, s, [3000, 900, 41], 2, 128, 16, seed=i) for i, s in enumerate(("bf16", "u8"))]
    want = [decode_and_check(p, gpu, 8) for p in pools]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for p, s, (q, _, _) in zip(pools, streams, want):
            with torch.cuda.stream(s):
                got.append(p.buffers.decode(q.to(gpu), p.table_gpu, p.lens_gpu, 128**-0.5, True))
        torch.cuda.synchronize()
        for (out, lse), (_, o, x) in zip(got, want):
            assert torch.equal(out, o) and torch.equal(lse, x)


# ---- write and read -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("tokens,Hkv,page", [(1, 1, 16), (37, 3, 16), (130, 2, 64)])
def test_write_of_rows(gpu, store, D, tokens, Hkv, page):
    """Rows where their slots say, the codes of the row quantiser, nothing else touched."""
    print("write", store, D, tokens, Hkv, page, flush=True)
    dtype, bits = STORES[store]
    pages = 2 * -(-tokens // page) + 1
    buffers = PagedKVCacheBuffers(pages, page, Hkv, D, dtype, bits, gpu)
    for t in (buffers.k, buffers.v):
        t.view(torch.uint8).fill_(0x5A)
    gen = torch.Generator().manual_seed(tokens + D)
    kv = torch.randn(tokens, 2 * Hkv, D, generator=gen) * 2.0 ** torch.randint(-12, 8, (tokens, 2 * Hkv, 1), generator=gen)
    kv[0, 0] = 0.25  # a constant row
    if tokens > 5:
        kv[3, 1, 7] = math.nan
        kv[4] = 0.0
    kv = kv.to(dtype).to(gpu)
    key, value = kv[:, :Hkv], kv[:, Hkv:]
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    dropped = torch.zeros(tokens, dtype=torch.bool)
    if tokens > 20:
        for i, s in ((2, -1), (9, pages * page), (10, -(2**62)), (11, 2**62), (tokens - 1, -1)):
            slots[i], dropped[i] = s, True
    before = [t.clone() for t in (buffers.k, buffers.v, *(buffers.quant or ()))]
    buffers.write(key, value, slots.to(gpu))
    want = [t.cpu() for t in before]
    keep = (~dropped).nonzero()[:, 0]
    at, place = slots[keep] // page, slots[keep] % page
    for i, x in enumerate((key, value)):
        if bits is None:
            want[i][at, :, place] = x.cpu()[keep]
            continue
        qz = RowQuantizer((1, Hkv, tokens, D), dtype, bits, allocate_buffers=True, device=gpu)
        qz.quantize(0, tokens, x.transpose(0, 1).contiguous()[None])
        for j, t in ((i, qz.quant_buffer), (2 + 2 * i, qz.quant_scales), (3 + 2 * i, qz.quant_zero_points)):
            t = t.cpu().view(Hkv, tokens, *t.shape[2:])
            want[j][at, :, place] = t[:, keep].transpose(0, 1)
    for got, w in zip((buffers.k, buffers.v, *(buffers.quant or ())), want):
        assert torch.equal(got.cpu().contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


def test_write_of_no_token(gpu):
    buffers = PagedKVCacheBuffers(2, 16, 2, 64, device=gpu)
    empty = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    buffers.write(empty, empty, torch.empty(0, dtype=torch.int64, device=gpu))
    assert (buffers.k == 0).all() and (buffers.v == 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", STORES)
def test_read_of_sequences(gpu, store, D):
    """The stored rows, rounded once; zeros behind the end and where the pool has no page."""
    print("read", store, D, flush=True)
    lens = [0, 1, 16, 47, 130]
    pool = Pool(gpu, store, lens, 3, D, 16, seed=D + 1)
    pool.table_gpu[3, 1], pool.table_gpu[4, 5] = pool.num_pages, -9
    for length in (1, 16, 100, 200):
        k, v = pool.buffers.read(pool.table_gpu, pool.lens_gpu, length)
        for i, got in enumerate((k, v)):
            assert got.shape == (5, 3, length, D) and got.dtype == pool.dtype
            for b, n in enumerate(lens):
                want = torch.zeros(3, length, D, dtype=torch.float64)
                m = min(n, length)
                want[:, :m] = pool.rows[i][b][:, :m]
                for at, bad in ((3, 1), (4, 5)):
                    if b == at:
                        want[:, 16 * bad : 16 * bad + 16] = 0
                # one product in fp32 (2^-24), one rounding to the type
                assert ((got[b].double().cpu() - want).abs() <= want.abs() * (HALF_STEP[pool.dtype] * (1 + 2.0**-10))).all()
                if pool.bits is None:
                    assert torch.equal(got[b].double().cpu(), want)
    k, v = pool.buffers.read(pool.table_gpu, pool.lens_gpu, 0)
    assert k.shape == v.shape == (5, 3, 0, D)


@pytest.mark.parametrize("store", ["u8", "u4_fp16"])
def test_read_gives_the_rows_of_the_quantiser(gpu, store):
    dtype, bits = STORES[store]
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(1, 2, 96, 128, generator=gen).to(dtype).to(gpu)
    buffers = PagedKVCacheBuffers(6, 16, 2, 128, dtype, bits, gpu)
    table = torch.tensor([[4, 1, 5, 0, 2, 3]], dtype=torch.int32, device=gpu)
    positions = torch.arange(96, device=gpu)[None]
    buffers.write(x[0].transpose(0, 1), x[0].transpose(0, 1), buffers.slots(table, positions))
    qz = RowQuantizer((1, 2, 96, 128), dtype, bits, allocate_buffers=True, device=gpu)
    qz.quantize(0, 96, x)
    want = qz.dequantize(0, 96).view(1, 2, 96, 128)
    for got in buffers.read(table, torch.tensor([96], dtype=torch.int32, device=gpu), 96):
        assert torch.equal(got, want)


def test_slots(gpu):
    buffers = PagedKVCacheBuffers(9, 32, 1, 64, device=gpu)
    table = torch.tensor([[5, 2, -1], [0, -1, -1]], dtype=torch.int32, device=gpu)
    positions = torch.tensor([[0, 33, 64, -1], [31, 32, 95, 96]], dtype=torch.int32, device=gpu)
    assert buffers.slots(table, positions).tolist() == [160, 65, -1, -1, 31, -1, -1, -1]


# ---- rotary ---------------------------------------------------------------------------------------------------------


def rotary64(x, weight, eps, cos, sin, interleaved):
    """x (tokens, heads, D) and its angles (tokens, n / 2) in 64 bits; also the sum of the magnitudes that a value is made of."""
    D, n = x.shape[-1], 2 * cos.shape[1]
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True).sqrt() / math.sqrt(D) + eps) * weight
    y, size = x.clone(), x.abs()
    cos, sin = cos[:, None], sin[:, None]
    a, b = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    size[..., a], size[..., b] = (x[..., a] * cos).abs() + (x[..., b] * sin).abs(), (x[..., b] * cos).abs() + (x[..., a] * sin).abs()
    return y, size


def check_rotary(before, after, Hq, Hkv, D, qw, kw, eps, cos, sin, positions, interleaved):
    before, after = before.cpu().view(-1, Hq + 2 * Hkv, D), after.cpu().view(-1, Hq + 2 * Hkv, D)
    pos = positions.cpu().flatten().long()
    there = (pos >= 0) & (pos < cos.shape[0])
    bits = torch.int16
    assert torch.equal(after[~there].contiguous().view(bits), before[~there].contiguous().view(bits))  # padding
    assert torch.equal(after[:, Hq + Hkv :].contiguous().view(bits), before[:, Hq + Hkv :].contiguous().view(bits))  # value heads
    x, angle = before[there, : Hq + Hkv].double(), pos[there]
    weight = None if qw is None else torch.cat((qw.cpu().double().expand(Hq, D), kw.cpu().double().expand(Hkv, D)))
    want, size = rotary64(x, weight, eps, cos.cpu().double()[angle], sin.cpu().double()[angle], interleaved)
    # the norm's sum of D squares and a few products in fp32, then one rounding
    u = HALF_STEP[before.dtype]
    tol = u * want.abs() + size * ((D + 16) * 2.0**-24) * (1 + u) + (2.0**-25 if before.dtype == torch.float16 else 0.0)
    err = (after[there, : Hq + Hkv].double() - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} tolerances"


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,part", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 48), (256, 256), (256, 32), (256, 240)])
def test_rotary(gpu, D, part, dtype, interleaved, norm):
    print("rotary", D, part, dtype, interleaved, norm, flush=True)
    gen = torch.Generator().manual_seed(D + part)
    for tokens, Hq, Hkv in ((1, 1, 1), (9, 7, 1), (70, 5, 2), (3, 64, 8)):
        qkv = torch.randn(tokens, (Hq + 2 * Hkv) * D, generator=gen).to(dtype).to(gpu)
        cos, sin = rows.rope_tables(3000, D, 1e4, gpu, rotary_dim=part)
        positions = torch.randint(0, 3000, (tokens,), generator=gen, dtype=torch.int32)
        if tokens > 8:
            positions[2], positions[3], positions[4], positions[-1] = -1, 3000, 2**31 - 1, -(2**31)
        qw, kw = ((1 + 0.3 * torch.randn(D, generator=gen)).to(gpu) for _ in range(2)) if norm else (None, None)
        before = qkv.clone()
        got = rows.rotary_(qkv, Hq, Hkv, D, qw, kw, 1e-5, cos, sin, positions.to(gpu), interleaved)
        assert got is qkv
        check_rotary(before, qkv, Hq, Hkv, D, qw, kw, 1e-5, cos, sin, positions, interleaved)


def test_rotary_of_batches_and_views(gpu):
    gen = torch.Generator().manual_seed(1)
    cos, sin = rows.rope_tables(500, 128, 1e6, gpu, scaling=rows.RopeScaling("yarn", 4.0, 256))
    wide = torch.randn(3, 5, 8 * 128 + 64, generator=gen).to(torch.bfloat16).to(gpu)
    before = wide.clone()
    positions = torch.randint(0, 500, (3, 5), generator=gen, dtype=torch.int32).to(gpu)
    rows.rotary_(wide[..., : 8 * 128], 4, 2, 128, None, None, 0.0, cos, sin, positions)
    check_rotary(before[..., :1024].reshape(15, -1), wide[..., :1024].reshape(15, -1), 4, 2, 128, None, None, 0.0, cos, sin, positions, False)
    assert torch.equal(wide[..., 1024:], before[..., 1024:])
    with pytest.raises(ValueError):  # every other batch element: no one stride
        rows.rotary_(torch.empty(4, 5, 1024, dtype=torch.bfloat16, device=gpu)[::2], 4, 2, 128, None, None, 0.0, cos, sin, positions[:2])
    one = torch.randn(4, 1, 1024, generator=gen).to(torch.bfloat16).to(gpu)
    first = one.clone()
    rows.rotary_(one[::2], 4, 2, 128, None, None, 0.0, cos, sin, positions[:2, :1].contiguous())
    assert torch.equal(one[1::2], first[1::2])
    check_rotary(first[::2, 0], one[::2, 0], 4, 2, 128, None, None, 0.0, cos, sin, positions[:2, :1], False)
    none = torch.empty(0, 1024, dtype=torch.bfloat16, device=gpu)
    rows.rotary_(none, 4, 2, 128, None, None, 0.0, cos, sin, torch.empty(0, dtype=torch.int32, device=gpu))


def test_rotary_of_empty_batches(gpu):
    cos, sin = rows.rope_tables(10, 64, 1e4, gpu)
    for shape in ((0,), (2, 0), (0, 3), (3, 1, 0)):
        x = torch.empty(*shape, 4 * 64, dtype=torch.bfloat16, device=gpu)
        assert rows.rotary_(x, 2, 1, 64, None, None, 0.0, cos, sin, torch.empty(shape, dtype=torch.int32, device=gpu)) is x


@pytest.mark.parametrize("interleaved,dtype", [(False, torch.bfloat16), (True, torch.float16)])
@pytest.mark.parametrize("tokens,Hq,Hkv,D", [(7000, 32, 8, 128), (18000, 14, 2, 128), (4300, 56, 8, 128), (4400, 28, 4, 256), (16600, 28, 4, 64)])
def test_rotary_of_many_tokens(gpu, tokens, Hq, Hkv, D, interleaved, dtype):
    """Batches beyond the caches, bit for bit as in parts."""
    print("rotary", tokens, Hq, Hkv, D, interleaved, flush=True)
    gen = torch.Generator().manual_seed(tokens)
    cos, sin = rows.rope_tables(3000, D, 1e6, gpu)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=gen)).to(gpu) for _ in range(2))
    whole = torch.randn(tokens, (Hq + 2 * Hkv) * D, generator=gen).to(dtype).to(gpu)
    positions = torch.randint(-1, 3001, (tokens,), generator=gen, dtype=torch.int32).to(gpu)
    parts = whole.clone()
    rows.rotary_(whole, Hq, Hkv, D, qw, kw, 1e-6, cos, sin, positions, interleaved)
    for at in range(0, tokens, 2500):
        rows.rotary_(parts[at : at + 2500], Hq, Hkv, D, qw, kw, 1e-6, cos, sin, positions[at : at + 2500], interleaved)
    assert torch.equal(whole.view(torch.int16), parts.view(torch.int16))


def test_rotary_agrees_with_the_batch_form(gpu):
    """One position a batch: what qk_norm_rope_ does, but for its rounding between the steps."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 12 * 128, generator=gen).to(torch.bfloat16).to(gpu)
    y = x.clone()
    cos, sin = rows.rope_tables(100, 128, 1e6, gpu)
    rows.qk_norm_rope_(x, 8, 2, 128, None, None, 0.0, cos, sin, 40)
    rows.rotary_(y, 8, 2, 128, None, None, 0.0, cos, sin, torch.arange(40, 46, dtype=torch.int32, device=gpu).repeat(2, 1))
    assert torch.equal(x, y)  # nothing is normalised: one rounding in both


# ---- together -------------------------------------------------------------------------------------------------------


class Layer:
    """One layer's step of generation: rotary, write, attention, on buffers that stay in place."""

    def __init__(self, gpu, store, lens, Hq, Hkv, D, page, seed):
        dtype, bits = STORES[store]
        self.Hq, self.Hkv, self.D, self.page, self.B = Hq, Hkv, D, page, len(lens)
        self.gen = torch.Generator().manual_seed(seed)
        width = -(-(max(lens) + 20) // page)
        self.buffers = PagedKVCacheBuffers(width * self.B, page, Hkv, D, dtype, bits, gpu)
        self.table = torch.randperm(width * self.B, generator=self.gen).view(self.B, width).to(torch.int32).to(gpu)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=gpu)
        self.cos, self.sin = rows.rope_tables(width * page, D, 1e6, gpu, rotary_dim=D)
        self.qw, self.kw = ((1 + 0.1 * torch.randn(D, generator=self.gen)).to(gpu) for _ in range(2))
        n = max(lens)
        positions = torch.arange(n, dtype=torch.int32, device=gpu)[None].repeat(self.B, 1)
        positions[positions >= self.lens[:, None]] = -1
        key, value = (torch.randn(self.B * n, Hkv, D, generator=self.gen).to(dtype).to(gpu) for _ in range(2))
        self.buffers.write(key, value, self.buffers.slots(self.table, positions))
        self.qkv = torch.empty(self.B, (Hq + 2 * Hkv) * D, dtype=dtype, device=gpu)
        self.positions = torch.empty(self.B, dtype=torch.int32, device=gpu)
        self.slots = torch.empty(self.B, dtype=torch.int64, device=gpu)

    def next(self):
        """New rows, one token longer; sequences of length 0 stay padding."""
        self.lens += (self.lens > 0).to(torch.int32)
        self.positions.copy_(self.lens - 1)
        self.slots.copy_(self.buffers.slots(self.table, self.positions[:, None]))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.gen).to(self.qkv.dtype))
        self.before = self.qkv.clone()

    def step(self):
        rows.rotary_(self.qkv, self.Hq, self.Hkv, self.D, self.qw, self.kw, 1e-6, self.cos, self.sin, self.positions)
        heads = self.qkv.view(self.B, -1, self.D)
        self.buffers.write(heads[:, self.Hq : -self.Hkv], heads[:, -self.Hkv :], self.slots)
        return self.buffers.decode(heads[:, : self.Hq], self.table, self.lens, return_lse=True)

    def check(self, out, lse):
        check_rotary(self.before, self.qkv, self.Hq, self.Hkv, self.D, self.qw, self.kw, 1e-6, self.cos, self.sin, self.positions, False)
        heads = self.qkv.view(self.B, -1, self.D).cpu()
        for b, n in enumerate(self.lens.tolist()):
            k, v = (stored_rows(self.buffers, i, self.table[b].cpu(), n) for i in (0, 1))
            check_decode(out[b].cpu(), lse[b].cpu(), heads[b, : self.Hq], k, v, self.D**-0.5, heads.dtype, stored_spans(self.buffers, self.table[b].cpu(), n))
            if n:  # the new row is the last
                new = heads[b, self.Hq : -self.Hkv].double()
                step = 0.0 if self.buffers.num_bits is None else (new.amax(-1, keepdim=True) - new.amin(-1, keepdim=True)) / ((1 << self.buffers.num_bits) - 1)
                assert ((k[:, -1] - new).abs() <= 1.01 * step + 1e-6).all()


@pytest.mark.parametrize("store", STORES)
def test_steps_of_generation(gpu, store):
    layer = Layer(gpu, store, [15, 0, 200, 31], 8, 2, 128, 16, 21)
    for _ in range(3):
        layer.next()
        layer.check(*layer.step())


@pytest.mark.parametrize("store", ["bf16", "u8", "u4_fp16"])
def test_captured_steps(gpu, store):
    """A captured step, replayed over growing lengths, with eager steps of another layer and the pool's other users between the replays."""
    layer = Layer(gpu, store, [130, 0, 2000, 1], 8, 2, 128, 16, 22)
    other = Layer(gpu, store, [40, 300], 8, 2, 128, 16, 23)
    layer.next()
    layer.step()  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    layer.next()
    with torch.cuda.graph(graph):
        out, lse = layer.step()
    for _ in range(4):
        layer.next()
        graph.replay()
        other.next()
        got = other.step()
        torch.cuda.synchronize()
        other.check(*got)
        layer.check(out, lse)
        again = layer.buffers.decode(layer.qkv.view(layer.B, -1, 128)[:, :8], layer.table, layer.lens, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)  # the eager result


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("store", ["fp16", "u8_fp16", "u4"])
def test_two_captured_steps_in_turn(gpu, store, shared):
    """Two graphs, replayed in either order on a stream of their own, each before the other's results are looked at. Of one memory pool in the order of their
    capture only, as torch asks for: the second graph's results may lie where the first one's workspace was."""
    layers = [Layer(gpu, store, lens, 6, 2, 64, 32, 24 + i) for i, lens in enumerate(([900, 33, 0], [5, 1500]))]
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
        for layer, (out, lse) in zip(layers, results):
            layer.check(out, lse)


def test_a_later_chunk_of_a_prompt(gpu):
    """A chunk attends over the rows read back, as over a contiguous cache."""
    gen = torch.Generator().manual_seed(31)
    T, q_len, Hq, Hkv, D = 300, 40, 8, 2, 128
    k, v = (torch.randn(1, Hkv, T, D, generator=gen).to(torch.bfloat16).to(gpu) for _ in range(2))
    q = torch.randn(1, Hq, q_len, D, generator=gen).to(torch.bfloat16).to(gpu)
    buffers = PagedKVCacheBuffers(30, 16, Hkv, D, device=gpu)
    table = torch.randperm(30, generator=gen).to(torch.int32)[None].to(gpu)
    buffers.write(k[0].transpose(0, 1), v[0].transpose(0, 1), buffers.slots(table, torch.arange(T, device=gpu)[None]))
    kr, vr = buffers.read(table, torch.tensor([T], dtype=torch.int32, device=gpu), T)
    assert torch.equal(kr, k) and torch.equal(vr, v)
    got, want = (ops.prefill_core(q, x, y, D**-0.5, T - q_len)[0] for x, y in ((kr, vr), (k, v)))
    assert torch.equal(got, want)
    # the chunk's last token, as a step over the pages, agrees to the roundings of its weights and of the output in both (2^-8 each)
    out, _ = buffers.decode(q[:, :, -1].contiguous(), table, torch.tensor([T], dtype=torch.int32, device=gpu))
    p = torch.softmax(q[0, :, -1:].double().cpu() @ k[0].double().cpu().repeat_interleave(4, 0).transpose(1, 2) * D**-0.5, -1)
    size = (p @ v[0].double().cpu().abs().repeat_interleave(4, 0))[:, 0]
    assert ((out[0].double() - got[0, -1].double()).abs().cpu() <= 4.2 * 2.0**-8 * size).all()
