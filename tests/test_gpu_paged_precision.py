"""How exact attention of one token over pages is, where looser bounds would not show a part of the arithmetic that is missing or cut off, against the same
mathematics in 64 bits."""
import math

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


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("store", ["u8_fp16", "u4_fp16"])
def test_codes_beside_rows_of_large_scales(gpu, store, D):
    """V rows of zeros with a scale 2^10 times that of the others, every fourth: code and zero point in the middle. They have no part in the outputs, and what is multiplied
    with them must not cut the others' products short: a product of 2^10 w with a bare code, a subnormal number of exponent -14, would cut those with w at 2^-24 2^-14
    2^10, a sixteenth of a code.

    Weights are all equal (q = 0). In units of a small row's scale times its codes: a weight in two parts of fp16 is off by 2^-20 of itself at most (its second part may
    be subnormal, 2^-25 where the first is 2^-4 or more). Products are cut at 2^-24 of the largest of 8; one rounding of 2^-24 for each of the sums of 8 and of the joins, 72
    with those of the zero points' part. All of them relative to sum w (half the codes), of 4-bit codes' first half, which are whole bytes over 16, 9 / 8 of it."""
    pool = Pool(gpu, store, [96, 31], 2, D, 16, seed=D)
    bits, buffers = pool.bits, pool.buffers
    mid, packed = (8, 0x88) if bits == 4 else (128, 128)
    small = buffers.quant.v_scale.clone()
    buffers.v[:, :, ::4] = packed
    buffers.quant.v_zp[:, :, ::4] = mid
    buffers.quant.v_scale[:, :, ::4] *= 2.0**10
    q = torch.zeros(2, 4, D, dtype=pool.dtype)
    out, _ = buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu)
    for b, n in enumerate(pool.lens):
        values = pool.rows[1][b].clone()
        values[:, ::4] = 0.0
        ref = values.mean(1).repeat_interleave(2, 0)
        half = small.cpu()[pool.table[b, : -(-n // 16)].long()].transpose(0, 1).flatten(1)[:, :n].clone()
        half[:, ::4] = 0.0
        half = (half * 2.0 ** (bits - 1) * 1.125).double().mean(1).repeat_interleave(2, 0)[:, None]
        tol = 2.0**-11 * ref.abs() + half * (2.0**-20 + 80 * 2.0**-24) * (1 + 2.0**-11) + 2.0**-25
        err = (out[b].double().cpu() - ref).abs()
        assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} tolerances"


@pytest.mark.parametrize("store,Hq,D,factor", [("u4_fp16", 16, 64, 1.0), ("u4_fp16", 8, 128, 0.01), ("u8_fp16", 8, 128, 1.0), ("u8_fp16", 4, 256, 0.3)])
def test_long_sequences_of_codes_are_off_by_the_outputs_rounding(gpu, store, Hq, D, factor):
    """Root mean square over the outputs: the rounding to fp16 of the 64-bit result, and at most a fifth of that beside it (in quadrature, 1.02). One sequence is shared by all
    compute units, four wavefronts each, so 50000 keys are some 100 roundings of fp32 to a wavefront, with the joins: 100^(1/2) 2^-25 of sums that are, without the middle
    code, about |v| n^(-1/2), as the outputs are: a thousandth of the outputs' rounding. The weights' logits are off by D^(1/2) 2^-24 |q k| in the mean, 2^-18, which moves
    outputs by less than 2^-18, where the outputs' rounding is 2^-12."""
    n = 50000
    pool = Pool(gpu, store, [n], 1, D, 64, seed=D)
    q = (factor * torch.randn(1, Hq, D, generator=pool.gen)).to(pool.dtype)
    out, _ = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu)
    ref = torch.softmax(q[0].double() @ pool.rows[0][0][0].T * D**-0.5, -1) @ pool.rows[1][0][0]
    off, rounding = ((x.double().cpu() - ref).norm().item() for x in (out[0], ref.to(pool.dtype)))
    assert off <= 1.02 * rounding, f"{off / rounding:.4f} times the rounding"


def by_hand(pool, q, b):
    """The outputs' terms p v in 64 bits, (Hq, n, D): of weights that are all positive, so that an infinite value is not multiplied by 0."""
    keys, values = (pool.rows[i][b].repeat_interleave(q.shape[1] // pool.Hkv, 0) for i in (0, 1))
    p = torch.softmax((keys @ q[b].double()[..., None])[..., 0] * pool.D**-0.5, -1)
    assert (p > 0).all()
    return p[..., None] * values


@pytest.mark.parametrize("lens,page", [([1, 2, 300, 40], 16), ([20000, 1, 3], 64)])
@pytest.mark.parametrize("store,D", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp16", 64), ("fp16", 128), ("fp16", 256)])
def test_infinite_values(gpu, store, D, lens, page):
    """A live key's infinite value makes its column infinite, with any weight; two of either sign, or a NaN, make it NaN. Other columns are what they are without."""
    print("infinite", store, D, lens, flush=True)
    pool = Pool(gpu, store, lens, 2, D, page, seed=D)
    q = (3.0 * torch.randn(len(lens), 8, D, generator=pool.gen)).to(pool.dtype)
    plain, _ = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu)
    for b, n in enumerate(lens):
        for j, t in enumerate(sorted({0, n // 3, n // 2, n - 1})):  # some of them with weights that 16 bits do not hold
            at = (int(pool.table[b, t // page]), j % 2, t % page)
            for column, value in ((7 * j, math.inf), (7 * j + 1, -math.inf), (3, (-1.0) ** (j // 2) * math.inf), (D - 1 - j, math.nan)):
                pool.buffers.v[(*at, column)] = value
                pool.rows[1][b][j % 2, t, column] = value
    out, lse = pool.buffers.decode(q.to(gpu), pool.table_gpu, pool.lens_gpu, return_lse=True)
    assert torch.isfinite(lse).all()
    got, plain = out.double().cpu(), plain.double().cpu()
    for b in range(len(lens)):
        want = by_hand(pool, q, b).sum(1)
        infinite, finite = torch.isinf(want), torch.isfinite(want)
        assert torch.equal(torch.isnan(got[b]), torch.isnan(want)) and infinite.any() and finite.any()
        assert torch.equal(got[b][infinite], want[infinite]) and torch.equal(got[b][finite], plain[b][finite])


@pytest.mark.parametrize("store", ["u8", "u4_fp16"])
def test_infinite_scales(gpu, store):
    """Rows of codes whose scale is not finite make their heads' outputs infinite or NaN, and no others."""
    pool = Pool(gpu, store, [100, 31], 2, 64, 16, seed=5)
    q = torch.randn(2, 4, 64, generator=pool.gen).to(pool.dtype).to(gpu)
    before = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu)[0]
    pool.buffers.quant.v_scale[int(pool.table[0, 2]), 1, 3] = math.inf
    out = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu)[0]
    assert not torch.isfinite(out[0, 2:]).any() and torch.equal(out[0, :2], before[0, :2]) and torch.equal(out[1], before[1])


@pytest.mark.parametrize("store", ["bf16", "fp16", "u8", "u4_fp16"])
def test_infinite_values_in_masked_places(gpu, store):
    """Of tokens in pages that the pool does not have, and behind the end."""
    pool = Pool(gpu, store, [100, 31], 1, 64, 16, seed=5)
    q = torch.randn(2, 4, 64, generator=pool.gen).to(pool.dtype).to(gpu)
    pool.table_gpu[0, 2] = -1
    before = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu)[0]
    for p, places in ((int(pool.table[0, 2]), slice(0, 16)), (int(pool.table[0, 6]), slice(4, 16)), (int(pool.table[1, 1]), slice(15, 16))):
        if pool.bits is None:
            pool.buffers.v[p, 0, places] = math.inf
        else:
            pool.buffers.quant.v_scale[p, 0, places] = math.inf
    after = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu)[0]
    assert torch.isfinite(before).all() and torch.equal(before, after)


@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("store", ["bf16", "fp16"])
def test_infinite_values_beside_masked_ones(gpu, store, page):
    """The column of a live infinite value holds infinities of the other sign, and NaN, in masked places."""
    pool = Pool(gpu, store, [3 * page + 5, 2 * page, 7], 2, 128, page, seed=6)
    q = torch.randn(3, 8, 128, generator=pool.gen).to(pool.dtype).to(gpu)
    v = pool.buffers.v
    for b, n in enumerate(pool.lens):
        v[int(pool.table[b, 0]), :, 4, 9] = math.inf
        last = int(pool.table[b, (n - 1) // page])
        v[last, :, (n - 1) % page + 1 :, 9] = -math.inf
        v[last, :, (n - 1) % page + 1 :, 10] = math.nan
    for b, at, entry in ((0, 1, -1), (1, 1, pool.num_pages + 7)):
        v[int(pool.table[b, at]), :, :, 9] = math.nan
        pool.table_gpu[b, at] = entry
    out, lse = pool.buffers.decode(q, pool.table_gpu, pool.lens_gpu, return_lse=True)
    assert torch.isfinite(lse).all() and (out[..., 9] == math.inf).all()
    out[..., 9] = 0.0
    assert torch.isfinite(out).all()
