"""Both parts of the weights of attention of one token over pages. A weight meets V as two numbers of 16 bits, itself rounded and what the rounding drops, for plain rows
and for codes with fp16 outputs (codes with bf16 outputs: the first alone). Outputs are rounded to 16 bits too, which hides what a weight's rounding does to them, unless
they cancel: here the signs of every column of V are such that the terms p v of one query head add up to next to nothing, while sum p |v| stays.

Bound: u |o| for the output (u: half a step, bf16 2^-8, fp16 2^-11); (sum p |v|) times the weights' error, which is u^2 in two parts and u in one, with u = 2^-11 for codes;
and 2^-17 (sum p |v|) for fp32: logits are exact (a query of one value that is not 0), their factor and difference are rounded, 3 2^-24 of at most 16 binary orders, the
exponential is off by 2^-23, 8 products are cut at 2^-24 of the largest and 100 sums are rounded. fp16 weights that are not normal numbers are off by 2^-32 of the largest.
Of codes |v| is scale |code - middle|."""
import math

import pytest
import torch

from keys_values_amd.kvcache.paged import PagedKVCacheBuffers

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STORES = {"bf16": (torch.bfloat16, None), "fp16": (torch.float16, None), "u8": (torch.bfloat16, 8), "u8_fp16": (torch.float16, 8), "u4": (torch.bfloat16, 4),
          "u4_fp16": (torch.float16, 4)}
CASES = [(store, D, n) for store in STORES for D, n in ((64, 300), (128, 77), (256, 700))]
GROUP = 4


class Cancelling:
    """One KV head's rows and GROUP queries; column d of V cancels for query d % GROUP."""

    def __init__(self, store, D, n):
        self.dtype, self.bits = STORES[store]
        self.D, self.n, gen = D, n, torch.Generator().manual_seed(n + D)
        self.q = torch.zeros(GROUP, D, dtype=self.dtype)
        for g in range(GROUP):
            self.q[g, 5 * g] = (4.0, -2.0, 1.0, 8.0)[g]
        self.key = (torch.randint(-64, 65, (n, D), generator=gen) / 64.0).to(self.dtype)
        self.key_codes = (torch.randint(0, 1 << (self.bits or 1), (n, D), generator=gen), 2.0 ** -(self.bits or 1), 1 << ((self.bits or 1) - 1))  # codes, scale, zero point
        keys = self.key.double() if self.bits is None else (self.key_codes[0] - self.key_codes[2]).double() * self.key_codes[1]
        self.logits = self.q.double() @ keys.T
        self.p = torch.softmax(self.logits, -1)
        if self.bits is None:
            self.size = (0.5 + torch.rand(n, D, generator=gen)).to(self.dtype).double()
        else:
            self.scale = 0.5 + torch.rand(n, generator=gen)
            self.codes = torch.randint(1, 1 << (self.bits - 1), (n, D), generator=gen)
            self.size = self.codes * self.scale.double()[:, None]
        self.sign = torch.empty(n, D, dtype=torch.float64)
        for d in range(D):
            terms = self.p[d % GROUP] * self.size[:, d]
            total = 0.0
            for i in torch.argsort(terms, descending=True).tolist():
                s = -1.0 if total > 0 else 1.0
                self.sign[i, d] = s
                total += s * terms[i].item()
        self.value = self.sign * self.size
        self.exact = self.p @ self.value

    def bound(self):
        u, met = HALF_STEP[self.dtype], self.p @ self.size
        if self.bits is None:
            weights = u * u
        else:
            weights = 2.0**-22 if self.dtype == torch.float16 else 2.0**-11
        lost = 0.0 if self.bits is None and self.dtype == torch.bfloat16 else self.n * 2.0**-32 * self.size.max()
        return u * self.exact.abs() + (weights + 2.0**-17) * met * (1 + u) + lost + (2.0**-25 if self.dtype == torch.float16 else 0.0)

    def model(self, second):
        """The outputs before their rounding, of weights rounded as the operands are; the second part times ``second``."""
        kept = torch.float16 if self.bits else self.dtype
        w = torch.exp2(((self.logits - self.logits.amax(-1, keepdim=True)) / math.log(2.0)).float() + (7.0 if kept == torch.float16 else 0.0))
        total = w.double().sum(-1, keepdim=True)
        if self.bits is None:
            rows = self.value
        else:
            per = 2.0 ** -math.ceil(math.log2(self.scale.max().item()))
            w, rows = w * (self.scale * per), self.sign * self.codes / per
        first = w.to(kept)
        rest = (w - first.float()).to(kept)
        return (first.double() + second * rest.double()) @ rows / total


@pytest.mark.parametrize("store,D,n", CASES)
def test_the_bound_sees_the_second_part(store, D, n):
    """In the arithmetic's model: within the bound, and beyond it without the second part, or with its sign turned."""
    c = Cancelling(store, D, n)
    bound = c.bound()
    one_part = c.bits is not None and c.dtype == torch.bfloat16

    def off(second):
        return ((c.model(second).to(c.dtype).double() - c.exact).abs() / bound).max().item()

    assert off(0.0 if one_part else 1.0) <= 1.0
    if not one_part:
        assert off(0.0) > 2.0 and off(-1.0) > 4.0


@pytest.mark.gpu
@pytest.mark.parametrize("store,D,n", CASES)
def test_weights_in_two_parts(gpu, store, D, n):
    c, page = Cancelling(store, D, n), 16
    pages = -(-n // page)
    buffers = PagedKVCacheBuffers(pages, page, 1, D, c.dtype, c.bits, gpu)
    at = torch.arange(n)
    if c.bits is None:
        buffers.write(c.key[:, None].to(gpu), c.value[:, None].to(c.dtype).to(gpu), at.to(gpu))
    else:
        middle = 1 << (c.bits - 1)
        for pages_of, codes in ((buffers.k, c.key_codes[0]), (buffers.v, middle + (c.sign * c.codes).long())):
            if c.bits == 4:
                codes = codes[:, : D // 2] << 4 | codes[:, D // 2 :]
            rows = torch.zeros(pages * page, codes.shape[1], dtype=torch.uint8)
            rows[:n] = codes.to(torch.uint8)
            pages_of.copy_(rows.view(pages, 1, page, -1))
        scales = torch.ones(pages * page)
        scales[:n] = c.scale
        for t, x in zip(buffers.quant, (c.key_codes[1], c.key_codes[2], scales.view(pages, 1, page).to(gpu), middle)):
            t.copy_(x) if torch.is_tensor(x) else t.fill_(x)
    table = torch.arange(pages, dtype=torch.int32, device=gpu)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    out, _ = buffers.decode(c.q[None].to(gpu), table, lens, 1.0)
    err = (out[0].double().cpu() - c.exact).abs() / c.bound()
    assert (err <= 1.0).all(), f"off by {err.max().item():.2f} tolerances"
