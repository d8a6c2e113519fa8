"""Angles for long contexts through the chunked-prefill model: what its layers rotate queries and keys by."""
import math

import pytest
import torch

from keys_values_amd.longctx import ops
from keys_values_amd.longctx.model import LongContextPrefillModel, PrefillConfig

pytestmark = pytest.mark.gpu
BASE, D, CONTEXT = 1.0e4, 64, 64  # CONTEXT: that the scalings take for the trained one


def frequency(kind, factor, j):
    """Pair j's angle per position, and the amplitude, from the definitions."""
    f = BASE ** (-2 * j / D)
    turns = CONTEXT * f / (2 * math.pi)
    if kind == "linear":
        return f / factor, 1.0
    if kind == "ntk":
        return (BASE * factor ** (D / (D - 2))) ** (-2 * j / D), 1.0
    if kind == "banded":  # four turns and more over the trained context are kept, one and fewer divided
        keep = min(max((turns - 1.0) / 3.0, 0.0), 1.0)
        return keep * f + (1 - keep) * f / factor, 1.0
    pair = [D * math.log(CONTEXT / (2 * math.pi * t)) / (2 * math.log(BASE)) for t in (32.0, 1.0)]
    low, high = max(math.floor(pair[0]), 0), math.ceil(pair[1])
    ramp = min(max((j - low) / (high - low), 0.0), 1.0)
    return (1 - ramp) * f + ramp * f / factor, 0.1 * math.log(factor) + 1.0


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("kind,factor", [("linear", 4.0), ("ntk", 8.0), ("banded", 8.0), ("yarn", 4.0)])
def test_prefill_with_scaled_angles(gpu, monkeypatch, kind, factor, norm):
    cfg = PrefillConfig(n_layer=2, n_embd=128, n_head=4, n_query_groups=2, head_size=D, intermediate_size=256, vocab_size=200, rope_base=BASE, norm_qk=norm,
                        rope_scaling=ops.RopeScaling(kind, factor, original_context=CONTEXT))
    model = LongContextPrefillModel(cfg, cache_length=256, chunk_size=64, quantized=False, max_context=400, device=gpu)
    for layer in model.layers:
        if norm:
            layer.norm_q.uniform_(0.5, 1.5)
            layer.norm_k.uniform_(0.5, 1.5)
    rotated = []
    turn = ops.qk_norm_rope_

    def spy(qkv, *args):
        before = qkv.cpu()
        turn(qkv, *args)
        rotated.append((args[-1], before, qkv.cpu(), args[3], args[4]))
        return qkv

    monkeypatch.setattr(ops, "qk_norm_rope_", spy)
    ids = torch.randint(0, cfg.vocab_size, (1, 390), generator=torch.Generator().manual_seed(1))
    out = model.prefill(ids)
    assert torch.isfinite(out).all() and len(rotated) >= 4 and rotated[-1][0] + rotated[-1][1].shape[1] == 390
    freq, m = zip(*(frequency(kind, factor, j) for j in range(D // 2)))
    for start, before, after, *weights in rotated:
        x, got = (t.view(-1, 8, D).double() for t in (before, after))
        assert torch.equal(got[:, 6:], x[:, 6:])  # value heads
        x = x[:, :6].clone()
        if norm:
            x = x / (x.square().sum(-1, keepdim=True).sqrt() / math.sqrt(D) + cfg.norm_eps)
            x[:, :4] *= weights[0].cpu().double()
            x[:, 4:] *= weights[1].cpu().double()
        angle = (start + torch.arange(x.shape[0], dtype=torch.float64))[:, None] * torch.tensor(freq, dtype=torch.float64)
        cos, sin = (angle.cos() * m[0])[:, None], (angle.sin() * m[0])[:, None]
        a, b = x[..., : D // 2], x[..., D // 2 :]
        want = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        size = torch.cat((a.abs() * cos.abs() + b.abs() * sin.abs(), b.abs() * cos.abs() + a.abs() * sin.abs()), -1)
        # one rounding to bf16, fp32 before it; a normalised head is rounded to bf16 before it is rotated, too
        tol = 2.0**-8 * want.abs() + size * (2.0**-18 + (2.0**-8 * (1 + 2.0**-8) if norm else 0.0))
        err = (got[:, :6] - want).abs()
        assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} tolerances at {start}"
