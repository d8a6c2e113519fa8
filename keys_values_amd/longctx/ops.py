"""Host wrappers of the normalisation / rotary / gated-activation kernels (C ABI: kvx_rmsnorm_rows,
kvx_add_rmsnorm_rows, kvx_swiglu_rows, kvx_qk_norm_rope, kvx_rotary)."""
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from keys_values_amd import _lib


@dataclass(frozen=True)
class RopeScaling:
    """Angles for contexts longer than the ``original_context`` tokens that a model was trained on, by the frequencies f of the unscaled encoding
    (n = rotary_dim):

    ``"linear"``: f / factor (positions interpolated).
    ``"ntk"``: those of the base times factor^(n / (n - 2)), which leaves the highest alone and divides the lowest by ``factor``.
    ``"banded"``: f where a wave is shorter than original_context / high_freq_factor tokens, f / factor where it is longer than
    original_context / low_freq_factor, and between the two the mean of both, weighted linearly by original_context / wavelength.
    ``"yarn"`` (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models", 2023): f where it turns more than ``beta_fast`` times
    over the original context, f / factor where fewer than ``beta_slow``, a ramp linear in j between; cos and sin times
    ``attention_factor``, by default 0.1 ln(factor) + 1."""

    kind: str
    factor: float
    original_context: int = 8192
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: Optional[float] = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "banded", "yarn"):
            raise ValueError(f"kind = {self.kind!r}, must be 'linear', 'ntk', 'banded' or 'yarn'")
        if not (self.factor >= 1.0 and self.original_context >= 1):
            raise ValueError(f"factor = {self.factor}, original_context = {self.original_context}: must be at least 1")
        if self.kind == "banded" and not (0.0 < self.low_freq_factor < self.high_freq_factor):
            raise ValueError(f"low_freq_factor = {self.low_freq_factor} must be positive and below high_freq_factor = {self.high_freq_factor}")
        if self.kind == "yarn" and not (0.0 < self.beta_slow < self.beta_fast):
            raise ValueError(f"beta_slow = {self.beta_slow} must be positive and below beta_fast = {self.beta_fast}")
        if self.kind == "yarn" and not (self.original_context > 2.0 * math.pi * self.beta_slow):  # the first pair turns original_context / 2 pi times
            raise ValueError(f"original_context = {self.original_context}: no pair turns beta_slow = {self.beta_slow} times over it")

    def frequencies(self, rotary_dim: int, base: float) -> torch.Tensor:
        """Angle per position of pair j, float64 (rotary_dim / 2,)."""
        j = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
        if self.kind == "ntk" and rotary_dim > 2:
            base = base * self.factor ** (rotary_dim / (rotary_dim - 2))
        f = base ** (-j / rotary_dim)
        if self.kind == "linear" or (self.kind == "ntk" and rotary_dim == 2):
            return f / self.factor
        if self.kind == "banded":
            waves = self.original_context * f / (2.0 * math.pi)
            keep = ((waves - self.low_freq_factor) / (self.high_freq_factor - self.low_freq_factor)).clamp(0.0, 1.0)
            return f * keep + f / self.factor * (1.0 - keep)
        if self.kind == "yarn":
            def pair(turns):  # j (real) of the pair that turns so often over the original context
                return rotary_dim * math.log(self.original_context / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

            low, high = max(math.floor(pair(self.beta_fast)), 0), min(math.ceil(pair(self.beta_slow)), rotary_dim - 1)
            ramp = ((j / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
            return f * (1.0 - ramp) + f / self.factor * ramp
        return f

    def amplitude(self) -> float:
        if self.kind != "yarn":
            return 1.0
        return 0.1 * math.log(self.factor) + 1.0 if self.attention_factor is None else self.attention_factor


def rope_tables(context: int, head_size: int, base: float, device, rotary_dim: Optional[int] = None,
                scaling: Optional[RopeScaling] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 cos / sin tables (context, head_size / 2): row p holds cos / sin of p * base^(-2j / head_size).
    Half-split convention: element d of a head is paired with d +- head_size / 2
    (keys_values/fused/fused_rope.py:57-87,198-200).

    ``rotary_dim``: tables (context, rotary_dim / 2) for :func:`rotary_` on the first part of the heads. ``scaling``: for long contexts. With either of
    them the angles are formed in 64 bits (in 32, as without, the angles of position 131072 are off by up to 0.004)."""
    if rotary_dim is not None or scaling is not None:
        n = head_size if rotary_dim is None else rotary_dim
        if not (0 < n <= head_size and n % 2 == 0):
            raise ValueError(f"rotary_dim = {n} must be even, positive and at most head_size = {head_size}")
        f = base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) if scaling is None else scaling.frequencies(n, base)
        angle = torch.arange(context, dtype=torch.float64, device=device).unsqueeze(-1) * f.to(device)
        m = 1.0 if scaling is None else scaling.amplitude()
        return (angle.cos() * m).float().contiguous(), (angle.sin() * m).float().contiguous()
    inv = 1.0 / (base ** (torch.arange(0, head_size, 2, dtype=torch.float32, device=device) / head_size))
    ang = torch.arange(context, dtype=torch.float32, device=device).unsqueeze(-1) * inv
    return ang.cos().contiguous(), ang.sin().contiguous()


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMSNorm.forward over the last axis (keys_values/model.py:870-878). x bf16 (..., dim), rows contiguous."""
    return _lib.host().rmsnorm(x, weight, eps, out)


def add_rmsnorm_(x: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """``x += delta`` (in place, rounded to bf16) and ``RMSNorm(x)`` in one pass: the residual add of a
    block with the normalisation that follows it (keys_values/model.py:560-584). Returns the normed rows."""
    return _lib.host().add_rmsnorm(x, delta, weight, eps)


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` for ``gate_up = [gate | up]`` (..., 2 * dim), the output of one GEMM over the
    stacked fc_1 / fc_2 weights; same rounding as ``F.silu(gate) * up`` on bf16 tensors."""
    return _lib.host().swiglu(gate_up)


def qk_norm_rope_(qkv: torch.Tensor, n_head: int, n_query_groups: int, head_size: int, q_weight: Optional[torch.Tensor],
                  k_weight: Optional[torch.Tensor], eps: float, cos: torch.Tensor, sin: torch.Tensor, input_pos: int) -> torch.Tensor:
    """In place on qkv (B, num, (n_head + 2 n_query_groups) * head_size): norm_q / norm_k over each
    head and the rotary encoding at positions input_pos .. input_pos + num - 1
    (keys_values/model.py:733-775). Returns qkv."""
    _lib.host().qk_norm_rope(qkv, n_head, n_query_groups, head_size, q_weight, k_weight, eps, cos, sin, input_pos)
    return qkv


def rotary_(qkv: torch.Tensor, n_head: int, n_query_groups: int, head_size: int, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float,
            cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """In place on qkv (..., (n_head + 2 n_query_groups) * head_size), bfloat16 or float16: norm_q / norm_k over each head, where weights are given,
    and the rotary encoding of every token at its own position, ``positions`` int32 of qkv's leading shape. For batches whose sequences
    have positions of their own; :func:`qk_norm_rope_` is for one position a batch, and rounds between the two steps.

    The tables' width says how much of a head is rotated: its first 2 * cos.shape[1] values (a multiple of 16). Pairs are the halves of that part, or with
    ``interleaved`` neighbours; frequencies for long contexts come with the tables (``rope_tables``). Tokens of a negative
    position (padding), and of one behind the tables, are left as they are. The positions are read on the device alone, so nothing is raised for
    those behind the tables: make the tables as long as the cache's sequences can get. Returns qkv."""
    _lib.host().rotary(qkv, n_head, n_query_groups, head_size, q_weight, k_weight, eps, cos, sin, positions, interleaved)
    return qkv
