"""Attention of a decoder layer over a paged cache of keys and values in 4 bits.

The part of a layer between its two projections, which the layer schedules
(`tokenweave_with_fuse_only`, `tokenweave_overlap`) leave to `layer.self_attn`: positions are
turned into the queries and keys (`RotaryPositions`), the new tokens' keys and values go to their
pages (`KVCache4`), and the queries attend over their sequences' pages.  `PagedSelfAttention` is one
tensor-parallel rank's `self_attn` from these parts.

Head sizes of the cache are 64, 128 and 256, in pages of 16 to 256 tokens.
"""
from __future__ import annotations

import math
from typing import Any, Dict, Optional, Tuple

import torch
import torch.nn as nn
from torch.nn.parameter import Parameter

from . import _custom_ops as ops
from .linear import RowParallelLinear


def rotary_frequencies(rotary_dim: int, base: float = 10000.0,
                       scaling: Optional[Dict[str, Any]] = None) -> Tuple[torch.Tensor, float]:
    """(radians a position of each of the rotary_dim / 2 pairs in 64 bits, the factor on cos and sin).

    `scaling` stretches positions for contexts longer than those trained on, by its "type":
      "linear"  every wave `factor` times longer
      "ntk"     a larger base: the longest wave `factor` times longer, the shortest as it was
      "bands"   waves longer than original_max_position / low_freq_factor (default 1) `factor` times
                longer, those shorter than original_max_position / high_freq_factor (default 4)
                as they were, a slope between
      "yarn"    the same idea with the slope over the pairs' numbers, from the pair that turns
                beta_fast (32) times in original_max_position to the one that turns beta_slow (1)
                times; cos and sin are multiplied by attention_factor (0.1 ln(factor) + 1)
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    n = rotary_dim // 2
    pair = torch.arange(n, dtype=torch.float64)
    inv = float(base) ** (-pair / n)
    if scaling is None:
        return inv, 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 1.0))
    if factor <= 0:
        raise ValueError(f"the factor of a scaling must be positive, got {factor}")
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "ntk":
        larger = float(base) * factor ** (n / (n - 1)) if n > 1 else float(base)
        return larger ** (-pair / n), 1.0
    if kind not in ("bands", "yarn"):
        raise ValueError(f'unknown scaling type {kind!r}: "linear", "ntk", "bands" or "yarn"')
    length = float(scaling["original_max_position"])
    if kind == "bands":
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError(f"high_freq_factor {high} must be above low_freq_factor {low}")
        keep = ((length * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return inv * keep + inv / factor * (1 - keep), 1.0

    def pair_that_turns(times: float) -> float:
        return n * math.log(length / (times * 2 * math.pi)) / math.log(base)
    first = max(math.floor(pair_that_turns(float(scaling.get("beta_fast", 32.0)))), 0)
    last = min(math.ceil(pair_that_turns(float(scaling.get("beta_slow", 1.0)))), rotary_dim - 1)
    keep = 1 - ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
    by_default = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return inv * keep + inv / factor * (1 - keep), float(scaling.get("attention_factor", by_default))


class RotaryPositions(nn.Module):
    """A model's table of cosines and sines, and the turning of queries and keys by it.  The table is
    computed in 64 bits and kept in fp32, `rotary_dim * 4` bytes a position."""

    def __init__(self, head_size: int, rotary_dim: Optional[int] = None, max_position: int = 8192,
                 base: float = 10000.0, interleaved: bool = False, scaling: Optional[Dict[str, Any]] = None) -> None:
        super().__init__()
        self.head_size = head_size
        self.rotary_dim = head_size if rotary_dim is None else rotary_dim
        if self.rotary_dim > head_size:
            raise ValueError(f"rotary_dim {self.rotary_dim} is larger than head_size {head_size}")
        if max_position < 1:
            raise ValueError(f"max_position must be positive, got {max_position}")
        self.max_position, self.interleaved = max_position, bool(interleaved)
        inv, factor = rotary_frequencies(self.rotary_dim, base, scaling)
        angle = torch.arange(max_position, dtype=torch.float64)[:, None] * inv
        self.register_buffer("cos_sin", (torch.cat((angle.cos(), angle.sin()), 1) * factor).float(), persistent=False)

    def _apply(self, fn: Any, recurse: bool = True) -> "RotaryPositions":
        """A model's type (`model.bfloat16()`) is not the table's: it stays fp32, on the device it is moved to."""
        table = self.cos_sin
        super()._apply(fn, recurse)
        if self.cos_sin.dtype != torch.float32:
            self.cos_sin = table.to(self.cos_sin.device)
        return self

    def forward(self, positions: torch.Tensor, q: torch.Tensor, k: Optional[torch.Tensor] = None,
                q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """q and k [tokens, heads, head_size], turned in place or into q_out / k_out; returns what holds
        the results."""
        ops.rotary_positions(q, k, positions, self.cos_sin, self.interleaved, inverse, q_out, k_out)
        return q if q_out is None else q_out, k if k_out is None else k_out

    def extra_repr(self) -> str:
        return (f"head_size={self.head_size}, rotary_dim={self.rotary_dim}, max_position={self.max_position}, "
                f"interleaved={self.interleaved}")


class KVCache4:
    """Pages of keys and values in 4 bits (4.25 with the scales).  A slot is page * page_size + place."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_size: int, device: Any = "cuda") -> None:
        if head_size not in (64, 128, 256):
            raise ValueError(f"head_size must be 64, 128 or 256, got {head_size}")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be a power of two from 16 to 256, got {page_size}")
        self.num_pages, self.page_size = num_pages, page_size
        self.num_kv_heads, self.head_size = num_kv_heads, head_size
        self.pages = torch.empty((num_pages, num_kv_heads, self.head_bytes(page_size, head_size)), dtype=torch.uint8,
                                 device=device)

    @staticmethod
    def head_bytes(page_size: int, head_size: int) -> int:
        """Bytes of one head in one page."""
        return page_size * (head_size + head_size // 16)

    def _check(self, name: str, t: torch.Tensor) -> None:
        # (the ops tell a cache's head size from their tensors: pages of another would pass for it)
        if t.size(-1) != self.head_size:
            raise RuntimeError(f"{name} has shape {tuple(t.shape)}, the cache head_size {self.head_size}")

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
               rotary: Optional[RotaryPositions] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> None:
        """Lays the tokens' keys, turned by `rotary` where it is given, and values into their slots;
        turns `q` in the same launch."""
        self._check("k", k)
        ops.kv4_append(self.pages, k, v, slots, positions, None if rotary is None else rotary.cos_sin,
                       False if rotary is None else rotary.interleaved, q, q_out)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The slots' keys and values, [slots, kv_heads, head_size]."""
        k, v = (torch.empty((slots.numel(), self.num_kv_heads, self.head_size), dtype=dtype, device=self.pages.device)
                for _ in range(2))
        ops.kv4_read(k, v, self.pages, slots)
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               scale: Optional[float] = None, query_starts: Optional[torch.Tensor] = None,
               max_queries: Optional[int] = None, window: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the new tokens over their sequences' pages (`ops.kv4_attention`)."""
        self._check("q", q)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ops.kv4_attention(out, q, self.pages, block_table, seq_lens, self.head_size ** -0.5 if scale is None else scale,
                          query_starts, max_queries, window)
        return out


class CachedBatch:
    """What a step's attention needs to know of its tokens.

    slots         [tokens] int64: where each new token goes, -1 for padding
    block_table   [sequences, pages] int32;  seq_lens [sequences] int32, the new tokens among them
    query_starts  [sequences + 1] int32, or None: the same number of new tokens for each sequence
    max_queries   the most new tokens of a sequence
    """

    def __init__(self, slots: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 query_starts: Optional[torch.Tensor] = None, max_queries: Optional[int] = None) -> None:
        self.slots, self.block_table, self.seq_lens = slots, block_table, seq_lens
        self.query_starts, self.max_queries = query_starts, max_queries
        self._splits: Dict[int, Tuple["CachedBatch", "CachedBatch"]] = {}

    def split(self, tokens: int) -> Tuple["CachedBatch", "CachedBatch"]:
        """The first `tokens` tokens and the rest, as the woven schedule runs them one after the other.
        A sequence that both hold ends, in the first, with its last token there.  The halves hold no
        lengths or starts of their own: they follow this batch's tensors where those change in place."""
        whole = (self.slots, self.block_table, self.seq_lens, self.query_starts, self.max_queries)
        halves = self._splits.get(tokens)
        if halves is None or any(a is not b for a, b in zip(halves[0].whole, whole)):
            halves = self._splits[tokens] = (_Half(whole, tokens, False), _Half(whole, tokens, True))
        return halves

    def _operands(self) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[int]]:
        """block_table, seq_lens, query_starts, max_queries as `ops.kv4_attention` takes them."""
        return self.block_table, self.seq_lens, self.query_starts, self.max_queries


class _Half(CachedBatch):
    """A batch's first tokens or the others.  What it says of them is computed from the whole batch's
    tensors every time it is asked for: lengths and starts may change in place, and where the question
    is part of a captured step, so is the answer.  Whole sequences with the same number of new tokens each
    are views, without any operation."""

    def __init__(self, whole: Tuple[Any, ...], tokens: int, second: bool) -> None:
        self.whole, self.tokens, self.second = whole, tokens, second
        self._splits = {}
        slots, _, lens, starts, _ = whole
        # new tokens of each sequence; 0: not the same for all
        self._each = slots.numel() // max(lens.numel(), 1) if starts is None else 0
        if starts is None and slots.numel() != self._each * lens.numel():
            raise RuntimeError(f"{slots.numel()} tokens are not the same number for each of {lens.numel()} sequences: "
                               "pass query_starts")
        # the sequences of this half, where none is in both
        self._rows = None
        if self._each and tokens % self._each == 0:
            at = tokens // self._each
            self._rows = slice(at, None) if second else slice(0, at)

    def _starts(self) -> torch.Tensor:
        """The whole batch's query_starts."""
        lens, starts = self.whole[2:4]
        if starts is None:
            starts = torch.arange(lens.numel() + 1, dtype=torch.int32, device=lens.device) * self._each
        return starts

    @property
    def slots(self) -> torch.Tensor:
        return self.whole[0][self.tokens:] if self.second else self.whole[0][:self.tokens]

    @property
    def block_table(self) -> torch.Tensor:
        return self.whole[1] if self._rows is None else self.whole[1][self._rows]

    @property
    def seq_lens(self) -> torch.Tensor:
        if self._rows is not None:
            return self.whole[2][self._rows]
        if self.second:
            return self.whole[2]
        behind = (self._starts() - self.tokens).clamp_(min=0)
        return self.whole[2] - (behind[1:] - behind[:-1])

    @property
    def query_starts(self) -> Optional[torch.Tensor]:
        if self._rows is not None:
            return None
        return (self._starts() - self.tokens).clamp_(min=0) if self.second else self._starts().clamp(max=self.tokens)

    @property
    def max_queries(self) -> Optional[int]:
        """The whole batch's bound; where it names none and its sequences have the same number, that number."""
        bound = self.whole[4]
        return self._each if bound is None and self.whole[3] is None else bound

    def _operands(self) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[int]]:
        if self._rows is not None:
            return super()._operands()
        # the whole batch's lengths and starts: the op leaves out what is not in this half.  One operation instead of
        # seven for the halves' own: 61 us for both halves of a captured layer of 512 channels instead of 70.
        starts = self._starts()
        return self.whole[1], self.whole[2], starts - self.tokens if self.second else starts, self.max_queries


class PagedSelfAttention(nn.Module):
    """One rank's self-attention: qkv projection, rotation, append, attention, and the row-parallel
    output projection that leaves this rank's partial sum in `hidden_states`, for the layer schedules to
    reduce.  `num_heads` and `num_kv_heads` are this rank's.  `begin(batch)` names the step's tokens."""

    def __init__(self, hidden_size: int, num_heads: int, num_kv_heads: int, head_size: int, rotary: RotaryPositions,
                 cache: KVCache4, window: int = 0, qkv_bias: bool = False, *, tp_rank: int = 0, tp_size: int = 1) -> None:
        super().__init__()
        if num_heads % num_kv_heads:
            raise ValueError(f"{num_heads} query heads over {num_kv_heads} key heads")
        self.num_heads, self.num_kv_heads, self.head_size, self.window = num_heads, num_kv_heads, head_size, window
        width = (num_heads + 2 * num_kv_heads) * head_size
        self.qkv_weight = Parameter(torch.empty(width, hidden_size, dtype=torch.bfloat16), requires_grad=False)
        if qkv_bias:
            self.qkv_bias = Parameter(torch.empty(width, dtype=torch.bfloat16), requires_grad=False)
        else:
            self.register_parameter("qkv_bias", None)
        self.o_proj = RowParallelLinear(num_heads * head_size * tp_size, hidden_size, bias=False, tp_rank=tp_rank,
                                        tp_size=tp_size)
        self.rotary, self.cache = rotary, cache
        self.batch: Optional[CachedBatch] = None

    def begin(self, batch: CachedBatch) -> None:
        """The tokens of the calls that follow."""
        self.batch = batch

    def forward(self, positions: torch.Tensor, hidden_states: torch.Tensor, split_id: Optional[int] = None,
                split_size: int = 0, num_actual_tokens: Optional[int] = None,
                gemm_cus: Optional[int] = None) -> torch.Tensor:
        if self.batch is None:
            raise RuntimeError("PagedSelfAttention: begin(batch) names the step's tokens before the first call")
        batch = self.batch if split_id is None else self.batch.split(split_size)[split_id]
        n = hidden_states.shape[0] if num_actual_tokens is None else num_actual_tokens
        x, D, Hq, Hk = hidden_states[:n], self.head_size, self.num_heads, self.num_kv_heads
        qkv = torch.empty((n, self.qkv_weight.shape[0]), dtype=x.dtype, device=x.device)
        ops.gemm_bf16_nt(qkv, x, self.qkv_weight.data, None, None if self.qkv_bias is None else self.qkv_bias.data)
        q, k, v = (t.view(n, t.shape[1] // D, D) for t in qkv.split((Hq * D, Hk * D, Hk * D), 1))
        self.cache.append(k, v, batch.slots, positions[:n], self.rotary, q)
        table, lens, starts, bound = batch._operands()
        out = self.cache.attend(q, table, lens, None, starts, bound, self.window,
                                torch.empty((n, Hq, D), dtype=q.dtype, device=q.device))
        self.o_proj(out.view(n, Hq * D), x, is_tokenweave=True, gemm_cus=gemm_cus)
        return hidden_states
