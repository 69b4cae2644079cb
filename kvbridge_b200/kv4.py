"""The 4-bit paged KV cache: append, read back, attention, accumulated
attention weights and eviction (include/kvbridge/attention_kv4.h).

The classes hold the device buffers of a call and its checked description, so
that a serving loop builds them once and each call is one trip through the C
ABI. Buffers are CUDA tensors; their types, shapes and strides are checked
when the object is made (``ValueError``), and the objects keep them alive.
Calls run on the given stream, or on torch's current one, and need the
buffers' device to be the current device.
"""
from __future__ import annotations

import ctypes
from ctypes import byref
from typing import Optional

import torch

from . import _lib
from ._lib import KvbKv4Eviction, KvbKv4Pool, KvbKv4Query, KvbKv4Rows, check

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _tensor(name: str, x, dtype, shape=None, like=None) -> int:
    """Address of a contiguous CUDA tensor of this dtype (and shape, a tuple)."""
    try:
        if (
            x.dtype is dtype
            and x.is_cuda
            and (shape is None or x.shape == shape)
            and (like is None or x.device == like)
            and x.is_contiguous()
        ):
            return x.data_ptr()
    except AttributeError:
        pass
    _device(name, x, like)
    if x.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {x.dtype}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(x.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _device(name: str, x, like=None) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if like is not None and x.device != like:
        raise ValueError(f"{name} is on {x.device}, the other buffers on {like}")


def _optional(name: str, x, dtype, shape, like) -> Optional[int]:
    return None if x is None else _tensor(name, x, dtype, shape, like)


def _strides(name: str, x, inner: int) -> tuple:
    """The outer strides of a tensor whose last `inner` dims are contiguous."""
    want = 1
    for size, stride in zip(reversed(x.shape[-inner:]), reversed(x.stride()[-inner:])):
        if size != 1 and stride != want:
            raise ValueError(f"the last {inner} dims of {name} must be contiguous")
        want *= size
    return x.stride()[:-inner]


# The stream's handle without a Stream object around it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream
)


def _stream(stream, device) -> Optional[int]:
    index = device.index
    if index != torch.cuda.current_device():
        raise ValueError(f"the buffers are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    if stream is None:
        return _raw_stream(index) or None
    if not isinstance(stream, int):
        stream = stream.cuda_stream
    return stream or None


class Kv4Pool:
    """Pages of 4-bit K and V: ``k`` uint8 [pages, kv_heads, page_tokens,
    dim / 2], ``v`` uint8 [pages, kv_heads, dim / 2, page_tokens], ``k_params``
    and ``v_params`` float32 [pages, kv_heads, page_tokens, 2] (scale, lo) and
    optionally ``positions`` int32 [pages, kv_heads, page_tokens]."""

    def __init__(self, k, v, k_params, v_params, positions=None):
        _device("k", k)
        if k.dim() != 4:
            raise ValueError("k must have shape [pages, kv_heads, page_tokens, dim / 2]")
        pages, heads, page, half = k.shape
        self.pages, self.kv_heads, self.page_tokens, self.dim = pages, heads, page, 2 * half
        self.k, self.v, self.k_params, self.v_params, self.positions = k, v, k_params, v_params, positions
        self.device = k.device
        self._c = KvbKv4Pool(
            heads, 2 * half, page, pages,
            _tensor("k", k, torch.uint8, None, self.device),
            _tensor("v", v, torch.uint8, (pages, heads, half, page), self.device),
            _tensor("k_params", k_params, torch.float32, (pages, heads, page, 2), self.device),
            _tensor("v_params", v_params, torch.float32, (pages, heads, page, 2), self.device),
            _optional("positions", positions, torch.int32, (pages, heads, page), self.device),
        )
        error = _lib.load().kvb_kv4_pool_error(byref(self._c))
        if error:
            raise ValueError(error.decode())
        self._ref = byref(self._c)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_tokens: int, dim: int, device="cuda", positions: bool = False):
        """A pool of unwritten pages."""
        half = dim // 2
        params = (pages, kv_heads, page_tokens, 2)
        return cls(
            torch.empty((pages, kv_heads, page_tokens, half), dtype=torch.uint8, device=device),
            torch.empty((pages, kv_heads, half, page_tokens), dtype=torch.uint8, device=device),
            torch.empty(params, device=device),
            torch.empty(params, device=device),
            torch.empty(params[:-1], dtype=torch.int32, device=device) if positions else None,
        )


class Kv4Rows:
    """Dense K and V rows [tokens, kv_heads, dim] (float32, float16 or
    bfloat16; tokens may be strided) and the int64 slots [tokens] they belong
    to: page * page_tokens + slot, negative to skip. ``positions`` int32
    [tokens] is for pools that keep positions."""

    def __init__(self, k, v, slots, positions=None):
        _device("k", k)
        self.device = k.device
        _device("v", v, self.device)
        if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have the same type and shape [tokens, kv_heads, dim]")
        if k.dtype not in TYPES:
            raise ValueError(f"k and v must be float32, float16 or bfloat16, not {k.dtype}")
        self.k, self.v, self.slots, self.positions = k, v, slots, positions
        tokens, self.kv_heads, self.dim = k.shape
        self._c = KvbKv4Rows(
            tokens, TYPES[k.dtype], k.data_ptr(), v.data_ptr(), _strides("k", k, 2)[0], _strides("v", v, 2)[0],
            _tensor("slots", slots, torch.int64, (tokens,), self.device),
            _optional("positions", positions, torch.int32, (tokens,), self.device),
        )
        self._ref = byref(self._c)


def _match(pool: Kv4Pool, rows: Kv4Rows) -> None:
    if (rows.kv_heads, rows.dim) != (pool.kv_heads, pool.dim) or rows.device != pool.device:
        raise ValueError("the rows' kv_heads, dim or device differ from the pool's")


def append_kv4(pool: Kv4Pool, rows: Kv4Rows, stream=None) -> None:
    """Quantise the rows and write them to their slots (distinct in a call)."""
    _match(pool, rows)
    check(_lib.load().kvb_append_kv4(pool._ref, rows._ref, _stream(stream, pool.device)))


def load_kv4(pool: Kv4Pool, rows: Kv4Rows, stream=None) -> None:
    """Write the values that the slots hold to the rows (zeros where skipped)."""
    _match(pool, rows)
    check(_lib.load().kvb_load_kv4(pool._ref, rows._ref, _stream(stream, pool.device)))


class Kv4Query:
    """Query rows ``q`` [batch, rows, q_heads, dim] (float32, float16 or
    bfloat16; batch and rows may be strided) of sequences of ``seq_lens`` int32
    [batch] cached tokens on the pages of ``block_table`` int32 [batch, width].

    The score of a row at position pq and a token at pk is scale * q.k, then
    softcap * tanh(x / softcap) if ``softcap``, then minus slopes[head] * |pq -
    pk| if ``slopes`` (float32 [q_heads]). A token is visible if pk <= pq and,
    with a ``window``, pq - pk < window, or if pk < prefix_lens[b] (int32
    [batch]; a negative one counts as 0 and is reported as a length). pq is ``q_positions`` int32 [batch, rows], or seq_len - rows + r."""

    def __init__(self, q, seq_lens, block_table, max_tokens: int, kv_heads: int, scale: float, softcap: float = 0.0,
                 slopes=None, window: int = 0, prefix_lens=None, q_positions=None):
        _device("q", q)
        self.device = q.device
        if q.dim() != 4:
            raise ValueError("q must have shape [batch, rows, q_heads, dim]")
        if q.dtype not in TYPES:
            raise ValueError(f"q must be float32, float16 or bfloat16, not {q.dtype}")
        batch, rows, q_heads, dim = q.shape
        _device("block_table", block_table, self.device)
        if block_table.dim() != 2:
            raise ValueError("block_table must have shape [batch, width]")
        if kv_heads < 1 or q_heads % kv_heads:
            raise ValueError("q_heads must be divisible by kv_heads")
        if not 0 <= window < 1 << 32 or not 0 <= max_tokens < 1 << 31:
            raise ValueError("window and max_tokens must not be negative")
        self.q, self.dtype, self.shape, self.kv_heads = q, q.dtype, q.shape, kv_heads
        self.lse_shape = q.shape[:3]
        self.max_tokens = max_tokens
        self._kept = (seq_lens, block_table, slopes, prefix_lens, q_positions)
        strides = _strides("q", q, 2)
        width = block_table.shape[1]
        self._c = KvbKv4Query(
            batch, rows, q_heads, width, max_tokens, TYPES[q.dtype], scale, softcap, window,
            q.data_ptr(), strides[0], strides[1],
            _tensor("seq_lens", seq_lens, torch.int32, (batch,), self.device),
            _tensor("block_table", block_table, torch.int32, (batch, width), self.device),
            _optional("q_positions", q_positions, torch.int32, (batch, rows), self.device),
            _optional("slopes", slopes, torch.float32, (q_heads,), self.device),
            _optional("prefix_lens", prefix_lens, torch.int32, (batch,), self.device),
        )
        self._ref = byref(self._c)


def _match_query(pool: Kv4Pool, query: Kv4Query) -> None:
    if query.kv_heads != pool.kv_heads or query.shape[3] != pool.dim or query.device != pool.device:
        raise ValueError("the query's kv_heads, dim or device differ from the pool's")


def attention_kv4_workspace_bytes(pool: Kv4Pool, query: Kv4Query) -> int:
    _match_query(pool, query)
    out = ctypes.c_size_t()
    check(_lib.load().kvb_attention_kv4_workspace_bytes(pool._ref, query._ref, byref(out)))
    return out.value


def launch_attention_kv4(pool: Kv4Pool, query: Kv4Query, workspace, out, lse=None, stream=None) -> None:
    """Attention of the query over the pool: ``out`` like q but contiguous,
    ``lse`` float32 [batch, rows, q_heads] (natural log), -inf and zeros for a
    row that sees nothing. ``workspace`` uint8, attention_kv4_workspace_bytes."""
    _match_query(pool, query)
    check(
        _lib.load().kvb_launch_attention_kv4(
            pool._ref, query._ref, _tensor("workspace", workspace, torch.uint8, None, pool.device), workspace.numel(),
            _tensor("out", out, query.dtype, query.shape, pool.device),
            None if lse is None else _tensor("lse", lse, torch.float32, query.lse_shape, pool.device),
            _stream(stream, pool.device),
        )
    )


def accumulate_weights_kv4(pool: Kv4Pool, query: Kv4Query, lse, weights, stream=None) -> None:
    """Add to ``weights`` float32 [batch, kv_heads, >= max_tokens] the attention
    weight each token gets from the query rows, given their ``lse``."""
    _match_query(pool, query)
    batch = query.shape[0]
    _device("weights", weights, pool.device)
    if weights.dim() != 3 or weights.shape[:2] != (batch, pool.kv_heads):
        raise ValueError("weights must have shape [batch, kv_heads, >= max_tokens]")
    check(
        _lib.load().kvb_accumulate_weights_kv4(
            pool._ref, query._ref, _tensor("lse", lse, torch.float32, query.lse_shape, pool.device),
            _tensor("weights", weights, torch.float32, None, pool.device), weights.shape[2],
            _stream(stream, pool.device),
        )
    )


class EvictPlan:
    """Keep ``budget`` tokens of every sequence and KV head: the first
    ``sinks``, the last ``recent`` and those of the largest ``weights`` (float32
    [batch, kv_heads, width]) among the rest. ``seq_lens`` int32 [batch] (at most
    width), ``block_table`` int32 [batch, pages]."""

    def __init__(self, weights, seq_lens, block_table, budget: int, sinks: int = 0, recent: int = 0):
        _device("weights", weights)
        if weights.dim() != 3:
            raise ValueError("weights must have shape [batch, kv_heads, tokens]")
        if min(budget, sinks, recent) < 0 or max(budget, sinks, recent) >= 1 << 31:
            raise ValueError("budget, sinks and recent must not be negative")
        self.batch, self.kv_heads, width = weights.shape
        self.device, self.budget = weights.device, budget
        self.weights, self.block_table = weights, block_table
        self._kept = seq_lens
        self._keep_shape, self._lens_shape = (self.batch, self.kv_heads, budget), (self.batch,)
        self._table = _tensor("block_table", block_table, torch.int32, None, self.device)
        if block_table.dim() != 2 or block_table.shape[0] != self.batch:
            raise ValueError("block_table must have shape [batch, pages]")
        self._width = block_table.shape[1]
        self._c = KvbKv4Eviction(
            self.batch, self.kv_heads, width, budget, sinks, recent,
            _tensor("seq_lens", seq_lens, torch.int32, (self.batch,), self.device),
            _tensor("weights", weights, torch.float32, None, self.device), width,
        )
        error = _lib.load().kvb_kv4_eviction_error(byref(self._c))
        if error:
            raise ValueError(error.decode())
        self._ref = byref(self._c)


def select_tokens(plan: EvictPlan, keep, kept_lens, stream=None) -> None:
    """``keep`` int32 [batch, kv_heads, budget]: the kept tokens, ascending, then
    zeros; ``kept_lens`` int32 [batch], a tensor apart from ``seq_lens``."""
    check(
        _lib.load().kvb_select_tokens(
            plan._ref, _tensor("keep", keep, torch.int32, plan._keep_shape, plan.device),
            _tensor("kept_lens", kept_lens, torch.int32, plan._lens_shape, plan.device), _stream(stream, plan.device),
        )
    )


def compact_kv4(pool: Kv4Pool, plan: EvictPlan, keep, new_table, new_weights=None, stream=None) -> None:
    """Copy the kept tokens in order to the pages of ``new_table`` int32 [batch,
    pages] (pages that the plan's block table does not use) and their weights to
    ``new_weights`` float32 [batch, kv_heads, >= budget] (the first budget of each),
    a tensor apart from the plan's."""
    if pool.device != plan.device:
        raise ValueError("the plan's device differs from the pool's")
    _device("new_table", new_table, pool.device)
    if new_weights is not None:
        _device("new_weights", new_weights, pool.device)
    if new_table.dim() != 2 or new_table.shape[0] != plan.batch:
        raise ValueError("new_table must have shape [batch, pages]")
    if new_weights is not None and (new_weights.dim() != 3 or new_weights.shape[:2] != (plan.batch, plan.kv_heads)):
        raise ValueError("new_weights must have shape [batch, kv_heads, >= budget]")
    check(
        _lib.load().kvb_compact_kv4(
            pool._ref, plan._ref, plan._table, plan._width,
            _tensor("keep", keep, torch.int32, plan._keep_shape, plan.device),
            _tensor("new_table", new_table, torch.int32, None, plan.device), new_table.shape[1],
            _optional("new_weights", new_weights, torch.float32, None, plan.device),
            0 if new_weights is None else new_weights.shape[2], _stream(stream, plan.device),
        )
    )
