"""The prompt pass: what a decoder needs to take whole prompts at once.

* ``plan_kv_blocks``: block tables and slot maps of a packed batch, from its
  requests' lengths, on the device (``sl_plan_kv_blocks``);
* ``Rotary``: rotary positions of query and key heads (``sl_rotary``);
* ``prompt_attention``: causal attention over packed sequences with grouped
  heads (``sl_prompt_attention``).

None of them is part of the reference's operator surface (it runs inside
vLLM, whose block manager, rotary embedding and prefill attention they stand
in for); ``harness.DecoderHarness.prefill`` is the decoder that calls them.
All calls enqueue on the current CUDA stream of their tensors' device and
never synchronise, so they can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib, ptr

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16,
           torch.float32: _lib.DTYPE_FP32}


def _same_device(first: torch.Tensor, **others) -> torch.device:
    """The CUDA device of ``first``, which every other tensor is on too."""
    if not first.is_cuda:
        raise ValueError("sluice_b200 ops take CUDA tensors")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, expected {first.device}")
    return first.device


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _vector(name: str, t: torch.Tensor, dtype: torch.dtype, length: int | None = None) -> None:
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} vector")
    if length is not None and t.numel() != length:
        raise ValueError(f"{name} has {t.numel()} entries, expected {length}")


# ------------------------------------------------------------ block planner
class KvPlanError(_lib.SluiceError):
    """The device found that a plan could not be made in full."""

    def __init__(self, status: int):
        RuntimeError.__init__(self, "plan_kv_blocks: " + (
            "the free cache blocks, or the room in a block table row, ran out"
            if status == _lib.KV_PLAN_NO_BLOCKS else
            "lengths, token counts or a free range that cannot be"))
        self.status = status


class KvPlan(NamedTuple):
    """A packed batch, as ``plan_kv_blocks`` lays it out."""

    cu_new: torch.Tensor            # int32 [B + 1] offsets of the new tokens
    cu_total: torch.Tensor          # int32 [B + 1] offsets of context + new tokens
    positions: torch.Tensor         # int64 [num_tokens] position in its sequence
    slots: torch.Tensor             # int64 [num_tokens] cache row, -1: none
    kv_slots: torch.Tensor | None   # int64 [num_kv_tokens] cache rows of all tokens
    status: torch.Tensor            # int32 [2] KV_PLAN_*, blocks taken

    def check(self) -> None:
        """Raise ``KvPlanError`` if the plan ran out of blocks or was given
        bad lengths (synchronises)."""
        status = int(self.status[0].item())
        if status != _lib.KV_PLAN_OK:
            raise KvPlanError(status)


def plan_kv_blocks(context_lens: torch.Tensor, new_lens: torch.Tensor,
                   block_table: torch.Tensor, free_blocks: torch.Tensor,
                   free_range: torch.Tensor, block_size: int, num_tokens: int, *,
                   num_kv_tokens: int = 0,
                   free_range_out: torch.Tensor | None = None) -> KvPlan:
    """Give every request the cache blocks its new tokens need and map the
    batch's tokens to cache rows.

    ``context_lens`` / ``new_lens`` int32 [B]: tokens cached and to add.
    ``block_table`` int32 [B, width]: row r's first ceil(context / block_size)
    entries are its blocks; the blocks it takes are written behind them.
    ``free_blocks`` int32 [N] is a ring of free block ids whose entries
    [free_range[0], free_range[1]) (int64 [2], taken modulo N) are free: blocks
    are taken from the front in request order, and ``free_range_out`` (default:
    ``free_range`` itself) receives the range that is left. ``num_tokens`` is
    the number of packed rows to fill (at least the sum of ``new_lens``: rows
    behind the last request get position and slot -1); ``num_kv_tokens`` > 0
    asks for the cache rows of all context + new tokens too. A request that
    the ring or its table row cannot hold takes nothing and its new tokens get
    slot -1; ``KvPlan.check`` raises for it.
    """
    B = context_lens.numel()
    _vector("context_lens", context_lens, torch.int32)
    _vector("new_lens", new_lens, torch.int32, B)
    _vector("free_blocks", free_blocks, torch.int32)
    _vector("free_range", free_range, torch.int64, 2)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 \
            or block_table.shape[0] != B:
        raise ValueError(f"block_table must be int32 [{B}, width] with contiguous rows")
    if B > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table's rows overlap")
    if free_range_out is None:
        free_range_out = free_range
    _vector("free_range_out", free_range_out, torch.int64, 2)
    if num_tokens < 0 or num_kv_tokens < 0:
        raise ValueError("num_tokens and num_kv_tokens are counts")
    dev = _same_device(context_lens, new_lens=new_lens, block_table=block_table,
                       free_blocks=free_blocks, free_range=free_range,
                       free_range_out=free_range_out)
    with torch.cuda.device(dev):
        # (the two vectors of a size from one allocation)
        cu = torch.empty(2, B + 1, dtype=torch.int32, device=dev)
        rows = torch.empty(2, num_tokens, dtype=torch.int64, device=dev)
        kv = torch.empty(num_kv_tokens, dtype=torch.int64, device=dev) if num_kv_tokens else None
        status = torch.empty(2, dtype=torch.int32, device=dev)
        check(lib().sl_plan_kv_blocks(
            ptr(context_lens), ptr(new_lens), B, int(block_size), ptr(block_table),
            max(block_table.stride(0), block_table.shape[1]), block_table.shape[1],
            ptr(free_blocks), free_blocks.numel(), ptr(free_range), ptr(free_range_out),
            num_tokens, num_kv_tokens, ptr(cu[0]), ptr(cu[1]), ptr(rows[0]), ptr(rows[1]),
            ptr(kv), ptr(status), _stream(dev)), "sl_plan_kv_blocks")
    return KvPlan(cu[0], cu[1], rows[0], rows[1], kv, status)


# ------------------------------------------------------------------- rotary
def rotary_frequencies(rotary_dim: int, base: float = 10000.0,
                       scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """(radians per position of each pair, float64 [rotary_dim / 2]; the
    factor on the rotated values).

    ``scaling`` None: base^(-2i / rotary_dim). ``{"type": "linear", "factor"}``
    divides the frequencies (positions interpolated); ``"ntk"`` raises the base
    by factor^(d / (d - 2)); ``"yarn"`` (``factor``, ``original_max``,
    ``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor`` 0.1 ln factor + 1)
    keeps the pairs that turn more than ``beta_fast`` times over the trained
    length, divides those that turn less than ``beta_slow`` times and blends in
    between by the pair's index; ``"llama3"`` (``factor``, ``original_max``,
    ``low_freq_factor``, ``high_freq_factor``) does so by wavelength.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even number")
    if not base > 0:
        raise ValueError("base must be positive")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)

    def powers(b: float) -> torch.Tensor:
        return float(b) ** (-2.0 * i / rotary_dim)

    plain = powers(base)
    if scaling is None:
        return plain, 1.0
    kind = scaling.get("type")
    if kind not in ("linear", "ntk", "yarn", "llama3"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    factor = float(scaling["factor"])
    if not factor > 0:
        raise ValueError("the scaling factor must be positive")
    if kind == "linear":
        return plain / factor, 1.0
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        return powers(base * factor ** (rotary_dim / (rotary_dim - 2.0))), 1.0
    trained = float(scaling["original_max"])
    if kind == "yarn":
        def pair_of(turns: float) -> float:
            # the pair index that turns so many times over the trained length
            return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_of(float(scaling.get("beta_fast", 32.0)))), 0)
        high = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1.0)))), rotary_dim - 1)
        stretched = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        m = scaling.get("attention_factor")
        return plain / factor * stretched + plain * (1.0 - stretched), \
            float(m) if m is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    lo_f, hi_f = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
    if not hi_f > lo_f:
        raise ValueError("high_freq_factor must exceed low_freq_factor")
    turns = trained * plain / (2 * math.pi)   # over the trained length
    keep = ((turns - lo_f) / (hi_f - lo_f)).clamp(0.0, 1.0)
    return (1.0 - keep) * plain / factor + keep * plain, 1.0


class Rotary:
    """Rotary positions of ``rotary_dim`` columns of query and key heads.

    ``interleaved``: pairs are adjacent columns; otherwise columns
    ``rotary_dim / 2`` apart. ``base`` and ``scaling`` as in
    ``rotary_frequencies``. Angles are reduced in 64 bits, so there is no
    table and no largest position.
    """

    def __init__(self, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                 interleaved: bool = True, device="cuda"):
        freqs, self.factor = rotary_frequencies(rotary_dim, base, scaling)
        self.rotary_dim = rotary_dim
        self.interleaved = bool(interleaved)
        # turns per position
        self.turns = (freqs / (2 * math.pi)).to(device)

    def _part(self, name: str, x: torch.Tensor, out: torch.Tensor | None, offset: int, T: int):
        if x.dim() != 3 or x.shape[0] != T:
            raise ValueError(f"{name} must be [{T}, heads, dim], got {tuple(x.shape)}")
        if not 0 <= offset <= x.shape[2] - self.rotary_dim:
            raise ValueError(f"{name}'s columns [{offset}, {offset + self.rotary_dim}) are not "
                             f"within its {x.shape[2]}")
        in_place = out is x
        # pairs are read as two elements at once, so they start on even ones
        odd = self.interleaved and any(s % 2 for s, n in zip(x.stride()[:2], x.shape) if n > 1) \
            or self.interleaved and x.data_ptr() % (2 * x.element_size())
        if x.shape[2] > 1 and x.stride(2) != 1 or odd:
            if in_place:
                raise ValueError(f"{name} cannot be rotated in place: its columns must be "
                                 "contiguous and its pairs aligned")
            x = x.contiguous().clone() if x.is_contiguous() else x.contiguous()
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        elif not in_place:
            if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
                raise ValueError(f"out_{name} must match {name}'s shape, type and device")
            if out.shape[2] > 1 and out.stride(2) != 1:
                raise ValueError(f"out_{name}'s columns must be contiguous")
            same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
            if not same and _ranges_meet(x, out):
                raise ValueError(f"out_{name} overlaps {name}; pass {name} itself to rotate it "
                                 "in place")
        if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
            raise ValueError(f"out_{name} has rows that share memory")
        part = _lib.RotaryPart(ptr(x), ptr(out), x.stride(0), x.stride(1), out.stride(0),
                               out.stride(1), x.shape[1], x.shape[2], offset)
        # (x: a copy made above has to outlive the launch)
        return part, out, x

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None,
                 *, q_offset: int = 0, k_offset: int = 0, out_q: torch.Tensor | None = None,
                 out_k: torch.Tensor | None = None):
        """``q`` [T, heads, dim] and ``k`` [T, kv_heads, k_dim] at
        ``positions`` (int64 [T]), columns [offset, offset + rotary_dim) of
        each head rotated and the others copied. Returns (q', k') (q' alone
        without ``k``), new tensors or ``out_q`` / ``out_k``; passing ``q``
        itself as ``out_q`` rotates in place. Rows at negative positions
        (padding) keep their values."""
        if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
            raise ValueError("q and k must share one of bfloat16, float16, float32")
        T = positions.numel()
        _vector("positions", positions, torch.int64)
        if k is None and out_k is not None:
            raise ValueError("out_k without k")
        pq, out_q, _keep_q = self._part("q", q, out_q, q_offset, T)
        pk, _keep_k = None, None
        if k is not None:
            pk, out_k, _keep_k = self._part("k", k, out_k, k_offset, T)
        dev = _same_device(q, positions=positions, k=k, out_q=out_q, out_k=out_k,
                           turns=self.turns)
        with torch.cuda.device(dev):
            check(lib().sl_rotary(ptr(positions), ptr(self.turns), T, self.rotary_dim,
                                  int(self.interleaved), float(self.factor), _DTYPES[q.dtype],
                                  ctypes.byref(pq), ctypes.byref(pk) if pk is not None else None,
                                  _stream(dev)), "sl_rotary")
        return out_q if k is None else (out_q, out_k)


def _ranges_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges that two strided tensors span meet."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


# ---------------------------------------------------------------- attention
def _tiled(t: torch.Tensor) -> torch.Tensor:
    """``t`` in a layout the kernel's tile loads take: contiguous columns,
    strides in multiples of 16 bytes, a 16-byte aligned address."""
    ok = t.data_ptr() % 16 == 0 and (t.shape[-1] == 1 or t.stride(-1) == 1) and \
        all(s % 8 == 0 and s > 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1)
    if ok:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor) -> list[int]:
    """Strides of all but the last dimension; a dimension of one entry is
    given the extent of what is inside it."""
    s = []
    inner = t.shape[-1]
    for n, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        s.append(st if n > 1 else inner)
        inner = max(inner, s[-1] * n)
    return s[::-1]


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: torch.Tensor, *, k_shared: torch.Tensor | None = None,
                     scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed sequences: ``out`` [Tq, heads, v_dim].

    ``q`` [Tq, heads, dim], ``k`` [Tk, kv_heads, dim], ``v`` [Tk, kv_heads,
    v_dim], bfloat16 or float16, (dim, v_dim) one of (64, 64), (128, 128),
    (192, 128); heads a multiple of kv_heads (head h reads key head
    h // (heads // kv_heads)). Sequence b's queries are rows
    [cu_q[b], cu_q[b + 1]) and its keys rows [cu_k[b], cu_k[b + 1]) (int32
    [B + 1]); its queries are its last tokens, so a prompt behind a cached
    beginning, or a single next token, has fewer queries than keys. With
    ``k_shared`` [Tk, 64] (dim 192), ``k`` has the first 128 columns and the
    last 64 are one row for all heads. ``scale`` defaults to dim^-0.5. A query
    that sees no key gets zeros; rows of ``q`` outside every sequence leave
    ``out`` as it was there (a new ``out`` is not initialised).
    """
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v are [tokens, heads, dim]")
    Tq, heads, dim = q.shape
    Tk, kv_heads, own = k.shape
    v_dim = v.shape[2]
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"prompt_attention takes bfloat16 or float16, got {q.dtype}")
    for name, t in (("k", k), ("v", v), ("k_shared", k_shared), ("out", out)):
        if t is not None and t.dtype != q.dtype:
            raise ValueError(f"{name} is {t.dtype}, q is {q.dtype}")
    if v.shape[:2] != k.shape[:2]:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ in tokens or heads")
    shared = 0
    if k_shared is not None:
        if k_shared.dim() != 2 or k_shared.shape[0] != Tk:
            raise ValueError(f"k_shared must be [{Tk}, columns], got {tuple(k_shared.shape)}")
        shared = k_shared.shape[1]
    if own + shared != dim:
        raise ValueError(f"q has {dim} columns per head, k {own} + {shared}")
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of {kv_heads} key heads")
    B = cu_q.numel() - 1
    _vector("cu_q", cu_q, torch.int32)
    _vector("cu_k", cu_k, torch.int32, B + 1)
    if B < 0:
        raise ValueError("cu_q needs at least one entry")
    if out is None:
        out = torch.empty(Tq, heads, v_dim, dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != (Tq, heads, v_dim):
        raise ValueError(f"out must be [{Tq}, {heads}, {v_dim}], got {tuple(out.shape)}")
    elif out.data_ptr() % 16 or out.stride(2) != 1 or any(
            s % 8 or s <= 0 for s, n in zip(out.stride()[:2], out.shape) if n > 1):
        raise ValueError("out needs contiguous columns, strides in multiples of 8 elements and "
                         "a 16-byte aligned address")
    elif any(_ranges_meet(out, t) for t in (q, k, v, k_shared) if t is not None):
        raise ValueError("out overlaps an input")
    dev = _same_device(q, k=k, v=v, cu_q=cu_q, cu_k=cu_k, k_shared=k_shared, out=out)
    if B == 0 or Tq == 0:
        return out
    with torch.cuda.device(dev):
        q, k, v = _tiled(q), _tiled(k), _tiled(v)
        a = _lib.AttentionArgs()
        a.q, a.k, a.v, a.out = ptr(q), ptr(k), ptr(v), ptr(out)
        a.q_token, a.q_head = _strides(q)
        a.k_token, a.k_head = _strides(k)
        a.v_token, a.v_head = _strides(v)
        a.out_token, a.out_head = _strides(out)
        if shared:
            k_shared = _tiled(k_shared)
            a.k_shared = ptr(k_shared)
            a.k_shared_token, = _strides(k_shared)
        a.cu_q, a.cu_k = ptr(cu_q), ptr(cu_k)
        a.Tq, a.Tk, a.B = Tq, Tk, B
        a.heads, a.kv_heads, a.dim, a.v_dim, a.shared_dim = heads, kv_heads, dim, v_dim, shared
        a.dtype = _DTYPES[q.dtype]
        a.scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
        n = lib().sl_prompt_attention_workspace_bytes(B, Tq, Tk, heads, kv_heads, v_dim)
        workspace = torch.empty(max(n, 256), dtype=torch.uint8, device=dev)
        check(lib().sl_prompt_attention(ctypes.byref(a), ptr(workspace), workspace.numel(),
                                        _stream(dev)), "sl_prompt_attention")
    prompt_attention.last_workspace = workspace
    return out


prompt_attention.last_workspace = None
