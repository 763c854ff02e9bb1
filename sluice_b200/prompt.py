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
import functools
import math
import operator
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib, ptr

# the current stream's handle without the object around it (a few microseconds
# a call; the same value as torch.cuda.current_stream(device).cuda_stream)
_raw_stream = torch._C._cuda_getCurrentRawStream

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16,
           torch.float32: _lib.DTYPE_FP32}


_INT_MAX = 0x7fffffff
_ROTARY_ROWS = _INT_MAX - 64   # of one call


def _device_index(first: torch.Tensor, *others) -> int:
    """The index of the CUDA device of ``first``, which every other tensor is
    on too."""
    if not first.is_cuda:
        raise ValueError("sluice_b200 ops take CUDA tensors")
    dev = first.get_device()
    for t in others:
        if t is not None and (not t.is_cuda or t.get_device() != dev):
            raise ValueError(f"a tensor is on {t.device}, expected {first.device}")
    return dev


def _no_gradient(*tensors) -> None:
    """Refuse what autograd would silently cut off."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("this operator has no backward pass: call it under torch.no_grad(), "
                             "or with detached tensors")


def _call(dev: int, name: str, *args) -> None:
    """``name`` of the library with ``args`` and the current stream of device
    ``dev``, which is made the current one where it is not."""
    fn = getattr(lib(), name)
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    check(rc, name)


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
                   block_table: torch.Tensor, free_blocks: torch.Tensor | None,
                   free_range: torch.Tensor | None, block_size: int, num_tokens: int, *,
                   num_kv_tokens: int = 0,
                   free_range_out: torch.Tensor | None = None) -> KvPlan:
    """Give every request the cache blocks its new tokens need and map the
    batch's tokens to cache rows.

    ``context_lens`` / ``new_lens`` int32 [B], B at most 8192: tokens cached and
    to add.
    ``block_table`` int32 [B, width]: row r's first ceil(context / block_size)
    entries are its blocks; the blocks it takes are written behind them.
    ``free_blocks`` int32 [N] is a ring of free block ids whose entries
    [free_range[0], free_range[1]) (int64 [2], taken modulo N) are free: blocks
    are taken from the front in request order, and ``free_range_out`` (default:
    ``free_range`` itself) receives the range that is left. With ``free_blocks``
    and ``free_range`` None the table rows are complete and nothing is taken
    (a cache whose sequences own their blocks). ``num_tokens`` is
    the number of packed rows to fill (at least the sum of ``new_lens``: rows
    behind the last request get position and slot -1); ``num_kv_tokens`` > 0
    asks for the cache rows of all context + new tokens too. A request that
    the ring or its table row cannot hold takes nothing and its new tokens get
    slot -1; ``KvPlan.check`` raises for it.
    """
    _vector("context_lens", context_lens, torch.int32)
    B = len(context_lens)
    _vector("new_lens", new_lens, torch.int32, B)
    if (free_blocks is None) != (free_range is None) or \
            (free_blocks is None and free_range_out is not None):
        raise ValueError("free_blocks and free_range come together")
    if free_blocks is not None:
        _vector("free_blocks", free_blocks, torch.int32)
        _vector("free_range", free_range, torch.int64, 2)
    shape, strides = block_table.shape, block_table.stride()
    if block_table.dtype != torch.int32 or len(shape) != 2 or strides[1] != 1 or shape[0] != B:
        raise ValueError(f"block_table must be int32 [{B}, width] with contiguous rows")
    width = shape[1]
    ld = strides[0] if B > 1 else width
    if ld < width:
        raise ValueError("block_table's rows overlap")
    if free_range_out is None:
        free_range_out = free_range
    else:
        _vector("free_range_out", free_range_out, torch.int64, 2)
        if abs(free_range_out.data_ptr() - free_range.data_ptr()) == 8:
            raise ValueError("free_range_out overlaps half of free_range")
    if num_tokens < 0 or num_kv_tokens < 0:
        raise ValueError("num_tokens and num_kv_tokens are counts")
    block_size = int(block_size)
    ring = 0 if free_blocks is None else free_blocks.numel()
    if max(block_size, width, ring) > _INT_MAX:
        raise ValueError("block_size, the table's width and the ring's size are 32-bit numbers")
    dev = _device_index(context_lens, new_lens, block_table, free_blocks, free_range,
                        free_range_out)
    # one allocation: the 64-bit outputs, then the 32-bit ones
    n64 = 2 * num_tokens + num_kv_tokens
    buf = torch.empty(n64 + B + 2, dtype=torch.int64, device=context_lens.device)
    r = buf.data_ptr()
    c = r + 8 * n64
    _call(dev, "sl_plan_kv_blocks", context_lens.data_ptr(), new_lens.data_ptr(), B,
          block_size, block_table.data_ptr(), ld, width, ptr(free_blocks), ring, ptr(free_range),
          ptr(free_range_out), num_tokens, num_kv_tokens, c, c + 4 * (B + 1), r,
          r + 8 * num_tokens, r + 16 * num_tokens if num_kv_tokens else None, c + 8 * (B + 1))
    # (views; "unsafe" to autograd only, which has no part in this)
    positions, slots, kv, rest = torch.unsafe_split_with_sizes(
        buf, (num_tokens, num_tokens, num_kv_tokens, B + 2))
    cu_new, cu_total, status = torch.unsafe_split_with_sizes(rest.view(torch.int32),
                                                             (B + 1, B + 1, 2))
    return KvPlan(cu_new, cu_total, positions, slots, kv if num_kv_tokens else None, status)


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
        """(the call's description of one tensor, its output, its input)."""
        in_place = out is x
        offset = operator.index(offset)   # (layouts are kept by value)
        copied, x_strides, new = _rotary_input(name, x.shape, x.stride(), offset, T,
                                               self.rotary_dim)
        if out is None and new is not None:
            # the usual call: a new output like a contiguous input
            out = torch.empty_like(x)
            part = _lib.RotaryPart.from_buffer_copy(new)
            part.x, part.y = x.data_ptr(), out.data_ptr()
            return part, out, x
        if copied:
            if in_place:
                raise ValueError(f"{name} cannot be rotated in place: its columns must be "
                                 "contiguous")
            x = x.clone(memory_format=torch.contiguous_format)
            x_strides = x.stride()
        if out is None:
            out = x.new_empty(x.shape)
        elif not in_place:
            if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
                raise ValueError(f"out_{name} must match {name}'s shape, type and device")
            if out.shape[2] > 1 and out.stride(2) != 1:
                raise ValueError(f"out_{name}'s columns must be contiguous")
            same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
            if not same and _ranges_meet(x, out):
                raise ValueError(f"out_{name} overlaps {name}; pass {name} itself to rotate it "
                                 "in place")
        y_strides = out.stride()
        if not _own_rows(out.shape, y_strides):
            raise ValueError(f"out_{name} has rows that share memory")
        _, heads, dim = x.shape
        return _lib.RotaryPart(x.data_ptr(), out.data_ptr(), x_strides[0], x_strides[1],
                               y_strides[0], y_strides[1], heads, dim, offset), out, x

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None,
                 *, q_offset: int = 0, k_offset: int = 0, out_q: torch.Tensor | None = None,
                 out_k: torch.Tensor | None = None):
        """``q`` [T, heads, dim] and ``k`` [T, kv_heads, k_dim] at
        ``positions`` (int64 [T]), columns [offset, offset + rotary_dim) of
        each head rotated and the others copied. Returns (q', k') (q' alone
        without ``k``), new tensors or ``out_q`` / ``out_k``; passing ``q``
        itself as ``out_q`` rotates in place. Rows at negative positions
        (padding) keep their values. Up to 512 rotated columns of up to 4096,
        fewer than 2^20 columns in all heads of a token, and fewer than
        2^31 - 64 rows."""
        dtype = _DTYPES.get(q.dtype)
        if dtype is None or (k is not None and k.dtype != q.dtype):
            raise ValueError("q and k must share one of bfloat16, float16, float32")
        T = positions.numel()
        _vector("positions", positions, torch.int64)
        _no_gradient(q, k, out_q, out_k)
        if k is None and out_k is not None:
            raise ValueError("out_k without k")
        given_q, given_k = out_q, out_k
        pq, out_q, q = self._part("q", q, out_q, q_offset, T)
        pk = None
        if k is not None:
            pk, out_k, k = self._part("k", k, out_k, k_offset, T)
            if given_q is not None and (_meet(out_q, k) or _meet(out_q, out_k)):
                raise ValueError("out_q overlaps k or out_k")
            if given_k is not None and _meet(out_k, q):
                raise ValueError("out_k overlaps q")
        _call(_device_index(q, positions, k, self.turns), "sl_rotary", ptr(positions),
              ptr(self.turns), T, self.rotary_dim, self.interleaved, self.factor, dtype,
              ctypes.byref(pq), None if pk is None else ctypes.byref(pk))
        return out_q if k is None else (out_q, out_k)


@functools.lru_cache(maxsize=512)
def _rotary_input(name: str, shape, strides, offset: int, T: int, rot: int):
    """(whether the input has to be copied first, its strides, and, for a
    contiguous input, the description of a call that writes a new tensor,
    without the addresses), by its layout."""
    if len(shape) != 3 or shape[0] != T:
        raise ValueError(f"{name} must be [{T}, heads, dim], got {tuple(shape)}")
    if T > _ROTARY_ROWS:
        raise ValueError(f"{T} rows in one call, at most {_ROTARY_ROWS}")
    if not 0 <= offset <= shape[2] - rot:
        raise ValueError(f"{name}'s columns [{offset}, {offset + rot}) are not within its "
                         f"{shape[2]}")
    copied = shape[2] > 1 and strides[2] != 1
    new = None
    if not copied and strides == (shape[1] * shape[2], shape[2], 1):
        new = _lib.RotaryPart(None, None, strides[0], strides[1], strides[0], strides[1],
                              shape[1], shape[2], offset)
    return copied, strides, new


def _ranges_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges that two strided tensors span meet."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [T, heads, columns] tensors with contiguous columns may
    share memory: their address ranges meet, and not just because they are
    different columns, or heads, of the rows of one buffer."""
    if not _ranges_meet(a, b):
        return False
    apart, rest = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    if rest or a.element_size() != b.element_size():
        return True
    for d in range(2):
        # every address modulo the step of a token, or of a head (a divisor of
        # the tokens')
        step = a.stride(d)
        if step <= 0 or b.stride(d) != step or \
                (d == 1 and any(t.shape[0] > 1 and t.stride(0) % step for t in (a, b))):
            continue
        of_a, of_b = (1 + sum((n - 1) * s for n, s in zip(t.shape[d + 1:], t.stride()[d + 1:]))
                      for t in (a, b))
        if of_a <= apart % step and apart % step + of_b <= step:
            return False
    return True


@functools.lru_cache(maxsize=512)
def _own_rows(shape, strides) -> bool:
    """Whether every row (contiguous columns) of such a layout has memory of
    its own: each step goes past all that is inside it."""
    inner = shape[-1]
    for step, n in sorted((s, n) for s, n in zip(strides[:-1], shape) if n > 1):
        if step < inner:
            return False
        inner += step * (n - 1)
    return True


# ---------------------------------------------------------------- attention
def _tiled(t: torch.Tensor) -> torch.Tensor:
    """``t`` in a layout the kernel's tile loads take: contiguous columns,
    strides in multiples of 16 bytes, a 16-byte aligned address."""
    if t.data_ptr() % 16 or not _tile_strides(t.shape, t.stride()):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _tile_strides(shape, strides) -> bool:
    return (shape[-1] <= 1 or strides[-1] == 1) and \
        all(s % 8 == 0 and s > 0 for s, n in zip(strides[:-1], shape) if n > 1)


def _strides(shape, strides) -> list[int]:
    """Strides of all but the last dimension; a dimension of one entry is
    given the extent of what is inside it."""
    s = []
    inner = shape[-1]
    for n, st in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        s.append(st if n > 1 else inner)
        inner = max(inner, s[-1] * n)
    return s[::-1]


@functools.lru_cache(maxsize=512)
def _attention_layout(q, k, v, k_shared, out, dtype, nq: int, nk: int, scale):
    """The call's description by its tensors' layouts, each (shape, strides)
    (``k_shared`` None; ``out`` None: a new one), without the addresses; the
    output's shape; whether the tile loads take the inputs' strides."""
    if len(q[0]) != 3 or len(k[0]) != 3 or len(v[0]) != 3:
        raise ValueError("q, k and v are [tokens, heads, dim]")
    Tq, heads, dim = q[0]
    Tk, kv_heads, own = k[0]
    v_dim = v[0][2]
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"prompt_attention takes bfloat16 or float16, got {dtype}")
    if v[0][:2] != k[0][:2]:
        raise ValueError(f"k {tuple(k[0])} and v {tuple(v[0])} differ in tokens or heads")
    shared = 0
    if k_shared is not None:
        if len(k_shared[0]) != 2 or k_shared[0][0] != Tk:
            raise ValueError(f"k_shared must be [{Tk}, columns], got {tuple(k_shared[0])}")
        shared = k_shared[0][1]
    if own + shared != dim:
        raise ValueError(f"q has {dim} columns per head, k {own} + {shared}")
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of {kv_heads} key heads")
    if nq > _INT_MAX:
        raise ValueError(f"{nq - 1} sequences in one call")
    if nq < 1 or nk != nq:
        raise ValueError(f"cu_q has {nq} entries and cu_k {nk}: both have one per sequence and "
                         "one more")
    if out is None:
        out = ((Tq, heads, v_dim), (heads * v_dim, v_dim, 1))
    elif tuple(out[0]) != (Tq, heads, v_dim):
        raise ValueError(f"out must be [{Tq}, {heads}, {v_dim}], got {tuple(out[0])}")
    elif out[1][2] != 1 or any(s % 8 or s <= 0 for s, n in zip(out[1][:2], out[0]) if n > 1):
        raise ValueError("out needs contiguous columns and strides in multiples of 8 elements")
    elif not _own_rows(*out):
        raise ValueError("out has rows that share memory")
    a = _lib.AttentionArgs()
    a.q_token, a.q_head = _strides(*q)
    a.k_token, a.k_head = _strides(*k)
    a.v_token, a.v_head = _strides(*v)
    a.out_token, a.out_head = _strides(*out)
    if shared:
        a.k_shared_token, = _strides(*k_shared)
    a.Tq, a.Tk, a.B = Tq, Tk, nq - 1
    a.heads, a.kv_heads, a.dim, a.v_dim, a.shared_dim = heads, kv_heads, dim, v_dim, shared
    a.dtype = _DTYPES[dtype]
    a.scale = 1.0 / math.sqrt(dim) if scale is None else scale
    tiled = all(t is None or _tile_strides(*t) for t in (q, k, v, k_shared))
    return a, (Tq, heads, v_dim), tiled


@functools.lru_cache(maxsize=512)
def _workspace_bytes(B: int, Tq: int, Tk: int, heads: int, kv_heads: int, v_dim: int,
                     dev: int) -> int:
    with torch.cuda.device(dev):   # (the size goes by the device's SMs)
        return max(256, lib().sl_prompt_attention_workspace_bytes(B, Tq, Tk, heads, kv_heads,
                                                                  v_dim))


# a status word per device, which its calls raise and ``check_attention`` reads
# and clears; kept for good, as captured calls hold its address
_failed: dict[int, torch.Tensor] = {}


def _failed_word(dev: int) -> torch.Tensor | None:
    word = _failed.get(dev)
    if word is None:
        with torch.cuda.device(dev), torch.inference_mode(False):
            # (what a capture allocates belongs to its graph: the word of a
            # process whose first call is captured comes with a later call)
            if not torch.cuda.is_current_stream_capturing():
                word = _failed.setdefault(dev, torch.zeros(1, dtype=torch.int32, device="cuda"))
    return word


def check_attention(device="cuda") -> None:
    """Raise if a bounded wait ran out in a ``prompt_attention`` call without
    a ``status`` of its own, on this device since the last check, so that its
    output is not to be used (synchronises)."""
    device = torch.device(device)
    word = _failed.get(torch.cuda.current_device() if device.index is None else device.index)
    if word is None:
        return
    status = int(word.item())
    word.zero_()
    check(status, "prompt_attention")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: torch.Tensor, *, k_shared: torch.Tensor | None = None,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed sequences: ``out`` [Tq, heads, v_dim].

    ``q`` [Tq, heads, dim], ``k`` [Tk, kv_heads, dim], ``v`` [Tk, kv_heads,
    v_dim], bfloat16 or float16, (dim, v_dim) one of (64, 64), (128, 128),
    (192, 128); heads a multiple of kv_heads (head h reads key head
    h // (heads // kv_heads)). Sequence b's queries are rows
    [cu_q[b], cu_q[b + 1]) and its keys rows [cu_k[b], cu_k[b + 1]) (int32
    [B + 1]); its queries are its last tokens, so a prompt behind a cached
    beginning, or a single next token, has fewer queries than keys. With
    ``k_shared`` [Tk, 64] (dim 192), ``k`` has the first 128 columns and the
    last 64 are one row for all heads. ``scale`` (positive) defaults to dim^-0.5. A query
    that sees no key gets zeros; rows of ``q`` outside every sequence leave
    ``out`` as it was there (a new ``out`` is not initialised).

    ``status`` (int32 [1]; default: a word of the device's, which
    ``check_attention`` reads) is raised to the code of the error, and never
    lowered, when a bounded wait of the device ran out.
    """
    for name, t in (("k", k), ("v", v), ("k_shared", k_shared), ("out", out)):
        if t is not None and t.dtype != q.dtype:
            raise ValueError(f"{name} is {t.dtype}, q is {q.dtype}")
    _no_gradient(q, k, v, k_shared, out)
    _vector("cu_q", cu_q, torch.int32)
    _vector("cu_k", cu_k, torch.int32)
    if status is not None:
        _vector("status", status, torch.int32, 1)
    if scale is not None:
        scale = float(scale)   # (layouts are kept by value)
    for copied in (False, True):
        layout, shape, tiled = _attention_layout(
            (q.shape, q.stride()), (k.shape, k.stride()), (v.shape, v.stride()),
            None if k_shared is None else (k_shared.shape, k_shared.stride()),
            None if out is None else (out.shape, out.stride()), q.dtype, len(cu_q), len(cu_k),
            scale)
        addresses = q.data_ptr() | k.data_ptr() | v.data_ptr()
        if k_shared is not None:
            addresses |= k_shared.data_ptr()
        if copied or (tiled and not addresses % 16):
            break
        q, k, v = _tiled(q), _tiled(k), _tiled(v)
        k_shared = None if k_shared is None else _tiled(k_shared)
    a = _lib.AttentionArgs.from_buffer_copy(layout)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    elif out.data_ptr() % 16:
        raise ValueError("out needs a 16-byte aligned address")
    elif any(_ranges_meet(out, t) for t in (q, k, v, k_shared) if t is not None):
        raise ValueError("out overlaps an input")
    dev = _device_index(q, k, v, cu_q, cu_k, k_shared, out, status)
    if a.B == 0 or a.Tq == 0:
        return out
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.cu_q, a.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
    if a.shared_dim:
        a.k_shared = k_shared.data_ptr()
    n = _workspace_bytes(a.B, a.Tq, a.Tk, a.heads, a.kv_heads, a.v_dim, dev)
    workspace = torch.empty(n, dtype=torch.uint8, device=q.device)
    if status is None:
        status = _failed_word(dev)
    _call(dev, "sl_prompt_attention_ex", ctypes.byref(a), workspace.data_ptr(), n, ptr(status))
    # (as other operators name the tensor that starts with their status)
    prompt_attention.last_workspace = status
    return out


prompt_attention.last_workspace = None
