"""CPU tier of the prompt pass: rotary frequencies, the plan oracle against a
token-by-token allocator, and the calls that are refused."""

import ctypes
import math

import pytest
import torch

from oracle import prompt as oprompt
from sluice_b200 import _lib, prompt


def test_plain_linear_and_ntk_frequencies():
    f, m = prompt.rotary_frequencies(64)
    assert m == 1.0 and f.dtype == torch.float64 and f.numel() == 32
    assert f[0] == 1.0
    # a ratio of 10000^(-2/64) from pair to pair: 2^-53 relative per power,
    # so 4 of them bound a quotient
    assert torch.allclose(f[1:] / f[:-1], torch.full((31,), 10000.0 ** (-2 / 64),
                                                     dtype=torch.float64), rtol=2 ** -50, atol=0)
    assert torch.equal(prompt.rotary_frequencies(64, scaling={"type": "linear", "factor": 4.0})[0],
                       f / 4.0)
    n, _ = prompt.rotary_frequencies(64, scaling={"type": "ntk", "factor": 4.0})
    # the base is chosen so that the slowest pair is stretched by the factor
    # and the fastest is kept
    assert n[0] == 1.0 and math.isclose(n[-1], f[-1] / 4.0, rel_tol=1e-13)


def test_yarn_frequencies_keep_fast_pairs_and_stretch_slow_ones():
    f, _ = prompt.rotary_frequencies(128)
    s = {"type": "yarn", "factor": 40.0, "original_max": 4096}
    y, m = prompt.rotary_frequencies(128, scaling=s)
    assert math.isclose(m, 0.1 * math.log(40.0) + 1.0)
    turns = 4096 * f / (2 * math.pi)
    # one pair around each limit is blended (the limits are rounded outwards)
    fast = int((turns > 32.0).sum())
    slow = int((turns > 1.0).sum())
    assert torch.equal(y[:fast - 1], f[:fast - 1])
    assert torch.allclose(y[slow + 1:], f[slow + 1:] / 40.0, rtol=1e-14, atol=0)
    assert (y[1:] < y[:-1]).all() and (y <= f).all() and (y >= f / 40.0 * (1 - 1e-14)).all()
    assert prompt.rotary_frequencies(128, scaling={**s, "attention_factor": 1.0})[1] == 1.0


def test_llama3_frequencies_split_by_wavelength():
    f, _ = prompt.rotary_frequencies(128, base=500000.0)
    s = {"type": "llama3", "factor": 8.0, "original_max": 8192, "low_freq_factor": 1.0,
         "high_freq_factor": 4.0}
    y, m = prompt.rotary_frequencies(128, base=500000.0, scaling=s)
    wave = 2 * math.pi / f
    assert m == 1.0
    assert torch.equal(y[wave < 8192 / 4], f[wave < 8192 / 4])
    assert torch.equal(y[wave > 8192], f[wave > 8192] / 8.0)
    mid = (wave > 8192 / 4) & (wave < 8192)
    assert mid.any() and (y[mid] < f[mid]).all() and (y[mid] > f[mid] / 8.0).all()


@pytest.mark.parametrize("args", [dict(rotary_dim=63), dict(rotary_dim=0),
                                  dict(rotary_dim=64, base=0.0),
                                  dict(rotary_dim=64, scaling={"type": "other", "factor": 2.0}),
                                  dict(rotary_dim=64, scaling={"type": "linear", "factor": 0.0}),
                                  dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2.0}),
                                  dict(rotary_dim=64, scaling={
                                      "type": "llama3", "factor": 8.0, "original_max": 8192,
                                      "low_freq_factor": 4.0, "high_freq_factor": 4.0})])
def test_rotary_refuses_bad_parameters(args):
    with pytest.raises(ValueError):
        prompt.rotary_frequencies(**args)


def test_plan_oracle_is_a_block_allocator():
    """Requests fed token by token to an allocator that opens a block whenever
    the last one is full get the oracle's slots."""
    g = torch.Generator().manual_seed(3)
    for bs in (1, 4, 64):
        context = torch.randint(0, 40, (6,), generator=g).tolist()
        new = torch.randint(0, 20, (6,), generator=g).tolist()
        ids = torch.randperm(400, generator=g).tolist()
        width = max(-(-(c + n) // bs) for c, n in zip(context, new)) + 1
        table, at = [], 0
        for c in context:
            h = -(-c // bs)
            table.append(ids[at:at + h] + [-1] * (width - h))
            at += h
        ring = ids[at:]
        ring = ring[7:] + ring[:7]
        head = len(ring) - 7
        got = oprompt.plan(context, new, table, ring, head, head + len(ring), bs, sum(new) + 3,
                           sum(new) + sum(context))
        free = (ring[head:] + ring[:head])
        slots, kv = [], []
        for c, n, row in zip(context, new, table):
            row = [b for b in row if b >= 0]
            for p in range(c + n):
                if p // bs == len(row):
                    row.append(free.pop(0))
                kv.append(row[p // bs] * bs + p % bs)
            slots += kv[len(kv) - n:] if n else []
        assert got[3] == slots + [-1] * 3 and got[4] == kv and not got[7]
        assert got[6] == head + len(ring) - len(free)


_THREE = torch.tensor([0, 8, 8])


def _plan_args(B=2, width=4):
    return dict(context_lens=torch.zeros(B, dtype=torch.int32),
                new_lens=torch.ones(B, dtype=torch.int32),
                block_table=torch.zeros(B, width, dtype=torch.int32),
                free_blocks=torch.arange(8, dtype=torch.int32),
                free_range=torch.tensor([0, 8]), block_size=16, num_tokens=2)


@pytest.mark.parametrize("change", [
    dict(new_lens=torch.ones(3, dtype=torch.int32)), dict(new_lens=torch.ones(2)),
    dict(context_lens=torch.zeros(2, 1, dtype=torch.int32)),
    dict(block_table=torch.zeros(3, 4, dtype=torch.int32)),
    dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()),
    dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)),
    dict(free_range=torch.tensor([0, 8], dtype=torch.int32)),
    dict(free_blocks=torch.zeros(16, dtype=torch.int32)[::2]), dict(num_tokens=-1),
    dict(free_range_out=torch.zeros(3, dtype=torch.int64)),
    dict(free_range=_THREE[:2], free_range_out=_THREE[1:]),
    dict(free_blocks=None), dict(free_range=None),
    dict(free_blocks=None, free_range=None, free_range_out=torch.tensor([0, 8])),
    dict(free_blocks=None, free_range=None),   # (CPU tensors)
    dict()])   # (CPU tensors)
def test_plan_refuses(change):
    with pytest.raises(ValueError):
        prompt.plan_kv_blocks(**{**_plan_args(), **change})


def _qkv(heads=4, kv_heads=2, dim=128, v_dim=128, own=None, T=8, dtype=torch.bfloat16):
    return dict(q=torch.zeros(T, heads, dim, dtype=dtype),
                k=torch.zeros(T, kv_heads, dim if own is None else own, dtype=dtype),
                v=torch.zeros(T, kv_heads, v_dim, dtype=dtype),
                cu_q=torch.tensor([0, T], dtype=torch.int32),
                cu_k=torch.tensor([0, T], dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(8, 4, 128)), dict(k=torch.zeros(8, 2, 128, dtype=torch.float16)),
    dict(v=torch.zeros(7, 2, 128, dtype=torch.bfloat16)),
    dict(k=torch.zeros(8, 3, 128, dtype=torch.bfloat16),
         v=torch.zeros(8, 3, 128, dtype=torch.bfloat16)),
    dict(k=torch.zeros(8, 2, 64, dtype=torch.bfloat16)),
    dict(k_shared=torch.zeros(8, 64, dtype=torch.bfloat16)),
    dict(k_shared=torch.zeros(7, 0, dtype=torch.bfloat16)),
    dict(cu_k=torch.tensor([0, 4, 8], dtype=torch.int32)),
    dict(cu_q=torch.tensor([0, 8])), dict(out=torch.zeros(8, 4, 64, dtype=torch.bfloat16)),
    dict(out=torch.zeros(8, 4, 128)),
    dict(out=torch.zeros(8, 4, 256, dtype=torch.bfloat16)[..., ::2]),
    dict()])   # (CPU tensors)
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        prompt.prompt_attention(**{**_qkv(), **change})


def test_attention_refuses_an_output_over_an_input():
    a = _qkv(heads=2)
    with pytest.raises(ValueError, match="overlaps"):
        prompt.prompt_attention(**a, out=a["q"])


def test_operators_without_a_backward_pass_refuse_gradients():
    a = _qkv()
    a["k"].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        prompt.prompt_attention(**a)
    with pytest.raises(ValueError, match="backward"):
        prompt.Rotary(64, device="cpu")(torch.arange(8), a["v"].clone().requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        prompt.prompt_attention(**a)


def test_rotary_refuses():
    r = prompt.Rotary(64, device="cpu")
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    pos = torch.arange(4)
    for bad in (dict(positions=pos.int(), q=x), dict(positions=pos, q=x.double()),
                dict(positions=pos[:3], q=x), dict(positions=pos, q=x[0]),
                dict(positions=pos, q=x, q_offset=65), dict(positions=pos, q=x, q_offset=-1),
                dict(positions=pos, q=x, k=x.float()), dict(positions=pos, q=x, out_k=x),
                dict(positions=pos, q=x[:, :, :32]),
                dict(positions=pos, q=x, out_q=torch.zeros(4, 2, 64, dtype=torch.bfloat16)),
                dict(positions=pos, q=x[:, :1], out_q=x[:, :1].expand(4, 1, 128).flip(0)[:3]),
                dict(positions=pos, q=x, k=x, out_k=torch.zeros(1, 2, 128, dtype=torch.bfloat16)
                     .expand(4, 2, 128)),
                dict(positions=pos, q=x)):   # (CPU tensors)
        with pytest.raises(ValueError):
            r(**bad)
    # an output over part of its input, and a tensor that cannot be rotated in
    # place
    buf = torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps"):
        r(pos, buf[:4], out_q=buf[1:])
    wide = torch.zeros(4, 2, 256, dtype=torch.bfloat16)[..., ::2]
    with pytest.raises(ValueError, match="in place"):
        r(pos, wide, out_q=wide)


def test_c_entries_refuse_without_a_gpu():
    L = _lib.lib()
    BAD, UNS, OK = _lib.SL_ERR_INVALID, _lib.SL_ERR_UNSUPPORTED, _lib.SL_OK

    def plan(B=4, bs=16, ld=8, width=8, n=8, T=4, Tk=0):
        return L.sl_plan_kv_blocks(None, None, B, bs, None, ld, width, None, n, None, None, T, Tk,
                                   None, None, None, None, None, None, None)

    assert plan() == BAD and plan(B=0) == BAD and plan(bs=0) == BAD and plan(ld=7) == BAD
    assert plan(width=0) == BAD and plan(n=0) == BAD and plan(T=-1) == BAD and plan(Tk=4) == BAD
    assert plan(B=8193) == UNS

    def paged(blocks=8, bs=64, ld=4, width=4, max_len=256, rank=512):
        return L.sl_mla_decode_paged(None, 16 * 192 + rank + 64, None, 1e-6, None, None, None,
                                     None, None, blocks, bs, None, ld, width, 8, 16, 128, 64, rank,
                                     128, max_len, 0.07, None, None)

    assert paged() == BAD and paged(blocks=0) == BAD and paged(ld=3) == BAD
    assert paged(width=0) == BAD and paged(max_len=257) == BAD
    assert paged(bs=48, max_len=192) == UNS

    def rot(T=4, rot=64, inter=1, dtype=0, heads=2, dim=128, offset=0, stride=128, x=16):
        p = _lib.RotaryPart(x, x, heads * stride, stride, heads * stride, stride, heads, dim,
                            offset)
        return L.sl_rotary(None, None, T, rot, inter, 1.0, dtype, ctypes.byref(p), None, None)

    assert rot() == BAD and rot(T=0) == OK and rot(T=-1) == BAD and rot(rot=63) == BAD
    assert rot(dtype=3) == BAD and rot(heads=0) == BAD and rot(offset=65) == BAD
    assert rot(dim=32) == BAD and rot(x=None) == BAD
    assert rot(rot=1024, dim=2048) == UNS and rot(dim=8192) == UNS

    def att(**kw):
        a = _lib.AttentionArgs()
        for n in ("q", "k", "v", "out", "cu_q", "cu_k"):
            setattr(a, n, 256)
        for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "out_token",
                  "out_head"):
            setattr(a, n, 128)
        a.Tq, a.Tk, a.B, a.heads, a.kv_heads, a.dim, a.v_dim = 4, 4, 1, 2, 2, 128, 128
        a.scale = 1.0
        ws, n = 256, 1 << 30
        for key, val in kw.items():
            if key == "ws":
                ws = val
            elif key == "n":
                n = val
            else:
                setattr(a, key, val)
        return L.sl_prompt_attention(ctypes.byref(a), ws, n, None)

    assert L.sl_prompt_attention(None, 256, 256, None) == BAD
    assert att(B=0) == BAD and att(Tq=-1) == BAD and att(heads=3) == BAD and att(scale=0.0) == BAD
    assert att(scale=float("nan")) == BAD and att(scale=float("inf")) == BAD
    assert att(dim=96) == UNS and att(v_dim=64) == UNS and att(dtype=2) == UNS
    assert att(shared_dim=64) == UNS and att(dim=192, shared_dim=32) == UNS
    assert att(heads=258, kv_heads=2) == UNS and att(Tk=1 << 31) == UNS
    assert att(Tq=0) == OK
    assert att(q=None) == BAD and att(k=None) == BAD and att(cu_k=None) == BAD
    assert att(ws=None) == BAD and att(n=0) == BAD
    assert att(q=264) == BAD and att(k_token=132) == BAD and att(dim=192, shared_dim=64) == BAD
    assert L.sl_prompt_attention_workspace_bytes(0, 1, 1, 1, 1, 64) == 0
    assert L.sl_prompt_attention_workspace_bytes(1, 1, 1, 1, 1, 64) >= 256


def test_prefill_refuses_expert_parallel_layers():
    from sluice_b200.ep import EPDecodeStack
    from sluice_b200.harness import OffloadedDecoder
    d = OffloadedDecoder.__new__(OffloadedDecoder)
    d.stack = EPDecodeStack.__new__(EPDecodeStack)
    with pytest.raises(ValueError, match="EPDecodeStack"):
        d.prefill(torch.zeros(2, dtype=torch.long), [1, 1])


def test_rotary_refuses_outputs_over_the_other_tensor():
    r = prompt.Rotary(64, device="cpu")
    pos = torch.arange(4)
    fused = torch.zeros(4, 5 * 64, dtype=torch.bfloat16)
    q, k = fused[:, :192].view(4, 3, 64), fused[:, 192:].view(4, 2, 64)
    for bad in (dict(q=k, k=k, out_q=k, out_k=k),             # rotated twice
                dict(q=torch.zeros_like(q), k=k, out_q=fused[:, 64:256].view(4, 3, 64)),
                dict(q=q, k=k, out_k=fused[:, :128].view(4, 2, 64)),
                dict(q=q, k=q, out_q=fused.new_empty(4, 3, 64),
                     out_k=torch.as_strided(q, (4, 3, 64), (320, 32, 1)))):
        with pytest.raises(ValueError, match="overlaps|share"):
            r(pos, **bad)
    # columns, or heads, of one buffer do not meet: only the device is refused
    rows = torch.zeros(4, 3, 128, dtype=torch.bfloat16)
    for a, b in ((q, k), (q[:1], k[:1]), (rows[..., :64], rows[..., 64:]),
                 (rows[:1, :, 64:], rows[:1, :, :64])):
        with pytest.raises(ValueError, match="CUDA"):
            r(pos[:a.shape[0]], a, b, out_q=a, out_k=b)


def test_outputs_whose_rows_share_memory_are_refused():
    buf = torch.zeros(8 * 4 * 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share"):
        prompt.prompt_attention(**_qkv(), out=buf.as_strided((8, 4, 128), (256, 64, 1)))
    with pytest.raises(ValueError, match="share"):
        prompt.prompt_attention(**_qkv(), out=buf.as_strided((8, 4, 128), (128, 128, 1)))
    with pytest.raises(ValueError, match="backward"):
        prompt.prompt_attention(**_qkv(), out=torch.zeros(8, 4, 128, dtype=torch.bfloat16,
                                                          requires_grad=True))
    with pytest.raises(ValueError, match="share"):
        x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
        prompt.Rotary(64, device="cpu")(torch.arange(4), x,
                                        out_q=buf.as_strided((4, 2, 64), (64, 64, 1)))


def test_attention_of_columns_that_no_copy_aligns_ends_in_a_refusal():
    with pytest.raises(ValueError, match="CUDA"):
        prompt.prompt_attention(**_qkv(dim=67, v_dim=67))


def test_decoder_angles_of_far_positions():
    """The decode step's table of angles has the phase of the prompt pass's
    64-bit ones, as far as the cache reaches."""
    from dataclasses import replace

    from sluice_b200.harness import V2_LITE_DECODER, DecoderHarness
    cfg = replace(V2_LITE_DECODER, num_layers=1, vocab=16)
    n = 70001
    h = DecoderHarness(cfg, None, batch=1, max_len=n, device="cpu")
    freqs, _ = prompt.rotary_frequencies(cfg.qk_rope, cfg.rope_theta)
    for p in (0, 1, 4095, 65537, n - 1):
        angle = p * freqs
        want = torch.stack([angle.cos(), angle.sin()], dim=-1)
        # one rounding to 32 bits of values up to one
        assert (h.rope_cs[p].double() - want).abs().max() <= 2.0 ** -24
        assert torch.equal(torch.view_as_real(h.freqs[p]), h.rope_cs[p])


def test_rotary_offsets_count_by_value():
    """An offset that is a tensor, changed between two calls."""
    r, x, at = prompt.Rotary(64, device="cpu"), torch.zeros(4, 2, 128), torch.tensor(64)
    with pytest.raises(ValueError, match="CUDA"):
        r(torch.arange(4), x, q_offset=at)
    at.fill_(65)
    with pytest.raises(ValueError, match="columns"):
        r(torch.arange(4), x, q_offset=at)
    with pytest.raises(TypeError):
        r(torch.arange(4), x, q_offset=1.5)


def test_sizes_past_32_bits_are_refused():
    """Not taken modulo 2^32, which is what a C int would keep of them."""
    meta = dict(device="meta")
    big = 2 ** 32 + 16
    for change in (dict(block_size=big), dict(block_table=torch.empty(2, big, dtype=torch.int32, **meta)),
                   dict(free_blocks=torch.empty(big, dtype=torch.int32, **meta))):
        with pytest.raises(ValueError, match="32-bit"):
            prompt.plan_kv_blocks(**{**_plan_args(), **change})
    r = prompt.Rotary(2, device="cpu")
    for T in (big, 2 ** 31 - 1):
        x = torch.empty(T, 1, 2, dtype=torch.bfloat16, **meta)
        with pytest.raises(ValueError, match="rows"):
            r(torch.empty(T, dtype=torch.long, **meta), x)
    cu = torch.empty(big, dtype=torch.int32, **meta)
    with pytest.raises(ValueError, match="sequences"):
        prompt.prompt_attention(**{**_qkv(), "cu_q": cu, "cu_k": cu})
    p = _lib.RotaryPart(16, 16, 2, 2, 2, 2, 1, 2, 0)
    assert _lib.lib().sl_rotary(256, 256, 2 ** 31 - 1, 2, 1, 1.0, 0, ctypes.byref(p), None, None) == \
        _lib.SL_ERR_UNSUPPORTED


def test_restore_of_a_state_without_blocks():
    """A state that holds caches, positions and ids only, as a contiguous cache
    needs them."""
    from dataclasses import replace

    from sluice_b200.harness import V2_LITE_DECODER, DecoderHarness, OffloadedDecoder
    d = OffloadedDecoder.__new__(OffloadedDecoder)
    d.model = DecoderHarness(replace(V2_LITE_DECODER, num_layers=1, vocab=16), None, batch=2,
                             max_len=8, device="cpu")
    d._ids = torch.tensor([3, 4])
    saved = {n: t for n, t in d.save().items() if n != "blocks"}
    d.model.pos.add_(5)
    d._ids.zero_()
    d.restore(saved)
    assert d.model.pos.tolist() == [0, 0] and d._ids.tolist() == [3, 4]
