"""The prompt pass's operators against their 64-bit and integer oracles."""

import math
import threading

import pytest
import torch

from oracle import prompt as oprompt
from sluice_b200 import _lib, ops, prompt

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------ block planner
def _plan_case(context, new, bs, extra=3, width_extra=1, seed=0, head=5):
    g = torch.Generator().manual_seed(seed)
    held = [-(-c // bs) for c in context]
    need = [-(-(c + n) // bs) for c, n in zip(context, new)]
    width = max(max(need), 1) + width_extra
    blocks = max(sum(need) + extra, sum(held) + 1)
    ids = torch.randperm(blocks, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    free = ids[at:]
    ring = [-7] * blocks
    for i, b in enumerate(free):
        ring[(head + i) % blocks] = b
    return table, ring, head, head + len(free)


def _run_plan(context, new, table, ring, head, tail, bs, T, Tk, in_place=True):
    i32 = dict(dtype=torch.int32, device="cuda")
    tab = torch.tensor(table, **i32)
    rng = torch.tensor([head, tail], device="cuda")
    out = rng if in_place else torch.full((2,), -1, dtype=torch.int64, device="cuda")
    p = prompt.plan_kv_blocks(torch.tensor(context, **i32), torch.tensor(new, **i32), tab,
                              torch.tensor(ring, **i32), rng, bs, T, num_kv_tokens=Tk,
                              free_range_out=None if in_place else out)
    return p, tab, out


def _check_plan(context, new, bs, T=None, kv=True, in_place=True, **case):
    table, ring, head, tail = _plan_case(context, new, bs, **case)
    T = sum(new) if T is None else T
    Tk = sum(new) + sum(context) if kv else 0
    p, tab, out = _run_plan(context, new, table, ring, head, tail, bs, T, Tk, in_place)
    ref = oprompt.plan(context, new, table, ring, head, tail, bs, T, Tk)
    assert p.cu_new.tolist() == ref[0] and p.cu_total.tolist() == ref[1]
    assert p.positions.tolist() == ref[2]
    assert p.slots.tolist() == ref[3]
    assert (p.kv_slots.tolist() if Tk else []) == ref[4]
    assert tab.tolist() == ref[5]
    assert out.tolist() == [ref[6], tail]
    assert p.status.tolist()[1] == ref[6] - head
    return p, ref


@pytest.mark.parametrize("bs", [1, 16, 48, 64, 128])
@pytest.mark.parametrize("context,new", [
    ([0], [1]), ([0], [0]), ([15, 16, 17], [1, 1, 1]), ([0, 0, 0], [137, 1, 255]),
    ([63, 64, 65, 0, 1], [1, 0, 64, 63, 200]), ([4096], [1])])
def test_plan_matches_the_oracle(bs, context, new):
    p, ref = _check_plan(context, new, bs)
    assert not ref[7]
    p.check()


@pytest.mark.parametrize("B", [31, 1024, 1025, 3001])
@pytest.mark.parametrize("in_place", [True, False])
def test_plan_of_many_requests(B, in_place):
    g = torch.Generator().manual_seed(B)
    context = torch.randint(0, 300, (B,), generator=g).tolist()
    new = torch.randint(0, 40, (B,), generator=g).tolist()
    p, _ = _check_plan(context, new, 16, in_place=in_place)   # several CTAs
    p.check()


@pytest.mark.parametrize("bs", [1, 4, 16])
def test_plan_of_requests_that_take_few_and_many_blocks(bs):
    """Runs of none to many blocks side by side, in one CTA and in several."""
    g = torch.Generator().manual_seed(bs)
    for B, most in ((40, 9), (300, 9), (600, 40)):
        new = torch.randint(0, most, (B,), generator=g).tolist()
        context = torch.randint(0, 30, (B,), generator=g).tolist()
        _check_plan(context, new, bs, seed=B)
        _check_plan(context, new, bs, seed=B, in_place=False)


def test_plan_of_long_requests_and_rows_behind_the_last():
    _check_plan([0, 100000], [70000, 1], 64, T=70500)[0].check()


def test_plan_without_blocks_left():
    """Requests that the ring or the table row cannot hold take nothing, the
    rest are served, and the status says so."""
    for in_place in (True, False):
        p, ref = _check_plan([0, 10, 15, 3, 16], [33, 6, 2, 2, 40], 16, extra=-3,
                             in_place=in_place)
        assert ref[7] and p.status[0].item() == _lib.KV_PLAN_NO_BLOCKS
        with pytest.raises(prompt.KvPlanError, match="free cache blocks"):
            p.check()
    p, ref = _check_plan([0, 10, 40], [90, 6, 20], 16, width_extra=-2)
    assert ref[7] and p.status[0].item() == _lib.KV_PLAN_NO_BLOCKS


def test_plan_of_complete_tables_and_large_block_ids():
    """Without a ring every block is in the table, and none is taken; slots pass
    32 bits."""
    i32 = dict(dtype=torch.int32, device="cuda")
    ids = [[2 ** 30 + 5, 7, -1], [2 ** 31 - 1, 2 ** 27, 3]]
    table = torch.tensor(ids, **i32)
    for bs in (64, 100):
        context, new = [10, 0], [bs + 20, 2 * bs + 1]
        p = prompt.plan_kv_blocks(torch.tensor(context, **i32), torch.tensor(new, **i32), table, None,
                                  None, bs, sum(new), num_kv_tokens=sum(new) + sum(context))
        p.check()
        want = [ids[r][q // bs] * bs + q % bs for r in (0, 1)
                for q in range(context[r], context[r] + new[r])]
        assert p.slots.tolist() == want and table.tolist() == ids
        assert p.kv_slots.tolist() == [ids[0][q // bs] * bs + q % bs
                                       for q in range(context[0] + new[0])] + want[new[0]:]
        assert p.status.tolist() == [0, 0]
    # a row that is too narrow, and an entry that is no block
    p = prompt.plan_kv_blocks(torch.tensor([0, 0], **i32), torch.tensor([193, 5], **i32), table, None,
                              None, 64, 198)
    assert p.status[0].item() == _lib.KV_PLAN_NO_BLOCKS
    assert p.slots[:193].eq(-1).all() and p.slots[193:].ge(0).all()
    p = prompt.plan_kv_blocks(torch.tensor([0, 0], **i32), torch.tensor([140, 5], **i32), table, None,
                              None, 64, 145)
    assert p.slots[128:140].eq(-1).all() and p.slots[:128].ge(0).all()
    # the same from a ring of such ids
    free = torch.tensor([2 ** 31 - 2, 2 ** 28], **i32)
    p = prompt.plan_kv_blocks(torch.tensor([0], **i32), torch.tensor([100], **i32),
                              torch.full((1, 2), -1, **i32), free,
                              torch.tensor([1, 3], device="cuda"), 64, 100)
    assert p.slots.tolist() == [2 ** 28 * 64 + q for q in range(64)] + \
        [(2 ** 31 - 2) * 64 + q for q in range(36)]


def test_plan_survives_bad_lengths_and_ranges():
    """Lengths below zero, more tokens than the outputs hold, contexts past the
    table row, a range larger than its ring: flagged, nothing out of place."""
    table, ring, head, tail = _plan_case([0, 0], [20, 20], 16)
    guard = 64
    p, _, _ = _run_plan([-5, 0], [20, -1], table, ring, head, tail, 16, 20, 0)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT and p.cu_new.tolist() == [0, 20, 20]
    p, _, _ = _run_plan([0, 0], [20, 20], table, ring, head, tail, 16, 30, 30)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT
    assert p.cu_new.tolist() == [0, 20, 30] and p.cu_total.tolist() == [0, 20, 30]
    width = len(table[0])
    p, _, _ = _run_plan([width * 16 + 1, 0], [1, 20], table, ring, head, tail, 16, 21, 0)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT and p.slots[0].item() == -1 and p.slots[1].item() >= 0
    p, _, out = _run_plan([0, 0], [20, 20], table, ring, 0, len(ring) + 1, 16, 40, 0)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT and p.slots.eq(-1).all() and out.tolist() == [0, len(ring) + 1]
    p, _, _ = _run_plan([2 ** 31 - 1, 2 ** 31 - 1], [2 ** 31 - 1, 5], table, ring, head, tail, 16,
                        guard, guard)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT and p.slots.eq(-1).all() and p.cu_total.max().item() <= guard


def test_plan_replays_in_a_graph_and_moves_its_range():
    """Captured with the range in place, every replay takes the next blocks."""
    i32 = dict(dtype=torch.int32, device="cuda")
    B, bs, N = 3, 16, 32
    context, new = torch.zeros(B, **i32), torch.tensor([16, 16, 16], **i32)
    table = torch.full((B, 8), -1, **i32)
    free, rng = torch.arange(N, **i32), torch.tensor([0, N], device="cuda")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    prompt.plan_kv_blocks(context, new, table.clone(), free, rng.clone(), bs, 48)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        p = prompt.plan_kv_blocks(context, new, table, free, rng, bs, 48)
        context += new
    for step in range(4):
        g.replay()
        torch.cuda.synchronize()
        assert rng.tolist() == [3 * (step + 1), N]
        assert table[:, step].tolist() == [3 * step, 3 * step + 1, 3 * step + 2]
        assert p.slots.tolist() == list(range(48 * step, 48 * (step + 1)))
        assert p.positions.tolist() == 3 * list(range(16 * step, 16 * (step + 1)))


# ------------------------------------------------------------------- rotary
def _rotary_close(got, ref, x, dtype, factor):
    """One rounding to the type, on values whose products and sine and cosine
    carry 32-bit errors: 8 of its half steps on the pair's magnitude bound the
    angle's rounding (pi times half a step), the sine's, and the products'."""
    tol = U[dtype] * ref.abs() + factor * 8 * 2.0 ** -24 * 2 * x.double().abs().amax()
    tol += 2.0 ** -25 if dtype == torch.float16 else 1e-38
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (err - tol).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,heads,kv_heads,dim,rot,offset", [
    (1, 1, 1, 64, 64, 0), (8, 16, 1, 192, 64, 128), (37, 5, 2, 80, 20, 60), (130, 3, 3, 96, 48, 8),
    (5, 40, 8, 128, 2, 0), (3, 2, 1, 514, 512, 2), (300, 7, 7, 66, 22, 30)])
def test_rotary_matches_64_bits(dtype, interleaved, T, heads, kv_heads, dim, rot, offset):
    g = _gen(T + dim)
    q = torch.randn(T, heads, dim, device="cuda", generator=g).to(dtype)
    k = torch.randn(T, kv_heads, dim, device="cuda", generator=g).to(dtype)
    pos = torch.randint(0, 1 << 21, (T,), device="cuda", generator=g)
    pos[0] = 0
    scaling = {"type": "yarn", "factor": 40.0, "original_max": 4096} if rot > 2 else None
    r = prompt.Rotary(rot, scaling=scaling, interleaved=interleaved)
    freqs, factor = prompt.rotary_frequencies(rot, scaling=scaling)
    yq, yk = r(pos, q, k, q_offset=offset, k_offset=0)
    for y, x, off in ((yq, q, offset), (yk, k, 0)):
        ref = oprompt.rotary(x, pos, freqs, factor, off, interleaved)
        _rotary_close(y, ref, x, dtype, factor)
        rest = [c for c in range(dim) if not off <= c < off + rot]
        assert torch.equal(y[..., rest], x[..., rest])
    # in place, on strided views of one buffer, the same bits; the columns
    # around them untouched
    buf = torch.full((T, heads + kv_heads + 1, dim + 8), 7.0, dtype=dtype, device="cuda")
    vq, vk = buf[:, :heads, :dim], buf[:, heads:heads + kv_heads, :dim]
    vq.copy_(q)
    vk.copy_(k)
    oq, ok = r(pos, vq, vk, q_offset=offset, out_q=vq, out_k=vk)
    assert oq is vq and ok is vk
    assert torch.equal(vq, yq) and torch.equal(vk, yk)
    assert buf[..., dim:].eq(7.0).all() and buf[:, -1].eq(7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,heads,kv_heads,dim,rot,offset", [
    (7, 3, 2, 112, 32, 16), (5, 2, 1, 72, 16, 8), (9, 1, 1, 48, 32, 0), (9, 1, 1, 80, 32, 32),
    (300, 4, 1, 160, 32, 112), (3, 2, 2, 9, 2, 3)])
def test_rotary_copies_an_odd_number_of_vectors(dtype, T, heads, kv_heads, dim, rot, offset):
    """Columns that are not rotated go in twos of the widest vectors: odd
    numbers of them, and twos that lie on both sides of the rotated ones."""
    for interleaved in (True, False):
        test_rotary_matches_64_bits(dtype, interleaved, T, heads, kv_heads, dim, rot, offset)


@pytest.mark.parametrize("rot", [512, 256])
def test_rotary_of_many_rows_of_wide_heads(rot):
    T = 40001
    x = torch.randn(T, 1, rot, device="cuda", generator=_gen(rot)).bfloat16()
    pos = torch.arange(T, device="cuda")
    freqs, factor = prompt.rotary_frequencies(rot)
    for interleaved in (True, False):
        y = prompt.Rotary(rot, interleaved=interleaved)(pos, x)
        _rotary_close(y, oprompt.rotary(x, pos, freqs, factor, 0, interleaved), x, x.dtype, factor)


def test_rotary_far_positions_keep_their_phase():
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 + 12345, 10 ** 12], device="cuda")
    x = torch.zeros(5, 1, 64, device="cuda")
    x[..., 0::2] = 1.0
    freqs, _ = prompt.rotary_frequencies(64)
    y = prompt.Rotary(64)(pos, x)
    # at 1e12 the 64-bit angle itself is off by 1e12 * 2^-52 of its turns
    ref = oprompt.rotary(x, pos, freqs, 1.0, 0, True)
    tol = 1e-6 + pos.double()[:, None, None] * 2.0 ** -50
    assert ((y.double() - ref).abs() <= tol).all()


def test_rotary_of_rows_past_32_bit_offsets():
    big = torch.empty(3, 1 << 30, device="cuda", dtype=torch.bfloat16)
    x = big[:, -256:].view(3, 2, 128)
    x.copy_(torch.randn(3, 2, 128, device="cuda", generator=_gen(2)))
    pos, r = torch.tensor([5, 77, 12345], device="cuda"), prompt.Rotary(128)
    want = r(pos, x.contiguous())
    assert torch.equal(r(pos, x), want)
    r(pos, x, out_q=x)
    assert torch.equal(x, want)


def test_rotary_leaves_padding_rows_and_other_layouts():
    """Rows at negative positions keep their bits, NaN among them; unaligned
    and transposed inputs are read as they are."""
    g = _gen(1)
    for dtype in (torch.bfloat16, torch.float32):
        for interleaved in (True, False):
            r = prompt.Rotary(32, interleaved=interleaved)
            x = torch.randn(6, 2, 64, device="cuda", generator=g).to(dtype)
            pos = torch.tensor([0, 3, -1, 9, -5, -1], device="cuda")
            x[2, 0, 3] = float("nan")
            x[4] = float("inf")
            y = r(pos, x)
            for i in (2, 4, 5):
                assert torch.equal(y[i].view(torch.uint8), x[i].view(torch.uint8))
            z = x.clone()
            r(pos, z, out_q=z)
            assert torch.equal(z.view(torch.uint8), y.view(torch.uint8))
            base = torch.randn(2, 6, 67, device="cuda", generator=g).to(dtype)
            odd = base.transpose(0, 1)[..., 3:]
            keep = odd.clone()
            assert torch.equal(r(pos, odd), r(pos, odd.contiguous()))
            assert torch.equal(odd, keep)
            r(pos, odd, out_q=odd)   # in place, whatever the alignment
            assert torch.equal(odd, r(pos, keep))
    empty = torch.empty(0, 2, 64, device="cuda")
    assert r(torch.empty(0, dtype=torch.long, device="cuda"), empty).shape == empty.shape


# ---------------------------------------------------------------- attention
def _bounds(o, mag, dtype, k_len, vmax):
    """|error| of an output o of weights p and values v, mag = sum p |v|: half
    a step on o; half a step on each weight as it is fed to the second product,
    hence on mag; and 2^-11 on mag for the 32-bit scores (their largest, of a
    few hundred, times 2^-24 times the length of a dot product), exponentials
    and sums. fp16 weights below 2^-14 are off by half of 2^-24 absolute, on
    k_len keys at most, against a sum of weights of at least one."""
    t = U[dtype] * o.abs() + (U[dtype] + 2.0 ** -11) * mag
    if dtype == torch.float16:
        t = t + 2.0 ** -25 * k_len * vmax + 2.0 ** -25
    return t + 1e-30


def _inputs(q_lens, k_lens, heads, kv_heads, dim, v_dim, shared, dtype, seed, tail=0, spread=1.0):
    g = _gen(seed)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    tq, tk = sum(q_lens) + tail, sum(k_lens) + tail
    q = (spread * rand(tq, heads, dim)).to(dtype)
    k = rand(tk, kv_heads, dim - shared).to(dtype)
    v = rand(tk, kv_heads, v_dim).to(dtype)
    ks = rand(tk, shared).to(dtype) if shared else None

    def cu(lens):
        return torch.tensor([0] + list(lens), device="cuda").cumsum(0).int()

    return q, k, v, ks, cu(q_lens), cu(k_lens)


def _check_attention(q_lens, k_lens, heads, kv_heads, dim, v_dim, shared=0, dtype=torch.bfloat16,
                     seed=0, spread=1.0, scale=None):
    q, k, v, ks, cu_q, cu_k = _inputs(q_lens, k_lens, heads, kv_heads, dim, v_dim, shared, dtype,
                                      seed, spread=spread)
    out = prompt.prompt_attention(q, k, v, cu_q, cu_k, k_shared=ks, scale=scale)
    assert ops.workspace_status(prompt.prompt_attention.last_workspace) == 0
    ref, mag = oprompt.attention(q, k, v, q_lens, k_lens,
                                 1 / math.sqrt(dim) if scale is None else scale, ks)
    err = (out.double() - ref).abs()
    vmax = v.abs().max().item() if v.numel() else 0.0
    tol = _bounds(ref, mag, dtype, max(k_lens), vmax)
    assert out.isfinite().all()
    assert (err <= tol).all(), ((err - tol).max().item(), (err / tol).max().item())
    return out


LAYOUTS = [(2, 2, 192, 128, 64), (2, 1, 192, 128, 0), (8, 1, 128, 128, 0), (3, 3, 128, 128, 0),
           (7, 1, 128, 128, 0), (4, 2, 64, 64, 0)]
LENGTHS = [([1], [1]), ([1], [200]), ([5], [3]), ([3], [0]), ([0, 7, 0], [3, 7, 0]),
           ([128], [128]), ([127, 129], [127, 129]), ([257], [300]), ([64, 1, 300], [700, 129, 300]),
           ([1, 1, 1, 1], [1, 128, 1000, 257])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("lens", LENGTHS)
def test_attention_matches_64_bits(dtype, layout, lens):
    heads, kv_heads, dim, v_dim, shared = layout
    _check_attention(*lens, heads, kv_heads, dim, v_dim, shared, dtype)


@pytest.mark.parametrize("layout", [(1, 1, 128, 128, 0), (2, 2, 192, 128, 64), (2, 1, 64, 64, 0)])
def test_attention_of_longer_prompts(layout):
    heads, kv_heads, dim, v_dim, shared = layout
    _check_attention([1100], [1100], heads, kv_heads, dim, v_dim, shared, seed=2)
    _check_attention([600, 150], [2000, 900], heads, kv_heads, dim, v_dim, shared, seed=3)


@pytest.mark.parametrize("heads,kv_heads", [(128, 1), (48, 1), (100, 2), (5, 1), (20, 4)])
def test_attention_group_sizes(heads, kv_heads):
    _check_attention([9, 1], [40, 300], heads, kv_heads, 64, 64, dtype=torch.float16)


@pytest.mark.parametrize("k_len", [9000, 40001])
def test_attention_of_a_single_token_over_a_long_cache(k_len):
    _check_attention([1], [k_len], 8, 2, 128, 128, seed=k_len)
    _check_attention([2, 1], [k_len, 30], 4, 1, 64, 64, dtype=torch.float16, seed=k_len)


def test_attention_of_sharp_flat_and_scaled_scores():
    """Scores of hundreds (one key takes all), all equal, and a given scale."""
    _check_attention([200], [333], 4, 2, 128, 128, spread=30.0)
    _check_attention([200], [333], 4, 2, 128, 128, spread=0.0)
    _check_attention([200], [333], 4, 2, 128, 128, dtype=torch.float16, scale=0.01)
    _check_attention([70], [555], 2, 2, 192, 128, 64, spread=30.0, dtype=torch.float16)


def test_attention_growing_scores_move_the_maximum():
    """Each key scores above all before it, by more and by less than the
    factor that a running maximum may lag behind."""
    for step in (0.02, 0.5, 3.0):
        T = 700
        q = torch.ones(T, 1, 128, device="cuda", dtype=torch.bfloat16)
        ramp = (torch.arange(T, device="cuda") * step / 128).bfloat16()
        k = ramp[:, None, None].expand(T, 1, 128).contiguous()
        v = torch.randn(T, 1, 128, device="cuda", generator=_gen(4)).bfloat16()
        cu = torch.tensor([0, T], device="cuda", dtype=torch.int32)
        for kk in (k, k.flip(0).contiguous()):
            out = prompt.prompt_attention(q, kk, v, cu, cu, scale=1.0)
            ref, mag = oprompt.attention(q, kk, v, [T], [T], 1.0)
            # scores reach T * step: 2^-24 of that, times the dot product's
            # length, on every weight
            tol = _bounds(ref, mag, torch.bfloat16, T, 5.0) + T * step * 2.0 ** -17 * mag
            assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("layout", [(4, 2, 128, 128, 0), (2, 2, 192, 128, 64)])
def test_attention_ignores_what_it_may_not_see(bad, layout):
    """Rows behind the last sequence and the next sequence's, and keys and
    values after a query, do not reach it."""
    heads, kv_heads, dim, v_dim, shared = layout
    q_lens, k_lens = [70, 150], [100, 201]
    q, k, v, ks, cu_q, cu_k = _inputs(q_lens, k_lens, heads, kv_heads, dim, v_dim, shared,
                                      torch.bfloat16, 5, tail=200)
    clean = prompt.prompt_attention(q, k, v, cu_q, cu_k, k_shared=ks)
    for t in (q, k, v, ks):
        if t is not None:
            t[-200:] = bad
    out = torch.full_like(clean, 3.0)
    got = prompt.prompt_attention(q, k, v, cu_q, cu_k, k_shared=ks, out=out)
    assert got is out and out[220:].eq(3.0).all()
    assert torch.equal(out[:220], clean[:220])
    # the second sequence spoilt from its 120th key on: its queries before
    # that one (query i sits at key i + 51), and the first sequence, as before
    for what in (k, v):
        kk, vv = k.clone(), v.clone()
        (kk if what is k else vv)[100 + 120:] = bad
        o = prompt.prompt_attention(q, kk, vv, cu_q, cu_k, k_shared=ks)
        assert torch.equal(o[:70 + 69], clean[:70 + 69])
        if what is v:
            assert not o[70 + 69:220].isfinite().any()
    # a spoilt value column spoils that column alone
    vv = v.clone()
    vv[100 + 120, 0, 5] = bad
    o = prompt.prompt_attention(q, k, vv, cu_q, cu_k, k_shared=ks)
    assert torch.equal(o[:70 + 69], clean[:70 + 69])
    per = heads // kv_heads
    assert not o[70 + 69:220, :per, 5].isfinite().any()
    rest = [c for c in range(v_dim) if c != 5]
    assert torch.equal(o[:220, :, rest], clean[:220, :, rest])
    assert torch.equal(o[:220, per:], clean[:220, per:])


def test_attention_of_spoilt_queries_and_visible_keys():
    """NaN in a query, or in a key that it sees, makes its own row NaN; a key
    at minus infinity takes no weight."""
    q, k, v, _, cu_q, cu_k = _inputs([150], [150], 2, 2, 64, 64, 0, torch.bfloat16, 6)
    clean = prompt.prompt_attention(q, k, v, cu_q, cu_k)
    q2 = q.clone()
    q2[40, 1, 3] = float("nan")
    o = prompt.prompt_attention(q2, k, v, cu_q, cu_k)
    assert o[40, 1].isnan().all()
    keep = torch.ones(150, 2, dtype=torch.bool)
    keep[40, 1] = False
    assert torch.equal(o[keep], clean[keep])
    for col in range(0, 64, 5):
        k2 = k.clone()
        k2[30, 0, col] = float("nan")
        o = prompt.prompt_attention(q, k2, v, cu_q, cu_k)
        assert o[30:, 0].isnan().all() and torch.equal(o[:30], clean[:30])
        assert torch.equal(o[:, 1], clean[:, 1])
    q3, k3 = q.abs() + 0.1, k.clone()
    k3[10, :, 0] = float("-inf")
    o = prompt.prompt_attention(q3, k3, v, cu_q, cu_k)
    v4, k4 = v.clone(), k3.clone()
    ref, mag = oprompt.attention(q3, k4, v4, [150], [150], 64 ** -0.5)
    live = torch.ones(150, dtype=torch.bool)
    live[10] = True
    assert ((o.double() - ref).abs() <= _bounds(ref, mag, torch.bfloat16, 150, 5.0))[live].all()


def test_attention_takes_strided_views():
    """Queries, keys and values as slices of one projection's output, an output
    inside a larger buffer: equal to contiguous inputs bit for bit."""
    T, g = 333, _gen(7)
    buf = torch.randn(T, 6 * 128 + 2 * 256 + 64, device="cuda", generator=g).bfloat16()
    q = buf[:, :768].view(T, 4, 192)
    kv = buf[:, 768:1280].view(T, 2, 256)
    k, v, ks = kv[..., :128], kv[..., 128:], buf[:, 1280:]
    cu = torch.tensor([0, 100, T], device="cuda", dtype=torch.int32)
    want = prompt.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu,
                                   k_shared=ks.contiguous())
    assert torch.equal(prompt.prompt_attention(q, k, v, cu, cu, k_shared=ks), want)
    big = torch.full((T, 5, 256), 2.0, device="cuda", dtype=torch.bfloat16)
    prompt.prompt_attention(q, k, v, cu, cu, k_shared=ks, out=big[:, 1:, 64:192])
    assert torch.equal(big[:, 1:, 64:192], want)
    assert big[:, 0].eq(2.0).all() and big[..., :64].eq(2.0).all() and big[..., 192:].eq(2.0).all()
    # layouts that the tile loads do not take are copied first
    qt = q.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    odd = torch.randn(T, 2, 129, device="cuda", generator=g).bfloat16()
    assert torch.equal(prompt.prompt_attention(qt, k, v, cu, cu, k_shared=ks), want)
    assert torch.equal(
        prompt.prompt_attention(q, k, odd[..., 1:], cu, cu, k_shared=ks),
        prompt.prompt_attention(q, k, odd[..., 1:].contiguous(), cu, cu, k_shared=ks))
    one = prompt.prompt_attention(q, k[:, :1].expand(T, 2, 128), v, cu, cu, k_shared=ks)
    assert one.isfinite().all()


def test_attention_survives_bad_offsets():
    """Offsets past the tensors, or running backwards, fault nothing and leave
    the rows around alone."""
    q, k, v, _, _, _ = _inputs([64], [64], 2, 2, 64, 64, 0, torch.bfloat16, 8)
    for cq, ck in (([0, 1000], [0, 64]), ([0, 64], [0, 5000]), ([0, 64], [60, 10]),
                   ([0, 40, 20, 64], [0, 64, 64, 64]), ([-50, 64], [-9, 64]),
                   ([0, 64], [2000000000, 2000000100])):
        big = torch.full((96, 2, 64), 5.0, device="cuda", dtype=torch.bfloat16)
        prompt.prompt_attention(q, k, v, torch.tensor(cq, device="cuda", dtype=torch.int32),
                                torch.tensor(ck, device="cuda", dtype=torch.int32),
                                out=big[16:80])
        torch.cuda.synchronize()
        assert big[:16].eq(5.0).all() and big[80:].eq(5.0).all()


def test_attention_over_a_cache_past_32_bit_offsets():
    """2.2 million keys of 8 heads: element offsets past 2^31."""
    Tk, g = 2_200_003, _gen(20)
    q = torch.randn(3, 16, 128, device="cuda", generator=g).bfloat16()
    k = torch.empty(Tk, 8, 128, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    v = torch.empty(Tk, 8, 128, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    lens = [5, Tk - 1005, 1000]
    cu_q = torch.tensor([0, 1, 2, 3], device="cuda", dtype=torch.int32)
    cu_k = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    out = prompt.prompt_attention(q, k, v, cu_q, cu_k)
    for b, h in ((1, 0), (1, 15), (2, 9)):
        kk = k[cu_k[b]:cu_k[b + 1], h // 2].double()
        vv = v[cu_k[b]:cu_k[b + 1], h // 2].double()
        p = torch.softmax(kk @ q[b, h].double() * 128 ** -0.5, dim=0)
        ref, mag = p @ vv, p @ vv.abs()
        # (sums of 17 000 tiles in 32 bits on top: 2^-24 each, half of them
        # rounding alike at most)
        tol = _bounds(ref, mag, torch.bfloat16, lens[b], 6.0) + 2.0 ** -11 * mag
        assert ((out[b, h].double() - ref).abs() <= tol).all()


def test_first_call_of_a_process_in_a_capture():
    """A process whose first calls are captured ones, replayed twice."""
    import os
    import subprocess
    import sys

    code = (
        "import torch\n"
        "from sluice_b200 import prompt\n"
        "cu = torch.tensor([0, 1], device='cuda', dtype=torch.int32)\n"
        "ck = torch.tensor([0, 3000], device='cuda', dtype=torch.int32)\n"
        "q = torch.randn(1, 8, 128, device='cuda').bfloat16()\n"
        "k = torch.randn(3000, 2, 128, device='cuda').bfloat16()\n"
        "pos = torch.tensor([7], device='cuda')\n"
        "r = prompt.Rotary(128)\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    o = prompt.prompt_attention(r(pos, q), k, k, cu, ck)\n"
        "g.replay(); a = o.clone(); g.replay()\n"
        "assert torch.equal(a, o) and torch.equal(o, prompt.prompt_attention(r(pos, q), k, k, cu, ck))\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_attention_empty_calls():
    q, k, v, _, cu_q, cu_k = _inputs([4], [4], 2, 2, 64, 64, 0, torch.bfloat16, 9)
    none = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 4.0)
    assert prompt.prompt_attention(q, k, v, none, none, out=out).eq(4.0).all()
    assert prompt.prompt_attention(q[:0], k, v, cu_q * 0, cu_k).shape == (0, 2, 64)
    assert prompt.prompt_attention(q, k[:0], v[:0], cu_q, cu_k * 0).eq(0).all()


def test_attention_on_a_side_stream_and_in_two_graphs():
    """Two captured calls that replay at the same time, on streams of their
    own, keep apart (each has its own workspace), and follow their inputs."""
    cases = []
    for seed, lens in ((10, ([1, 1], [5000, 70])), (11, ([300], [900]))):
        q, k, v, ks, cu_q, cu_k = _inputs(*lens, 8, 2, 128, 128, 0, torch.bfloat16, seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            want = prompt.prompt_attention(q, k, v, cu_q, cu_k)
        s.synchronize()
        assert torch.equal(want, prompt.prompt_attention(q, k, v, cu_q, cu_k))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = prompt.prompt_attention(q, k, v, cu_q, cu_k)
        cases.append((g, s, out, want, (q, k, v, cu_q, cu_k)))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s, *_ in cases:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for g, s, out, want, args in cases:
        assert torch.equal(out, want)
        args[2].mul_(-1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, -want)


def test_attention_repeats_bit_for_bit():
    q, k, v, _, cu_q, cu_k = _inputs([513, 1, 77], [900, 3000, 77], 4, 2, 128, 128, 0,
                                     torch.bfloat16, 12)
    first = prompt.prompt_attention(q, k, v, cu_q, cu_k)
    for _ in range(5):
        assert torch.equal(prompt.prompt_attention(q, k, v, cu_q, cu_k), first)


@pytest.mark.parametrize("B", [32, 33, 300, 700])
@pytest.mark.parametrize("most", [3, 150])
def test_attention_of_many_sequences(B, most):
    """Lengths from none to ``most`` tokens, some behind a beginning, sequences
    without queries or keys among them, more of them than the work table has
    entries."""
    g = torch.Generator().manual_seed(B + most)
    q_lens = torch.randint(0, most + 1, (B,), generator=g).tolist()
    k_lens = [n + int(c) for n, c in zip(q_lens, torch.randint(0, most, (B,), generator=g))]
    k_lens[3] = 0
    _check_attention(q_lens, k_lens, 2, 1, 128, 128, seed=B)


def test_attention_of_more_sequences_than_a_table_entry_has_lanes():
    g = torch.Generator().manual_seed(4)
    q_lens = torch.randint(0, 2, (9000,), generator=g).tolist()
    k_lens = [n * (1 + i % 5) for i, n in enumerate(q_lens)]
    _check_attention(q_lens, k_lens, 2, 2, 64, 64, seed=1)


@pytest.mark.parametrize("q_lens,k_lens", [
    ([150], [6000]), ([3, 150], [40, 6000]), ([1] * 40, [3000 + 7 * i for i in range(40)])])
def test_attention_of_many_items_in_shares(q_lens, k_lens):
    """More items than a warp has lanes in one sequence, and more sequences than
    lanes, their key tiles shared out."""
    _check_attention(q_lens, k_lens, 128, 1, 128, 128, seed=2)


# ------------------------------------------------------------- all together
def test_steps_of_all_three_in_one_graph():
    """Plan, rotary positions, cache and attention captured as one step of a
    padded batch; each replay has other lengths, down to none at all."""
    B, T, Tk, bs, width, heads, kv_heads, dim = 4, 256, 700, 32, 9, 4, 2, 128
    gen = _gen(21)
    spare = B * width * bs   # the cache row of padding
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.randperm(B * width, device="cuda", generator=gen).int().view(B, width)
    context, new = torch.zeros(B, **i32), torch.zeros(B, **i32)
    q, k, v = (torch.empty(T, n, dim, device="cuda", dtype=torch.bfloat16)
               for n in (heads, kv_heads, kv_heads))
    kc, vc = (torch.zeros(spare + 1, kv_heads, dim, device="cuda", dtype=torch.bfloat16)
              for _ in range(2))
    out = torch.empty(T, heads, dim, device="cuda", dtype=torch.bfloat16)
    rot = prompt.Rotary(64)

    def step():
        plan = prompt.plan_kv_blocks(context, new, table, None, None, bs, T, num_kv_tokens=Tk)
        rot(plan.positions, q, k, q_offset=64, k_offset=64, out_q=q, out_k=k)
        rows = torch.where(plan.slots < 0, spare, plan.slots)
        kc.index_copy_(0, rows, k)
        vc.index_copy_(0, rows, v)
        rows = torch.where(plan.kv_slots < 0, spare, plan.kv_slots)
        prompt.prompt_attention(q, kc[rows], vc[rows], plan.cu_new, plan.cu_total, out=out)
        context.add_(new)
        return plan

    def fill():
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
        out.fill_(7.0)

    fill()
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = step()
    context.zero_()
    keys = [k[:0].clone() for _ in range(B)]
    values = [v[:0].clone() for _ in range(B)]
    for lens in ([100, 1, 0, 155], [20, 1, 30, 1], [1, 1, 1, 1], [0, 0, 0, 0], [0, 250, 1, 5]):
        fill()
        new.copy_(torch.tensor(lens))
        pos = torch.cat([torch.arange(len(keys[b]), len(keys[b]) + n) for b, n in enumerate(lens)]
                        + [torch.full((T - sum(lens),), -1)]).cuda()
        want_q, want_k = rot(pos, q, k, q_offset=64, k_offset=64)
        g.replay()
        torch.cuda.synchronize()
        plan.check()
        assert torch.equal(plan.positions, pos)
        assert torch.equal(q, want_q) and torch.equal(k, want_k)
        at = 0
        for b, n in enumerate(lens):
            keys[b] = torch.cat([keys[b], k[at:at + n]])
            values[b] = torch.cat([values[b], v[at:at + n]])
            at += n
        k_lens = [len(x) for x in keys]
        assert context.tolist() == k_lens and plan.cu_total.tolist()[-1] == sum(k_lens)
        assert out[at:].eq(7.0).all()
        if at == 0:
            continue
        ref, mag = oprompt.attention(q[:at], torch.cat(keys), torch.cat(values), lens, k_lens,
                                     1 / math.sqrt(dim))
        tol = _bounds(ref, mag, torch.bfloat16, max(k_lens), torch.cat(values).abs().max().item())
        assert ((out[:at].double() - ref).abs() <= tol).all()


def test_two_threads_at_once():
    """Calls of two host threads, each on a stream of its own, keep apart."""
    def inputs(seed):
        q, k, v, _, cu_q, cu_k = _inputs([70 + seed, 1], [300, 900 + seed], 4, 2, 128, 128, 0,
                                         torch.bfloat16, seed)
        return q, k, v, cu_q, cu_k, torch.arange(len(q), device="cuda")

    rot = prompt.Rotary(128, interleaved=False)
    cases = [inputs(s) for s in (1, 2)]

    def run(q, k, v, cu_q, cu_k, pos):
        return prompt.prompt_attention(rot(pos, q), k, v, cu_q, cu_k)

    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(run(*cases[i]), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
