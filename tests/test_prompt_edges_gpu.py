"""The prompt pass's operators at the edges of what their calls allow."""

import math
import threading

import pytest
import torch

from oracle import prompt as oprompt
from sluice_b200 import _lib, ops, prompt

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ block planner
@pytest.mark.parametrize("bs", [64, 48, 1])
def test_plan_of_a_context_past_its_complete_table_row(bs):
    """Without a ring, the cached rows behind the table row's last block have
    no slot; those before it, and the requests beside, keep theirs."""
    width = 4
    table = torch.tensor([[5, 9, 2, 7], [1, 0, 3, 4]], **I32)
    context, new = [width * bs + 2 * bs + 3, bs], [1, 2 * bs]
    T, Tk = sum(new), sum(context) + sum(new)
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.tensor(new, **I32), table,
                              None, None, bs, T, num_kv_tokens=Tk)
    ids = table.tolist()

    def slot(r, q):
        return ids[r][q // bs] * bs + q % bs if q < width * bs else -1

    assert p.status.tolist() == [_lib.KV_PLAN_BAD_INPUT, 0]
    assert p.slots.tolist() == [-1] + [slot(1, q) for q in range(bs, 3 * bs)]
    assert p.positions.tolist() == [context[0]] + list(range(bs, 3 * bs))
    assert p.kv_slots.tolist() == [slot(0, q) for q in range(context[0])] + [-1] + \
        [slot(1, q) for q in range(3 * bs)]
    assert table.tolist() == ids


def test_plan_of_a_context_past_its_row_among_many():
    """The same in several CTAs, several rows a lane."""
    bs, width, B = 16, 3, 700
    context = [width * bs + 100 if r % 3 == 0 else 20 for r in range(B)]
    table = torch.arange(B * width, **I32).view(B, width)
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.ones(B, **I32), table, None, None,
                              bs, B, num_kv_tokens=sum(context) + B)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT
    want, want_kv = [], []
    for r, c in enumerate(context):
        rows = [(r * width + q // bs) * bs + q % bs if q < width * bs else -1 for q in range(c + 1)]
        want_kv += rows
        want.append(rows[-1])
    assert p.slots.tolist() == want and p.kv_slots.tolist() == want_kv


@pytest.mark.parametrize("bs", [16, 96, 1])
@pytest.mark.parametrize("ring", [True, False])
@pytest.mark.parametrize("huge", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 5), (2 ** 31 - 40, 7)])
def test_plan_of_requests_behind_a_huge_one(bs, ring, huge):
    """A request whose lengths pass its table row, and with it the sums pass
    2^31 - 1, is reported; the ones behind it get their own positions and
    blocks."""
    context, new = [huge[0], 10, 3, 0], [huge[1], 5, 30, 2]
    width, rest = 40, 3
    held = [-(-c // bs) for c in context]
    need = [-(-(c + n) // bs) for c, n in zip(context, new)]
    ids = torch.randperm(400, generator=torch.Generator().manual_seed(bs)).tolist()
    rows, at = [ids[:width]], width
    for r in (1, 2, 3):
        n = held[r] if ring else need[r]
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    table = torch.tensor(rows, **I32)
    free, rng = (torch.tensor(ids[300:364], **I32), torch.tensor([60, 124], device="cuda")) \
        if ring else (None, None)
    T, Tk = sum(new) + rest, 100
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.tensor(new, **I32), table, free,
                              rng, bs, T, num_kv_tokens=Tk)
    taken = 0
    for r in (1, 2, 3):
        for i in range(held[r], need[r] if ring else held[r]):
            rows[r][i] = ids[300 + (60 + taken) % 64]
            taken += 1
    assert p.status.tolist() == [_lib.KV_PLAN_BAD_INPUT, taken]
    assert table.tolist() == rows
    positions = [c + i for c, n in zip(context, new) for i in range(n)]
    slots = [-1] * new[0] + [rows[r][q // bs] * bs + q % bs for r in (1, 2, 3)
                             for q in range(context[r], context[r] + new[r])]
    assert p.positions.tolist() == positions + [-1] * rest
    assert p.slots.tolist() == slots + [-1] * rest
    assert p.cu_new.tolist() == [0, new[0], new[0] + 5, new[0] + 35, new[0] + 37]
    assert p.cu_total.tolist() == [0] + 4 * [Tk]
    assert p.kv_slots.tolist() == [rows[0][q // bs] * bs + q % bs if q < width * bs else -1
                                   for q in range(Tk)]


def test_plan_of_sums_that_end_inside_a_request():
    """The sum of all rows passes 2^31 - 1 within a request that fits its row,
    behind one that found no blocks."""
    bs, width = 1 << 20, 2048
    context, new = [2 ** 31 - 6000, 0, 1023], [0, 5 * bs, 1]
    table = torch.full((3, width), -1, **I32)
    table[0] = torch.arange(width)
    table[2, 0] = 77
    T = 16
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.tensor(new, **I32), table,
                              torch.tensor([9], **I32), torch.tensor([0, 1], device="cuda"), bs, T)
    assert p.status.tolist() == [_lib.KV_PLAN_BAD_INPUT, 0]
    assert p.slots.eq(-1).all() and p.positions.tolist() == list(range(T))
    T = sum(new) + 1
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.tensor(new, **I32), table,
                              torch.tensor([9], **I32), torch.tensor([0, 1], device="cuda"), bs, T)
    assert p.slots[:5 * bs].eq(-1).all()
    assert p.slots[5 * bs:].tolist() == [77 * bs + 1023, -1]
    assert p.positions[5 * bs:].tolist() == [1023, -1]
    assert torch.equal(p.positions[:5 * bs], torch.arange(5 * bs, device="cuda"))


def test_plan_of_the_most_requests():
    """8192 requests, the most that a plan takes, against the oracle."""
    B, bs, width = 8192, 16, 3
    g = torch.Generator().manual_seed(8)
    context = torch.randint(0, 20, (B,), generator=g)
    new = torch.randint(0, 20, (B,), generator=g)
    held = (context + bs - 1) // bs
    table = torch.where(torch.arange(width) < held[:, None],
                        torch.arange(B * width).view(B, width), -1).int()
    free = (torch.randperm(2 * B, generator=g) + B * width).int()
    T, Tk = int(new.sum()), int((context + new).sum())
    tab = table.cuda()
    rng = torch.tensor([7, 7 + len(free)], device="cuda")
    p = prompt.plan_kv_blocks(context.int().cuda(), new.int().cuda(), tab, free.cuda(), rng, bs, T,
                              num_kv_tokens=Tk)
    ref = oprompt.plan(context.tolist(), new.tolist(), table.tolist(), free.tolist(), 7,
                       7 + len(free), bs, T, Tk)
    assert p.cu_new.tolist() == ref[0] and p.cu_total.tolist() == ref[1]
    assert p.positions.tolist() == ref[2] and p.slots.tolist() == ref[3]
    assert p.kv_slots.tolist() == ref[4] and tab.tolist() == ref[5]
    assert rng.tolist() == [ref[6], 7 + len(free)] and not ref[7]
    p.check()


# ---------------------------------------------------------------- attention
def _attend(q_lens, k_lens, heads, kv_heads, dim, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q, k, v = (torch.randn(n, h, dim, device="cuda", generator=g).to(dtype)
               for n, h in ((sum(q_lens), heads), (sum(k_lens), kv_heads), (sum(k_lens), kv_heads)))
    cu_q, cu_k = (torch.tensor([0] + list(n), device="cuda").cumsum(0).int()
                  for n in (q_lens, k_lens))
    out = prompt.prompt_attention(q, k, v, cu_q, cu_k)
    assert ops.workspace_status(prompt.prompt_attention.last_workspace) == 0
    return out, q, k, v


def _close(out, ref, mag, dtype=torch.bfloat16, more=0.0):
    """Half a step on the output, half a step on each weight as it is fed to the
    second product (hence on mag = sum p |v|), and 2^-11 of mag for the 32-bit
    scores, exponentials and sums."""
    u = torch.finfo(dtype).eps / 2
    err = (out.double() - ref).abs()
    tol = u * ref.abs() + (u + 2.0 ** -11) * mag + more
    assert out.isfinite().all() and (err <= tol).all(), (err - tol).max().item()


def _shared_out(q_lens, k_lens, heads, kv_heads, v_dim):
    """Whether the key tiles are shared out (only then the workspace is more
    than its header)."""
    return _lib.lib().sl_prompt_attention_workspace_bytes(
        len(q_lens), sum(q_lens), sum(k_lens), heads, kv_heads, v_dim) > 256


@pytest.mark.parametrize("q_lens,k_lens", [
    ([700] + [1] * 256, [3700] + [1300] * 256),                  # a work table entry of several
    ([1] * 200 + [900] + [1] * 99, [1600 + r % 7 for r in range(200)] + [4900] + [1600] * 99)])
def test_attention_of_a_long_prompt_among_many_in_shares(q_lens, k_lens):
    """Looking up a stretch takes long (hundreds of items of one sequence, added
    up by one lane) while the tiles of the one before pass by."""
    assert _shared_out(q_lens, k_lens, 128, 1, 128)
    out, q, k, v = _attend(q_lens, k_lens, 128, 1, 128, seed=len(q_lens))
    ref, mag = oprompt.attention(q, k, v, q_lens, k_lens, 128 ** -0.5)
    _close(out, ref, mag)


@pytest.mark.parametrize("heads,dim,q_len,k_len", [(128, 128, 4000, 12000), (128, 64, 4000, 12000),
                                                   (64, 128, 16001, 56003)])
def test_attention_of_thousands_of_items_in_shares(heads, dim, q_len, k_len):
    """Thousands of items of one sequence and many key tiles that no row is
    masked in; every 97th query is compared."""
    assert _shared_out([q_len], [k_len], heads, 1, dim)
    out, q, k, v = _attend([q_len], [k_len], heads, 1, dim, seed=q_len)
    kk, vv = k[:, 0].double(), v[:, 0].double()
    for i in list(range(0, q_len, 97)) + [q_len - 1]:
        n = i + 1 + k_len - q_len
        p = torch.softmax(q[i].double() @ kk[:n].T * dim ** -0.5, dim=-1)
        _close(out[i], p @ vv[:n], p @ vv[:n].abs())


def test_attention_raises_a_status_and_never_lowers_it():
    """A call that ran through leaves the caller's word, and the device's, as
    they were, whatever they hold; what the device's holds is raised once."""
    def call(**kw):
        return prompt.prompt_attention(q, q, q, cu, cu, **kw)

    q = torch.randn(40, 2, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 40], **I32)
    want = call()
    prompt.check_attention()
    word = torch.zeros(1, **I32)
    assert torch.equal(call(status=word), want) and word.item() == 0
    word.fill_(_lib.SL_ERR_TIMEOUT)
    call(status=word)
    assert word.item() == _lib.SL_ERR_TIMEOUT
    prompt.check_attention()            # (the call had a word of its own)
    call()
    shared = prompt.prompt_attention.last_workspace
    shared.fill_(_lib.SL_ERR_TIMEOUT)   # as a wait that ran out does
    call()
    with pytest.raises(_lib.SluiceError, match="wait ran out"):
        prompt.check_attention(torch.device("cuda", 0))
    prompt.check_attention("cuda")
    with pytest.raises(ValueError, match="status"):
        call(status=torch.zeros(2, **I32))
    with pytest.raises(ValueError):
        call(status=torch.zeros(1, dtype=torch.int32))


def test_attention_keeps_no_workspace():
    """Key tiles in shares take tens of MB while the call runs, none after."""
    assert _shared_out([1, 1], [30000, 30000], 8, 2, 128)
    out, *rest = _attend([1, 1], [30000, 30000], 8, 2, 128, seed=1)
    del out, rest
    assert prompt.prompt_attention.last_workspace.untyped_storage().nbytes() <= 512


@pytest.mark.parametrize("size", [3.3e38, 1e-20])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim", [
    ([300, 1], [300, 700], 2, 1, 128), ([1, 2], [40001, 30], 8, 2, 128), ([130], [1500], 4, 4, 64)])
def test_attention_of_the_largest_and_of_small_values(size, q_lens, k_lens, heads, kv_heads, dim):
    """No weighted sum passes the largest value, for scores at random, all alike
    and growing from key to key."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    tq, tk = sum(q_lens), sum(k_lens)
    v = size * (1 - 0.9 * torch.rand(tk, kv_heads, dim, device="cuda", generator=g))
    v = (v * torch.randint(0, 2, (tk, 1, 1), device="cuda", generator=g).sub(0.5).sign()).bfloat16()
    cu_q, cu_k = (torch.tensor([0] + n, device="cuda").cumsum(0).int() for n in (q_lens, k_lens))
    for step in (None, 0.0, 0.05, 0.7):
        if step is None:
            q, k = (torch.randn(n, h, dim, device="cuda", generator=g).bfloat16()
                    for n, h in ((tq, heads), (tk, kv_heads)))
        else:
            # (steps of 1/16 in the last column: exact in bf16 up to 256 of them)
            q = torch.zeros(tq, heads, dim, device="cuda", dtype=torch.bfloat16)
            q[..., -1] = 16 * step * dim ** 0.5
            k = torch.zeros(tk, kv_heads, dim, device="cuda", dtype=torch.bfloat16)
            k[..., -1] = ((torch.arange(tk, device="cuda") % 256) / 16)[:, None].bfloat16()
        out = prompt.prompt_attention(q, k, v, cu_q, cu_k)
        ref, mag = oprompt.attention(q, k, v, q_lens, k_lens, dim ** -0.5)
        # scores reach 256 * step, rounded at 2^-24 of that
        _close(out, ref, mag, more=(256 * (step or 0.0) * 2.0 ** -22) * mag)


@pytest.mark.parametrize("strong", [0, 30000, -1])
@pytest.mark.parametrize("q_len,n,heads", [(1, 60001, 2), (130, 60001, 2), (1, 30101, 148)])
def test_attention_of_a_flat_tail_behind_one_strong_key_in_fp16(strong, q_len, n, heads):
    """Weights of 2^-26.3 of the strong key's, tens of thousands of them, make a
    difference together; in shares (few heads) and in whole items."""
    q = torch.zeros(q_len, heads, 64, device="cuda", dtype=torch.float16)
    q[..., 0] = 1.0
    at = strong if strong >= 0 else n - q_len   # (every query sees it)
    k = torch.zeros(n, heads, 64, device="cuda", dtype=torch.float16)
    k[at, :, 0] = 18.25
    v = torch.ones(n, heads, 64, device="cuda", dtype=torch.float16)
    v[at, :, :32] = 0.0
    cu_q, cu_k = torch.tensor([0, q_len], **I32), torch.tensor([0, n], **I32)
    out = prompt.prompt_attention(q, k, v, cu_q, cu_k, scale=1.0)
    ref, mag = oprompt.attention(q, k, v, [q_len], [n], 1.0)
    assert ref[..., :32].min() > 3e-4
    # a weight of 2^7 w in fp16 is off by half of 2^-24 at most where it has no
    # bits below that, against a sum of at least 2^7; and the output by half of
    # its own last bit
    _close(out, ref, mag, torch.float16, more=2.0 ** -32 * n + 2.0 ** -25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim,v_dim,shared", [(2, 2, 64, 64, 0), (4, 2, 128, 128, 0),
                                                             (2, 2, 192, 128, 64)])
@pytest.mark.parametrize("q_len,k_len", [(150, 150), (2, 3000), (40, 700)])
def test_attention_of_an_infinite_value_at_a_weight_of_zero(dtype, heads, kv_heads, dim, v_dim,
                                                            shared, q_len, k_len):
    """0 times inf: a key that scores -inf, or too low for a weight, makes NaN
    of its value's infinite columns, as the formula does, wherever it lies; a
    key with a weight makes inf of them."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    q = (torch.rand(q_len, heads, dim, device="cuda", generator=g) + 0.1).to(dtype)
    k = torch.randn(k_len, kv_heads, dim - shared, device="cuda", generator=g).to(dtype)
    v = torch.randn(k_len, kv_heads, v_dim, device="cuda", generator=g).to(dtype)
    ks = torch.randn(k_len, shared, device="cuda", generator=g).to(dtype) if shared else None
    cu_q, cu_k = torch.tensor([0, q_len], **I32), torch.tensor([0, k_len], **I32)
    clean = prompt.prompt_attention(q, k, v, cu_q, cu_k, k_shared=ks)
    for at in (k_len - q_len, k_len - q_len // 2 - 1, k_len - 1):
        first = max(0, at - (k_len - q_len))   # the first query that sees it
        for low in (float("-inf"), -30000.0, None):
            k2, v2, s2 = k.clone(), v.clone(), None if ks is None else ks.clone()
            if low is not None:
                (k2[at, :, 3] if s2 is None else s2[at, 3:4])[:] = low
            v2[at, :, 5] = float("inf")
            v2[at, :, 40] = float("-inf")
            o = prompt.prompt_attention(q, k2, v2, cu_q, cu_k, k_shared=s2)
            assert torch.equal(o[:first], clean[:first])
            seen = o[first:]
            if at == 0 and low == float("-inf"):
                assert seen[0].isnan().all()   # it is all that this query sees
                seen = seen[1:]
            if at == 0 and low == -30000.0:
                # ... with all the weight there is
                assert seen[0, :, 5].eq(float("inf")).all() and seen[0, :, 40].eq(-float("inf")).all()
                seen = seen[1:]
            if low is None:
                assert seen[..., 5].eq(float("inf")).all()
                assert seen[..., 40].eq(-float("inf")).all()
            else:
                assert seen[..., [5, 40]].isnan().all()
            rest = [c for c in range(v_dim) if c not in (5, 40)]
            assert seen[..., rest].isfinite().all()


def test_attention_scales_count_by_value():
    """A scale that is a tensor, changed between two calls."""
    q = torch.randn(40, 2, 64, device="cuda").bfloat16()
    cu, scale = torch.tensor([0, 40], **I32), torch.tensor(0.05)
    for value in (0.05, 2.0):
        scale.fill_(value)
        assert torch.equal(prompt.prompt_attention(q, q, q, cu, cu, scale=scale),
                           prompt.prompt_attention(q, q, q, cu, cu, scale=value))


@pytest.mark.parametrize("cq,ck,q_len,k_len,rows", [
    ([0, 1000], [0, 64], 64, 64, (0, 64)), ([0, 64], [0, 5000], 64, 64, (0, 64)),
    ([-50, 64], [-9, 64], 64, 64, (0, 64)), ([0, 64], [60, 10], 64, 0, (0, 64)),
    ([0, 64], [2000000000, 2000000100], 64, 0, (0, 64)),
    # (rows 20 to 39 belong to two sequences; those behind see no keys)
    ([0, 40, 20, 64], [0, 64, 64, 64], 40, 64, (0, 20)), ([0, 40, 20, 64], [0, 64, 64, 64], 64, 0, (40, 64))])
def test_attention_of_offsets_cut_to_the_tensors(cq, ck, q_len, k_len, rows):
    """Offsets past the tensors count as their ends, and a sequence that runs
    backwards is empty; no wait runs out."""
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    q, k, v = (torch.randn(64, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(3))
    word = torch.zeros(1, **I32)
    out = prompt.prompt_attention(q, k, v, torch.tensor(cq, **I32), torch.tensor(ck, **I32),
                                  status=word)
    assert word.item() == 0
    ref, mag = oprompt.attention(q, k, v, [q_len], [k_len], 64 ** -0.5)
    a, b = rows
    _close(out[a:b], ref[a:b], mag[a:b])


# ------------------------------------------------------------------- rotary
def _frequencies(kind, rot, base=10000.0):
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if kind == "linear":
        return [x / 4.0 for x in f], {"type": kind, "factor": 4.0}
    if kind == "ntk":
        b = base * 3.0 ** (rot / (rot - 2))
        return [b ** (-2.0 * i / rot) for i in range(rot // 2)], {"type": kind, "factor": 3.0}

    def llama3(x):
        wave = 2 * math.pi / x
        if wave < 8192 / 4.0:
            return x
        if wave > 8192 / 1.0:
            return x / 8.0
        smooth = (8192 / wave - 1.0) / (4.0 - 1.0)
        return (1 - smooth) * x / 8.0 + smooth * x

    return [llama3(x) for x in f], {"type": kind, "factor": 8.0, "original_max": 8192,
                                    "low_freq_factor": 1.0, "high_freq_factor": 4.0}


@pytest.mark.parametrize("kind", ["linear", "ntk", "llama3"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotary_of_scaled_frequencies(kind, interleaved, dtype):
    T, rot = 37, 64
    freqs, scaling = _frequencies(kind, rot)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = torch.randn(T, 3, 96, device="cuda", generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), device="cuda", generator=g)
    y = prompt.Rotary(rot, scaling=scaling, interleaved=interleaved)(pos, x, q_offset=8)
    ref = oprompt.rotary(x, pos, torch.tensor(freqs, dtype=torch.float64), 1.0, 8, interleaved)
    # half a step of the result; 8 half steps of 32 bits of a pair's magnitude for
    # the angle, the sine and the products; and the frequencies' own powers, 4 steps
    # of 2^-52 relative to an angle of 2^20 at most
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + \
        (8 * 2.0 ** -24 + 2.0 ** 20 * 2.0 ** -50) * 2 * x.double().abs().amax() + 2.0 ** -25
    assert ((y.double() - ref).abs() <= tol).all()


def test_the_devices_status_word_of_two_threads_and_inference_mode(monkeypatch):
    """First calls at the same time, in inference mode: one word, which is read
    and cleared outside of it."""
    monkeypatch.setattr(prompt, "_failed", {})
    q = torch.randn(9, 2, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 9], **I32)
    gate, words = threading.Barrier(4), []

    def work():
        with torch.inference_mode():
            gate.wait()
            prompt.prompt_attention(q, q, q, cu, cu)
            words.append(prompt._failed_word(0).data_ptr())

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(words) == 4 and len(set(words)) == 1
    prompt._failed[0].fill_(_lib.SL_ERR_TIMEOUT)
    with pytest.raises(_lib.SluiceError):
        prompt.check_attention()
    prompt.check_attention()


def test_attention_as_the_first_call_of_a_thread():
    """A host thread that has called nothing of the device yet."""
    q = torch.randn(50, 4, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 50], **I32)
    outs = [prompt.prompt_attention(q, q, q, cu, cu) for _ in range(2)]
    want = outs.pop().clone()
    outs.clear()   # (the thread's allocations come from the cache)
    t = threading.Thread(target=lambda: outs.append(prompt.prompt_attention(q, q, q, cu, cu)))
    t.start()
    t.join()
    assert outs and torch.equal(outs[0], want)
