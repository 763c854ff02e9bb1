"""Prompts in one pass through the decoder harness: the block planner, rotary
positions, the latent cache and the packed attention together, against the
same tokens fed one position per step; paged against contiguous caches."""

from dataclasses import replace

import pytest
import torch

from sluice_b200 import configs, prompt
from sluice_b200.harness import V2_LITE_DECODER, DecoderHarness, OffloadedDecoder
from sluice_b200.layer import MoEDecodeStack

pytestmark = pytest.mark.gpu


def _harness(batch=3, max_len=320, layers=3, seed=4, **kw):
    dcfg = replace(V2_LITE_DECODER, num_layers=layers, vocab=2048)
    # the MoE layers stand aside: a fixed map of the rows that keeps them apart
    return DecoderHarness(dcfg, lambda li, x: x.roll(1, dims=-1), batch=batch, max_len=max_len,
                          seed=seed, **kw)


def _tokens(lengths, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 2048, (n,), generator=g) for n in lengths]


def _by_steps(h, tokens):
    """The tokens fed one position per step, every sequence at its own pace."""
    out = [None] * len(tokens)
    n = max(len(t) for t in tokens)
    for p in range(n):
        ids = torch.tensor([int(t[min(p, len(t) - 1)]) for t in tokens], device="cuda")
        h.pos.copy_(torch.tensor([min(p, len(t) - 1) for t in tokens], device="cuda"))
        nxt = h.step(ids)
        for b, t in enumerate(tokens):
            if p == len(t) - 1:
                out[b] = int(nxt[b])
    h.pos.copy_(torch.tensor([len(t) for t in tokens], device="cuda"))
    return out


def _row(h, li, b, p):
    """The cache row of a sequence's position."""
    if not h.paged:
        return h.cache[li, b, p]
    blk = int(h.block_table[b, p // h.block_size])
    return h.cache[li, blk, p % h.block_size]


def _rows(h, li, b, n):
    return torch.stack([_row(h, li, b, p) for p in range(n)]).float()


# Both ways round to bf16 after each product, norm and sum, about a dozen times
# a layer and at different places (the steps absorb the key map into the query,
# the pass expands it): 36 roundings of half a step of 2^-8 each, added up as
# independent errors over three layers, are 2.4e-2 of the values' size.
TOL = 2.4e-2


@pytest.mark.parametrize("lengths", [[1, 1, 1], [37, 1, 130], [129, 300, 64], [5, 0, 40]])
def test_prefill_matches_single_steps(lengths):
    a, b = _harness(), _harness()
    tokens = _tokens(lengths)
    nxt = a.prefill(torch.cat(tokens).cuda(), lengths)
    live = [i for i, n in enumerate(lengths) if n]
    # (a sequence without tokens is fed a stand-in whose rows are not compared)
    _by_steps(b, [t if len(t) else torch.zeros(1, dtype=torch.long) for t in tokens])
    assert a.pos.tolist() == lengths
    assert nxt.tolist() == [int(v) if n else -1 for v, n in zip(nxt, lengths)]
    for li in range(3):
        for s in live:
            got, ref = _rows(a, li, s, lengths[s]), _rows(b, li, s, lengths[s])
            assert (got - ref).norm() <= TOL * ref.norm(), (li, s)
    # rows behind a sequence's last position were not touched
    for s, n in enumerate(lengths):
        assert a.cache[:, s, n:].eq(0).all()
    # decode goes on from either cache alike
    ids = torch.randint(0, 2048, (3,), device="cuda")
    a.step(ids)
    b.step(ids)
    for s in live:
        got, ref = _row(a, 2, s, lengths[s]).float(), _row(b, 2, s, lengths[s]).float()
        assert (got - ref).norm() <= TOL * ref.norm()


def test_prefill_in_chunks_matches_one_pass():
    lengths = [200, 33, 130]
    tokens = _tokens(lengths)
    whole, chunked = _harness(), _harness()
    whole.prefill(torch.cat(tokens).cuda(), lengths)
    done = [0, 0, 0]
    for chunk in ([64, 33, 1], [136, 0, 100], [0, 0, 29]):
        ids = torch.cat([t[d:d + c] for t, d, c in zip(tokens, done, chunk)])
        nxt = chunked.prefill(ids.cuda(), chunk)
        done = [d + c for d, c in zip(done, chunk)]
        assert [v >= 0 for v in nxt.tolist()] == [c > 0 for c in chunk]
    assert done == lengths and chunked.pos.tolist() == lengths
    for li in range(3):
        for s, n in enumerate(lengths):
            got, ref = _rows(chunked, li, s, n), _rows(whole, li, s, n)
            assert (got - ref).norm() <= TOL * ref.norm(), (li, s)
    # positions given by the caller: the same, without reading them back
    again = _harness()
    again.prefill(torch.cat([t[:10] for t in tokens]).cuda(), [10] * 3, context=[0] * 3)
    again.prefill(torch.cat([t[10:20] for t in tokens]).cuda(), [10] * 3, context=[10] * 3)
    assert again.pos.tolist() == [20] * 3


@pytest.mark.parametrize("block_size", [32, 64, 96])
def test_paged_cache_gives_the_contiguous_results(block_size):
    """Prompts, single steps across block borders and further chunks: the same
    bits from a pool of blocks as from one run of rows per sequence."""
    flat, paged = _harness(), _harness(cache_blocks=24, block_size=block_size)
    lengths = [70, 31, 128]
    tokens = torch.cat(_tokens(lengths)).cuda()
    ids_f, ids_p = flat.prefill(tokens, lengths), paged.prefill(tokens, lengths)
    assert torch.equal(ids_f, ids_p)
    for _ in range(5):
        ids_f, ids_p = flat.step(ids_f), paged.step(ids_p)
        assert torch.equal(ids_f, ids_p)
    more = torch.cat(_tokens([3, 90, 1], seed=6)).cuda()
    assert torch.equal(flat.prefill(more, [3, 90, 1]), paged.prefill(more, [3, 90, 1]))
    total = flat.pos.tolist()
    assert total == paged.pos.tolist() == [78, 126, 134]
    for li in range(3):
        for s, n in enumerate(total):
            assert torch.equal(_rows(flat, li, s, n), _rows(paged, li, s, n))
    used = sum(-(-n // block_size) for n in total)
    assert paged.free_range.tolist() == [used, 24]
    blocks = paged.block_table[paged.block_table >= 0].tolist()
    assert sorted(blocks) == list(range(used))
    paged.check_blocks()
    paged.reset()
    assert paged.free_range.tolist() == [0, 24] and paged.block_table.eq(-1).all()


def test_pool_that_runs_out():
    h = _harness(cache_blocks=4, block_size=32)
    with pytest.raises(prompt.KvPlanError):
        h.prefill(torch.cat(_tokens([60, 60, 60])).cuda(), [60, 60, 60])
    # nothing was taken or moved: a smaller batch fits
    assert h.free_range.tolist() == [0, 4] and h.pos.tolist() == [0, 0, 0]
    h.check_blocks()
    ids = h.prefill(torch.cat(_tokens([32, 20, 32])).cuda(), [32, 20, 32])
    assert h.free_range.tolist() == [3, 4]
    # the next step wants two more blocks, one is left: it is reported, and the
    # served sequences' rows are written
    h.step(ids)
    with pytest.raises(prompt.KvPlanError):
        h.check_blocks()
    assert h.block_table[:, 1].tolist() == [3, -1, -1]
    # a prompt goes on only behind positions that have cache rows: sequence 2's
    # last one found no block, and no sequence may be said to be further than
    # its blocks reach
    state = [t.clone() for t in (h.cache, h.block_table, h.free_range)]
    for lengths, context in (([0, 0, 3], None), ([3, 3, 3], [33, 21, 33]), ([0, 5, 0], [0, 40, 0])):
        with pytest.raises(prompt.KvPlanError):
            h.prefill(torch.cat(_tokens(lengths)).cuda(), lengths, context=context)
        assert all(torch.equal(a, b) for a, b in zip(state, (h.cache, h.block_table, h.free_range)))
    h.prefill(torch.cat(_tokens([4, 11, 0])).cuda(), [4, 11, 0])
    assert h.pos.tolist() == [37, 32, 33]


def test_prefill_refuses():
    h = _harness()
    ids = torch.zeros(6, dtype=torch.long, device="cuda")
    for bad in ([2, 2], [2, 2, 3], [4, -1, 3]):
        with pytest.raises(ValueError):
            h.prefill(ids, bad)
    with pytest.raises(ValueError, match="max_len"):
        h.prefill(torch.zeros(321, dtype=torch.long, device="cuda"), [321, 0, 0])
    with pytest.raises(ValueError):
        h.prefill(ids, [2, 2, 2], context=[0, 0])
    assert h.prefill(ids[:0], [0, 0, 0]).tolist() == [-1, -1, -1]
    with pytest.raises(ValueError):
        _harness(cache_blocks=4, block_size=48)
    with pytest.raises(ValueError):
        _harness(cache_blocks=4, fused_attention=False)
    with pytest.raises(ValueError):
        _harness(fused_attention=False).prefill(ids, [2, 2, 2])


def test_offloaded_decoder_from_prompts_to_captured_steps():
    """The whole decoder: prompts through the prompt pass (the MoE layers in
    expert waves), then captured decode steps, on a contiguous and on a paged
    cache; restoring the state repeats the same tokens."""
    dcfg = replace(V2_LITE_DECODER, num_layers=3, vocab=4096)
    runs = []
    for kw in ({}, dict(cache_blocks=40, block_size=32)):
        stack = MoEDecodeStack(configs.V2_LITE, slots=40, seed=3, num_layers=2)
        d = OffloadedDecoder(dcfg, stack, 4, 256, 3, **kw)
        g = torch.Generator().manual_seed(9)
        lengths = [100, 7, 1, 63]
        ids = torch.randint(0, 4096, (sum(lengths),), generator=g).cuda()
        first = d.prefill(ids, lengths)
        d.capture()
        state = d.save()
        seen = [d.replay().tolist() for _ in range(40)]
        assert d.model.pos.tolist() == [n + 40 for n in lengths]
        d.check()
        assert d.stats()["fills"] > 0
        d.restore(state)
        again = [d.replay().tolist() for _ in range(40)]
        assert d.model.pos.tolist() == [n + 40 for n in lengths]
        runs.append((first.tolist(), seen[:4], again[:4]))
        d.release()
    # the experts' slots differ in order only, so the tokens are the same
    assert runs[0][0] == runs[1][0] and runs[0][1] == runs[1][1]


@pytest.mark.parametrize("kw", [{}, dict(cache_blocks=24, block_size=32)])
def test_prefill_reports_a_wait_that_ran_out(kw, monkeypatch):
    """One layer's attention gives up (its status says so): no position moves,
    no block is taken, and the same prompts can be taken again."""
    h, calls = _harness(**kw), []
    real = prompt.prompt_attention

    def gives_up(*args, status=None, **rest):
        out = real(*args, status=status, **rest)
        calls.append(status)
        if len(calls) == 2:
            status.fill_(5)   # SL_ERR_TIMEOUT
        return out

    tokens = _tokens([30, 1, 50])
    monkeypatch.setattr(prompt, "prompt_attention", gives_up)
    before = h.save_blocks()
    with pytest.raises(RuntimeError, match="wait ran out"):
        h.prefill(torch.cat(tokens).cuda(), [30, 1, 50])
    assert len(calls) == 3 and h.pos.tolist() == [0, 0, 0]
    assert all(torch.equal(v, before[n]) for n, v in h.save_blocks().items())
    monkeypatch.undo()
    again = h.prefill(torch.cat(tokens).cuda(), [30, 1, 50])
    assert torch.equal(again, _harness(**kw).prefill(torch.cat(tokens).cuda(), [30, 1, 50]))
    h.check_blocks()


def test_far_positions_have_the_same_keys_from_steps_and_prompts():
    """A million positions on, the first layer's rotated keys of two tokens as
    single steps and as a prompt's chunk write them."""
    P, rope = 10 ** 6, V2_LITE_DECODER.qk_rope
    ids = torch.tensor([7, 1999], device="cuda")
    rows = []
    for chunk in (False, True):
        h = _harness(batch=1, max_len=P + 8, layers=1)
        h.pos.fill_(P)
        if chunk:
            h.prefill(ids, [2], context=[P])
        else:
            for i in range(2):
                h.step(ids[i:i + 1])
        assert h.pos.tolist() == [P + 2]
        rows.append(h.cache[0, 0, P:P + 2, -rope:].float())
    a, b = (r.view(2, rope // 2, 2) for r in rows)
    # a step of the projection's rounding between them, half a step of each
    # result's: four half steps of a pair's length
    assert ((a - b).abs().amax(-1) <= 4 * 2.0 ** -8 * a.norm(dim=-1)).all()


def test_prefill_that_fails_in_a_layer_takes_no_blocks():
    h = _harness(cache_blocks=8, block_size=32)
    h.prefill(torch.cat(_tokens([20, 40, 1])).cuda(), [20, 40, 1])
    before, pos, moe = h.save_blocks(), h.pos.tolist(), h.moe

    def fails(li, x):
        raise OSError("no experts")

    h.moe = fails
    more = torch.cat(_tokens([60, 0, 31], seed=6)).cuda()
    for _ in range(3):
        with pytest.raises(OSError):
            h.prefill(more, [60, 0, 31])
        assert h.pos.tolist() == pos
        assert all(torch.equal(v, before[n]) for n, v in h.save_blocks().items())
    h.moe = moe
    nxt = h.prefill(more, [60, 0, 31])
    assert nxt.tolist()[1] == -1 and h.pos.tolist() == [80, 40, 32]
    assert h.free_range.tolist() == [6, 8]   # ceil(80 / 32) + ceil(40 / 32) + ceil(32 / 32)
    h.check_blocks()


@pytest.mark.parametrize("kw", [{}, dict(cache_blocks=8, block_size=32),
                                dict(cache_blocks=8, block_size=96)])
def test_steps_past_the_last_position_are_reported(kw):
    h = _harness(batch=2, max_len=96 if kw.get("block_size") == 32 else 80, **kw)
    n = h.max_len - 1
    ids = h.prefill(torch.cat(_tokens([n, 20])).cuda(), [n, 20])
    other = _rows(h, 0, 1, 20)
    ids = h.step(ids)   # the last position
    h.check_blocks()
    for _ in range(2):
        ids = h.step(ids)
        with pytest.raises(prompt.KvPlanError):
            h.check_blocks()
    assert torch.equal(_rows(h, 0, 1, 20), other)
    h.reset()
    h.check_blocks()
