"""The operators of a prompt pass, measured: their cases, inputs, plain forms and exact values.

Three operators, in the order in which a packed batch of prompts uses them:

* ``plan``: block tables and slot maps from request lengths
  (``prompt.plan_kv_blocks``);
* ``rotary``: rotary positions of query and key heads (``prompt.Rotary``);
* ``attention``: causal attention over packed sequences with grouped heads,
  whose queries are the last tokens of their sequences
  (``prompt.prompt_attention``).

``run`` computes the plain form in elementary torch operations where ``own``
is false, and calls this package's operators where it is true.
"""

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# scores of one step of the plain form and of the exact one, at most this many
_SCORES = 1 << 28


def _ints(text):
    return [int(v) for v in text.split(",")]


# ------------------------------------------------------------------- cases
def _attention(name, dtype, heads, kv_heads, dim, v_dim, shared, new, context):
    """``new`` tokens of each sequence behind ``context`` earlier ones; the
    last ``shared`` columns of a key are one row for all heads."""
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "v_dim": v_dim, "shared": shared, "new": new,
            "context": context}


def _rotary(name, dtype, tokens, heads, kv_heads, dim, k_dim, rot, offset, interleaved, scaling,
            start):
    """``tokens`` rows at positions that begin at ``start``; the rotated
    columns are [offset, offset + rot) of a query head and the last ``rot``
    of a key head's ``k_dim``."""
    return {"name": name, "op": "rotary", "dtype": dtype, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "k_dim": k_dim, "rot": rot, "offset": offset,
            "interleaved": interleaved, "scaling": scaling, "start": start}


def _plan(name, requests, block, new_most, context_most, kv_map, lengths):
    """``requests`` requests with up to ``new_most`` new tokens each behind up
    to ``context_most`` cached ones, drawn from the number ``lengths``."""
    return {"name": name, "op": "plan", "requests": requests, "block": block,
            "new_most": new_most, "context_most": context_most, "kv_map": kv_map,
            "lengths": lengths}


def listed():
    return [
        # a 512-token step of a latent-attention decoder, four ragged prompts
        # (one of a single token): where launch and tail latency count
        _attention("attention_step", "bf16", 16, 16, 192, 128, 64, "137,1,255,119", "0,0,0,0"),
        # one whole prompt of the same decoder
        _attention("attention_prompt", "bf16", 16, 16, 192, 128, 64, "4096", "0"),
        # a long document on eight query heads per key head
        _attention("attention_long", "bf16", 32, 4, 128, 128, 0, "16384", "0"),
        # chunks of prompts behind their cached beginnings, seven query heads
        # per key head, an empty context among them
        _attention("attention_chunks", "fp16", 28, 4, 128, 128, 0, "512,509,3,1000",
                   "8192,4099,0,130"),
        # the next token of eight sequences of unlike lengths
        _attention("attention_tokens", "bf16", 32, 4, 128, 128, 0, "1,1,1,1,1,1,1,1",
                   "4095,17,32767,8191,0,12345,1000,2047"),
        # many short prompts on narrow heads
        _attention("attention_narrow", "fp16", 16, 8, 64, 64, 0,
                   "700,33,1024,5,260,411,129,128,1,900,77,350,640,2,513,255", ",".join(["0"] * 16)),
        # a decode step of eight sequences: the last 64 columns of each query
        # head and the one key row that all heads share
        _rotary("rotary_step", "bf16", 8, 16, 1, 192, 64, 64, 128, True, "none", 300),
        # a long prompt with whole heads and positions far past the trained ones
        _rotary("rotary_prompt", "bf16", 16384, 32, 4, 128, 128, 128, 0, False, "yarn", 98304),
        # a quarter of each head, an odd number of rows
        _rotary("rotary_partial", "fp16", 4099, 28, 4, 128, 128, 32, 0, False, "llama3", 5),
        # a decode step of eight sequences over blocks of 64
        _plan("plan_step", 8, 64, 1, 4096, False, 1),
        # a batch of ragged prompts, with the map of all their cached rows
        _plan("plan_prompts", 48, 64, 512, 2048, True, 2),
        # a full server: many requests, mixed lengths, blocks of 16
        _plan("plan_server", 1024, 16, 192, 4096, True, 3),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "plan"])
    if op == "attention":
        heads, kv_heads, dim, v_dim, shared = rng.choice([
            (16, 16, 192, 128, 64), (16, 16, 192, 128, 0), (32, 4, 128, 128, 0),
            (28, 4, 128, 128, 0), (40, 8, 128, 128, 0), (9, 3, 64, 64, 0), (16, 8, 64, 64, 0),
            (32, 1, 128, 128, 0)])
        most = listed()[2]
        most = work(most)["flops"]
        while True:
            n = _spread(rng, 1, 24)
            tokens = rng.random() < 0.25   # a step of single tokens
            new = [1 if tokens else _spread(rng, 1, 8192) for _ in range(n)]
            context = [_spread(rng, 1, 65536) - 1 if tokens or rng.random() < 0.3 else 0
                       for _ in range(n)]
            case = _attention("", rng.choice(["bf16", "fp16"]), heads, kv_heads, dim, v_dim,
                              shared, ",".join(map(str, new)), ",".join(map(str, context)))
            w = work(case)
            if w["flops"] <= most and w["bytes"] <= 2 << 30:
                break
    elif op == "rotary":
        dim, k_dim, rot, offset = rng.choice([(192, 64, 64, 128), (128, 128, 128, 0),
                                              (128, 128, 32, 0), (64, 64, 64, 0), (96, 96, 48, 0),
                                              (80, 80, 20, 60)])
        kv_heads = 1 if dim != k_dim else rng.choice([1, 2, 4, 8])
        case = _rotary("", rng.choice(["bf16", "fp16", "fp32"]), _spread(rng, 1, 16384),
                       kv_heads * rng.choice([1, 2, 3, 4]), kv_heads, dim, k_dim, rot, offset,
                       rng.random() < 0.5, rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                       _spread(rng, 1, 1 << 20) - 1)
    else:
        requests = _spread(rng, 1, 1024)
        case = _plan("", requests, rng.choice([16, 32, 64, 96, 128]),
                     rng.choice([1, _spread(rng, 1, 192)]), _spread(rng, 1, 4096),
                     rng.random() < 0.5, rng.randrange(1 << 30))
    del case["name"]
    return case


def _plan_lengths(case):
    """(context, new) token counts of the case's requests: some have nothing
    cached, some have nothing to add."""
    r = random.Random(case["lengths"])
    context, new = [], []
    for _ in range(case["requests"]):
        context.append(0 if r.random() < 0.2 else r.randint(0, case["context_most"]))
        new.append(0 if case["new_most"] > 1 and r.random() < 0.05 else
                   r.randint(1, case["new_most"]))
    return context, new


def work(case):
    if case["op"] == "attention":
        new, context = _ints(case["new"]), _ints(case["context"])
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, context))
        tq, tk = sum(new), sum(new) + sum(context)
        item = 2
        own_dim = case["dim"] - case["shared"]
        return {"bytes": item * (tq * case["heads"] * (case["dim"] + case["v_dim"]) +
                                 tk * case["kv_heads"] * (own_dim + case["v_dim"]) +
                                 tk * case["shared"]),
                "flops": 2 * pairs * case["heads"] * (case["dim"] + case["v_dim"])}
    if case["op"] == "rotary":
        item = 4 if case["dtype"] == "fp32" else 2
        wide = case["heads"] * case["dim"] + case["kv_heads"] * case["k_dim"]
        turned = (case["heads"] + case["kv_heads"]) * case["rot"]
        return {"bytes": case["tokens"] * (2 * item * wide + 8), "flops": 3 * case["tokens"] * turned}
    context, new = _plan_lengths(case)
    b, tq = case["requests"], sum(new)
    tk = tq + sum(context) if case["kv_map"] else 0
    bs = case["block"]
    taken = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(context, new))
    held = sum(-(-c // bs) for c in context) if case["kv_map"] else b
    return {"bytes": 16 * b + 4 * held + 8 * taken + 16 * tq + 8 * tk, "flops": 0}


# ------------------------------------------------------------------ inputs
def _scaling(case):
    kind = case["scaling"]
    if kind == "none":
        return None
    if kind in ("linear", "ntk"):
        return {"type": kind, "factor": 4.0}
    if kind == "yarn":
        return {"type": "yarn", "factor": 40.0, "original_max": 4096, "beta_fast": 32.0,
                "beta_slow": 1.0}
    return {"type": "llama3", "factor": 8.0, "original_max": 8192, "low_freq_factor": 1.0,
            "high_freq_factor": 4.0}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "attention":
        t = _TYPES[case["dtype"]]
        new, context = _ints(case["new"]), _ints(case["context"])
        total = [n + c for n, c in zip(new, context)]
        tq, tk = sum(new), sum(total)
        own_dim = case["dim"] - case["shared"]

        def rand(*shape):
            return torch.randn(*shape, generator=g, device=dev)

        # queries sharper than unit scores, so that some keys stand out
        state["q"] = (1.5 * rand(tq, case["heads"], case["dim"])).to(t)
        state["k"] = rand(tk, case["kv_heads"], own_dim).to(t)
        state["v"] = rand(tk, case["kv_heads"], case["v_dim"]).to(t)
        state["k_shared"] = rand(tk, case["shared"]).to(t) if case["shared"] else None
        state["cu_q"] = _cumulated(new, dev)
        state["cu_k"] = _cumulated(total, dev)
        state["new"], state["total"] = new, total
    elif case["op"] == "rotary":
        t = _TYPES[case["dtype"]]
        n = case["tokens"]
        state["q"] = torch.randn(n, case["heads"], case["dim"], generator=g, device=dev).to(t)
        state["k"] = torch.randn(n, case["kv_heads"], case["k_dim"], generator=g, device=dev).to(t)
        # a run of positions cut into two sequences, the second from the start
        pos = torch.arange(n, device=dev) + case["start"]
        cut = 2 * n // 3
        pos[cut:] -= case["start"] + cut
        state["positions"] = pos
        # the frequencies are a constant of the model, made when it is loaded
        state["freqs"] = _frequencies(case, dev)
        if own:
            from sluice_b200 import prompt
            state["rotary"] = prompt.Rotary(case["rot"], base=10000.0, scaling=_scaling(case),
                                            interleaved=case["interleaved"], device=dev)
    else:
        context, new = _plan_lengths(case)
        bs, b = case["block"], case["requests"]
        held = [-(-c // bs) for c in context]
        need = [-(-(c + n) // bs) for c, n in zip(context, new)]
        width = max(max(need), 1)
        blocks = sum(need) + 7
        r = random.Random(seed)
        ids = list(range(blocks))
        r.shuffle(ids)
        table = torch.full((b, width), -1, dtype=torch.int32)
        at = 0
        for i, h in enumerate(held):
            table[i, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
            at += h
        free = ids[at:]
        head = r.randrange(blocks)
        ring = torch.full((blocks,), -1, dtype=torch.int32)
        for i, v in enumerate(free):
            ring[(head + i) % blocks] = v
        state["table"] = table.to(dev)
        state["free"] = ring.to(dev)
        state["range"] = torch.tensor([head, head + len(free)], dtype=torch.int64, device=dev)
        state["range_out"] = torch.zeros(2, dtype=torch.int64, device=dev)
        state["context"] = torch.tensor(context, dtype=torch.int32, device=dev)
        state["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
        # a server knows how many tokens it has packed into the step
        state["tokens"] = sum(new)
        state["kv_tokens"] = sum(new) + sum(context) if case["kv_map"] else 0
    return state


def _cumulated(lengths, dev):
    c = [0]
    for n in lengths:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=dev)


def _frequencies(case, dev):
    """(angle per position of each pair in 64 bits, factor on the rotated values)."""
    rot, base = case["rot"], 10000.0
    i = torch.arange(rot // 2, dtype=torch.float64, device=dev)
    s = _scaling(case)
    if s is None:
        return base ** (-2.0 * i / rot), 1.0
    f = s["factor"]
    if s["type"] == "linear":
        return base ** (-2.0 * i / rot) / f, 1.0
    if s["type"] == "ntk":
        return (base * f ** (rot / (rot - 2.0))) ** (-2.0 * i / rot), 1.0
    plain = base ** (-2.0 * i / rot)
    if s["type"] == "yarn":
        # pairs that turn more than beta_fast times over the trained length
        # keep their frequency, those below beta_slow turns are stretched
        def pair(turns):
            return rot * math.log(s["original_max"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(math.floor(pair(s["beta_fast"])), 0)
        hi = min(math.ceil(pair(s["beta_slow"])), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return plain / f * ramp + plain * (1 - ramp), 0.1 * math.log(f) + 1.0
    wave = 2 * math.pi / plain
    low = s["original_max"] / s["low_freq_factor"]
    high = s["original_max"] / s["high_freq_factor"]
    mix = (s["original_max"] / wave - s["low_freq_factor"]) / \
        (s["high_freq_factor"] - s["low_freq_factor"])
    mid = (1 - mix) * plain / f + mix * plain
    return torch.where(wave > low, plain / f, torch.where(wave < high, plain, mid)), 1.0


# ------------------------------------------------------------------- passes
def run(state):
    op = state["case"]["op"]
    if own:
        from sluice_b200 import prompt
        if op == "attention":
            return prompt.prompt_attention(state["q"], state["k"], state["v"], state["cu_q"],
                                           state["cu_k"], k_shared=state["k_shared"])
        if op == "rotary":
            return state["rotary"](state["positions"], state["q"], state["k"],
                                   q_offset=state["case"]["offset"],
                                   k_offset=state["case"]["k_dim"] - state["case"]["rot"]
                                   if state["case"]["offset"] else 0)
        p = prompt.plan_kv_blocks(state["context"], state["new"], state["table"], state["free"],
                                  state["range"], state["case"]["block"], state["tokens"],
                                  num_kv_tokens=state["kv_tokens"], free_range_out=state["range_out"])
        out = [p.cu_new, p.cu_total, p.positions, p.slots, state["table"], state["range_out"]]
        return out + [p.kv_slots] if state["kv_tokens"] else out
    if op == "attention":
        return _plain_attention(state)
    if op == "rotary":
        return _plain_rotary(state)
    return _plain_plan(state)


def _plain_attention(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    per = heads // kv_heads
    scale = 1.0 / math.sqrt(case["dim"])
    out = torch.empty(q.shape[0], heads, case["v_dim"], dtype=q.dtype, device=q.device)
    q0 = k0 = 0
    for n, total in zip(state["new"], state["total"]):
        kf = k[k0:k0 + total].float()
        if state["k_shared"] is not None:
            pe = state["k_shared"][k0:k0 + total].float()
            kf = torch.cat([kf, pe[:, None, :].expand(-1, kv_heads, -1)], dim=-1)
        kf = kf.permute(1, 2, 0).contiguous()                      # [kv_heads, dim, total]
        vf = v[k0:k0 + total].float().transpose(0, 1).contiguous()  # [kv_heads, total, v_dim]
        rows = max(1, _SCORES // (total * heads))
        for a in range(0, n, rows):
            b = min(n, a + rows)
            last = total - n + b                                   # keys that row b - 1 sees
            qf = q[q0 + a:q0 + b].float().view(b - a, kv_heads, per, -1)
            qf = qf.permute(1, 2, 0, 3).reshape(kv_heads, per * (b - a), -1)
            s = torch.bmm(qf, kf[:, :, :last]).mul_(scale).view(kv_heads, per, b - a, last)
            at = torch.arange(total - n + a, total - n + b, device=q.device)
            hidden = torch.arange(last, device=q.device)[None, :] > at[:, None]
            s.masked_fill_(hidden, float("-inf"))
            s -= s.amax(dim=-1, keepdim=True)
            s.exp_()
            s /= s.sum(dim=-1, keepdim=True)
            o = torch.bmm(s.view(kv_heads, per * (b - a), last), vf[:, :last])
            o = o.view(kv_heads, per, b - a, -1).permute(2, 0, 1, 3).reshape(b - a, heads, -1)
            out[q0 + a:q0 + b] = o.to(q.dtype)
        q0, k0 = q0 + n, k0 + total
    return out


def _plain_rotary(state):
    case = state["case"]
    freq, factor = state["freqs"]
    rot = case["rot"]
    # angles in 64 bits: far positions lose their phase in 32
    angle = state["positions"].double()[:, None] * freq[None, :]
    cos = (angle.cos() * factor).float()[:, None, :]
    sin = (angle.sin() * factor).float()[:, None, :]

    def turn(x, offset):
        y = x.clone()
        part = x[..., offset:offset + rot].float()
        if case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            z = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = part[..., :rot // 2], part[..., rot // 2:]
            z = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        y[..., offset:offset + rot] = z.to(x.dtype)
        return y

    return (turn(state["q"], case["offset"]),
            turn(state["k"], case["k_dim"] - rot if case["offset"] else 0))


def _plain_plan(state):
    case = state["case"]
    bs, table, free = case["block"], state["table"], state["free"]
    context, new = state["context"].long(), state["new"].long()
    total = context + new
    dev = table.device

    def cumulated(x):
        return torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(x, 0)])

    cu_new, cu_total = cumulated(new), cumulated(total)
    held = (context + bs - 1) // bs
    need = (total + bs - 1) // bs
    cu_taken = cumulated(need - held)
    # the blocks that each request takes, in request order
    col = torch.arange(table.shape[1], device=dev)[None, :]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    at = state["range"][0] + cu_taken[:-1, None] + (col - held[:, None])
    table.copy_(torch.where(fresh, free[at.remainder(free.numel())], table))
    state["range_out"].copy_(torch.stack([state["range"][0] + cu_taken[-1], state["range"][1]]))

    def slots(first, count, starts, size):
        row = torch.repeat_interleave(torch.arange(table.shape[0], device=dev), count,
                                      output_size=size)
        pos = first[row] + torch.arange(size, device=dev) - starts[row]
        return pos, table[row, pos // bs].long() * bs + pos % bs

    positions, new_slots = slots(context, new, cu_new, state["tokens"])
    out = [cu_new.int(), cu_total.int(), positions, new_slots, table, state["range_out"]]
    if state["kv_tokens"]:
        out.append(slots(torch.zeros_like(context), total, cu_total, state["kv_tokens"])[1])
    return out


# -------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(state)
    if case["op"] == "rotary":
        return _exact_rotary(state)
    return _exact_plan(state)


def _exact_attention(state):
    """One head and a band of rows at a time, in 64 bits, over all keys of the
    sequence: weights exp(s - max) with zeros past the diagonal, divided last."""
    case, q = state["case"], state["q"]
    per = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape[0], case["heads"], case["v_dim"], dtype=torch.float64,
                      device=q.device)
    q0 = k0 = 0
    for n, total in zip(state["new"], state["total"]):
        band = max(1, (_SCORES // 2) // total)
        for h in range(case["heads"]):
            keys = state["k"][k0:k0 + total, h // per].double()
            if state["k_shared"] is not None:
                keys = torch.hstack([keys, state["k_shared"][k0:k0 + total].double()])
            values = state["v"][k0:k0 + total, h // per].double()
            for a in range(0, n, band):
                z = q[q0 + a:q0 + min(n, a + band), h].double() @ keys.T / case["dim"] ** 0.5
                seen = torch.ones_like(z, dtype=torch.bool).tril_(total - n + a)
                top = torch.where(seen, z, torch.full_like(z, -1e300)).max(1, keepdim=True).values
                w = torch.where(seen, (z - top).exp(), torch.zeros_like(z))
                out[q0 + a:q0 + a + z.shape[0], h] = (w @ values) / w.sum(1, keepdim=True)
        q0, k0 = q0 + n, k0 + total
    return out


def _exact_rotary(state):
    """Each pair as a complex number times factor * exp(i position freq)."""
    case = state["case"]
    freq, factor = state["freqs"]
    rot = case["rot"]
    pos = state["positions"].double()
    turns = torch.polar(torch.full((pos.numel(), rot // 2), factor, dtype=torch.float64,
                                   device=pos.device), torch.outer(pos, freq)).unsqueeze(1)
    res = []
    for x, offset in ((state["q"], case["offset"]),
                      (state["k"], case["k_dim"] - rot if case["offset"] else 0)):
        y = x.double()
        first = torch.arange(rot // 2, device=pos.device)
        first, step = (2 * first, 1) if case["interleaved"] else (first, rot // 2)
        a, b = offset + first, offset + first + step
        z = torch.complex(y[:, :, a], y[:, :, b]) * turns
        y[:, :, a], y[:, :, b] = z.real, z.imag
        res.append(y)
    return tuple(res)


def _exact_plan(state):
    """Request after request on the host, as a block allocator hands blocks out."""
    case = state["case"]
    bs = case["block"]
    table, ring = state["table"].cpu(), state["free"].cpu().tolist()
    head, tail = state["range"].cpu().tolist()
    cu_new, cu_total, positions, slots, kv = [0], [0], [], [], []
    for r, (c, n) in enumerate(zip(state["context"].tolist(), state["new"].tolist())):
        have = (c + bs - 1) // bs
        while have * bs < c + n:
            table[r, have] = ring[head % len(ring)]
            head, have = head + 1, have + 1
        blocks = table[r].tolist()
        every = [blocks[p // bs] * bs + p % bs for p in range(c + n if state["kv_tokens"] else 0)]
        kv += every
        positions += range(c, c + n)
        slots += every[c:] if every else [blocks[p // bs] * bs + p % bs for p in range(c, c + n)]
        cu_new.append(cu_new[-1] + n)
        cu_total.append(cu_total[-1] + c + n)

    def whole(x, t=torch.int64):
        return torch.tensor(x, dtype=t)

    out = [whole(cu_new, torch.int32), whole(cu_total, torch.int32), whole(positions), whole(slots),
           table, whole([head, tail])]
    return out + [whole(kv)] if state["kv_tokens"] else out
