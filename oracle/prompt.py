"""The prompt pass's operators restated on plain Python and 64-bit torch: the
block planner request by request, rotary positions as complex products,
causal attention over packed sequences with its absolute sums (for error
bounds)."""

from __future__ import annotations

import torch


def plan(context, new, table, free, head, tail, block_size, T, Tk=0):
    """(cu_new, cu_total, positions, slots, kv_slots, table, head, overflow)
    as lists; ``table`` a list of rows. A request whose blocks do not fit the
    ring or its row takes nothing, and neither does any later one that needs
    blocks (in the ring's case)."""
    table = [list(r) for r in table]
    n, width = len(free), len(table[0])
    used, at, overflow = 0, 0, False
    cu_new, cu_total, positions, slots, kv = [0], [0], [], [], []
    for r, (c, f) in enumerate(zip(context, new)):
        held, need = -(-c // block_size), -(-(c + f) // block_size)
        served = True
        if need > width:
            served, overflow = False, True
        else:
            at += need - held
            if need > held and at > tail - head:
                served, overflow = False, True
            elif need > held:
                for i in range(held, need):
                    table[r][i] = free[(head + at - need + i) % n]
                used = at

        def slot(p):
            if p >= c and not served:
                return -1
            b = table[r][p // block_size]
            return -1 if b < 0 else b * block_size + p % block_size

        positions += range(c, c + f)
        slots += [slot(p) for p in range(c, c + f)]
        if Tk:
            kv += [slot(p) for p in range(c + f)]
        cu_new.append(cu_new[-1] + f)
        cu_total.append(cu_total[-1] + c + f)
    positions += [-1] * (T - len(positions))
    slots += [-1] * (T - len(slots))
    kv += [-1] * (Tk - len(kv))
    return cu_new, cu_total, positions, slots, kv, table, head + used, overflow


def rotary(x, positions, freqs, factor, offset, interleaved):
    """x [T, heads, dim] rotated in 64 bits; rows at negative positions kept."""
    y = x.double().clone()
    half = freqs.numel()
    j = torch.arange(half, device=x.device)
    a, b = (offset + 2 * j, offset + 2 * j + 1) if interleaved else (offset + j, offset + half + j)
    t = torch.outer(positions.double(), freqs.double().to(x.device))
    cos, sin = (t.cos() * factor)[:, None], (t.sin() * factor)[:, None]
    live = (positions >= 0)[:, None, None]
    y[..., a] = torch.where(live, x[..., a].double() * cos - x[..., b].double() * sin,
                            x[..., a].double())
    y[..., b] = torch.where(live, x[..., b].double() * cos + x[..., a].double() * sin,
                            x[..., b].double())
    return y


def attention(q, k, v, q_lens, k_lens, scale, k_shared=None):
    """(out, sums of weight * |v|), both [Tq, heads, v_dim] in 64 bits, rows
    outside the sequences NaN. Keys that a query does not see are never read
    for it."""
    Tq, heads, _ = q.shape
    per = heads // k.shape[1]
    out = torch.full((Tq, heads, v.shape[2]), float("nan"), dtype=torch.float64, device=q.device)
    mag = out.clone()
    q0 = k0 = 0
    for n, m in zip(q_lens, k_lens):
        kk = k[k0:k0 + m].double()
        if k_shared is not None:
            kk = torch.cat([kk, k_shared[k0:k0 + m, None].double().expand(-1, k.shape[1], -1)], -1)
        kk = kk.repeat_interleave(per, dim=1)
        vv = v[k0:k0 + m].double().repeat_interleave(per, dim=1)
        for i in range(n):
            seen = i + 1 + m - n
            if seen <= 0:
                out[q0 + i] = 0
                mag[q0 + i] = 0
                continue
            s = torch.einsum("hd,jhd->hj", q[q0 + i].double(), kk[:seen]) * scale
            p = torch.softmax(s, dim=-1)
            out[q0 + i] = torch.einsum("hj,jhd->hd", p, vv[:seen])
            mag[q0 + i] = torch.einsum("hj,jhd->hd", p, vv[:seen].abs())
        q0, k0 = q0 + n, k0 + m
    return out, mag
