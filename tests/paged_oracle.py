"""The operators over a paged cache from their definitions, in 64 bits and
one sequence and head at a time, with how far a right answer may be off.

The bounds count roundings, u being half a step of the type: a score of d
products summed in 32 bits is off by ds = (d + 8) 2^-24 sum|q k| |scale| +
2^-21 (|s| + cap + bias) at most, so a weight is off by the factor
exp(2 ds), and a sum of n weights by n 2^-24. An output is rounded once
(u |o|), and its weights may be rounded to the inputs' type before they
meet the values: (u + 2 ds + n 2^-24) sum w|v|.
"""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24


def attend(q, k, v, scale, softcap, bias, dtype):
    """One query over n visible keys, all float64: output, log-sum-exp,
    weights, and the bounds of each."""
    n, d = k.shape
    if n == 0:
        zero = torch.zeros(v.shape[1], dtype=torch.float64)
        return zero, -math.inf, torch.zeros(0, dtype=torch.float64), \
            zero, 0.0, torch.zeros(0, dtype=torch.float64)
    s = (k @ q) * scale
    ds = (d + 8) * F32 * (k.abs() @ q.abs()) * abs(scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s - bias
    ds = ds + 8 * F32 * (s.abs() + softcap + bias.abs())
    top = s.max()
    e = torch.exp(s - top)
    w = e / e.sum()
    lse = float(top + torch.log(e.sum()))
    o = w @ v
    u = HALF_STEP[dtype]
    # a weight that underflows in 32 bits may vanish: 2^-126 each
    off = 2 * ds + 2 * ds.max() + (n + 16) * F32
    o_tol = u * o.abs() + (w * (u + off)) @ v.abs() * 1.02 + 1e-30
    if dtype == torch.float16:  # subnormal steps of the weights and outputs
        o_tol = o_tol + 2.0 ** -25 * (1 + v.abs().sum(0))
    lse_tol = float(2 * ds.max()) + (n + 16) * F32 + 4 * F32 * abs(lse)
    return o, lse, w, o_tol, lse_tol, w * off * 1.02 + 1e-30


def gather(pool, table_row, slots, head):
    """Rows of one sequence's slots and whether their pages are there."""
    block = pool.shape[1]
    slots = torch.tensor(list(slots), dtype=torch.long)
    page = table_row.long()[slots // block]
    there = (page >= 0) & (page < pool.shape[0])
    rows = pool[page[there], slots[there] % block, head].double()
    return rows, there.tolist()


def decode(q, k_pool, v_pool, table, lens, scale=None, softcap=0.0,
           slopes=None, key_pos=None, q_pos=None, mass=None):
    """All on the CPU. Returns {name: (value, bound)}."""
    b, qh, d = q.shape
    kvh, block = k_pool.shape[2], k_pool.shape[1]
    room = table.shape[1] * block
    scale = d ** -0.5 if scale is None else scale
    g = qh // kvh
    out = torch.zeros(b, qh, d, dtype=torch.float64)
    out_tol = torch.zeros_like(out)
    lse = torch.full((b, qh), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    m, m_tol = None, None
    if mass is not None:
        m = mass.double().clone()
        m_tol = 4 * F32 * m.abs()
    for i in range(b):
        n = min(max(int(lens[i]), 0), room)
        if m is not None:
            m[i, :, n:] = 0
            m_tol[i, :, n:] = 0
        for h in range(qh):
            kh = h // g
            k, there = gather(k_pool, table[i], range(n), kh)
            v, _ = gather(v_pool, table[i], range(n), kh)
            at = [s for s, ok in enumerate(there) if ok]
            bias = torch.zeros(len(at), dtype=torch.float64)
            if slopes is not None:
                for x, s in enumerate(at):
                    gap = int(q_pos[i]) - int(key_pos[i, kh, s]) \
                        if key_pos is not None else n - 1 - s
                    bias[x] = float(slopes[h]) * abs(gap)
            o, total, w, ot, lt, wt = attend(
                q[i, h].double(), k, v, scale, softcap, bias, q.dtype)
            out[i, h], out_tol[i, h] = o, ot
            lse[i, h], lse_tol[i, h] = total, lt
            if m is not None and at:
                m[i, kh, at] += w
                m_tol[i, kh, at] += wt + 4 * F32 * g * w
    got = {"out": (out, out_tol), "lse": (lse, lse_tol)}
    if m is not None:
        got["mass"] = (m, m_tol)
    return got


def packed(q, k, v, cu_q, cu_k=None, causal=True, prefix=None, scale=None,
           softcap=0.0, slopes=None):
    """All on the CPU. Rows of no document are zeros and -inf."""
    rows, qh, d = q.shape
    kvh = k.shape[1]
    cu_k = cu_q if cu_k is None else cu_k
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(rows, qh, d, dtype=torch.float64)
    out_tol = torch.zeros_like(out)
    lse = torch.full((rows, qh), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    kd, vd, qd = k.double(), v.double(), q.double()
    for i in range(len(cu_q) - 1):
        q0, q1, k0, k1 = (int(x) for x in (cu_q[i], cu_q[i + 1], cu_k[i],
                                           cu_k[i + 1]))
        m, n = q1 - q0, k1 - k0
        j = torch.arange(n)
        for r in range(m):
            at = r + n - m
            seen = torch.ones(n, dtype=torch.bool)
            if causal:
                seen = j <= at
                if prefix is not None:
                    seen = seen | (j < int(prefix[i]))
            keys = j[seen]
            for h in range(qh):
                kh = h * kvh // qh
                bias = torch.zeros(len(keys), dtype=torch.float64)
                if slopes is not None:
                    bias = float(slopes[h]) * (at - keys).abs().double()
                o, total, _, ot, lt, _ = attend(
                    qd[q0 + r, h], kd[k0 + keys, kh], vd[k0 + keys, kh],
                    scale, softcap, bias, q.dtype)
                out[q0 + r, h], out_tol[q0 + r, h] = o, ot
                lse[q0 + r, h], lse_tol[q0 + r, h] = total, lt
    return {"out": (out, out_tol), "lse": (lse, lse_tol)}


def evict(k_pool, v_pool, table, lens, mass, key_pos, budget, recent):
    """All on the CPU, exactly: the five tensors afterwards."""
    k, v = k_pool.clone(), v_pool.clone()
    block, kvh = k.shape[1], k.shape[2]
    room = table.shape[1] * block
    new_lens, new_mass, new_pos = lens.clone(), mass.clone(), key_pos.clone()
    for i in range(len(lens)):
        n = min(max(int(lens[i]), 0), room)
        keep = min(n, budget)
        for h in range(kvh):
            if n > keep:
                newest = int(key_pos[i, h, :n].max())

                def rank(s):
                    w = float(mass[i, h, s])
                    if int(key_pos[i, h, s]) > newest - recent:
                        return (0, 0.0, s)
                    if math.isnan(w):
                        return (1, 0.0, s)
                    return (2, -w, s)
                kept = set(sorted(range(n), key=rank)[:keep])
                holes = [s for s in range(keep) if s not in kept]
                movers = sorted(s for s in kept if s >= keep)
                assert len(holes) == len(movers)
                for to, frm in zip(holes, movers):
                    new_mass[i, h, to] = mass[i, h, frm]
                    new_pos[i, h, to] = key_pos[i, h, frm]
                    pt, pf = (int(table[i, x // block]) for x in (to, frm))
                    if 0 <= pt < len(k) and 0 <= pf < len(k):
                        k[pt, to % block, h] = k_pool[pf, frm % block, h]
                        v[pt, to % block, h] = v_pool[pf, frm % block, h]
            new_mass[i, h, keep:] = 0
            new_pos[i, h, keep:] = -1
        new_lens[i] = keep
    return k, v, new_lens, new_mass, new_pos


def check(name, got, want):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    same = (got == value) | (torch.isnan(got) & torch.isnan(value))
    off = torch.where(same, torch.zeros_like(value), (got - value).abs())
    worst = off - bound
    bad = ~(worst <= 0) & ~same
    assert not bad.any(), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, first at "
        f"{bad.nonzero()[0].tolist()}: {float(got[bad][0])} for "
        f"{float(value[bad][0])}, {float(off[bad][0]):.3g} over a bound of "
        f"{float(bound[bad][0]):.3g}")
