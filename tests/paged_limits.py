"""Inputs at the ends of what the operators over a paged cache and packed
prompts take, and what a right answer is there."""
import torch

import paged_cases as cases
import paged_oracle as oracle

F32 = oracle.F32


def whole(gen, shape, dtype, size=1.0):
    """Whole numbers from -4 to 4, times a power of two: their products add
    up without a rounding in 32 bits."""
    return (torch.randint(-4, 5, shape, generator=gen) * size).to(dtype)


def seen_by(m, n, causal, prefix):
    at, j = torch.arange(m)[:, None] + n - m, torch.arange(n)
    if not causal:
        return at, j, torch.ones(m, n, dtype=torch.bool)
    return at, j, (j <= at) | (j < prefix)


def pick(s, off, seen, v, dtype):
    """Scores s [m, n] in 64 bits, which 32 bits hold to `off`, over values
    v [n, d]: the least and largest output that scores so far off can give.
    Other keys than those within 60 of the top weigh e^-60 at most. Where
    `off` is 0 the keys at the top share it evenly, if no other is near."""
    s = torch.where(seen, s, float("-inf"))
    top, at = s.max(1, keepdim=True)
    slack = off + off.gather(1, at)
    near = seen & (s >= top - slack - 60)
    even = ((s == top) == near).all() and not off.any()
    low = torch.empty(len(s), v.shape[1], dtype=torch.float64)
    high = low.clone()
    for r in range(len(s)):
        x = v[near[r]]
        if even:
            low[r] = high[r] = x.mean(0)
        else:
            low[r], high[r] = x.min(0).values, x.max(0).values
        # a weight and the output are rounded once each
        tol = (2 * oracle.HALF_STEP[dtype] + 2 * len(s[0]) * F32) \
            * x.abs().mean(0) if even else \
            2 * oracle.HALF_STEP[dtype] * x.abs().max(0).values
        low[r] -= tol + 1e-12
        high[r] += tol + 1e-12
    return low, high, torch.logsumexp(s, 1), slack[:, 0]


# name: type, d, scale, size of q and k, slope, cap, causal
LARGE = {
    "below": (torch.bfloat16, 64, 3e3, 1, 0.0, 0.0, True),
    "about": (torch.float16, 128, -2e4, 1, 0.0, 0.0, True),
    "million": (torch.bfloat16, 128, 1e6, 1, 0.0, 0.0, False),
    "1e8": (torch.bfloat16, 64, 1e8, 1, 0.0, 0.0, True),
    "-1e10": (torch.bfloat16, 128, -1e10, 1, 0.0, 0.0, True),
    "1e30": (torch.float16, 128, 1e30, 1, 0.0, 0.0, True),
    "1e30_64": (torch.float16, 64, 1e30, 1, 0.0, 0.0, False),
    "inputs": (torch.bfloat16, 128, 1.0, 2.0 ** 40, 0.0, 0.0, True),
    "inputs_16": (torch.float16, 64, 1.0, 1024, 0.0, 0.0, True),
    "both": (torch.bfloat16, 64, 1e8, 1, 1e8, 0.0, True),
    "both_16": (torch.float16, 128, 1e10, 1, 3e9, 0.0, True),
    "slope": (torch.bfloat16, 128, 1.0, 1, 1e9, 0.0, False),
    "slope_16": (torch.float16, 64, 0.5, 1, 1e12, 0.0, True),
    "capped": (torch.bfloat16, 64, 1.0, 1, 1e9, 30.0, True),
    "capped_16": (torch.float16, 128, 1.0, 1, 1e7, 50.0, False),
    "flat": (torch.bfloat16, 128, 1e9, 1, 1.0, 0.0, True),
    "cap_alone": (torch.bfloat16, 64, 1e9, 1, 0.0, 1000.0, True),
}


def scores(q, k, scale, cap, bias):
    """In 64 bits, and how far 32 bits may be off: whole numbers' products
    are exact, and a scale alone keeps their order and what is equal."""
    s = (q.double() @ k.double().t()) * scale
    off = torch.zeros_like(s)
    if cap:
        s = cap * torch.tanh(s / cap)
        off += 8 * F32 * cap
    if bias is not None:
        off += 16 * F32 * (s.abs() + bias.abs())
        s = s - bias
    return s, off


def packed_large(name):
    """Two documents; returns the call's arguments and what to hold the
    outputs against."""
    dtype, d, scale, size, slope, cap, causal = LARGE[name]
    gen = torch.Generator().manual_seed(len(name))
    lens, qh, kvh = [300, 65], 4, 2
    rows = sum(lens)
    q = whole(gen, (rows, qh, d), dtype, size)
    k = whole(gen, (rows, kvh, d), dtype, size)
    v = torch.randn(rows, kvh, d, generator=gen).to(dtype)
    prefix = torch.tensor([0, 40], dtype=torch.int32)
    cu = torch.tensor([0, 300, 365], dtype=torch.int32)
    kw = dict(scale=scale, softcap=cap, causal=causal, prefix_lens=prefix)
    if slope:
        kw["slopes"] = slope * 2.0 ** -torch.arange(qh)
    want = {x: torch.zeros(rows, qh, d, dtype=torch.float64)
            for x in ("low", "high")}
    want["lse"] = torch.zeros(rows, qh, dtype=torch.float64)
    want["off"] = torch.zeros_like(want["lse"])
    for i, n in enumerate(lens):
        a, e = int(cu[i]), int(cu[i + 1])
        at, j, seen = seen_by(n, n, causal, int(prefix[i]))
        for h in range(qh):
            bias = float(kw["slopes"][h]) * (at - j).abs().double() \
                if slope else None
            s, off = scores(q[a:e, h], k[a:e, h * kvh // qh], scale, cap,
                            bias)
            low, high, lse, slack = pick(
                s, off, seen, v[a:e, h * kvh // qh].double(), dtype)
            want["low"][a:e, h], want["high"][a:e, h] = low, high
            want["lse"][a:e, h], want["off"][a:e, h] = lse, slack
    return (q, k, v, cu), kw, want


def hold(out, lse, want):
    out, lse = out.detach().cpu().double(), lse.detach().cpu().double()
    ok = (out >= want["low"]) & (out <= want["high"])
    bad = (~ok).nonzero()
    assert not len(bad), (
        f"{len(bad)} of {ok.numel()}, first at {bad[0].tolist()}: "
        f"{float(out[~ok][0])}, not from {float(want['low'][~ok][0])} to "
        f"{float(want['high'][~ok][0])}")
    tol = 8 * F32 * want["lse"].abs() + want["off"] + 1e-5
    assert ((lse == want["lse"]) | ((lse - want["lse"]).abs() <= tol)).all()


def decode_large(name):
    """Three sequences, one of them of many chunks with ties in several, and
    what their outputs and weights have to be."""
    dtype, d, scale, size, slope, cap, _ = LARGE[name]
    gen = torch.Generator().manual_seed(len(name) + 7)
    lens, qh, kvh, block = [2500, 0, 130], 6, 2, 64
    need = [-(-n // block) for n in lens]
    width = max(need) + 1
    table = torch.full((len(lens), width), -1)
    ids = torch.randperm(sum(need), generator=gen)
    table[0, :need[0]], table[2, :need[2]] = ids[:need[0]], ids[need[0]:]
    k = whole(gen, (len(ids), block, kvh, d), dtype, size)
    v = torch.randn(len(ids), block, kvh, d, generator=gen).to(dtype)
    q = whole(gen, (len(lens), qh, d), dtype, size)
    # the last key of all and some before it hold the same row
    for i, n in enumerate(lens):
        for s in range(n - 1, 0, -700):
            k[table[i, s // block], s % block] = \
                q[i, ::qh // kvh] if scale > 0 else -q[i, ::qh // kvh]
    kw = dict(scale=scale, softcap=cap,
              mass=torch.rand(len(lens), kvh, width * block, generator=gen))
    if slope:
        kw["slopes"] = slope * 2.0 ** -torch.arange(qh)
    want = {x: torch.zeros(len(lens), qh, d, dtype=torch.float64)
            for x in ("low", "high")}
    want["lse"] = torch.full((len(lens), qh), -float("inf"),
                             dtype=torch.float64)
    want["off"] = torch.zeros_like(want["lse"])
    want["mass"] = kw["mass"].double().clone()
    want["even"] = not slope and not cap
    want["sums"] = torch.full((len(lens), kvh), float(qh // kvh),
                              dtype=torch.float64)
    for i, n in enumerate(lens):
        want["mass"][i, :, n:] = 0
        want["sums"][i] = want["mass"][i].sum(-1) + (qh // kvh if n else 0)
        for h in range(qh if n else 0):
            kh = h * kvh // qh
            rows = table[i, :need[i]]
            bias = None
            if slope:
                bias = float(kw["slopes"][h]) \
                    * (n - 1 - torch.arange(n)).double()[None]
            s, off = scores(q[i, h:h + 1],
                            k[rows].reshape(-1, kvh, d)[:n, kh], scale, cap,
                            bias)
            low, high, lse, slack = pick(
                s, off, torch.ones(1, n, dtype=torch.bool),
                v[rows].reshape(-1, kvh, d)[:n, kh].double(), dtype)
            want["low"][i, h], want["high"][i, h] = low[0], high[0]
            want["lse"][i, h], want["off"][i, h] = lse[0], slack[0]
            want["mass"][i, kh, :n] += torch.softmax(s[0], 0)
    args = (q, k, v, table, torch.tensor(lens))
    return args, kw, want


def hold_mass(mass, want):
    """Each query head hands out a weight of one in all; where the scores
    are exact, by the definition."""
    mass = mass.detach().cpu().double()
    assert ((mass.sum(-1) - want["sums"]).abs()
            <= 2 * mass.shape[-1] * F32 * (1 + want["sums"])).all()
    if want["even"]:
        # equal keys share evenly, others get nothing: a few roundings
        assert ((mass - want["mass"]).abs()
                <= 64 * F32 * (1 + want["mass"])).all()


def plant(rows):
    """Infinities and NaN into rows [n, ...] of values that are seen."""
    n = len(rows)
    rows[n - 1, ..., ::7] = float("inf")
    rows[n // 2, ..., 5::16] = float("nan")
    rows[0, ..., 3::11] = -float("inf")


def wild_sums(v, seen):
    """What values v [n, d] that are not finite make of outputs whose keys
    are `seen` [m, n], whatever the weights; 0 where there are none."""
    wild = torch.where(torch.isfinite(v), 0.0, v.double())
    total = torch.zeros(len(seen), v.shape[1], dtype=torch.float64)
    for j in wild.ne(0).any(1).nonzero()[:, 0].tolist():
        total[seen[:, j]] += wild[j]
    return total


# cases of decode whose chunks are cut alike and unlike, and one whose
# weights mostly underflow
DECODE_WILD = ["odd", "ten_to_one", "sixteen", "fp16", "long", "sloped",
               "moved", "mass", "missing", "head_major", "strong",
               "bigger_mass", "bigger_groups", "big_ragged"]


def decode_wild(name):
    q, st, kw = cases.decode_inputs(name)
    k, v, table, lens = st["k"], st["v"], st["table"], st["lens"]
    n_blocks, block, kvh, d = v.shape
    calm = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    for b in range(len(lens)):  # the oracle has its rows without them
        slots = torch.arange(int(lens[b]))
        page = table[b].long()[slots // block]
        there = (page >= 0) & (page < n_blocks)
        if there.any():
            at = page[there], slots[there] % block
            rows = v[at].clone()
            plant(rows)
            v[at] = rows
    want = oracle.decode(q, k, calm, table, lens, **kw)
    out = want["out"][0]
    for b in range(len(lens)):
        for h in range(q.shape[1]):
            rows, _ = oracle.gather(v, table[b], range(int(lens[b])),
                                    h * kvh // q.shape[1])
            more = wild_sums(rows, torch.ones(1, len(rows)).bool())[0]
            out[b, h] = torch.where(more == 0, out[b, h], more)
    return q, st, kw, want


PACKED_WILD = ["odd", "ten_to_one", "fp16", "long", "full", "capped",
               "prefix", "all", "more_keys", "fewer_keys", "tail", "strong",
               "steep", "rising", "wild_16", "many_128"]


def packed_wild(name):
    q, k, v, cu, kw = cases.packed_inputs(name)
    kcu = kw.get("cu_seqlens_k", cu)
    docs = range(len(cu) - 1)
    calm = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    for i in docs:
        a, e = int(kcu[i]), int(kcu[i + 1])
        if a < e:
            plant(v[a:e])
    want = cases.packed_expected(q, k, calm, cu, kw)
    out = want["out"][0]
    for i in docs:
        q0, q1, k0, k1 = (int(x) for x in (cu[i], cu[i + 1], kcu[i],
                                           kcu[i + 1]))
        p = int(kw["prefix_lens"][i]) if "prefix_lens" in kw else 0
        _, _, seen = seen_by(q1 - q0, k1 - k0, kw["causal"], p)
        for h in range(q.shape[1]):
            more = wild_sums(v[k0:k1, h * k.shape[1] // q.shape[1]], seen)
            # where a score is none, nothing else counts
            out[q0:q1, h] = torch.where((more == 0) | out[q0:q1, h].isnan(),
                                        out[q0:q1, h], more)
    return (q, k, v, cu), kw, want


# many keys of a small weight beside a few of a large one that hold zeros:
# d, keys, steps of 2 of the small weight, and how the large ones come
FAINT = {
    "first": (64, 700, 25.5, "first"), "last": (128, 700, 25.5, "last"),
    "rising": (64, 900, 22.0, "rising"), "fainter": (128, 3000, 28.0,
                                                     "first"),
    "mild": (64, 500, 15.5, "last"),
}


def faint(name):
    """fp16: one query head of two sees `n` keys. Returns q [1, 2, d], k and
    v [n, 1, d], the outputs and how far each kernel's may be off them: a
    weight is held to a step of 2^-24 after it was lifted by `lift`."""
    d, n, down, how = FAINT[name]
    log2 = 0.6931471805599453
    q = torch.zeros(1, 2, d, dtype=torch.float16)
    q[0, :, 0] = 1
    gen = torch.Generator().manual_seed(n)
    k = torch.zeros(n, 1, d, dtype=torch.float16)
    v = (30000 + 30000 * torch.rand(n, 1, d, generator=gen)).half()
    k[:, 0, 0] = -down * log2
    top = {"first": [(0, 0.0)], "last": [(n - 1, 0.0)],
           "rising": [(0, -5.5), (n // 3, -2.75), (n - 1, 0.0)]}[how]
    for at, value in top:
        k[at, 0, 0] = value * log2
        v[at] = 0
    w = torch.softmax(k[:, 0, 0].double(), 0)
    out = (w @ v[:, 0].double())[None, None].expand(1, 2, d)

    def tol(lift):
        u = oracle.HALF_STEP[torch.float16]
        off = u + 2 * (d + 32) * F32 * down + (n + 16) * F32
        return u * out.abs() + off * out.abs() \
            + 2.0 ** (-25 - lift) * v[:, 0].double().sum(0)

    return q, k, v, out, tol


# block, budget, recent, pages that are not there, and what is kept of 100
EVICT_GONE = {
    "few": (16, 40, 4, [1, 5]), "first": (8, 90, 10, [0]),
    "recent_gone": (16, 30, 20, [5, 6]), "most": (4, 40, 8, range(0, 25, 2)),
    "more_than_budget": (4, 80, 8, [0, 3, 7, 9, 12, 20, 24]),
    "nearly_all": (8, 20, 4, range(1, 13)), "all": (8, 20, 4, range(13)),
    "block_one": (1, 37, 9, range(0, 100, 3)),
}


def evict_gone(name, n=100, heads=2):
    """A sequence some of whose pages are not there, and the slots that
    stay: present ones by age and weight, then the others by number."""
    block, budget, recent, gone = EVICT_GONE[name]
    gen = torch.Generator().manual_seed(len(name))
    pages = -(-n // block)
    table = torch.randperm(pages, generator=gen)[None].clone()
    for p in gone:
        table[0, p] = -1 if p % 2 else pages + 5
    room = pages * block
    k = torch.randn(pages, block, heads, 64, generator=gen).bfloat16()
    v = torch.randn(pages, block, heads, 64, generator=gen).bfloat16()
    mass = torch.rand(1, heads, room, generator=gen)
    mass[..., ::9] = float("nan")
    pos = torch.randperm(room, generator=gen).int().repeat(1, heads, 1)
    there = [0 <= int(table[0, s // block]) < pages for s in range(n)]
    kept = []
    for h in range(heads):
        newest = int(pos[0, h, :n].max())

        def rank(s):
            m = float(mass[0, h, s])
            if not there[s]:
                return 3, 0, s
            if int(pos[0, h, s]) > newest - recent:
                return 0, 0, s
            return (1, 0, s) if m != m else (2, -m, s)
        kept.append(sorted(sorted(range(n), key=rank)[:budget]))
    return (k, v, table, torch.tensor([n])), mass, pos, budget, recent, \
        there, kept


def hold_evicted(before, after, mass, pos, got, budget, there, kept):
    """Every slot that has a row now holds a kept row, its weight and its
    position, and no kept row that a present slot is named for is another's."""
    k, v, table, _ = before
    gk, gv = after
    lens, new_mass, new_pos = (x.cpu() for x in got)
    assert lens.tolist() == [budget]
    block = k.shape[1]

    def row(pool, h, s):
        return pool[table[0, s // block], s % block, h]

    for h, slots in enumerate(kept):
        stay = [s for s in slots if s < budget]
        holes = [s for s in range(budget) if s not in slots]
        movers = [s for s in slots if s >= budget]
        of = dict(zip(stay + holes, stay + movers))
        for s in range(budget):
            at = of[s]
            assert int(new_pos[0, h, s]) == int(pos[0, h, at])
            x, y = float(new_mass[0, h, s]), float(mass[0, h, at])
            assert x == y or x != x and y != y
            if there[s]:  # then what it holds is the row it is named for
                assert there[at]
                assert torch.equal(row(gk.cpu(), h, s), row(k, h, at))
                assert torch.equal(row(gv.cpu(), h, s), row(v, h, at))
        assert (new_mass[0, h, budget:] == 0).all()
        assert (new_pos[0, h, budget:] == -1).all()
