"""What the serving operators over a paged key-value cache are measured on.

Four operators, in the order in which a serving step calls them:

  prefill  attention of packed prompts: scores capped by a tanh, a bias that
           grows with distance, a document mask, a prefix that is seen whole
  append   the new tokens' keys and values go to their pages
  decode   attention of one new token a sequence over its pages
  evict    the cache is cut to a budget by accumulated attention weight

`own` chooses between the plain form and the framework's kernels.
"""
import random

import torch

own = False

# query heads, key heads, head width: the shards and models that the
# framework's configurations name, and one without shared heads
HEADS = {
    "4/2x64": (4, 2, 64), "8/8x64": (8, 8, 64), "16/2x128": (16, 2, 128),
    "32/4x128": (32, 4, 128), "32/8x128": (32, 8, 128),
    "64/8x128": (64, 8, 128), "80/8x128": (80, 8, 128),
    "8/1x128": (8, 1, 128),
}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 64  # PagedKVCache's own default


def _case(op, name=None, **over):
    case = {"op": op, "heads": "32/8x128", "type": "bf16", "seqs": 1,
            "longest": 1, "ragged": 0, "block": BLOCK, "softcap": 0.0,
            "slopes": False, "prefix": False, "causal": True, "mass": False,
            "moved": False, "single": True, "budget": 0, "recent": 0,
            "tail": 0}
    case.update(over)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a short chat prompt on the small test geometry: launch cost
        _case("prefill", "prefill_short", heads="4/2x64", longest=37),
        # a batch of prompts packed without padding, some with a part that
        # is seen from both sides (a system prompt), scores capped
        _case("prefill", "prefill_packed", heads="64/8x128", seqs=9,
              longest=2048, ragged=11, softcap=30.0, prefix=True, tail=5),
        # one long document, distance bias instead of rotary positions
        _case("prefill", "prefill_long", type="fp16", longest=16384,
              slopes=True),
        # one new token of one chat: launch cost
        _case("append", "append_one", longest=700),
        # keys of a packed batch of prompts go to their pages
        _case("append", "append_prompts", heads="64/8x128", seqs=24,
              longest=4096, ragged=5, single=False),
        # one chat on one card: latency
        _case("decode", "decode_one", longest=700),
        # the large equal batch of offline generation
        _case("decode", "decode_batch", heads="64/8x128", seqs=512,
              longest=131),
        # a serving batch of unlike lengths, ten query heads to a key head
        _case("decode", "decode_ragged", heads="80/8x128", type="fp16",
              seqs=48, longest=16384, ragged=3, softcap=30.0),
        # two very long contexts, distance bias
        _case("decode", "decode_long", heads="64/8x128", seqs=2,
              longest=130001, slopes=True),
        # a cache under a budget: weights are accumulated on the way, and
        # the slots' own positions give the distances
        _case("decode", "decode_mass", heads="32/4x128", seqs=32,
              longest=4100, ragged=2, mass=True, moved=True, slopes=True),
        # the steady state of a cache under a budget: one row goes
        _case("evict", "evict_step", heads="32/4x128", seqs=8,
              longest=1025, budget=1024, recent=128),
        # long prompts are cut to the budget after their prefill
        _case("evict", "evict_prompts", heads="32/4x128", seqs=32,
              longest=8191, ragged=9, budget=2048, recent=256),
    ]


def _span(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["prefill", "append", "decode", "evict"])
    case = _case(op, heads=rng.choice(sorted(HEADS)),
                 type=rng.choice(["bf16", "bf16", "fp16"]),
                 block=rng.choice([16, 32, 64, 64, 128]))
    case["ragged"] = rng.choice([0, rng.randrange(1, 1 << 20)])
    if op == "prefill":
        case["seqs"] = _span(rng, 1, 32)
        case["longest"] = _span(rng, 1, 16384)
        case["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
        case["slopes"] = rng.random() < 0.4
        case["prefix"] = rng.random() < 0.4
        case["causal"] = rng.random() < 0.85
        case["tail"] = rng.choice([0, 0, _span(rng, 1, 100)])
    elif op == "append":
        case["seqs"] = _span(rng, 1, 512)
        case["longest"] = _span(rng, 1, 16384)
        case["single"] = rng.random() < 0.5
    elif op == "decode":
        case["seqs"] = _span(rng, 1, 512)
        case["longest"] = _span(rng, 1, 131072)
        case["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
        case["slopes"] = rng.random() < 0.4
        case["mass"] = rng.random() < 0.4
        case["moved"] = case["mass"] and rng.random() < 0.5
    else:
        case["seqs"] = _span(rng, 1, 64)
        case["longest"] = _span(rng, 64, 16384)
        case["budget"] = max(1, int(case["longest"] * rng.uniform(0.2, 1.0)))
        case["recent"] = rng.randrange(0, case["budget"] + 1)
    top = {"prefill": ("flops", "prefill_long"),
           "append": ("bytes", "append_prompts"),
           "decode": ("bytes", "decode_long"),
           "evict": ("room", "evict_prompts")}[op]
    most = _cost(next(c for c in listed() if c["name"] == top[1]), top[0])
    while _cost(case, top[0]) > most:  # shrink what would cost too much
        if case["seqs"] > 1 and rng.random() < 0.5:
            case["seqs"] = max(1, case["seqs"] * 2 // 3)
        else:
            case["longest"] = max(1, case["longest"] * 2 // 3)
            if op == "evict":
                case["budget"] = max(1, case["budget"] * 2 // 3)
                case["recent"] = min(case["recent"], case["budget"])
    return case


def _cost(case, what):
    if what == "room":  # the pool's rows
        return sum(_lens(case)) * HEADS[case["heads"]][1]
    if what == "flops":  # the plain form forms whole score matrices
        qh, _, d = HEADS[case["heads"]]
        rows = sum(_lens(case)) + case["tail"]
        return 4 * qh * d * rows * rows
    return work(case)[what]


def _lens(case):
    """The sequences' lengths: all `longest`, or spread below it."""
    n, top = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    rng = random.Random(case["ragged"])
    return [top] + [_span(rng, max(1, top // 32), top) for _ in range(n - 1)]


def _prefixes(case):
    """How many leading tokens of each prompt all of its tokens see."""
    rng = random.Random(case["ragged"] + 1)
    return [rng.choice([0, n // 4, n // 2]) if case["prefix"] else 0
            for n in _lens(case)]


def _pairs(case):
    """Query-key pairs that a prompt's mask leaves."""
    total = 0
    for n, p in zip(_lens(case), _prefixes(case)):
        total += n * (n + 1) // 2 + p * (p - 1) // 2 if case["causal"] \
            else n * n
    return total


def work(case):
    qh, kvh, d = HEADS[case["heads"]]
    lens = _lens(case)
    n, seqs = sum(lens), case["seqs"]
    if case["op"] == "prefill":
        return {"bytes": 4 * n * d * (qh + kvh), "flops":
                4 * qh * d * _pairs(case)}
    if case["op"] == "append":
        rows = seqs if case["single"] else n
        return {"bytes": 8 * rows * kvh * d, "flops": 0}
    if case["op"] == "decode":
        size = 4 * n * kvh * d + 4 * seqs * qh * d
        if case["mass"]:  # read, added to and written
            size += 8 * n * kvh
        if case["moved"] and case["slopes"]:
            size += 4 * n * kvh
        return {"bytes": size, "flops": 4 * n * qh * d}
    # evict: weights and positions are read and written; of the rows that
    # stay, the share that sits above the budget moves (read and written)
    size = 0
    for m in lens:
        keep = min(m, case["budget"])
        moved = (m - keep) * (keep / m)
        size += 8 * m + 8 * keep + 8 * moved * d
    return {"bytes": int(size * kvh), "flops": 0}


def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda",
                        dtype=torch.float32) * std).to(dtype)


def _pool(gen, pages, block, kvh, d, dtype):
    pool = torch.empty(pages, block, kvh, d, device="cuda", dtype=dtype)
    step = max(1, (1 << 26) // (block * kvh * d))
    for i in range(0, pages, step):
        part = pool[i:i + step]
        part.copy_(_normal(gen, part.shape, dtype))
    return pool


def _table(rng, lens, block, width):
    """Pages in the order in which a busy allocator hands them out."""
    need = [-(-n // block) for n in lens]
    ids = list(range(sum(need)))
    rng.shuffle(ids)
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int64, device="cuda"), max(at, 1)


def prepare(case, seed):
    qh, kvh, d = HEADS[case["heads"]]
    dtype, block = TYPES[case["type"]], case["block"]
    lens, seqs = _lens(case), case["seqs"]
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    rng = random.Random(seed)
    state = {"case": case, "scale": d ** -0.5}
    state["slopes"] = torch.tensor(
        [2.0 ** (-8.0 * (h + 1) / qh) for h in range(qh)],
        dtype=torch.float32, device="cuda") if case["slopes"] else None
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    cu = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case["op"] == "prefill":
        rows = starts[-1] + case["tail"]
        state.update(
            q=_normal(gen, (rows, qh, d), dtype, 3.0),
            k=_normal(gen, (rows, kvh, d), dtype),
            v=_normal(gen, (rows, kvh, d), dtype), cu=cu,
            prefix=torch.tensor(_prefixes(case), dtype=torch.int32,
                                device="cuda") if case["prefix"] else None)
        return state
    room = lens if case["op"] != "append" or not case["single"] \
        else [n + 1 for n in lens]
    width = -(-max(room) // block) + 1
    table, pages = _table(rng, room, block, width)
    state.update(table=table,
                 k_pool=_pool(gen, pages, block, kvh, d, dtype),
                 v_pool=_pool(gen, pages, block, kvh, d, dtype),
                 lens=torch.tensor(lens, dtype=torch.int64, device="cuda"))
    if case["op"] == "append":
        rows = seqs if case["single"] else starts[-1]
        if not case["single"]:
            state["lens"] = torch.zeros(seqs, dtype=torch.int64,
                                        device="cuda")
            state["cu"] = cu
        # the projection's output as it comes: keys and values side by side
        kv = _normal(gen, (rows, 2 * kvh, d), dtype)
        state.update(k=kv[:, :kvh], v=kv[:, kvh:])
        return state
    room = width * block
    if case["op"] == "decode":
        state["q"] = _normal(gen, (seqs, qh, d), dtype, 3.0)
        if case["mass"]:
            state["mass"] = torch.rand(seqs, kvh, room, generator=gen,
                                       device="cuda")
        if case["moved"]:
            # a cache that has been cut before: positions out of order
            jump = torch.rand(seqs, kvh, room, generator=gen, device="cuda")
            state["key_pos"] = (jump * 2 * room).to(torch.int32)
            state["q_pos"] = torch.full((seqs,), 2 * room,
                                        dtype=torch.int64, device="cuda")
        return state
    # accumulated weights have a heavy tail; some slots never got any
    mass = torch.randn(seqs, kvh, room, generator=gen, device="cuda")
    mass = torch.exp(2.0 * mass)
    mass *= torch.rand(seqs, kvh, room, generator=gen, device="cuda") > 0.1
    slot = torch.arange(room, device="cuda", dtype=torch.int32)
    live = slot < state["lens"].view(-1, 1, 1)
    state["mass"] = torch.where(live, mass, torch.zeros_like(mass))
    state["key_pos"] = torch.where(live, slot, -1).expand(
        seqs, kvh, room).to(torch.int32).contiguous()
    return state


# ------------------------------------------------------------ plain forms
def _capped(s, cap):
    return cap * torch.tanh(s / cap) if cap else s


def _weights(s, seen):
    """Softmax over the last axis where `seen`; rows that see nothing
    weigh nothing."""
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _plain_prefill(st):
    case = st["case"]
    qh, kvh, _ = HEADS[case["heads"]]
    q, k, v, cu = st["q"], st["k"], st["v"], st["cu"]
    rows = q.shape[0]
    at = torch.arange(rows, device=q.device)
    doc = (at[:, None] >= cu[None, 1:]).sum(-1)  # seqs: behind the last
    inside = doc < case["seqs"]
    begin = cu.long()[doc.clamp(max=case["seqs"] - 1)]
    pos = at - begin
    if st["prefix"] is None:
        prefix = torch.zeros_like(pos)
    else:
        prefix = st["prefix"].long()[doc.clamp(max=case["seqs"] - 1)]
    g, d = qh // kvh, q.shape[2]
    # [kvh, d, rows] and [kvh, rows, d], shared by g query heads each
    kf = k.permute(1, 2, 0).float().contiguous()
    vf = v.permute(1, 0, 2).float().contiguous()
    slopes = st["slopes"].view(kvh, g, 1, 1) if case["slopes"] else None
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // (qh * rows))  # 1 GiB of scores at once
    for r in range(0, rows, step):
        e = min(rows, r + step)
        qf = q[r:e].view(e - r, kvh, g, d).permute(1, 2, 0, 3).float()
        s = torch.matmul(qf.reshape(kvh, g * (e - r), d), kf)
        s = _capped(s.view(kvh, g, e - r, rows) * st["scale"],
                    case["softcap"])
        if slopes is not None:
            s = s - slopes * (pos[r:e, None] - pos[None]).abs().float()
        seen = (doc[r:e, None] == doc[None]) & inside[r:e, None]
        if case["causal"]:
            seen &= (pos[None] <= pos[r:e, None]) \
                | (pos[None] < prefix[r:e, None])
        o = torch.matmul(_weights(s, seen).view(kvh, g * (e - r), rows), vf)
        out[r:e] = o.view(qh, e - r, d).transpose(0, 1).to(out.dtype)
    return out


def _plain_append(st):
    k_pool, v_pool, table = st["k_pool"], st["v_pool"], st["table"]
    block, rows = st["case"]["block"], st["k"].shape[0]
    at = torch.arange(rows, device=k_pool.device)
    if st["case"]["single"]:
        seq, slot = at, st["lens"]
    else:
        seq = (at[:, None] >= st["cu"][None, 1:]).sum(-1)
        slot = st["lens"][seq] + at - st["cu"][seq]
    page = table[seq, slot // block]
    k_pool[page, slot % block] = st["k"]
    v_pool[page, slot % block] = st["v"]
    return k_pool, v_pool


def _plain_decode(st):
    case, q, table = st["case"], st["q"], st["table"]
    qh, kvh, d = HEADS[case["heads"]]
    room = table.shape[1] * case["block"]
    slot = torch.arange(room, device=q.device)
    out = torch.empty_like(q)
    mass = torch.zeros_like(st["mass"]) if case["mass"] else None
    step = max(1, (1 << 28) // (room * kvh * d))
    for b in range(0, case["seqs"], step):
        e = min(case["seqs"], b + step)
        n = e - b
        pages = table[b:e].clamp(min=0)
        kf = st["k_pool"][pages].view(n, room, kvh, d).float()
        vf = st["v_pool"][pages].view(n, room, kvh, d).float()
        seen = (slot < st["lens"][b:e, None])[:, None, None]
        vf = torch.where(seen.view(n, room, 1, 1), vf, 0.0)
        qf = q[b:e].view(n, kvh, qh // kvh, d).float()
        s = torch.matmul(qf, kf.permute(0, 2, 3, 1).contiguous())
        s = _capped(s * st["scale"], case["softcap"])
        if st["slopes"] is not None:
            if case["moved"]:
                gap = st["q_pos"][b:e, None, None] - st["key_pos"][b:e]
            else:
                gap = (st["lens"][b:e, None, None] - 1 - slot)
            gap = gap.abs().float()[:, :, None]
            s = s - st["slopes"].view(1, kvh, qh // kvh, 1) * gap
        w = _weights(s, seen)
        o = torch.matmul(w, vf.permute(0, 2, 1, 3).contiguous())
        out[b:e] = o.view(n, qh, d).to(out.dtype)
        if case["mass"]:
            mass[b:e] = torch.where(seen[:, 0], st["mass"][b:e] + w.sum(2),
                                    0.0)
    return (out, mass) if case["mass"] else out


def _plain_evict(st):
    case, lens = st["case"], st["lens"]
    seqs, kvh, room = st["mass"].shape
    budget, recent = case["budget"], case["recent"]
    slot = torch.arange(room, device=lens.device)
    live = slot < lens.view(-1, 1, 1)
    pos = torch.where(live, st["key_pos"], -1)
    newest = pos.amax(-1, keepdim=True)
    score = torch.where(pos > newest - recent, float("inf"), st["mass"])
    score = torch.where(live, score, -1.0)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(live.expand(seqs, kvh, room))
    kept.scatter_(-1, order[..., :budget], True)
    kept &= live
    # the i-th free slot below the budget takes the i-th row above it
    hole = live & ~kept & (slot < budget)
    mover = kept & (slot >= budget)
    none = torch.full_like(order, room)
    holes = torch.sort(torch.where(hole, slot, none), dim=-1).values
    movers = torch.sort(torch.where(mover, slot, none), dim=-1).values
    to, frm = holes[..., :budget], movers[..., :budget]
    # a pair that is not there repeats the first one; where nothing moves,
    # slot 0 is copied onto itself
    none = frm[..., :1] == room
    some = frm < room
    to = torch.where(some, to, torch.where(none, 0, to[..., :1]))
    frm = torch.where(some, frm, torch.where(none, 0, frm[..., :1]))
    block, table = case["block"], st["table"]

    head = torch.arange(kvh, device=lens.device).view(1, -1, 1)

    def rows(at):
        page = torch.gather(table[:, None].expand(-1, kvh, -1), 2,
                            at // block)
        return page, at % block, head

    st["k_pool"][rows(to)] = st["k_pool"][rows(frm)]
    st["v_pool"][rows(to)] = st["v_pool"][rows(frm)]
    new_lens = lens.clamp(max=budget)
    stay = slot < new_lens.view(-1, 1, 1)
    mass, key_pos = st["mass"].clone(), st["key_pos"].clone()
    mass.scatter_(-1, to, torch.gather(st["mass"], -1, frm))
    key_pos.scatter_(-1, to, torch.gather(st["key_pos"], -1, frm))
    mass = torch.where(stay, mass, 0.0)
    key_pos = torch.where(stay, key_pos, -1)
    return st["k_pool"], st["v_pool"], new_lens, mass, key_pos


# ------------------------------------------------------- the framework's
def _own(st):
    from triton_dist_amd import ops

    case = st["case"]
    if case["op"] == "prefill":
        return ops.flash_prefill_packed_op(
            st["q"], st["k"], st["v"], st["cu"], causal=case["causal"],
            prefix_lens=st["prefix"], scale=st["scale"],
            softcap=case["softcap"], slopes=st["slopes"])
    if case["op"] == "append":
        ops.paged_append_op(
            st["k"], st["v"], st["k_pool"], st["v_pool"], st["table"],
            st["lens"], cu_seqlens=None if case["single"] else st["cu"])
        return st["k_pool"], st["v_pool"]
    if case["op"] == "decode":
        return ops.paged_decode_op(
            st["q"], st["k_pool"], st["v_pool"], st["table"], st["lens"],
            scale=st["scale"], softcap=case["softcap"],
            slopes=st["slopes"], key_pos=st.get("key_pos"),
            q_pos=st.get("q_pos"), mass=st.get("mass"))
    lens, mass, key_pos = ops.kv_evict_op(
        st["k_pool"], st["v_pool"], st["table"], st["lens"], st["mass"],
        st["key_pos"], case["budget"], case["recent"])
    return st["k_pool"], st["v_pool"], lens, mass, key_pos


def run(state):
    if own:
        return _own(state)
    return {"prefill": _plain_prefill, "append": _plain_append,
            "decode": _plain_decode, "evict": _plain_evict}[
                state["case"]["op"]](state)


# ------------------------------------------------- the definition, 64 bits
def _attend64(q, k, v, scale, cap, bias, seen):
    """q [m, d], k and v [n, d], bias and seen [m, n] or None, all float64:
    the outputs and the weights."""
    s = torch.mm(q, k.t()).mul_(scale)
    if cap:
        s = torch.tanh(s.div_(cap)).mul_(cap)
    if bias is not None:
        s += bias
    if seen is not None:
        s.masked_fill_(~seen, float("-inf"))
    lse = torch.logsumexp(s, 1, keepdim=True)
    w = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse))
    return torch.mm(w, v), w


def _exact_prefill(st):
    case = st["case"]
    qh, kvh, _ = HEADS[case["heads"]]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for n, p in zip(_lens(case), _prefixes(case)):
        j = torch.arange(n, device="cuda", dtype=torch.float64)
        for h in range(qh):
            g = h // (qh // kvh)
            k = st["k"][start:start + n, g].double()
            v = st["v"][start:start + n, g].double()
            for r in range(0, n, 2048):
                e = min(n, r + 2048)
                i = j[r:e, None]
                bias = -st["slopes"][h].double() * (i - j).abs() \
                    if case["slopes"] else None
                seen = (i >= j) | (j < p) if case["causal"] else None
                q = st["q"][start + r:start + e, h].double()
                out[start + r:start + e, h] = _attend64(
                    q, k, v, st["scale"], case["softcap"], bias, seen)[0]
        start += n
    return out


def _exact_append(st):
    case, block = st["case"], st["case"]["block"]
    k_pool, v_pool = st["k_pool"].clone(), st["v_pool"].clone()
    table = st["table"].cpu()
    row = 0
    for b, n in enumerate(_lens(case)):
        first, count = (n, 1) if case["single"] else (0, n)
        slot = first
        while slot < first + count:
            end = min(first + count, (slot // block + 1) * block)
            page, at, m = int(table[b, slot // block]), slot % block, \
                end - slot
            k_pool[page, at:at + m] = st["k"][row:row + m]
            v_pool[page, at:at + m] = st["v"][row:row + m]
            row, slot = row + m, end
    return k_pool, v_pool


def _exact_decode(st):
    case = st["case"]
    qh, kvh, d = HEADS[case["heads"]]
    g, block = qh // kvh, case["block"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    mass = torch.zeros(st["mass"].shape, dtype=torch.float64,
                       device="cuda") if case["mass"] else None
    for b, n in enumerate(_lens(case)):
        pages = st["table"][b, :-(-n // block)]
        k = st["k_pool"][pages].reshape(-1, kvh, d)[:n].double()
        v = st["v_pool"][pages].reshape(-1, kvh, d)[:n].double()
        j = torch.arange(n, device="cuda", dtype=torch.float64)
        for h in range(kvh):
            bias = None
            if case["slopes"]:
                if case["moved"]:
                    gap = (st["q_pos"][b] - st["key_pos"][b, h, :n]).double()
                else:
                    gap = n - 1 - j
                bias = -st["slopes"][h * g:h * g + g, None].double() * \
                    gap.abs()[None]
            q = st["q"][b, h * g:h * g + g].double()
            o, w = _attend64(q, k[:, h], v[:, h], st["scale"],
                             case["softcap"], bias, None)
            out[b, h * g:h * g + g] = o
            if case["mass"]:
                mass[b, h, :n] = st["mass"][b, h, :n].double() + w.sum(0)
    return (out, mass) if case["mass"] else out


def _exact_evict(st):
    case, block = st["case"], st["case"]["block"]
    budget, recent = case["budget"], case["recent"]
    k_pool, v_pool = st["k_pool"].clone(), st["v_pool"].clone()
    old_mass, old_pos = st["mass"].cpu().numpy(), st["key_pos"].cpu().numpy()
    new_mass, new_pos = old_mass * 0, old_pos * 0 - 1
    lens = _lens(case)
    src, dst = [], []
    table = st["table"].cpu().tolist()
    for b, n in enumerate(lens):
        for h in range(old_mass.shape[1]):
            m, p = old_mass[b, h, :n].tolist(), old_pos[b, h, :n].tolist()
            last = max(p)
            order = sorted(range(n), key=lambda i: (
                p[i] <= last - recent, -m[i] if p[i] <= last - recent else 0,
                i))
            kept = sorted(order[:budget])
            low = [i for i in kept if i < budget]
            free = sorted(set(range(min(n, budget))) - set(low))
            for i in low:
                new_mass[b, h, i], new_pos[b, h, i] = m[i], p[i]
            for i, j in zip(free, kept[len(low):]):
                new_mass[b, h, i], new_pos[b, h, i] = m[j], p[j]
                src.append((table[b][j // block], j % block, h))
                dst.append((table[b][i // block], i % block, h))
    if src:
        frm = torch.tensor(src, device="cuda").t()
        to = torch.tensor(dst, device="cuda").t()
        for old, new in ((st["k_pool"], k_pool), (st["v_pool"], v_pool)):
            new[to[0], to[1], to[2]] = old[frm[0], frm[1], frm[2]]
    return (k_pool, v_pool, torch.tensor([min(n, budget) for n in lens]),
            torch.from_numpy(new_mass), torch.from_numpy(new_pos))


def exact(case, seed):
    state = prepare(case, seed)
    return {"prefill": _exact_prefill, "append": _exact_append,
            "decode": _exact_decode, "evict": _exact_evict}[
                case["op"]](state)
