"""Inputs of the tests of the operators over a paged cache: made on the CPU,
with the places that nothing may read filled with NaN and infinities."""
import torch

import paged_oracle as oracle

BAD = (float("nan"), float("inf"), float("-inf"))


def normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dtype)


def cache(seed, lens, kvh, d, block, dtype=torch.bfloat16, index=torch.int64,
          spare=1, missing=(), wide=0, head_major=False, extra=0):
    """Pools whose pages come in a shuffled order; rows past a length hold
    no numbers, nor do pages of nobody. `missing`: (sequence, page of it)
    without a page. `wide`: columns of the table beside the ones used."""
    gen = torch.Generator().manual_seed(seed)
    b = len(lens)
    need = [-(-(n + extra) // block) for n in lens]
    width = max(need + [1]) + spare
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen)
    shape = (total, block, kvh, d)
    if head_major:
        k = normal(gen, (total, kvh, block, d), dtype).transpose(1, 2)
        v = normal(gen, (total, kvh, block, d), dtype).transpose(1, 2)
    else:
        k, v = normal(gen, shape, dtype), normal(gen, shape, dtype)
    table = torch.full((b, width + wide), -1, dtype=index)
    used = 0
    live = torch.zeros(total, block, dtype=torch.bool)
    for i, n in enumerate(need):
        table[i, :n] = order[used:used + n].to(index)
        for p in range(n):
            rows = min(max(lens[i] - p * block, 0), block)
            live[order[used + p], :rows] = True
        used += n
    for i, p in missing:
        table[i, p] = -1 if (i + p) % 2 else total + 7
    dead = ~live
    fill = torch.tensor(BAD * (int(dead.sum()) // 3 + 1))[:int(dead.sum())]
    k[dead] = fill.to(dtype)[:, None, None]
    v[dead] = fill.flip(0).to(dtype)[:, None, None]
    return {"k": k, "v": v, "table": table[:, :width], "gen": gen,
            "lens": torch.tensor(lens, dtype=index), "room": width * block}


# name: lens, qh, kvh, d, block, and what differs
DECODE = {
    "one": dict(lens=[1], qh=1, kvh=1, d=64, block=16),
    "odd": dict(lens=[0, 1, 15, 16, 17, 33], qh=4, kvh=2, d=64, block=16),
    "ten_to_one": dict(lens=[5, 130, 64], qh=20, kvh=2, d=128, block=64),
    "many_to_one": dict(lens=[40, 7], qh=48, kvh=1, d=128, block=32),
    "sixteen": dict(lens=[100, 0, 31], qh=32, kvh=2, d=64, block=8),
    "fp16": dict(lens=[77, 260], qh=8, kvh=8, d=128, block=64,
                 dtype=torch.float16),
    "long": dict(lens=[1500, 3, 700], qh=8, kvh=2, d=128, block=64),
    "uneven_block": dict(lens=[100, 50], qh=6, kvh=3, d=64, block=7),
    "block_one": dict(lens=[37, 20], qh=2, kvh=1, d=128, block=1),
    "int32": dict(lens=[90, 130], qh=4, kvh=4, d=64, block=16,
                  index=torch.int32),
    "capped": dict(lens=[300, 64], qh=8, kvh=2, d=128, block=32,
                   softcap=2.0, std=4.0),
    "sloped": dict(lens=[513, 128, 1], qh=8, kvh=2, d=64, block=64,
                   slopes=True),
    "both_fp16": dict(lens=[257, 90], qh=10, kvh=2, d=128, block=16,
                      softcap=20.0, slopes=True, dtype=torch.float16),
    "moved": dict(lens=[200, 65], qh=8, kvh=4, d=128, block=64, slopes=True,
                  moved=True, mass=True),
    "mass": dict(lens=[0, 300, 64, 1], qh=10, kvh=2, d=64, block=16,
                 mass=True),
    "mass_many": dict(lens=[129, 5], qh=40, kvh=1, d=128, block=64,
                      mass=True, softcap=5.0),
    "missing": dict(lens=[100, 40, 16], qh=4, kvh=2, d=64, block=16,
                    missing=[(0, 0), (0, 5), (1, 1), (2, 0)], mass=True,
                    slopes=True),
    "head_major": dict(lens=[70, 33], qh=8, kvh=2, d=128, block=32,
                       head_major=True, wide=3),
    "past_room": dict(lens=[64, 32], qh=4, kvh=2, d=64, block=32, spare=0,
                      tell=[1 << 40, -5], mass=True),
    "strong": dict(lens=[400], qh=8, kvh=1, d=128, block=64, std=30.0),
    "no_scale": dict(lens=[50], qh=2, kvh=2, d=64, block=16, scale=0.0),
    "large_cap": dict(lens=[50, 300], qh=2, kvh=2, d=64, block=16,
                      softcap=1000.0),
    "small_cap": dict(lens=[50], qh=2, kvh=2, d=64, block=16, softcap=1e-6),
    "negative": dict(lens=[90, 3], qh=4, kvh=2, d=64, block=16, scale=-0.4),
    "batch": dict(lens=[(i * 37) % 90 for i in range(70)], qh=4, kvh=2,
                  d=64, block=16),
    "big_batch": dict(lens=[(i * 37) % 70 for i in range(515)], qh=3, kvh=3,
                      d=64, block=16, slopes=True),
    "big_ragged": dict(lens=[1900] + [(i * 7) % 5 for i in range(300)]
                       + [700] + [0] * 230, qh=10, kvh=1, d=128, block=64,
                       mass=True),
    "bigger_batch": dict(lens=[(i * 37) % 33 for i in range(1024)] + [700],
                         qh=6, kvh=3, d=64, block=16, mass=True),
    "bigger_ragged": dict(lens=[(i * 97) % 601 for i in range(24)], qh=64,
                          kvh=64, d=64, block=32, slopes=True),
    "bigger_mass": dict(lens=[900, 0, 385, 1, 640, 513, 129, 770], qh=100,
                        kvh=100, d=128, block=64, mass=True, moved=True,
                        slopes=True),
    "bigger_groups": dict(lens=[3000, 2500], qh=2 * 34, kvh=34, d=64,
                          block=64, softcap=9.0),
    "big_heads": dict(lens=[(i * 11) % 40 for i in range(130)], qh=34,
                      kvh=17, d=64, block=8),
}


def decode_inputs(name):
    c = dict(DECODE[name])
    lens, dtype = c["lens"], c.get("dtype", torch.bfloat16)
    st = cache(len(name), lens, c["kvh"], c["d"], c["block"], dtype,
               c.get("index", torch.int64), c.get("spare", 1),
               c.get("missing", ()), c.get("wide", 0),
               c.get("head_major", False))
    gen, b, qh = st.pop("gen"), len(lens), c["qh"]
    room = st.pop("room")
    if "tell" in c:  # what the lengths' tensor says
        st["lens"] = torch.tensor(c["tell"])
    q = normal(gen, (b, qh, c["d"]), dtype, c.get("std", 1.0))
    kw = {"scale": c.get("scale"), "softcap": c.get("softcap", 0.0)}
    if c.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, qh + 1) / qh)
    if c.get("moved"):
        kw["key_pos"] = torch.randint(0, 2 * room, (b, c["kvh"], room),
                                      generator=gen, dtype=torch.int32)
        kw["q_pos"] = torch.full((b,), room)
    if c.get("mass"):
        kw["mass"] = torch.rand(b, c["kvh"], room, generator=gen)
    return q, st, kw


def decode_expected(q, st, kw):
    return oracle.decode(q, st["k"], st["v"], st["table"], st["lens"], **kw)


PACKED = {
    "one": dict(lens=[1], qh=1, kvh=1, d=64),
    "odd": dict(lens=[3, 0, 1, 65, 31], qh=4, kvh=2, d=64),
    "ten_to_one": dict(lens=[33, 40], qh=10, kvh=1, d=128),
    "fp16": dict(lens=[129, 20], qh=4, kvh=4, d=128, dtype=torch.float16),
    "long": dict(lens=[300, 257], qh=4, kvh=1, d=128),
    "long_64": dict(lens=[260, 7], qh=2, kvh=1, d=64),
    "full": dict(lens=[70, 130], qh=2, kvh=2, d=64, causal=False),
    "capped": dict(lens=[140], qh=4, kvh=2, d=128, softcap=2.0, std=4.0),
    "large_cap": dict(lens=[90, 33], qh=2, kvh=1, d=128, softcap=1000.0),
    "small_cap": dict(lens=[90, 33], qh=2, kvh=1, d=64, softcap=1e-6),
    "sloped": dict(lens=[200, 10], qh=8, kvh=2, d=64, slopes=True),
    "prefix": dict(lens=[150, 5, 90], qh=2, kvh=1, d=128,
                   prefix=[70, 99, 0]),
    "all": dict(lens=[130, 66], qh=4, kvh=2, d=128, prefix=[33, 64],
                softcap=10.0, slopes=True, dtype=torch.float16),
    "more_keys": dict(lens=[5, 64, 1], keys=[200, 70, 129], qh=4, kvh=2,
                      d=64, slopes=True),
    "fewer_keys": dict(lens=[150, 8, 4], keys=[20, 0, 4], qh=2, kvh=1,
                       d=128),
    "full_prefix": dict(lens=[70, 30], qh=2, kvh=1, d=64, causal=False,
                        prefix=[20, 0], slopes=True),
    "full_other": dict(lens=[5, 40], keys=[100, 0], qh=2, kvh=1, d=128,
                       causal=False, slopes=True),
    "tail": dict(lens=[40, 9], tail=30, qh=2, kvh=1, d=64),
    "head": dict(lens=[40, 9], head=5, tail=3, qh=2, kvh=1, d=64),
    "strong": dict(lens=[300], qh=2, kvh=1, d=128, std=30.0),
    "steep": dict(lens=[280], qh=2, kvh=1, d=64, slopes=True, steep=40.0),
    "rising": dict(lens=[280], qh=2, kvh=1, d=64, slopes=True, steep=-0.5),
    "strided": dict(lens=[90, 20], qh=4, kvh=2, d=128, strided=True),
    "int64": dict(lens=[9, 80], qh=2, kvh=1, d=64, index=torch.int64,
                  prefix=[3, 200]),
    "wild": dict(lens=[100, 33, 257], qh=4, kvh=2, d=64, wild=True),
    "wild_16": dict(lens=[70, 200], qh=3, kvh=1, d=128, wild=True,
                    dtype=torch.float16, prefix=[65, 20], slopes=True),
    "wild_other": dict(lens=[90, 40], keys=[30, 120], qh=2, kvh=1, d=128,
                       wild=True, softcap=7.0),
    "many": dict(lens=[(i * 29) % 7 for i in range(150)], qh=2, kvh=1, d=64),
    "many_128": dict(lens=[(i * 29) % 5 for i in range(80)] + [90], qh=6,
                     kvh=2, d=128, prefix=[(i * 3) % 4 for i in range(81)]),
    "very_many": dict(lens=[(i * 29) % 4 for i in range(1300)], qh=1, kvh=1,
                      d=64, tail=9),
}


def packed_inputs(name):
    c = dict(PACKED[name])
    gen = torch.Generator().manual_seed(len(name) + 100)
    dtype, qh, kvh, d = c.get("dtype", torch.bfloat16), c["qh"], c["kvh"], \
        c["d"]
    index = c.get("index", torch.int32)
    head, tail = c.get("head", 0), c.get("tail", 0)
    lens, keys = c["lens"], c.get("keys")

    def starts(ns):
        at = [head]
        for n in ns:
            at.append(at[-1] + n)
        return torch.tensor(at, dtype=index), at[-1] + tail

    cu, rows = starts(lens)
    kw = {"causal": c.get("causal", True), "softcap": c.get("softcap", 0.0)}
    nkeys = rows
    if keys is not None:
        kw["cu_seqlens_k"], nkeys = starts(keys)
    if c.get("strided"):  # as a projection leaves them, side by side
        qkv = normal(gen, (rows, qh + 2 * kvh, d), dtype)
        q, k, v = qkv[:, :qh], qkv[:, qh:qh + kvh], qkv[:, qh + kvh:]
    else:
        q = normal(gen, (rows, qh, d), dtype, c.get("std", 1.0))
        k = normal(gen, (nkeys, kvh, d), dtype)
        v = normal(gen, (nkeys, kvh, d), dtype)
    kcu = kw.get("cu_seqlens_k", cu)
    if c.get("wild"):  # late keys of each document, which few queries see
        for e in kcu[1:].tolist():
            k[e - 1, :, ::3] = BAD[0]
            v[e - 1] = BAD[0]
            v[e - 5, :, ::2] = BAD[1]
            v[e - 5, :, 1::4] = BAD[2]
            v[e - 20, -1, 3] = BAD[2]
    for t in (k, v):  # rows of no document hold no numbers
        t[:int(kcu[0])] = BAD[0]
        t[int(kcu[-1]):] = BAD[1]
    if c.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, qh + 1) / qh) \
            * c.get("steep", 1.0)
    if "prefix" in c:
        kw["prefix_lens"] = torch.tensor(c["prefix"], dtype=index)
    return q, k, v, cu, kw


def packed_expected(q, k, v, cu, kw):
    kw = dict(kw)
    return oracle.packed(q, k, v, cu, kw.pop("cu_seqlens_k", None),
                         prefix=kw.pop("prefix_lens", None), **kw)


EVICT = {
    "one_over": dict(lens=[65, 64, 10], kvh=2, budget=64, recent=8),
    "half": dict(lens=[200, 90, 0, 100], kvh=3, budget=100, recent=30),
    "to_one": dict(lens=[130, 1], kvh=1, budget=1, recent=0),
    "all_recent": dict(lens=[150], kvh=2, budget=40, recent=40),
    "ties": dict(lens=[120, 77], kvh=2, budget=50, recent=5, ties=True),
    "special": dict(lens=[100], kvh=2, budget=30, recent=3, special=True),
    "shuffled": dict(lens=[140, 66], kvh=2, budget=60, recent=20,
                     shuffled=True),
    "same_pos": dict(lens=[90], kvh=1, budget=30, recent=30, same=True),
    "wide_row": dict(lens=[90, 70], kvh=1, budget=32, recent=4, d=128,
                     block=64, dtype=torch.float16),
    "thin_row": dict(lens=[40], kvh=2, budget=9, recent=2, d=8, block=3),
    "missing": dict(lens=[100], kvh=2, budget=40, recent=4,
                    missing=[(0, 1), (0, 5)]),
    "long": dict(lens=[5000, 1300], kvh=1, budget=1200, recent=100, d=8,
                 block=128),
    "part_equal": dict(lens=[4097, 16384], kvh=1, budget=4000, recent=50, d=8,
                       block=128, ties=True),
    "very_long": dict(lens=[40000, 16500, 9], kvh=1, budget=16400, recent=300,
                      d=8, block=128),
    "very_long_ties": dict(lens=[36000], kvh=1, budget=17000, recent=0, d=8,
                           block=128, ties=True),
    "roomy": dict(lens=[30, 20], kvh=2, budget=1 << 30, recent=7),
    "past_room": dict(lens=[48], kvh=1, budget=20, recent=3, tell=[1 << 50],
                      spare=0),
}


def evict_inputs(name):
    c = EVICT[name]
    lens, kvh = c["lens"], c["kvh"]
    st = cache(len(name) + 50, lens, kvh, c.get("d", 64), c.get("block", 16),
               c.get("dtype", torch.bfloat16), spare=c.get("spare", 1),
               missing=c.get("missing", ()))
    gen, room, b = st.pop("gen"), st.pop("room"), len(lens)
    if "tell" in c:
        st["lens"] = torch.tensor(c["tell"])
    mass = torch.exp(2 * torch.randn(b, kvh, room, generator=gen))
    if c.get("ties"):
        mass = torch.randint(0, 3, mass.shape, generator=gen).float()
    if c.get("special"):
        odd = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0,
                            -0.0, -1.0, 1e-42])
        mass[..., ::2] = odd[torch.randint(0, 7, mass[..., ::2].shape,
                                           generator=gen)]
    pos = torch.arange(room, dtype=torch.int32).expand(b, kvh, room).clone()
    if c.get("shuffled"):
        pos = torch.stack([torch.stack([
            torch.randperm(room, generator=gen) for _ in range(kvh)])
            for _ in range(b)]).to(torch.int32)
    if c.get("same"):
        pos.zero_()
    return st, mass, pos, c["budget"], c["recent"]
