"""Every form that the attention kernels over packed prompts and pages are
built in: type, row, cap and bias crossed, at odd lengths and at long ones.
The bounds are paged_oracle.attend's, a document and head at a time."""
import itertools

import torch

import paged_cases as cases
import paged_limits as limits
import paged_oracle as oracle

F32 = oracle.F32
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCORES = {"plain": {}, "cap": dict(softcap=15.0), "bias": dict(slopes=True),
          "both": dict(softcap=15.0, slopes=True)}

PACKED = {
    f"{t}-{d}-{s}": dict(dtype=TYPES[t], d=d, lens=[77, 130, 1, 33, 257],
                         prefix=[20, 0, 1, 40, 100], qh=6, kvh=2, **SCORES[s])
    for t, d, s in itertools.product(TYPES, (64, 128), SCORES)}
PACKED.update({
    "long-bf16-128": dict(dtype=torch.bfloat16, d=128, lens=[2001, 65],
                          qh=2, kvh=1, slopes=True),
    "long-bf16-64": dict(dtype=torch.bfloat16, d=64, lens=[1987], qh=3,
                         kvh=1, softcap=15.0, slopes=True, prefix=[700]),
    "long-fp16-128": dict(dtype=torch.float16, d=128, lens=[13, 2050], qh=2,
                          kvh=2),
    "long-fp16-64": dict(dtype=torch.float16, d=64, lens=[2011], qh=2, kvh=1,
                         softcap=15.0, causal=False),
    "long-fp16-64-bias": dict(dtype=torch.float16, d=64, lens=[1500, 500],
                              qh=2, kvh=1, slopes=True),
})


def packed(name):
    c = PACKED[name]
    gen = torch.Generator().manual_seed(len(name))
    dtype, d, qh, kvh = c["dtype"], c["d"], c["qh"], c["kvh"]
    starts = torch.tensor([0] + c["lens"]).cumsum(0)
    rows = int(starts[-1])
    q = cases.normal(gen, (rows, qh, d), dtype, 3.0)
    k = cases.normal(gen, (rows, kvh, d), dtype)
    v = cases.normal(gen, (rows, kvh, d), dtype)
    cap, causal = c.get("softcap", 0.0), c.get("causal", True)
    kw = dict(softcap=cap, causal=causal)
    if c.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, qh + 1) / qh)
    if "prefix" in c:
        kw["prefix_lens"] = torch.tensor(c["prefix"])
    out = torch.zeros(rows, qh, d, dtype=torch.float64)
    lse = torch.zeros(rows, qh, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    u, scale = oracle.HALF_STEP[dtype], d ** -0.5
    for i, n in enumerate(c["lens"]):
        a, e = int(starts[i]), int(starts[i + 1])
        at, j, seen = limits.seen_by(n, n, causal,
                                     c.get("prefix", [0] * 9)[i])
        for h in range(qh):
            x = q[a:e, h].double()
            y, z = (t[a:e, h * kvh // qh].double() for t in (k, v))
            s = x @ y.t() * scale
            off = (d + 8) * F32 * (x.abs() @ y.abs().t()) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            if "slopes" in kw:
                bias = float(kw["slopes"][h]) * (at - j).abs().double()
                s = s - bias
                off += 8 * F32 * bias
            off += 8 * F32 * (s.abs() + cap)
            off = torch.where(seen, off, 0.0)
            s = torch.where(seen, s, float("-inf"))
            w = torch.softmax(s, 1)
            most = off.max(1, keepdim=True).values
            many = seen.sum(1, keepdim=True)
            out[a:e, h] = w @ z
            lse[a:e, h] = torch.logsumexp(s, 1)
            off = u + 2 * off + 2 * most + (many + 16) * F32
            out_tol[a:e, h] = u * out[a:e, h].abs() + 1e-30 \
                + 1.02 * (w * off) @ z.abs()
            if dtype == torch.float16:  # steps of outputs and lifted weights
                out_tol[a:e, h] += 2.0 ** -25 \
                    + 2.0 ** -34 * seen.double() @ z.abs()
            lse_tol[a:e, h] = (2 * most + (many + 16) * F32)[:, 0] \
                + 4 * F32 * lse[a:e, h].abs()
    return (q, k, v, starts), kw, {"out": (out, out_tol),
                                   "lse": (lse, lse_tol)}


DECODE = {
    f"{t}-{d}-{s}{m}": dict(dtype=TYPES[t], d=d, mass=bool(m),
                            lens=[700, 0, 33, 1300], **SCORES[s])
    for t, d, s, m in itertools.product(TYPES, (64, 128), SCORES,
                                        ("", "-mass"))}

# key heads and keys enough that waves share no chunk
DECODE.update({
    f"many-{t}-{d}": dict(dtype=TYPES[t], d=d, mass=True, qh=64, kvh=64,
                          lens=[900, 0, 1300, 2001, 1500, 700],
                          **SCORES["both"])
    for t, d in itertools.product(TYPES, (64, 128))})


def decode(name):
    c = DECODE[name]
    qh, kvh = c.get("qh", 6), c.get("kvh", 2)
    st = cases.cache(len(name), c["lens"], kvh, c["d"], 32, c["dtype"])
    gen, b = st.pop("gen"), len(c["lens"])
    q = cases.normal(gen, (b, qh, c["d"]), c["dtype"], 3.0)
    kw = dict(softcap=c.get("softcap", 0.0))
    if c.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, qh + 1) / qh)
    room = st.pop("room")
    if c["mass"]:
        kw["mass"] = torch.rand(b, kvh, room, generator=gen)
    return q, st, kw, cases.decode_expected(q, st, kw)
