"""The operators over a paged cache and packed prompts on the GPU, against
their definition in 64 bits, and as a serving loop uses them together."""
import pytest
import torch

import paged_cases as cases
import paged_oracle as oracle
from triton_dist_amd import ops

pytestmark = pytest.mark.gpu


def _gpu(x):
    if isinstance(x, dict):
        return {k: _gpu(v) for k, v in x.items()}
    if isinstance(x, torch.Tensor):  # keeps strides
        y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype,
                                device="cuda")
        return y.copy_(x)
    return x


def _same(x, y):
    x, y = x.cpu(), y.cpu()
    if x.is_floating_point():
        as_int = torch.int32 if x.dtype == torch.float32 else torch.int16
        x, y = x.contiguous().view(as_int), y.contiguous().view(as_int)
    return torch.equal(x, y)


def _decode(q, st, kw, **more):
    return ops.paged_decode_op(q, st["k"], st["v"], st["table"], st["lens"],
                               **kw, **more)


@pytest.mark.parametrize("name", cases.DECODE)
def test_decode(name):
    q, st, kw = cases.decode_inputs(name)
    want = cases.decode_expected(q, st, kw)
    q, st, kw = _gpu(q), _gpu(st), _gpu(kw)
    got = _decode(q, st, kw, return_lse=True)
    for x, key in zip(got, ("out", "lse", "mass")):
        oracle.check(key, x, want[key])
    again = _decode(q, st, kw, return_lse=True)
    assert all(_same(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("name", cases.PACKED)
def test_packed(name):
    args = cases.packed_inputs(name)
    want = cases.packed_expected(*args)
    q, k, v, cu, kw = (_gpu(x) for x in args)
    got = ops.flash_prefill_packed_op(q, k, v, cu, return_lse=True, **kw)
    for x, key in zip(got, ("out", "lse")):
        oracle.check(key, x, want[key])
    again = ops.flash_prefill_packed_op(q, k, v, cu, **kw)
    assert _same(got[0], again)


def test_packed_leaves_rows_of_no_document():
    q, k, v, cu, kw = (_gpu(x) for x in cases.packed_inputs("head"))
    whole = torch.full((q.shape[0], q.shape[1], 2, q.shape[2]), 7.0,
                       dtype=q.dtype, device="cuda")
    out = whole[:, :, 0]  # strided, with rows of nobody between
    got = ops.flash_prefill_packed_op(q, k, v, cu, out=out, **kw)
    assert got is out and (whole[:, :, 1] == 7).all()
    lo, hi = int(cu[0]), int(cu[-1])
    assert (out[:lo] == 7).all() and (out[hi:] == 7).all()
    assert _same(out[lo:hi], ops.flash_prefill_packed_op(
        q, k, v, cu, **kw)[lo:hi])


@pytest.mark.parametrize("cu", [[0, 500], [-3, 20], [10, 5, 40], [0, 20, 9],
                                [30, 40]])
def test_packed_keeps_to_its_rows(cu):
    """Offsets that are not a packing's: nothing outside is touched."""
    whole = torch.randn(3, 40, 2, 64, device="cuda").bfloat16()
    q, k, v = whole[0], whole[1, :, :1], whole[2, :, :1]
    guard = torch.full((80, 2, 64), 7.0, device="cuda").bfloat16()
    ops.flash_prefill_packed_op(
        q[:35], k[:35], v[:35], torch.tensor(cu, device="cuda"),
        out=guard[20:55])
    assert (guard[:20] == 7).all() and (guard[55:] == 7).all()


@pytest.mark.parametrize("name", cases.EVICT)
@pytest.mark.parametrize("inplace", [False, True])
def test_evict(name, inplace):
    st, mass, pos, budget, recent = cases.evict_inputs(name)
    want = oracle.evict(st["k"], st["v"], st["table"], st["lens"], mass, pos,
                        budget, recent)
    st, mass, pos = _gpu(st), _gpu(mass), _gpu(pos)
    before = mass.clone(), pos.clone(), st["lens"].clone()
    got = ops.kv_evict_op(
        st["k"], st["v"], st["table"], st["lens"], mass, pos, budget, recent,
        out=(st["lens"], mass, pos) if inplace else None)
    for x, y in zip((st["k"], st["v"], *got), want):
        assert _same(x, y)
    if not inplace:
        assert all(_same(x, y) for x, y in zip((mass, pos, st["lens"]),
                                               before))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("heads, d, block", [(2, 16, 8), (5, 128, 7),
                                             (8, 64, 64)])
@pytest.mark.parametrize("tell", [None, [-3, 1 << 40, 5, 80]])
def test_append(dtype, single, heads, d, block, tell):
    lens = [5, 16, 0, 63]
    st = cases.cache(3, lens, heads, d, block, dtype, extra=11,
                     missing=[(1, 2)])
    if tell:  # what the lengths' tensor says
        st["lens"] = torch.tensor(tell)
    gen = st["gen"]
    cu = torch.tensor([2, 2, 9, 10, 21])
    rows = 4 if single else 23
    kv = cases.normal(gen, (rows, 2 * heads, d), dtype)
    pos = torch.randint(0, 1000, (rows,), generator=gen, dtype=torch.int32)
    key_pos = torch.full((4, heads, st["room"]), -1, dtype=torch.int32)
    wk, wv, wp = st["k"].clone(), st["v"].clone(), key_pos.clone()
    kw = {} if single else {"cu_seqlens": cu}
    ops.paged_append_op(kv[:, :heads], kv[:, heads:], wk, wv, st["table"],
                        st["lens"], key_pos=wp, pos=pos, **kw)
    g = _gpu(dict(k=st["k"], v=st["v"], t=st["table"], n=st["lens"], p=pos,
                  key_pos=key_pos, kv=kv, **kw))
    ops.paged_append_op(g["kv"][:, :heads], g["kv"][:, heads:], g["k"],
                        g["v"], g["t"], g["n"], key_pos=g["key_pos"],
                        pos=g["p"], **({} if single else
                                       {"cu_seqlens": g["cu_seqlens"]}))
    for x, y in ((g["k"], wk), (g["v"], wv), (g["key_pos"], wp)):
        assert _same(x, y)


@pytest.mark.parametrize("first, lens", [
    (0, [(1 << 63) - 1, 5]), (-(1 << 63), [5, 5]),
    (-(1 << 63), [(1 << 63) - 1] * 2), (-(1 << 40), [-(1 << 63), 16]),
    (-3, [-(1 << 63), 16])])
def test_append_with_any_number(first, lens):
    """Slots that a sum in 64 bits would turn negative are dropped."""
    st = cases.cache(8, [5, 16], 2, 64, 8, extra=9)
    cu = torch.tensor([first, 4, 9])
    k = cases.normal(st["gen"], (9, 2, 64), torch.bfloat16)
    lens = torch.tensor(lens)
    g = _gpu(dict(k=st["k"], v=st["v"], t=st["table"], n=lens, cu=cu, new=k))
    ops.paged_append_op(k, k, st["k"], st["v"], st["table"], lens,
                        cu_seqlens=cu)
    ops.paged_append_op(g["new"], g["new"], g["k"], g["v"], g["t"], g["n"],
                        cu_seqlens=g["cu"])
    assert _same(g["k"], st["k"]) and _same(g["v"], st["v"])


def test_far_pages_need_64_bits():
    """Pages whose rows start past 2^31 elements."""
    block, kvh, d = 64, 8, 128
    pages = (1 << 32) // (block * kvh * d) // 2 + 8  # past 2^31 elements
    k = torch.zeros(pages, block, kvh, d, dtype=torch.bfloat16,
                    device="cuda")
    v = torch.zeros_like(k)
    ids = [pages - 1, 0, pages - 2]
    table = torch.tensor([ids], device="cuda")
    lens = torch.zeros(1, dtype=torch.int64, device="cuda")
    gen = torch.Generator().manual_seed(1)
    new = cases.normal(gen, (150, 2 * kvh, d), torch.bfloat16)
    nk, nv = _gpu(new)[:, :kvh], _gpu(new)[:, kvh:]
    cu = torch.tensor([0, 150], device="cuda")
    ops.paged_append_op(nk, nv, k, v, table, lens, cu_seqlens=cu)
    lens += 150
    q = cases.normal(gen, (1, 8, d), torch.bfloat16)
    small = dict(k=k[ids].cpu(), v=v[ids].cpu())
    want = oracle.decode(q, small["k"], small["v"],
                         torch.tensor([[0, 1, 2]]), [150])
    got = ops.paged_decode_op(q.cuda(), k, v, table, lens)
    oracle.check("out", got, want["out"])
    mass = torch.rand(1, kvh, 192, device="cuda")
    pos = torch.arange(192, dtype=torch.int32,
                       device="cuda").repeat(1, kvh, 1)
    wk, wv, *rest = oracle.evict(
        small["k"], small["v"], torch.tensor([[0, 1, 2]]), lens.cpu(),
        mass.cpu(), pos.cpu(), 40, 4)
    got = ops.kv_evict_op(k, v, table, lens, mass, pos, 40, 4)
    for x, y in zip((k[ids], v[ids], *got), (wk, wv, *rest)):
        assert _same(x, y)


def test_no_sequences_and_no_tokens():
    st = _gpu({k: x for k, x in cases.cache(1, [5], 2, 64, 16).items()
               if isinstance(x, torch.Tensor)})
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    at = (st["k"], st["v"], st["table"][:0], none)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert ops.paged_decode_op(q, *at).shape == (0, 4, 64)
    ops.paged_append_op(q[:, :2], q[:, :2], *at)
    z = torch.zeros(0, 2, 32, device="cuda")
    ops.kv_evict_op(*at, z, z.int(), 4, 1)
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.flash_prefill_packed_op(q, q[:, :2], q[:, :2],
                                       cu).shape == (0, 4, 64)
    # rows, but no document; documents, but no keys
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert (ops.flash_prefill_packed_op(q, q, q, cu) == 0).all()
    two = torch.tensor([0, 3], device="cuda")
    out, lse = ops.flash_prefill_packed_op(
        q, q[:0], q[:0], two, cu_seqlens_k=two * 0, return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()
    # a table without a page
    got = ops.paged_decode_op(q[:1], st["k"], st["v"], st["table"][:, :0],
                              st["lens"]) if st["k"].shape[2] == 2 else None
    assert (got == 0).all()


def _loop(st, mass, key_pos, nxt, q, k, v, budget, slopes):
    """One step of a cache under a budget, all state in place."""
    at = (st["k"], st["v"], st["table"], st["lens"])
    ops.paged_append_op(k, v, *at, key_pos=key_pos, pos=nxt)
    st["lens"] += 1
    out, _ = ops.paged_decode_op(q, *at, slopes=slopes, key_pos=key_pos,
                                 q_pos=nxt, mass=mass, mass_out=mass)
    ops.kv_evict_op(*at, mass, key_pos, budget, 4,
                    out=(st["lens"], mass, key_pos))
    nxt += 1
    return out


def _loop_state(seed):
    lens, kvh, d, block = [40, 17, 0], 2, 64, 16
    st = cases.cache(seed, lens, kvh, d, block, extra=40)
    gen = st.pop("gen")
    room = st.pop("room")
    mass = torch.rand(3, kvh, room, generator=gen)
    pos = torch.arange(room, dtype=torch.int32).repeat(3, kvh, 1)
    for i, n in enumerate(lens):
        mass[i, :, n:], pos[i, :, n:] = 0, -1
    new = [cases.normal(gen, (3, 8, d), torch.bfloat16) for _ in range(8)]
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0])
    return st, mass, pos, st["lens"].clone(), new, slopes


@pytest.mark.parametrize("graph", [False, True])
def test_serving_loop(graph):
    """Append, attend and evict together for some steps, eagerly and as one
    replayed graph, against the CPU's run of the same loop."""
    st, mass, pos, nxt, new, slopes = _loop_state(5)
    g = _gpu(dict(st=st, mass=mass, pos=pos, nxt=nxt))
    gs, buf = _gpu(slopes), _gpu(new[0].clone())

    def step():
        return _loop(g["st"], g["mass"], g["pos"], g["nxt"], buf[:, :4],
                     buf[:, 4:6], buf[:, 6:], 32, gs)

    if graph:
        keep = {k: v.clone() for k, v in (("mass", g["mass"]),
                                          ("pos", g["pos"]),
                                          ("nxt", g["nxt"]), *(
            (k, v) for k, v in g["st"].items()))}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        for k, v in keep.items():
            (g[k] if k in g else g["st"][k]).copy_(v)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            out = step()
    for x in new:
        buf.copy_(x)
        if graph:
            captured.replay()
            torch.cuda.synchronize()
            torch.ones(1000, device="cuda").sum().item()
        else:
            out = step()
        lens = st["lens"].clone()
        # every step starts from the same state: the weights that the GPU
        # accumulated decide what is evicted
        want = oracle.decode(
            x[:, :4], *_appended(st, pos, nxt, x), lens + 1,
            slopes=slopes, key_pos=pos, q_pos=nxt, mass=mass)
        oracle.check("out", out, want["out"])
        at = (st["k"], st["v"], st["table"], lens + 1)
        ek, ev, el, em, ep = oracle.evict(*at, want["mass"][0].float(), pos,
                                          32, 4)
        oracle.check("mass", g["mass"].sort().values,
                     (em.double().sort().values,
                      torch.full(em.shape, 2e-5, dtype=torch.float64)))
        assert _same(g["st"]["lens"], el) and _same(g["pos"], ep)
        assert _same(g["st"]["k"], ek) and _same(g["st"]["v"], ev)
        st["k"], st["v"], st["lens"], pos = ek, ev, el, ep
        mass = g["mass"].cpu()
        nxt += 1
        assert _same(g["nxt"], nxt)


def _appended(st, pos, nxt, x):
    ops.paged_append_op(x[:, 4:6], x[:, 6:], st["k"], st["v"], st["table"],
                        st["lens"], key_pos=pos, pos=nxt)
    return st["k"], st["v"], st["table"]


def test_two_streams_at_once():
    """Two calls of each kind in flight, each with its own workspace."""
    runs = []
    for name in ("moved", "mass_many"):
        q, st, kw = cases.decode_inputs(name)
        want = cases.decode_expected(q, st, kw)
        runs.append((_gpu(q), _gpu(st), _gpu(kw), want,
                     torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for q, st, kw, want, stream in runs:
            with torch.cuda.stream(stream):
                got.append((_decode(q, st, kw), want))
    torch.cuda.synchronize()
    for (out, mass), want in got:
        oracle.check("out", out, want["out"])
        oracle.check("mass", mass, want["mass"])


def test_captured_prefill_follows_its_lengths():
    """One graph of packed prompts, replayed for other packings."""
    gen = torch.Generator().manual_seed(2)
    q = cases.normal(gen, (200, 4, 64), torch.bfloat16)
    k = cases.normal(gen, (200, 2, 64), torch.bfloat16)
    v = cases.normal(gen, (200, 2, 64), torch.bfloat16)
    gq, gk, gv = _gpu(q), _gpu(k), _gpu(v)
    cu = torch.tensor([0, 60, 200], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    ops.flash_prefill_packed_op(gq, gk, gv, cu, prefix_lens=prefix)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.flash_prefill_packed_op(gq, gk, gv, cu, prefix_lens=prefix)
    for starts, pre in (([0, 60, 200], [0, 9]), ([0, 199, 200], [150, 1]),
                        ([0, 0, 31], [4, 4]), ([0, 64, 128], [64, 0])):
        cu.copy_(torch.tensor(starts))
        prefix.copy_(torch.tensor(pre))
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.flash_prefill_packed_op(gq, gk, gv, cu,
                                            prefix_lens=prefix)
        assert _same(out, eager)
        want = oracle.packed(q, k, v, starts, prefix=pre)
        oracle.check("out", out, want["out"])


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_cache_steps(weights, graph):
    """A PagedKVCache through prompts, steps and cuts."""
    import paged_cache_loop

    paged_cache_loop.run("cuda", weights, graph)
