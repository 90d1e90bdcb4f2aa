"""The operators over a paged cache and packed prompts on the CPU, at the
ends of what they take."""
import pytest
import torch

import paged_limits as limits
import paged_oracle as oracle
from triton_dist_amd import ops


@pytest.mark.parametrize("name", limits.LARGE)
def test_packed_large_logits(name):
    args, kw, want = limits.packed_large(name)
    out, lse = ops.flash_prefill_packed_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)


@pytest.mark.parametrize("name", limits.LARGE)
def test_decode_large_logits(name):
    args, kw, want = limits.decode_large(name)
    out, lse, mass = ops.paged_decode_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)
    limits.hold_mass(mass, want)


@pytest.mark.parametrize("name", limits.DECODE_WILD)
def test_decode_wild_values(name):
    q, st, kw, want = limits.decode_wild(name)
    out = ops.paged_decode_op(q, st["k"], st["v"], st["table"], st["lens"],
                              **kw)
    oracle.check("out", out[0] if "mass" in kw else out, want["out"])


@pytest.mark.parametrize("name", limits.PACKED_WILD)
def test_packed_wild_values(name):
    args, kw, want = limits.packed_wild(name)
    oracle.check("out", ops.flash_prefill_packed_op(*args, **kw),
                 want["out"])


@pytest.mark.parametrize("name", limits.EVICT_GONE)
def test_evict_where_pages_are_gone(name):
    before, mass, pos, budget, recent, there, kept = limits.evict_gone(name)
    k, v, table, lens = (x.clone() for x in before)
    got = ops.kv_evict_op(k, v, table, lens, mass, pos, budget, recent)
    limits.hold_evicted(before, (k, v), mass, pos, got, budget, there, kept)


def test_decode_after_a_cut_where_a_page_is_gone():
    """An evicted row is not attended to under the name of one that was
    never there."""
    k = torch.zeros(2, 1, 1, 64).bfloat16()
    v = torch.zeros_like(k)
    v[0], v[1] = 5, 7
    table, lens = torch.tensor([[0, 1, -1]]), torch.tensor([3])
    mass, pos = torch.tensor([[[0.0, 5.0, 9.0]]]), torch.arange(3).int()
    pos = pos.view(1, 1, 3)
    lens, mass, pos = ops.kv_evict_op(k, v, table, lens, mass, pos, 1, 0)
    assert pos.tolist() == [[[1, -1, -1]]]
    q = torch.zeros(1, 1, 64).bfloat16()
    assert (ops.paged_decode_op(q, k, v, table, lens) == 7).all()


def _cache_fields(b=1, block=64, kvh=8, width=8):
    """A cache as the native functions take it, at no address."""
    return [0, 0, block * kvh * 64, kvh * 64, 64, block * kvh * 64, kvh * 64,
            64, 1, block, kvh, 64, 0, 0, 0, width, width, 0, 1, b]


@pytest.mark.skipif(torch.cuda.is_available(),
                    reason="what is not refused would run")
@pytest.mark.parametrize("name, args", [
    ("paged_append", (_cache_fields(), 0, 0, 0, 0, 0, 0, 1 << 27, 0, 0, 0, 0,
                      0, 0)),
    ("paged_decode", (_cache_fields(b=1 << 24), 0, 0, 0, 8, 1.0, 0.0, 0, 0,
                      0, 0, 0, 0, 0, 0, 0, 0)),
    # as many slots as there may be without weights, and one of 65535 less
    # than the joins and the spans of 1024 slots need with them
    ("paged_decode", (_cache_fields(kvh=1, width=(65535 - 31) * 16), 0, 0, 0,
                      32, 1.0, 0.0, 0, 0, 0, 0, 0, 0, 1, 1, 0, 0)),
    ("paged_decode", (_cache_fields(kvh=1 << 16), 0, 0, 0, 1 << 16, 1.0, 0.0,
                      0, 0, 0, 0, 0, 0, 0, 0, 0, 0)),
    ("kv_evict", (_cache_fields(b=1 << 22), 0, 0, 5, 1, 0, 0, 0, 0, 0)),
    ("kv_evict", (_cache_fields(width=1 << 17), 0, 0, 1 << 22, 1, 0, 0, 0, 0,
                  0)),
    ("packed_prefill", (0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1 << 30, 1,
                        64, 8, 128, 0, 1, 0, 0, 0, 0, 0, 0, 1, 1, 1.0, 0.0,
                        0, 0)),
])
def test_too_large_for_a_launch(name, args):
    """Refused before anything is launched."""
    from triton_dist_amd import _C

    with pytest.raises(RuntimeError, match="too (large|many)"):
        getattr(_C, name)(*args)


def _pools(kind, n=3, block=4, heads=2, d=16):
    """Pools and whether rows of theirs share memory."""
    store = torch.zeros(4 * n * block * heads * d).bfloat16()
    shape, row = (n, block, heads, d), heads * d
    whole = (block * row, row, d, 1)
    if kind == "apart":
        return torch.zeros(shape).bfloat16(), torch.zeros(shape).bfloat16()
    if kind == "one":
        k = store.as_strided(shape, whole)
        return k, store.as_strided(shape, whole)
    if kind == "heads_side_by_side":
        kv = store[:2 * n * block * row].view(n, block, 2 * heads, d)
        return kv[:, :, :heads], kv[:, :, heads:]
    if kind == "heads_in_turn":
        kv = store[:2 * n * block * row].view(n, block, heads, 2, d)
        return kv[..., 0, :], kv[..., 1, :]
    if kind == "pages_in_turn":
        kv = store[:2 * n * block * row].view(n, 2, block, heads, d)
        return kv[:, 1], kv[:, 0]
    if kind == "head_major":
        kv = store[:2 * n * block * row].view(2, n, heads, block, d)
        return kv[0].transpose(1, 2), kv[1].transpose(1, 2)
    if kind == "one_page_each":  # a stride that nothing steps by
        return store[:block * row].view(1, block, heads, d).expand(
            1, -1, -1, -1), torch.zeros(1, *shape[1:]).bfloat16()
    k = store.as_strided(shape, whole)
    return {
        "a_page_on": lambda: (k, store.as_strided(shape, whole,
                                                  block * row)),
        "a_row_back": lambda: (store.as_strided(shape, whole, row), k),
        "half_a_row_on": lambda: (k, store.as_strided(shape, whole, d // 2)),
        "other_strides": lambda: (k, store.as_strided(
            shape, (row, n * row, d, 1))),
        "expanded_pages": lambda: (k[:1].expand(shape), k.clone()),
        "expanded_heads": lambda: (k.clone(), k[:, :, :1].expand(shape)),
        "folded_rows": lambda: (k.clone(), store.as_strided(
            shape, (block * row, 8, d, 1))),
    }[kind]()


GOOD = ["apart", "one", "heads_side_by_side", "heads_in_turn",
        "pages_in_turn", "head_major", "one_page_each"]
SHARING = ["a_page_on", "a_row_back", "half_a_row_on", "other_strides",
           "expanded_pages", "expanded_heads", "folded_rows"]


@pytest.mark.parametrize("kind", GOOD + SHARING)
def test_pools_that_share_memory(kind):
    """Refused where they are written; reading them is fine."""
    k_pool, v_pool = _pools(kind)
    table, lens = torch.tensor([[0, 2], [1, -1]]), torch.tensor([5, 0])
    if len(k_pool) == 1:
        table = table.clamp(max=0)
    k = torch.randn(2, 2, 16).bfloat16()
    v = k if kind == "one" else torch.randn(2, 2, 16).bfloat16()
    mass = torch.zeros(2, 2, 8)
    calls = [lambda: ops.paged_append_op(k, v, k_pool, v_pool, table, lens),
             lambda: ops.kv_evict_op(k_pool, v_pool, table, lens, mass,
                                     mass.int(), 2, 1)]
    for call in calls:
        if kind in SHARING:
            with pytest.raises(ValueError, match="pool: "):
                call()
        else:
            call()
    if kind in GOOD and kind != "one_page_each":
        ops.paged_append_op(k, v, k_pool, v_pool, table, lens)
        assert torch.equal(k_pool[2, 1], k[0])
        assert torch.equal(v_pool[2, 1], v[0])
        assert torch.equal(k_pool[1, 0], k[1])
        assert torch.equal(v_pool[1, 0], v[1])


def test_pools_in_decode_may_share_memory():
    store = torch.randn(3 * 16 * 64).bfloat16()
    pool = store.view(3, 16, 1, 64)
    q = torch.randn(1, 2, 64).bfloat16()
    table, lens = torch.tensor([[2, 1]]), torch.tensor([20])
    want = ops.paged_decode_op(q, pool, pool.clone(), table, lens)
    assert torch.equal(ops.paged_decode_op(q, pool, pool, table, lens), want)


def test_append_refuses_rows_of_the_pools():
    pool = torch.zeros(3, 4, 2, 16).bfloat16()
    at = (pool, pool.clone(), torch.tensor([[0], [1]]), torch.tensor([0, 0]))
    new = torch.randn(2, 2, 16).bfloat16()
    for k, v in ((pool[2, :2], new), (new, pool[2, :2]),
                 (at[1][2, :2], new), (pool[1:, 0], new)):
        with pytest.raises(ValueError, match="apart from the pools"):
            ops.paged_append_op(k, v, *at)
    ops.paged_append_op(pool[2, :2].clone(), new, *at)
    with pytest.raises(ValueError, match="one k as v"):
        ops.paged_append_op(new, new.clone(), pool, pool, *at[2:])


def test_forward_derivatives_are_refused():
    """Each input that could carry one; the same calls go through without."""
    import torch.autograd.forward_ad as forward

    def call(name, change):
        def f(key, shape, dtype=torch.bfloat16):
            return change(key, torch.zeros(shape, dtype=dtype))
        pools = f("k_pool", (2, 4, 1, 64)), f("v_pool", (2, 4, 1, 64))
        at = torch.tensor([[0, 1]]), torch.tensor([6])
        mass = f("mass", (1, 1, 8), torch.float32)
        slopes = f("slopes", (1,), torch.float32)
        q = f("q", (1, 1, 64))
        if name == "append":
            ops.paged_append_op(f("k", (1, 1, 64)), f("v", (1, 1, 64)),
                                *pools, *at)
        elif name == "decode":
            ops.paged_decode_op(q, *pools, *at, mass=mass, slopes=slopes)
        elif name == "evict":
            ops.kv_evict_op(*pools, *at, mass,
                            torch.zeros(1, 1, 8, dtype=torch.int32), 3, 1)
        else:
            ops.flash_prefill_packed_op(
                q, f("k", (1, 1, 64)), f("v", (1, 1, 64)),
                torch.tensor([0, 1]), slopes=slopes)

    with forward.dual_level():
        for name, keys in (("append", "k v k_pool v_pool"),
                           ("decode", "q k_pool v_pool mass slopes"),
                           ("evict", "k_pool v_pool mass"),
                           ("prefill", "q k v slopes")):
            call(name, lambda key, t: t)
            for which in keys.split():
                with pytest.raises(RuntimeError, match="forward derivative"):
                    call(name, lambda key, t: forward.make_dual(
                        t, torch.ones_like(t)) if key == which else t)
