"""The operators over a paged cache and packed prompts on the CPU: values
against their definition in 64 bits, and what they refuse."""
import pytest
import torch

import paged_cases as cases
import paged_oracle as oracle
from triton_dist_amd import ops


@pytest.mark.parametrize("name", cases.DECODE)
def test_decode(name):
    q, st, kw = cases.decode_inputs(name)
    got = ops.paged_decode_op(q, st["k"], st["v"], st["table"], st["lens"],
                              return_lse=True, **kw)
    want = cases.decode_expected(q, st, kw)
    for x, key in zip(got, ("out", "lse", "mass")):
        oracle.check(key, x, want[key])


@pytest.mark.parametrize("name", cases.PACKED)
def test_packed(name):
    q, k, v, cu, kw = cases.packed_inputs(name)
    got = ops.flash_prefill_packed_op(q, k, v, cu, return_lse=True, **kw)
    want = cases.packed_expected(q, k, v, cu, kw)
    for x, key in zip(got, ("out", "lse")):
        oracle.check(key, x, want[key])


@pytest.mark.parametrize("name", cases.EVICT)
def test_evict(name):
    st, mass, pos, budget, recent = cases.evict_inputs(name)
    want = oracle.evict(st["k"], st["v"], st["table"], st["lens"], mass, pos,
                        budget, recent)
    got = ops.kv_evict_op(st["k"], st["v"], st["table"], st["lens"], mass,
                          pos, budget, recent)
    for x, y in zip((st["k"], st["v"], *got), want):
        assert torch.equal(x.view(torch.int16) if x.dtype in
                           oracle.HALF_STEP else x,
                           y.view(torch.int16) if y.dtype in
                           oracle.HALF_STEP else y) or (
            x.dtype == torch.float32
            and torch.equal(x.view(torch.int32), y.view(torch.int32)))


def test_append_single_and_packed():
    st = cases.cache(3, [5, 16, 0], 2, 16, 8, extra=9)
    k = torch.randn(3, 2, 16).bfloat16()
    pos = torch.tensor([50, 60, 70])
    key_pos = torch.full((3, 2, st["room"]), -1, dtype=torch.int32)
    ops.paged_append_op(k, -k, st["k"], st["v"], st["table"], st["lens"],
                        key_pos=key_pos, pos=pos)
    for b in range(3):
        s = int(st["lens"][b])
        page = st["table"][b, s // 8]
        assert torch.equal(st["k"][page, s % 8], k[b])
        assert torch.equal(st["v"][page, s % 8], -k[b])
        assert key_pos[b, :, s].tolist() == [int(pos[b])] * 2
    assert int((key_pos >= 0).sum()) == 6
    cu = torch.tensor([1, 4, 4, 13], dtype=torch.int32)
    k = torch.randn(15, 2, 16).bfloat16()
    before = st["k"].clone()
    ops.paged_append_op(k, k, st["k"], st["v"], st["table"], st["lens"],
                        cu_seqlens=cu)
    changed = 0
    for b in range(3):
        for i in range(int(cu[b]), int(cu[b + 1])):
            s = int(st["lens"][b]) + i - int(cu[b])
            page = int(st["table"][b, s // 8])
            if page < 0:
                continue
            assert torch.equal(st["k"][page, s % 8], k[i])
            changed += 1
    same = (st["k"].view(torch.int16) == before.view(torch.int16)).all(-1)
    assert int((~same.all(-1)).sum()) == changed


def _decode_args():
    st = cases.cache(1, [5, 20], 2, 64, 16)
    q = torch.randn(2, 4, 64).bfloat16()
    return [q, st["k"], st["v"], st["table"], st["lens"]], st["room"]


@pytest.mark.parametrize("change, words", [
    (dict(at=0, to=lambda t: t.half()), "bfloat16"),
    (dict(at=0, to=lambda t: t[:1]), "q: "),
    (dict(at=0, to=lambda t: t[:, :3]), "multiple"),
    (dict(at=0, to=lambda t: t.transpose(1, 2).contiguous()
          .transpose(1, 2)), "contiguous"),
    (dict(at=1, to=lambda t: t.float()), "bfloat16 or float16"),
    (dict(at=2, to=lambda t: t[:1]), "v_pool"),
    (dict(at=3, to=lambda t: t.float()), "int32 or int64"),
    (dict(at=3, to=lambda t: t.t().contiguous().t()), "rows"),
    (dict(at=4, to=lambda t: t[:1]), "seq_lens"),
    (dict(kw=dict(softcap=-1.0)), "softcap"),
    (dict(kw=dict(softcap=float("nan"))), "softcap"),
    (dict(kw=dict(scale=float("inf"))), "scale"),
    (dict(kw=dict(slopes=torch.ones(3))), "slopes"),
    (dict(kw=dict(slopes=torch.ones(4).double())), "slopes"),
    (dict(kw=dict(q_pos=torch.zeros(2).long())), "both"),
    (dict(kw=dict(mass=torch.zeros(2, 2, 7))), "mass"),
    (dict(kw=dict(mass_out=torch.zeros(2, 2, 48))), "needs mass"),
])
def test_decode_refuses(change, words):
    args, _ = _decode_args()
    if "at" in change:
        args[change["at"]] = change["to"](args[change["at"]])
    with pytest.raises(ValueError, match=words):
        ops.paged_decode_op(*args, **change.get("kw", {}))


@pytest.mark.parametrize("kw, words", [
    (dict(softcap=-1.0), "softcap"), (dict(softcap=1e-7), "softcap"),
    (dict(softcap=1e4), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(scale=1e31), "scale"), (dict(scale=-float("inf")), "scale"),
    (dict(scale=float("nan")), "scale")])
def test_scores_refuse(kw, words):
    with pytest.raises(ValueError, match=words):
        ops.paged_decode_op(*_decode_args()[0], **kw)
    with pytest.raises(ValueError, match=words):
        ops.flash_prefill_packed_op(*_packed_args(), **kw)


def test_decode_refuses_overlap_and_gradients():
    args, room = _decode_args()
    store = torch.zeros(2 * 2 * room + 8)
    mass = store[:2 * 2 * room].view(2, 2, room)
    with pytest.raises(ValueError, match="apart"):
        ops.paged_decode_op(*args, mass=mass,
                            mass_out=store[8:].view(2, 2, room))
    args[0].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        ops.paged_decode_op(*args)
    with torch.no_grad():
        ops.paged_decode_op(*args)
    args[0].requires_grad_(False)
    args[2] = args[2].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        ops.paged_decode_op(*args)


def _packed_args():
    q = torch.randn(9, 4, 64).bfloat16()
    k = torch.randn(9, 2, 64).bfloat16()
    return [q, k, k.clone(), torch.tensor([0, 4, 9], dtype=torch.int32)]


@pytest.mark.parametrize("change, words", [
    (dict(at=0, to=lambda t: t.float()), "bfloat16 or float16"),
    (dict(at=0, to=lambda t: t[:, :3]), "multiple"),
    (dict(at=0, to=lambda t: t[..., :32]), "64 or 128"),
    (dict(at=0, to=lambda t: t[:8]), "as many rows"),
    (dict(at=1, to=lambda t: t.half()), "k: "),
    (dict(at=2, to=lambda t: t[:, :1]), "v: "),
    (dict(at=3, to=lambda t: t.float()), "cu_seqlens"),
    (dict(at=3, to=lambda t: t[:, None]), "cu_seqlens"),
    (dict(kw=dict(cu_seqlens_k=torch.tensor([0, 9]))), "cu_seqlens"),
    (dict(kw=dict(prefix_lens=torch.tensor([1]))), "prefix_lens"),
    (dict(kw=dict(out=torch.zeros(9, 4, 64))), "out"),
])
def test_packed_refuses(change, words):
    args = _packed_args()
    if "at" in change:
        args[change["at"]] = change["to"](args[change["at"]])
    with pytest.raises(ValueError, match=words):
        ops.flash_prefill_packed_op(*args, **change.get("kw", {}))


def test_packed_refuses_overlap_and_keeps_rows():
    q, k, v, cu = _packed_args()
    with pytest.raises(ValueError, match="apart"):
        ops.flash_prefill_packed_op(q, k, v, cu, out=q)
    row = torch.zeros(64 * 40).bfloat16()
    for strides in ((256, 0, 1), (0, 64, 1), (64, 64, 1), (256, 56, 1),
                    (200, 64, 1)):
        with pytest.raises(ValueError, match="share"):
            ops.flash_prefill_packed_op(
                q, k, v, cu, out=row.as_strided((9, 4, 64), strides))
    for strides in ((256, 64, 1), (64, 9 * 64, 1), (264, 64, 1)):
        ops.flash_prefill_packed_op(
            q, k, v, cu, out=row.as_strided((9, 4, 64), strides))
    for one in (q[:1], q[:, :1]):  # a stride that nothing steps by
        args = [one, k[:len(one), :1], v[:len(one), :1], cu[:1].repeat(2)]
        ops.flash_prefill_packed_op(
            *args, out=row.as_strided(one.shape, (
                (0, 64, 1) if len(one) == 1 else (64, 0, 1))))
    out = torch.full_like(q, 7.0)
    ops.flash_prefill_packed_op(q, k, v, cu[:2], out=out)
    assert (out[4:] == 7).all() and not (out[:4] == 7).any()


@pytest.mark.parametrize("kw, words", [
    (dict(budget=0), "budget"), (dict(budget=1 << 31), "budget"),
    (dict(recent=-1), "recent"), (dict(recent=9, budget=8), "recent"),
    (dict(mass=torch.zeros(1, 2, 3)), "mass"),
    (dict(key_pos=torch.zeros(2, 2, 48)), "key_pos"),
])
def test_evict_refuses(kw, words):
    st = cases.cache(1, [5, 20], 2, 64, 16)
    args = dict(mass=torch.zeros(2, 2, st["room"]), budget=8, recent=2,
                key_pos=torch.zeros(2, 2, st["room"], dtype=torch.int32))
    args.update(kw)
    with pytest.raises(ValueError, match=words):
        ops.kv_evict_op(st["k"], st["v"], st["table"], st["lens"], **args)


def test_append_refuses():
    st = cases.cache(1, [5, 20], 2, 64, 16)
    at = (st["k"], st["v"], st["table"], st["lens"])
    k = torch.randn(2, 2, 64).bfloat16()
    for new, kw, words in [
            (k[:1], {}, "one token"), (k.half(), {}, "k: "),
            (k[:, :1], {}, "k: "),
            (k, dict(cu_seqlens=torch.tensor([0, 2])), "cu_seqlens"),
            (k, dict(pos=torch.tensor([0, 2])), "both")]:
        with pytest.raises(ValueError, match=words):
            ops.paged_append_op(new, new, *at, **kw)


@pytest.mark.parametrize("weights", [False, True])
def test_cache_steps(weights):
    import paged_cache_loop

    paged_cache_loop.run("cpu", weights)


def test_cache_refuses():
    from triton_dist_amd.models import PagedKVCache

    cache = PagedKVCache(1, 2, 64, 2, 64, block=16)
    with pytest.raises(RuntimeError, match="without weights"):
        cache.evict(8, 2)
    with pytest.raises(ValueError, match="reserve"):
        cache.reserve(65)
    cache = PagedKVCache(1, 2, 64, 2, 64, block=16, weights=True)
    with pytest.raises(RuntimeError, match="by write"):
        cache.append(0, torch.zeros(2, 1, 2, 64), torch.zeros(2, 1, 2, 64), 0)
