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
