"""The operators over a paged cache and packed prompts on the GPU, at the
ends of what they take."""
import pytest
import torch

import paged_limits as limits
import paged_oracle as oracle
from triton_dist_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", limits.LARGE)
def test_packed_large_logits(name):
    """Logits that 32 bits hold to many units: the largest takes it all, and
    equal ones share it."""
    args, kw, want = limits.packed_large(name)
    args = [x.cuda() for x in args]
    kw = {k: x.cuda() if isinstance(x, torch.Tensor) else x
          for k, x in kw.items()}
    out, lse = ops.flash_prefill_packed_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)


@pytest.mark.parametrize("name", limits.LARGE)
def test_decode_large_logits(name):
    """The same, with equal keys in chunks apart, and their weights."""
    args, kw, want = limits.decode_large(name)
    args = [x.cuda() for x in args]
    kw = {k: x.cuda() if isinstance(x, torch.Tensor) else x
          for k, x in kw.items()}
    out, lse, mass = ops.paged_decode_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)
    limits.hold_mass(mass, want)


def _cuda(x):
    return {k: _cuda(v) for k, v in x.items()} if isinstance(x, dict) else \
        x.cuda() if isinstance(x, torch.Tensor) else x


@pytest.mark.parametrize("name", limits.DECODE_WILD)
def test_decode_wild_values(name):
    """Values that are no finite numbers, among slots that are seen."""
    q, st, kw, want = limits.decode_wild(name)
    g = _cuda(st)
    out = ops.paged_decode_op(q.cuda(), g["k"], g["v"], g["table"],
                              g["lens"], **_cuda(kw))
    oracle.check("out", out[0] if "mass" in kw else out, want["out"])


@pytest.mark.parametrize("name", limits.PACKED_WILD)
def test_packed_wild_values(name):
    args, kw, want = limits.packed_wild(name)
    out = ops.flash_prefill_packed_op(*(x.cuda() for x in args), **_cuda(kw))
    oracle.check("out", out, want["out"])


@pytest.mark.parametrize("name", limits.FAINT)
def test_faint_weights_in_fp16(name):
    """Weights that 16 bits do not hold as they are."""
    q, k, v, out, tol = limits.faint(name)
    n, pages = len(k), -(-len(k) // 16)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    got = ops.flash_prefill_packed_op(q.cuda(), k.cuda(), v.cuda(), cu,
                                      cu_seqlens_k=cu * n, scale=1.0)
    oracle.check("prefill", got, (out, tol(9)))
    pool = torch.zeros(2, pages * 16, 1, k.shape[2], dtype=k.dtype)
    pool[0, :n], pool[1, :n] = k, v
    pool = pool.view(2, pages, 16, 1, -1).cuda()
    got = ops.paged_decode_op(
        q.cuda(), pool[0], pool[1], torch.arange(pages, device="cuda")[None],
        torch.tensor([n], device="cuda"), scale=1.0)
    oracle.check("decode", got, (out, tol(15)))


@pytest.mark.parametrize("weights", [False, True])
def test_replays_past_the_table(weights):
    """Steps that the host does not see: what has no slot is dropped, and
    told; the rest is what eager steps leave. Then the host looks again."""
    from triton_dist_amd.models import PagedKVCache

    cache = PagedKVCache(1, 2, 32, 1, 64, block=16, device="cuda",
                         weights=weights)
    cache.reserve(16)
    cache.begin_step(torch.tensor([13, 2], device="cuda"))
    cu = torch.tensor([0, 13, 15], device="cuda")
    x = torch.ones(15, 1, 64, device="cuda").bfloat16()
    cache.write(0, x, x, cu)
    cache.end_step()
    x = torch.ones(2, 1, 64, device="cuda").bfloat16()

    def step():
        cache.begin_step()
        cache.write(0, x, x)
        out = cache.attend(0, x)
        cache.end_step()
        return out

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(20):
        graph.replay()
        torch.cuda.synchronize()
        n = [14 + turn + 1, 3 + turn + 1]
        assert cache.lost().tolist() == [m > 16 for m in n]
        assert cache.seq_len.tolist() == [min(m, 32) for m in n]
        assert (out == 1).all()
    with pytest.raises(RuntimeError, match="no room"):
        step()
    cache.reserve(32)
    assert cache.lost().tolist() == [True, True]
    cache.reset()
    cache.reserve(32)
    for _ in range(32):
        step()
    with pytest.raises(RuntimeError, match="no room"):
        step()
    assert not cache.lost().any()


@pytest.mark.parametrize("name", limits.EVICT_GONE)
@pytest.mark.parametrize("n, spare", [(100, 0), (100, 5000), (100, 20000)])
def test_evict_where_pages_are_gone(name, n, spare):
    """In each of the selection's forms, which go by the table's width."""
    before, mass, pos, budget, recent, there, kept = limits.evict_gone(name,
                                                                       n)
    k, v, table, lens = (x.cuda() for x in before)
    room = mass.shape[2] + -(-spare // k.shape[1]) * k.shape[1]
    wide = torch.full((1, room // k.shape[1]), -1, device="cuda")
    wide[:, :table.shape[1]] = table
    more = torch.zeros(1, mass.shape[1], room - mass.shape[2], device="cuda")
    got = ops.kv_evict_op(
        k, v, wide, lens, torch.cat([mass.cuda(), more], 2),
        torch.cat([pos.cuda(), more.int()], 2), budget, recent)
    limits.hold_evicted(before, (k, v), mass, pos, got, budget, there, kept)
