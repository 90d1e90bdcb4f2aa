"""What a PagedKVCache does when a step has no room."""
import pytest
import torch

from triton_dist_amd.models import PagedKVCache


def _cache(weights, **kw):
    return PagedKVCache(2, 2, 16, 1, 64, block=8, weights=weights, **kw)


def _step(cache, value, counts=1):
    x = torch.full((2, 1, 64), float(value)).bfloat16()
    cache.begin_step(counts)
    out = []
    for layer in range(2):
        cache.write(layer, x, x)
        out.append(cache.attend(layer, x))
    cache.end_step()
    return out


def _state(cache):
    return [t.clone() for t in (cache.seq_len, cache.next_pos, cache.k_pool,
                                cache.v_pool, cache._live, cache._count)]


def _refused(cache, counts=1, words="no room"):
    before = _state(cache)
    with pytest.raises(RuntimeError, match=words):
        _step(cache, 1.0, counts)
    assert all(torch.equal(x, y) for x, y in zip(before, _state(cache)))
    assert not cache.lost().any()


@pytest.mark.parametrize("weights", [False, True])
def test_steps_past_the_table(weights):
    cache = _cache(weights)
    cache.reserve(16)
    for i in range(16):
        _step(cache, i)
    _refused(cache)
    _refused(cache)
    cache.seq_len[0] = 3  # one sequence made shorter is not enough
    _refused(cache, words=r"\[1\]")
    cache.seq_len[1] = 5
    _step(cache, 1.0)
    assert cache.seq_len.tolist() == [4, 6]


def test_a_budget_that_frees_nothing():
    """Every token's own row is there for it, or the step is refused."""
    cache = _cache(True)
    cache.reserve(16)
    for i in range(16):
        _step(cache, i)
        cache.evict(16, 4)
    _refused(cache)
    cache.evict(15, 4)
    out = _step(cache, 99.0)
    assert cache.key_pos[:, :, :, :16].amax(-1).eq(16).all()
    assert all((o > 6).all() for o in out)  # 99 takes it nearly all


def test_a_budget_that_frees_some():
    cache = _cache(True)
    cache.reserve(16)
    for i in range(60):
        _step(cache, i)
        cache.evict(12, 4)
    assert cache.seq_len.tolist() == [12, 12]
    assert cache.next_pos.tolist() == [60, 60] and not cache.lost().any()


def test_no_pages():
    cache = _cache(False)
    _refused(cache)
    cache.reserve(8)
    for i in range(8):
        _step(cache, i)
    _refused(cache)
    cache.reserve(9)
    _step(cache, 8)
    assert cache.seq_len.tolist() == [9, 9]
    cache.reset()
    _refused(cache)


def test_counts_of_each_sequence():
    cache = _cache(False)
    cache.reserve(16)
    _step(cache, 1.0, torch.tensor([1, 16]))
    _refused(cache, torch.tensor([1, 1]))
    _step(cache, 1.0, torch.tensor([1, 0]))
    assert cache.seq_len.tolist() == [2, 16]


def test_pages_of_the_callers_own():
    """A table that the caller fills needs no reserve."""
    cache = _cache(False)
    cache.block_table.copy_(torch.tensor([[2, -1], [3, 1]]))
    for i in range(8):
        _step(cache, i)
    _refused(cache, words=r"\[0\]")
    _step(cache, 1.0, torch.tensor([0, 1]))
    cache.block_table[0, 1] = 0
    _step(cache, 1.0)
    assert cache.seq_len.tolist() == [9, 10]


def test_append_and_then_steps():
    cache = _cache(False)
    x = torch.zeros(2, 7, 1, 64).bfloat16()
    for layer in range(2):
        cache.append(layer, x, x, 0)
    _step(cache, 1.0)
    _refused(cache)
    assert cache.seq_len.tolist() == [8, 8]


def test_lost_is_remembered():
    """What the host cannot refuse is told afterwards, also once there are
    pages."""
    cache = _cache(False)
    cache.reserve(8)
    cache.seq_len.copy_(torch.tensor([8, 2]))
    cache._live.copy_(torch.tensor([9, 3]))  # as a replayed step leaves it
    cache.end_step()
    assert cache.lost().tolist() == [True, False]
    cache.reserve(16)
    assert cache.lost().tolist() == [True, False]
    cache._live.fill_(40)
    cache.end_step()
    assert cache.seq_len.tolist() == [16, 16]
    assert cache.lost().tolist() == [True, True]
    cache.reset()
    assert not cache.lost().any()
