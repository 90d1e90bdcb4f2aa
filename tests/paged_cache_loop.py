"""A PagedKVCache step by step beside a list of the tokens that should be in
it: shared by the tests on the CPU and on the GPU."""
import torch

import paged_oracle as oracle
from triton_dist_amd.models import PagedKVCache


def run(device, weights, graph=False):
    """Prompts of unlike lengths, then steps of one token, cut to a budget
    from time to time. What is attended is checked against all tokens that
    the cache should still hold, by what it says of their positions."""
    layers, b, qh, kvh, d, budget = 2, 3, 4, 2, 64, 24
    gen = torch.Generator().manual_seed(11)
    lens = [17, 1, 30]
    cache = PagedKVCache(layers, b, 64, kvh, d, block=16, device=device,
                         weights=weights)
    cache.reserve(64)
    told = [[[] for _ in range(b)] for _ in range(layers)]  # (k, v) by pos

    def token(n):
        return torch.randn(n, 2 * kvh + qh, d, generator=gen).bfloat16()

    starts = torch.tensor([0, 17, 18, 48], dtype=torch.int32)
    cache.begin_step(torch.tensor(lens, device=device))
    for layer in range(layers):
        x = token(sum(lens))
        for i in range(b):
            told[layer][i] = list(x[starts[i]:starts[i + 1]])
        x = x.to(device)
        cache.write(layer, x[:, :kvh], x[:, kvh:2 * kvh],
                    starts.to(device))
    cache.end_step()
    assert cache.seq_len.tolist() == lens

    x = [token(b).to(device) for _ in range(layers)]
    slopes = torch.tensor([0.3, 0.1, 0.02, 0.0], device=device)

    def step():
        cache.begin_step()
        out = []
        for layer in range(layers):
            cache.write(layer, x[layer][:, :kvh], x[layer][:, kvh:2 * kvh])
            out.append(cache.attend(layer, x[layer][:, 2 * kvh:],
                                    slopes=slopes, softcap=20.0))
        cache.end_step()
        if weights:
            cache.evict(budget, 6)
        return out

    play = step
    if graph:
        state = [cache.k_pool, cache.v_pool, cache.seq_len, cache.next_pos]
        state += [cache.mass, cache.key_pos] if weights else []
        saved = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        for t, old in zip(state, saved):
            t.copy_(old)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            out = step()

        def play():
            captured.replay()
            return out
    for turn in range(10):
        held = None
        if weights:
            held = cache.key_pos.cpu().clone()
            mass = cache.mass.cpu().clone()
        before = cache.seq_len.tolist()
        for layer in range(layers):
            new = token(b)
            x[layer].copy_(new)
            for i in range(b):
                told[layer][i].append(new[i])
        got = play()
        for layer in range(layers):
            for i in range(b):
                n = len(told[layer][i])
                for h in range(qh):
                    kh = h // (qh // kvh)
                    pos = list(range(n))
                    if weights:
                        pos = held[layer, i, kh, :before[i]].tolist() \
                            + [n - 1]
                        assert len(set(pos)) == len(pos)
                    rows = torch.stack([told[layer][i][p] for p in pos])
                    gap = n - 1 - torch.tensor(pos).double()
                    o, _, _, tol, _, _ = oracle.attend(
                        told[layer][i][-1][2 * kvh + h].double(),
                        rows[:, kh].double(), rows[:, kvh + kh].double(),
                        d ** -0.5, 20.0, float(slopes[h]) * gap,
                        torch.bfloat16)
                    oracle.check(f"turn {turn} layer {layer} seq {i}",
                                 got[layer][i, h], (o, tol))
        want = [min(n + 1, budget) if weights else n + 1 for n in before]
        assert cache.seq_len.tolist() == want
        assert cache.next_pos.tolist() == [n + turn + 1 for n in lens]
        if weights:  # every step hands out one weight a query head
            total = cache.mass.double().sum().item()
            assert total <= mass.double().sum().item() \
                + layers * b * qh + 1e-3
            for i, n in enumerate(want):
                live = cache.key_pos[:, i, :, :n]
                newest = lens[i] + turn
                for back in range(min(6, n)):
                    assert (live == newest - back).sum() == layers * kvh
                assert (cache.key_pos[:, i, :, n:] == -1).all()
                assert (cache.mass[:, i, :, n:] == 0).all()
