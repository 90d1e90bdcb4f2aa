"""Operators over a paged key-value cache, and the attention of packed
prompts that fills it: HIP kernels on GPU, torch references on CPU.

A cache's layer is a pair of pools [n_blocks, block, kvh, d] (a
`PagedKVCache.k_pool[layer]`), a table [B, max_blocks] of page numbers and
the sequences' lengths [B]; sequence b's slot s is row s % block of page
table[b, s // block]. Lengths and page numbers stay on the device, so every
operator can be captured into a graph and replayed while they change. They
are not copied to the host, so what they hold is bounded on the device
instead: a length counts as at most max_blocks * block and at least 0, and
a page number outside the pool as a page that is not there. Keys of such a
page are left out of attention, rows meant for it are dropped.

The operators run on the device of their tensors and on its current stream,
allocate what they need from torch's allocator, and offer no gradients.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

_INDEX = (torch.int32, torch.int64)
_HALF = (torch.bfloat16, torch.float16)


def _need(ok: bool, message: str):
    if not ok:
        raise ValueError(message)


def _C():
    from .. import _C as mod

    if mod is None:
        raise RuntimeError("triton_dist_amd._C missing on a GPU host")
    return mod


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("this operator has no backward: call it under "
                           "torch.no_grad() or detach its inputs")


def _rows16(name: str, t: torch.Tensor):
    """The kernels move rows in pieces of 16 bytes."""
    if t.numel() == 0:
        return
    _need(t.stride(-1) == 1 or t.shape[-1] == 1,
          f"{name}: the last dimension has to be contiguous")
    _need(all(st % 8 == 0 for st, n in zip(t.stride()[:-1], t.shape[:-1])
              if n > 1) and t.data_ptr() % 16 == 0,
          f"{name}: rows have to start at multiples of 16 bytes")


def _index(name: str, t: torch.Tensor, shape, device):
    _need(t.dtype in _INDEX, f"{name}: int32 or int64, got {t.dtype}")
    _need(tuple(t.shape) == tuple(shape),
          f"{name}: shape {tuple(shape)}, got {tuple(t.shape)}")
    _need(t.device == device, f"{name}: on {t.device}, not on {device}")
    _need(t.is_contiguous(), f"{name}: has to be contiguous")


def _plane(name: str, t: torch.Tensor, dtype, shape, device):
    _need(t.dtype == dtype, f"{name}: {dtype}, got {t.dtype}")
    _need(tuple(t.shape) == tuple(shape),
          f"{name}: shape {tuple(shape)}, got {tuple(t.shape)}")
    _need(t.device == device, f"{name}: on {t.device}, not on {device}")
    _need(t.is_contiguous(), f"{name}: has to be contiguous")


def _overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    if not x.numel() or not y.numel():
        return False

    def ends(t):
        reach = sum((n - 1) * abs(st) for n, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (reach + 1) * t.element_size()

    (a, b), (c, d) = ends(x), ends(y)
    return a < d and c < b


def _cache(k_pool, v_pool, block_table, seq_lens):
    """Checks a cache's layer; returns (n_blocks, block, kvh, d, B, room)."""
    _need(k_pool.dim() == 4, "k_pool: [n_blocks, block, kvh, d]")
    _need(k_pool.dtype in _HALF,
          f"k_pool: bfloat16 or float16, got {k_pool.dtype}")
    _need(v_pool.dtype == k_pool.dtype and v_pool.shape == k_pool.shape
          and v_pool.device == k_pool.device,
          "v_pool: of k_pool's type, shape and device")
    n, block, kvh, d = k_pool.shape
    _need(block >= 1 and kvh >= 1, "k_pool: empty blocks")
    _need(1 <= n < 1 << 31, f"k_pool: from 1 to 2^31 - 1 pages, got {n}")
    _need(d % 8 == 0 and d >= 8, f"k_pool: d a multiple of 8, got {d}")
    _rows16("k_pool", k_pool)
    _rows16("v_pool", v_pool)
    _need(block_table.dim() == 2, "block_table: [B, max_blocks]")
    _need(block_table.dtype in _INDEX,
          f"block_table: int32 or int64, got {block_table.dtype}")
    _need(block_table.device == k_pool.device,
          f"block_table: on {block_table.device}, not on {k_pool.device}")
    b, width = block_table.shape
    _need(width <= 1 or block_table.stride(1) == 1,
          "block_table: rows have to be contiguous")
    _need(width * block < (1 << 31) - 4096,
          "block_table: a sequence has room for 2^31 - 4096 slots at most")
    _index("seq_lens", seq_lens, (b,), k_pool.device)
    return n, block, kvh, d, b, width * block


def _fields(k_pool, v_pool, block_table, seq_lens):
    n, block, kvh, d = k_pool.shape
    return [k_pool.data_ptr(), v_pool.data_ptr(), *k_pool.stride()[:3],
            *v_pool.stride()[:3], n, block, kvh, d,
            int(k_pool.dtype == torch.float16), block_table.data_ptr(),
            int(block_table.dtype == torch.int64), block_table.stride(0),
            block_table.shape[1], seq_lens.data_ptr(),
            int(seq_lens.dtype == torch.int64), block_table.shape[0]]


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _is64(t: Optional[torch.Tensor]) -> int:
    return int(t is not None and t.dtype == torch.int64)


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _grouped(qh: int, kvh: int):
    _need(qh >= kvh and qh % kvh == 0,
          f"q: {qh} heads are no multiple of the {kvh} key heads")


def _score_args(scale, softcap, slopes, d, qh, device):
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    _need(math.isfinite(scale), f"scale: finite, got {scale}")
    _need(math.isfinite(softcap) and softcap >= 0,
          f"softcap: finite and not negative, got {softcap}")
    if slopes is not None:
        _plane("slopes", slopes, torch.float32, (qh,), device)
    return scale, softcap


def _rows_of(table, lens, n_blocks, block):
    """CPU: per sequence the slots whose page is there, with (page, row)."""
    room = table.shape[1] * block
    for b in range(table.shape[0]):
        slot = torch.arange(min(max(int(lens[b]), 0), room))
        page = table[b].long()[slot // block]
        yield b, slot, page, slot % block, (page >= 0) & (page < n_blocks)


# ------------------------------------------------------------------ append
def paged_append_op(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor,
                    v_pool: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, *,
                    cu_seqlens: Optional[torch.Tensor] = None,
                    key_pos: Optional[torch.Tensor] = None,
                    pos: Optional[torch.Tensor] = None) -> None:
    """Write new keys and values [T, kvh, d] to the pages of a cache.

    Without `cu_seqlens` token b is sequence b's one new token (T = B) and
    goes to its slot seq_lens[b]. With `cu_seqlens` [B + 1] the tokens of
    sequence b are the rows cu_seqlens[b] to cu_seqlens[b + 1], for the
    slots from seq_lens[b] on; rows behind the last sequence are ignored.
    Lengths are left to the caller, who adds to them once per step. A row
    without room (past the table, or on a page that is not there) is
    dropped. `key_pos` [B, kvh, room] int32, if given, gets the tokens'
    positions `pos` [T] at their slots.
    """
    n, block, kvh, d, b, room = _cache(k_pool, v_pool, block_table, seq_lens)
    dev = k_pool.device
    _no_grad(k, v)
    for name, t in (("k", k), ("v", v)):
        _need(t.dim() == 3 and t.shape[1:] == (kvh, d),
              f"{name}: [T, {kvh}, {d}], got {tuple(t.shape)}")
        _need(t.dtype == k_pool.dtype,
              f"{name}: the pools' {k_pool.dtype}, got {t.dtype}")
        _need(t.device == dev, f"{name}: on {t.device}, not on {dev}")
        _rows16(name, t)
    tokens = k.shape[0]
    _need(v.shape[0] == tokens, "k and v: as many tokens each")
    if cu_seqlens is None:
        _need(tokens == b, f"k: one token for each of {b} sequences, got "
                           f"{tokens}; packed tokens need cu_seqlens")
    else:
        _index("cu_seqlens", cu_seqlens, (b + 1,), dev)
    _need((key_pos is None) == (pos is None),
          "key_pos and pos: both or neither")
    if key_pos is not None:
        _plane("key_pos", key_pos, torch.int32, (b, kvh, room), dev)
        _index("pos", pos, (tokens,), dev)
    if not tokens or not b:
        return
    if k_pool.is_cuda:
        with torch.cuda.device(dev):
            _C().paged_append(
                _fields(k_pool, v_pool, block_table, seq_lens),
                k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                v.stride(0), v.stride(1), tokens, _ptr(cu_seqlens),
                _is64(cu_seqlens), _ptr(key_pos), _ptr(pos), _is64(pos),
                _stream(dev))
        return
    for i in range(b):
        lo = i if cu_seqlens is None else max(int(cu_seqlens[i]), 0)
        hi = i + 1 if cu_seqlens is None else min(int(cu_seqlens[i + 1]),
                                                  tokens)
        first = lo if cu_seqlens is None else int(cu_seqlens[i])
        for t in range(lo, hi):
            slot = int(seq_lens[i]) + t - first
            if not 0 <= slot < room:
                continue
            page = int(block_table[i, slot // block])
            if not 0 <= page < n:
                continue
            k_pool[page, slot % block] = k[t]
            v_pool[page, slot % block] = v[t]
            if key_pos is not None:
                key_pos[i, :, slot] = pos[t]


# ------------------------------------------------------------------ decode
def paged_decode_op(q: torch.Tensor, k_pool: torch.Tensor,
                    v_pool: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, *,
                    scale: Optional[float] = None, softcap: float = 0.0,
                    slopes: Optional[torch.Tensor] = None,
                    key_pos: Optional[torch.Tensor] = None,
                    q_pos: Optional[torch.Tensor] = None,
                    mass: Optional[torch.Tensor] = None,
                    mass_out: Optional[torch.Tensor] = None,
                    return_lse: bool = False):
    """Attention of one new token a sequence, q [B, qh, d], over the first
    seq_lens[b] slots of its pages (the new token's own row among them:
    append first). d is 64 or 128; qh is a multiple of kvh.

    A score is s = scale * q.k (scale: d ** -0.5 by default), then
    softcap * tanh(s / softcap) if softcap > 0, then less slopes[h] * |i-j|
    if `slopes` [qh] fp32 are given, with the query's position i and the
    key's position j: the last slot's and the key's slot number, or
    `q_pos` [B] and `key_pos` [B, kvh, room] int32 for a cache whose rows
    have moved.

    `mass` [B, kvh, room] fp32 asks for the attention weights: returned is
    mass plus, for each slot, the weights that the key head's query heads
    gave it, and 0 for the slots past the length. It is a new tensor, or
    `mass_out`, which may be `mass` itself.

    Returns out [B, qh, d], and in this order, where asked for, the log of
    the sum of exponentials [B, qh] fp32 and the weights. A sequence that
    sees no key gets zeros and -inf.
    """
    n, block, kvh, d, b, room = _cache(k_pool, v_pool, block_table, seq_lens)
    dev = k_pool.device
    _no_grad(q, slopes, mass)
    _need(q.dim() == 3 and q.shape[0] == b and q.shape[2] == d,
          f"q: [{b}, qh, {d}], got {tuple(q.shape)}")
    _need(q.dtype == k_pool.dtype,
          f"q: the pools' {k_pool.dtype}, got {q.dtype}")
    _need(q.device == dev, f"q: on {q.device}, not on {dev}")
    _need(d in (64, 128), f"q: d of 64 or 128, got {d}")
    qh = q.shape[1]
    _grouped(qh, kvh)
    _rows16("q", q)
    scale, softcap = _score_args(scale, softcap, slopes, d, qh, dev)
    _need((key_pos is None) == (q_pos is None),
          "key_pos and q_pos: both or neither")
    if key_pos is not None:
        _plane("key_pos", key_pos, torch.int32, (b, kvh, room), dev)
        _index("q_pos", q_pos, (b,), dev)
    if mass is None:
        _need(mass_out is None, "mass_out: needs mass")
    else:
        _plane("mass", mass, torch.float32, (b, kvh, room), dev)
        if mass_out is None:
            mass_out = torch.empty_like(mass)
        else:
            _plane("mass_out", mass_out, torch.float32, (b, kvh, room), dev)
            _need(mass_out.data_ptr() == mass.data_ptr()
                  or not _overlap(mass, mass_out),
                  "mass_out: mass itself, or apart from it")
    out = torch.empty(b, qh, d, dtype=q.dtype, device=dev)
    lse = torch.empty(b, qh, dtype=torch.float32, device=dev)
    if b and k_pool.is_cuda:
        with torch.cuda.device(dev):
            ws = torch.empty(
                _C().paged_decode_workspace(b, qh, kvh, d, room,
                                            mass is not None),
                dtype=torch.uint8, device=dev)
            _C().paged_decode(
                _fields(k_pool, v_pool, block_table, seq_lens),
                q.data_ptr(), q.stride(0), q.stride(1), qh, scale, softcap,
                _ptr(slopes), _ptr(key_pos), _ptr(q_pos), _is64(q_pos),
                out.data_ptr(), lse.data_ptr(), _ptr(mass), _ptr(mass_out),
                ws.data_ptr(), _stream(dev))
    elif b:
        _decode_cpu(q, k_pool, v_pool, block_table, seq_lens, scale, softcap,
                    slopes, key_pos, q_pos, mass, mass_out, out, lse)
    got = [out] + ([lse] if return_lse else []) \
        + ([mass_out] if mass is not None else [])
    return got[0] if len(got) == 1 else tuple(got)


def _weights_cpu(s: torch.Tensor):
    """Softmax over the last axis and its log-sum-exp; rows of -inf weigh
    nothing."""
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    return torch.where(torch.isinf(s) & (s < 0), 0.0, w), lse


def _decode_cpu(q, k_pool, v_pool, table, lens, scale, softcap, slopes,
                key_pos, q_pos, mass, mass_out, out, lse):
    n_blocks, block, kvh, d = k_pool.shape
    g = q.shape[1] // kvh
    for b, slot, page, row, there in _rows_of(table, lens, n_blocks, block):
        n = int(slot.numel())
        gap = slot.new_tensor(n - 1) - slot
        page, row, at = page[there], row[there], slot[there]
        k = k_pool[page, row].float().permute(1, 2, 0)     # [kvh, d, n]
        v = v_pool[page, row].float().transpose(0, 1)      # [kvh, n, d]
        s = torch.matmul(q[b].float().view(kvh, g, d), k) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            if key_pos is not None:
                gap = q_pos[b].long() - key_pos[b].long()[:, at]
            else:
                gap = gap[there].expand(kvh, -1)
            s = s - slopes.view(kvh, g, 1) * gap.abs().float()[:, None]
        w, total = _weights_cpu(s)
        out[b] = torch.matmul(w, v).view(-1, d).to(out.dtype)
        lse[b] = total.view(-1)
        if mass is not None:
            new = mass[b].clone()
            new[:, at] += w.sum(1)
            new[:, n:] = 0
            mass_out[b] = new


# ------------------------------------------------------------------- evict
def kv_evict_op(k_pool: torch.Tensor, v_pool: torch.Tensor,
                block_table: torch.Tensor, seq_lens: torch.Tensor,
                mass: torch.Tensor, key_pos: torch.Tensor, budget: int,
                recent: int, *, out: Optional[Tuple] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence longer than `budget` slots to `budget`, per key
    head: the slots of the `recent` newest positions stay, and of the others
    those of the largest weight `mass` [B, kvh, room] fp32 (a NaN counts as
    the largest, of equal ones the lowest slot stays).

    The rows that stay are moved into the slots below the budget in place:
    the i-th slot below it that became free takes the i-th kept row from
    above it, all others stay where they are. So the slots' order is lost,
    and `key_pos` [B, kvh, room] int32 holds each slot's position. A newest
    position is the largest of a sequence's slots.

    Returns the lengths, weights and positions afterwards, with 0 and -1 in
    the slots past the new length: new tensors, or those of `out`, which may
    be the inputs themselves. A page is moved by the one sequence that holds
    it: pages that sequences share must not be evicted from.
    """
    n, block, kvh, d, b, room = _cache(k_pool, v_pool, block_table, seq_lens)
    dev = k_pool.device
    _plane("mass", mass, torch.float32, (b, kvh, room), dev)
    _plane("key_pos", key_pos, torch.int32, (b, kvh, room), dev)
    _no_grad(mass)
    budget, recent = int(budget), int(recent)
    _need(1 <= budget < 1 << 31, f"budget: at least 1, got {budget}")
    _need(0 <= recent <= budget,
          f"recent: from 0 to the budget of {budget}, got {recent}")
    if out is None:
        out = (torch.empty_like(seq_lens), torch.empty_like(mass),
               torch.empty_like(key_pos))
    else:
        _need(len(out) == 3, "out: (seq_lens, mass, key_pos)")
        _plane("out[0]", out[0], seq_lens.dtype, (b,), dev)
        _plane("out[1]", out[1], torch.float32, (b, kvh, room), dev)
        _plane("out[2]", out[2], torch.int32, (b, kvh, room), dev)
        for new, old in zip(out, (seq_lens, mass, key_pos)):
            _need(new.data_ptr() == old.data_ptr()
                  or not _overlap(new, old),
                  "out: the inputs themselves, or apart from them")
        for i, x in enumerate(out):
            for j, y in enumerate((seq_lens, mass, key_pos)):
                _need(i == j or not _overlap(x, y),
                      "out: not over another input")
            for y in out[:i]:
                _need(not _overlap(x, y), "out: apart from each other")
    if not b:
        return out
    if k_pool.is_cuda:
        with torch.cuda.device(dev):
            ws = torch.empty(
                _C().kv_evict_workspace(b, kvh, room, budget),
                dtype=torch.uint8, device=dev)
            _C().kv_evict(_fields(k_pool, v_pool, block_table, seq_lens),
                          mass.data_ptr(), key_pos.data_ptr(), budget,
                          recent, out[1].data_ptr(), out[2].data_ptr(),
                          out[0].data_ptr(), ws.data_ptr(), _stream(dev))
        return out
    new_lens, new_mass = seq_lens.clone(), mass.clone()
    new_pos = key_pos.clone()
    for i in range(b):
        length = min(max(int(seq_lens[i]), 0), room)
        keep = min(length, budget)
        for h in range(kvh if length > keep else 0):
            m, p = mass[i, h, :length], key_pos[i, h, :length].long()
            fresh = p > int(p.max()) - recent
            order = torch.sort(m, descending=True, stable=True).indices
            order = torch.cat([torch.nonzero(fresh)[:, 0],
                               order[~fresh[order]]])
            kept = torch.zeros(length, dtype=torch.bool)
            kept[order[:keep]] = True
            holes = torch.nonzero(~kept[:keep])[:, 0].tolist()
            movers = (torch.nonzero(kept[keep:])[:, 0] + keep).tolist()
            for to, frm in zip(holes, movers):
                new_mass[i, h, to] = m[frm]
                new_pos[i, h, to] = key_pos[i, h, frm]
                pt = int(block_table[i, to // block])
                pf = int(block_table[i, frm // block])
                if 0 <= pt < n and 0 <= pf < n:
                    for pool in (k_pool, v_pool):
                        pool[pt, to % block, h] = pool[pf, frm % block, h]
        new_lens[i] = keep
        new_mass[i, :, keep:] = 0
        new_pos[i, :, keep:] = -1
    for new, got in zip(out, (new_lens, new_mass, new_pos)):
        new.copy_(got)
    return out


# ----------------------------------------------------------------- prefill
def flash_prefill_packed_op(q: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                            cu_seqlens_k: Optional[torch.Tensor] = None,
                            causal: bool = True,
                            prefix_lens: Optional[torch.Tensor] = None,
                            scale: Optional[float] = None,
                            softcap: float = 0.0,
                            slopes: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None,
                            return_lse: bool = False):
    """Attention of documents packed side by side: q [T, qh, d], k and v
    [Tk, kvh, d], d 64 or 128, qh a multiple of kvh. Document i's queries
    are rows cu_seqlens[i] to cu_seqlens[i + 1], its keys the same rows, or
    those of `cu_seqlens_k`. A token sees its own document only.

    With `causal`, query i of a document with m queries and n keys sees the
    keys up to i + n - m (the last query sees them all), and besides them
    the document's first prefix_lens[i] keys. Scores are capped by `softcap`
    and lowered by `slopes` as in `paged_decode_op`, the distance being that
    from key position i + n - m.

    Returns out [T, qh, d] and, if asked for, the log of the sum of
    exponentials [T, qh] fp32. A row that sees no key gets zeros and -inf.
    Rows that belong to no document are left as they were in a given `out`,
    and are zeros and -inf in tensors that the call makes (a `lse` always).
    Keys and values of rows that a document's mask hides from part of its
    queries have to be finite.
    """
    dev = q.device
    _need(q.dim() == 3 and k.dim() == 3,
          "q and k: [tokens, heads, d]")
    _need(q.dtype in _HALF, f"q: bfloat16 or float16, got {q.dtype}")
    rows, qh, d = q.shape
    keys, kvh = k.shape[:2]
    _need(d in (64, 128), f"q: d of 64 or 128, got {d}")
    _need(kvh >= 1 and k.shape[2] == d, f"k: [Tk, kvh, {d}], got "
                                        f"{tuple(k.shape)}")
    _need(v.shape == k.shape, "v: of k's shape")
    for name, t in (("k", k), ("v", v)):
        _need(t.dtype == q.dtype, f"{name}: q's {q.dtype}, got {t.dtype}")
        _need(t.device == dev, f"{name}: on {t.device}, not on {dev}")
    _grouped(qh, kvh)
    _no_grad(q, k, v, slopes)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _rows16(name, t)
        _need(t.shape[0] < 1 << 31, f"{name}: 2^31 rows at most")
    _need(cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1,
          "cu_seqlens: [documents + 1]")
    docs = cu_seqlens.numel() - 1
    _index("cu_seqlens", cu_seqlens, (docs + 1,), dev)
    if cu_seqlens_k is None:
        _need(keys == rows, "k: as many rows as q, or cu_seqlens_k")
        cu_seqlens_k = cu_seqlens
    else:
        _index("cu_seqlens_k", cu_seqlens_k, (docs + 1,), dev)
    if prefix_lens is not None:
        _need(causal, "prefix_lens: without causal every key is seen")
        _index("prefix_lens", prefix_lens, (docs,), dev)
    scale, softcap = _score_args(scale, softcap, slopes, d, qh, dev)
    clear = out is None
    if out is None:
        out = torch.empty(rows, qh, d, dtype=q.dtype, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype
              and out.device == dev, "out: of q's shape, type and device")
        _rows16("out", out)
        _need(not any(_overlap(out, t) for t in (q, k, v)),
              "out: apart from q, k and v")
    lse = torch.empty(rows, qh, dtype=torch.float32, device=dev) \
        if return_lse else None
    if rows and q.is_cuda:
        with torch.cuda.device(dev):
            _C().packed_prefill(
                q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(),
                k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                v.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                _ptr(lse), rows, keys, qh, kvh, d,
                int(q.dtype == torch.float16), docs, cu_seqlens.data_ptr(),
                _is64(cu_seqlens), cu_seqlens_k.data_ptr(),
                _is64(cu_seqlens_k), _ptr(prefix_lens), _is64(prefix_lens),
                int(causal), int(clear), scale, softcap, _ptr(slopes),
                _stream(dev))
    elif rows:
        if clear:
            out.zero_()
        if lse is not None:
            lse.fill_(float("-inf"))
        _packed_cpu(q, k, v, cu_seqlens, cu_seqlens_k, causal, prefix_lens,
                    scale, softcap, slopes, out, lse)
    return (out, lse) if return_lse else out


def _packed_cpu(q, k, v, cu_q, cu_k, causal, prefix, scale, softcap, slopes,
                out, lse):
    rows, qh, d = q.shape
    keys, kvh = k.shape[:2]
    for i in range(cu_q.numel() - 1):
        q0, q1 = (min(max(int(c), 0), rows) for c in cu_q[i:i + 2])
        k0, k1 = (min(max(int(c), 0), keys) for c in cu_k[i:i + 2])
        m, n = q1 - q0, max(k1 - k0, 0)
        if m <= 0:
            continue
        qf = q[q0:q1].float().view(m, kvh, qh // kvh, d).permute(1, 2, 0, 3)
        kf = k[k0:k0 + n].float().permute(1, 2, 0)[:, None]
        s = torch.matmul(qf, kf) * scale            # [kvh, g, m, n]
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        at = torch.arange(m)[:, None] + n - m
        j = torch.arange(n)
        if slopes is not None:
            s = s - slopes.view(kvh, -1, 1, 1) * (at - j).abs().float()
        if causal:
            seen = j <= at
            if prefix is not None:
                seen = seen | (j < int(prefix[i]))
            s = s.masked_fill(~seen, float("-inf"))
        w, total = _weights_cpu(s)
        o = torch.matmul(w, v[k0:k0 + n].float().transpose(0, 1)[:, None])
        out[q0:q1] = o.permute(2, 0, 1, 3).reshape(m, qh, d).to(out.dtype)
        if lse is not None:
            lse[q0:q1] = total.permute(2, 0, 1).reshape(m, qh)
