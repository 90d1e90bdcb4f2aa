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

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward

_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_BF16, _FP16 = torch.bfloat16, torch.float16
# the stream as a number, without a Stream object around it
_raw_stream = torch._C._cuda_getCurrentRawStream \
    if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _native():
    from .. import _C as mod

    if mod is None:
        raise RuntimeError("triton_dist_amd._C missing on a GPU host")
    return mod


def _call(name: str, dev: torch.device, *args):
    """The native function on the tensors' device and its current stream."""
    fn = getattr(_native(), name)
    if dev.index == torch.cuda.current_device():
        fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            fn(*args, _raw_stream(dev.index))


# Every check costs host time that a decode step of a few microseconds
# waits for, so the common case goes by in one comparison or two and
# messages are put together when they are needed.
def _refuse(message: str):
    raise ValueError(message)


def _no_backward():
    raise RuntimeError("this operator has no backward: call it under "
                       "torch.no_grad() or detach its inputs")


def _no_tangents(*tensors):
    """Forward-mode derivatives, which need no requires_grad, would vanish."""
    if _forward._current_level < 0:
        return
    if any(t is not None and _forward.unpack_dual(t).tangent is not None
           for t in tensors):
        raise RuntimeError("this operator has no forward derivative: give it "
                           "the primal of its inputs")


def _rows16(name: str, t: torch.Tensor):
    """The kernels move rows in pieces of 16 bytes."""
    if t.numel() == 0:
        return
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        _refuse(f"{name}: the last dimension has to be contiguous")
    if t.data_ptr() % 16 or any(
            st % 8 and n > 1 for st, n in zip(t.stride()[:-1], t.shape)):
        _refuse(f"{name}: rows have to start at multiples of 16 bytes")


def _heads(name: str, t: torch.Tensor, dtype, dev):
    """A tensor [tokens, heads, d] beside others of `dtype` on `dev`."""
    if t.dtype != dtype:
        _refuse(f"{name}: {dtype} as the others, got {t.dtype}")
    if t.device != dev:
        _refuse(f"{name}: on {t.device}, not on {dev}")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s0 | s1) & 7 or t.data_ptr() & 15:
        _rows16(name, t)


def _array(name: str, t: torch.Tensor, dtype, shape, dev):
    """Contiguous, of a type (None: a whole number's) and shape."""
    if t.dtype != dtype and (dtype is not None or t.dtype != _I32
                             and t.dtype != _I64):
        _refuse(f"{name}: {dtype or 'int32 or int64'}, got {t.dtype}")
    if t.shape != shape:
        _refuse(f"{name}: shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != dev:
        _refuse(f"{name}: on {t.device}, not on {dev}")
    if not t.is_contiguous():
        _refuse(f"{name}: has to be contiguous")


def _overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    if not x.numel() or not y.numel():
        return False

    def ends(t):
        reach = sum((n - 1) * abs(st) for n, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (reach + 1) * t.element_size()

    (a, b), (c, d) = ends(x), ends(y)
    return a < d and c < b


def _cache(k_pool, v_pool, block_table, seq_lens):
    """Checks a cache's layer; returns what the native functions want of it
    and (block, kvh, d, B, slots of a sequence)."""
    dtype, dev, shape = k_pool.dtype, k_pool.device, k_pool.shape
    if len(shape) != 4:
        _refuse("k_pool: [n_blocks, block, kvh, d]")
    if dtype != _BF16 and dtype != _FP16:
        _refuse(f"k_pool: bfloat16 or float16, got {dtype}")
    if v_pool.dtype != dtype or v_pool.shape != shape or v_pool.device != dev:
        _refuse("v_pool: of k_pool's type, shape and device")
    if (k_pool.requires_grad or v_pool.requires_grad) \
            and torch.is_grad_enabled():
        _no_backward()
    n, block, kvh, d = shape
    if not (0 < n < 1 << 31 and block > 0 and kvh > 0 and d > 0) or d & 7:
        _refuse("k_pool: from 1 to 2^31 - 1 pages of at least one slot and "
                f"head, d a multiple of 8, got {tuple(shape)}")
    k, v = k_pool.data_ptr(), v_pool.data_ptr()
    k0, k1, k2, k3 = k_pool.stride()
    v0, v1, v2, v3 = v_pool.stride()
    if k3 != 1 or v3 != 1 or (k0 | k1 | k2 | v0 | v1 | v2) & 7 \
            or (k | v) & 15:
        _rows16("k_pool", k_pool)
        _rows16("v_pool", v_pool)
    if block_table.dim() != 2:
        _refuse("block_table: [B, max_blocks]")
    if block_table.dtype != _I64 and block_table.dtype != _I32:
        _refuse(f"block_table: int32 or int64, got {block_table.dtype}")
    if block_table.device != dev:
        _refuse(f"block_table: on {block_table.device}, not on {dev}")
    b, width = block_table.shape
    row, one = block_table.stride()
    if one != 1 and width > 1:
        _refuse("block_table: rows have to be contiguous")
    if width * block >= (1 << 31) - 4096:
        _refuse("block_table: fewer than 2^31 - 4096 slots a sequence")
    _array("seq_lens", seq_lens, None, (b,), dev)
    return [k, v, k0, k1, k2, v0, v1, v2, n, block, kvh, d, dtype == _FP16,
            block_table.data_ptr(), block_table.dtype == _I64, row, width,
            seq_lens.data_ptr(), seq_lens.dtype == _I64, b], \
        (block, kvh, d, b, width * block)


def _meet(apart: int, dims, d: int) -> bool:
    """Whether rows of d elements of two tensors of the same strides `dims`
    (from the largest, with sizes), whose first elements lie `apart`, have an
    element in common."""
    if not dims:
        return abs(apart) < d
    (stride, size), rest = dims[0], dims[1:]
    if stride == 0 or size == 1:
        return _meet(apart, rest, d)
    near = apart // stride
    return any(_meet(apart - i * stride, rest, d) for i in (near, near + 1)
               if abs(i) < size)


def _writes(k_pool, v_pool, fields):
    """Pools that a call writes: rows have memory of their own, also in the
    other pool unless both are one. Returns where each begins and ends."""
    k, v, k0, k1, k2, v0, v1, v2, n, block, kvh, d = fields[:12]
    if k_pool.is_contiguous() and v_pool.is_contiguous():
        size = 2 * n * block * kvh * d
        k_end, v_end = k + size, v + size
        if k_end <= v or v_end <= k or k == v:
            return k, k_end, v, v_end
    else:
        for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
            reach = d
            for stride, size in sorted(zip(t.stride(), t.shape[:3])):
                if size > 1:
                    if stride < reach:
                        _refuse(f"{name}: rows that do not share memory")
                    reach += stride * (size - 1)
        k_end = k + 2 * ((n - 1) * k0 + (block - 1) * k1 + (kvh - 1) * k2 + d)
        v_end = v + 2 * ((n - 1) * v0 + (block - 1) * v1 + (kvh - 1) * v2 + d)
    if k < v_end and v < k_end:
        same = (k0, k1, k2) == (v0, v1, v2)
        if not (same and k == v) and (not same or _meet(
                (v - k) // 2, sorted(((k0, n), (k1, block), (k2, kvh)),
                                     reverse=True), d)):
            _refuse("v_pool: k_pool itself, or apart from it")
    return k, k_end, v, v_end


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _is64(t: Optional[torch.Tensor]) -> int:
    return t is not None and t.dtype == _I64


def _score_args(scale, softcap, slopes, d, qh, kvh, dev):
    if qh < kvh or qh % kvh:
        _refuse(f"q: {qh} heads are no multiple of the {kvh} key heads")
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not -1e30 <= scale <= 1e30:  # and its quotient by a cap in 32 bits
        _refuse(f"scale: from -1e30 to 1e30, got {scale}")
    # The kernels take the tanh from one exponential, whose error is the
    # cap's size times 2^-23: 3e-4 of a logit at the largest.
    if softcap and not 1e-6 <= softcap <= 1000.0:
        _refuse(f"softcap: 0 or from 1e-6 to 1000, got {softcap}")
    if slopes is not None:
        _array("slopes", slopes, _F32, (qh,), dev)
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

    The pools' rows have memory of their own, apart from each other (one pool
    may hold what serves as both) and from k and v. No two tokens may be for
    the same row: sequences that share a page write behind it.
    """
    fields, (block, kvh, d, b, room) = _cache(k_pool, v_pool, block_table,
                                              seq_lens)
    dev, dtype = k_pool.device, k_pool.dtype
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        _no_backward()
    _no_tangents(k, v, k_pool, v_pool)
    tokens = k.shape[0]
    if k.shape != (tokens, kvh, d) or v.shape != k.shape:
        _refuse(f"k: and v: [T, {kvh}, {d}], got {tuple(k.shape)} and "
                f"{tuple(v.shape)}")
    _heads("k", k, dtype, dev)
    _heads("v", v, dtype, dev)
    if cu_seqlens is not None:
        _array("cu_seqlens", cu_seqlens, None, (b + 1,), dev)
    elif tokens != b:
        _refuse(f"k: one token for each of {b} sequences, got {tokens}; "
                "packed tokens need cu_seqlens")
    if key_pos is not None and pos is not None:
        _array("key_pos", key_pos, _I32, (b, kvh, room), dev)
        _array("pos", pos, None, (tokens,), dev)
    elif key_pos is not pos:
        _refuse("key_pos and pos: both or neither")
    if not tokens or not b:
        return
    x, y = k.data_ptr(), v.data_ptr()
    x0, x1, _ = k.stride()
    y0, y1, _ = v.stride()
    begin, end, begin2, end2 = _writes(k_pool, v_pool, fields)
    x_end = x + 2 * ((tokens - 1) * x0 + (kvh - 1) * x1 + d)
    y_end = y + 2 * ((tokens - 1) * y0 + (kvh - 1) * y1 + d)
    if x < end and begin < x_end or x < end2 and begin2 < x_end \
            or y < end and begin < y_end or y < end2 and begin2 < y_end:
        _refuse("k and v: apart from the pools")
    if begin == begin2 and (x, x0, x1) != (y, y0, y1):
        _refuse("k_pool and v_pool: one pool takes one k as v")
    if dev.type == "cuda":
        _call("paged_append", dev, fields, x, x0, x1, y, y0, y1, tokens,
              _ptr(cu_seqlens), _is64(cu_seqlens), _ptr(key_pos), _ptr(pos),
              _is64(pos))
        return
    n = k_pool.shape[0]
    for i in range(b):
        lo = i if cu_seqlens is None else max(int(cu_seqlens[i]), 0)
        hi = i + 1 if cu_seqlens is None else min(int(cu_seqlens[i + 1]),
                                                  tokens)
        first = lo if cu_seqlens is None else int(cu_seqlens[i])
        for t in range(lo, hi):
            slot = max(int(seq_lens[i]), 0) + t - first
            if slot >= room:
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
    softcap * tanh(s / softcap) for a softcap from 1e-6 to 1000 (0: none),
    then less slopes[h] * |i-j| if `slopes` [qh] fp32 are given, with the
    query's position i and the key's position j: the last slot's and the
    key's slot number, or `q_pos` [B] and `key_pos` [B, kvh, room] int32 for
    a cache whose rows have moved.

    `mass` [B, kvh, room] fp32 asks for the attention weights: returned is
    mass plus, for each slot, the weights that the key head's query heads
    gave it, and 0 for the slots past the length. It is a new tensor, or
    `mass_out`, which may be `mass` itself.

    Returns out [B, qh, d], and in this order, where asked for, the log of
    the sum of exponentials [B, qh] fp32 and the weights. A sequence that
    sees no key gets zeros and -inf. A value that is no finite number counts
    in full, however small its weight is. Values are summed in 32 bits before
    the weights' sum divides them, so finite ones are to stay below 2^90.
    """
    fields, (block, kvh, d, b, room) = _cache(k_pool, v_pool, block_table,
                                              seq_lens)
    dev = k_pool.device
    if torch.is_grad_enabled() and (
            q.requires_grad or mass is not None and mass.requires_grad
            or slopes is not None and slopes.requires_grad):
        _no_backward()
    _no_tangents(q, k_pool, v_pool, mass, slopes)
    if q.dim() != 3 or q.shape[0] != b or q.shape[2] != d:
        _refuse(f"q: [{b}, qh, {d}], got {tuple(q.shape)}")
    qh = q.shape[1]
    if d != 128 and d != 64:
        _refuse(f"q: d of 64 or 128, got {d}")
    _heads("q", q, k_pool.dtype, dev)
    scale, softcap = _score_args(scale, softcap, slopes, d, qh, kvh, dev)
    if key_pos is not None and q_pos is not None:
        _array("key_pos", key_pos, _I32, (b, kvh, room), dev)
        _array("q_pos", q_pos, None, (b,), dev)
    elif key_pos is not q_pos:
        _refuse("key_pos and q_pos: both or neither")
    if mass is not None:
        _array("mass", mass, _F32, (b, kvh, room), dev)
        if mass_out is None:
            mass_out = torch.empty_like(mass)
        else:
            _array("mass_out", mass_out, _F32, (b, kvh, room), dev)
            if mass_out.data_ptr() != mass.data_ptr() \
                    and _overlap(mass, mass_out):
                _refuse("mass_out: mass itself, or apart from it")
    elif mass_out is not None:
        _refuse("mass_out: needs mass")
    cuda = dev.type == "cuda"
    out = torch.empty((b, qh, d), dtype=q.dtype, device=dev)
    lse = torch.empty((b, qh), dtype=_F32, device=dev) \
        if return_lse or not cuda else None
    if b and cuda:
        ws = torch.empty(_native().paged_decode_workspace(
            b, qh, kvh, d, room, mass is not None), dtype=torch.uint8,
            device=dev)
        _call("paged_decode", dev, fields, q.data_ptr(), q.stride(0),
              q.stride(1), qh, scale, softcap, _ptr(slopes), _ptr(key_pos),
              _ptr(q_pos), _is64(q_pos), out.data_ptr(), _ptr(lse),
              _ptr(mass), _ptr(mass_out), ws.data_ptr())
    elif b:
        _decode_cpu(q, k_pool, v_pool, block_table, seq_lens, scale, softcap,
                    slopes, key_pos, q_pos, mass, mass_out, out, lse)
    if mass is not None:
        return (out, lse, mass_out) if return_lse else (out, mass_out)
    return (out, lse) if return_lse else out


def _weights_cpu(s: torch.Tensor):
    """Softmax over the last axis and its log-sum-exp; rows of -inf weigh
    nothing. The maximum and the sum stay apart, since a large maximum
    swallows the log of the sum."""
    if not s.shape[-1]:
        return s, s.new_full(s.shape[:-1], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    return w, (top + torch.log(total))[..., 0]


def _sums_cpu(w, v, seen):
    """w [..., m, n] times v [..., n, d]; a value that is no finite number
    counts for the rows that see it, `seen` [m, n], however small its weight
    is, and for no other."""
    wild = ~torch.isfinite(v)
    o = torch.matmul(w, torch.where(wild, 0.0, v))
    keys = wild.any(-1).flatten(0, -2).any(0).nonzero()[:, 0]
    for j in keys.tolist():
        o[..., seen[:, j], :] += torch.where(
            wild[..., j, None, :], v[..., j, None, :], 0.0)
    return o


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
        out[b] = _sums_cpu(w, v, torch.ones(g, len(at), dtype=torch.bool)) \
            .view(-1, d).to(out.dtype)
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
    the largest, of equal ones the lowest slot stays). A slot whose page is
    not there holds no row: it stays only if all that have one do, the lowest
    first.

    The rows that stay are moved into the slots below the budget in place:
    the i-th slot below it that became free takes the i-th kept row from
    above it, all others stay where they are. So the slots' order is lost,
    and `key_pos` [B, kvh, room] int32 holds each slot's position. A newest
    position is the largest of a sequence's slots.

    Returns the lengths, weights and positions afterwards, with 0 and -1 in
    the slots past the new length: new tensors, or those of `out`, which may
    be the inputs themselves. A row that would move to a page that is not
    there is dropped. A page is moved by the one sequence that holds
    it: pages that sequences share must not be evicted from.
    """
    fields, (block, kvh, d, b, room) = _cache(k_pool, v_pool, block_table,
                                              seq_lens)
    dev = k_pool.device
    _writes(k_pool, v_pool, fields)
    if mass.requires_grad and torch.is_grad_enabled():
        _no_backward()
    _no_tangents(k_pool, v_pool, mass)
    _array("mass", mass, _F32, (b, kvh, room), dev)
    _array("key_pos", key_pos, _I32, (b, kvh, room), dev)
    budget, recent = int(budget), int(recent)
    if not 1 <= budget < 1 << 31:
        _refuse(f"budget: at least 1, got {budget}")
    if not 0 <= recent <= budget:
        _refuse(f"recent: from 0 to the budget of {budget}, got {recent}")
    if out is None:
        out = (torch.empty_like(seq_lens), torch.empty_like(mass),
               torch.empty_like(key_pos))
    else:
        out = tuple(out)
        if len(out) != 3:
            _refuse("out: (seq_lens, mass, key_pos)")
        _array("out[0]", out[0], seq_lens.dtype, (b,), dev)
        _array("out[1]", out[1], _F32, (b, kvh, room), dev)
        _array("out[2]", out[2], _I32, (b, kvh, room), dev)
        for i, x in enumerate(out):
            for j, y in enumerate((seq_lens, mass, key_pos)):
                if (i != j or x.data_ptr() != y.data_ptr()) \
                        and _overlap(x, y):
                    _refuse("out: the inputs themselves, or apart from them")
            if any(_overlap(x, y) for y in out[:i]):
                _refuse("out: apart from each other")
    if not b:
        return out
    if dev.type == "cuda":
        ws = torch.empty(_native().kv_evict_workspace(b, kvh, room, budget),
                         dtype=torch.uint8, device=dev)
        _call("kv_evict", dev, fields, mass.data_ptr(), key_pos.data_ptr(),
              budget, recent, out[1].data_ptr(), out[2].data_ptr(),
              out[0].data_ptr(), ws.data_ptr())
        return out
    n = k_pool.shape[0]
    new_lens, new_mass = seq_lens.clone(), mass.clone()
    new_pos = key_pos.clone()
    for i in range(b):
        length = min(max(int(seq_lens[i]), 0), room)
        keep = min(length, budget)
        page = block_table[i].long()[torch.arange(length) // block]
        there = (page >= 0) & (page < n)
        for h in range(kvh if length > keep else 0):
            m, p = mass[i, h, :length], key_pos[i, h, :length].long()
            fresh = p > int(p.max()) - recent
            order = torch.sort(m, descending=True, stable=True).indices
            order = torch.cat([torch.nonzero(fresh & there)[:, 0],
                               order[(~fresh & there)[order]],
                               torch.nonzero(~there)[:, 0]])
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
    the document's first prefix_lens[i] keys; without it every query sees
    every key of its document. Scores are capped by `softcap`
    and lowered by `slopes` as in `paged_decode_op`, the distance being that
    from key position i + n - m.

    Returns out [T, qh, d] and, if asked for, the log of the sum of
    exponentials [T, qh] fp32. A row that sees no key gets zeros and -inf.
    Rows that belong to no document are left as they were in a given `out`,
    and are zeros and -inf in tensors that the call makes (a `lse` always).
    What the mask hides from a query does not count, whatever it holds; a
    value that is seen and is no finite number counts in full, however small
    its weight is, and finite ones are to stay below 2^90, as in
    `paged_decode_op`.
    """
    dev, dtype = q.device, q.dtype
    if q.dim() != 3 or k.dim() != 3:
        _refuse("q and k: [tokens, heads, d]")
    if dtype != _BF16 and dtype != _FP16:
        _refuse(f"q: bfloat16 or float16, got {dtype}")
    rows, qh, d = q.shape
    keys, kvh, dk = k.shape
    if d != 128 and d != 64:
        _refuse(f"q: d of 64 or 128, got {d}")
    if kvh < 1 or dk != d:
        _refuse(f"k: [Tk, kvh, {d}], got {tuple(k.shape)}")
    if v.shape != k.shape:
        _refuse("v: of k's shape")
    if rows >= 1 << 31 or keys >= 1 << 31:
        _refuse("q and k: fewer than 2^31 rows")
    if torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or v.requires_grad
            or slopes is not None and slopes.requires_grad):
        _no_backward()
    _no_tangents(q, k, v, slopes, out)
    _heads("q", q, dtype, dev)
    _heads("k", k, dtype, dev)
    _heads("v", v, dtype, dev)
    scale, softcap = _score_args(scale, softcap, slopes, d, qh, kvh, dev)
    if cu_seqlens.dim() != 1 or not cu_seqlens.shape[0]:
        _refuse("cu_seqlens: [documents + 1]")
    docs = cu_seqlens.shape[0] - 1
    _array("cu_seqlens", cu_seqlens, None, (docs + 1,), dev)
    if cu_seqlens_k is not None:
        _array("cu_seqlens_k", cu_seqlens_k, None, (docs + 1,), dev)
    elif keys != rows:
        _refuse("k: as many rows as q, or cu_seqlens_k")
    else:
        cu_seqlens_k = cu_seqlens
    if prefix_lens is not None:
        _array("prefix_lens", prefix_lens, None, (docs,), dev)
    clear = out is None
    if clear:
        out = torch.empty((rows, qh, d), dtype=dtype, device=dev)
    else:
        if out.shape != q.shape:
            _refuse(f"out: of q's shape, got {tuple(out.shape)}")
        _heads("out", out, dtype, dev)
        (x, n), (y, more) = sorted(zip(out.stride(), out.shape[:2]))
        if n > 1 and x < d or more > 1 and y < (x * (n - 1) if n > 1
                                                else 0) + d:
            _refuse("out: rows that do not share memory")
        if out.requires_grad and torch.is_grad_enabled():
            _no_backward()
        if _overlap(out, q) or _overlap(out, k) or _overlap(out, v):
            _refuse("out: apart from q, k and v")
    lse = torch.empty((rows, qh), dtype=_F32, device=dev) \
        if return_lse else None
    if rows and dev.type == "cuda":
        _call("packed_prefill", dev, q.data_ptr(), q.stride(0), q.stride(1),
              k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
              v.stride(0), v.stride(1), out.data_ptr(), out.stride(0),
              out.stride(1), _ptr(lse), rows, keys, qh, kvh, d,
              dtype == _FP16, docs, cu_seqlens.data_ptr(),
              cu_seqlens.dtype == _I64, cu_seqlens_k.data_ptr(),
              cu_seqlens_k.dtype == _I64, _ptr(prefix_lens),
              _is64(prefix_lens), causal, clear, scale, softcap,
              _ptr(slopes))
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
        seen = torch.ones(m, n, dtype=torch.bool)
        if causal:
            seen = j <= at
            if prefix is not None:
                seen = seen | (j < int(prefix[i]))
            s = s.masked_fill(~seen, float("-inf"))
        w, total = _weights_cpu(s)
        vf = v[k0:k0 + n].float().transpose(0, 1)   # [kvh, n, d]
        o = _sums_cpu(w, vf[:, None], seen)
        out[q0:q1] = o.permute(2, 0, 1, 3).reshape(m, qh, d).to(out.dtype)
        if lse is not None:
            lse[q0:q1] = total.permute(2, 0, 1).reshape(m, qh)
