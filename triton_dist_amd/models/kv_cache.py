"""Static KV cache (capability parity with Triton-distributed
python/triton_dist/models/kv_cache.py:29-66: [L, B, maxlen, H, D] tensors +
an offset vector). The offset lives on DEVICE and all indexing/masking is
computed from it, so decode steps replay correctly under hipGraph capture.
"""
from __future__ import annotations

import torch


class KVCache:
    def __init__(self, n_layers: int, batch: int, max_len: int,
                 n_kv_heads: int, head_dim: int, device="cpu",
                 dtype=torch.bfloat16):
        self.n_layers, self.batch, self.max_len = n_layers, batch, max_len
        self.kvh, self.head_dim = n_kv_heads, head_dim
        shape = (n_layers, batch, max_len, n_kv_heads, head_dim)
        self.k = torch.zeros(shape, device=device, dtype=dtype)
        self.v = torch.zeros(shape, device=device, dtype=dtype)
        # device-resident so graph replays see the advancing offset
        self.offset = torch.zeros((), device=device, dtype=torch.int64)
        self._range = torch.arange(max_len, device=device)

    def reset(self):
        self.offset.zero_()

    def fill_prefill(self, layer: int, k: torch.Tensor, v: torch.Tensor):
        """k/v: [B, S, kvh, D]; writes positions [0, S). Host-shape static."""
        s = k.shape[1]
        self.k[layer, :, :s].copy_(k)
        self.v[layer, :, :s].copy_(v)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor):
        """Decode append at the device offset (graph-safe dynamic index)."""
        s = k.shape[1]
        idx = self.offset + torch.arange(s, device=k.device)
        self.k[layer].index_copy_(1, idx, k)
        self.v[layer].index_copy_(1, idx, v)

    def advance(self, s: int = 1):
        self.offset += s

    def view(self, layer: int, s_new: int):
        """Full-length K/V [B, kvh, maxlen, D] plus a bool mask [1,1,s,maxlen]
        marking valid key positions (<= offset + query index)."""
        ks = self.k[layer].transpose(1, 2)
        vs = self.v[layer].transpose(1, 2)
        qpos = self.offset + torch.arange(s_new, device=ks.device)
        mask = self._range.unsqueeze(0) <= qpos.unsqueeze(1)  # [s, maxlen]
        return ks, vs, mask.view(1, 1, s_new, self.max_len)


class PagedKVCache:
    """Block-paged KV pool (capability parity with the reference
    megakernel's paged cache, mega_triton_kernel/models/paged_kv_cache.py
    — behavior only): a shared pool of fixed-size blocks
    [n_blocks, block, kvh, D] per side with a per-sequence block table,
    blocks allocated on first touch. Serving engines get allocation at
    block granularity instead of max_len * batch up front.

    `gather_layer` materializes a contiguous [B, L, kvh, D] view for the
    kernels that want one. A decode step reads the pages themselves: after
    `reserve` has handed out pages, `begin_step`, for every layer `write`
    and `attend`, then `end_step`, all of it without the host and for
    sequences of unlike lengths, so that a step can be captured. With
    `weights` the cache also keeps the attention weight that each slot got
    and each slot's position, and `evict` cuts it to a budget by them.

    A step that the pages have no room for is refused by `begin_step`, where
    the host knows of it. Where it does not, in a replayed graph or with
    counts on the device, rows without a slot are dropped and `lost` tells
    of them."""

    def __init__(self, n_layers: int, batch: int, max_len: int,
                 n_kv_heads: int, head_dim: int, block: int = 64,
                 n_blocks: int = 0, device="cpu", dtype=torch.bfloat16,
                 weights: bool = False):
        assert max_len % block == 0
        self.n_layers, self.batch = n_layers, batch
        self.max_len, self.block = max_len, block
        self.kvh, self.head_dim = n_kv_heads, head_dim
        self.blocks_per_seq = max_len // block
        if n_blocks <= 0:
            n_blocks = batch * self.blocks_per_seq  # worst case
        self.n_blocks = n_blocks
        pool = (n_layers, n_blocks, block, n_kv_heads, head_dim)
        self.k_pool = torch.zeros(pool, device=device, dtype=dtype)
        self.v_pool = torch.zeros(pool, device=device, dtype=dtype)
        # block_table[b, j] = pool block id of sequence b's j-th block
        # (-1 = unallocated); shared across layers (same shape every layer)
        self.block_table = torch.full((batch, self.blocks_per_seq), -1,
                                      dtype=torch.int64, device=device)
        self.seq_len = torch.zeros(batch, dtype=torch.int64, device=device)
        self._free_top = 0
        # of the step under way: its tokens, and the lengths with them
        self._count = torch.ones_like(self.seq_len)
        self._live = torch.zeros_like(self.seq_len)
        # slots that every sequence has pages for, and what no length is
        # above (None: not known), as far as the host was told; a captured
        # step moves lengths whenever it is replayed
        self._room, self._most, self._captured = 0, 0, False
        # the longest that a sequence was to become, and which lost rows
        self._peak = torch.zeros_like(self.seq_len)
        self._lost = torch.zeros_like(self.seq_len, dtype=torch.bool)
        # the position of a sequence's next token, which eviction leaves
        self.next_pos = torch.zeros_like(self.seq_len)
        self.mass = self.key_pos = None
        if weights:
            plane = (n_layers, batch, n_kv_heads, max_len)
            self.mass = torch.zeros(plane, device=device)
            self.key_pos = torch.full(plane, -1, device=device,
                                      dtype=torch.int32)

    def reset(self):
        self.block_table.fill_(-1)
        self.seq_len.zero_()
        self.next_pos.zero_()
        self._free_top = 0
        self._room, self._most = 0, 0
        self._peak.zero_()
        self._lost.zero_()
        if self.mass is not None:
            self.mass.zero_()
            self.key_pos.fill_(-1)

    # ------------------------------------------------- steps over the pages
    def reserve(self, upto_len: int):
        """Hand out pages for every sequence up to `upto_len` slots (on the
        host: once, outside of a captured step)."""
        if upto_len > self.max_len:
            raise ValueError(f"reserve: {upto_len} of {self.max_len} slots")
        self._lost.logical_or_(self.lost())  # before there are more pages
        self._ensure_blocks(upto_len)

    def _slots(self) -> torch.Tensor:
        """[B]: slots from a sequence's first on whose pages are there."""
        there = (self.block_table >= 0) & (self.block_table < self.n_blocks)
        return there.long().cumprod(1).sum(1) * self.block

    def lost(self) -> torch.Tensor:
        """[B] bool: sequences that steps since the last `reset` wanted more
        slots for than there are pages now, or were at a `reserve` since; rows
        of theirs were dropped."""
        return self._lost | (self._peak > self._slots())

    def _make_sure(self, counts):
        """Refuses a step that has no room. What the host was told decides;
        if that does not, lengths and pages are looked at."""
        if self.seq_len.is_cuda and torch.cuda.is_current_stream_capturing():
            self._captured = True
            return
        if isinstance(counts, torch.Tensor):
            if counts.is_cuda:
                self._most = None
                return
            new = int(counts.max()) if counts.numel() else 0
        else:
            new = int(counts)
        if self._captured or self._most is None \
                or self._most + new > self._room:
            lens, slots = self.seq_len.cpu(), self._slots().cpu()
            short = (lens + counts > slots).nonzero()[:, 0].tolist()
            if short:
                i = short[0]
                raise RuntimeError(
                    f"PagedKVCache: no room for the step in sequences "
                    f"{short}; {i} holds {int(lens[i])} tokens and has pages "
                    f"for {int(slots[i])} of {self.max_len} slots")
            self._room = int(slots.min()) if self.batch else 0
            self._most = int(lens.max()) if self.batch else 0
        self._most += new

    def begin_step(self, counts=1):
        """A step that adds `counts` tokens to the sequences: one number, or
        [B] of them. Raises RuntimeError, and changes nothing, if a sequence
        has no pages for them; counts on the device are not looked at."""
        self._make_sure(counts)
        if isinstance(counts, torch.Tensor):
            self._count.copy_(counts)
        else:
            self._count.fill_(counts)
        torch.add(self.seq_len, self._count, out=self._live)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor,
              cu_seqlens: "torch.Tensor | None" = None):
        """The step's keys and values: [B, kvh, D] with one token a
        sequence, or packed [T, kvh, D] with `cu_seqlens` [B + 1]."""
        from ..ops.paged import paged_append_op

        key_pos = pos = None
        if self.mass is not None:
            key_pos, pos = self.key_pos[layer], self.next_pos
            if cu_seqlens is not None:
                at = torch.arange(k.shape[0], device=k.device)
                cu = cu_seqlens.to(torch.int64)
                seq = torch.searchsorted(cu[1:].contiguous(), at, right=True)
                seq.clamp_(max=self.batch - 1)
                pos = pos[seq] + at - cu[seq]
        paged_append_op(k, v, self.k_pool[layer], self.v_pool[layer],
                        self.block_table, self.seq_len,
                        cu_seqlens=cu_seqlens, key_pos=key_pos, pos=pos)

    def attend(self, layer: int, q: torch.Tensor, **score) -> torch.Tensor:
        """Attention of the step's last token of each sequence, q [B, qh, D]
        to [B, qh, D], over the slots with the step's own. `score`: scale,
        softcap and slopes of `paged_decode_op`."""
        from ..ops.paged import paged_decode_op

        at = (q, self.k_pool[layer], self.v_pool[layer], self.block_table,
              self._live)
        if self.mass is None:
            return paged_decode_op(*at, **score)
        last = self.next_pos + self._count - 1
        return paged_decode_op(*at, key_pos=self.key_pos[layer], q_pos=last,
                               mass=self.mass[layer],
                               mass_out=self.mass[layer], **score)[0]

    def end_step(self):
        torch.clamp(self._live, max=self.max_len, out=self.seq_len)
        torch.maximum(self._peak, self._live, out=self._peak)
        self.next_pos.add_(self._count)

    def evict(self, budget: int, recent: int):
        """Between steps: cut every sequence to `budget` slots, in every
        layer and for every key head by its own weights (`kv_evict_op`). A
        next step needs a slot: the budget is to lie below what is reserved.
        """
        from ..ops.paged import kv_evict_op

        if self.mass is None:
            raise RuntimeError("PagedKVCache.evict: made without weights")
        for layer in range(self.n_layers):
            kv_evict_op(self.k_pool[layer], self.v_pool[layer],
                        self.block_table, self.seq_len, self.mass[layer],
                        self.key_pos[layer], budget, recent,
                        out=(self._live, self.mass[layer],
                             self.key_pos[layer]))
        self.seq_len.copy_(self._live)
        if self._most is not None:
            self._most = min(self._most, budget)

    def _ensure_blocks(self, upto_len: int):
        """Allocate pool blocks for every sequence up to `upto_len`
        positions (host-side allocator; block ids land in the table)."""
        need = (upto_len + self.block - 1) // self.block
        table = self.block_table
        for j in range(need):
            col = table[:, j]
            missing = (col < 0).nonzero(as_tuple=True)[0]
            if missing.numel():
                n = missing.numel()
                if self._free_top + n > self.n_blocks:
                    raise RuntimeError("PagedKVCache: pool exhausted")
                ids = torch.arange(self._free_top, self._free_top + n,
                                   device=table.device)
                table[missing, j] = ids
                self._free_top += n
        self._room = max(self._room, need * self.block)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor,
               pos0: int):
        """k/v: [B, S, kvh, D] written at positions [pos0, pos0+S)."""
        if self.mass is not None:
            raise RuntimeError("PagedKVCache.append: a cache with weights "
                               "takes its tokens by write")
        b, s = k.shape[0], k.shape[1]
        self._ensure_blocks(pos0 + s)
        for off in range(s):
            p = pos0 + off
            blk = self.block_table[:, p // self.block]     # [B]
            self.k_pool[layer, blk, p % self.block] = k[:, off]
            self.v_pool[layer, blk, p % self.block] = v[:, off]
        if layer == self.n_layers - 1:
            self.seq_len.fill_(pos0 + s)
            self._most = pos0 + s

    def gather_layer(self, layer: int, upto_len: int):
        """Contiguous [B, upto_len, kvh, D] views for the decode kernels."""
        nb = (upto_len + self.block - 1) // self.block
        blk = self.block_table[:, :nb].clamp(min=0)        # [B, nb]
        k = self.k_pool[layer, blk]                        # [B, nb, blk,...]
        v = self.v_pool[layer, blk]
        shp = (self.batch, nb * self.block, self.kvh, self.head_dim)
        return k.reshape(shp)[:, :upto_len], v.reshape(shp)[:, :upto_len]


class HybridCache(KVCache):
    """KVCache + per-GDN-layer recurrent state for hybrid (Qwen3-Next
    style) stacks. GDN state is positionless fp32 [B, local_heads, K, V],
    zeroed on reset; attention layers use the inherited paged-less KV
    slots (GDN layers simply never touch theirs)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self._gdn = {}

    def gdn_state(self, layer: int, batch: int, lh: int, dk: int,
                  dv: int) -> "torch.Tensor":
        key = layer
        if key not in self._gdn:
            self._gdn[key] = torch.zeros(batch, lh, dk, dv,
                                         dtype=torch.float32,
                                         device=self.k.device)
        return self._gdn[key]

    def reset(self):
        super().reset()
        for t in self._gdn.values():
            t.zero_()
