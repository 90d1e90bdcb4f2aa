// td/paged.hpp — what the operators over a paged key-value cache share: the
// description of a cache, the way from a position to its row, and the score
// of one query-key pair.
#pragma once

#include <hip/hip_runtime.h>

#include "td/device.hpp"

namespace td {

// An int32 or int64 array on the device. Lengths, offsets and page numbers
// come in either; the branch is uniform and costs one scalar compare.
struct IdxPtr {
  const void *p;
  int is64;
  TD_DEV long operator[](long i) const {
    return is64 ? ((const long *)p)[i] : (long)((const int *)p)[i];
  }
};

// One layer of a paged cache: k and v are [n_blocks, block, kvh, d] with
// strides in elements (the innermost is 1), table is [batch, max_blocks].
struct PagedArgs {
  void *k, *v;
  long k_page, k_row, k_head;
  long v_page, v_row, v_head;
  long n_blocks;
  int block, kvh, d;
  int is_fp16;
  IdxPtr table;
  long table_stride;
  int max_blocks;
  IdxPtr lens;
  int batch;

  __host__ __device__ int room() const { return max_blocks * block; }
  // A length below zero counts as zero, one past the table as the table's.
  TD_DEV int len(int b) const {
    long n = lens[b];
    return n < 0 ? 0 : n > room() ? room() : (int)n;
  }
  // The page of a sequence's slot; -1 where the table names none. Nothing
  // is ever read or written through a page outside the pool.
  TD_DEV long page(int b, int slot) const {
    long p = table[b * table_stride + (unsigned)slot / (unsigned)block];
    return p >= 0 && p < n_blocks ? p : -1;
  }
};

// Of all lanes, to all lanes: lane i takes from lanes 1, 2, 4 and 8 before it
// in its row of 16, then rows 1 and 3 from the row before, then 2 and 3 from
// lane 31, which leaves the whole in lane 63.
#define TD_WAVE_STEPS(X) \
  X(0x111, 0xf) X(0x112, 0xf) X(0x114, 0xf) X(0x118, 0xf) X(0x142, 0xa) \
  X(0x143, 0xc)
TD_DEV float wave_max(float x) {
#define TD_STEP(ctrl, rows)                                                 \
  x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(                 \
                   __float_as_uint(x), __float_as_uint(x), ctrl, rows, 0xf, \
                   false)));
  TD_WAVE_STEPS(TD_STEP)
#undef TD_STEP
  return __uint_as_float(
      __builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
TD_DEV int wave_max(int x) {
#define TD_STEP(ctrl, rows) \
  x = max(x, __builtin_amdgcn_update_dpp(x, x, ctrl, rows, 0xf, false));
  TD_WAVE_STEPS(TD_STEP)
#undef TD_STEP
  return __builtin_amdgcn_readlane(x, 63);
}
TD_DEV float wave_sum(float x) {
#define TD_STEP(ctrl, rows)                                             \
  x += __uint_as_float(__builtin_amdgcn_update_dpp(                     \
      0, __float_as_uint(x), ctrl, rows, 0xf, true));
  TD_WAVE_STEPS(TD_STEP)
#undef TD_STEP
  return __uint_as_float(
      __builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
// Sums over the lanes up to and with this one.
TD_DEV int wave_scan(int x) {
#define TD_STEP(ctrl, rows) \
  x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, true);
  TD_WAVE_STEPS(TD_STEP)
#undef TD_STEP
  return x;
}

// Infinite or not a number.
TD_DEV bool wild(__bf16 x) {
  return (__builtin_bit_cast(unsigned short, x) & 0x7f80) == 0x7f80;
}
TD_DEV bool wild(_Float16 x) {
  return (__builtin_bit_cast(unsigned short, x) & 0x7c00) == 0x7c00;
}

// How a score becomes a logit: capped by a tanh, then lowered by the
// distance between the query's and the key's position.
struct ScoreArgs {
  float scale;
  float softcap;        // 0: none
  const float *slopes;  // [qh] or null
};

void launch_paged_append(const PagedArgs &a, const void *k, long k_tok,
                         long k_head, const void *v, long v_tok, long v_head,
                         long tokens, IdxPtr cu, int *key_pos, IdxPtr pos,
                         hipStream_t stream);

struct PagedDecodeArgs {
  PagedArgs c;
  ScoreArgs s;
  const void *q;  // [batch, qh, d], strides in elements
  long q_tok, q_head;
  int qh;
  const int *key_pos;  // [batch, kvh, room] or null
  IdxPtr q_pos;        // [batch], read where key_pos is
  void *out;           // [batch, qh, d]
  float *lse;          // [batch, qh] or null
  const float *mass;   // [batch, kvh, room] or null
  float *mass_out;     // [batch, kvh, room], may be mass itself
  void *ws;
};
size_t paged_decode_workspace(int batch, int qh, int kvh, int d, long room,
                              bool mass);
void launch_paged_decode(const PagedDecodeArgs &a, hipStream_t stream);

struct EvictArgs {
  PagedArgs c;
  const float *mass;
  const int *key_pos;
  int budget, recent;
  float *mass_out;
  int *key_pos_out;
  void *lens_out;  // of the type of c.lens
  void *ws;
};
size_t kv_evict_workspace(int batch, int kvh, long room, int budget);
void launch_kv_evict(const EvictArgs &a, hipStream_t stream);

// kernels/packed_attn.hip
struct PackedArgs {
  const void *q, *k, *v;
  long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void *out;  // [rows, qh, d], strides in elements
  long out_tok, out_head;
  float *lse;  // [rows, qh] or null
  long rows, keys;
  int qh, kvh, d, is_fp16, seqs;
  IdxPtr cu_q, cu_k;  // [seqs + 1]
  IdxPtr prefix;      // [seqs] or null
  int causal;
  int clear_tail;  // write zeros behind the last sequence
  ScoreArgs s;
};
void launch_packed_prefill(const PackedArgs &a, hipStream_t stream);

}  // namespace td
