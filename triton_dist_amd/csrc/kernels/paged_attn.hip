// Operators over a paged key-value cache: new rows go to their pages,
// attention of one new token a sequence, eviction by accumulated weight.
#include <stdexcept>
#include <string>

#include "td/api.hpp"
#include "td/paged.hpp"

namespace td {

namespace {

using bf16 = __bf16;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

void launched(const char *what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}

// A launch counts threads in 32 bits, and workgroups past the first dimension
// in 16.
void check_grid(const char *what, long x, long threads, long y = 1,
                long z = 1) {
  if (x * threads > 0xffffffffL || y > 0xffff || z > 0xffff)
    throw std::runtime_error(
        std::string(what) + ": too large, " + std::to_string(x) + " x " +
        std::to_string(y) + " x " + std::to_string(z) + " workgroups");
}

// ---------------------------------------------------------------------------
// append: one thread moves 16 bytes of a token's keys and values.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_paged_append(
    PagedArgs a, const bf16 *__restrict__ k, long k_tok, long k_head,
    const bf16 *__restrict__ v, long v_tok, long v_head, long tokens,
    IdxPtr cu, int *key_pos, IdxPtr pos) {
  const int chunks = a.d / 8;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long t = i / (a.kvh * chunks);
  if (t >= tokens) return;
  const int h = (int)(i / chunks % a.kvh), c = (int)(i % chunks);
  int b = (int)t;
  unsigned long past = 0;  // slots behind the length; an offset may be anything
  if (cu.p) {
    int lo = 0, hi = a.batch;  // the sequence with cu[b] <= t < cu[b + 1]
    while (lo < hi) {
      int mid = (lo + hi) >> 1;
      if (cu[mid + 1] <= t) lo = mid + 1; else hi = mid;
    }
    if (lo >= a.batch || t < cu[lo]) return;
    b = lo;
    past = (unsigned long)t - (unsigned long)cu[b];
  }
  const unsigned long slot = a.len(b) + past;
  if (past >= (unsigned long)a.room() || slot >= (unsigned long)a.room())
    return;
  const long page = a.page(b, (int)slot);
  if (page < 0) return;
  const int row = (int)slot % a.block;
  *(u32x4 *)((bf16 *)a.k + page * a.k_page + row * a.k_row + h * a.k_head +
             c * 8) = *(const u32x4 *)(k + t * k_tok + h * k_head + c * 8);
  *(u32x4 *)((bf16 *)a.v + page * a.v_page + row * a.v_row + h * a.v_head +
             c * 8) = *(const u32x4 *)(v + t * v_tok + h * v_head + c * 8);
  if (key_pos && c == 0)
    key_pos[((long)b * a.kvh + h) * a.room() + slot] = (int)pos[t];
}

// ---------------------------------------------------------------------------
// decode
//
// Bound by reading K and V once. The batch's keys are cut into chunks of
// equal length on the device, from the lengths as they are, so a long
// sequence among short ones is spread over the card as well. A wave takes a
// key head of one and up to 16 of its query heads, or a quarter of the tiles
// of that (find_cut).
//
// A wave goes through its 32-key tiles without a barrier. S^T = K Q^T and
// O^T = V^T P^T, so that a lane holds the scores of one query head all the
// way: lane (n, qd) = (lane & 15, lane >> 4) gets from the 16x16x32 matrix
// instructions the scores of head n and keys 16 t + 4 qd + i, which are the
// elements that the second product wants from it, once its 32 keys are
// numbered (qd, t, i). K goes from global memory to the operand's registers;
// V takes a way through the wave's piece of LDS, where it is read transposed.
//
// The weights meet V in the inputs' type, as a rounded part and the rounded
// rest: the second product is far from bounding the kernel, and with it the
// output's own rounding is the only one that counts. fp16 has no numbers
// below 2^-24, so its weights are lifted by 2^15 while they are summed: of
// those less than 2^-39 of the maximum nothing is left (2^-24 without).
// ---------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
template <typename T> constexpr float kLift = 1.f;
template <> constexpr float kLift<_Float16> = 32768.f;
constexpr int kTile = 32;              // keys of a wave's step
constexpr int kStep = 4 * kTile;       // keys that chunks are measured in
constexpr int kSlots = 512;            // workgroups that the card holds
// Steps that a workgroup starts for. Neither side of it suits all: at 12,
// 16 sequences of 4000 keys with 8 key heads take 55 us for 61 and 100 of 500
// 50 for 58, but 512 of 131 take 70 for 63; at 3, 64 of up to 4100 with 4 key
// heads take 58 for 61, but one of 30000 with 8 takes 37 for 33.
constexpr int kFew = 6;

template <typename T> using vec8 = __attribute__((ext_vector_type(8))) T;
template <typename T> using vec4 = __attribute__((ext_vector_type(4))) T;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
// at any float's address
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(4)));

TD_DEV f32x4 mfma16(vec8<bf16> a, vec8<bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
TD_DEV f32x4 mfma16(vec8<_Float16> a, vec8<_Float16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Of each 16 lanes, lane l gets column l of the 4x16 block whose row l / 4
// and columns 4 (l % 4) on its pointer names.
TD_DEV s16x4 read_transposed(const void *lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4 *)(unsigned)(uintptr_t)lds);
}
// Orders a wave's own LDS traffic for the compiler; the hardware keeps it
// in order.
TD_DEV void wave_fence() {
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// The power of two of a rounded logit less a maximum of such: taken off the
// unrounded product, the largest would differ by its maximum's rounding.
TD_DEV float power_of(float logit, float top) {
#pragma clang fp contract(off)
  return __builtin_amdgcn_exp2f(logit - top);
}

TD_DEV float lse_of(float top, float sum) {
  return sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// A part's share in a sum. One that is no finite number counts in full,
// however small its share is.
TD_DEV float share_of(float r, float x) {
  return fabsf(x) < INFINITY ? r * x : x;
}

struct Chunk {
  int b, len;        // sequence and its length
  int first, count;  // this chunk's number among the sequence's, how many
};

// Where a call keeps what its kernels hand on.
struct DecodeWork {
  float *part;    // [chunks, qh, d]: outputs of one chunk among several
  // [chunks, qh]: a chunk's largest logit, in units of log2, and the sum of
  // its powers less that one. They stay apart, since past 2^24 a maximum
  // swallows the log of its sum.
  float2 *sum;
  int *plan;      // [batch, 2]: a sequence's chunks, its first further one
  float *logits;  // [batch, qh, room], in units of log2, where weights are
  int groups;     // of up to 16 query heads of a key head
  int apart;      // waves never share a chunk
  int least;      // steps of a chunk
  int joins;      // workgroups that join a key head's query heads
};

// How the batch's keys are cut, from the lengths as they are. A sequence's
// first chunk has the sequence's number; further ones are numbered behind
// those, sequence by sequence. All of a workgroup of 256 threads calls this.
struct Cut {
  int steps;   // a chunk's length
  int most;    // further chunks at most
  bool shared; // a workgroup's waves share one head's chunk
};
TD_DEV int steps_of(int len) { return (len + kStep - 1) / kStep; }
TD_DEV int chunks_of(int len, int steps) {
  return max(1, (steps_of(len) + steps - 1) / steps);
}
TD_DEV Cut find_cut(const PagedArgs &c, const DecodeWork &w, int *lds) {
  const int tid = threadIdx.x, each = (c.batch + 255) / 256;
  int sum = 0;
  for (int i = tid * each; i < min((tid + 1) * each, c.batch); ++i)
    sum += steps_of(c.len(i));
  sum = wave_scan(sum);
  if ((tid & 63) == 63) lds[tid >> 6] = sum;
  __syncthreads();
  const long total = (long)lds[0] + lds[1] + lds[2] + lds[3];
  const int per = c.kvh * w.groups, own = (per + 3) / 4;
  Cut cut;
  // Few steps for a workgroup: its waves share one, which is done soonest
  // (32 sequences of up to 4100 keys, 4 key heads: 24 us for 28). Else each
  // wave has a key head of its own, so that a workgroup reads neighbouring
  // heads' rows and joins nothing (48 of up to 16384, 8 key heads: 203 us
  // for 228), in twice the chunks that the card holds, which evens out what
  // ragged sequences leave over.
  cut.shared = !w.apart && total * per < kFew * kSlots;
  const long target = cut.shared ? (kSlots + per - 1) / per
                                 : (2 * kSlots + own - 1) / own;
  cut.steps = max(w.least, (int)((total + target - 1) / target));
  cut.most = (int)(total / cut.steps);
  return cut;
}
// The further chunk `at`; false where there are not so many.
TD_DEV bool find_further(const PagedArgs &c, const Cut &cut, int at,
                         int *lds, Chunk &out) {
  if (at >= cut.most) return false;
  const int tid = threadIdx.x, each = (c.batch + 255) / 256;
  int own = 0;
  for (int i = tid * each; i < min((tid + 1) * each, c.batch); ++i)
    own += chunks_of(c.len(i), cut.steps) - 1;
  const int upto = wave_scan(own);
  __syncthreads();
  if ((tid & 63) == 63) lds[tid >> 6] = upto;
  __syncthreads();
  int before = upto - own, all = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < tid >> 6) before += lds[i];
    all += lds[i];
  }
  if (at >= all) return false;
  for (int i = tid * each; i < min((tid + 1) * each, c.batch); ++i) {
    const int n = chunks_of(c.len(i), cut.steps) - 1;
    if (at >= before && at < before + n) {
      lds[4] = i;
      lds[5] = at - before + 1;
    }
    before += n;
  }
  __syncthreads();
  out.b = lds[4];
  out.first = lds[5];
  out.len = c.len(out.b);
  out.count = chunks_of(out.len, cut.steps);
  return true;
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_paged_decode(PagedDecodeArgs a,
                                                         DecodeWork w) {
  constexpr int kC = D / 32, kT = D / 16;  // pieces of a row, tiles of it
  constexpr int kRow = D + 16;   // of V in LDS: 8 rows take all 64 banks
  constexpr int kORow = D + 4;   // of the outputs there, floats
  constexpr int kBytes = kTile * kRow * 2;
  static_assert(16 * kORow * 4 <= kBytes, "outputs fit where V was");
  __shared__ __attribute__((aligned(16))) char lds[4][kBytes];
  __shared__ float lds_m[4][16], lds_l[4][16];
  __shared__ int found[8];

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int n = lane & 15, qd = lane >> 4;
  const Cut cut = find_cut(a.c, w, found);
  const int per = a.c.kvh * w.groups;
  const int blocks = cut.shared ? per : (per + 3) / 4;  // of a chunk
  const int id = blockIdx.x / blocks;
  Chunk ch{id, 0, 0, 1};
  if (id >= a.c.batch) {
    if (!find_further(a.c, cut, id - a.c.batch, found, ch)) return;
  } else {
    ch.len = a.c.len(id);
    ch.count = chunks_of(ch.len, cut.steps);
  }
  if (tid == 0 && blockIdx.x % blocks == 0) {
    if (ch.first == 0) w.plan[2 * ch.b] = ch.count;
    if (ch.first == 1) w.plan[2 * ch.b + 1] = id;
  }
  const int stride = cut.shared ? kStep : kTile;
  const int share = cut.shared ? blockIdx.x % per
                               : blockIdx.x % blocks * 4 + wave;
  if (share >= per) return;  // and with it no barrier follows
  const int kh = share / w.groups, group = share % w.groups;
  const int g = a.qh / a.c.kvh;
  const int h0 = kh * g + group * 16;       // first query head here
  const int heads = min(16, g - group * 16);
  const int b = ch.b;
  const long long_cut = (long)cut.steps * kStep;
  const int k0 = (int)(ch.first * long_cut);
  const int k1 = (int)min((long)ch.len, k0 + long_cut);

  vec8<T> qf[kC] = {};
  if (n < heads) {
    const T *q = (const T *)a.q + b * a.q_tok + (h0 + n) * a.q_head + qd * 8;
#pragma unroll
    for (int c = 0; c < kC; ++c) qf[c] = *(const vec8<T> *)(q + c * 32);
  }
  const float scale = a.s.scale * kLog2e;
  const float cap = a.s.softcap * kLog2e;
  const float in_cap = a.s.softcap > 0.f ? 2.f * kLog2e * a.s.scale /
                                               a.s.softcap : 0.f;
  const float slope = a.s.slopes && n < heads ? a.s.slopes[h0 + n] * kLog2e
                                              : 0.f;
  const int *key_pos = a.key_pos ? a.key_pos + ((long)b * a.c.kvh + kh) *
                                                   a.c.room()
                                 : nullptr;
  const long q_at = key_pos ? a.q_pos[b] : (long)ch.len - 1;

  const T *kbase = (const T *)a.c.k + kh * a.c.k_head + qd * 8;
  const T *vbase = (const T *)a.c.v + kh * a.c.v_head + qd * 8;
  vec8<T> kf[2][kC], vf[2][kC];
  i32x4_any kp[2];  // positions of the loaded tile's keys 16 t + 4 qd + i
  int page[2];     // of the tile to load next
  bool ok[2];      // this lane's rows of the loaded tile are there
  auto look_up = [&](int base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int slot = base + 16 * t + n;
      page[t] = slot < k1 ? (int)a.c.page(b, slot) : -1;
    }
  };
  // Rows that are not there are read from the pool's first page instead,
  // masked as keys and cleared as values before they are used.
  auto load_k = [&](int base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const long p = max(page[t], 0);
      const unsigned r = (unsigned)(base + 16 * t + n) % (unsigned)a.c.block;
      const T *row = kbase + p * a.c.k_page + r * a.c.k_row;
#pragma unroll
      for (int c = 0; c < kC; ++c)
        kf[t][c] = *(const vec8<T> *)(row + c * 32);
      if (key_pos) {
        const int slot = base + 16 * t + 4 * qd;
        if (slot + 4 <= k1) {
          kp[t] = *(const i32x4_any *)(key_pos + slot);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            kp[t][i] = key_pos[min(slot + i, k1 - 1)];
        }
      }
    }
  };
  auto load_v = [&](int base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      ok[t] = page[t] >= 0;
      const long p = max(page[t], 0);
      const unsigned r = (unsigned)(base + 16 * t + n) % (unsigned)a.c.block;
      const T *row = vbase + p * a.c.v_page + r * a.c.v_row;
#pragma unroll
      for (int c = 0; c < kC; ++c)
        vf[t][c] = *(const vec8<T> *)(row + c * 32);
    }
  };

  float m = -INFINITY, l = 0.f;  // m of all quads alike, l of this lane
  f32x4 acc[kT] = {};
  T *vl = (T *)lds[wave];
  int base = k0 + (cut.shared ? wave * kTile : 0);
  if (base < k1) {
    look_up(base);
    load_k(base);
    load_v(base);
    look_up(base + stride);
  }
  for (; base < k1; base += stride) {
    const bool more = base + stride < k1;
    f32x4 s[2] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < kC; ++c) s[t] = mfma16(kf[t][c], qf[c], s[t]);
    float far[2][4];
    if (a.s.slopes) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          far[t][i] = fabsf((float)(
              key_pos ? q_at - kp[t][i]
                      : q_at - (base + 16 * t + 4 * qd + i)));
    }
    // which of the tile's 32 rows are there, seen by every lane
    const unsigned here = (unsigned)(__ballot(ok[0]) & 0xffff) |
                          (unsigned)(__ballot(ok[1]) & 0xffff) << 16;
    if (here != 0xffffffffu) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (!ok[t])
#pragma unroll
          for (int c = 0; c < kC; ++c) vf[t][c] = vec8<T>{};
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < kC; ++c)
        *(vec8<T> *)(vl + (16 * t + n) * kRow + c * 32 + qd * 8) = vf[t][c];
    wave_fence();
    if (more) {
      load_k(base + stride);
      load_v(base + stride);
      look_up(base + 2 * stride);
    }
    // scores, in units of log2
    if (a.s.softcap > 0.f) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][i] = cap - 2.f * cap *
                              __builtin_amdgcn_rcpf(
                                  1.f + __builtin_amdgcn_exp2f(s[t][i] *
                                                               in_cap));
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] *= scale;
    }
    if (a.s.slopes) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] -= slope * far[t][i];
    }
    if (here != 0xffffffffu) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(here >> (16 * t + 4 * qd + i) & 1)) s[t][i] = -INFINITY;
    }
    if (w.logits && n < heads) {
      float *to = w.logits + ((long)b * a.qh + h0 + n) * a.c.room() + base +
                  4 * qd;
      if (base + kTile <= k1) {
#pragma unroll
        for (int t = 0; t < 2; ++t) *(f32x4_any *)(to + 16 * t) = s[t];
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (base + 16 * t + 4 * qd + i < k1) to[16 * t + i] = s[t][i];
      }
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]),
                            fmaxf(s[0][2], s[0][3])),
                      fmaxf(fmaxf(s[1][0], s[1][1]),
                            fmaxf(s[1][2], s[1][3])));
    if (__any(top > m)) {  // seldom after the first tiles
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = fmaxf(m, top);
      const float r = __builtin_amdgcn_exp2f(
          m - (to == -INFINITY ? 0.f : to));
      m = to;
      l *= r;
#pragma unroll
      for (int t = 0; t < kT; ++t) acc[t] *= r;
    }
    const float safe = m == -INFINITY ? 0.f : m;
    vec8<T> hi, lo;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = power_of(s[t][i], safe) * kLift<T>;
        l += p;
        hi[4 * t + i] = (T)p;
        lo[4 * t + i] = (T)(p - (float)hi[4 * t + i]);
      }
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const T *at = vl + (4 * qd + (n >> 2)) * kRow + t * 16 + 4 * (n & 3);
      union { s16x4 half[2]; vec8<T> all; } v;
      v.half[0] = read_transposed(at);
      v.half[1] = read_transposed(at + 16 * kRow);
      acc[t] = mfma16(v.all, hi, acc[t]);
      acc[t] = mfma16(v.all, lo, acc[t]);
    }
    wave_fence();  // the next tile's values go where these were
  }

  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // A value that is no finite number makes its outputs so, however small its
  // weight. Times a weight that underflows, or a rounded weight's rest of
  // zero or less, an infinite one is NaN, so outputs that are NaN without a
  // score being one are summed again from such values alone.
  bool spoilt = false;
#pragma unroll
  for (int t = 0; t < kT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) spoilt |= acc[t][i] != acc[t][i];
  if (__any(spoilt && l == l)) {
    f32x4 alone[kT] = {};
    for (base = k0 + (cut.shared ? wave * kTile : 0); base < k1;
         base += stride) {
      bool open = false;  // NaN, and not yet by a value
#pragma unroll
      for (int t = 0; t < kT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          open |= acc[t][i] != acc[t][i] && alone[t][i] == alone[t][i];
      if (!__any(open)) break;
#pragma unroll 4
      for (int slot = base; slot < min(base + kTile, k1); ++slot) {
        const long p = a.c.page(b, slot);
        if (p < 0) continue;
        const T *row = (const T *)a.c.v + kh * a.c.v_head + p * a.c.v_page +
                       (long)((unsigned)slot % (unsigned)a.c.block) *
                           a.c.v_row + qd * 4;
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          const vec4<T> x = *(const vec4<T> *)(row + t * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            alone[t][i] += wild(x[i]) ? (float)x[i] : 0.f;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (acc[t][i] != acc[t][i] && alone[t][i] != 0.f)
          acc[t][i] = alone[t][i];
  }
  l *= 1.f / kLift<T>;
#pragma unroll
  for (int t = 0; t < kT; ++t) acc[t] *= 1.f / kLift<T>;
  if (!cut.shared) {
    if (n >= heads) return;
    const float r = l == 0.f ? 0.f : 1.f / l;
    const long at = (long)id * a.qh + h0 + n, to = (long)b * a.qh + h0 + n;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      acc[t] *= r;
      if (ch.count == 1) {
        vec4<T> o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = (T)acc[t][i];
        *(vec4<T> *)((T *)a.out + to * D + t * 16 + qd * 4) = o;
      } else {
        *(f32x4 *)(w.part + at * D + t * 16 + qd * 4) = acc[t];
      }
    }
    if (qd == 0) {
      w.sum[at] = make_float2(m, l);
      if (ch.count == 1 && a.lse) a.lse[to] = lse_of(m, l);
    }
    return;
  }
  // join the four waves
  float *ol = (float *)lds[wave];
#pragma unroll
  for (int t = 0; t < kT; ++t)
    *(f32x4 *)(ol + n * kORow + t * 16 + qd * 4) = acc[t];
  if (qd == 0) {
    lds_m[wave][n] = m;
    lds_l[wave][n] = l;
  }
  __syncthreads();
  for (int i = tid; i < heads * (D / 4); i += 256) {
    const int h = i / (D / 4), c = i % (D / 4) * 4;
    const float top = fmaxf(fmaxf(lds_m[0][h], lds_m[1][h]),
                            fmaxf(lds_m[2][h], lds_m[3][h]));
    const float safe = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o = {};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float r = __builtin_amdgcn_exp2f(lds_m[x][h] - safe);
      sum += r * lds_l[x][h];
      const f32x4 y = *(const f32x4 *)((const float *)lds[x] + h * kORow + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += share_of(r, y[e]);
    }
    o *= sum == 0.f ? 0.f : 1.f / sum;
    const long at = (long)id * a.qh + h0 + h, to = (long)b * a.qh + h0 + h;
    if (ch.count == 1) {
#pragma unroll
      for (int x = 0; x < 4; ++x) ((T *)a.out)[to * D + c + x] = (T)o[x];
      if (c == 0 && a.lse) a.lse[to] = lse_of(top, sum);
    } else {
      *(f32x4 *)(w.part + at * D + c) = o;
    }
    if (c == 0) w.sum[at] = make_float2(top, sum);
  }
}

// Joins a sequence's chunks and hands out its weights: of the workgroups
// (sequence, key head, z) the first w.joins share out the query heads, and
// each further one adds the weights of 1024 slots, from the logits that the
// first kernel kept.
constexpr int kSpan = 1024;    // slots
constexpr int kSpanWaves = 8;
template <typename T, int D>
__global__ __launch_bounds__(64 * kSpanWaves) void k_decode_finish(PagedDecodeArgs a,
                                                         DecodeWork w) {
  __shared__ float lds_top[kSpanWaves], lds_sum[kSpanWaves];
  __shared__ float lds_o[kSpanWaves][D];
  const int b = blockIdx.x, kh = blockIdx.y, z = blockIdx.z;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int g = a.qh / a.c.kvh, room = a.c.room();
  const int count = w.plan[2 * b], more = w.plan[2 * b + 1];
  auto row = [&](int i, int h) {  // a chunk's outputs of a query head
    return (long)(i ? more + i - 1 : b) * a.qh + h;
  };
  // all chunks' maximum and the sum of powers less that, by the whole wave
  auto sum_of = [&](int h, float &top, float &sum) {
    top = -INFINITY, sum = 0.f;
    for (int i = lane; i < count; i += 64)
      top = fmaxf(top, w.sum[row(i, h)].x);
    top = wave_max(top);
    if (top == -INFINITY) top = 0.f;  // nothing to sum
    for (int i = lane; i < count; i += 64) {
      const float2 x = w.sum[row(i, h)];
      sum += __builtin_amdgcn_exp2f(x.x - top) * x.y;
    }
    sum = wave_sum(sum);
  };
  if (z < w.joins) {
    if (count == 1) return;
    // heads of this workgroup, waves to a head, heads at once
    const int heads = (g + w.joins - 1) / w.joins;
    const int each = max(1, kSpanWaves / heads), at_once = kSpanWaves / each;
    for (int x = 0; x < heads; x += at_once) {
      const int y = x + wave / each, h = kh * g + z * heads + y;
      const bool live = wave < each * at_once && y < heads &&
                        z * heads + y < g;
      if (live) {
        float top, sum;
        sum_of(h, top, sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        float o[D / 64] = {};
#pragma unroll 4
        for (int i = wave % each; i < count; i += each) {
          const long at = row(i, h);
          const float2 x = w.sum[at];
          const float r = __builtin_amdgcn_exp2f(x.x - top) * x.y * inv;
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            o[c] += share_of(r, w.part[at * D + lane * (D / 64) + c]);
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          lds_o[wave][lane * (D / 64) + c] = o[c];
        if (wave % each == 0 && lane == 0 && a.lse)
          a.lse[(long)b * a.qh + h] = lse_of(top, sum);
      }
      __syncthreads();
      for (int i = tid; i < at_once * D; i += 64 * kSpanWaves) {
        const int p = i / D, c = i % D;
        if (x + p >= heads || z * heads + x + p >= g) continue;
        float sum = 0.f;
        for (int v = 0; v < each; ++v) sum += lds_o[p * each + v][c];
        ((T *)a.out)[((long)b * a.qh + kh * g + z * heads + x + p) * D + c] =
            (T)sum;
      }
      __syncthreads();
    }
    return;
  }
  constexpr int kOwn = kSpan / 64 / kSpanWaves;
  const int len = a.c.len(b), from = (z - w.joins) * kSpan + tid;
  const long plane = ((long)b * a.c.kvh + kh) * room;
  float sum[kOwn] = {};
  if ((z - w.joins) * kSpan < len)
    for (int x = 0; x < g; x += kSpanWaves) {
      const float *s = w.logits + ((long)b * a.qh + kh * g + x) * room + from;
      float logit[kSpanWaves][kOwn];
#pragma unroll
      for (int y = 0; y < kSpanWaves; ++y)
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int slot = from + i * 64 * kSpanWaves;
          logit[y][i] = x + y < g && slot < len
                            ? s[(long)y * room + i * 64 * kSpanWaves]
                            : -INFINITY;
        }
      float top = 0.f, total = 0.f;
      if (x + wave < g) sum_of(kh * g + x + wave, top, total);
      __syncthreads();
      if (lane == 0) lds_top[wave] = top, lds_sum[wave] = total;
      __syncthreads();
#pragma unroll
      for (int y = 0; y < kSpanWaves; ++y) {
        const float most = lds_top[y], all = lds_sum[y];
        if (all == 0.f) continue;  // also a head that is not there
        const float inv = 1.f / all;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          sum[i] += __builtin_amdgcn_exp2f(logit[y][i] - most) * inv;
      }
    }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int slot = from + i * 64 * kSpanWaves;
    if (slot < room)
      a.mass_out[plane + slot] = slot < len ? a.mass[plane + slot] + sum[i]
                                            : 0.f;
  }
}

// ---------------------------------------------------------------------------
// evict
//
// Two launches: a workgroup per sequence and key head finds what stays, does
// the bookkeeping and lists which row goes where; then all the card moves
// rows. Bound by latency in the first (up to four counts of the keys in
// LDS, each with its barriers), by the rows' bytes in the second. Rows that stay below the
// budget are not touched, so the steady state, one row over, moves one.
// ---------------------------------------------------------------------------
// Order of what stays: slots of the `recent` newest positions first, then
// by weight, NaN above all as a sort has it. Unsigned compare. 0 is no slot,
// and kGone one whose page is not there: it holds no row that could move, so
// it comes behind all others.
constexpr unsigned kGone = 1;
TD_DEV unsigned rank_key(float mass, bool is_recent) {
  if (is_recent) return 0xFFFFFFFFu;
  if (mass != mass) return 0xFFFFFFFEu;
  unsigned u = __float_as_uint(mass + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvict = 1024;              // threads, and slots of a pass
constexpr int kEvictWaves = kEvict / 64;
constexpr int kPairs = 32;                // rows that a workgroup moves

// What goes where: the i-th free slot below the budget takes the i-th kept
// row above it. ws: [batch, kvh, pairs] of these, then [batch, kvh] counts.
struct Pair {
  int to, from;
  float mass;  // the moved row's
  int pos;
};

// R passes of slots are kept in registers as keys; longer sequences (MANY)
// go by in parts of as many and are read again for each threshold.
template <int R, bool MANY>
__global__ __launch_bounds__(kEvict) void k_evict_select(EvictArgs a,
                                                         int pairs) {
  __shared__ int lds_n[kEvictWaves], lds_gone[kEvictWaves], hists[4][256];
  __shared__ int lds_c[2][R][kEvictWaves], lds_all[2];
  const int b = blockIdx.x / a.c.kvh, h = blockIdx.x % a.c.kvh;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int room = a.c.room(), len = a.c.len(b);
  const int keep = min(len, a.budget);
  const long row = ((long)b * a.c.kvh + h) * room;
  const float *mass = a.mass + row;
  const int *pos = a.key_pos + row;
  float *mass_out = a.mass_out + row;
  int *pos_out = a.key_pos_out + row;
  int *count = (int *)((Pair *)a.ws + (long)gridDim.x * pairs) + blockIdx.x;
  Pair *list = (Pair *)a.ws + (long)blockIdx.x * pairs;
  if (keep == len) {
    for (int i = tid; i < room; i += kEvict) {
      const float m = i < len ? mass[i] : 0.f;
      const int p = i < len ? pos[i] : -1;
      mass_out[i] = m;
      pos_out[i] = p;
    }
    if (tid == 0) *count = 0;
    return;
  }

  (&hists[0][0])[tid] = 0;
  // positions from the first one on count as recent
  unsigned key[R];
  float m[R];
  int p[R];
  long since = 0;
  bool gone = false;  // some page of the sequence's is not there
  constexpr int kPart = R * kEvict;
  auto read = [&](int part) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = part + r * kEvict + tid;
      m[r] = i < len ? mass[i] : 0.f;
      p[r] = i < len ? pos[i] : INT_MIN;
    }
  };
  {
    int newest = INT_MIN;
    for (int part = 0; part < (MANY ? len : 1); part += kPart) {
      read(part);
#pragma unroll
      for (int r = 0; r < R; ++r) newest = max(newest, p[r]);
    }
    const int used = (len - 1) / a.c.block + 1;
    for (int i = tid; i < used; i += kEvict) {
      const long page = a.c.table[b * a.c.table_stride + i];
      gone |= page < 0 || page >= a.c.n_blocks;
    }
    newest = wave_max(newest);
    gone = __any(gone);
    if (lane == 0) lds_n[wave] = newest, lds_gone[wave] = gone;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEvictWaves; ++i) {
      newest = max(newest, lds_n[i]);
      gone |= lds_gone[i] != 0;
    }
    since = (long)newest - a.recent + 1;
  }
  auto load = [&](int part) {
    if (MANY) read(part);
    unsigned lacks = 0;  // bit r: a slot without a page
    if (gone)
#pragma unroll 1
      for (int r = 0; r < R; ++r) {
        const int i = part + r * kEvict + tid;
        if (i < len && a.c.page(b, i) < 0) lacks |= 1u << r;
      }
#pragma unroll
    for (int r = 0; r < R; ++r)
      key[r] = part + r * kEvict + tid >= len ? 0
               : lacks >> r & 1               ? kGone
                                              : rank_key(m[r], p[r] >= since);
  };
  if (!MANY) load(0);

  // The keep-th largest key, eight bits at a time from the top, by counts of
  // the keys that agree so far. Of those that equal it, `need` stay.
  unsigned t = 0;
  int need = keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    int *hist = hists[shift / 8];
    for (int part = 0; part < (MANY ? len : 1); part += kPart) {
      if (MANY) load(part);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = key[r] && (shift == 24 || (key[r] ^ t) >> shift < 256);
        const int bin = key[r] >> shift & 255;
        const unsigned long long who = __ballot(in);
        if (!who) continue;
        // often all lanes want one bin: weights of one size, recent slots
        const int first = __builtin_amdgcn_readlane(bin, __builtin_ctzll(who));
        if (__ballot(in && bin == first) == who) {
          if (lane == 0) atomicAdd(&hist[first], (int)__popcll(who));
        } else if (in) {
          atomicAdd(&hist[bin], 1);
        }
      }
    }
    __syncthreads();
    // lane i has bins 255 - 4 i down, so sums come from the largest
    int n[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += n[i] = hist[255 - 4 * lane - i];
    int above = wave_scan(sum) - sum;
    const int at = __builtin_ctzll(__ballot(above + sum >= need));
    above = __builtin_amdgcn_readlane(above, at);
    int digit = 255 - 4 * at, in_bin = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = __builtin_amdgcn_readlane(n[i], at);
      if (in_bin == 0 && above + x >= need) in_bin = x, digit -= i;
      else if (in_bin == 0) above += x;
    }
    need -= above;
    t |= (unsigned)digit << shift;
    if (in_bin == need) {
      t -= 1;  // those above it are just enough
      need = 0;
      break;
    }
  }

  // Ranks in order of the slots, part by part. A wave puts its counts of a
  // pass into lds_c; `sum_up` makes of them what comes before each.
  auto sum_up = [&](int which) {
    __syncthreads();
    if (wave == 0) {
      constexpr int kEach = R * kEvictWaves / 64;
      int *c = &lds_c[which][0][0] + lane * kEach, n[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum += n[i] = c[i];
      int before = wave_scan(sum) - sum;
      if (lane == 63) lds_all[which] = before + sum;
#pragma unroll
      for (int i = 0; i < kEach; ++i) c[i] = before, before += n[i];
    }
    __syncthreads();
  };
  int ties = 0, holes = 0, movers = 0;
  const unsigned long long below = (1ull << lane) - 1;
  for (int part = 0; part < (MANY ? len : 1); part += kPart) {
    if (MANY) load(part);
    unsigned stays = 0;  // bit r
    if (need) {  // of the equal ones the first stay
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int n = __popcll(__ballot(key[r] == t));
        if (lane == 0) lds_c[0][r][wave] = n;
      }
      sum_up(0);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      bool stay = key[r] > t;
      if (need) {
        const unsigned long long equal = __ballot(key[r] == t);
        const int rank = ties + lds_c[0][r][wave] + __popcll(equal & below);
        stay = stay || (key[r] == t && rank < need);
      }
      stays |= (unsigned)stay << r;
    }
    if (need) {
      ties += lds_all[0];
      __syncthreads();
    }
    // free slots below the budget, and kept rows above it
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = part + r * kEvict + tid;
      const bool stay = stays >> r & 1;
      const int nh = __popcll(__ballot(i < keep && !stay));
      const int nm = __popcll(__ballot(i >= keep && stay));
      if (lane == 0) lds_c[0][r][wave] = nh, lds_c[1][r][wave] = nm;
    }
    sum_up(0);
    sum_up(1);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = part + r * kEvict + tid;
      const bool stay = stays >> r & 1;
      const bool hole = i < keep && !stay, mover = i >= keep && stay;
      const unsigned long long some_h = __ballot(hole);
      const unsigned long long some_m = __ballot(mover);
      if (some_h && hole)
        list[holes + lds_c[0][r][wave] + __popcll(some_h & below)].to = i;
      if (some_m && mover) {
        Pair *to = list + movers + lds_c[1][r][wave] +
                   __popcll(some_m & below);
        to->from = i;
        to->mass = m[r];
        to->pos = p[r];
      }
      if (i < keep && stay) {
        if (mass_out != mass) mass_out[i] = m[r];
        if (pos_out != pos) pos_out[i] = p[r];
      }
    }
    holes += lds_all[0];
    movers += lds_all[1];
    if (MANY) __syncthreads();
  }
  if (tid == 0) *count = movers;
  // All of the old has been read, and the list is whole.
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < movers; i += kEvict) {
    const Pair x = list[i];
    mass_out[x.to] = x.mass;
    pos_out[x.to] = x.pos;
  }
  for (int i = keep + tid; i < room; i += kEvict) {
    mass_out[i] = 0.f;
    pos_out[i] = -1;
  }
}

// Sixteen bytes of a key's and of a value's row per thread. Lengths are
// written here, since the launch before reads the old ones, which may be the
// same array.
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a, int pairs) {
  const int b = blockIdx.x / a.c.kvh, h = blockIdx.x % a.c.kvh;
  const int tid = threadIdx.x;
  const int *count = (const int *)((const Pair *)a.ws +
                                   (long)gridDim.x * pairs);
  const int n = min(count[blockIdx.x] - (int)blockIdx.y * kPairs, kPairs);
  const Pair *list = (const Pair *)a.ws + (long)blockIdx.x * pairs +
                     (long)blockIdx.y * kPairs;
  const int chunks = a.c.d / 8;
#pragma unroll 4
  for (int i = tid; i < n * chunks; i += 256) {
    const Pair &p = list[i / chunks];
    const long pt = a.c.page(b, p.to), pf = a.c.page(b, p.from);
    if (pt < 0 || pf < 0) continue;
    const int c = i % chunks * 8;
    const int rt = (unsigned)p.to % (unsigned)a.c.block;
    const int rf = (unsigned)p.from % (unsigned)a.c.block;
    bf16 *k = (bf16 *)a.c.k + h * a.c.k_head + c;
    bf16 *v = (bf16 *)a.c.v + h * a.c.v_head + c;
    const u32x4 kr = *(const u32x4 *)(k + pf * a.c.k_page + rf * a.c.k_row);
    const u32x4 vr = *(const u32x4 *)(v + pf * a.c.v_page + rf * a.c.v_row);
    *(u32x4 *)(k + pt * a.c.k_page + rt * a.c.k_row) = kr;
    *(u32x4 *)(v + pt * a.c.v_page + rt * a.c.v_row) = vr;
  }
  if (h == 0 && blockIdx.y == 0 && tid == 0) {
    const int keep = min(a.c.len(b), a.budget);
    if (a.c.lens.is64) ((long *)a.lens_out)[b] = keep;
    else ((int *)a.lens_out)[b] = keep;
  }
}

}  // namespace

void launch_paged_append(const PagedArgs &a, const void *k, long k_tok,
                         long k_head, const void *v, long v_tok, long v_head,
                         long tokens, IdxPtr cu, int *key_pos, IdxPtr pos,
                         hipStream_t stream) {
  const long threads = tokens * a.kvh * (a.d / 8);
  if (!threads || !a.batch) return;
  check_grid("paged_append", (threads + 255) / 256, 256);
  k_paged_append<<<dim3((unsigned)((threads + 255) / 256)), 256, 0, stream>>>(
      a, (const bf16 *)k, k_tok, k_head, (const bf16 *)v, v_tok, v_head,
      tokens, cu, key_pos, pos);
  launched("paged_append");
}

static DecodeWork decode_work(int batch, int qh, int kvh) {
  DecodeWork w{};
  w.groups = (qh / kvh + 15) / 16;
  // so many sequences that there are steps enough, if none is empty
  w.apart = (long)batch * kvh * w.groups >= kFew * kSlots;
  // ... and of these each then takes two at least, since a sequence of one to
  // two steps in two chunks costs a join (512 of 131 keys, 8 key heads: 65 us
  // for 63; 400 of 131 in rows of 64: 36 for 33; longer ones the same)
  w.least = w.apart ? 2 : 1;
  // a workgroup to a query head, unless so many would take longer to start
  // than to join (512 sequences, 8 key heads, nothing to join: 17 us)
  const long most = 4 * kSlots / ((long)batch * kvh);
  w.joins = (int)max(1L, min((long)(qh / kvh), most));
  return w;
}

// Chunks at most: those of a cut that is shared and of one that is not, over
// the blocks that each takes.
static long decode_chunks(int batch, int kvh, const DecodeWork &w) {
  const int per = kvh * w.groups, own = (per + 3) / 4;
  return batch + max((kSlots + per - 1) / per, (2 * kSlots + own - 1) / own);
}

size_t paged_decode_workspace(int batch, int qh, int kvh, int d, long room,
                              bool mass) {
  const size_t chunks = decode_chunks(batch, kvh, decode_work(batch, qh, kvh));
  return (chunks * qh * (d + 2) + 2 * (size_t)batch +
          (mass ? (size_t)batch * qh * room : 0)) *
         sizeof(float);
}

template <typename T, int D>
static void decode(const PagedDecodeArgs &a, const DecodeWork &w,
                   hipStream_t stream) {
  const int per = a.c.kvh * w.groups, own = (per + 3) / 4;
  const long shared = a.c.batch + (kSlots + per - 1) / per;
  const long apart = a.c.batch + (2 * kSlots + own - 1) / own;
  const long blocks = max(w.apart ? 0 : shared * per, apart * own);
  // nothing to join where no sequence can have two chunks
  const long spans = a.mass ? (a.c.room() + kSpan - 1L) / kSpan : 0;
  const bool more = spans || a.c.room() > w.least * kStep;
  check_grid("paged_decode", blocks, 256);
  if (more)
    check_grid("paged_decode", a.c.batch, 64 * kSpanWaves, a.c.kvh,
               w.joins + spans);
  k_paged_decode<T, D><<<dim3((unsigned)blocks), 256, 0, stream>>>(a, w);
  launched("paged_decode");
  if (more) {
    const dim3 finish(a.c.batch, a.c.kvh, w.joins + spans);
    k_decode_finish<T, D><<<finish, 64 * kSpanWaves, 0, stream>>>(a, w);
    launched("paged_decode");
  }
}

void launch_paged_decode(const PagedDecodeArgs &a, hipStream_t stream) {
  if (!a.c.batch) return;
  if ((long)a.c.batch * (a.c.room() / kStep + 1) > 1L << 30)
    throw std::runtime_error("paged_decode: 2^37 slots in all at most");
  DecodeWork w = decode_work(a.c.batch, a.qh, a.c.kvh);
  w.part = (float *)a.ws;
  const size_t chunks = decode_chunks(a.c.batch, a.c.kvh, w);
  w.sum = (float2 *)(w.part + chunks * a.qh * a.c.d);
  w.plan = (int *)(w.sum + chunks * a.qh);
  w.logits = a.mass ? (float *)(w.plan + 2 * (size_t)a.c.batch) : nullptr;
  if (a.c.is_fp16)
    a.c.d == 64 ? decode<_Float16, 64>(a, w, stream)
                : decode<_Float16, 128>(a, w, stream);
  else
    a.c.d == 64 ? decode<bf16, 64>(a, w, stream)
                : decode<bf16, 128>(a, w, stream);
}

static int evict_pairs(long room, int budget) {  // most rows that can move
  const long pairs = budget < room - budget ? budget : room - budget;
  return (int)(pairs > 0 ? pairs : 0);
}

size_t kv_evict_workspace(int batch, int kvh, long room, int budget) {
  return (size_t)batch * kvh *
         (sizeof(int) + evict_pairs(room, budget) * sizeof(Pair));
}

void launch_kv_evict(const EvictArgs &a, hipStream_t stream) {
  if (!a.c.batch) return;
  const int room = a.c.room(), pairs = evict_pairs(room, a.budget);
  const long rows = (long)a.c.batch * a.c.kvh;
  const long parts = (pairs + kPairs - 1) / kPairs;
  if (room > 1 << 30)
    throw std::runtime_error("kv_evict: 2^30 slots of a sequence at most");
  check_grid("kv_evict", rows, kEvict);
  check_grid("kv_evict", rows, 256, parts);
  // registers for as many keys as a sequence can have, in steps that each
  // cost the shorter ones something
  if (room <= 4 * kEvict)
    k_evict_select<4, false><<<rows, kEvict, 0, stream>>>(a, pairs);
  else if (room <= 16 * kEvict)
    k_evict_select<16, false><<<rows, kEvict, 0, stream>>>(a, pairs);
  else
    k_evict_select<16, true><<<rows, kEvict, 0, stream>>>(a, pairs);
  launched("kv_evict");
  const dim3 grid((unsigned)rows, (unsigned)(parts ? parts : 1));
  k_evict_move<<<grid, 256, 0, stream>>>(a, pairs);
  launched("kv_evict");
}

}  // namespace td
