// Attention of packed prompts: documents side by side without padding, each
// token seeing only its own document, causally or not, with a prefix that
// all of a document's tokens see.
//
// Bound by the matrix instructions: 4 d operations per query head and seen
// pair, against a few bytes per token. One pass over the keys with running
// maxima and sums.
//
// A wave owns a unit: 32 rows of one query head. The eight units of a
// workgroup share one key head's K and V, and units are numbered heads
// first, so that with eight query heads to a key head a workgroup's units
// are the same 32 rows: they need the same keys, and the causal boundary
// costs one partly seen tile. Any number of query heads per key head packs
// without a gap.
//
// S^T = K Q^T and O^T = V^T P^T on 32x32x16 matrix instructions. Lane
// (c, h) = (lane & 31, lane >> 5) gets the scores of row c with keys
// 8 (r / 4) + 4 h + r % 4, r = 0..15, so maxima and sums need one exchange
// with the other half of the wave, and those scores are just what the second
// product wants from this lane once its keys are numbered that way: the
// weights never leave the registers. K and V come as they lie, by direct
// loads to LDS, 64 keys a step and two steps deep; V is read transposed.
#include <stdexcept>
#include <string>

#include "td/api.hpp"
#include "td/paged.hpp"

namespace td {

namespace {

using bf16 = __bf16;
template <typename T> using vec8 = __attribute__((ext_vector_type(8))) T;
template <typename T> using vec4 = __attribute__((ext_vector_type(4))) T;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kWaves = 8, kRows = 32, kKeys = 64;
// A maximum may fall behind by this many powers of two before the sums are
// rescaled: weights up to 2^6 cost no precision.
constexpr float kSlack = 6.f;

TD_DEV f32x16 mfma32(vec8<bf16> a, vec8<bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
TD_DEV f32x16 mfma32(vec8<_Float16> a, vec8<_Float16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// Of each 16 lanes, lane l gets column l of the 4x16 block whose row l / 4
// and columns 4 (l % 4) on its pointer names.
TD_DEV s16x4 read_transposed(const void *lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4 *)(unsigned)(uintptr_t)lds);
}
// Where a row's 16-byte pieces lie in LDS. K: eight rows' pieces of one
// column take all banks. V: the 64 bytes of four rows that 32 lanes read
// transposed do.
template <int D> TD_DEV int k_piece(int row, int piece) {
  return piece ^ (row & (D / 8 - 1));
}
template <int D> TD_DEV int v_piece(int row, int piece) {
  return D == 128 ? piece ^ (row & 3) << 2 : piece ^ (row >> 1 & 1) << 2;
}

struct Doc {
  long q0, k0;
  int m, n;   // rows, keys
  int index;
  int block;  // the workgroup's number in the document, from its end
};

// The document's workgroup `at`, or what is left of `at` where there is
// none: the number of the workgroup among the spare ones.
TD_DEV bool find_doc(const PackedArgs &a, int &at, Doc &out) {
  const int lane = threadIdx.x & 63, g = a.qh / a.kvh;
  for (int base = 0; base < a.seqs; base += 64) {
    const int i = base + lane;
    long q0 = 0;
    int m = 0, blocks = 0;
    if (i < a.seqs) {
      q0 = min(max(a.cu_q[i], 0L), a.rows);
      m = (int)(min(max(a.cu_q[i + 1], q0), a.rows) - q0);
      blocks = (int)(((long)((m + kRows - 1) / kRows) * g + kWaves - 1) /
                     kWaves);
    }
    int upto = blocks;
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned long long found = __ballot(upto > at);
    if (found) {
      const int f = __builtin_ctzll(found);
      out.index = base + f;
      // heavy blocks, which see most keys, first
      out.block = __builtin_amdgcn_readlane(upto, f) - 1 - at;
      out.m = __builtin_amdgcn_readlane(m, f);
      out.q0 = min(max(a.cu_q[out.index], 0L), a.rows);
      out.k0 = min(max(a.cu_k[out.index], 0L), a.keys);
      out.n = (int)(min(max(a.cu_k[out.index + 1], out.k0), a.keys) -
                    out.k0);
      return true;
    }
    at -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// Rows of no document: zeros, in what the call itself has made.
template <typename T>
TD_DEV void clear_tail(const PackedArgs &a, int spare, int spares, int kh) {
  const long first = a.seqs ? min(max(a.cu_q[0], 0L), a.rows) : 0;
  const long last = a.seqs ? min(max(a.cu_q[a.seqs], first), a.rows) : 0;
  const int g = a.qh / a.kvh, pieces = a.d / 8;
  const long rows = first + a.rows - last;
  for (long i = (long)spare * blockDim.x + threadIdx.x;
       i < rows * g * pieces; i += (long)spares * blockDim.x) {
    const long r = i / (g * pieces), row = r < first ? r : last + r - first;
    const int h = kh * g + (int)(i / pieces % g), c = (int)(i % pieces);
    if (a.clear_tail)
      *(vec8<T> *)((T *)a.out + row * a.out_tok + h * a.out_head + c * 8) =
          vec8<T>{};
    if (a.lse && c == 0) a.lse[row * a.qh + h] = -INFINITY;
  }
}

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves, 2) void k_packed_prefill(
    PackedArgs a, int tiles) {
  constexpr int kP = D / 8;          // 16-byte pieces of a row
  constexpr int kStage = kKeys * D;  // elements of a staged K or V
  constexpr int kLoads = kKeys * kP / (64 * kWaves);
  __shared__ __attribute__((aligned(16))) T lds_k[2][kStage];
  __shared__ __attribute__((aligned(16))) T lds_v[2][kStage];
  __shared__ int lds_see[kWaves];

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int c = lane & 31, h = lane >> 5;
  const int kh = blockIdx.x % a.kvh, g = a.qh / a.kvh;
  int at = blockIdx.x / a.kvh;
  Doc doc;
  if (!find_doc(a, at, doc)) {
    if (a.clear_tail || a.lse)  // `at` is past the documents' workgroups
      clear_tail<T>(a, at, tiles - ((int)(blockIdx.x / a.kvh) - at), kh);
    return;
  }
  const int units = (doc.m + kRows - 1) / kRows * g;
  const int unit = doc.block * kWaves + wave;
  const bool live = unit < units;
  const int head = kh * g + (live ? unit % g : 0);
  const int row0 = live ? unit / g * kRows : 0;
  const int row = min(row0 + c, doc.m - 1);  // a last unit repeats its last
  // keys that this row sees: those below `lim`
  const int pos = row + doc.n - doc.m;
  int lim = doc.n;
  if (a.causal) {
    lim = min(max(pos + 1, 0), doc.n);
    if (a.prefix.p)
      lim = max(lim, (int)min(a.prefix[doc.index], (long)doc.n));
  }
  if (!live) lim = 0;
  int most = lim, least = lim;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = max(most, __shfl_xor(most, o));
    least = min(least, __shfl_xor(least, o));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  if (lane == 0) lds_see[wave] = most;

  // A negative scale turns the queries' sign, so that maxima stay maxima; a
  // scale of zero clears them, so that a hidden key's -inf stays one.
  const float c1 = (a.s.scale == 0.f ? 1.f : fabsf(a.s.scale)) * kLog2e;
  vec8<T> qf[D / 16];
  {
    const T *q = (const T *)a.q + (doc.q0 + row) * a.q_tok +
                 head * a.q_head + h * 8;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qf[s] = *(const vec8<T> *)(q + s * 16);
      if (a.s.scale < 0.f) qf[s] = -qf[s];
      if (a.s.scale == 0.f) qf[s] = vec8<T>{};
    }
  }
  const float cap = a.s.softcap * kLog2e;
  const float in_cap = CAP ? 2.f * c1 / a.s.softcap : 0.f;
  const float slope = BIAS ? a.s.slopes[head] * kLog2e : 0.f;
  __syncthreads();
  int see = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) see = max(see, lds_see[w]);
  const int steps = (see + kKeys - 1) / kKeys;

  const T *kbase = (const T *)a.k + doc.k0 * a.k_tok + kh * a.k_head;
  const T *vbase = (const T *)a.v + doc.k0 * a.v_tok + kh * a.v_head;
  // Keys past the document repeat its last one: their weights are zero.
  vec8<T> nk[kLoads], nv[kLoads];
  auto fetch = [&](int step) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (i * 64 * kWaves + tid) / kP, p = tid % kP;
      const long key = min(step * kKeys + r, doc.n - 1);
      nk[i] = *(const vec8<T> *)(kbase + key * a.k_tok + p * 8);
      nv[i] = *(const vec8<T> *)(vbase + key * a.v_tok + p * 8);
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (i * 64 * kWaves + tid) / kP, p = tid % kP;
      *(vec8<T> *)&lds_k[buf][r * D + k_piece<D>(r, p) * 8] = nk[i];
      *(vec8<T> *)&lds_v[buf][r * D + v_piece<D>(r, p) * 8] = nv[i];
    }
  };

  float m = -INFINITY, l = 0.f;
  f32x16 acc[D / 32] = {};
  if (steps) {
    fetch(0);
    stage(0);
    if (steps > 1) fetch(1);
  }
  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1, base = step * kKeys;
    __syncthreads();  // this step is there, the other buffer is free
    if (step + 1 < steps) {
      stage(buf ^ 1);
      if (step + 2 < steps) fetch(step + 2);
    }
    if (base >= most) continue;
    f32x16 s[2] = {};
#pragma unroll
    for (int x = 0; x < D / 16; ++x)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 32 * t + c;
        const vec8<T> kf = *(const vec8<T> *)(
            &lds_k[buf][r * D + k_piece<D>(r, 2 * x + h) * 8]);
        s[t] = mfma32(kf, qf[x], s[t]);
      }
    if (CAP) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[t][r] = cap - 2.f * cap *
                              __builtin_amdgcn_rcpf(
                                  1.f + __builtin_amdgcn_exp2f(s[t][r] *
                                                               in_cap));
    }
    if (BIAS) {
      const float gap = (float)(pos - base - 4 * h);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float z = CAP ? s[t][r] : s[t][r] * c1;
          const float far = gap - (float)(32 * t + 8 * (r / 4) + r % 4);
          s[t][r] = z - slope * fabsf(far);
        }
    }
    if (base + kKeys > least) {  // not all of the wave's rows see all keys
      const int left = lim - base - 4 * h;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * t + 8 * (r / 4) + r % 4 >= left) s[t][r] = -INFINITY;
    }
    // plain scores are scaled in the exponent's multiply-add
    const float f = CAP || BIAS ? 1.f : c1;
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
    top = fmaxf(top, __shfl_xor(top, 32)) * f;
    if (__any(top > m + kSlack)) {
      const float to = fmaxf(m, top);
      const float x = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f
                                                                  : to));
      m = to;
      l *= x;
#pragma unroll
      for (int t = 0; t < D / 32; ++t) acc[t] *= x;
    }
    const float safe = m == -INFINITY ? 0.f : m;
    vec8<T> p[4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[t][r] * f - safe);
        l += e;
        p[2 * t + r / 8][r % 8] = (T)e;
      }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        const int r = 16 * x + 4 * h + ((lane & 15) >> 2);
        const int col = 32 * t + (lane & 16) + 4 * (lane & 3);
        union { s16x4 half[2]; vec8<T> all; } v;
        v.half[0] = read_transposed(
            &lds_v[buf][r * D + v_piece<D>(r, col / 8) * 8 + col % 8]);
        v.half[1] = read_transposed(
            &lds_v[buf][(r + 8) * D + v_piece<D>(r + 8, col / 8) * 8 +
                        col % 8]);
        acc[t] = mfma32(v.all, p[x], acc[t]);
      }
  }
  if (!live || row0 + c >= doc.m) return;
  l += __shfl_xor(l, 32);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *out = (T *)a.out + (doc.q0 + row) * a.out_tok + head * a.out_head +
           4 * h;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      vec4<T> o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (T)(acc[t][r + i] * inv);
      *(vec4<T> *)(out + 32 * t + 2 * r) = o;
    }
  if (a.lse && h == 0)
    a.lse[(doc.q0 + row) * a.qh + head] =
        l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int D>
void prefill(const PackedArgs &a, hipStream_t stream) {
  // as many workgroups a key head as any cutting of the rows into documents
  // can need, and spare ones for the rows of no document
  const long g = a.qh / a.kvh;
  const long tiles = (a.rows / kRows + a.seqs) * g / kWaves + a.seqs + 4;
  if (tiles * a.kvh > 0x7fffffffL)
    throw std::runtime_error("packed_prefill: too many rows and heads");
  const dim3 grid((unsigned)(tiles * a.kvh));
  const int n = 64 * kWaves, t = (int)tiles;
  if (a.s.softcap > 0.f && a.s.slopes)
    k_packed_prefill<T, D, true, true><<<grid, n, 0, stream>>>(a, t);
  else if (a.s.softcap > 0.f)
    k_packed_prefill<T, D, true, false><<<grid, n, 0, stream>>>(a, t);
  else if (a.s.slopes)
    k_packed_prefill<T, D, false, true><<<grid, n, 0, stream>>>(a, t);
  else
    k_packed_prefill<T, D, false, false><<<grid, n, 0, stream>>>(a, t);
}

}  // namespace

void launch_packed_prefill(const PackedArgs &a, hipStream_t stream) {
  if (!a.rows) return;
  if (a.is_fp16)
    a.d == 64 ? prefill<_Float16, 64>(a, stream)
              : prefill<_Float16, 128>(a, stream);
  else
    a.d == 64 ? prefill<bf16, 64>(a, stream) : prefill<bf16, 128>(a, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    throw std::runtime_error(std::string("packed_prefill: ") +
                             hipGetErrorString(e));
}

}  // namespace td
