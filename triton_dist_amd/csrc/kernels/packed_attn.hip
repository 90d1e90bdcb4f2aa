// Attention of packed prompts: documents side by side without padding, each
// token seeing only its own document, causally or not, with a prefix that
// all of a document's tokens see.
//
// Bound by the matrix instructions: 4 d operations per query head and seen
// pair, against a few bytes per token. One pass over the keys with running
// maxima and sums.
//
// A wave owns a unit: 32 rows of one query head. The units of a workgroup
// share one key head's K and V, and units are numbered heads first, so that
// with eight query heads to a key head a workgroup's units are the same 32
// rows: they need the same keys, and the causal boundary
// costs one partly seen tile. Any number of query heads per key head packs
// without a gap.
//
// S^T = K Q^T and O^T = V^T P^T on 32x32x16 matrix instructions. Lane
// (c, h) = (lane & 31, lane >> 5) gets the scores of row c with keys
// 8 (r / 4) + 4 h + r % 4, r = 0..15, so maxima and sums need one exchange
// with the other half of the wave, and those scores are just what the second
// product wants from this lane once its keys are numbered that way: the
// weights never leave the registers. K and V go through registers to LDS,
// 64 keys a step; V is read transposed.
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
constexpr int kRows = 32, kKeys = 64;
// Of a workgroup. With rows of 64 elements more of a step's work is vector
// instructions, and two workgroups of four on a SIMD's waves overlap better:
// 8 heads, 8192 tokens plain 139 us for 156 with eight, capped 171 for 240,
// 1000 tokens 22 for 25, 64 documents of 256 24 for 29, 8 of 1000 the same.
// With 128 sharing K and V among eight does where documents are long: 8192
// tokens, 32 query heads plain 569 us for 610 with four, capped 675 for 702.
// Where they are short four would do better: 64 documents of 256 146 for 116,
// one of 1000 35 for 30.
template <int D> constexpr int kWavesOf = D == 64 ? 4 : 8;
// A maximum may fall behind by this many powers of two before the sums are
// rescaled: weights up to 2^6 cost no precision.
constexpr float kSlack = 6.f;
// Weights meet V in the inputs' type, the sum taken of them as they are before
// that rounding: of bf16 2^-8 of each at most, which adds a quarter to an
// output's error against 64 bits (packed prompts with a cap: 0.0017 to 0.0021),
// where a second product for the rest would add half to the matrix work. fp16
// has no numbers below 2^-24, so its weights are lifted by as much as the
// slack leaves room for: they keep all bits down to 2^-23 of the maximum and
// vanish below 2^-34 (2^-14 and 2^-25 without).
template <typename T> constexpr float kLift = 0.f;
template <> constexpr float kLift<_Float16> = 9.f;
// Below this, in units of log2, a maximum is rounded by 2^-4 at most, which
// scales a row's weights and their sum alike; logits past it are rounded like
// the maximum before it is taken off. To keep both forms costs 8192 tokens
// of 8 heads of 64 6 us of 145, 16384 with a bias 0.02 ms of 2.60, and those
// without one nothing.
constexpr float kFar = 1 << 20;

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
// Elements from row to row in LDS. K: 16 bytes more than a row, so that the
// same piece of eight rows takes different banks. V: 64 bytes more, so that
// the 64 bytes of four rows that 32 lanes read transposed do. With fixed
// steps every read of a step is one address and an offset.
template <int D> constexpr int kRowK = D + 8;
template <int D> constexpr int kRowV = D + 32;

struct Doc {
  int q0, k0;  // first row, first key
  int m, n;    // rows, keys
  int prefix;  // keys that all rows see
  int block;   // the workgroup's number in the document, from its end
};

// Document i, by offsets that may be anything: nothing outside of the rows
// and keys comes out. Returns its workgroups.
template <int D>
TD_DEV int read_doc(const PackedArgs &a, int i, Doc &out) {
  const long q0 = a.cu_q[i], q1 = a.cu_q[i + 1], k0 = a.cu_k[i],
             k1 = a.cu_k[i + 1];  // all loads at once
  const long prefix = a.causal && a.prefix.p ? a.prefix[i] : 0;
  out.q0 = (int)min(max(q0, 0L), a.rows);
  out.k0 = (int)min(max(k0, 0L), a.keys);
  out.m = (int)min(max(q1, (long)out.q0), a.rows) - out.q0;
  out.n = (int)min(max(k1, (long)out.k0), a.keys) - out.k0;
  out.prefix = (int)min(max(prefix, 0L), a.keys);
  return (int)(((out.m + kRows - 1L) / kRows * (a.qh / a.kvh) +
                kWavesOf<D> - 1) / kWavesOf<D>);
}

// The document's workgroup `at`, or what is left of `at` where there is
// none: the number of the workgroup among the spare ones. Heavy workgroups
// of a document, which see most keys, come first. A wave finds it among up
// to 64 documents, which needs no barrier; among more the waves share the
// offsets (16384 tokens, 64 heads of 128, 8 tokens a document: 0.70 ms, and
// 2.40 where each wave goes through all offsets).
template <int D>
TD_DEV bool find_doc(const PackedArgs &a, int &at, Doc &out) {
  constexpr int kWaves = kWavesOf<D>, kThreads = 64 * kWaves;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (a.seqs <= 64) {
    Doc doc{};
    const int blocks = lane < a.seqs ? read_doc<D>(a, lane, doc) : 0;
    const int upto = wave_scan(blocks);
    const unsigned long long found = __ballot(blocks && upto > at);
    if (found) {
      const int f = __builtin_ctzll(found);
      out.block = __builtin_amdgcn_readlane(upto, f) - 1 - at;
      out.q0 = __builtin_amdgcn_readlane(doc.q0, f);
      out.k0 = __builtin_amdgcn_readlane(doc.k0, f);
      out.m = __builtin_amdgcn_readlane(doc.m, f);
      out.n = __builtin_amdgcn_readlane(doc.n, f);
      out.prefix = __builtin_amdgcn_readlane(doc.prefix, f);
      return true;
    }
    at -= __builtin_amdgcn_readlane(upto, 63);
    return false;
  }
  __shared__ int lds_n[kWaves];
  __shared__ Doc lds_doc;
  const int each = (a.seqs + kThreads - 1) / kThreads;
  const int last = min((tid + 1) * each, a.seqs);
  int own = 0;
  Doc doc;
  for (int i = tid * each; i < last; ++i) own += read_doc<D>(a, i, doc);
  const int upto = wave_scan(own);
  if (lane == 63) lds_n[wave] = upto;
  if (tid == 0) lds_doc.m = 0;
  __syncthreads();
  int before = upto - own, all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave) before += lds_n[i];
    all += lds_n[i];
  }
  if (at < all && at >= before && at < before + own)
    for (int i = tid * each; i < last; ++i) {
      const int blocks = read_doc<D>(a, i, doc);
      if (at >= before && at < before + blocks) {
        doc.block = before + blocks - 1 - at;
        lds_doc = doc;
      }
      before += blocks;
    }
  __syncthreads();
  out = lds_doc;
  if (at < all && out.m > 0) return true;
  at = max(at - all, 0);
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
__global__ __launch_bounds__(64 * kWavesOf<D>, 2) void k_packed_prefill(
    PackedArgs a, int tiles) {
  constexpr int kWaves = kWavesOf<D>;
  constexpr int kP = D / 8;          // 16-byte pieces of a row
  constexpr int kLoads = kKeys * kP / (64 * kWaves);
  constexpr int kStageK = kKeys * kRowK<D>, kStageV = kKeys * kRowV<D>;
  __shared__ __attribute__((aligned(16))) T stage_lds[2 * (kStageK + kStageV)];
  T *const lds_k = stage_lds, *const lds_v = stage_lds + 2 * kStageK;
  __shared__ int lds_see[kWaves], lds_all[kWaves], lds_wild;

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int c = lane & 31, h = lane >> 5;
  const int kh = blockIdx.x % a.kvh, g = a.qh / a.kvh;
  int at = blockIdx.x / a.kvh;
  Doc doc;
  if (!find_doc<D>(a, at, doc)) {
    if (a.clear_tail || a.lse)  // `at` is past the documents' workgroups
      clear_tail<T>(a, at, tiles - ((int)(blockIdx.x / a.kvh) - at), kh);
    return;
  }
  // Keys past the document repeat its last one: their weights are zero.
  constexpr int kPer = 64 * kWaves / kP;  // rows that the workgroup moves
  const int srow = tid / kP, piece = tid % kP;
  const T *kfrom = (const T *)a.k + (long)doc.k0 * a.k_tok + kh * a.k_head +
                   piece * 8;
  const T *vfrom = (const T *)a.v + (long)doc.k0 * a.v_tok + kh * a.v_head +
                   piece * 8;
  vec8<T> nk[kLoads], nv[kLoads];
  int see = doc.n;  // keys that some row sees
  auto fetch = [&](vec8<T> *to, const T *from, long tok, int first) {
    if (see <= 0 || first >= see) return;  // also a document without keys
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int key = max(0, min(first + i * kPer + srow, doc.n - 1));
      to[i] = *(const vec8<T> *)(from + (long)key * tok);
    }
  };
  vec8<T> after[kLoads];
  fetch(nk, kfrom, a.k_tok, -32);
  fetch(after, kfrom, a.k_tok, 32);
  fetch(nv, vfrom, a.v_tok, 0);

  const int units = (doc.m + kRows - 1) / kRows * g;
  const int unit = doc.block * kWaves + wave;
  const bool live = unit < units;
  const int head = kh * g + (live ? unit % g : 0);
  const int row0 = live ? unit / g * kRows : 0;
  const int row = min(row0 + c, doc.m - 1);  // a last unit repeats its last
  vec8<T> qf[D / 16];
  {
    const T *q = (const T *)a.q + (long)(doc.q0 + row) * a.q_tok +
                 head * a.q_head + h * 8;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *(const vec8<T> *)(q + s * 16);
  }
  // keys that this row sees: those below `lim`
  const int pos = row + doc.n - doc.m;
  int lim = doc.n;
  if (a.causal) {
    lim = max(min(max(pos + 1, 0), doc.n), min(doc.prefix, doc.n));
  }
  if (!live) lim = 0;
  const bool only_back = a.causal && !a.prefix.p;
  const int first_pos = row0 + doc.n - doc.m;
  int most = lim, least = lim;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = max(most, __shfl_xor(most, o));
    least = min(least, __shfl_xor(least, o));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  if (lane == 0) lds_see[wave] = most, lds_all[wave] = live ? least : doc.n;
  if (tid == 0) lds_wild = 0;

  const float c1 = (a.s.scale == 0.f ? 1.f : fabsf(a.s.scale)) * kLog2e;
  // A logit in units of log2 is cf x + c0, less slope times the distance:
  // x is the score itself, or with a cap 1 / (1 + e^(2 s / cap)), of which
  // cap tanh is cap - 2 cap x.
  float cf = CAP ? -2.f * kLog2e * a.s.softcap : c1;
  const float c0 = CAP ? kLog2e * a.s.softcap : 0.f;
  const float in_cap = CAP ? 2.f * c1 / a.s.softcap : 0.f;
  // The distance to key 4 h + 8 (r / 4) + r % 4 of 32 is gap less that, so
  // what a lane's 16 keys differ by is the same for the whole wave.
  const float slope = BIAS ? a.s.slopes[head] * kLog2e : 0.f;
  float step_up[BIAS ? 16 : 1];
  if (BIAS)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      step_up[r] = __uint_as_float(__builtin_amdgcn_readfirstlane(
          __float_as_uint(slope * (float)(8 * (r / 4) + r % 4))));
  // an instruction takes one scalar register: leave it to these
  asm("" : "+v"(cf));
  __syncthreads();
  see = 0;
  int all_see = doc.n;  // keys that all rows see
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    see = max(see, lds_see[w]);
    all_see = min(all_see, lds_all[w]);
  }
  const int steps = (see + kKeys - 1) / kKeys;

  auto stage_k = [&](const vec8<T> *from, int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kPer + srow;
      *(vec8<T> *)&lds_k[buf * kStageK + r * kRowK<D> + piece * 8] = from[i];
    }
  };
  // A weight of zero does not hide a value that is no number, so where some
  // row does not see some key such values are staged as zeros, and added to
  // the rows that see them at the end.
  auto some_hidden = [&](int step) { return (step + 1) * kKeys > all_see; };
  auto stage_v = [&](int step) {
    const int buf = step & 1;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kPer + srow;
      if (some_hidden(step)) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (wild(nv[i][e])) any = true, nv[i][e] = (T)0.f;
        if (any) lds_wild = 1;
      }
      *(vec8<T> *)&lds_v[buf * kStageV + r * kRowV<D> + piece * 8] = nv[i];
    }
  };

  float m = -INFINITY, l = 0.f;
  f32x16 acc[D / 32] = {};
  const int kread = c * kRowK<D> + h * 8;
  const int vread = (4 * h + ((lane & 15) >> 2)) * kRowV<D> + (lane & 16) +
                    4 * (lane & 3);
  auto k_frag = [&](int buf, int sub, int x) {
    return *(const vec8<T> *)(&lds_k[buf * kStageK + kread +
                                        32 * sub * kRowK<D> + 16 * x]);
  };
  auto v_frag = [&](int buf, int sub, int j) {
    constexpr int n = D / 32;
    union { s16x4 half[2]; vec8<T> all; } v;
    const T *at = &lds_v[buf * kStageV + vread +
                            (32 * sub + 16 * (j / n)) * kRowV<D> +
                            32 * (j % n)];
    v.half[0] = read_transposed(at);
    v.half[1] = read_transposed(at + 8 * kRowV<D>);
    return v.all;
  };
  // What is kept of a score until it is weighed: x, or with a bias the logit
  // but for c0 and slope times gap.
  auto keep = [&](float x, int r) {
    if (CAP)
      x = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * in_cap));
    return BIAS ? x * cf + step_up[r] : x;
  };
  constexpr bool kLow = CAP && !BIAS;  // a small x is a large logit
  constexpr float kHidden = kLow ? INFINITY : -INFINITY;
  auto larger = [](float x, float y) {
    return kLow ? fminf(x, y) : fmaxf(x, y);
  };
  // Slope times gap, for the 32 keys from `base` on.
  auto lean = [&](int base) {
    return BIAS ? slope * (float)(pos - base - 4 * h) : 0.f;
  };
  // Where not all of the wave's rows see the 32 keys from `base` on, hides
  // what they do not see; where keys behind a row are seen, turns their
  // distance's sign. Then finds the largest again.
  auto mend = [&](f32x16 &s, int base, float &top) {
    const bool turn = BIAS && !only_back && base + 32 > first_pos;
    if (base + 32 <= least && !turn) return;
    const int left = lim - base - 4 * h, gap = pos - base - 4 * h;
    top = kHidden;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = 8 * (r / 4) + r % 4;
      if (BIAS && j > gap) s[r] -= 2.f * slope * (float)(j - gap);
      if (j >= left) s[r] = kHidden;
      top = larger(top, s[r]);
    }
  };
  // Rows' maxima follow the scores `s` of the 32 keys from `base` on. A weight
  // is then the power of s * cf + from (s + from with a bias): one operation
  // a score, which takes the maximum off the unrounded product, so that the
  // largest weight is 2 to the rounding of the maximum. Where that could be
  // far from 1, logits are rounded like the maximum before it is taken off (and
  // divided by the cf that the power multiplies them by).
  float from = 0.f;
  const unsigned long long far_off =
      BIAS ? __ballot(fabsf(slope) * (float)max(abs(pos), abs(pos - doc.n)) +
                          c0 > kFar)
           : 0;
  unsigned long long far = far_off;  // of the whole wave
  auto raise = [&](f32x16 &s, float top, int base) {
#pragma clang fp contract(off)
    const float add = BIAS ? c0 - lean(base) : c0;
    top = BIAS ? top + add : top * cf + add;
    if (__any(top > m + kSlack)) {
      const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float x = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f
                                                                  : to));
      m = to;
      l *= x;
#pragma unroll
      for (int t = 0; t < D / 32; ++t) acc[t] *= x;
      // a cap alone leaves logits of 1443 at most
      if (!CAP || BIAS)
        far = far_off | __ballot(m != -INFINITY && fabsf(m) > kFar);
    }
    const float safe = m == -INFINITY ? 0.f : m;
    from = add - safe + kLift<T>;
    if (far) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[r] = BIAS ? (s[r] + add) - safe : (s[r] * cf - safe) / cf;
      from = kLift<T>;
    }
  };
  // 32 keys' scores in `s` are weighed and their values collected while the
  // next 32 keys' scores are made in `next`, `base` on. The order is written
  // out, so that reads run two or three products ahead and each product of
  // 32 cycles has about as much vector work beside it: the weights beside
  // the scores' products, the next logits beside the values'.
  auto work = [&](f32x16 &s, f32x16 &next, int step, int sub) {
    constexpr int nx = D / 16, nj = D / 16;
    const int buf = step & 1, base = step * kKeys + 32 * (sub + 1);
    const float from_s = from;
    vec8<T> kq[3], vq[3], p[2];
#pragma unroll
    for (int x = 0; x < 3; ++x) kq[x] = k_frag(buf, sub, x);
    // behind the last keys the products are of no use and no harm
#pragma unroll
    for (int x = 0; x < nx; ++x) {
      __builtin_amdgcn_sched_barrier(0);
      next = mfma32(kq[x % 3], qf[x], x ? next : f32x16{});
      if (x + 3 < nx) kq[x % 3] = k_frag(buf, sub, x + 3);
      else vq[x + 3 - nx] = v_frag(buf, sub, x + 3 - nx);
#pragma unroll
      for (int r = 16 / nx * x; r < 16 / nx * (x + 1); ++r) {
        const float e =
            __builtin_amdgcn_exp2f(BIAS ? s[r] + from_s : s[r] * cf + from_s);
        l += e;
        p[r / 8][r % 8] = (T)e;
      }
    }
    float top = kHidden;
#pragma unroll
    for (int j = 0; j < nj; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      acc[j % (D / 32)] = mfma32(vq[j % 3], p[j / (D / 32)],
                                 acc[j % (D / 32)]);
      if (j + 3 < nj) vq[j % 3] = v_frag(buf, sub, j + 3);
      if (j < 2) continue;  // the scores are still on their way
#pragma unroll
      for (int r = 16 * (j - 2) / (nj - 2); r < 16 * (j - 1) / (nj - 2);
           ++r) {
        next[r] = keep(next[r], r);
        top = larger(top, next[r]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (base < most) {
      mend(next, base, top);
      raise(next, top, base);
    }
  };

  // A step's V are the keys from 64 step on; its K are those of the
  // products made in it, 32 keys further.
  f32x16 sa, sb;
  if (steps) {
    stage_k(nk, 1);
    stage_k(after, 0);
    stage_v(0);
    fetch(nk, kfrom, a.k_tok, kKeys + 32);
    fetch(nv, vfrom, a.v_tok, kKeys);
    __syncthreads();
    // A negative scale turns the queries' sign, so that maxima stay maxima;
    // a scale of zero clears them, so that a hidden key's -inf stays one.
    if (!(a.s.scale > 0.f))
#pragma unroll
      for (int x = 0; x < D / 16; ++x)
        qf[x] = a.s.scale < 0.f ? -qf[x] : vec8<T>{};
    if (most > 0) {
#pragma unroll
      for (int x = 0; x < D / 16; ++x)
        sa = mfma32(k_frag(1, 1, x), qf[x], x ? sa : f32x16{});
      float top = kHidden;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sa[r] = keep(sa[r], r);
        top = larger(top, sa[r]);
      }
      mend(sa, 0, top);
      raise(sa, top, 0);
    }
  }
  for (int step = 0; step < steps; ++step) {
    const int base = step * kKeys;
    __syncthreads();  // this step is there, the other buffers are free
    if (step + 1 < steps) {
      stage_k(nk, (step & 1) ^ 1);
      stage_v(step + 1);
      fetch(nk, kfrom, a.k_tok, base + 2 * kKeys + 32);
      fetch(nv, vfrom, a.v_tok, base + 2 * kKeys);
    }
    if (base < most) {
      work(sa, sb, step, 0);
      if (base + 32 < most) work(sb, sa, step, 1);
    }
  }
  __syncthreads();
  if (lds_wild)
    for (int key = all_see / kKeys * kKeys; key < see; ++key) {
      if (key >= lim) continue;
      const T *v = (const T *)a.v + (long)(doc.k0 + key) * a.v_tok +
                   kh * a.v_head + 4 * h;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const T x = v[32 * t + 8 * (r / 4) + r % 4];
          if (wild(x)) acc[t][r] += (float)x;
        }
    }
  l += __shfl_xor(l, 32);
  // A value that is no finite number makes its outputs so, however small its
  // weight; times one that underflows an infinite value is NaN. So outputs
  // that are NaN without a score being one are summed from such values alone.
  bool spoilt = false;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) spoilt |= acc[t][r] != acc[t][r];
  if (__any(spoilt && l == l)) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      f32x16 alone = {};
#pragma unroll 4
      for (int key = 0; key < most; ++key) {
        if (key % 64 == 0) {  // done where all that were NaN are by a value
          bool open = false;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            open |= acc[t][r] != acc[t][r] && alone[r] == alone[r];
          if (!__any(open && key < lim)) break;
        }
        if (key >= lim) continue;
        const T *v = (const T *)a.v + (long)(doc.k0 + key) * a.v_tok +
                     kh * a.v_head + 4 * h + 32 * t;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const T x = v[8 * (r / 4) + r % 4];
          alone[r] += wild(x) ? (float)x : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (acc[t][r] != acc[t][r] && alone[r] != 0.f) acc[t][r] = alone[r];
    }
  }
  if (!live) return;
  if (a.lse && h == 0 && row0 + c < doc.m)
    a.lse[(long)(doc.q0 + row) * a.qh + head] =
        l == 0.f ? -INFINITY
                 : (m - kLift<T> + __builtin_amdgcn_logf(l)) * kLn2;
  // Through LDS, where nothing is read any more, so that whole rows go out.
  constexpr int kRowO = D + 8;
  static_assert(kWaves * kRows * kRowO <= 2 * (kStageK + kStageV),
                "outputs fit where K and V were");
  T *mine = &stage_lds[wave * kRows * kRowO];
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      vec4<T> o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (T)(acc[t][r + i] * inv);
      *(vec4<T> *)(mine + c * kRowO + 32 * t + 2 * r + 4 * h) = o;
    }
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
  T *out = (T *)a.out + (long)(doc.q0 + row0) * a.out_tok + head * a.out_head;
#pragma unroll
  for (int i = 0; i < kRows * kP / 64; ++i) {
    const int r = (i * 64 + lane) / kP, e = lane % kP * 8;
    if (row0 + r < doc.m)
      *(vec8<T> *)(out + r * a.out_tok + e) =
          *(const vec8<T> *)(mine + r * kRowO + e);
  }
}

template <typename T, int D>
void prefill(const PackedArgs &a, hipStream_t stream) {
  // as many workgroups a key head as any cutting of the rows into documents
  // can need, and spare ones for the rows of no document
  constexpr int kWaves = kWavesOf<D>;
  const long g = a.qh / a.kvh;
  const long tiles = (a.rows / kRows + a.seqs) * g / kWaves + a.seqs + 4;
  if (tiles * a.kvh * 64 * kWaves > 0xffffffffL)  // threads of a launch
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
  if (a.rows > 0x7fffffffL || a.keys > 0x7fffffffL)
    throw std::runtime_error("packed_prefill: too many rows");
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
