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

TD_DEV float wave_max(float x) {
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
TD_DEV float wave_sum(float x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
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
  long slot;
  if (cu.p) {
    int lo = 0, hi = a.batch;  // the sequence with cu[b] <= t < cu[b + 1]
    while (lo < hi) {
      int mid = (lo + hi) >> 1;
      if (cu[mid + 1] <= t) lo = mid + 1; else hi = mid;
    }
    if (lo >= a.batch || t < cu[lo]) return;
    b = lo;
    slot = a.lens[b] + t - cu[b];
  } else {
    slot = a.lens[b];
  }
  if (slot < 0 || slot >= a.room()) return;
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
// decode: a workgroup per sequence and query head, a thread per key for the
// scores, a thread per element of the output for the sums.
// ---------------------------------------------------------------------------
template <typename T>
TD_DEV float score(const PagedDecodeArgs &a, const float *q, int b, int h,
                   int slot, int len, long page) {
  const int kh = h / (a.qh / a.c.kvh);
  const T *row = (const T *)a.c.k + page * a.c.k_page +
                 (slot % a.c.block) * a.c.k_row + kh * a.c.k_head;
  float s = 0.f;
  for (int i = 0; i < a.c.d; ++i) s += q[i] * (float)row[i];
  s *= a.s.scale;
  if (a.s.softcap > 0.f) s = a.s.softcap * tanhf(s / a.s.softcap);
  if (a.s.slopes) {
    long far = a.key_pos ? a.q_pos[b] - a.key_pos[((long)b * a.c.kvh + kh) *
                                                      a.c.room() + slot]
                         : (long)len - 1 - slot;
    s -= a.s.slopes[h] * (float)(far < 0 ? -far : far);
  }
  return s;
}

template <typename T>
__global__ __launch_bounds__(256) void k_paged_decode(PagedDecodeArgs a) {
  __shared__ float q[256], p[256], red[4], part[256];
  const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int d = a.c.d, kh = h / (a.qh / a.c.kvh);
  const int len = a.c.len(b);
  if (tid < d) q[tid] = (float)((const T *)a.q)[b * a.q_tok + h * a.q_head +
                                                tid];
  float m = -INFINITY, l = 0.f, acc = 0.f;
  const int col = tid % d, lane = tid / d, lanes = 256 / d;
  for (int base = 0; base < len; base += 256) {
    __syncthreads();
    const int slot = base + tid;
    float s = -INFINITY;
    if (slot < len) {
      const long page = a.c.page(b, slot);
      if (page >= 0) s = score<T>(a, q, b, h, slot, len, page);
    }
    float top = wave_max(s);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, top);
    const float safe = mn == -INFINITY ? 0.f : mn;
    const float r = expf(m - safe);
    p[tid] = expf(s - safe);
    m = mn;
    acc *= r;
    l *= r;
    __syncthreads();
    for (int i = 0; i < 256; ++i) l += p[i];
    const int top_i = min(256, len - base);
    for (int i = lane; i < top_i; i += lanes) {
      if (p[i] == 0.f) continue;  // also a slot whose page is missing
      const long page = a.c.page(b, base + i);
      acc += p[i] * (float)((const T *)a.c.v)[page * a.c.v_page +
                                              ((base + i) % a.c.block) *
                                                  a.c.v_row +
                                              kh * a.c.v_head + col];
    }
  }
  __syncthreads();
  part[tid] = acc;
  __syncthreads();
  if (tid < d) {
    for (int i = 1; i < lanes; ++i) acc += part[i * d + tid];
    ((T *)a.out)[((long)b * a.qh + h) * d + tid] =
        (T)(l > 0.f ? acc / l : 0.f);
    if (tid == 0)
      a.lse[(long)b * a.qh + h] = l > 0.f ? m + logf(l) : -INFINITY;
  }
}

// The weights that the query heads of a key head gave each slot.
template <typename T>
__global__ __launch_bounds__(256) void k_paged_mass(PagedDecodeArgs a) {
  extern __shared__ float qs[];
  const int b = blockIdx.y, kh = blockIdx.z, g = a.qh / a.c.kvh;
  const int d = a.c.d, slot = blockIdx.x * 256 + threadIdx.x;
  for (int i = threadIdx.x; i < g * d; i += 256)
    qs[i] = (float)((const T *)a.q)[b * a.q_tok + (kh * g + i / d) *
                                                      a.q_head + i % d];
  __syncthreads();
  const int len = a.c.len(b);
  if (slot >= a.c.room()) return;
  const long at = ((long)b * a.c.kvh + kh) * a.c.room() + slot;
  if (slot >= len) {
    a.mass_out[at] = 0.f;
    return;
  }
  float w = 0.f;
  const long page = a.c.page(b, slot);
  if (page >= 0)
    for (int i = 0; i < g; ++i) {
      const float lse = a.lse[(long)b * a.qh + kh * g + i];
      if (lse == -INFINITY) continue;
      w += expf(score<T>(a, qs + i * d, b, kh * g + i, slot, len, page) -
                lse);
    }
  a.mass_out[at] = a.mass[at] + w;
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
// Order of what stays: slots of the `recent` newest positions first, then
// by weight, NaN above all as a sort has it. Unsigned compare.
TD_DEV unsigned rank_key(float mass, bool is_recent) {
  if (is_recent) return 0xFFFFFFFFu;
  if (mass != mass) return 0xFFFFFFFEu;
  unsigned u = __float_as_uint(mass + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A workgroup per sequence and key head finds the kept slots and writes
// which row goes where: the i-th free slot below the budget takes the i-th
// kept row above it. ws: [batch, kvh] counts, then [batch, kvh, pairs, 2].
__global__ __launch_bounds__(256) void k_evict_select(EvictArgs a,
                                                      int pairs) {
  __shared__ int red[256];
  __shared__ unsigned pick;
  __shared__ int need, off_hole, off_mover;
  const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int room = a.c.room(), len = a.c.len(b);
  const long row = ((long)b * a.c.kvh + h) * room;
  const float *mass = a.mass + row;
  const int *pos = a.key_pos + row;
  int *count = (int *)a.ws + (long)b * a.c.kvh + h;
  int *list = (int *)a.ws + (long)a.c.batch * a.c.kvh +
              ((long)b * a.c.kvh + h) * pairs * 2;
  const int keep = min(len, a.budget);
  if (keep < len) {
    int newest = INT_MIN;
    for (int i = tid; i < len; i += 256) newest = max(newest, pos[i]);
    red[tid] = newest;
    __syncthreads();
    if (tid == 0)
      for (int i = 1; i < 256; ++i) newest = max(newest, red[i]);
    if (tid == 0) red[0] = newest;
    __syncthreads();
    const long since = (long)red[0] - a.recent;
    // the keep-th largest key, a bit at a time from the top
    unsigned t = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned with = t | 1u << bit;
      int n = 0;
      for (int i = tid; i < len; i += 256)
        n += rank_key(mass[i], pos[i] > since) >= with;
      __syncthreads();
      red[tid] = n;
      __syncthreads();
      if (tid == 0) {
        for (int i = 1; i < 256; ++i) n += red[i];
        pick = n >= keep ? with : t;
      }
      __syncthreads();
      t = pick;
    }
    int over = 0;
    for (int i = tid; i < len; i += 256)
      over += rank_key(mass[i], pos[i] > since) > t;
    __syncthreads();
    red[tid] = over;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < 256; ++i) over += red[i];
      need = keep - over;  // of those that equal t, the first ones stay
      int ties = 0, holes = 0, movers = 0;
      for (int i = 0; i < len; ++i) {
        const unsigned key = rank_key(mass[i], pos[i] > since);
        const bool stays = key > t || (key == t && ties++ < need);
        if (!stays && i < keep) list[2 * holes++] = i;
        if (stays && i >= keep) list[2 * movers++ + 1] = i;
      }
      *count = movers;
    }
  } else if (tid == 0) {
    *count = 0;
  }
}

__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a, int pairs) {
  const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int room = a.c.room(), len = a.c.len(b);
  const int keep = min(len, a.budget);
  const long row = ((long)b * a.c.kvh + h) * room;
  const int n = ((const int *)a.ws)[(long)b * a.c.kvh + h];
  const int *list = (const int *)a.ws + (long)a.c.batch * a.c.kvh +
                    ((long)b * a.c.kvh + h) * pairs * 2;
  if (a.mass_out != a.mass)
    for (int i = tid; i < keep; i += 256) a.mass_out[row + i] = a.mass[row + i];
  if (a.key_pos_out != a.key_pos)
    for (int i = tid; i < keep; i += 256)
      a.key_pos_out[row + i] = a.key_pos[row + i];
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const int to = list[2 * i], from = list[2 * i + 1];
    a.mass_out[row + to] = a.mass[row + from];
    a.key_pos_out[row + to] = a.key_pos[row + from];
  }
  __syncthreads();
  for (int i = keep + tid; i < room; i += 256) {
    a.mass_out[row + i] = 0.f;
    a.key_pos_out[row + i] = -1;
  }
  const int chunks = a.c.d / 8;
  for (int i = tid; i < n * chunks; i += 256) {
    const int to = list[i / chunks * 2], from = list[i / chunks * 2 + 1];
    const long pt = a.c.page(b, to), pf = a.c.page(b, from);
    if (pt < 0 || pf < 0) continue;
    const int c = i % chunks * 8, rt = to % a.c.block, rf = from % a.c.block;
    bf16 *k = (bf16 *)a.c.k + h * a.c.k_head + c;
    bf16 *v = (bf16 *)a.c.v + h * a.c.v_head + c;
    *(u32x4 *)(k + pt * a.c.k_page + rt * a.c.k_row) =
        *(u32x4 *)(k + pf * a.c.k_page + rf * a.c.k_row);
    *(u32x4 *)(v + pt * a.c.v_page + rt * a.c.v_row) =
        *(u32x4 *)(v + pf * a.c.v_page + rf * a.c.v_row);
  }
}

// Lengths last: the kernels before it read the old ones, which may be the
// same array.
__global__ __launch_bounds__(256) void k_evict_lens(EvictArgs a) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= a.c.batch) return;
  const int keep = min(a.c.len(b), a.budget);
  if (a.c.lens.is64) ((long *)a.lens_out)[b] = keep;
  else ((int *)a.lens_out)[b] = keep;
}

}  // namespace

void launch_paged_append(const PagedArgs &a, const void *k, long k_tok,
                         long k_head, const void *v, long v_tok, long v_head,
                         long tokens, IdxPtr cu, int *key_pos, IdxPtr pos,
                         hipStream_t stream) {
  const long threads = tokens * a.kvh * (a.d / 8);
  if (!threads || !a.batch) return;
  if (threads > 0x7fffffffL * 256)
    throw std::runtime_error("paged_append: too many tokens");
  k_paged_append<<<dim3((unsigned)((threads + 255) / 256)), 256, 0, stream>>>(
      a, (const bf16 *)k, k_tok, k_head, (const bf16 *)v, v_tok, v_head,
      tokens, cu, key_pos, pos);
  launched("paged_append");
}

size_t paged_decode_workspace(int, int, int, int, long, bool) { return 0; }

void launch_paged_decode(const PagedDecodeArgs &a, hipStream_t stream) {
  if (!a.c.batch) return;
  const dim3 grid(a.c.batch, a.qh);
  if (a.c.is_fp16) k_paged_decode<_Float16><<<grid, 256, 0, stream>>>(a);
  else k_paged_decode<bf16><<<grid, 256, 0, stream>>>(a);
  launched("paged_decode");
  if (a.mass && a.c.room()) {
    const dim3 mg((a.c.room() + 255) / 256, a.c.batch, a.c.kvh);
    const size_t lds = (size_t)(a.qh / a.c.kvh) * a.c.d * 4;
    if (a.c.is_fp16) k_paged_mass<_Float16><<<mg, 256, lds, stream>>>(a);
    else k_paged_mass<bf16><<<mg, 256, lds, stream>>>(a);
    launched("paged_decode");
  }
}

size_t kv_evict_workspace(int batch, int kvh, long room, int budget) {
  const long pairs = budget < room - budget ? budget : room - budget;
  return (size_t)batch * kvh * (1 + 2 * (pairs > 0 ? pairs : 0)) *
         sizeof(int);
}

void launch_kv_evict(const EvictArgs &a, hipStream_t stream) {
  if (!a.c.batch) return;
  const int room = a.c.max_blocks * a.c.block;
  const int pairs = max(0, min(a.budget, room - a.budget));
  const dim3 grid(a.c.batch, a.c.kvh);
  k_evict_select<<<grid, 256, 0, stream>>>(a, pairs);
  launched("kv_evict");
  k_evict_move<<<grid, 256, 0, stream>>>(a, pairs);
  launched("kv_evict");
  k_evict_lens<<<(a.c.batch + 255) / 256, 256, 0, stream>>>(a);
  launched("kv_evict");
}

}  // namespace td
