// Attention of packed prompts: documents side by side without padding, each
// token seeing only its own document, causally or not, with a prefix that
// all of a document's tokens see.
#include <stdexcept>
#include <string>

#include "td/api.hpp"
#include "td/paged.hpp"

namespace td {

namespace {

using bf16 = __bf16;

// A workgroup per row and query head.
template <typename T>
__global__ __launch_bounds__(256) void k_packed_rows(PackedArgs a) {
  __shared__ float q[256], p[256], red[4], part[256];
  const long row = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x, d = a.d;
  const int kh = h / (a.qh / a.kvh);
  int lo = 0, hi = a.seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid + 1] <= row) lo = mid + 1; else hi = mid;
  }
  T *out = (T *)a.out + row * a.out_tok + h * a.out_head;
  if (lo >= a.seqs || row < a.cu_q[lo]) {  // behind the last document
    if (a.clear_tail) {
      if (tid < d) out[tid] = (T)0.f;
      if (a.lse && tid == 0) a.lse[row * a.qh + h] = -INFINITY;
    }
    return;
  }
  const long k0 = min(max(a.cu_k[lo], 0L), a.keys);
  const long k1 = min(max(a.cu_k[lo + 1], k0), a.keys);
  const long q0 = a.cu_q[lo], q1 = min(a.cu_q[lo + 1], a.rows);
  const long n = k1 - k0;
  const long at = row - q0 + n - (q1 - q0);  // the row's own key position
  long see = n;
  if (a.causal) {
    see = min(n, max(at + 1, 0L));
    if (a.prefix.p) see = max(see, min(n, a.prefix[lo]));
  }
  if (tid < d)
    q[tid] = (float)((const T *)a.q)[row * a.q_tok + h * a.q_head + tid];
  float m = -INFINITY, l = 0.f, acc = 0.f;
  const int col = tid % d, lane = tid / d, lanes = 256 / d;
  for (long base = 0; base < see; base += 256) {
    __syncthreads();
    const long j = base + tid;
    float s = -INFINITY;
    if (j < see) {
      const T *kr = (const T *)a.k + (k0 + j) * a.k_tok + kh * a.k_head;
      s = 0.f;
      for (int i = 0; i < d; ++i) s += q[i] * (float)kr[i];
      s *= a.s.scale;
      if (a.s.softcap > 0.f) s = a.s.softcap * tanhf(s / a.s.softcap);
      if (a.s.slopes) s -= a.s.slopes[h] * (float)(at > j ? at - j : j - at);
    }
    float top = s;
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    const float mn = fmaxf(
        m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float safe = mn == -INFINITY ? 0.f : mn;
    const float r = expf(m - safe);
    p[tid] = expf(s - safe);
    m = mn;
    acc *= r;
    l *= r;
    __syncthreads();
    for (int i = 0; i < 256; ++i) l += p[i];
    const int some = (int)min(256L, see - base);
    for (int i = lane; i < some; i += lanes)
      acc += p[i] * (float)((const T *)a.v)[(k0 + base + i) * a.v_tok +
                                            kh * a.v_head + col];
  }
  __syncthreads();
  part[tid] = acc;
  __syncthreads();
  if (tid < d) {
    for (int i = 1; i < lanes; ++i) acc += part[i * d + tid];
    out[tid] = (T)(l > 0.f ? acc / l : 0.f);
    if (a.lse && tid == 0)
      a.lse[row * a.qh + h] = l > 0.f ? m + logf(l) : -INFINITY;
  }
}

}  // namespace

void launch_packed_prefill(const PackedArgs &a, hipStream_t stream) {
  if (!a.rows) return;
  if (a.rows > 0x7fffffffL)
    throw std::runtime_error("packed_prefill: too many rows");
  const dim3 grid((unsigned)a.rows, a.qh);
  if (a.is_fp16) k_packed_rows<_Float16><<<grid, 256, 0, stream>>>(a);
  else k_packed_rows<bf16><<<grid, 256, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    throw std::runtime_error(std::string("packed_prefill: ") +
                             hipGetErrorString(e));
}

}  // namespace td
