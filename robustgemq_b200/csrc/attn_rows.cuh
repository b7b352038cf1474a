// One attention row by one block over a cache of 16 bits, in fp32 on the CUDA cores: the
// plainest form, which the kernel for chunks falls back on for rows its tiles cannot keep
// apart (codes need no such form: a key's factors say what is no number).
#pragma once

#include "paged.cuh"

namespace gemq {

// Eight elements of a row, from element 8 * c.
template <typename T>
__device__ __forceinline__ void load8(const uint8_t* row, int c, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(row + c * 16);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(u[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

constexpr int kAttnRowThreads = 128;
constexpr int kAttnMaxDim = 256;

struct AttnRowSmem {
  float q[kAttnMaxDim];
  float p[kAttnRowThreads];
  float red[kAttnRowThreads / 32];
};

__device__ __forceinline__ float row_reduce(float v, bool is_max, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = is_max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();  // red may still be read by the previous reduction
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < kAttnRowThreads / 32; ++i) r = is_max ? fmaxf(r, red[i]) : r + red[i];
  return r;
}

// One row by one block of kAttnRowThreads threads, in fp32 throughout: a thread takes whole
// keys for the scores and then elements of the output. Keys that the row does not see
// are never read.
template <typename T>
__device__ void attn_one_row(const AttnArgs& a, int b, const SeqRange& r, int i, int h, AttnRowSmem& sm) {
  const int D = a.kv.head_dim;
  const int kvh = h / a.group;
  const T* q = static_cast<const T*>(a.q) + (r.start + i) * a.q_token_stride + static_cast<int64_t>(h) * D;
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kAttnRowThreads) sm.q[d] = to_f32(q[d]);
  __syncthreads();
  const int pos = r.kv_len - r.q_len + i;
  const int j1 = min(pos, r.kv_len - 1) + 1;
  const int j0 = first_seen(pos, a.window);
  const int mask = (1 << a.kv.page_shift) - 1;
  float m = -INFINITY, l = 0.f, o[kAttnMaxDim / kAttnRowThreads] = {};
  for (int jb = j0; jb < j1; jb += kAttnRowThreads) {
    const int j = jb + static_cast<int>(threadIdx.x);
    float s = -INFINITY;
    if (j < j1) {
      const int page = page_of(a, b, j >> a.kv.page_shift);
      if (page >= 0) {
        const uint8_t* row = a.kv.k + a.kv.row(page, kvh, j & mask);
        float dot = 0.f;
        for (int c = 0; c < D / 8; ++c) {
          float x[8];
          load8<T>(row, c, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = fmaf(sm.q[8 * c + e], x[e], dot);
        }
        s = dot * (a.scale * kLog2e);
      }
    }
    // a NaN score has to reach the sums: fmaxf alone would drop it
    const float top = fmaxf(m, row_reduce(s, true, sm.red));
    const float ref = top == -INFINITY ? 0.f : top;
    const float keep = exp2f(m - ref);
    const float p = j < j1 ? exp2f(s - ref) : 0.f;
    sm.p[threadIdx.x] = p;
    l = l * keep + row_reduce(p, false, sm.red);  // its barriers also publish p
    m = top;
    const int cnt = min(kAttnRowThreads, j1 - jb);
#pragma unroll
    for (int u = 0; u < kAttnMaxDim / kAttnRowThreads; ++u) {
      const int d = threadIdx.x + u * kAttnRowThreads;
      if (d >= D) continue;
      float acc = o[u] * keep;
      for (int t = 0; t < cnt; ++t) {
        const int jj = jb + t;
        const int page = page_of(a, b, jj >> a.kv.page_shift);
        if (page < 0) continue;
        const uint8_t* row = a.kv.v + a.kv.row(page, kvh, jj & mask);
        acc = fmaf(sm.p[t], to_f32(reinterpret_cast<const T*>(row)[d]), acc);
      }
      o[u] = acc;
    }
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // an empty row gives 0, a NaN one NaN
  T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(r.start + i) * a.q_heads + h) * D;
#pragma unroll
  for (int u = 0; u < kAttnMaxDim / kAttnRowThreads; ++u) {
    const int d = threadIdx.x + u * kAttnRowThreads;
    if (d < D) out[d] = from_f32<T>(o[u] * inv);
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[static_cast<int64_t>(r.start + i) * a.q_heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace gemq
