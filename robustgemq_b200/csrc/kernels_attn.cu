// Attention of a chunk of new tokens over a paged KV cache.
//
// Row (token i of the n new ones of a sequence of length L with them, query head h) has
// position p = L - n + i and sees the keys j <= p (j > p - window where there is one):
//   o = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j - m),  c = scale log2(e),
//   lse = (m + log2 sum_j w_j) ln(2)
// A row that sees nothing gives o = 0 and lse = -inf. What a row does not see does not
// reach it whatever it holds.
#include "paged.cuh"

namespace gemq {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Eight elements of a stored row, from element 8 * c.
template <typename T, int BITS>
__device__ __forceinline__ void load8(const uint8_t* row, int c, float step, float base, float (&x)[8]) {
  if constexpr (BITS == 16) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + c * 16);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else if constexpr (BITS == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(row + c * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * step;
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + c * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>((w >> (4 * i)) & 15u), step, base);
  }
}

constexpr int kRowThreads = 128;
constexpr int kRowMaxDim = 256;

struct RowSmem {
  float q[kRowMaxDim];
  float p[kRowThreads];
  float red[kRowThreads / 32];
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
  for (int i = 1; i < kRowThreads / 32; ++i) r = is_max ? fmaxf(r, red[i]) : r + red[i];
  return r;
}

// One row by one block of kRowThreads threads, in fp32 throughout: a thread takes whole
// keys for the scores and then elements of the output. Keys that the row does not see
// are never read.
template <typename T, int BITS>
__device__ void attn_one_row(const AttnArgs& a, int b, const SeqRange& r, int i, int h, RowSmem& sm) {
  const int D = a.kv.head_dim;
  const int kvh = h / a.group;
  const T* q = static_cast<const T*>(a.q) + (r.start + i) * a.q_token_stride + static_cast<int64_t>(h) * D;
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kRowThreads) sm.q[d] = to_f32(q[d]);
  __syncthreads();
  const int pos = r.kv_len - r.q_len + i;
  const int j1 = min(pos, r.kv_len - 1) + 1;
  const int j0 = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int mask = (1 << a.kv.page_shift) - 1;
  float m = -INFINITY, l = 0.f, o[kRowMaxDim / kRowThreads] = {};
  for (int jb = j0; jb < j1; jb += kRowThreads) {
    const int j = jb + static_cast<int>(threadIdx.x);
    float s = -INFINITY;
    if (j < j1) {
      const int page = page_of(a, b, j >> a.kv.page_shift);
      if (page >= 0) {
        const uint8_t* row = a.kv.k + a.kv.row(page, kvh, j & mask);
        float step = 1.f, base = 0.f;
        if constexpr (BITS != 16) {
          const float* sc = a.kv.k_scale + a.kv.scale_row(page, kvh, j & mask);
          step = sc[0];
          if constexpr (BITS == 4) base = sc[1];
        }
        float dot = 0.f;
        for (int c = 0; c < D / 8; ++c) {
          float x[8];
          load8<T, BITS>(row, c, step, base, x);
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
    const int cnt = min(kRowThreads, j1 - jb);
#pragma unroll
    for (int u = 0; u < kRowMaxDim / kRowThreads; ++u) {
      const int d = threadIdx.x + u * kRowThreads;
      if (d >= D) continue;
      float acc = o[u] * keep;
      for (int t = 0; t < cnt; ++t) {
        const int jj = jb + t;
        const int page = page_of(a, b, jj >> a.kv.page_shift);
        if (page < 0) continue;
        const uint8_t* row = a.kv.v + a.kv.row(page, kvh, jj & mask);
        float x;
        if constexpr (BITS == 16) {
          x = to_f32(reinterpret_cast<const T*>(row)[d]);
        } else {
          const float* sc = a.kv.v_scale + a.kv.scale_row(page, kvh, jj & mask);
          if constexpr (BITS == 8) x = static_cast<float>(reinterpret_cast<const int8_t*>(row)[d]) * sc[0];
          else x = fmaf(static_cast<float>((row[d >> 1] >> (4 * (d & 1))) & 15), sc[0], sc[1]);
        }
        acc = fmaf(sm.p[t], x, acc);
      }
      o[u] = acc;
    }
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // an empty row gives 0, a NaN one NaN
  T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(r.start + i) * a.q_heads + h) * D;
#pragma unroll
  for (int u = 0; u < kRowMaxDim / kRowThreads; ++u) {
    const int d = threadIdx.x + u * kRowThreads;
    if (d < D) out[d] = from_f32<T>(o[u] * inv);
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[static_cast<int64_t>(r.start + i) * a.q_heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// One block a row: the simplest form.
template <typename T, int BITS>
__global__ void __launch_bounds__(kRowThreads) k_attn_rows(const AttnArgs a) {
  __shared__ RowSmem sm;
  grid_dep_wait();
  const int h = blockIdx.x % a.q_heads;
  const int t = blockIdx.x / a.q_heads;
  for (int b = 0; b < a.num_seqs; ++b) {
    const SeqRange r = seq_range(a, b);
    if (t >= r.start && t < r.start + r.q_len) {
      attn_one_row<T, BITS>(a, b, r, t - r.start, h, sm);
      return;
    }
  }
}

}  // namespace

size_t attention_workspace(const AttnArgs&, int, int, int) { return 0; }

cudaError_t launch_attention(const AttnArgs& a, int bits, bool bf16, int, int, void*, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.num_tokens) * static_cast<unsigned>(a.q_heads)), block(kRowThreads);
  if (bf16) {
    if (bits == 16) return launch_dep(k_attn_rows<__nv_bfloat16, 16>, grid, block, 0, s, a);
    if (bits == 8) return launch_dep(k_attn_rows<__nv_bfloat16, 8>, grid, block, 0, s, a);
    return launch_dep(k_attn_rows<__nv_bfloat16, 4>, grid, block, 0, s, a);
  }
  if (bits == 16) return launch_dep(k_attn_rows<__half, 16>, grid, block, 0, s, a);
  if (bits == 8) return launch_dep(k_attn_rows<__half, 8>, grid, block, 0, s, a);
  return launch_dep(k_attn_rows<__half, 4>, grid, block, 0, s, a);
}

}  // namespace gemq
