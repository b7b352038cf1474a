// What the paged KV cache's kernels share: the cache's device description, one row's
// address, and the 16-bit types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "gemq_common.cuh"
#include "gemq_internal.h"

namespace gemq {

// The smallest step a quantised row is stored with. Attention weights each value row by
// its step (2^log2 step), so the step must not be zero; 2^-64 is far below any real
// row's (a fp16 row's step is at least 2^-31 unless it is constant) and keeps 1 / step
// times any sequence length inside fp32.
constexpr float kMinScale = 5.421010862427522e-20f;  // 2^-64

// The step t with which a value row counts in attention, `base` its offset (the value of
// code 8 at 4 bits): what is stored, but at least 2^-64 (a step of zero) and 2^-100 |base|,
// so that base / t stays in fp32 for a row of large equal values, whose codes say nothing.
// Either moves a value by less than 2^-96 of it. A NaN stays. A step above 2^38 (only bf16
// rows of values above 10^12 have one) is none: a weight is held as 2^x t beside the largest
// one that the row sees, and where steps reach from 2^-64 (rows of zeros) further than that,
// keys of equal weight fall out of fp32 and were lost from the sum of the weights.
constexpr float kMaxValueStep = 274877906944.f;  // 2^38
__device__ __forceinline__ float value_step(float stored, float base) {
  const float least = fmaxf(kMinScale, fabsf(base) * 7.888609052210118e-31f);
  const float step = stored < least ? least : stored;
  return step > kMaxValueStep ? NAN : step;
}

// gemq_kv_cache_t as the kernels take it. Strides between pages, heads and tokens: of the
// codes in units of 8 bytes, of the scales in floats; below 2^31 each, so that a row's
// address takes three 32 x 32 -> 64 bit multiply-adds.
struct KvDev {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  uint32_t page_stride, head_stride, token_stride;
  uint32_t scale_page_stride, scale_head_stride, scale_token_stride;
  int num_pages, kv_heads, page_shift, head_dim;

  __device__ __forceinline__ int64_t row(int page, int head, int off) const {
    return static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_stride +
                                 static_cast<uint64_t>(static_cast<uint32_t>(head)) * head_stride +
                                 static_cast<uint64_t>(static_cast<uint32_t>(off)) * token_stride) << 3);
  }
  __device__ __forceinline__ int64_t scale_row(int page, int head, int off) const {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * scale_page_stride +
                                static_cast<uint64_t>(static_cast<uint32_t>(head)) * scale_head_stride +
                                static_cast<uint64_t>(static_cast<uint32_t>(off)) * scale_token_stride);
  }
};

template <typename T>
struct Vec2;
template <>
struct Vec2<__half> {
  using type = __half2;
};
template <>
struct Vec2<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two fp32 values rounded to a pair of T, as the 32 bits of the pair.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}

constexpr float kHalfMin = 6.103515625e-5f;  // 2^-14, the smallest normal fp16 number
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Pairs of fp32 and their arithmetic in one instruction a pair.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Positions of a sequence that attention takes: below 2^31 by more than a kernel's tiles and
// units of keys, and the tiles asked for ahead, reach past the last one.
constexpr int kMaxPositions = 0x7fffffff - 1023;

// Everything an attention launch needs.
struct AttnArgs {
  KvDev kv;
  const void* q;
  int64_t q_token_stride;  // elements
  const int32_t* page_table;
  int64_t page_table_stride;
  int max_pages;
  const int32_t* kv_lens;
  const int32_t* q_starts;  // null: every sequence has num_tokens / num_seqs tokens
  int num_tokens, num_seqs, q_heads, group;
  float scale;
  int window;  // 0: none
  void* out;
  float* lse;  // may be null
};

// New tokens [start, start + len) of sequence b and its length with them, clamped to the
// buffers (a value outside them is recorded in the device error word).
struct SeqRange {
  int start, q_len, kv_len;
};
__device__ __forceinline__ SeqRange seq_range(const AttnArgs& a, int b) {
  SeqRange r;
  int lo, hi;
  if (a.q_starts != nullptr) {
    lo = a.q_starts[b];
    hi = a.q_starts[b + 1];
  } else {
    const int n = a.num_tokens / a.num_seqs;
    lo = b * n;
    hi = lo + n;
  }
  const int kv = a.kv_lens[b];
  const int cap = min(a.max_pages << a.kv.page_shift, kMaxPositions);
  r.start = min(max(lo, 0), a.num_tokens);
  r.q_len = min(max(hi, r.start), a.num_tokens) - r.start;
  r.kv_len = min(max(kv, 0), cap);
  if (lo != r.start || hi != r.start + r.q_len || kv != r.kv_len) set_device_error(kDevBadCachePos);
  return r;
}

// The first position that a row at position `last` sees. (Neither of the two may be taken
// from the other as they are: a row before position 0 with the widest window leaves 32 bits.)
__device__ __forceinline__ int first_seen(int last, int window) {
  return window > 0 && last >= window ? last - window + 1 : 0;
}

// The page of a sequence's page index, or -1 (recorded) for an id outside the cache.
__device__ __forceinline__ int page_of(const AttnArgs& a, int b, int index) {
  const int p = a.page_table[b * a.page_table_stride + index];
  if (p >= 0 && p < a.kv.num_pages) return p;
  set_device_error(kDevBadCachePos);
  return -1;
}

// Launchers (kernels_cache.cu, kernels_attn.cu, kernels_verify.cu). Arguments are checked
// by the C ABI before they come here.
cudaError_t launch_cache_write(const KvDev& c, int bits, bool bf16, const void* k, const void* v, int64_t k_ts,
                               int64_t k_hs, int64_t v_ts, int64_t v_hs, const int64_t* slots, int tokens,
                               cudaStream_t s);
cudaError_t launch_cache_read(const KvDev& c, int bits, bool bf16, const int64_t* slots, int tokens, void* k, void* v,
                              cudaStream_t s);
size_t attention_workspace(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len);
cudaError_t launch_attention(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len, void* workspace,
                             cudaStream_t s);
// (kernels_attn_tc.cu: many rows a KV head)
size_t many_workspace(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len);
cudaError_t launch_many(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len, void* workspace,
                        cudaStream_t s);
size_t verify_workspace(int B, int n, int V);
cudaError_t launch_verify(const gemq_verify_t& v, int B, int n, int V, void* workspace, cudaStream_t s);

}  // namespace gemq
