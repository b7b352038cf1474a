// Paged KV cache: rows quantised as they are written, and read back.
//
// Stored forms of one token's key (or value) of one head, x[0..D):
//   16 bits  x
//   8 bits   m = max(max|x|, 127 * 2^-64); code rint(127 x / m) in [-127, 127]; step m / 127
//   4 bits   lo = min x, r = max(max x - lo, 15 * 2^-64); code rint(15 (x - lo) / r) in
//            [0, 15]; (step, value of code 0) = (r / 15, lo). Two codes to a byte, the
//            even element in the low half.
// A row with a NaN, an infinity, or a range whose product above leaves fp32 stores NaN
// as its step and reads back as NaN throughout: the damage stays in that token and head.
//
// Multiplying before the one division (both products are exact for 16-bit inputs whose
// differences fit fp32) makes the halves that the rounding meets exact halves, so a code
// does not hang on the division's last bit.
#include "paged.cuh"

namespace gemq {

namespace {

constexpr int kRowThreads = 256;

// Which row a group of GL lanes handles: K rows of all tokens, then V rows.
struct RowId {
  int kv, token, head;
};
__device__ __forceinline__ RowId row_id(int64_t r, int64_t rows, int heads) {
  RowId id;
  id.kv = r >= rows;
  const uint32_t i = static_cast<uint32_t>(id.kv ? r - rows : r);
  id.token = static_cast<int>(i / static_cast<uint32_t>(heads));
  id.head = static_cast<int>(i - static_cast<uint32_t>(id.token) * static_cast<uint32_t>(heads));
  return id;
}

// rint(num / den) of the rounded fp32 quotient. The reciprocal's product is good to 4e-5
// here (|quotient| <= 127); only a quotient that near a half takes the division.
__device__ __forceinline__ int code_of(float num, float den, float inv) {
  const float y = num * inv, r = rintf(y);
  if (fabsf(fabsf(y - r) - 0.5f) < 1e-4f) return __float2int_rn(__fdiv_rn(num, den));
  return static_cast<int>(r);
}

// One group of GL lanes a row, eight elements a lane; U rows a group, their loads issued
// together (one row at a time a block has too few bytes on the way: the 50,001-token
// 8-bit case of 391 MB took 254 us).
template <typename T, int BITS, int GL, int U>
__global__ void __launch_bounds__(kRowThreads) k_cache_write(const KvDev c, const T* __restrict__ k,
                                                            const T* __restrict__ v, int64_t k_ts, int64_t k_hs,
                                                            int64_t v_ts, int64_t v_hs,
                                                            const int64_t* __restrict__ slots, int tokens) {
  constexpr int kGroups = kRowThreads / GL;
  const int64_t rows = static_cast<int64_t>(tokens) * c.kv_heads;
  const int sub = threadIdx.x % GL;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * (kGroups * U) + threadIdx.x / GL;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  grid_dep_wait();
  uint4 raw[U];
  int64_t slot[U];
  RowId id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * kGroups;
    const bool live = r < 2 * rows;
    id[u] = row_id(live ? r : 0, rows, c.kv_heads);
    slot[u] = live ? slots[id[u].token] : -1;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (live && sub * 8 < c.head_dim)
      raw[u] = __ldcs(reinterpret_cast<const uint4*>((id[u].kv ? v : k) + id[u].token * (id[u].kv ? v_ts : k_ts) +
                                                     id[u].head * (id[u].kv ? v_hs : k_hs) + sub * 8));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= total && sub == 0) set_device_error(kDevBadCachePos);
    const bool put = slot[u] >= 0 && slot[u] < total;
    const bool mine = put && sub * 8 < c.head_dim;
    const int page = static_cast<int>(slot[u] >> c.page_shift);
    const int off = static_cast<int>(slot[u] & ((int64_t(1) << c.page_shift) - 1));
    uint8_t* dst = (id[u].kv ? c.v : c.k) + (put ? c.row(page, id[u].head, off) : 0);
    if constexpr (BITS == 16) {
      if (mine) *reinterpret_cast<uint4*>(dst + sub * 16) = raw[u];
    } else {
      float x[8];
      const uint32_t ws[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(ws[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
      float lo = mine ? x[0] : INFINITY, hi = mine ? x[0] : -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = fmaf(x[i], 0.f, sum);  // a NaN or an infinity makes it a NaN
        if (mine) {
          lo = fminf(lo, x[i]);
          hi = fmaxf(hi, x[i]);
        }
      }
#pragma unroll
      for (int o = GL / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const uint32_t group = GL == 32 ? 0xffffffffu : ((1u << (GL & 31)) - 1u) << ((threadIdx.x & 31) / GL * GL);
      const bool any_bad = (__ballot_sync(0xffffffffu, isnan(sum)) & group) != 0;
      constexpr float kTop = BITS == 8 ? 127.f : 15.f;
      const float base = BITS == 8 ? 0.f : lo;
      const float range = fmaxf(BITS == 8 ? fmaxf(fabsf(lo), fabsf(hi)) : hi - lo, kTop * kMinScale);
      const bool poison = any_bad || !isfinite(range * kTop);
      if (mine) {
        const float inv = __frcp_rn(range);
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          q[i] = poison ? 0u : static_cast<uint32_t>(code_of((x[i] - base) * kTop, range, inv));
        if constexpr (BITS == 8) {
          uint2 w;
          w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
          w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
          *reinterpret_cast<uint2*>(dst + sub * 8) = w;
        } else {
          uint32_t w = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) w |= q[i] << (4 * i);
          *reinterpret_cast<uint32_t*>(dst + sub * 4) = w;
        }
        if (sub == 0) {
          float* s = (id[u].kv ? c.v_scale : c.k_scale) + c.scale_row(page, id[u].head, off);
          const float step = poison ? NAN : __fdiv_rn(range, kTop);
          if constexpr (BITS == 8) *s = step;
          else *reinterpret_cast<float2*>(s) = make_float2(step, poison ? NAN : lo);
        }
      }
    }
  }
}

// The mirror: out [tokens, heads, D] of T, one rounding. A negative slot reads zeros.
template <typename T, int BITS, int GL, int U>
__global__ void __launch_bounds__(kRowThreads) k_cache_read(const KvDev c, const int64_t* __restrict__ slots,
                                                           int tokens, T* __restrict__ k, T* __restrict__ v) {
  constexpr int kGroups = kRowThreads / GL;
  const int64_t rows = static_cast<int64_t>(tokens) * c.kv_heads;
  const int sub = threadIdx.x % GL;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * (kGroups * U) + threadIdx.x / GL;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  grid_dep_wait();
  if (sub * 8 >= c.head_dim) return;
  RowId id[U];
  bool live[U];
  uint4 raw[U];
  float2 sc[U];
  int64_t slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * kGroups;
    live[u] = r < 2 * rows;
    id[u] = row_id(live[u] ? r : 0, rows, c.kv_heads);
    slot[u] = live[u] ? slots[id[u].token] : -1;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= total && sub == 0) set_device_error(kDevBadCachePos);
    raw[u] = make_uint4(0, 0, 0, 0);
    sc[u] = make_float2(0.f, 0.f);
    if (slot[u] >= 0 && slot[u] < total) {
      const int page = static_cast<int>(slot[u] >> c.page_shift);
      const int off = static_cast<int>(slot[u] & ((int64_t(1) << c.page_shift) - 1));
      const uint8_t* src = (id[u].kv ? c.v : c.k) + c.row(page, id[u].head, off) + sub * BITS;
      if constexpr (BITS == 16) {
        raw[u] = __ldcs(reinterpret_cast<const uint4*>(src));
      } else {
        const float* s = (id[u].kv ? c.v_scale : c.k_scale) + c.scale_row(page, id[u].head, off);
        if constexpr (BITS == 8) {
          const uint2 w = __ldcs(reinterpret_cast<const uint2*>(src));
          raw[u].x = w.x;
          raw[u].y = w.y;
          sc[u].x = *s;
        } else {
          raw[u].x = __ldcs(reinterpret_cast<const uint32_t*>(src));
          sc[u] = *reinterpret_cast<const float2*>(s);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!live[u]) continue;
    uint4 out = raw[u];
    if constexpr (BITS != 16) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (BITS == 8)
          x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? raw[u].x : raw[u].y) >> (8 * (i & 3)))) * sc[u].x;
        else
          x[i] = fmaf(static_cast<float>((raw[u].x >> (4 * i)) & 15u), sc[u].x, sc[u].y);
      }
      out = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
    T* dst = (id[u].kv ? v : k) + (static_cast<int64_t>(id[u].token) * c.kv_heads + id[u].head) * c.head_dim + sub * 8;
    __stcs(reinterpret_cast<uint4*>(dst), out);
  }
}

struct WriteCall {
  KvDev c;
  const void *k, *v;
  int64_t k_ts, k_hs, v_ts, v_hs;
  const int64_t* slots;
  int tokens;
};

// Rows a group: four once that still gives every SM its blocks, else one.
int rows_a_group(const KvDev& c, int tokens, int gl) {
  const int64_t blocks = 2 * static_cast<int64_t>(tokens) * c.kv_heads * gl / (4 * kRowThreads);
  return blocks >= 4 * device_sm_count() ? 4 : 1;
}
unsigned row_blocks(const KvDev& c, int tokens, int gl, int rows) {
  const int64_t groups = (2 * static_cast<int64_t>(tokens) * c.kv_heads + rows - 1) / rows;
  return static_cast<unsigned>((groups * gl + kRowThreads - 1) / kRowThreads);
}

template <typename T, int BITS, int GL, int U>
cudaError_t write_u(const WriteCall& a, cudaStream_t s) {
  return launch_dep(k_cache_write<T, BITS, GL, U>, dim3(row_blocks(a.c, a.tokens, GL, U)), dim3(kRowThreads), 0, s, a.c,
                    static_cast<const T*>(a.k), static_cast<const T*>(a.v), a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.slots,
                    a.tokens);
}
template <typename T, int BITS, int GL>
cudaError_t write_gl(const WriteCall& a, cudaStream_t s) {
  return rows_a_group(a.c, a.tokens, GL) == 4 ? write_u<T, BITS, GL, 4>(a, s) : write_u<T, BITS, GL, 1>(a, s);
}
template <typename T, int BITS, int GL, int U>
cudaError_t read_u(const KvDev& c, const int64_t* slots, int tokens, void* k, void* v, cudaStream_t s) {
  return launch_dep(k_cache_read<T, BITS, GL, U>, dim3(row_blocks(c, tokens, GL, U)), dim3(kRowThreads), 0, s, c, slots,
                    tokens, static_cast<T*>(k), static_cast<T*>(v));
}
template <typename T, int BITS, int GL>
cudaError_t read_gl(const KvDev& c, const int64_t* slots, int tokens, void* k, void* v, cudaStream_t s) {
  return rows_a_group(c, tokens, GL) == 4 ? read_u<T, BITS, GL, 4>(c, slots, tokens, k, v, s)
                                          : read_u<T, BITS, GL, 1>(c, slots, tokens, k, v, s);
}

// Calls f with the lane group of the head size (the power of two that holds head_dim / 8
// lanes) as a compile-time constant.
template <typename F>
cudaError_t with_group(int head_dim, F&& f) {
  if (head_dim <= 16) return f(std::integral_constant<int, 2>());
  if (head_dim <= 32) return f(std::integral_constant<int, 4>());
  if (head_dim <= 64) return f(std::integral_constant<int, 8>());
  if (head_dim <= 128) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}
template <typename F>
cudaError_t with_form(bool bf16, int bits, F&& f) {
  auto g = [&](auto t) {
    if (bits == 16) return f(t, std::integral_constant<int, 16>());
    if (bits == 8) return f(t, std::integral_constant<int, 8>());
    return f(t, std::integral_constant<int, 4>());
  };
  return bf16 ? g(__nv_bfloat16()) : g(__half());
}

}  // namespace

cudaError_t launch_cache_write(const KvDev& c, int bits, bool bf16, const void* k, const void* v, int64_t k_ts,
                               int64_t k_hs, int64_t v_ts, int64_t v_hs, const int64_t* slots, int tokens,
                               cudaStream_t s) {
  const WriteCall a{c, k, v, k_ts, k_hs, v_ts, v_hs, slots, tokens};
  return with_form(bf16, bits, [&](auto t, auto b) {
    return with_group(c.head_dim, [&](auto gl) { return write_gl<decltype(t), decltype(b)::value, decltype(gl)::value>(a, s); });
  });
}

cudaError_t launch_cache_read(const KvDev& c, int bits, bool bf16, const int64_t* slots, int tokens, void* k, void* v,
                              cudaStream_t s) {
  return with_form(bf16, bits, [&](auto t, auto b) {
    return with_group(c.head_dim, [&](auto gl) {
      return read_gl<decltype(t), decltype(b)::value, decltype(gl)::value>(c, slots, tokens, k, v, s);
    });
  });
}

}  // namespace gemq
