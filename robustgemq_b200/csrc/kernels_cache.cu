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

// i / heads for i < 2^30 as a multiplication: with 2^(l - 1) < d <= 2^l and
// m = floor(2^(31 + l) / d) + 1, i / d = floor(i m / 2^(31 + l)) for every i < 2^31.
struct HeadDiv {
  uint32_t m;
  int shift;  // l - 1; -1: one head
};
HeadDiv head_div(int d) {
  if (d == 1) return {0u, -1};
  int l = 1;
  while ((1 << l) < d) ++l;
  return {static_cast<uint32_t>((uint64_t{1} << (31 + l)) / static_cast<uint32_t>(d) + 1), l - 1};
}

// Which row a group of GL lanes handles: K rows of all tokens, then V rows.
struct RowId {
  bool v;
  uint32_t token, head;
};
__device__ __forceinline__ RowId row_id(uint32_t r, uint32_t rows, uint32_t heads, HeadDiv d) {
  RowId id;
  id.v = r >= rows;
  const uint32_t i = id.v ? r - rows : r;
  id.token = d.shift < 0 ? i : __umulhi(i, d.m) >> d.shift;
  id.head = i - id.token * heads;
  return id;
}

// Where a slot's row lies. Slots are below 2^31 once checked.
__device__ __forceinline__ int64_t slot_row(const KvDev& c, uint32_t slot, uint32_t head) {
  return c.row(static_cast<int>(slot >> c.page_shift), static_cast<int>(head),
               static_cast<int>(slot & ((1u << c.page_shift) - 1u)));
}
__device__ __forceinline__ int64_t slot_scale(const KvDev& c, uint32_t slot, uint32_t head) {
  return c.scale_row(static_cast<int>(slot >> c.page_shift), static_cast<int>(head),
                     static_cast<int>(slot & ((1u << c.page_shift) - 1u)));
}

// Maximum of pairs; a NaN in either wins.
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }

// One group of GL lanes a row, eight elements a lane; U rows a group, their loads issued
// together. The first form (one row, every step in fp32, a division an element) executed
// 350 instructions a lane and row and was bound by their issue at 1.6 TB/s; the extremes
// are now taken on 16-bit pairs and the codes by one multiply and one add.
template <typename T, int BITS, int GL, int U>
__global__ void __launch_bounds__(kRowThreads) k_cache_write(const KvDev c, const T* __restrict__ k,
                                                            const T* __restrict__ v, int64_t k_ts, int64_t k_hs,
                                                            int64_t v_ts, int64_t v_hs,
                                                            const int64_t* __restrict__ slots, uint32_t rows,
                                                            HeadDiv div) {
  using T2 = typename Vec2<T>::type;
  constexpr int kGroups = kRowThreads / GL;
  const int sub = threadIdx.x % GL;
  const bool inside = sub * 8 < c.head_dim;
  const uint32_t r0 = blockIdx.x * static_cast<uint32_t>(kGroups * U) + threadIdx.x / GL;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  uint4 raw[U];
  int64_t slot[U];
  RowId id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = r0 + u * kGroups;
    const bool live = r < 2 * rows;
    id[u] = row_id(live ? r : 0u, rows, static_cast<uint32_t>(c.kv_heads), div);
    slot[u] = live ? __ldg(slots + id[u].token) : -1;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (live && inside) {
      const T* src = id[u].v ? v + id[u].token * v_ts + id[u].head * v_hs : k + id[u].token * k_ts + id[u].head * k_hs;
      raw[u] = __ldcs(reinterpret_cast<const uint4*>(src + sub * 8));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= total && sub == 0) set_device_error(kDevBadCachePos);
    const bool put = slot[u] >= 0 && slot[u] < total;
    const uint32_t at = put ? static_cast<uint32_t>(slot[u]) : 0u;
    uint8_t* dst = (id[u].v ? c.v : c.k) + slot_row(c, at, id[u].head) + sub * BITS;
    const uint32_t ws[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
    if constexpr (BITS == 16) {
      if (put && inside) *reinterpret_cast<uint4*>(dst) = raw[u];
    } else {
      // (max |x|, the same) or (max x, max -x) of the row
      T2 top;
      {
        T2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const T2*>(&ws[i]);
        if constexpr (BITS == 8) {
          top = max2(max2(__habs2(p[0]), __habs2(p[1])), max2(__habs2(p[2]), __habs2(p[3])));
          top = max2(top, __lowhigh2highlow(top));
        } else {
          T2 hi = max2(max2(p[0], p[1]), max2(p[2], p[3]));
          T2 lo = max2(max2(__hneg2(p[0]), __hneg2(p[1])), max2(__hneg2(p[2]), __hneg2(p[3])));
          hi = max2(hi, __lowhigh2highlow(hi));
          lo = max2(lo, __lowhigh2highlow(lo));
          const uint32_t both = __byte_perm(*reinterpret_cast<const uint32_t*>(&hi), *reinterpret_cast<const uint32_t*>(&lo), 0x5410);
          top = *reinterpret_cast<const T2*>(&both);
          // lanes past the row's end must not bring a zero
          const uint32_t none = std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
          if (!inside) top = *reinterpret_cast<const T2*>(&none);
        }
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) top = max2(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      const float2 ext = unpack2<T>(*reinterpret_cast<const uint32_t*>(&top));
      constexpr float kTop = BITS == 8 ? 127.f : 15.f;
      const float base = BITS == 8 ? 0.f : -ext.y;
      const float wide = BITS == 8 ? ext.x : ext.x - base;
      const bool poison = !isfinite(wide * kTop);  // also where a NaN or an infinity came up
      const float range = fmaxf(wide, kTop * kMinScale);
      // Codes: y = kTop (x - base) / range to within 5e-5, plus 1.5 * 2^23, whose sum's
      // low bits are rint(y). Only where some y comes that near a half is the rounded
      // fp32 quotient of the definition taken.
      constexpr float kMagic = 12582912.f;
      const float inv = poison ? 0.f : __frcp_rn(range) * kTop;
      float x[8], worst = 0.f;
      uint32_t q[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(ws[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = (BITS == 8 ? x[i] : x[i] - base) * inv;
        const float r = y + kMagic;
        worst = fmaxf(worst, fabsf(y - (r - kMagic)));
        q[i] = __float_as_uint(r);
      }
      if (worst > 0.4999f) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          q[i] = __float_as_uint(__fdiv_rn((BITS == 8 ? x[i] : x[i] - base) * kTop, range) + kMagic);
      }
      if (poison) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = 0;
      }
      if (put && inside) {
        uint2 w;
        w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
        if constexpr (BITS == 8) {
          *reinterpret_cast<uint2*>(dst) = w;
        } else {
          // bytes of one code each to two codes a byte
          const uint32_t a = (w.x | w.x >> 4) & 0x00ff00ffu, b = (w.y | w.y >> 4) & 0x00ff00ffu;
          *reinterpret_cast<uint32_t*>(dst) = __byte_perm(a, b, 0x6420);
        }
        if (sub == 0) {
          float* s = (id[u].v ? c.v_scale : c.k_scale) + slot_scale(c, at, id[u].head);
          const float step = poison ? NAN : __fdiv_rn(range, kTop);
          if constexpr (BITS == 8) *s = step;
          else *reinterpret_cast<float2*>(s) = make_float2(step, poison ? NAN : base);
        }
      }
    }
  }
}

// The mirror: out [tokens, heads, D] of T, one rounding. A negative slot reads zeros.
template <typename T, int BITS, int GL, int U>
__global__ void __launch_bounds__(kRowThreads) k_cache_read(const KvDev c, const int64_t* __restrict__ slots,
                                                           uint32_t rows, HeadDiv div, T* __restrict__ k,
                                                           T* __restrict__ v) {
  constexpr int kGroups = kRowThreads / GL;
  const int sub = threadIdx.x % GL;
  const uint32_t r0 = blockIdx.x * static_cast<uint32_t>(kGroups * U) + threadIdx.x / GL;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  if (sub * 8 >= c.head_dim) return;
  RowId id[U];
  bool live[U];
  uint4 raw[U];
  float2 sc[U];
  int64_t slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = r0 + u * kGroups;
    live[u] = r < 2 * rows;
    id[u] = row_id(live[u] ? r : 0u, rows, static_cast<uint32_t>(c.kv_heads), div);
    slot[u] = live[u] ? __ldg(slots + id[u].token) : -1;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= total && sub == 0) set_device_error(kDevBadCachePos);
    raw[u] = make_uint4(0, 0, 0, 0);
    sc[u] = make_float2(0.f, 0.f);
    if (slot[u] >= 0 && slot[u] < total) {
      const uint32_t at = static_cast<uint32_t>(slot[u]);
      const uint8_t* src = (id[u].v ? c.v : c.k) + slot_row(c, at, id[u].head) + sub * BITS;
      if constexpr (BITS == 16) {
        raw[u] = __ldcs(reinterpret_cast<const uint4*>(src));
      } else {
        const float* s = (id[u].v ? c.v_scale : c.k_scale) + slot_scale(c, at, id[u].head);
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
      // a code in the low byte of 2^23's pattern reads as 2^23 + code
      float x[8];
      uint32_t b0 = raw[u].x, b1 = raw[u].y;
      if constexpr (BITS == 8) {
        b0 ^= 0x80808080u;
        b1 ^= 0x80808080u;
      } else {
        b1 = (raw[u].x >> 4) & 0x0f0f0f0fu;  // odd elements
        b0 = raw[u].x & 0x0f0f0f0fu;         // even ones
      }
      constexpr float kBias = 8388608.f + (BITS == 8 ? 128.f : 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = BITS == 8 ? (i < 4 ? b0 : b1) : (i & 1 ? b1 : b0);
        const uint32_t byte = BITS == 8 ? i & 3 : i >> 1;
        const float f = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540u | byte)) - kBias;
        x[i] = BITS == 8 ? f * sc[u].x : fmaf(f, sc[u].x, sc[u].y);
      }
      out = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
    T* dst = (id[u].v ? v : k) + (static_cast<int64_t>(id[u].token) * c.kv_heads + id[u].head) * c.head_dim + sub * 8;
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
                    static_cast<uint32_t>(a.tokens) * static_cast<uint32_t>(a.c.kv_heads), head_div(a.c.kv_heads));
}
template <typename T, int BITS, int GL>
cudaError_t write_gl(const WriteCall& a, cudaStream_t s) {
  return rows_a_group(a.c, a.tokens, GL) == 4 ? write_u<T, BITS, GL, 4>(a, s) : write_u<T, BITS, GL, 1>(a, s);
}
template <typename T, int BITS, int GL, int U>
cudaError_t read_u(const KvDev& c, const int64_t* slots, int tokens, void* k, void* v, cudaStream_t s) {
  return launch_dep(k_cache_read<T, BITS, GL, U>, dim3(row_blocks(c, tokens, GL, U)), dim3(kRowThreads), 0, s, c, slots,
                    static_cast<uint32_t>(tokens) * static_cast<uint32_t>(c.kv_heads), head_div(c.kv_heads),
                    static_cast<T*>(k), static_cast<T*>(v));
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
