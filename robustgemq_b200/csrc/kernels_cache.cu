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
// Of two tokens written to one slot parts of both may stay: a row's pieces and its scale are
// separate stores of separate warps.
//
// Each pass reads its rows once and writes them once. Measured on a B200, written and read
// back in one graph, 50,001 tokens of 8 heads x 80, 8 bits: 81 us for 391 MB (4.8 TB/s of
// the copy's 6.56; the read is at 6.0; the write takes 54 for 30 us of bytes, a warp's loads,
// reductions and stores one after the other and 68% of its issue slots used); 8,192 of
// 4 x 128, 4 bits: 15 us for 43 MB, two launches that each last a few memory latencies; 64
// of 16 x 128: 4 us, one latency each.
//
// Multiplying before the one division (both products are exact for 16-bit inputs whose
// differences fit fp32) makes the halves that the rounding meets exact halves, so a code
// does not hang on the division's last bit.
#include "paged.cuh"

namespace gemq {

namespace {

constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;

// How a warp takes rows: a lane takes two chunks of eight elements, half a row apart, so
// G = D / 16 lanes a row and 32 / G rows a warp (D is a multiple of 16). The lanes of a
// half are neighbours in memory in every form.
struct Lanes {
  int g, rows;      // lanes a row, rows a warp
  uint32_t inv_g;   // floor(65536 / g) + 1: l / g = l inv_g >> 16 for l < 32
};
Lanes lanes_of(int head_dim) {
  const int g = head_dim / 16;
  return {g, 32 / g, 65536u / static_cast<uint32_t>(g) + 1u};
}
struct Lane {
  int row, sub;  // of the warp's rows; of the row's lanes
  bool has_row;  // the last 32 % G lanes have none
};
__device__ __forceinline__ Lane lane_of(const Lanes& l) {
  const int lane = threadIdx.x & 31;
  Lane x;
  x.row = static_cast<int>(static_cast<uint32_t>(lane) * l.inv_g >> 16);
  x.sub = lane - x.row * l.g;
  x.has_row = x.row < l.rows;
  return x;
}

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

// Codes of eight elements, one to a byte, and how near any of them is to a half:
// y = kTop (x - base) / range to within 5e-5, plus 1.5 * 2^23, whose sum's low bits are
// rint(y).
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ uint2 bytes_of(const uint32_t (&q)[8]) {
  return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
}
template <typename T, int BITS>
__device__ __forceinline__ uint2 encode(const uint4& raw, float base, float inv, float& worst) {
  const uint32_t ws[4] = {raw.x, raw.y, raw.z, raw.w};
  const F2 inv2 = f2(inv, inv), magic = f2(kMagic, kMagic), neg = f2(-1.f, -1.f), from = f2(-base, -base);
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(ws[i]);
    F2 x = f2(f.x, f.y);
    if constexpr (BITS == 4) x = add2(x, from);
    const F2 r = fma2(x, inv2, magic);
    float e0, e1, r0, r1;
    split(fma2(x, inv2, fma2(r, neg, magic)), e0, e1);
    split(r, r0, r1);
    worst = fmaxf(worst, fmaxf(fabsf(e0), fabsf(e1)));
    q[2 * i] = __float_as_uint(r0);
    q[2 * i + 1] = __float_as_uint(r1);
  }
  return bytes_of(q);
}
// The definition's rounded quotients where an element's y comes near a half (halves are
// common: an element of half the row's maximum is one at 8 bits).
template <typename T, int BITS>
__device__ __forceinline__ uint2 encode_near(const uint4& raw, float base, float inv, float range, uint2 w) {
  const uint32_t ws[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    constexpr float kTop = BITS == 8 ? 127.f : 15.f;
    const float2 f = unpack2<T>(ws[i / 2]);
    const float x = (i & 1 ? f.y : f.x) - base, y = x * inv;
    if (fabsf(y - rintf(y)) > 0.4998f) {
      const uint32_t q = __float_as_uint(__fdiv_rn(x * kTop, range) + kMagic);
      // byte i % 4 of its word
      uint32_t& to = i < 4 ? w.x : w.y;
      to = __byte_perm(to, q, i % 4 == 0 ? 0x3214 : i % 4 == 1 ? 0x3240 : i % 4 == 2 ? 0x3410 : 0x4210);
    }
  }
  return w;
}
template <int BITS>
__device__ __forceinline__ void put_codes(uint8_t* dst, uint2 w) {
  if constexpr (BITS == 8) {
    *reinterpret_cast<uint2*>(dst) = w;
  } else {
    // bytes of one code each to two codes a byte
    const uint32_t a = (w.x | w.x >> 4) & 0x00ff00ffu, b = (w.y | w.y >> 4) & 0x00ff00ffu;
    *reinterpret_cast<uint32_t*>(dst) = __byte_perm(a, b, 0x6420);
  }
}

// U rows a group, their loads issued together. The first form (a row to 16 lanes, every
// step in fp32, a division an element) executed 350 instructions a lane of eight elements
// and was bound by their issue; the extremes are now taken on 16-bit pairs, the codes in
// three packed operations a pair, and a row's addresses and scales serve twice the
// elements (280 a lane of sixteen). Two blocks more an SM (64 registers a thread instead
// of 78) are worth 9%.
template <typename T, int BITS, int U>
__global__ void __launch_bounds__(kRowThreads, 8) k_cache_write(const KvDev c, const T* __restrict__ k,
                                                            const T* __restrict__ v, int64_t k_ts, int64_t k_hs,
                                                            int64_t v_ts, int64_t v_hs,
                                                            const int64_t* __restrict__ slots, uint32_t rows,
                                                            HeadDiv div, Lanes lanes) {
  using T2 = typename Vec2<T>::type;
  const Lane me = lane_of(lanes);
  const uint32_t r0 = (blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * static_cast<uint32_t>(U * lanes.rows) + me.row;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  uint4 raw[U][2];
  int64_t slot[U];
  RowId id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = r0 + u * lanes.rows;
    const bool live = me.has_row && r < 2 * rows;
    id[u] = row_id(live ? r : 0u, rows, static_cast<uint32_t>(c.kv_heads), div);
    slot[u] = -1;
    raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
    if (live) {
      slot[u] = __ldg(slots + id[u].token);
      const T* src = id[u].v ? v + id[u].token * v_ts + id[u].head * v_hs : k + id[u].token * k_ts + id[u].head * k_hs;
      raw[u][0] = __ldcs(reinterpret_cast<const uint4*>(src + me.sub * 8));
      raw[u][1] = __ldcs(reinterpret_cast<const uint4*>(src + (me.sub + lanes.g) * 8));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= total && me.sub == 0) set_device_error(kDevBadCachePos);
    const bool put = slot[u] >= 0 && slot[u] < total;
    const uint32_t at = put ? static_cast<uint32_t>(slot[u]) : 0u;
    uint8_t* dst = (id[u].v ? c.v : c.k) + slot_row(c, at, id[u].head) + me.sub * BITS;
    if constexpr (BITS == 16) {
      if (put) {
        *reinterpret_cast<uint4*>(dst) = raw[u][0];
        *reinterpret_cast<uint4*>(dst + lanes.g * BITS) = raw[u][1];
      }
    } else {
      // (max |x|, the same) or (max x, max -x) of the row
      T2 top;
      {
        T2 p[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t ws[4] = {raw[u][i].x, raw[u][i].y, raw[u][i].z, raw[u][i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) p[4 * i + e] = *reinterpret_cast<const T2*>(&ws[e]);
        }
        if constexpr (BITS == 8) {
          top = __habs2(p[0]);
#pragma unroll
          for (int i = 1; i < 8; ++i) top = max2(top, __habs2(p[i]));
          top = max2(top, __lowhigh2highlow(top));
        } else {
          T2 hi = p[0], lo = __hneg2(p[0]);
#pragma unroll
          for (int i = 1; i < 8; ++i) {
            hi = max2(hi, p[i]);
            lo = max2(lo, __hneg2(p[i]));
          }
          hi = max2(hi, __lowhigh2highlow(hi));
          lo = max2(lo, __lowhigh2highlow(lo));
          const uint32_t both = __byte_perm(*reinterpret_cast<const uint32_t*>(&hi), *reinterpret_cast<const uint32_t*>(&lo), 0x5410);
          top = *reinterpret_cast<const T2*>(&both);
        }
        // round the row's lanes, each step doubling what a lane has seen
#pragma unroll
        for (int o = 1; o < 16; o *= 2) {
          if (o >= lanes.g) break;
          const int to = me.sub + o;
          top = max2(top, __shfl_sync(0xffffffffu, top, me.row * lanes.g + (to < lanes.g ? to : to - lanes.g)));
        }
      }
      const float2 ext = unpack2<T>(*reinterpret_cast<const uint32_t*>(&top));
      constexpr float kTop = BITS == 8 ? 127.f : 15.f;
      const float base = BITS == 8 ? 0.f : -ext.y;
      const float wide = BITS == 8 ? ext.x : ext.x - base;
      const bool poison = !isfinite(wide * kTop);  // also where a NaN or an infinity came up
      const float range = fmaxf(wide, kTop * kMinScale);
      const float inv = poison ? 0.f : __frcp_rn(range) * kTop;
      float worst = 0.f;
      uint2 w0 = encode<T, BITS>(raw[u][0], base, inv, worst), w1 = encode<T, BITS>(raw[u][1], base, inv, worst);
      // only where some y comes that near a half is the rounded fp32 quotient taken
      if (worst > 0.4999f) {
        w0 = encode_near<T, BITS>(raw[u][0], base, inv, range, w0);
        w1 = encode_near<T, BITS>(raw[u][1], base, inv, range, w1);
      }
      if (poison) w0 = w1 = make_uint2(0, 0);
      if (put) {
        put_codes<BITS>(dst, w0);
        put_codes<BITS>(dst + lanes.g * BITS, w1);
        if (me.sub == 0) {
          float* s = (id[u].v ? c.v_scale : c.k_scale) + slot_scale(c, at, id[u].head);
          const float step = poison ? NAN : __fdiv_rn(range, kTop);
          if constexpr (BITS == 8) *s = step;
          else *reinterpret_cast<float2*>(s) = make_float2(step, poison ? NAN : base);
        }
      }
    }
  }
}

// Eight elements from their codes: a code in the low byte of 2^23's pattern reads as
// 2^23 + code.
template <typename T, int BITS>
__device__ __forceinline__ uint4 decode(const uint4& raw, float step, float base) {
  uint32_t b0 = raw.x, b1 = raw.y;
  if constexpr (BITS == 8) {
    b0 ^= 0x80808080u;
    b1 ^= 0x80808080u;
  } else {
    b1 = (raw.x >> 4) & 0x0f0f0f0fu;  // odd elements
    b0 = raw.x & 0x0f0f0f0fu;         // even ones
  }
  constexpr float kBias = 8388608.f + (BITS == 8 ? 128.f : 0.f);
  const F2 bias = f2(-kBias, -kBias), step2 = f2(step, step), base2 = f2(base, base);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t w = BITS == 8 ? (i < 2 ? b0 : b1) : (j ? b1 : b0);
      const uint32_t byte = BITS == 8 ? (2 * i + j) & 3 : i;
      x[j] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540u | byte));
    }
    const F2 f = add2(f2(x[0], x[1]), bias);
    split(BITS == 8 ? mul2(f, step2) : fma2(f, step2, base2), x[0], x[1]);
    out[i] = pack2<T>(x[0], x[1]);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}
template <int BITS>
__device__ __forceinline__ uint4 get_codes(const uint8_t* src) {
  if constexpr (BITS == 16) return __ldcs(reinterpret_cast<const uint4*>(src));
  if constexpr (BITS == 8) {
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(src));
    return make_uint4(w.x, w.y, 0, 0);
  }
  return make_uint4(__ldcs(reinterpret_cast<const uint32_t*>(src)), 0, 0, 0);
}

// The mirror: out [tokens, heads, D] of T, one rounding. A negative slot reads zeros.
template <typename T, int BITS, int U>
__global__ void __launch_bounds__(kRowThreads) k_cache_read(const KvDev c, const int64_t* __restrict__ slots,
                                                           uint32_t rows, HeadDiv div, Lanes lanes, T* __restrict__ k,
                                                           T* __restrict__ v) {
  const Lane me = lane_of(lanes);
  const uint32_t r0 = (blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * static_cast<uint32_t>(U * lanes.rows) + me.row;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  if (!me.has_row) return;
  RowId id[U];
  bool live[U];
  uint4 raw[U][2];
  float2 sc[U];
  int64_t slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = r0 + u * lanes.rows;
    live[u] = r < 2 * rows;
    id[u] = row_id(live[u] ? r : 0u, rows, static_cast<uint32_t>(c.kv_heads), div);
    slot[u] = live[u] ? __ldg(slots + id[u].token) : -1;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= total && me.sub == 0) set_device_error(kDevBadCachePos);
    raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
    sc[u] = make_float2(0.f, 0.f);
    if (slot[u] >= 0 && slot[u] < total) {
      const uint32_t at = static_cast<uint32_t>(slot[u]);
      const uint8_t* src = (id[u].v ? c.v : c.k) + slot_row(c, at, id[u].head) + me.sub * BITS;
      raw[u][0] = get_codes<BITS>(src);
      raw[u][1] = get_codes<BITS>(src + lanes.g * BITS);
      if constexpr (BITS != 16) {
        const float* s = (id[u].v ? c.v_scale : c.k_scale) + slot_scale(c, at, id[u].head);
        if constexpr (BITS == 8) sc[u].x = *s;
        else sc[u] = *reinterpret_cast<const float2*>(s);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!live[u]) continue;
    uint4 out[2] = {raw[u][0], raw[u][1]};
    if constexpr (BITS != 16) {
      out[0] = decode<T, BITS>(raw[u][0], sc[u].x, sc[u].y);
      out[1] = decode<T, BITS>(raw[u][1], sc[u].x, sc[u].y);
    }
    T* dst = (id[u].v ? v : k) + (static_cast<int64_t>(id[u].token) * c.kv_heads + id[u].head) * c.head_dim + me.sub * 8;
    __stcs(reinterpret_cast<uint4*>(dst), out[0]);
    __stcs(reinterpret_cast<uint4*>(dst + lanes.g * 8), out[1]);
  }
}

struct WriteCall {
  KvDev c;
  const void *k, *v;
  int64_t k_ts, k_hs, v_ts, v_hs;
  const int64_t* slots;
  int tokens;
};

// Rows a group: two once that still gives every SM its blocks, else one. (50,001 tokens of 8
// heads x 80: 81 us with two, 87 with one, 106 with four.)
constexpr int kMoreRows = 2;
unsigned row_blocks(int64_t rows, const Lanes& l, int u) {
  const int64_t each = static_cast<int64_t>(kRowWarps) * l.rows * u;
  return static_cast<unsigned>((rows + each - 1) / each);
}
bool takes_more(int64_t rows, const Lanes& l) { return row_blocks(rows, l, kMoreRows) >= 8u * static_cast<unsigned>(device_sm_count()); }

template <typename T, int BITS, int U>
cudaError_t write_u(const WriteCall& a, const Lanes& l, cudaStream_t s) {
  const uint32_t rows = static_cast<uint32_t>(a.tokens) * static_cast<uint32_t>(a.c.kv_heads);
  return launch_dep(k_cache_write<T, BITS, U>, dim3(row_blocks(2 * static_cast<int64_t>(rows), l, U)), dim3(kRowThreads), 0,
                    s, a.c, static_cast<const T*>(a.k), static_cast<const T*>(a.v), a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.slots,
                    rows, head_div(a.c.kv_heads), l);
}
template <typename T, int BITS, int U>
cudaError_t read_u(const KvDev& c, const int64_t* slots, int tokens, void* k, void* v, const Lanes& l, cudaStream_t s) {
  const uint32_t rows = static_cast<uint32_t>(tokens) * static_cast<uint32_t>(c.kv_heads);
  return launch_dep(k_cache_read<T, BITS, U>, dim3(row_blocks(2 * static_cast<int64_t>(rows), l, U)), dim3(kRowThreads), 0, s,
                    c, slots, rows, head_div(c.kv_heads), l, static_cast<T*>(k), static_cast<T*>(v));
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
  const Lanes l = lanes_of(c.head_dim);
  const bool more = takes_more(2 * static_cast<int64_t>(tokens) * c.kv_heads, l);
  return with_form(bf16, bits, [&](auto t, auto b) {
    using T = decltype(t);
    constexpr int kBits = decltype(b)::value;
    return more ? write_u<T, kBits, kMoreRows>(a, l, s) : write_u<T, kBits, 1>(a, l, s);
  });
}

cudaError_t launch_cache_read(const KvDev& c, int bits, bool bf16, const int64_t* slots, int tokens, void* k, void* v,
                              cudaStream_t s) {
  const Lanes l = lanes_of(c.head_dim);
  const bool more = takes_more(2 * static_cast<int64_t>(tokens) * c.kv_heads, l);
  return with_form(bf16, bits, [&](auto t, auto b) {
    using T = decltype(t);
    constexpr int kBits = decltype(b)::value;
    return more ? read_u<T, kBits, kMoreRows>(c, slots, tokens, k, v, l, s) : read_u<T, kBits, 1>(c, slots, tokens, k, v, l, s);
  });
}

}  // namespace gemq
