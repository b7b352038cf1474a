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

// One group of GL lanes a row, eight elements a lane.
template <typename T, int BITS, int GL>
__global__ void __launch_bounds__(kRowThreads) k_cache_write(const KvDev c, const T* __restrict__ k,
                                                            const T* __restrict__ v, int64_t k_ts, int64_t k_hs,
                                                            int64_t v_ts, int64_t v_hs,
                                                            const int64_t* __restrict__ slots, int tokens) {
  const int64_t rows = static_cast<int64_t>(tokens) * c.kv_heads;
  const int sub = threadIdx.x % GL;
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) / GL;
  grid_dep_wait();
  const bool live = r < 2 * rows;
  const RowId id = row_id(live ? r : 0, rows, c.kv_heads);
  const int64_t slot = live ? slots[id.token] : -1;
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  if (slot >= total && sub == 0) set_device_error(kDevBadCachePos);
  const bool put = slot >= 0 && slot < total;
  const bool mine = put && sub * 8 < c.head_dim;
  const T* src = (id.kv ? v : k) + id.token * (id.kv ? v_ts : k_ts) + id.head * (id.kv ? v_hs : k_hs) + sub * 8;
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (mine) raw = *reinterpret_cast<const uint4*>(src);
  const int page = static_cast<int>(slot >> c.page_shift);
  const int off = static_cast<int>(slot & ((int64_t(1) << c.page_shift) - 1));
  uint8_t* dst = (id.kv ? c.v : c.k) + (put ? c.row(page, id.head, off) : 0);
  if constexpr (BITS == 16) {
    if (mine) *reinterpret_cast<uint4*>(dst + sub * 16) = raw;
    return;
  }
  float x[8];
  {
    const float2 a = unpack2<T>(raw.x), b = unpack2<T>(raw.y), d = unpack2<T>(raw.z), e = unpack2<T>(raw.w);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = d.x; x[5] = d.y; x[6] = e.x; x[7] = e.y;
  }
  float lo = mine ? x[0] : INFINITY, hi = mine ? x[0] : -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bad |= !isfinite(x[i]);
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
  const bool any_bad = (__ballot_sync(0xffffffffu, bad) & group) != 0;
  constexpr float kTop = BITS == 8 ? 127.f : 15.f;
  const float base = BITS == 8 ? 0.f : lo;
  const float range = fmaxf(BITS == 8 ? fmaxf(fabsf(lo), fabsf(hi)) : hi - lo, kTop * kMinScale);
  const bool poison = any_bad || !isfinite(range * kTop);
  if (!mine) return;
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    q[i] = poison ? 0u : static_cast<uint32_t>(__float2int_rn(__fdiv_rn((x[i] - base) * kTop, range)));
  if constexpr (BITS == 8) {
    uint2 w;
    w.x = (q[0] & 255u) | (q[1] & 255u) << 8 | (q[2] & 255u) << 16 | q[3] << 24;
    w.y = (q[4] & 255u) | (q[5] & 255u) << 8 | (q[6] & 255u) << 16 | q[7] << 24;
    *reinterpret_cast<uint2*>(dst + sub * 8) = w;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (q[i] & 15u) << (4 * i);
    *reinterpret_cast<uint32_t*>(dst + sub * 4) = w;
  }
  if (sub == 0) {
    float* s = (id.kv ? c.v_scale : c.k_scale) + c.scale_row(page, id.head, off);
    s[0] = poison ? NAN : __fdiv_rn(range, kTop);
    if constexpr (BITS == 4) s[1] = poison ? NAN : lo;
  }
}

// The mirror: out [tokens, heads, D] of T, one rounding. A negative slot reads zeros.
template <typename T, int BITS, int GL>
__global__ void __launch_bounds__(kRowThreads) k_cache_read(const KvDev c, const int64_t* __restrict__ slots,
                                                           int tokens, T* __restrict__ k, T* __restrict__ v) {
  const int64_t rows = static_cast<int64_t>(tokens) * c.kv_heads;
  const int sub = threadIdx.x % GL;
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) / GL;
  grid_dep_wait();
  if (r >= 2 * rows || sub * 8 >= c.head_dim) return;
  const RowId id = row_id(r, rows, c.kv_heads);
  const int64_t slot = slots[id.token];
  const int64_t total = static_cast<int64_t>(c.num_pages) << c.page_shift;
  if (slot >= total && sub == 0) set_device_error(kDevBadCachePos);
  uint4 out = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < total) {
    const int page = static_cast<int>(slot >> c.page_shift);
    const int off = static_cast<int>(slot & ((int64_t(1) << c.page_shift) - 1));
    const uint8_t* src = (id.kv ? c.v : c.k) + c.row(page, id.head, off);
    if constexpr (BITS == 16) {
      out = *reinterpret_cast<const uint4*>(src + sub * 16);
    } else {
      const float* s = (id.kv ? c.v_scale : c.k_scale) + c.scale_row(page, id.head, off);
      const float step = s[0];
      float x[8];
      if constexpr (BITS == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(src + sub * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * step;
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(src + sub * 4);
        const float base = s[1];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>((w >> (4 * i)) & 15u), step, base);
      }
      out = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
  }
  T* dst = (id.kv ? v : k) + (static_cast<int64_t>(id.token) * c.kv_heads + id.head) * c.head_dim + sub * 8;
  *reinterpret_cast<uint4*>(dst) = out;
}

struct WriteCall {
  KvDev c;
  const void *k, *v;
  int64_t k_ts, k_hs, v_ts, v_hs;
  const int64_t* slots;
  int tokens;
};

unsigned row_blocks(const KvDev& c, int tokens, int gl) {
  const int64_t threads = 2 * static_cast<int64_t>(tokens) * c.kv_heads * gl;
  return static_cast<unsigned>((threads + kRowThreads - 1) / kRowThreads);
}

template <typename T, int BITS, int GL>
cudaError_t write_gl(const WriteCall& a, cudaStream_t s) {
  return launch_dep(k_cache_write<T, BITS, GL>, dim3(row_blocks(a.c, a.tokens, GL)), dim3(kRowThreads), 0, s, a.c,
                    static_cast<const T*>(a.k), static_cast<const T*>(a.v), a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.slots,
                    a.tokens);
}
template <typename T, int BITS, int GL>
cudaError_t read_gl(const KvDev& c, const int64_t* slots, int tokens, void* k, void* v, cudaStream_t s) {
  return launch_dep(k_cache_read<T, BITS, GL>, dim3(row_blocks(c, tokens, GL)), dim3(kRowThreads), 0, s, c, slots,
                    tokens, static_cast<T*>(k), static_cast<T*>(v));
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
