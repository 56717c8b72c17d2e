// The quantised KV cache: writing rows (optionally picked by an index, so that
// a compression step's kept rows go straight into it) and reading them back.
//
//   lo, hi = a group's least and greatest value within +-61440
//   z = f16(lo)   s = f16((hi - lo) c)   i = 1 / s (0 where s = 0)
//   n = rint((x - z) i) kept in 0..N,    c = f32(1 / N), N = 15 or 255
//
// Every step is one correctly rounded f32 operation, so the codes are the same
// on any machine.  A NaN in a group makes its scale and zero NaN: the group
// reads back as NaN.
//
// Both kernels move each byte once, eight lanes a row, a block 16 rows of one KV
// head (no division a row).  Writing: a lane has 16 channels of K and 16 of V in
// flight, group extrema come from shuffles (16-bit types: least and minus greatest
// in one register), the codes from shifted sums of the floats' bit patterns, the
// clamp only for groups that need it.  It is bound by the instructions it issues
// (460 for 16 channels of K and V a lane, 84% of the issue slots) close to the
// memory's time: 16384 tokens of 8 heads in bf16 16.3 us (5.3 TB/s), 8 x 32768 242
// us (5.8 TB/s).  From f32, eight blocks an SM, it is bound by memory: 16384 tokens 24.4
// us (6.3 TB/s).  So is reading back: 8 x 32768 tokens 213 us (6.6 TB/s), 16384 tokens
// 15.0 us.  Blocks of 128 threads, twelve an SM, gave 5% over
// blocks of 256.
#include <cuda_bf16.h>

#include <climits>

#include "common.cuh"
#include "host_util.h"
#include "kvq_common.cuh"

namespace core {
namespace kvq {

struct Cache {
  uint8_t* codes[2];   // K, V
  uint32_t* meta[2];
  int B, H, cap;
};

struct WriteParams {
  Cache c;
  const void* src[2];
  long long sb[2], sh[2], sl[2];  // element strides of (B, H, L)
  int L, T;
  const int* index;   // (B, T) source rows, or null
  const int* start;   // (B) first slots, or null
  const int* counts;  // (B) rows to write of the T, or null
  int start0;
  DeviceStatus* status;
};

struct ReadParams {
  Cache c;
  void* dst[2];
  int T;
  const int* index;  // (B, T) slots, or null
  const int* start;
  int start0;
  DeviceStatus* status;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Eight neighbouring channels as f32.
template <typename T>
struct Piece {
  uint4 v[sizeof(T) * 8 / 16];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const;
};
template <>
__device__ __forceinline__ void Piece<float>::get(float (&x)[8]) const {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __uint_as_float(v[i].x);
    x[4 * i + 1] = __uint_as_float(v[i].y);
    x[4 * i + 2] = __uint_as_float(v[i].z);
    x[4 * i + 3] = __uint_as_float(v[i].w);
  }
}
template <>
__device__ __forceinline__ void Piece<__nv_bfloat16>::get(float (&x)[8]) const {
  const uint32_t u[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void Piece<__half>::get(float (&x)[8]) const {
  const uint32_t u[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(as_half2(u[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// A group's scale and zero (the word of both as it is stored), and what its
// codes are computed with.
struct Grid {
  float z, inv;
  uint32_t word;
  bool plain;  // none of the group's channels needs a clamp
};

template <int kBits>
__device__ __forceinline__ Grid grid_of(float lo, float hi) {
  constexpr float c = kBits == 4 ? 1.0f / 15.0f : 1.0f / 255.0f, top = kBits == 4 ? 15.f : 255.f;
  const float lo0 = lo, hi0 = hi;
  lo = max_nan(min_nan(lo, kLimit), -kLimit);
  hi = max_nan(min_nan(hi, kLimit), -kLimit);
  const __half2 sz = __floats2half2_rn(__fmul_rn(__fsub_rn(hi, lo), c), lo);
  const float2 f = __half22float2(sz);
  Grid g;
  g.z = f.y;
  g.inv = f.x > 0.f ? __frcp_rn(f.x) : 0.f;
  g.word = as_u32(sz);
  // the extrema fall on codes 0 .. N, and neither was saturated (NaN: false)
  const float first = __fmul_rn(__fsub_rn(lo, g.z), g.inv), last = __fmul_rn(__fsub_rn(hi, g.z), g.inv);
  g.plain = lo == lo0 && hi == hi0 && first >= -0.5f && last < top + 0.5f;
  return g;
}

// Eight codes of kBits each from floats 1.5 2^23 + n: the integer lies in the low
// bits, so shifted sums of the bit patterns give the word once the patterns of
// 1.5 2^23 are taken off again (modulo 2^32).
template <int kBits>
__device__ __forceinline__ void pack_codes(const float (&r)[8], uint32_t* w) {
  constexpr uint32_t m = 0x4B400000u;  // the bits of 1.5 2^23
  if constexpr (kBits == 4) {
    constexpr int at[8] = {0, 16, 4, 20, 8, 24, 12, 28};
    constexpr uint32_t off = m + (m << 4) + (m << 8) + (m << 12) + (m << 16) + (m << 20) + (m << 24) + (m << 28);
    uint32_t x = 0u - off;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += __float_as_uint(r[i]) << at[i];
    w[0] = x;
  } else {
    constexpr int at[4] = {0, 16, 8, 24};
    constexpr uint32_t off = m + (m << 8) + (m << 16) + (m << 24);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t x = 0u - off;
#pragma unroll
      for (int i = 0; i < 4; ++i) x += __float_as_uint(r[4 * h + i]) << at[i];
      w[h] = x;
    }
  }
}

// Codes of a lane's sixteen channels: two words (4 bits) or four (8 bits).
template <typename T, int kBits>
__device__ __forceinline__ void encode(const Piece<T>& p0, const Piece<T>& p1, const Grid& g, uint32_t (&w)[kBits / 2]) {
  constexpr float top = kBits == 4 ? 15.f : 255.f;
  constexpr float magic = 12582912.f;  // 1.5 2^23: adding it rounds to the nearest integer, ties to even
  float x[2][8], r[2][8];
  p0.get(x[0]);
  p1.get(x[1]);
  if (g.plain) {
    const unsigned long long nz = f2_pack(-g.z, -g.z), mg = f2_pack(magic, magic);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        // the product is one scalar multiplication a channel: the assembler joins a
        // packed one with the addition into an fma, whose single rounding moves ties
        const unsigned long long d = f2_add(f2_pack(x[h][i], x[h][i + 1]), nz);
        const unsigned long long y = f2_add(f2_pack(__fmul_rn(f2_lo(d), g.inv), __fmul_rn(f2_hi(d), g.inv)), mg);
        r[h][i] = f2_lo(y);
        r[h][i + 1] = f2_hi(y);
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = fmaxf(fminf(x[h][i], kLimit), -kLimit);  // NaN: any code, its scale is NaN
        r[h][i] = __fadd_rn(fminf(fmaxf(__fmul_rn(__fsub_rn(v, g.z), g.inv), 0.f), top), magic);
      }
    }
  }
  pack_codes<kBits>(r[0], w);
  pack_codes<kBits>(r[1], w + kBits / 4);
}

// Extrema of 16 channels (or of 8), as a (least, greatest) pair that NaN passes
// through: f32, or both as the halves of one register, which the shuffles then
// move at once.
template <typename T>
struct Extrema;
template <>
struct Extrema<float> {
  float lo, hi;
  __device__ __forceinline__ void of(const Piece<float>& p) {
    float x[8];
    p.get(x);
    lo = hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, x[i]);
      hi = max_nan(hi, x[i]);
    }
  }
  __device__ __forceinline__ void with(const Extrema& o) {
    lo = min_nan(lo, o.lo);
    hi = max_nan(hi, o.hi);
  }
  __device__ __forceinline__ void close() {}
  __device__ __forceinline__ void across(int bit) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, bit));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, bit));
  }
  __device__ __forceinline__ float least() const { return lo; }
  __device__ __forceinline__ float greatest() const { return hi; }
};
template <typename T2>
__device__ __forceinline__ T2 pair_of(uint32_t u) {
  return *reinterpret_cast<T2*>(&u);
}
template <typename T, typename T2>
struct Extrema16 {
  T2 lo, hi;  // of even and odd channels; after close(): lo = (least, -greatest)
  __device__ __forceinline__ void of(const Piece<T>& p) {
    const uint32_t u[4] = {p.v[0].x, p.v[0].y, p.v[0].z, p.v[0].w};
    lo = hi = pair_of<T2>(u[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      lo = __hmin2_nan(lo, pair_of<T2>(u[i]));
      hi = __hmax2_nan(hi, pair_of<T2>(u[i]));
    }
  }
  __device__ __forceinline__ void with(const Extrema16& o) {
    lo = __hmin2_nan(lo, o.lo);
    hi = __hmax2_nan(hi, o.hi);
  }
  __device__ __forceinline__ void close() {
    const T2 n = __hneg2(hi);
    // (lo.x, -hi.x) and (lo.y, -hi.y): one minimum leaves (least, -greatest)
    lo = __hmin2_nan(__halves2(__low2(lo), __low2(n)), __halves2(__high2(lo), __high2(n)));
  }
  __device__ __forceinline__ void across(int bit) { lo = __hmin2_nan(lo, __shfl_xor_sync(0xffffffffu, lo, bit)); }
  __device__ __forceinline__ float least() const { return to_float(__low2(lo)); }
  __device__ __forceinline__ float greatest() const { return -to_float(__high2(lo)); }
  static __device__ __forceinline__ __half2 __halves2(__half a, __half b) { return __halves2half2(a, b); }
  static __device__ __forceinline__ __nv_bfloat162 __halves2(__nv_bfloat16 a, __nv_bfloat16 b) {
    return __halves2bfloat162(a, b);
  }
  static __device__ __forceinline__ __half __low2(__half2 a) { return __low2half(a); }
  static __device__ __forceinline__ __half __high2(__half2 a) { return __high2half(a); }
  static __device__ __forceinline__ __nv_bfloat16 __low2(__nv_bfloat162 a) { return __low2bfloat16(a); }
  static __device__ __forceinline__ __nv_bfloat16 __high2(__nv_bfloat162 a) { return __high2bfloat16(a); }
  static __device__ __forceinline__ float to_float(__half a) { return __half2float(a); }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 a) { return __bfloat162float(a); }
};
template <>
struct Extrema<__half> : Extrema16<__half, __half2> {};
template <>
struct Extrema<__nv_bfloat16> : Extrema16<__nv_bfloat16, __nv_bfloat162> {};

constexpr int kThreads = 128;
constexpr int kRows = kThreads / 8;  // rows of a block: eight lanes each

// Lane m of a row's eight holds channels 16 m .. 16 m + 15.
template <typename T, int kBits, int kG>
__device__ __forceinline__ void write_row(const Piece<T>& p0, const Piece<T>& p1, bool keys, int m, uint32_t tok,
                                          bool live, uint8_t* codes, uint32_t* meta) {
  Extrema<T> e, e1;
  e.of(p0);
  e1.of(p1);
  e.with(e1);
  e.close();
  e.across(1);
  if (kG <= 2) e.across(2);
  if (kG == 1) e.across(4);
  const Grid g = grid_of<kBits>(e.least(), e.greatest());
  uint32_t w[kBits / 2];
  encode<T, kBits>(p0, p1, g, w);
  if (!live) return;
  if (keys) {
    // channels 32 b + 8 t .. with b = m / 2 and t = 2 (m & 1), then t + 1
    if constexpr (kBits == 4) {
      uint32_t* to = reinterpret_cast<uint32_t*>(codes) + 8 * (m & 1) + (m >> 1);
      to[0] = w[0];
      to[4] = w[1];
    } else {
      const uint32_t at = (64u * (m >> 2) + 32u * (m & 1) + 8u * ((m >> 1) & 1)) ^ key_swizzle<8>(tok);
      *reinterpret_cast<uint2*>(codes + at) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(codes + at + 16) = make_uint2(w[2], w[3]);
    }
  } else {
    if constexpr (kBits == 4)
      *reinterpret_cast<uint2*>(codes + ((8u * m) ^ value_swizzle<4>(tok))) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4*>(codes + ((16u * m) ^ value_swizzle<8>(tok))) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if ((m & (8 / kG - 1)) == 0) meta[m / (8 / kG)] = g.word;
}

template <typename T, int kBits, int kG>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 8 : 12) quantize_kernel(const WriteParams p) {
  const int m = threadIdx.x & 7;
  const unsigned chunks = ((unsigned)p.T + kRows - 1) / kRows, units = (unsigned)(p.c.B * p.c.H) * chunks;
  // whole warps stay in the loop: the shuffles need every lane of a row
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    const int bh = (int)(u / chunks), t = (int)(u - (unsigned)bh * chunks) * kRows + (int)(threadIdx.x >> 3);
    const int b = bh / p.c.H, h = bh - b * p.c.H;
    int n = p.T;
    if (p.counts != nullptr) n = min(n, p.counts[b]);
    bool live = t < n;
    const long long slot = (long long)(p.start != nullptr ? p.start[b] : p.start0) + t;
    int src = t;
    if (live && p.index != nullptr) src = p.index[(long long)b * p.T + t];
    if (live && (slot < 0 || slot >= p.c.cap || src < 0 || src >= p.L)) {
      if (m == 0) record_error(p.status, CORE_ERR_INVALID_ARG, slot < 0 || slot >= p.c.cap ? 1401 : 1402, t);
      live = false;
    }
    Piece<T> k0{}, k1{}, v0{}, v1{};
    if (live) {
      const T* k = static_cast<const T*>(p.src[0]) + b * p.sb[0] + h * p.sh[0] + src * p.sl[0] + 16 * m;
      const T* v = static_cast<const T*>(p.src[1]) + b * p.sb[1] + h * p.sh[1] + src * p.sl[1] + 16 * m;
      k0.load(k);
      k1.load(k + 8);
      v0.load(v);
      v1.load(v + 8);
    }
    const long long row = (long long)bh * p.c.cap + slot;
    write_row<T, kBits, kG>(k0, k1, true, m, (uint32_t)slot, live, p.c.codes[0] + row * (16 * kBits),
                            p.c.meta[0] + row * kG);
    write_row<T, kBits, kG>(v0, v1, false, m, (uint32_t)slot, live, p.c.codes[1] + row * (16 * kBits),
                            p.c.meta[1] + row * kG);
  }
}

// Eight channels in the output type; `apart`: how far the pieces of an even and
// the next odd lane lie from one another.  f32 pieces of two lanes are exchanged
// by halves, so that each store covers whole 32-byte sectors (16384 tokens read
// back as f32: 38 -> 26 us).
__device__ __forceinline__ void store8(float* o, const float (&x)[8], int apart) {
  const int lane = threadIdx.x & 31;
  const uint32_t row = 0xffu << (lane & 24);  // the lanes of a row go the same way
  const bool odd = lane & 1;
  float own[4], other[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    own[i] = odd ? x[4 + i] : x[i];
    other[i] = __shfl_xor_sync(row, odd ? x[i] : x[4 + i], 1);
  }
  float* first = odd ? o - apart + 4 : o;   // of the even lane's piece
  float* second = odd ? o + 4 : o + apart;  // of the odd lane's piece
  const float4 a = make_float4(own[0], own[1], own[2], own[3]), b = make_float4(other[0], other[1], other[2], other[3]);
  *reinterpret_cast<float4*>(first) = odd ? b : a;
  *reinterpret_cast<float4*>(second) = odd ? a : b;
}
__device__ __forceinline__ void store8(__nv_bfloat16* o, const float (&x)[8], int) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(__half* o, const float (&x)[8], int) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = as_u32(__floats2half2_rn(x[2 * i], x[2 * i + 1]));
  *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
}

template <typename T, int kBits>
__device__ __forceinline__ void decode_store(const uint32_t* w, uint32_t meta, T* o, int apart) {
  const float2 sz = __half22float2(as_half2(meta));
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 n = __half22float2(kBits == 4 ? code_pair<4>(w[0], i) : code_pair<8>(w[i >> 1], i & 1));
    x[2 * i] = __fmaf_rn(n.x, sz.x, sz.y);
    x[2 * i + 1] = __fmaf_rn(n.y, sz.x, sz.y);
  }
  store8(o, x, apart);
}

template <typename T, int kBits, int kG>
__global__ void __launch_bounds__(kThreads, 12) dequantize_kernel(const ReadParams p) {
  const int m = threadIdx.x & 7, a = m >> 2, q = m & 3;
  const unsigned chunks = ((unsigned)p.T + kRows - 1) / kRows, units = (unsigned)(p.c.B * p.c.H) * chunks;
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    const int bh = (int)(u / chunks), t = (int)(u - (unsigned)bh * chunks) * kRows + (int)(threadIdx.x >> 3);
    if (t >= p.T) continue;
    const int b = bh / p.c.H;
    long long slot;
    if (p.index != nullptr)
      slot = p.index[(long long)b * p.T + t];
    else
      slot = (long long)(p.start != nullptr ? p.start[b] : p.start0) + t;
    const long long to = ((long long)bh * p.T + t) * kD;
    // K: lane m = 4 a + q decodes channels 64 a + 8 q and 64 a + 32 + 8 q; V: 16 m
    T* ok = static_cast<T*>(p.dst[0]) + to + 64 * a + 8 * q;
    T* ov = static_cast<T*>(p.dst[1]) + to + 16 * m;
    if (slot < 0 || slot >= p.c.cap) {
      if (m == 0) record_error(p.status, CORE_ERR_INVALID_ARG, 1411, t);
      const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      store8(ok, zero, 8);
      store8(ok + 32, zero, 8);
      store8(ov, zero, 16);
      store8(ov + 8, zero, 16);
      continue;
    }
    const long long row = (long long)bh * p.c.cap + slot;
    const uint8_t* kc = p.c.codes[0] + row * (16 * kBits);
    const uint8_t* vc = p.c.codes[1] + row * (16 * kBits);
    const uint32_t* km = p.c.meta[0] + row * kG;
    const uint32_t* vm = p.c.meta[1] + row * kG;
    uint32_t kw[kBits / 2], vw[kBits / 2];
    if constexpr (kBits == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(kc + 16 * q + 8 * a);
      const uint2 y = *reinterpret_cast<const uint2*>(vc + ((8u * m) ^ value_swizzle<4>((uint32_t)slot)));
      kw[0] = x.x; kw[1] = x.y;
      vw[0] = y.x; vw[1] = y.y;
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(kc + ((16u * m) ^ key_swizzle<8>((uint32_t)slot)));
      const uint4 y = *reinterpret_cast<const uint4*>(vc + ((16u * m) ^ value_swizzle<8>((uint32_t)slot)));
      kw[0] = x.x; kw[1] = x.y; kw[2] = x.z; kw[3] = x.w;
      vw[0] = y.x; vw[1] = y.y; vw[2] = y.z; vw[3] = y.w;
    }
    const uint32_t k0 = km[kG == 4 ? 2 * a : kG == 2 ? a : 0], k1 = kG == 4 ? km[2 * a + 1] : k0;
    const uint32_t v0 = vm[kG == 4 ? m >> 1 : kG == 2 ? a : 0];
    decode_store<T, kBits>(kw, k0, ok, 8);
    decode_store<T, kBits>(kw + kBits / 4, k1, ok + 32, 8);
    decode_store<T, kBits>(vw, v0, ov, 16);
    decode_store<T, kBits>(vw + kBits / 4, v0, ov + 8, 16);
  }
}

}  // namespace kvq

int check_kvq(const core_kvq_t* c, const char* fn) {
  const std::string f(fn);
  if (c == nullptr || c->k_codes == nullptr || c->k_meta == nullptr || c->v_codes == nullptr || c->v_meta == nullptr)
    return set_error(CORE_ERR_INVALID_ARG, f + ": NULL cache buffer");
  if (c->batch <= 0 || c->n_kv_heads <= 0 || c->capacity <= 0)
    return set_error(CORE_ERR_INVALID_ARG, f + ": non-positive cache dimension");
  if ((int64_t)c->batch * c->n_kv_heads > INT_MAX)
    return set_error(CORE_ERR_UNSUPPORTED, f + ": batch x n_kv_heads does not fit 31 bits");
  if (c->capacity % 128 != 0 || c->capacity > INT_MAX - 256)
    return set_error(CORE_ERR_INVALID_ARG, f + ": capacity must be a multiple of 128 below 2^31");
  if (c->bits != 4 && c->bits != 8) return set_error(CORE_ERR_UNSUPPORTED, f + ": bits must be 4 or 8");
  if (c->group != 32 && c->group != 64 && c->group != 128)
    return set_error(CORE_ERR_UNSUPPORTED, f + ": group must be 32, 64 or 128");
  if (!aligned16(c->k_codes) || !aligned16(c->k_meta) || !aligned16(c->v_codes) || !aligned16(c->v_meta))
    return set_error(CORE_ERR_INVALID_ARG, f + ": cache buffers must be 16-byte aligned");
  return CORE_OK;
}

}  // namespace core

using namespace core;

namespace {

kvq::Cache device_cache(const core_kvq_t* c) {
  kvq::Cache d;
  d.codes[0] = static_cast<uint8_t*>(c->k_codes);
  d.codes[1] = static_cast<uint8_t*>(c->v_codes);
  d.meta[0] = static_cast<uint32_t*>(c->k_meta);
  d.meta[1] = static_cast<uint32_t*>(c->v_meta);
  d.B = c->batch;
  d.H = c->n_kv_heads;
  d.cap = c->capacity;
  return d;
}

// Units of kRows rows of one KV head, one block each.
long long row_units(const core_kvq_t* c, int n_rows) {
  return (long long)c->batch * c->n_kv_heads * ((n_rows + kvq::kRows - 1) / kvq::kRows);
}

template <template <typename, int, int> class F, typename T, typename... A>
void by_format(int bits, int group, A&&... a) {
  if (bits == 4) {
    if (group == 32) F<T, 4, 4>::run(a...);
    else if (group == 64) F<T, 4, 2>::run(a...);
    else F<T, 4, 1>::run(a...);
  } else {
    if (group == 32) F<T, 8, 4>::run(a...);
    else if (group == 64) F<T, 8, 2>::run(a...);
    else F<T, 8, 1>::run(a...);
  }
}

template <template <typename, int, int> class F, typename... A>
bool by_type(int dtype, int bits, int group, A&&... a) {
  if (dtype == CORE_DTYPE_BF16) by_format<F, __nv_bfloat16>(bits, group, a...);
  else if (dtype == CORE_DTYPE_F16) by_format<F, __half>(bits, group, a...);
  else if (dtype == CORE_DTYPE_F32) by_format<F, float>(bits, group, a...);
  else return false;
  return true;
}

template <typename T, int kBits, int kG>
struct Write {
  static void run(int blocks, cudaStream_t s, const kvq::WriteParams& p) {
    kvq::quantize_kernel<T, kBits, kG><<<blocks, kvq::kThreads, 0, s>>>(p);
  }
};
template <typename T, int kBits, int kG>
struct Read {
  static void run(int blocks, cudaStream_t s, const kvq::ReadParams& p) {
    kvq::dequantize_kernel<T, kBits, kG><<<blocks, kvq::kThreads, 0, s>>>(p);
  }
};

}  // namespace

extern "C" int core_kvq_quantize(const core_kvq_t* cache, int32_t dtype, const void* k, const int64_t* k_strides,
                                 const void* v, const int64_t* v_strides, int32_t src_len, int32_t n_rows,
                                 const int32_t* index, const int32_t* start, int32_t start_all,
                                 const int32_t* counts, void* stream) {
  const char* fn = "core_kvq_quantize";
  int rc = check_kvq(cache, fn);
  if (rc != CORE_OK) return rc;
  const std::string f(fn);
  if (k == nullptr || v == nullptr || k_strides == nullptr || v_strides == nullptr)
    return set_error(CORE_ERR_INVALID_ARG, f + ": NULL argument");
  if (src_len <= 0 || n_rows <= 0 || n_rows > INT_MAX - 256 || (index == nullptr && n_rows > src_len))
    return set_error(CORE_ERR_INVALID_ARG, f + ": bad row count");
  if (start == nullptr && (start_all < 0 || (int64_t)start_all + n_rows > cache->capacity))
    return set_error(CORE_ERR_INVALID_ARG, f + ": rows outside the cache's capacity");
  const int size = dtype == CORE_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    if ((k_strides[i] * size) % 16 != 0 || (v_strides[i] * size) % 16 != 0)
      return set_error(CORE_ERR_INVALID_ARG, f + ": strides must be multiples of 16 bytes");
  if (!aligned16(k) || !aligned16(v)) return set_error(CORE_ERR_INVALID_ARG, f + ": rows must be 16-byte aligned");
  kvq::WriteParams p{};
  p.c = device_cache(cache);
  p.src[0] = k;
  p.src[1] = v;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? v_strides : k_strides;
    p.sb[i] = st[0];
    p.sh[i] = st[1];
    p.sl[i] = st[2];
  }
  p.L = src_len;
  p.T = n_rows;
  p.index = index;
  p.start = start;
  p.counts = counts;
  p.start0 = start_all;
  p.status = device_status();
  const long long units = row_units(cache, n_rows);
  if (units > INT_MAX) return set_error(CORE_ERR_UNSUPPORTED, f + ": too many rows");
  const int blocks = (int)units;
  if (!by_type<Write>(dtype, cache->bits, cache->group, blocks, static_cast<cudaStream_t>(stream), p))
    return set_error(CORE_ERR_UNSUPPORTED, f + ": dtype must be bf16, f16 or f32");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CORE_OK : cuda_error(e, "quantize_kernel launch");
}

extern "C" int core_kvq_dequantize(const core_kvq_t* cache, int32_t dtype, int32_t n_rows, const int32_t* index,
                                   const int32_t* start, int32_t start_all, void* out_k, void* out_v, void* stream) {
  const char* fn = "core_kvq_dequantize";
  int rc = check_kvq(cache, fn);
  if (rc != CORE_OK) return rc;
  const std::string f(fn);
  if (out_k == nullptr || out_v == nullptr) return set_error(CORE_ERR_INVALID_ARG, f + ": NULL argument");
  if (n_rows <= 0 || n_rows > INT_MAX - 256) return set_error(CORE_ERR_INVALID_ARG, f + ": bad row count");
  if (index == nullptr && start == nullptr && (start_all < 0 || (int64_t)start_all + n_rows > cache->capacity))
    return set_error(CORE_ERR_INVALID_ARG, f + ": rows outside the cache's capacity");
  if (!aligned16(out_k) || !aligned16(out_v))
    return set_error(CORE_ERR_INVALID_ARG, f + ": outputs must be 16-byte aligned");
  kvq::ReadParams p{};
  p.c = device_cache(cache);
  p.dst[0] = out_k;
  p.dst[1] = out_v;
  p.T = n_rows;
  p.index = index;
  p.start = start;
  p.start0 = start_all;
  p.status = device_status();
  const long long units = row_units(cache, n_rows);
  if (units > INT_MAX) return set_error(CORE_ERR_UNSUPPORTED, f + ": too many rows");
  const int blocks = (int)units;
  if (!by_type<Read>(dtype, cache->bits, cache->group, blocks, static_cast<cudaStream_t>(stream), p))
    return set_error(CORE_ERR_UNSUPPORTED, f + ": dtype must be bf16, f16 or f32");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CORE_OK : cuda_error(e, "dequantize_kernel launch");
}
