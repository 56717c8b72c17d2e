// The quantised KV cache: writing rows (optionally picked by an index, so that
// a compression step's kept rows go straight into it) and reading them back.
//
//   lo, hi = a group's least and greatest value within +-61440
//   z = f16(lo)   s = f16((hi - lo) c)   i = 1 / s (0 where s = 0)
//   n = rint((x - z) i) kept in 0..N,    c = f32(1 / N), N = 15 or 255
//
// Every step is one correctly rounded f32 operation, so the codes are the same
// on any machine.  A NaN in a group makes its scale and zero NaN: the group
// reads back as NaN.  Both kernels move each byte once: eight lanes take a row
// (16 channels of K and 16 of V each, loaded together), group extrema come from
// shuffles, and a row's codes leave as 8 or 16 bytes a lane.
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

struct Grid {  // a group's scale and zero, and what the codes are computed with
  float z, inv;
  uint32_t word;
};

template <int kBits>
__device__ __forceinline__ Grid make_grid(float lo, float hi) {
  constexpr float c = kBits == 4 ? 1.0f / 15.0f : 1.0f / 255.0f;
  lo = max_nan(min_nan(lo, kLimit), -kLimit);
  hi = max_nan(min_nan(hi, kLimit), -kLimit);
  const __half z = __float2half_rn(lo), s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), c));
  Grid g;
  g.z = __half2float(z);
  const float sf = __half2float(s);
  g.inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
  g.word = (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(z) << 16);
  return g;
}

// Codes of eight channels: one word (4 bits) or two (8 bits).  The extrema were
// saturated and the channels were not: a channel beyond the limit lands on the
// first or last code all the same, as the saturated one does, unless the whole
// group is (the saturated scale is then zero or tiny), so channels are clamped
// where an extremum was.
template <int kBits>
__device__ __forceinline__ void encode(const float (&x)[8], const Grid& g, bool clamp, uint32_t (&w)[kBits / 4]) {
  constexpr float top = kBits == 4 ? 15.f : 255.f;
  uint32_t n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = x[i];
    if (clamp) v = fmaxf(fminf(v, kLimit), -kLimit);
    const float y = fminf(fmaxf(__fmul_rn(__fsub_rn(v, g.z), g.inv), 0.f), top);
    // adding 1.5 2^23 rounds to the nearest integer (ties to even) in the low bits
    n[i] = __float_as_uint(__fadd_rn(y, 12582912.f)) & (kBits == 4 ? 15u : 255u);
  }
  if constexpr (kBits == 4) {
    w[0] = n[0] | n[2] << 4 | n[4] << 8 | n[6] << 12 | n[1] << 16 | n[3] << 20 | n[5] << 24 | n[7] << 28;
  } else {
    w[0] = n[0] | n[2] << 8 | n[1] << 16 | n[3] << 24;
    w[1] = n[4] | n[6] << 8 | n[5] << 16 | n[7] << 24;
  }
}

// kSteps-lane extrema of a group whose lanes differ in the given lane bits.
__device__ __forceinline__ void reduce(float& lo, float& hi, int bit) {
  lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, bit));
  hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, bit));
}
__device__ __forceinline__ void extrema(const float (&x)[8], float& lo, float& hi) {
  lo = hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
}

template <int kBits, int kG>
__device__ __forceinline__ void write_row(const float (&p0)[8], const float (&p1)[8], bool keys, int m,
                                          uint32_t tok, bool live, uint8_t* codes, uint32_t* meta) {
  // K: lane m = 4 a + t holds channels 64 a + 8 t and 64 a + 32 + 8 t;
  // V: channels 16 m and 16 m + 8
  float lo0, hi0, lo1, hi1;
  extrema(p0, lo0, hi0);
  extrema(p1, lo1, hi1);
  if (!(keys && kG == 4)) {  // both pieces in one group
    lo0 = min_nan(lo0, lo1);
    hi0 = max_nan(hi0, hi1);
  }
  reduce(lo0, hi0, 1);
  if (keys || kG <= 2) reduce(lo0, hi0, 2);
  if (kG == 1) reduce(lo0, hi0, 4);
  if (keys && kG == 4) {
    reduce(lo1, hi1, 1);
    reduce(lo1, hi1, 2);
  } else {
    lo1 = lo0;
    hi1 = hi0;
  }
  const Grid g0 = make_grid<kBits>(lo0, hi0);
  const Grid g1 = keys && kG == 4 ? make_grid<kBits>(lo1, hi1) : g0;
  const bool c0 = !(fabsf(lo0) <= kLimit && fabsf(hi0) <= kLimit);
  const bool c1 = !(fabsf(lo1) <= kLimit && fabsf(hi1) <= kLimit);
  uint32_t w0[kBits / 4], w1[kBits / 4];
  encode<kBits>(p0, g0, c0, w0);
  encode<kBits>(p1, g1, c1, w1);
  if (!live) return;
  const int a = m >> 2, t = m & 3;
  if constexpr (kBits == 4) {
    const uint32_t at = keys ? 16u * t + 8u * a : (8u * m) ^ value_swizzle<4>(tok);
    *reinterpret_cast<uint2*>(codes + at) = make_uint2(w0[0], w1[0]);
  } else {
    const uint32_t at = (16u * m) ^ (keys ? key_swizzle<8>(tok) : value_swizzle<8>(tok));
    *reinterpret_cast<uint4*>(codes + at) = make_uint4(w0[0], w0[1], w1[0], w1[1]);
  }
  if (keys) {
    if (kG == 4 && t == 0) *reinterpret_cast<uint2*>(meta + 2 * a) = make_uint2(g0.word, g1.word);
    if (kG == 2 && t == 0) meta[a] = g0.word;
  } else {
    if (kG == 4 && (m & 1) == 0) meta[m >> 1] = g0.word;
    if (kG == 2 && t == 0) meta[a] = g0.word;
  }
  if (kG == 1 && m == 0) meta[0] = g0.word;
}

constexpr int kThreads = 256;

template <typename T, int kBits, int kG>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const WriteParams p) {
  const long long total = (long long)p.c.B * p.c.H * p.T;
  const int m = threadIdx.x & 7;
  const long long step = (long long)gridDim.x * (kThreads / 8);
  // whole warps stay in the loop: the shuffles need every lane of a row
  for (long long r0 = (long long)blockIdx.x * (kThreads / 8); r0 < total; r0 += step) {
    const long long r = r0 + (threadIdx.x >> 3);
    bool live = r < total;
    int bh = 0, t = 0;
    if (live) {
      if (total <= UINT_MAX) {
        bh = (int)((unsigned)r / (unsigned)p.T);
        t = (int)((unsigned)r - (unsigned)bh * (unsigned)p.T);
      } else {
        bh = (int)(r / p.T);
        t = (int)(r - (long long)bh * p.T);
      }
    }
    const int b = bh / p.c.H, h = bh - b * p.c.H;
    if (live && p.counts != nullptr) live = t < p.counts[b];
    long long slot = 0;
    int src = t;
    if (live) {
      slot = (long long)(p.start != nullptr ? p.start[b] : p.start0) + t;
      if (p.index != nullptr) src = p.index[(long long)b * p.T + t];
      if (slot < 0 || slot >= p.c.cap || src < 0 || src >= p.L) {
        if (m == 0) record_error(p.status, CORE_ERR_INVALID_ARG, slot < 0 || slot >= p.c.cap ? 1401 : 1402, t);
        live = false;
      }
    }
    Piece<T> k0, k1, v0, v1;
    if (live) {
      const T* k = static_cast<const T*>(p.src[0]) + b * p.sb[0] + h * p.sh[0] + src * p.sl[0];
      const T* v = static_cast<const T*>(p.src[1]) + b * p.sb[1] + h * p.sh[1] + src * p.sl[1];
      const int at = 64 * (m >> 2) + 8 * (m & 3);
      k0.load(k + at);
      k1.load(k + at + 32);
      v0.load(v + 16 * m);
      v1.load(v + 16 * m + 8);
    } else {
      k0 = k1 = v0 = v1 = Piece<T>{};
    }
    const long long row = (long long)bh * p.c.cap + slot;
    float x[8], y[8];
    k0.get(x);
    k1.get(y);
    write_row<kBits, kG>(x, y, true, m, (uint32_t)slot, live, p.c.codes[0] + row * (16 * kBits), p.c.meta[0] + row * kG);
    v0.get(x);
    v1.get(y);
    write_row<kBits, kG>(x, y, false, m, (uint32_t)slot, live, p.c.codes[1] + row * (16 * kBits), p.c.meta[1] + row * kG);
  }
}

// Eight channels n s + z (one rounding in f32) in the output type.
__device__ __forceinline__ void store8(float* o, const float (&x)[8]) {
  reinterpret_cast<float4*>(o)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(o)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* o, const float (&x)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(__half* o, const float (&x)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = as_u32(__floats2half2_rn(x[2 * i], x[2 * i + 1]));
  *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
}

template <typename T, int kBits>
__device__ __forceinline__ void decode_store(const uint32_t* w, uint32_t meta, T* o) {
  const float2 sz = __half22float2(as_half2(meta));
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 n = __half22float2(kBits == 4 ? code_pair<4>(w[0], i) : code_pair<8>(w[i >> 1], i & 1));
    x[2 * i] = __fmaf_rn(n.x, sz.x, sz.y);
    x[2 * i + 1] = __fmaf_rn(n.y, sz.x, sz.y);
  }
  store8(o, x);
}

template <typename T, int kBits, int kG>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const ReadParams p) {
  const long long total = (long long)p.c.B * p.c.H * p.T;
  const int m = threadIdx.x & 7, a = m >> 2, q = m & 3;
  const long long step = (long long)gridDim.x * (kThreads / 8);
  for (long long r = (long long)blockIdx.x * (kThreads / 8) + (threadIdx.x >> 3); r < total; r += step) {
    int bh, t;
    if (total <= UINT_MAX) {
      bh = (int)((unsigned)r / (unsigned)p.T);
      t = (int)((unsigned)r - (unsigned)bh * (unsigned)p.T);
    } else {
      bh = (int)(r / p.T);
      t = (int)(r - (long long)bh * p.T);
    }
    const int b = bh / p.c.H;
    long long slot;
    if (p.index != nullptr)
      slot = p.index[(long long)b * p.T + t];
    else
      slot = (long long)(p.start != nullptr ? p.start[b] : p.start0) + t;
    T* ok = static_cast<T*>(p.dst[0]) + r * kD;
    T* ov = static_cast<T*>(p.dst[1]) + r * kD;
    const int at = 64 * a + 8 * q;
    if (slot < 0 || slot >= p.c.cap) {
      if (m == 0) record_error(p.status, CORE_ERR_INVALID_ARG, 1411, t);
      const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      store8(ok + at, zero);
      store8(ok + at + 32, zero);
      store8(ov + 16 * m, zero);
      store8(ov + 16 * m + 8, zero);
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
      kw[0] = x.x;
      kw[1] = x.y;
      vw[0] = y.x;
      vw[1] = y.y;
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(kc + ((16u * m) ^ key_swizzle<8>((uint32_t)slot)));
      const uint4 y = *reinterpret_cast<const uint4*>(vc + ((16u * m) ^ value_swizzle<8>((uint32_t)slot)));
      kw[0] = x.x;
      kw[1] = x.y;
      kw[2] = x.z;
      kw[3] = x.w;
      vw[0] = y.x;
      vw[1] = y.y;
      vw[2] = y.z;
      vw[3] = y.w;
    }
    const uint32_t k0 = km[kG == 4 ? 2 * a : kG == 2 ? a : 0], k1 = kG == 4 ? km[2 * a + 1] : k0;
    const uint32_t v0 = vm[kG == 4 ? m >> 1 : kG == 2 ? a : 0];
    decode_store<T, kBits>(kw, k0, ok + at);
    decode_store<T, kBits>(kw + kBits / 4, k1, ok + at + 32);
    decode_store<T, kBits>(vw, v0, ov + 16 * m);
    decode_store<T, kBits>(vw + kBits / 4, v0, ov + 16 * m + 8);
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

// Eight lanes a row, at most 8 resident blocks' worth of grid per SM.
int row_blocks(long long rows) {
  const long long need = (rows + kvq::kThreads / 8 - 1) / (kvq::kThreads / 8), cap = (long long)sm_count() * 8;
  return (int)(need < cap ? need : cap);
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
  if (src_len <= 0 || n_rows <= 0 || (index == nullptr && n_rows > src_len))
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
  const int blocks = row_blocks((long long)cache->batch * cache->n_kv_heads * n_rows);
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
  if (n_rows <= 0) return set_error(CORE_ERR_INVALID_ARG, f + ": bad row count");
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
  const int blocks = row_blocks((long long)cache->batch * cache->n_kv_heads * n_rows);
  if (!by_type<Read>(dtype, cache->bits, cache->group, blocks, static_cast<cudaStream_t>(stream), p))
    return set_error(CORE_ERR_UNSUPPORTED, f + ": dtype must be bf16, f16 or f32");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CORE_OK : cuda_error(e, "dequantize_kernel launch");
}
