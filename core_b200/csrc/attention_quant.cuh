// What the two kernels of the attention over the quantised cache share: their
// arguments, the places of rows and tokens, and the join of a sequence's parts.
#pragma once

#include <atomic>

#include "common.cuh"
#include "kvq_common.cuh"

namespace core {
namespace kvq {

// P = 2^(S - anchor): a row's anchor lies kLift (in powers of two) below its maximum when it
// was last raised, and is raised when a score passes it by more than kTop (a difference,
// which is exact).  So P is 2^14 at most, which leaves f16 room for what rounding adds to
// scores above 2^23, and goes down to 2^-25, 2^-32 of the row's largest.  With the maximum
// itself as anchor a long tail of weights of 2^-25 was lost.
constexpr float kLift = 7.0f, kTop = 14.0f;

struct AttnParams {
  const uint8_t* kc;
  const uint32_t* km;
  const uint8_t* vc;
  const uint32_t* vm;
  const void* q;
  long long qb, qh, ql;  // element strides of (B, Hq, Lq)
  const int* lengths;    // (B), or null: max_len for all
  const uint8_t* mask;   // (B, mask_stride), 0: hidden; or null
  long long mask_stride;
  int B, Hkv, G, Lq, cap, max_len;
  int n_rt, n_split;  // row tiles a KV head, parts of a sequence
  int causal, f16;
  float scale_log2;
  void* out;    // (B, Lq, Hq, d)
  float* lse;   // (B, Hq, Lq), natural log
  float* part_o;    // (B Hkv, row, split, d) f32 where n_split > 1
  float* part_lse;  // (B Hkv, row, split), base 2
  DeviceStatus* status;
};

// Tokens of one sequence that the kernel sees.
__device__ __forceinline__ int sequence_length(const AttnParams& p, int b) {
  int n = p.max_len;
  if (p.lengths != nullptr) {
    const int given = p.lengths[b];
    if (given < 0 || given > p.max_len) {
      if (threadIdx.x == 0) record_error(p.status, CORE_ERR_INVALID_ARG, 1421, b);
      n = given < 0 ? 0 : p.max_len;
    } else {
      n = given;
    }
  }
  return n;
}

// Last token (exclusive) that query row r of a KV head sees; rows past the end see none.
__device__ __forceinline__ int row_limit(const AttnParams& p, int r, int len) {
  const int i = r / p.G;
  if (i >= p.Lq) return 0;
  return p.causal ? max(len - p.Lq + i + 1, 0) : len;
}

// Tiles of `tok` tokens that each part of a sequence takes.
__device__ __forceinline__ int tiles_per_split(int end, int tok, int n_split) {
  const int tiles = (end + tok - 1) / tok;
  return (tiles + n_split - 1) / n_split;
}

// Power of two, as two factors within f32's range, that brings a query row whose
// largest element is `mx` into [2^7, 2^8).
struct RowShift {
  float f1, f2;  // their product scales the row
  float inv1, inv2;
};
__device__ __forceinline__ RowShift row_shift(float mx) {
  const int e = (int)((__float_as_uint(mx) >> 23) & 255u) - 127;
  const int sh = mx > 0.f && e < 128 ? 7 - e : 0;
  const int sh1 = sh / 2, sh2 = sh - sh1;
  RowShift r;
  r.f1 = __uint_as_float((uint32_t)(127 + sh1) << 23);
  r.f2 = __uint_as_float((uint32_t)(127 + sh2) << 23);
  r.inv1 = __uint_as_float((uint32_t)(127 - sh1) << 23);
  r.inv2 = __uint_as_float((uint32_t)(127 - sh2) << 23);
  return r;
}

// Two neighbouring elements of a bf16 or f16 row as f32.
__device__ __forceinline__ float2 query_pair(uint32_t w, bool f16) {
  if (f16) return __half22float2(as_half2(w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Programmatic dependent launch: the kernel of the parts lets the join start, and
// the join waits there until every part is written.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Sets a kernel's shared memory limits at its first launch on a device: `done`
// has a bit for each device that has them.
inline cudaError_t prepare_kernel(const void* kern, uint32_t smem, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// The kernel for many query rows (attention_quant_many.cu): rows and tokens of a
// tile, and its launch.
constexpr int kManyRows = 256, kManyTok = 128;
cudaError_t launch_many(int bits, int group, const AttnParams& p, long long blocks, cudaStream_t s);

}  // namespace kvq
}  // namespace core
