// Attention over the quantised KV cache (4 or 8 bits), for few query rows a KV
// head: single tokens, short runs of proposed tokens.
//
//   S = scale q (n s + z)^T,  out = softmax(S) (n s + z),  LSE = log sum exp S
//
// What bounds it: the packed cache is read once, 16 bits + 4 (128 / group) bytes a
// row of K or V; beside that, every code has to be turned into a matrix operand.
// In 8 bits the bytes bind: 8 x 32768 tokens of 8 heads 91-101 us by the group, 6.0-6.2
// TB/s; one sequence of 131072 tokens 49 us, 5.8 TB/s.  In 4 bits neither the bytes
// (8 x 32768 tokens 67-70 us, 4.3-4.9 TB/s; 131072 tokens 41 us, 24 of them at the
// rate of memory) nor the issue slots (62% and 58% used) are full: the 670
// instructions of a tile of 32 tokens and warp depend on one another (K's codes,
// products, maximum, exponent, transpose, V's codes), and the 16 or 12 warps that an SM
// holds do not cover all of it.  Half of the instructions go through the half-rate
// integer pipe that masks and pairs the nibbles (55% busy).
//
//  * The codes are the A operand (16 tokens, or 16 channels, a tile) and the
//    query rows the 8 columns of B (up to three such tiles a CTA), so that a GQA
//    group of up to 8 rows wastes little; S^T comes out with a token per row and goes
//    back in as the B operand of P V through movmatrix, without leaving the registers.
//  * K's codes enter as exact integers: a nibble masked out of its word is the
//    f16 subnormal n 2^-24 (or 16 n 2^-24; q then carries the 1/16).  A group's
//    products are multiplied by its scale in f32, and the zeros come in through
//    one more product, z times the row's sum of q over the group (as two f16
//    terms), so that S has no rounding but f32's.  q is scaled by a power of two
//    to f16's range per row; its elements stay exact down to 2^-18 of the row's largest.
//  * V's codes are spread over tokens in the scale that multiplies them, so
//    they become f16 values n s + z (one rounding, 2^-11) in registers.
//  * A warp owns 32-token tiles (every fourth of its CTA's) with its own ring of
//    bulk copies, running maxima and sums: nothing waits for another warp until
//    the CTA's four results are joined.  Sums are rescaled only when a score
//    passes the maximum that they were scaled with by 2^7.
//  * A sequence is cut over CTAs when there are few (batch row, KV head) pairs; a
//    second kernel, set up while the parts run, joins them.  Which kernel takes a
//    call and into how many parts is decided by modelled times (below).
//  * Sums, maxima and the LSE are f32.  P is rounded to f16 (2^7 at the running
//    maximum; below 2^-32 of the row's largest it vanishes) and so are V's values; scores are not.
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

#include "attention_quant.cuh"
#include "host_util.h"

namespace core {
namespace kvq {

constexpr int kWarps = 4;
constexpr int kAttnThreads = kWarps * 32;
constexpr int kTok = 32;  // tokens of a warp's tile


template <int kBits, int kG>
struct Stage {
  static constexpr uint32_t kCodes = kTok * 16 * kBits, kMeta = kTok * 4 * kG;
  static constexpr uint32_t kKc = 0, kVc = kCodes, kKm = 2 * kCodes, kVm = kKm + kMeta, kBytes = kVm + kMeta;
  static constexpr int kCount = 2;  // more stages gain nothing: 16 warps an SM have 150 KB on the way
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Four values in the output type.
__device__ __forceinline__ uint2 half4(float4 x, bool f16) {
  if (f16) return make_uint2(as_u32(__floats2half2_rn(x.x, x.y)), as_u32(__floats2half2_rn(x.z, x.w)));
  const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

__device__ __forceinline__ float low_half(uint32_t w) { return __low2float(as_half2(w)); }

// Query rows [8 nt, 8 nt + 8) of a tile as B operands: lane (g, t) holds of row g
// the channels 32 b + 8 t .. + 7, in pairs i = 0..3: reg 4 b + i.
struct QueryRow {
  uint4 u[4];
};
__device__ __forceinline__ QueryRow load_query(const AttnParams& p, int b, int kvh, int row, int t) {
  QueryRow r;
  const int i = row / p.G;
  const bool live = i < p.Lq;
  const uint16_t* src = static_cast<const uint16_t*>(p.q) + b * p.qb +
                        (long long)(kvh * p.G + (live ? row - i * p.G : 0)) * p.qh + (long long)(live ? i : 0) * p.ql;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    r.u[c] = live ? __ldg(reinterpret_cast<const uint4*>(src + 32 * c + 8 * t)) : make_uint4(0, 0, 0, 0);
  return r;
}
template <int kBits, int kG>
__device__ __forceinline__ void set_query(const AttnParams& p, const QueryRow& row, int t, uint32_t (&qf)[16],
                                          uint32_t& qsum, float& row_scale) {
  float x[32];
  float mx = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t w[4] = {row.u[c].x, row.u[c].y, row.u[c].z, row.u[c].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = query_pair(w[j], p.f16 != 0);
      x[8 * c + 2 * j] = f.x;
      x[8 * c + 2 * j + 1] = f.y;
      mx = fmax3(mx, fabsf(f.x), fabsf(f.y));
    }
  }
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const RowShift sh = row_shift(mx);
  float part[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    part[c] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(x[8 * c + 2 * j] * sh.f1 * sh.f2, x[8 * c + 2 * j + 1] * sh.f1 * sh.f2);
      const float2 r = __half22float2(h);
      part[c] += r.x + r.y;
      // 4 bits: odd pairs meet 16 n
      qf[4 * c + j] = as_u32(kBits == 4 && (j & 1) ? __hmul2(h, __floats2half2_rn(0.0625f, 0.0625f)) : h);
    }
    part[c] += __shfl_xor_sync(0xffffffffu, part[c], 1);
    part[c] += __shfl_xor_sync(0xffffffffu, part[c], 2);
  }
  // sum of q over group t (t < kG), as two f16 terms
  float s;
  if (kG == 4)
    s = t == 0 ? part[0] : t == 1 ? part[1] : t == 2 ? part[2] : part[3];
  else if (kG == 2)
    s = t == 0 ? part[0] + part[1] : t == 1 ? part[2] + part[3] : 0.f;
  else
    s = t == 0 ? (part[0] + part[1]) + (part[2] + part[3]) : 0.f;
  const __half hi = __float2half_rn(s);
  qsum = as_u32(__halves2half2(hi, __float2half_rn(s - __half2float(hi))));
  // the sums of products come in units of 2^-24 (the codes') and of the shift
  row_scale = p.scale_log2 * 16777216.f * sh.inv1 * sh.inv2;
}

template <int kBits, int kG, int kNT, int kCtas>
__global__ void __launch_bounds__(kAttnThreads, kCtas) attn_few_kernel(const AttnParams p) {
  using St = Stage<kBits, kG>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps * St::kCount];
  __shared__ int abort_storage;
  __shared__ float sm_m[kWarps][8 * kNT], sm_l[kWarps][8 * kNT];
  __shared__ long long sm_at[8 * kNT];
  volatile int* abort_flag = &abort_storage;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned u = blockIdx.x;
  const int rt = (int)(u % (unsigned)p.n_rt);
  u /= (unsigned)p.n_rt;
  const int split = (int)(u % (unsigned)p.n_split);
  const int bh = (int)(u / (unsigned)p.n_split);
  const int b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  const int row0 = rt * 8 * kNT;
  const int rows = p.G * p.Lq;

  // the queries and the length are asked for first: everything else of the start
  // happens while they come
  QueryRow qrow[kNT];
#pragma unroll
  for (int n = 0; n < kNT; ++n) qrow[n] = load_query(p, b, kvh, row0 + 8 * n + g, t);
  const int len = sequence_length(p, b);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * St::kCount; ++i) mbar_init(smem_u32(&bars[i]), 1);
    abort_storage = 0;
    fence_barrier_init();
  }
  __syncthreads();

  const int last_row = min(row0 + 8 * kNT, rows) - 1;
  const int end = row_limit(p, last_row, len);  // no row of the tile sees a token from here on
  const int first_end = row_limit(p, row0, len);  // every row sees the tokens before this
  const int per = tiles_per_split(end, kTok, p.n_split);
  const int tile0 = split * per, tile1 = min(tile0 + per, (end + kTok - 1) / kTok);
  if (p.n_split > 1) launch_dependents();
  if (p.n_split > 1 && tile0 >= tile1 && split > 0) return;  // the join does not read this part

  const long long base = (long long)bh * p.cap;
  const uint32_t ring = smem_u32(smem) + (uint32_t)warp * (St::kCount * St::kBytes);
  const uint32_t my_bars = smem_u32(&bars[warp * St::kCount]);
  const int n_mine = tile1 - tile0 > warp ? (tile1 - tile0 - warp + kWarps - 1) / kWarps : 0;
  auto issue = [&](int it) {
    const int s = it % St::kCount;
    const long long row = base + (long long)(tile0 + warp + it * kWarps) * kTok;
    const uint32_t bar = my_bars + 8u * s, dst = ring + s * St::kBytes;
    mbar_arrive_expect_tx(bar, St::kBytes);
    bulk_load(dst + St::kKc, p.kc + row * (16 * kBits), St::kCodes, bar);
    bulk_load(dst + St::kKm, p.km + row * kG, St::kMeta, bar);
    bulk_load(dst + St::kVc, p.vc + row * (16 * kBits), St::kCodes, bar);
    bulk_load(dst + St::kVm, p.vm + row * kG, St::kMeta, bar);
  };
  if (lane == 0)
    for (int it = 0; it < St::kCount && it < n_mine; ++it) issue(it);

  uint32_t qf[kNT][16], qsum[kNT];
  float rs[kNT][2];
  int lim[kNT][2];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    float r;
    set_query<kBits, kG>(p, qrow[n], t, qf[n], qsum[n], r);
    rs[n][0] = __shfl_sync(0xffffffffu, r, 8 * t);      // row 2 t of the eight
    rs[n][1] = __shfl_sync(0xffffffffu, r, 8 * t + 4);  // row 2 t + 1
    lim[n][0] = row_limit(p, row0 + 8 * n + 2 * t, len);
    lim[n][1] = row_limit(p, row0 + 8 * n + 2 * t + 1, len);
  }

  float o[8][kNT][4];
  float anchor[kNT][2], l[kNT][2];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    anchor[n][0] = anchor[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
  }

  // Row r of a 16-token tile holds token pi(r): pi(2 i) = i, pi(2 i + 1) = 4 +
  // (i ^ 1), pi(r + 8) = pi(r) + 8: lanes that read K or V together then never
  // meet in a bank.
  const int pig = (g & 1) ? 4 + ((g >> 1) ^ 1) : g >> 1;  // token of K row g
  const int va = t, vb = 4 + (t ^ 1);                     // tokens of V columns 2 t and 2 t + 1
  const int vgrp = (g * kG) >> 3;                         // group of V channels 16 g ..

  const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (long long)b * p.mask_stride;
  bool ok = true;
  // this lane's token of the tile, seen or not: asked for a tile ahead
  auto look = [&](int it) -> uint32_t {
    const int tok = (tile0 + warp + it * kWarps) * kTok + lane;
    if (it >= n_mine || tok >= end) return 0u;
    return mask == nullptr ? 1u : (uint32_t)__ldg(mask + tok);
  };
  uint32_t mine = look(0);
  for (int it = 0; it < n_mine; ++it) {
    const int s = it % St::kCount;
    const int tok0 = (tile0 + warp + it * kWarps) * kTok;
    const uint32_t bits = __ballot_sync(0xffffffffu, mine != 0);
    mine = look(it + 1);
    ok = bounded_wait(my_bars + 8u * s, (uint32_t)(it / St::kCount) & 1u, abort_flag, p.status, 1422);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {  // give up, but leave no copy of this warp's in flight
      for (int k = it; k < it + St::kCount && k < n_mine; ++k) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(my_bars + 8u * (k % St::kCount), (uint32_t)(k / St::kCount) & 1u) &&
               globaltimer_ns() - t0 < kWaitLimitNs) {
        }
      }
      break;
    }
    const uint32_t st = ring + s * St::kBytes;

    // ---- S^T: two tiles of 16 tokens, kNT tiles of 8 rows
    float sc[2][kNT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint32_t tk0 = 16 * mt + pig, tk1 = tk0 + 8;
      uint32_t m0[kG], m1[kG];
      const uint32_t ma = st + St::kKm;
      if constexpr (kG == 4) {
        const uint4 x = lds128(ma + tk0 * 16), y = lds128(ma + tk1 * 16);
        m0[0] = x.x; m0[1] = x.y; m0[2] = x.z; m0[3] = x.w;
        m1[0] = y.x; m1[1] = y.y; m1[2] = y.z; m1[3] = y.w;
      } else if constexpr (kG == 2) {
        const uint2 x = lds64(ma + tk0 * 8), y = lds64(ma + tk1 * 8);
        m0[0] = x.x; m0[1] = x.y;
        m1[0] = y.x; m1[1] = y.y;
      } else {
        m0[0] = lds32(ma + tk0 * 4);
        m1[0] = lds32(ma + tk1 * 4);
      }
      // zeros: column 2 t, 2 t + 1 of the product both hold group t's
      uint32_t z0 = 0, z1 = 0;
      if constexpr (kG == 4) {
        z0 = lds32(ma + tk0 * 16 + t * 4);
        z1 = lds32(ma + tk1 * 16 + t * 4);
      } else if constexpr (kG == 2) {
        z0 = t == 0 ? m0[0] : t == 1 ? m0[1] : 0u;
        z1 = t == 0 ? m1[0] : t == 1 ? m1[1] : 0u;
      } else {
        z0 = t == 0 ? m0[0] : 0u;
        z1 = t == 0 ? m1[0] : 0u;
      }
      z0 = prmt(z0, z0, 0x3232);
      z1 = prmt(z1, z1, 0x3232);
      float zs[kNT][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        zs[n][0] = zs[n][1] = zs[n][2] = zs[n][3] = 0.f;
        mma1688(zs[n], z0, z1, qsum[n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[mt][n][e] = zs[n][e] * 5.9604644775390625e-8f;  // 2^-24
      }
      // codes: words of block b of 32 channels (8 bits: two words)
      uint32_t w0[kBits], w1[kBits];
#pragma unroll
      for (int c = 0; c < kBits / 4; ++c) {
        const uint32_t at0 = (64u * c + 16u * t) ^ key_swizzle<kBits>(tk0), at1 = (64u * c + 16u * t) ^ key_swizzle<kBits>(tk1);
        const uint4 x = lds128(st + St::kKc + tk0 * (16 * kBits) + at0), y = lds128(st + St::kKc + tk1 * (16 * kBits) + at1);
        w0[4 * c] = x.x; w0[4 * c + 1] = x.y; w0[4 * c + 2] = x.z; w0[4 * c + 3] = x.w;
        w1[4 * c] = y.x; w1[4 * c + 1] = y.y; w1[4 * c + 2] = y.z; w1[4 * c + 3] = y.w;
      }
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        float acc[kNT][4];
#pragma unroll
        for (int n = 0; n < kNT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
        for (int bb = 0; bb < 4 / kG; ++bb) {
          const int blk = gr * (4 / kG) + bb;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // pairs 2 h and 2 h + 1: 16 channels of the quad
            uint32_t a0, a1, a2, a3;
            if constexpr (kBits == 4) {
              const uint32_t x0 = h ? w0[blk] >> 8 : w0[blk], x1 = h ? w1[blk] >> 8 : w1[blk];
              a0 = x0 & 0x000f000fu;
              a1 = x1 & 0x000f000fu;
              a2 = x0 & 0x00f000f0u;
              a3 = x1 & 0x00f000f0u;
            } else {
              const uint32_t x0 = w0[2 * blk + h], x1 = w1[2 * blk + h];
              a0 = x0 & 0x00ff00ffu;
              a1 = x1 & 0x00ff00ffu;
              a2 = (x0 >> 8) & 0x00ff00ffu;
              a3 = (x1 >> 8) & 0x00ff00ffu;
            }
#pragma unroll
            for (int n = 0; n < kNT; ++n)
              mma16816(acc[n], a0, a1, a2, a3, qf[n][4 * blk + 2 * h], qf[n][4 * blk + 2 * h + 1]);
          }
        }
        const float s0 = low_half(m0[gr]), s1 = low_half(m1[gr]);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          sc[mt][n][0] = fmaf(s0, acc[n][0], sc[mt][n][0]);
          sc[mt][n][1] = fmaf(s0, acc[n][1], sc[mt][n][1]);
          sc[mt][n][2] = fmaf(s1, acc[n][2], sc[mt][n][2]);
          sc[mt][n][3] = fmaf(s1, acc[n][3], sc[mt][n][3]);
        }
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[mt][n][e] *= rs[n][e & 1];
    }
    const bool full = bits == 0xffffffffu && tok0 + kTok <= first_end;
    if (!full) {
      // hidden tokens: value 0 whatever their bytes hold (scale and zero are
      // cleared in the tile), score -inf
      if (!((bits >> lane) & 1u)) {
#pragma unroll
        for (int c = 0; c < kG; ++c) sts32(st + St::kVm + (uint32_t)(lane * kG + c) * 4u, 0u);
      }
      fence_proxy_async_shared();  // before a copy may take the stage again
      __syncwarp();
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 16 * mt + pig + (e >> 1) * 8;
            if (!((bits >> k) & 1u) || tok0 + k >= lim[n][e & 1]) sc[mt][n][e] = -INFINITY;
          }
    }

    // ---- running maxima, as the anchors of P
    bool raise = false;
    float mx[kNT][2];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[n][h] = fmaxf(fmaxf(sc[0][n][h], sc[0][n][h + 2]), fmaxf(sc[1][n][h], sc[1][n][h + 2]));
        raise |= mx[n][h] - anchor[n][h] > kTop;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v = mx[n][h];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          if (v - anchor[n][h] > kTop) {
            const float f = ex2_approx(anchor[n][h] - (v - kLift));
            anchor[n][h] = v - kLift;
            l[n][h] *= f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[j][n][h] *= f;
              o[j][n][h + 2] *= f;
            }
          }
        }
    }

    // ---- P^T, and its transpose as the B operand
    uint32_t pf[2][kNT][2];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const float b0 = anchor[n][0] == -INFINITY ? 0.f : anchor[n][0];
      const float b1 = anchor[n][1] == -INFINITY ? 0.f : anchor[n][1];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float e0 = ex2_approx(sc[mt][n][0] - b0), e1 = ex2_approx(sc[mt][n][1] - b1);
        const float e2 = ex2_approx(sc[mt][n][2] - b0), e3 = ex2_approx(sc[mt][n][3] - b1);
        l[n][0] += e0 + e2;
        l[n][1] += e1 + e3;
        pf[mt][n][0] = movmatrix_trans(as_u32(__floats2half2_rn(e0, e1)));
        pf[mt][n][1] = movmatrix_trans(as_u32(__floats2half2_rn(e2, e3)));
      }
    }

    // ---- O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint32_t ta = 16 * mt + va, tb = 16 * mt + vb;
      const uint32_t ma = st + St::kVm + vgrp * 4;
      const uint32_t xa = lds32(ma + ta * (4 * kG)), xb = lds32(ma + tb * (4 * kG));
      const uint32_t ya = lds32(ma + (ta + 8) * (4 * kG)), yb = lds32(ma + (tb + 8) * (4 * kG));
      const __half2 sx = as_half2(prmt(xa, xb, 0x5410)), zx = as_half2(prmt(xa, xb, 0x7632));
      const __half2 sy = as_half2(prmt(ya, yb, 0x5410)), zy = as_half2(prmt(ya, yb, 0x7632));
      const uint32_t vs = st + St::kVc;
      uint32_t wa[kBits / 2], wb[kBits / 2], ua[kBits / 2], ub[kBits / 2];
      if constexpr (kBits == 4) {
        const uint32_t at = (8u * g) ^ value_swizzle<4>(ta);  // alike for all four tokens
        const uint2 r0 = lds64(vs + ta * 64 + at), r1 = lds64(vs + tb * 64 + at);
        const uint2 r2 = lds64(vs + (ta + 8) * 64 + at), r3 = lds64(vs + (tb + 8) * 64 + at);
        wa[0] = r0.x; wa[1] = r0.y; wb[0] = r1.x; wb[1] = r1.y;
        ua[0] = r2.x; ua[1] = r2.y; ub[0] = r3.x; ub[1] = r3.y;
      } else {
        const uint32_t ata = (16u * g) ^ value_swizzle<8>(ta), atb = (16u * g) ^ value_swizzle<8>(tb);
        const uint4 r0 = lds128(vs + ta * 128 + ata), r1 = lds128(vs + tb * 128 + atb);
        const uint4 r2 = lds128(vs + (ta + 8) * 128 + ata), r3 = lds128(vs + (tb + 8) * 128 + atb);
        wa[0] = r0.x; wa[1] = r0.y; wa[2] = r0.z; wa[3] = r0.w;
        wb[0] = r1.x; wb[1] = r1.y; wb[2] = r1.z; wb[3] = r1.w;
        ua[0] = r2.x; ua[1] = r2.y; ua[2] = r2.z; ua[3] = r2.w;
        ub[0] = r3.x; ub[1] = r3.y; ub[2] = r3.z; ub[3] = r3.w;
      }
#pragma unroll
      for (int w = 0; w < kBits / 2; ++w) {
        // even channels of the word for both tokens, and odd ones
        const uint32_t ex = prmt(wa[w], wb[w], 0x5410), ox = prmt(wa[w], wb[w], 0x7632);
        const uint32_t ey = prmt(ua[w], ub[w], 0x5410), oy = prmt(ua[w], ub[w], 0x7632);
#pragma unroll
        for (int i = 0; i < 16 / kBits; ++i) {
          const uint32_t a0 = as_u32(__hfma2(code_pair<kBits>(ex, i), sx, zx));
          const uint32_t a1 = as_u32(__hfma2(code_pair<kBits>(ox, i), sx, zx));
          const uint32_t a2 = as_u32(__hfma2(code_pair<kBits>(ey, i), sy, zy));
          const uint32_t a3 = as_u32(__hfma2(code_pair<kBits>(oy, i), sy, zy));
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816(o[w * (16 / kBits) + i][n], a0, a1, a2, a3, pf[mt][n][0], pf[mt][n][1]);
        }
      }
    }
    __syncwarp();
    if (lane == 0 && it + St::kCount < n_mine) issue(it + St::kCount);
  }

  // ---- join the warps: maxima and sums, then each row's weighted mean
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = l[n][h];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      if (g == 0) {
        sm_m[warp][8 * n + 2 * t + h] = anchor[n][h];
        sm_l[warp][8 * n + 2 * t + h] = v;
      }
    }
  __syncthreads();  // also: every warp's ring is idle
  if (*abort_flag) return;
  float* so = reinterpret_cast<float*>(smem);  // [warp][row][128]
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* dst = so + ((warp * 8 * kNT) + 8 * n + 2 * t + h) * kD + 16 * g;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        // m-tile j: channels 2 j (row g) and 2 j + 1 (row g + 8) of the sixteen
        *reinterpret_cast<float4*>(dst + 2 * j) =
            make_float4(o[j][n][h], o[j][n][h + 2], o[j + 1][n][h], o[j + 1][n][h + 2]);
      }
    }
  if (threadIdx.x < 8 * kNT) {  // one thread a row: the warps' weights, and where the row goes
    const int r = threadIdx.x, row = row0 + r;
    float m = -INFINITY, lt = 0.f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm_m[w][r]);
    const float mb = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = ex2_approx(sm_m[w][r] - mb);
      lt += f[w] * sm_l[w][r];
    }
    // a row that saw no token: output 0, LSE -inf.  (NaN scores leave lt NaN.)
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sm_m[w][r] = f[w] * inv;
    const float lse2 = lt == 0.f ? -INFINITY : m + log2f(lt);
    if (row < rows) {
      if (p.n_split > 1) {
        const long long at = ((long long)bh * rows + row) * p.n_split + split;
        sm_at[r] = at;
        p.part_lse[at] = lse2;
      } else {
        const int i = row / p.G, hq = kvh * p.G + row - i * p.G, Hq = p.Hkv * p.G;
        sm_at[r] = ((long long)b * p.Lq + i) * Hq + hq;
        p.lse[((long long)b * Hq + hq) * p.Lq + i] = lse2 * 0.69314718055994531f;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2 * kNT; ++k) {
    const int r = warp + kWarps * k;
    if (row0 + r >= rows) break;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm_m[w][r];
      const float4 x = reinterpret_cast<const float4*>(so + (w * 8 * kNT + r) * kD)[lane];
      acc.x += f * x.x;
      acc.y += f * x.y;
      acc.z += f * x.z;
      acc.w += f * x.w;
    }
    if (p.n_split > 1)
      reinterpret_cast<float4*>(p.part_o + sm_at[r] * kD)[lane] = acc;
    else
      reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + sm_at[r] * kD)[lane] = half4(acc, p.f16);
  }
}

// Joins the parts of a row: weights 2^(lse_i - max), then their mean.  A CTA of
// four warps takes a row: every warp works out the weights, takes every fourth
// part, four channels a lane, and the four sums meet in shared memory.
constexpr int kMaxSplit = 128;

__global__ void __launch_bounds__(128) attn_join_kernel(const AttnParams p, int rows_per_tile, int tok) {
  __shared__ float weight[kMaxSplit];
  __shared__ float4 sums[4][32];
  const int rows = p.G * p.Lq;
  const long long row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bh = (int)(row / rows), r = (int)(row - (long long)bh * rows);
  const int b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  int len = p.max_len;
  if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), p.max_len);
  // the parts that this row's tile wrote (part 0 always is)
  const int last_row = min(r / rows_per_tile * rows_per_tile + rows_per_tile, rows) - 1;
  const int end = row_limit(p, last_row, len);
  const int per = tiles_per_split(end, tok, p.n_split);
  const int n = per == 0 ? 1 : ((end + tok - 1) / tok + per - 1) / per;
  wait_primary();
  const float* lse = p.part_lse + row * p.n_split;
  float v[kMaxSplit / 32];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMaxSplit / 32; ++k) {
    v[k] = 32 * k + lane < n ? lse[32 * k + lane] : -INFINITY;
    m = fmaxf(m, v[k]);
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  const float mb = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxSplit / 32; ++k) {
    const float w = ex2_approx(v[k] - mb);
    l += w;
    if (warp == 0) weight[32 * k + lane] = w;
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  __syncthreads();
  const float4* po = reinterpret_cast<const float4*>(p.part_o + row * p.n_split * kD) + lane;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = warp; i < n; i += 4) {
    const float w = weight[i];
    const float4 x = po[(long long)i * 32];
    acc.x += w * x.x;
    acc.y += w * x.y;
    acc.z += w * x.z;
    acc.w += w * x.w;
  }
  sums[warp][lane] = acc;
  __syncthreads();
  const int c = threadIdx.x;
  const float* sf = reinterpret_cast<const float*>(sums);
  const float sum = (sf[c] + sf[kD + c]) + (sf[2 * kD + c] + sf[3 * kD + c]);
  const float val = l == 0.f ? 0.f : sum / l;
  const int i = r / p.G, hq = kvh * p.G + r - i * p.G, Hq = p.Hkv * p.G;
  const long long at = (((long long)b * p.Lq + i) * Hq + hq) * kD + c;
  if (p.f16)
    static_cast<__half*>(p.out)[at] = __float2half_rn(val);
  else
    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(val);
  if (c == 0)
    p.lse[((long long)b * Hq + hq) * p.Lq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// The same with a warp a row, for calls with enough rows to fill the SMs that way
// (a CTA a row spends 400 instructions a warp on each; with it 512 queries x 32 heads
// over 16384 tokens, two parts a row, took 171 us instead of 153).
__global__ void __launch_bounds__(128) attn_join_rows_kernel(const AttnParams p, int rows_per_tile, int tok) {
  const int rows = p.G * p.Lq;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  wait_primary();
  if (row >= (long long)p.B * p.Hkv * rows) return;
  const int bh = (int)(row / rows), r = (int)(row - (long long)bh * rows);
  const int b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  int len = p.max_len;
  if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), p.max_len);
  const int last_row = min(r / rows_per_tile * rows_per_tile + rows_per_tile, rows) - 1;
  const int end = row_limit(p, last_row, len);
  const int per = tiles_per_split(end, tok, p.n_split);
  const int n = per == 0 ? 1 : ((end + tok - 1) / tok + per - 1) / per;
  const float* lse = p.part_lse + row * p.n_split;
  const float4* po = reinterpret_cast<const float4*>(p.part_o + row * p.n_split * kD) + lane;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 32) m = fmaxf(m, lse[i]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  const float mb = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float w = ex2_approx(lse[i] - mb);
    const float4 x = po[(long long)i * 32];
    l += w;
    acc.x += w * x.x;
    acc.y += w * x.y;
    acc.z += w * x.z;
    acc.w += w * x.w;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  acc.x *= inv;
  acc.y *= inv;
  acc.z *= inv;
  acc.w *= inv;
  const int i = r / p.G, hq = kvh * p.G + r - i * p.G, Hq = p.Hkv * p.G;
  const long long at = ((long long)b * p.Lq + i) * Hq + hq;
  reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * kD)[lane] = half4(acc, p.f16);
  if (lane == 0)
    p.lse[((long long)b * Hq + hq) * p.Lq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// CTAs of attn_few_kernel that fit an SM: in 8 bits by shared memory (74 KB each at
// groups of 32), in 4 bits by registers.
constexpr int resident(int bits, int nt) { return nt > 1 ? 2 : bits == 8 ? 3 : 4; }

// Microseconds that the two kernels take on a B200, as measured over lengths of 1
// to 131072 and 1 to 2048 rows; the plan only compares them.
//
// attn_few_kernel: the longer of two times, rounded off where they meet (eighth
// powers).  A warp takes its tiles one after the other, `tile` each; and the SMs
// together need `all` for each of their tiles, by instructions issued (4 bits) or bytes
// (8 bits).  Starts grow with the CTAs on an SM, and later waves' are half hidden.
// Fitted to 600 calls of 333 to 131072 tokens and 2 to 512 sequences x heads; what it
// picks is 1% off the best of them (24 rows: 4% on top, for they gain little where
// the other choices are near).
struct FewTimes {
  double start, start_cta, tile, all;  // us; all: 1e-3 us over the 148 SMs
};
FewTimes few_times(int bits, int nt, int ctas_sm) {
  if (nt == 3) return bits == 4 ? FewTimes{4.4, 1.8, 1.7, 1.92} : FewTimes{3.9, 2.4, 1.72, 2.14};
  if (nt == 2) return bits == 4 ? FewTimes{2.7, 1.35, 1.35, 1.33} : FewTimes{2.9, 1.35, 1.3, 1.55};
  if (bits == 8) return {1.3, 1.0, 1.24, 1.29};
  return {1.2, 0.9, ctas_sm == 4 ? 1.36 : 1.22, 1.0};
}
double few_us(int bits, int ctas_sm, int nt, long long units, int tiles, int n) {
  const long long sms = sm_count(), ctas = units * n;
  const long long waves = (ctas + sms * ctas_sm - 1) / (sms * ctas_sm);
  const long long share = (ctas + sms - 1) / sms < ctas_sm ? (ctas + sms - 1) / sms : ctas_sm;
  const int rounds = ((tiles + n - 1) / n + kWarps - 1) / kWarps;
  const FewTimes c = few_times(bits, nt, ctas_sm);
  auto squared3 = [](double x) { return x *= x, x *= x, x * x; };
  // SMs wait for fuller ones where instructions bind; memory is one for all
  const double uneven = bits == 4 ? std::sqrt((double)(waves * share * sms) / ctas) : 1.0;
  const double in_turn = (double)waves * rounds * c.tile, all = (double)units * tiles * c.all * (0.148 / sms) * uneven;
  const double body = std::sqrt(std::sqrt(std::sqrt(squared3(in_turn) + squared3(all))));
  return (0.4 + 0.6 * waves) * (c.start + c.start_cta * share) + body + (n > 1 ? 3.3 + 0.022 * n : 0.0);
}
// attn_many_kernel: one CTA an SM; its start and end, and a tile of 128 keys, depend on
// whether it has one row tile of 128 or two; the join also moves every part's rows.
double many_us(int bits, long long units, long long rows, int tiles, int n) {
  const long long sms = sm_count(), waves = (units * n + sms - 1) / sms;
  const bool two = rows > 128;
  const double tile = bits == 8 ? 2.3 : two ? 2.0 : 1.75;
  const double part = 1e-6 * 2 * kD * 4 * units * (rows < kManyRows ? rows : kManyRows) / 8.0;
  return waves * ((two ? 14.5 : 9.3) + ((tiles + n - 1) / n) * tile) + (n > 1 ? 3.8 + n * (0.022 + part) : 0.0);
}

struct Plan {
  bool many;
  int nt, ctas, n_rt, n_split;  // few rows: tiles of 8 rows a CTA, CTAs an SM
  bool join_rows;               // the parts are joined by a warp a row, not a CTA
};

// Which kernel takes the call, and into how many parts it cuts the sequences.
// Tried are the counts that fill the SMs once, twice, .. , each lowered to the
// least that gives its parts as many tiles.
Plan make_plan(int bits, int B, int Hkv, long long rows, int max_len, bool exact) {
  const long long heads = (long long)B * Hkv, sms = sm_count();
  auto least = [](int tiles, int step, long long n) {  // same tiles a part (in `step`s), fewest parts
    const long long most = (tiles + step - 1) / step;
    n = n < kMaxSplit ? n : kMaxSplit;
    n = n < most ? n : most;
    if (n < 2) return 1;
    const int each = ((tiles + (int)n - 1) / (int)n + step - 1) / step * step;
    return (tiles + each - 1) / each;
  };
  Plan r{};
  double best = 0;
  // 8, 16 or 24 rows a CTA: its rows share the codes' turning into operands, but 24
  // take all 255 registers and a longer start.  24 against 2 x 16 for 20 rows: 44
  // and 60 us over 8 x 8192 tokens of 8 heads, 12.4 and 11.8 over 1 x 4096.  8 rows in 4
  // bits: built for three CTAs an SM or, with 128 registers instead of 168, for four:
  // 41.3 and 43.4 us over 1 x 131072 tokens, 78.3 and 69.9 over 8 x 32768.
  const int few_tiles = (max_len + kTok - 1) / kTok;
  for (int nt = rows <= 8 ? 1 : 2; nt <= (rows <= 8 ? 1 : rows <= 16 ? 2 : 3); ++nt) {
    const int most = resident(bits, nt), n_rt = (int)((rows + 8 * nt - 1) / (8 * nt));
    for (int ctas = most < 3 ? most : 3; ctas <= most; ++ctas) {
      for (int k = 0; k <= 3 * ctas; ++k) {
        const int n = k == 0 ? 1 : least(few_tiles, kWarps, sms * k / (heads * n_rt));
        const double us = few_us(bits, ctas, nt, heads * n_rt, few_tiles, n);
        if (r.n_split == 0 || us < best) {
          best = us;
          r = {false, nt, ctas, n_rt, n, false};
        }
      }
    }
  }
  // Up to 32 rows stay with the kernel that keeps the keys exact, more where that is asked for.
  if (rows <= 32 || exact) return r;
  const int many_rt = (int)((rows + kManyRows - 1) / kManyRows), many_tiles = (max_len + kManyTok - 1) / kManyTok;
  const long long many_units = heads * many_rt;
  for (int k = 0; k <= 6; ++k) {
    const int n = k == 0 ? 1 : least(many_tiles, 1, sms * k / many_units);
    const double us = many_us(bits, many_units, rows, many_tiles, n);
    if (us < best) {
      best = us;
      r = {true, 0, 1, many_rt, n, false};
    }
  }
  return r;
}

Plan whole_plan(int bits, int B, int Hkv, long long rows, int max_len, bool exact) {
  Plan p = make_plan(bits, B, Hkv, rows, max_len, exact);
  // A warp a row where rows are many for their parts, else a CTA a row: 16384 rows of
  // 2 parts 171 -> 153 us with the attention itself, 2048 rows of 8 parts 31.2 -> 34.9.
  p.join_rows = rows * B * Hkv > (long long)sm_count() * 8 * p.n_split;
  return p;
}

// The plan of the workspace query serves the call of the same sizes that follows it on
// this thread, also if the SMs to plan for were changed in between (another thread
// may): the workspace fits that plan.
Plan plan(int bits, int B, int Hkv, long long rows, int max_len, bool exact, bool query) {
  struct Last {
    long long key[6];
    int sms;
    Plan plan;
  };
  static thread_local Last last{{-1, 0, 0, 0, 0, 0}, 0, {}};
  const long long key[6] = {bits, B, Hkv, rows, max_len, exact};
  const int sms = sm_count();
  bool same = !query || sms == last.sms;
  for (int i = 0; i < 6; ++i) same = same && key[i] == last.key[i];
  if (!same) {
    last.plan = whole_plan(bits, B, Hkv, rows, max_len, exact);
    last.sms = sms;
    for (int i = 0; i < 6; ++i) last.key[i] = key[i];
  }
  return last.plan;
}

template <int kBits, int kG, int kNT, int kCtas = resident(kBits, kNT)>
cudaError_t launch_few(const AttnParams& p, long long blocks, cudaStream_t s) {
  using St = Stage<kBits, kG>;
  constexpr uint32_t ring = kWarps * St::kCount * St::kBytes, join = kWarps * 8 * kNT * kD * 4;
  constexpr uint32_t smem = ring > join ? ring : join;
  auto kern = attn_few_kernel<kBits, kG, kNT, kCtas>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)blocks, kAttnThreads, smem, s>>>(p);
  return cudaGetLastError();
}

template <int kBits, int kG>
cudaError_t launch_nt(const Plan& pl, const AttnParams& p, long long blocks, cudaStream_t s) {
  if (pl.nt == 3) return launch_few<kBits, kG, 3>(p, blocks, s);
  if (pl.nt == 2) return launch_few<kBits, kG, 2>(p, blocks, s);
  if (pl.ctas == 3) return launch_few<kBits, kG, 1, 3>(p, blocks, s);
  return launch_few<kBits, kG, 1>(p, blocks, s);
}

}  // namespace kvq
}  // namespace core

using namespace core;

namespace {
template <class C>
void carve_parts(C& c, int n_split, long long rows, float** o, float** lse) {
  if (n_split <= 1) return;
  *o = c.template take<float>((size_t)rows * n_split * kvq::kD);
  *lse = c.template take<float>((size_t)rows * n_split);
}
struct SizerOut : Sizer {
  template <class T>
  T* take(size_t n) {
    Sizer::take<T>(n);
    return nullptr;
  }
};
}  // namespace

extern "C" size_t core_kvq_attention_workspace_bytes(const core_kvq_t* cache, int32_t n_q_heads, int32_t n_queries,
                                                     int32_t max_length) {
  if (cache == nullptr || cache->n_kv_heads <= 0 || n_q_heads < cache->n_kv_heads || n_queries <= 0 ||
      cache->batch <= 0 || max_length < 0)
    return 0;
  const long long rows = (long long)(n_q_heads / cache->n_kv_heads) * n_queries;
  const kvq::Plan pl = kvq::plan(cache->bits, cache->batch, cache->n_kv_heads, rows, max_length, false, true);
  SizerOut z;
  float *a, *b;
  carve_parts(z, pl.n_split, rows * cache->batch * cache->n_kv_heads, &a, &b);
  return z.used;
}

extern "C" int core_kvq_attention_plan(const core_kvq_t* cache, int32_t n_q_heads, int32_t n_queries,
                                       int32_t max_length, int32_t causal, core_kvq_plan_t* out) {
  const char* fn = "core_kvq_attention_plan";
  int rc = check_kvq(cache, fn);
  if (rc != CORE_OK) return rc;
  const std::string f(fn);
  if (out == nullptr) return set_error(CORE_ERR_INVALID_ARG, f + ": NULL argument");
  if (n_q_heads <= 0 || n_queries <= 0 || n_q_heads % cache->n_kv_heads != 0)
    return set_error(CORE_ERR_INVALID_ARG, f + ": bad query dimensions");
  if (max_length < 0 || max_length > cache->capacity)
    return set_error(CORE_ERR_INVALID_ARG, f + ": max_length outside the cache's capacity");
  const long long rows = (long long)(n_q_heads / cache->n_kv_heads) * n_queries;
  if (rows > INT_MAX / 2) return set_error(CORE_ERR_UNSUPPORTED, f + ": too many query rows");
  const kvq::Plan pl = kvq::plan(cache->bits, cache->batch, cache->n_kv_heads, rows, max_length,
                                 (causal & CORE_KVQ_EXACT_KEYS) != 0, true);
  out->row_tile = pl.many ? kvq::kManyRows : 8 * pl.nt;
  out->ctas_per_sm = pl.ctas;
  out->parts = pl.n_split;
  out->join_rows = pl.n_split > 1 && pl.join_rows;
  out->f16_keys = pl.many;
  SizerOut z;
  float *a, *b;
  carve_parts(z, pl.n_split, rows * cache->batch * cache->n_kv_heads, &a, &b);
  out->workspace_bytes = z.used;
  return CORE_OK;
}

extern "C" int core_kvq_attention(const core_kvq_t* cache, int32_t dtype, int32_t n_q_heads, int32_t n_queries,
                                  const void* q, const int64_t* q_strides, const int32_t* lengths,
                                  int32_t max_length, const uint8_t* key_mask, int64_t mask_stride, int32_t causal,
                                  float softmax_scale, void* out, float* lse, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* fn = "core_kvq_attention";
  int rc = check_kvq(cache, fn);
  if (rc != CORE_OK) return rc;
  const std::string f(fn);
  if (q == nullptr || q_strides == nullptr || out == nullptr || lse == nullptr)
    return set_error(CORE_ERR_INVALID_ARG, f + ": NULL argument");
  if (n_q_heads <= 0 || n_queries <= 0) return set_error(CORE_ERR_INVALID_ARG, f + ": non-positive dimension");
  if (n_q_heads % cache->n_kv_heads != 0)
    return set_error(CORE_ERR_INVALID_ARG, f + ": n_q_heads must be a multiple of n_kv_heads");
  if (dtype != CORE_DTYPE_BF16 && dtype != CORE_DTYPE_F16)
    return set_error(CORE_ERR_UNSUPPORTED, f + ": dtype must be bf16 or f16");
  if (max_length < 0 || max_length > cache->capacity)
    return set_error(CORE_ERR_INVALID_ARG, f + ": max_length outside the cache's capacity");
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return set_error(CORE_ERR_INVALID_ARG, f + ": softmax_scale must be positive");
  if (!aligned16(q) || !aligned16(out)) return set_error(CORE_ERR_INVALID_ARG, f + ": q and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 != 0) return set_error(CORE_ERR_INVALID_ARG, f + ": q strides must be multiples of 8 elements");
  if (key_mask != nullptr && mask_stride < max_length)
    return set_error(CORE_ERR_INVALID_ARG, f + ": key_mask rows shorter than max_length");
  const long long rows = (long long)(n_q_heads / cache->n_kv_heads) * n_queries;
  if (rows > INT_MAX / 2) return set_error(CORE_ERR_UNSUPPORTED, f + ": too many query rows");

  kvq::AttnParams p{};
  p.kc = static_cast<const uint8_t*>(cache->k_codes);
  p.km = static_cast<const uint32_t*>(cache->k_meta);
  p.vc = static_cast<const uint8_t*>(cache->v_codes);
  p.vm = static_cast<const uint32_t*>(cache->v_meta);
  p.q = q;
  p.qb = q_strides[0];
  p.qh = q_strides[1];
  p.ql = q_strides[2];
  p.lengths = lengths;
  p.mask = key_mask;
  p.mask_stride = mask_stride;
  p.B = cache->batch;
  p.Hkv = cache->n_kv_heads;
  p.G = n_q_heads / cache->n_kv_heads;
  p.Lq = n_queries;
  p.cap = cache->capacity;
  p.max_len = max_length;
  p.causal = (causal & ~CORE_KVQ_EXACT_KEYS) != 0;
  p.f16 = dtype == CORE_DTYPE_F16;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out = out;
  p.lse = lse;
  p.status = device_status();
  const kvq::Plan pl = kvq::plan(cache->bits, p.B, p.Hkv, rows, max_length,
                                 (causal & CORE_KVQ_EXACT_KEYS) != 0, false);
  p.n_rt = pl.n_rt;
  p.n_split = pl.n_split;
  Carver c(workspace, workspace_bytes);
  carve_parts(c, pl.n_split, rows * p.B * p.Hkv, &p.part_o, &p.part_lse);
  if (c.overflow) return set_error(CORE_ERR_WORKSPACE, f + ": workspace too small");
  const long long blocks = (long long)p.B * p.Hkv * pl.n_rt * pl.n_split;
  const long long all_rows = rows * p.B * p.Hkv;
  const long long join_blocks = pl.join_rows ? (all_rows + 3) / 4 : all_rows;
  if (blocks > INT_MAX || join_blocks > INT_MAX)
    return set_error(CORE_ERR_UNSUPPORTED, f + ": too many query rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (pl.many)
    e = kvq::launch_many(cache->bits, cache->group, p, blocks, s);
  else if (cache->bits == 4)
    e = cache->group == 32   ? kvq::launch_nt<4, 4>(pl, p, blocks, s)
        : cache->group == 64 ? kvq::launch_nt<4, 2>(pl, p, blocks, s)
                             : kvq::launch_nt<4, 1>(pl, p, blocks, s);
  else
    e = cache->group == 32   ? kvq::launch_nt<8, 4>(pl, p, blocks, s)
        : cache->group == 64 ? kvq::launch_nt<8, 2>(pl, p, blocks, s)
                             : kvq::launch_nt<8, 1>(pl, p, blocks, s);
  if (e != cudaSuccess) return cuda_error(e, pl.many ? "attn_many_kernel launch" : "attn_few_kernel launch");
  if (pl.n_split > 1) {
    // the join may be set up while the parts are still computed: it waits for them
    // on the device
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)join_blocks);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, pl.join_rows ? kvq::attn_join_rows_kernel : kvq::attn_join_kernel, p,
                           pl.many ? kvq::kManyRows : 8 * pl.nt, pl.many ? kvq::kManyTok : kvq::kTok);
    if (e != cudaSuccess) return cuda_error(e, "attn_join_kernel launch");
  }
  return CORE_OK;
}
