// Attention over the quantised KV cache for many query rows a KV head (pieces of
// prompts): tcgen05, with the codes turned into f16 tiles on the way into shared
// memory.
//
// A CTA takes 256 rows of one KV head (rows pack the query heads that share it:
// row = query * G + head), as two tiles of 128, and walks its keys in tiles of
// 128:
//
//   S_x = Q_x K_j^T      128 x 128 x 128 into TMEM
//   P_x = exp2(S_x s log2e - m)   f16, written over S_x in TMEM
//   O_x += P_x V_j       A = P_x from TMEM, B = the V tile (MN-major)
//
// Roles: warps 0-3 and 4-7 run the softmax of tile 0 and 1, one thread a row;
// warps 8-11 read codes from global memory, a tile ahead in registers, and write
// n s + z as swizzled f16 tiles (two K and two V buffers); one thread of warp 12
// issues the MMAs.  The two tiles alternate: while one's softmax runs, the tensor
// cores take the other's P V and next Q K.  Turning codes into f16 costs the same
// for 256 rows as for one, about a quarter of the instructions that the softmax
// of the 256 rows takes.
//
// S_x of tile j + 1 is issued behind P_x V_j, so a full S_x also says that O_x
// holds all earlier tiles: the rare rescale (a maximum that passed by 2^8)
// needs no wait of its own.  Keys and values are rounded to f16 (2^-11), queries
// stay exact behind a power of two per row.
#include <cuda_bf16.h>

#include "attention_quant.cuh"
#include "host_util.h"

namespace core {
namespace kvq {

constexpr int kManyThreads = 512;
constexpr uint32_t kTileB = 128 * kD * 2;  // 32 KB: 128 rows of 128 f16
constexpr uint32_t kAtomB = kTileB / 2;    // 64 channels of the 128 rows

struct ManySmem {
  static constexpr uint32_t kQ = 0;                  // two tiles
  static constexpr uint32_t kK = kQ + 2 * kTileB;    // two buffers
  static constexpr uint32_t kV = kK + 2 * kTileB;
  static constexpr uint32_t kBar = kV + 2 * kTileB;
  static constexpr uint32_t kTotal = kBar + 256;
};

template <int kRegs>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 32 columns stored without waiting (tmem_wait_st before the data is handed on).
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Eight channels of one row: their words' codes as f16 n s + z, in channel order.
template <int kBits>
__device__ __forceinline__ void store_chunk(uint32_t dst, const uint32_t* w, __half2 s, __half2 z) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = as_u32(__hfma2(kBits == 4 ? code_pair<4>(w[0], i) : code_pair<8>(w[i >> 1], i & 1), s, z));
  sts128(dst, h[0], h[1], h[2], h[3]);
}

// One dequantising thread's share of a K tile: rows r0 + 8 i, the 16-byte chunk t
// (8 bits: t and 4 + t) of each.  Lanes that store together hold rows r and r + 4.
template <int kBits, int kG>
struct KeyPiece {
  uint4 c[4][kBits / 4];
  uint32_t m[4][kG];
  __device__ __forceinline__ void load(const AttnParams& p, long long row) {
    const int lane = threadIdx.x & 31, t = lane & 3, w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 32 + (lane >> 3) + (lane & 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 8 * i;
      const uint8_t* src = p.kc + (row + r) * (16 * kBits);
#pragma unroll
      for (int h = 0; h < kBits / 4; ++h)
        c[i][h] = __ldg(reinterpret_cast<const uint4*>(src + ((64u * h + 16u * t) ^ key_swizzle<kBits>(r))));
      const uint32_t* ms = p.km + (row + r) * kG;
      if constexpr (kG == 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(ms));
        m[i][0] = x.x; m[i][1] = x.y; m[i][2] = x.z; m[i][3] = x.w;
      } else if constexpr (kG == 2) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(ms));
        m[i][0] = x.x; m[i][1] = x.y;
      } else {
        m[i][0] = __ldg(ms);
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t tile) const {
    const int lane = threadIdx.x & 31, t = lane & 3, w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 32 + (lane >> 3) + (lane & 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 8 * i;
      const uint32_t rowa = tile + (uint32_t)r * 128u;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t x[2];
        if constexpr (kBits == 4) {
          x[0] = b == 0 ? c[i][0].x : b == 1 ? c[i][0].y : b == 2 ? c[i][0].z : c[i][0].w;
        } else {
          const uint4& u = c[i][b >> 1];
          x[0] = b & 1 ? u.z : u.x;
          x[1] = b & 1 ? u.w : u.y;
        }
        const uint32_t mw = m[i][b * kG / 4];
        store_chunk<kBits>(rowa + (uint32_t)(b >> 1) * kAtomB + ((uint32_t)(((b & 1) * 4 + t) ^ (r & 7)) << 4), x,
                           as_half2(prmt(mw, mw, 0x1010)), as_half2(prmt(mw, mw, 0x3232)));
      }
    }
  }
};

// The same for V: 16 channels of rows r0 + 4 i; a hidden token's row becomes 0.
template <int kBits, int kG>
struct ValuePiece {
  uint32_t c[8][kBits / 2];
  uint32_t m[8];
  __device__ __forceinline__ void load(const AttnParams& p, long long row, const uint8_t* mask, int tok0, int end) {
    const int lane = threadIdx.x & 31, g = (lane & 3) + ((lane >> 1) & 4), w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 32 + ((lane >> 2) & 1) + ((lane >> 3) & 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + 4 * i;
      const uint8_t* src = p.vc + (row + r) * (16 * kBits);
      if constexpr (kBits == 4) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(src + ((8u * g) ^ value_swizzle<4>(r))));
        c[i][0] = x.x; c[i][1] = x.y;
      } else {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(src + ((16u * g) ^ value_swizzle<8>(r))));
        c[i][0] = x.x; c[i][1] = x.y; c[i][2] = x.z; c[i][3] = x.w;
      }
      m[i] = __ldg(p.vm + (row + r) * kG + ((g * kG) >> 3));
      if (tok0 + r >= end || (mask != nullptr && mask[tok0 + r] == 0)) m[i] = 0;
    }
  }
  __device__ __forceinline__ void store(uint32_t tile) const {
    const int lane = threadIdx.x & 31, g = (lane & 3) + ((lane >> 1) & 4), w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 32 + ((lane >> 2) & 1) + ((lane >> 3) & 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + 4 * i;
      const uint32_t rowa = tile + (uint32_t)(g >> 2) * kAtomB + (uint32_t)r * 128u;
      const __half2 s = as_half2(prmt(m[i], m[i], 0x1010)), z = as_half2(prmt(m[i], m[i], 0x3232));
#pragma unroll
      for (int h = 0; h < 2; ++h)
        store_chunk<kBits>(rowa + ((uint32_t)((2 * (g & 3) + h) ^ (r & 7)) << 4), &c[i][h * (kBits / 4)], s, z);
    }
  }
};

template <int kBits, int kG>
__global__ void __launch_bounds__(kManyThreads, 1) attn_many_kernel(const AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t sQ = sbase + ManySmem::kQ, sK = sbase + ManySmem::kK, sV = sbase + ManySmem::kV;
  const uint32_t bar = sbase + ManySmem::kBar;
  auto bar_q_full = [&](int x) { return bar + 8u * x; };
  auto bar_k_full = [&](int s) { return bar + 16 + 8u * s; };
  auto bar_k_empty = [&](int s) { return bar + 32 + 8u * s; };
  auto bar_v_full = [&](int s) { return bar + 48 + 8u * s; };
  auto bar_v_empty = [&](int s) { return bar + 64 + 8u * s; };
  auto bar_s_full = [&](int x) { return bar + 80 + 8u * x; };
  auto bar_p_full = [&](int x) { return bar + 96 + 8u * x; };
  auto bar_o_full = [&](int x) { return bar + 112 + 8u * x; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + ManySmem::kBar + 200);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sgen + ManySmem::kBar + 208);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the last row tiles of every head first: under a causal limit they see most
  const unsigned bh_n = (unsigned)p.B * (unsigned)p.Hkv;
  unsigned u = blockIdx.x;
  const int bh = (int)(u % bh_n);
  u /= bh_n;
  const int split = (int)(u % (unsigned)p.n_split);
  const int rt = p.n_rt - 1 - (int)(u / (unsigned)p.n_split);
  const int b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  const int rows = p.G * p.Lq, row0 = rt * kManyRows;
  const int n_x = rows - row0 > 128 ? 2 : 1;  // row tiles in use

  const int len = sequence_length(p, b);
  const int end = row_limit(p, min(row0 + kManyRows, rows) - 1, len);
  const int per = tiles_per_split(end, kManyTok, p.n_split);
  const int tile0 = split * per, tile1 = min(tile0 + per, (end + kManyTok - 1) / kManyTok);
  const int n = max(tile1 - tile0, 0);
  if (n == 0 && split > 0) return;  // the join does not read this part
  const long long base = (long long)bh * p.cap;
  const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (long long)b * p.mask_stride;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q_full(i), 4);
      mbar_init(bar_k_full(i), 4);
      mbar_init(bar_k_empty(i), 1);
      mbar_init(bar_v_full(i), 4);
      mbar_init(bar_v_empty(i), 1);
      mbar_init(bar_s_full(i), 1);
      mbar_init(bar_p_full(i), 4);
      mbar_init(bar_o_full(i), 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    // S0 [0, 128), S1 [128, 256), O0 [256, 384), O1 [384, 512)
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint32_t bb, uint32_t parity, int where) -> bool {
    return bounded_wait(bb, parity, abort_flag, p.status, where);
  };

  if (warp >= 12) {
    reg_dec<40>();
    if (warp == 12 && lane == 0) {
      constexpr uint32_t idesc_qk = (1u << 4) | ((uint32_t)(kManyTok >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t idesc_pv = idesc_qk | (1u << 16);  // B (the V tile) MN-major
      auto qk = [&](int x, int j) {
        const uint32_t k = sK + (uint32_t)(j & 1) * kTileB, q = sQ + (uint32_t)x * kTileB;
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t off = (uint32_t)(ks >> 2) * kAtomB + (uint32_t)(ks & 3) * 32u;
          mma_bf16(tmem + 128u * x, sdesc_kmajor(q + off), sdesc_kmajor(k + off), idesc_qk, ks > 0 ? 1u : 0u);
        }
        mma_commit(bar_s_full(x));
      };
      bool ok = n > 0;
      for (int x = 0; x < n_x && ok; ++x) ok = wait(bar_q_full(x), 0, 1431);
      if (ok && (ok = wait(bar_k_full(0), 0, 1432))) {
        tc_fence_after();
        for (int x = 0; x < n_x; ++x) qk(x, 0);
        mma_commit(bar_k_empty(0));
      }
      for (int j = 0; j < n && ok; ++j) {
        const bool more = j + 1 < n;
        const int s = j & 1;
        if (more && !(ok = wait(bar_k_full(s ^ 1), (uint32_t)((j + 1) >> 1) & 1u, 1433))) break;
        if (!(ok = wait(bar_v_full(s), (uint32_t)(j >> 1) & 1u, 1434))) break;
        for (int x = 0; x < n_x; ++x) {
          if (!(ok = wait(bar_p_full(x), (uint32_t)j & 1u, 1435))) break;
          tc_fence_after();
          for (int ks = 0; ks < 8; ++ks)
            mma_ts(tmem + 256u + 128u * x, tmem + 128u * x + 8u * ks,
                   sdesc_sw128(sV + (uint32_t)s * kTileB + (uint32_t)ks * 16u * 128u, kAtomB, 1024u), idesc_pv,
                   (j > 0 || ks > 0) ? 1u : 0u);
          if (x == n_x - 1) mma_commit(bar_v_empty(s));
          if (more) {
            qk(x, j + 1);
            if (x == n_x - 1) mma_commit(bar_k_empty(s ^ 1));
          } else {
            mma_commit(bar_o_full(x));
          }
        }
      }
    }
  } else if (warp >= 8) {
    // ---------------- codes to f16 tiles ----------------
    reg_dec<112>();
    KeyPiece<kBits, kG> kp;
    ValuePiece<kBits, kG> vp;
    bool ok = true;
    if (n > 0) {
      kp.load(p, base + (long long)tile0 * kManyTok);
      vp.load(p, base + (long long)tile0 * kManyTok, mask, tile0 * kManyTok, end);
    }
    for (int j = 0; j < n; ++j) {
      const int s = j & 1, next = (tile0 + j + 1) * kManyTok;
      if (j >= 2) ok = __all_sync(0xffffffffu, wait(bar_k_empty(s), (uint32_t)((j >> 1) - 1) & 1u, 1441));
      if (!ok) break;
      kp.store(sK + (uint32_t)s * kTileB);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_k_full(s));
      if (j + 1 < n) kp.load(p, base + next);
      if (j >= 2) ok = __all_sync(0xffffffffu, wait(bar_v_empty(s), (uint32_t)((j >> 1) - 1) & 1u, 1442));
      if (!ok) break;
      vp.store(sV + (uint32_t)s * kTileB);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_v_full(s));
      if (j + 1 < n) vp.load(p, base + next, mask, next, end);
    }
  } else {
    // ---------------- softmax and epilogue: one thread a row ----------------
    reg_inc<176>();
    const int x = warp >> 2;
    if (x < n_x) {
      const int r = (warp & 3) * 32 + lane;  // row of the tile
      const int row = row0 + x * 128 + r;
      const int qi = row / p.G, hq = kvh * p.G + row - qi * p.G;
      const bool live = row < rows;
      const int lim = row_limit(p, row, len);
      const int first = row_limit(p, row0 + x * 128, len);  // every row sees the tokens before
      float sc;
      {
        // Q: f16 behind a power of two, into the swizzled tile
        uint4 v[16];
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + b * p.qb + (long long)hq * p.qh +
                                                          (long long)qi * p.ql);
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          v[c] = live ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = query_pair(w[e], p.f16 != 0);
            mx = fmax3(mx, fabsf(f.x), fabsf(f.y));
          }
        }
        const RowShift sh = row_shift(mx);
        sc = p.scale_log2 * sh.inv1 * sh.inv2;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = query_pair(w[e], p.f16 != 0);
            h[e] = as_u32(__floats2half2_rn(f.x * sh.f1 * sh.f2, f.y * sh.f1 * sh.f2));
          }
          sts128(sQ + (uint32_t)x * kTileB + (uint32_t)(c >> 3) * kAtomB + (uint32_t)r * 128u +
                     ((uint32_t)((c & 7) ^ (r & 7)) << 4),
                 h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q_full(x));
      }
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t tS = lanes + 128u * x, tO = lanes + 256u + 128u * x;
      float m_used = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        const int tok0 = (tile0 + j) * kManyTok;
        uint32_t bits[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (mask != nullptr) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int k = tok0 + 32 * c + lane;
            bits[c] = __ballot_sync(0xffffffffu, k < end && mask[k] != 0);
          }
        }
        const bool full = tok0 + kManyTok <= first && (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu;
        ok = __all_sync(0xffffffffu, wait(bar_s_full(x), (uint32_t)j & 1u, 1451));
        if (!ok) break;
        tc_fence_after();
        float v[4][32];
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld32(tS + 32u * c, v[c]);
          if (!full) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((bits[c] >> e) & 1u) || tok0 + 32 * c + e >= lim) v[c][e] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) mx = fmax3(mx, v[c][e], v[c][e + 1]);
        }
        const float mt = mx * sc;
        const bool raise = mt > m_used + kRaise;
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? ex2_approx(m_used - mt) : 1.0f;
          if (j > 0) {
            l *= f;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float o[32];
              tmem_ld32(tO + 32u * c, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= f;
              tmem_st32(tO + 32u * c, o);
            }
          }
          if (raise) m_used = mt;
        }
        const float neg = m_used == -INFINITY ? 0.f : -m_used;
        const unsigned long long sc2 = f2_pack(sc, sc), neg2 = f2_pack(neg, neg);
        unsigned long long acc = 0ull;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t h[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int k = 64 * c + 2 * e;
            const unsigned long long y = f2_fma(f2_pack(v[k >> 5][k & 31], v[k >> 5][(k & 31) + 1]), sc2, neg2);
            const float p0 = ex2_approx(f2_lo(y)), p1 = ex2_approx(f2_hi(y));
            acc = f2_add(acc, f2_pack(p0, p1));
            h[e] = as_u32(__floats2half2_rn(p0, p1));
          }
          tmem_st32u(tS + 32u * c, h);
        }
        l += f2_lo(acc) + f2_hi(acc);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p_full(x));
      }
      if (n > 0 && ok) ok = __all_sync(0xffffffffu, wait(bar_o_full(x), 0, 1452));
      if (ok) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that saw no token: output 0, LSE -inf
        const float lse2 = l == 0.f ? -INFINITY : m_used + log2f(l);
        const long long part = ((long long)bh * rows + row) * p.n_split + split;
        const int Hq = p.Hkv * p.G;
        float* of = p.n_split > 1 ? p.part_o + part * kD : nullptr;
        uint16_t* oh = static_cast<uint16_t*>(p.out) + (((long long)b * p.Lq + qi) * Hq + hq) * kD;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float o[32];
          if (n > 0) {
            tmem_ld32(tO + 32u * c, o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (!live) continue;
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = l == 0.f ? 0.f : o[e] * inv;
          if (p.n_split > 1) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(of + 32 * c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t h[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (p.f16) {
                  h[k] = as_u32(__floats2half2_rn(o[e + 2 * k], o[e + 2 * k + 1]));
                } else {
                  const __nv_bfloat162 y = __floats2bfloat162_rn(o[e + 2 * k], o[e + 2 * k + 1]);
                  h[k] = *reinterpret_cast<const uint32_t*>(&y);
                }
              }
              *reinterpret_cast<uint4*>(oh + 32 * c + e) = make_uint4(h[0], h[1], h[2], h[3]);
            }
          }
        }
        if (live) {
          if (p.n_split > 1)
            p.part_lse[part] = lse2;
          else
            p.lse[((long long)b * Hq + hq) * p.Lq + qi] = lse2 * 0.69314718055994531f;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

namespace {
template <int kBits, int kG>
cudaError_t launch_one(const AttnParams& p, long long blocks, cudaStream_t s) {
  constexpr uint32_t smem = ManySmem::kTotal + 1024;
  auto kern = attn_many_kernel<kBits, kG>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)blocks, kManyThreads, smem, s>>>(p);
  return cudaGetLastError();
}
}  // namespace

cudaError_t launch_many(int bits, int group, const AttnParams& p, long long blocks, cudaStream_t s) {
  if (bits == 4)
    return group == 32   ? launch_one<4, 4>(p, blocks, s)
           : group == 64 ? launch_one<4, 2>(p, blocks, s)
                         : launch_one<4, 1>(p, blocks, s);
  return group == 32   ? launch_one<8, 4>(p, blocks, s)
         : group == 64 ? launch_one<8, 2>(p, blocks, s)
                       : launch_one<8, 1>(p, blocks, s);
}

}  // namespace kvq
}  // namespace core
