// Attention over the quantised KV cache for many query rows a KV head (pieces of
// prompts): tcgen05, with the codes turned into f16 tiles on the way into shared
// memory.
//
// A CTA takes 256 rows of one KV head (rows pack the query heads that share it:
// row = query * G + head), as two tiles of 128, and walks its keys in tiles of 128:
//
//   S   = Q_x K_j^T      128 x 128 x 128 into TMEM, one buffer for both row tiles
//   P_x = exp2(S s log2e - m)     f16, into TMEM
//   O_x += P_x V_j       A = P_x from TMEM, B = the V tile (MN-major)
//
// TMEM holds O_0, O_1 (256 columns), S (128), P_0 and P_1 (64 each).  A softmax
// thread takes its row of S into registers at once and gives the buffer up, so
// the other row tile's scores are computed while it works, and its own next ones
// are there when it is done: softmax and tensor cores run side by side.  (S and P
// of a row tile in one buffer made softmax, P V and Q K^T follow one another,
// 4650 cycles a pair of tiles against 3500 now; 64-key tiles with two buffers each
// ran into M 128 x N 64 products taking as long as N 128 ones.)
//
// Roles: warps 0-3 and 4-7 run the softmax of row tile 0 and 1, one thread a row;
// warps 8-11 turn codes into the swizzled f16 tiles of K, warps 12-15 those of V
// (two buffers each; the codes come 64 tokens ahead in registers); warp 16 issues
// Q K^T, warp 17 P V.  Turning codes into f16 costs the same for 256 rows as for
// one, about a third of the instructions that the softmax of the 256 rows takes.
// With four warps for K and V together that work was the longest chain whenever
// the codes came from HBM, and the time hung on how far ahead the compiler happened
// to ask for them (475 to 590 us for 2048 queries over 16384 tokens; 492-522 now,
// in every format).
//
// What bounds it now: 512 queries (2048 rows a head) over 16384 tokens take 149 us,
// join included, 910 TFLOP/s, and 2048 queries 486 us, 1.06 PFLOP/s of the measured
// 1.65.  A pair of tiles takes about 3500 cycles, of which the MMAs need 2048: Q K^T
// reads 128 bytes of shared memory a cycle, all there are, and shares them with the
// tiles' writing; the rest is the way of S from tensor core to registers and back.  The
// softmax spills (116-120 bytes of stores in the six builds: 128 scores of a row and
// their state against 168 registers).
//
// Keys and values are rounded to f16 (2^-11; bf16 would lose three more bits), queries
// stay exact, behind a power of two per row, down to 2^-21 of the row's largest, P is f16
// (2^7 at the running maximum, at most 2^14), sums and statistics are f32.  O_x is
// rescaled only when a score passes the maximum that it was scaled with by 2^7.
#include <cuda_bf16.h>

#include "attention_quant.cuh"
#include "host_util.h"

namespace core {
namespace kvq {

constexpr int kManyThreads = 640;
constexpr uint32_t kTile = 128 * kD * 2;  // 32 KB: 128 rows (queries or tokens) of 128 f16
constexpr uint32_t kAtom = kTile / 2;     // 64 channels of the rows
constexpr uint32_t kHalf = 64 * 128;      // 64 rows of an atom

struct ManySmem {
  static constexpr uint32_t kQ = 0;               // two tiles
  static constexpr uint32_t kK = kQ + 2 * kTile;  // two buffers
  static constexpr uint32_t kV = kK + 2 * kTile;
  static constexpr uint32_t kBar = kV + 2 * kTile;
  static constexpr uint32_t kTotal = kBar + 512;
};
// TMEM columns
constexpr uint32_t kColO = 0, kColS = 256, kColP = 384;

template <int kRegs>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
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
// 32 lanes x 16 columns (store and wait).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 lanes x 128 columns.  Both loads and their wait are one statement: the registers
// hold nothing before the wait, and between statements the compiler may copy or spill
// them.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&v)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
      "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%129];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      :
        "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63]),
        "=f"(v[64]), "=f"(v[65]), "=f"(v[66]), "=f"(v[67]), "=f"(v[68]), "=f"(v[69]), "=f"(v[70]), "=f"(v[71]),
        "=f"(v[72]), "=f"(v[73]), "=f"(v[74]), "=f"(v[75]), "=f"(v[76]), "=f"(v[77]), "=f"(v[78]), "=f"(v[79]),
        "=f"(v[80]), "=f"(v[81]), "=f"(v[82]), "=f"(v[83]), "=f"(v[84]), "=f"(v[85]), "=f"(v[86]), "=f"(v[87]),
        "=f"(v[88]), "=f"(v[89]), "=f"(v[90]), "=f"(v[91]), "=f"(v[92]), "=f"(v[93]), "=f"(v[94]), "=f"(v[95]),
        "=f"(v[96]), "=f"(v[97]), "=f"(v[98]), "=f"(v[99]), "=f"(v[100]), "=f"(v[101]), "=f"(v[102]), "=f"(v[103]),
        "=f"(v[104]), "=f"(v[105]), "=f"(v[106]), "=f"(v[107]), "=f"(v[108]), "=f"(v[109]), "=f"(v[110]), "=f"(v[111]),
        "=f"(v[112]), "=f"(v[113]), "=f"(v[114]), "=f"(v[115]), "=f"(v[116]), "=f"(v[117]), "=f"(v[118]), "=f"(v[119]),
        "=f"(v[120]), "=f"(v[121]), "=f"(v[122]), "=f"(v[123]), "=f"(v[124]), "=f"(v[125]), "=f"(v[126]), "=f"(v[127])
      : "r"(taddr), "r"(taddr + 64u)
      : "memory");
}

// Loads that stay where they are written: the compiler would otherwise sink them
// to their first use, a tile later, and leave their latency in the open.
__device__ __forceinline__ uint4 ldg128(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg64(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ldg32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ldg8(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

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

// One thread's share of 64 tokens of K: rows r0 + 8 i, the 16-byte chunk t
// (8 bits: t and 4 + t) of each.  Lanes that store together hold rows r and r + 4.
template <int kBits, int kG>
struct KeyPiece {
  uint4 c[2][kBits / 4];
  uint32_t m[2][kG];
  __device__ __forceinline__ void load(const AttnParams& p, long long row) {
    const int lane = threadIdx.x & 31, t = lane & 3, w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 16 + (lane >> 3) + (lane & 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + 8 * i;
      const uint8_t* src = p.kc + (row + r) * (16 * kBits);
#pragma unroll
      for (int h = 0; h < kBits / 4; ++h)
        c[i][h] = ldg128(src + ((64u * h + 16u * t) ^ key_swizzle<kBits>(r)));
      const uint32_t* ms = p.km + (row + r) * kG;
      if constexpr (kG == 4) {
        const uint4 x = ldg128(ms);
        m[i][0] = x.x; m[i][1] = x.y; m[i][2] = x.z; m[i][3] = x.w;
      } else if constexpr (kG == 2) {
        const uint2 x = ldg64(ms);
        m[i][0] = x.x; m[i][1] = x.y;
      } else {
        m[i][0] = ldg32(ms);
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t tile) const {
    const int lane = threadIdx.x & 31, t = lane & 3, w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 16 + (lane >> 3) + (lane & 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
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
        store_chunk<kBits>(rowa + (uint32_t)(b >> 1) * kAtom + ((uint32_t)(((b & 1) * 4 + t) ^ (r & 7)) << 4), x,
                           as_half2(prmt(mw, mw, 0x1010)), as_half2(prmt(mw, mw, 0x3232)));
      }
    }
  }
};

// The same for V: 16 channels of rows r0 + 4 i; a hidden token's row becomes 0.
template <int kBits, int kG>
struct ValuePiece {
  uint32_t c[4][kBits / 2];
  uint32_t m[4], seen[4];
  __device__ __forceinline__ void load(const AttnParams& p, long long row, const uint8_t* mask, int tok0, int end) {
    const int lane = threadIdx.x & 31, g = (lane & 3) + ((lane >> 1) & 4), w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 16 + ((lane >> 2) & 1) + ((lane >> 3) & 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 4 * i;
      const uint8_t* src = p.vc + (row + r) * (16 * kBits);
      if constexpr (kBits == 4) {
        const uint2 x = ldg64(src + ((8u * g) ^ value_swizzle<4>(r)));
        c[i][0] = x.x; c[i][1] = x.y;
      } else {
        const uint4 x = ldg128(src + ((16u * g) ^ value_swizzle<8>(r)));
        c[i][0] = x.x; c[i][1] = x.y; c[i][2] = x.z; c[i][3] = x.w;
      }
      m[i] = ldg32(p.vm + (row + r) * kG + ((g * kG) >> 3));
      seen[i] = tok0 + r >= end ? 0u : mask == nullptr ? 1u : ldg8(mask + tok0 + r);
    }
  }
  __device__ __forceinline__ void store(uint32_t tile) const {
    const int lane = threadIdx.x & 31, g = (lane & 3) + ((lane >> 1) & 4), w = (threadIdx.x >> 5) & 3;
    const int r0 = w * 16 + ((lane >> 2) & 1) + ((lane >> 3) & 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 4 * i;
      const uint32_t rowa = tile + (uint32_t)(g >> 2) * kAtom + (uint32_t)r * 128u;
      const uint32_t mw = seen[i] ? m[i] : 0u;
      const __half2 s = as_half2(prmt(mw, mw, 0x1010)), z = as_half2(prmt(mw, mw, 0x3232));
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
  auto bar_s_full = [&](int x) { return bar + 80 + 8u * x; };   // S holds row tile x's scores
  auto bar_s_taken = [&](int x) { return bar + 96 + 8u * x; };  // they are in registers
  auto bar_p_full = [&](int x) { return bar + 112 + 8u * x; };
  auto bar_pv = [&](int x) { return bar + 128 + 8u * x; };
  auto bar_last = [&](int w) { return bar + 144 + 8u * w; };  // an MMA warp that gives up: its products are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + ManySmem::kBar + 400);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sgen + ManySmem::kBar + 408);

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
  if (p.n_split > 1) launch_dependents();
  if (n == 0 && split > 0) return;  // the join does not read this part
  const long long base = (long long)bh * p.cap;
  const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (long long)b * p.mask_stride;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q_full(i), 4);
      mbar_init(bar_k_full(i), 8);  // four warps, two halves
      mbar_init(bar_k_empty(i), 1);
      mbar_init(bar_v_full(i), 8);
      mbar_init(bar_v_empty(i), 1);
      mbar_init(bar_s_full(i), 1);
      mbar_init(bar_s_taken(i), 4);
      mbar_init(bar_p_full(i), 4);
      mbar_init(bar_pv(i), 1);
      mbar_init(bar_last(i), 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns are this CTA's, so they start at column 0, lane 0: the address
  // is a constant, and anything else an error.
  constexpr uint32_t tmem = 0;
  if (threadIdx.x == 0 && *tmem_slot != 0) {
    record_error(p.status, CORE_ERR_CUDA, 1430, (int)*tmem_slot);
    *abort_flag = 1;
  }
  auto wait = [&](uint32_t bb, uint32_t parity, int where) -> bool {
    return bounded_wait(bb, parity, abort_flag, p.status, where);
  };

  if (warp >= 16) {
    reg_dec<32>();
    // Two warps issue the MMAs, Q K^T and P V each in its own order, so that
    // neither waits behind the other's barriers.  A whole warp walks the tiles and
    // one elected lane issues: addresses and descriptors then stay in uniform
    // registers, where the MMAs take them (82 cycles an MMA before, 65 now).
    auto all = [&](uint32_t bb, uint32_t parity, int where) -> bool {
      const bool got = __all_sync(0xffffffffu, wait(bb, parity, where));
      tc_fence_after();
      return got;
    };
    bool ok = n > 0;
    const bool leader = elect_one();
    if (warp == 16) {
      constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kManyTok >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      for (int j = 0; j < n && ok; ++j) {
        if (!(ok = all(bar_k_full(j & 1), (uint32_t)(j >> 1) & 1u, 1431))) break;
        const uint64_t kd = sdesc_kmajor(sK + (uint32_t)(j & 1) * kTile);
        for (int x = 0; x < n_x; ++x) {
          if (j == 0 && !(ok = all(bar_q_full(x), 0, 1432))) break;
          // S is free when the row tile before this one has taken its scores
          const int prev = x > 0 ? 0 : n_x - 1, when = x > 0 ? j : j - 1;
          if (when >= 0 && !(ok = all(bar_s_taken(prev), (uint32_t)when & 1u, 1433))) break;
          const uint64_t qd = sdesc_kmajor(sQ + (uint32_t)x * kTile);
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
              const uint32_t off = ((uint32_t)(ks >> 2) * kAtom + (uint32_t)(ks & 3) * 32u) / 16;
              mma_bf16(tmem + kColS, qd + off, kd + off, idesc, ks > 0 ? 1u : 0u);
            }
            mma_commit(bar_s_full(x));
            if (x == n_x - 1) mma_commit(bar_k_empty(j & 1));
          }
          __syncwarp();
        }
      }
    } else if (warp == 17) {
      constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24) |
                                 (1u << 16);  // B (the V tile) MN-major
      for (int j = 0; j < n && ok; ++j) {
        if (!(ok = all(bar_v_full(j & 1), (uint32_t)(j >> 1) & 1u, 1434))) break;
        const uint64_t vd = sdesc_sw128(sV + (uint32_t)(j & 1) * kTile, kAtom, 1024u);
        for (int x = 0; x < n_x; ++x) {
          if (!(ok = all(bar_p_full(x), (uint32_t)j & 1u, 1435))) break;
          const uint32_t a = tmem + kColP + 64u * x, d = tmem + kColO + 128u * x;
          if (leader) {
            mma_ts(d, a, vd, idesc, j > 0 ? 1u : 0u);
#pragma unroll
            for (int ks = 1; ks < 8; ++ks) mma_ts(d, a + 8u * ks, vd + ks * 16 * 128 / 16, idesc, 1u);
            mma_commit(bar_pv(x));
            if (x == n_x - 1) mma_commit(bar_v_empty(j & 1));
          }
          __syncwarp();
        }
      }
    }
    if (!ok && n > 0) {  // given up: no product may be in flight when TMEM is freed
      if (leader) mma_commit(bar_last(warp - 16));
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(bar_last(warp - 16), 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
  } else if (warp >= 8) {
    // ---------------- codes to f16 tiles: K warps 8-11, V warps 12-15 ----------------
    reg_dec<56>();
    bool ok = true;
    const int first = tile0 * kManyTok;  // 64 tokens at a time, the next ones in registers
    auto put = [&](auto& piece, int i, uint32_t tiles, uint32_t empty, uint32_t full, auto&& get) -> bool {
      const uint32_t s = (uint32_t)(i >> 1) & 1u;
      if (i >= 4 && (i & 1) == 0) ok = __all_sync(0xffffffffu, wait(empty + 8u * s, (uint32_t)((i >> 2) - 1) & 1u, 1441));
      if (!ok) return false;
      piece.store(tiles + s * kTile + (uint32_t)(i & 1) * kHalf);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + 8u * s);
      if (i + 1 < 2 * n) get(i + 1);
      return true;
    };
    if (n > 0 && warp < 12) {
      KeyPiece<kBits, kG> piece;
      auto get = [&](int i) { piece.load(p, base + first + i * 64); };
      get(0);
      for (int i = 0; i < 2 * n; ++i)
        if (!put(piece, i, sK, bar_k_empty(0), bar_k_full(0), get)) break;
    } else if (n > 0) {
      ValuePiece<kBits, kG> piece;
      auto get = [&](int i) { piece.load(p, base + first + i * 64, mask, first + i * 64, end); };
      get(0);
      for (int i = 0; i < 2 * n; ++i)
        if (!put(piece, i, sV, bar_v_empty(0), bar_v_full(0), get)) break;
    }
  } else {
    // ---------------- softmax and epilogue: one thread a row ----------------
    reg_inc<168>();
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
          sts128(sQ + (uint32_t)x * kTile + (uint32_t)(c >> 3) * kAtom + (uint32_t)r * 128u +
                     ((uint32_t)((c & 7) ^ (r & 7)) << 4),
                 h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q_full(x));
      }
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t tS = lanes + kColS, tP = lanes + kColP + 64u * x, tO = lanes + kColO + 128u * x;
      const unsigned long long sc2 = f2_pack(sc, sc);
      float anchor = -INFINITY, l = 0.f;
      bool ok = true;
      // a tile's mask is asked for while the tile before it is worked on
      uint32_t seen[4] = {1u, 1u, 1u, 1u};
      auto look = [&](int j) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int k = (tile0 + j) * kManyTok + 32 * c + lane;
          seen[c] = j < n && k < end ? ldg8(mask + k) : 0u;
        }
      };
      if (mask != nullptr) look(0);
      for (int j = 0; j < n; ++j) {
        const int tok0 = (tile0 + j) * kManyTok;
        uint32_t bits[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (mask != nullptr) {
#pragma unroll
          for (int c = 0; c < 4; ++c) bits[c] = __ballot_sync(0xffffffffu, seen[c] != 0);
          look(j + 1);
        }
        const bool full = tok0 + kManyTok <= first && (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu;
        ok = __all_sync(0xffffffffu, wait(bar_s_full(x), (uint32_t)j & 1u, 1451));
        if (!ok) break;
        tc_fence_after();
        float v[128];
        tmem_ld128(tS, v);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_s_taken(x));
        if (!full) {
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (!((bits[e >> 5] >> (e & 31)) & 1u) || tok0 + e >= lim) v[e] = -INFINITY;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 128; e += 8) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = fmax3(mx[c], v[e + 2 * c], v[e + 2 * c + 1]);
        }
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        const bool raise = mt - anchor > kTop;
        // O_x holds every earlier tile, and P_x may be written again, once the last
        // P V has landed
        auto last_pv = [&]() -> bool {
          const bool got = j == 0 || wait(bar_pv(x), (uint32_t)(j - 1) & 1u, 1452);
          tc_fence_after();
          return __all_sync(0xffffffffu, got);
        };
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? ex2_approx(anchor - (mt - kLift)) : 1.0f;
          if (j > 0) {
            if (!(ok = last_pv())) break;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              float o[16];
              tmem_ld16(tO + 16u * c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              tmem_st16(tO + 16u * c, o);
            }
          }
          if (raise) anchor = mt - kLift;
        }
        const float neg = anchor == -INFINITY ? 0.f : -anchor;
        const unsigned long long neg2 = f2_pack(neg, neg);
        unsigned long long acc = 0ull;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t h[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const unsigned long long y = f2_fma(f2_pack(v[64 * c + 2 * e], v[64 * c + 2 * e + 1]), sc2, neg2);
            const float p0 = ex2_approx(f2_lo(y)), p1 = ex2_approx(f2_hi(y));
            acc = f2_add(acc, f2_pack(p0, p1));
            h[e] = as_u32(__floats2half2_rn(p0, p1));
          }
          if (c == 0 && !(ok = last_pv())) break;
          tmem_st32u(tP + 32u * c, h);
        }
        if (!ok) break;
        l += f2_lo(acc) + f2_hi(acc);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p_full(x));
      }
      if (n > 0 && ok) ok = __all_sync(0xffffffffu, wait(bar_pv(x), (uint32_t)(n - 1) & 1u, 1453));
      if (ok) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that saw no token: output 0, LSE -inf
        const float lse2 = l == 0.f ? -INFINITY : anchor + log2f(l);
        const long long part = ((long long)bh * rows + row) * p.n_split + split;
        const int Hq = p.Hkv * p.G;
        float* of = p.n_split > 1 ? p.part_o + part * kD : nullptr;
        uint16_t* oh = static_cast<uint16_t*>(p.out) + (((long long)b * p.Lq + qi) * Hq + hq) * kD;
        // all of O before rows past the end part from their warp: the loads take all of it
        float o[128];
        if (n > 0) {
          tmem_ld128(tO, o);
        } else {
#pragma unroll
          for (int e = 0; e < 128; ++e) o[e] = 0.f;
        }
        if (live && p.n_split > 1) {
#pragma unroll
          for (int e = 0; e < 128; e += 4)
            *reinterpret_cast<float4*>(of + e) =
                l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                         : make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
        } else if (live) {
#pragma unroll
          for (int e = 0; e < 128; e += 8) {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float x0 = l == 0.f ? 0.f : o[e + 2 * k] * inv, x1 = l == 0.f ? 0.f : o[e + 2 * k + 1] * inv;
              if (p.f16) {
                h[k] = as_u32(__floats2half2_rn(x0, x1));
              } else {
                const __nv_bfloat162 y = __floats2bfloat162_rn(x0, x1);
                h[k] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
            *reinterpret_cast<uint4*>(oh + e) = make_uint4(h[0], h[1], h[2], h[3]);
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
  if (warp == 16) {
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
