// Softmax cross entropy of an output head over its whole vocabulary, from the hidden states, with its gradients.
//
//   l[t, v] = h_t . w_v,   lse_t = log sum_v exp l[t, v],   nll_t = lse_t - l[t, y_t]
//   d[t, v] = g_t (exp(l[t, v] - lse_t) - [v = y_t]),   dH = d W,   dW = d^T H
//
// The forward product reduces each 128 columns of a token's logits to (max, sum of exp) in its epilogue and takes the
// label's logit out on the way; a second kernel joins them in order, nll = log1p(sum_{v != y} exp(l_v - l_y)), which
// keeps its digits where the label is nearly certain, and with it d[t, y] = g expm1(-nll).  The logits are not stored.  Where the caller has
// room for them, the first columns' distances below the largest of their 128 columns are kept for the backward pass, in
// 16 bits (log2 units, steps of 2^-11: exp(l) within 2^-12.5 of itself down to 2^-32 of the largest, nothing below that; a
// bf16 exponential would have rounded d a second time by 2^-9).  They save a quarter of a training step's products for two bytes an
// entry.  The backward pass takes the vocabulary in pieces: the kept columns first, then pieces whose logits it computes
// again, with d in 16 bits as the epilogue's result; it multiplies a piece's d with its rows of W (dH, summed over the
// pieces in FP32) and with H (dW's rows of the piece).  Every sum runs in a fixed order, so results repeat bit for bit.
//
// d is held as 2^k d / u, with u = max|g| (or g itself where all tokens share it), in units of its largest possible
// magnitude, and the products take the factor back in FP32: in f16 (k = 15) probabilities down to 2^-39 then stay normal
// numbers, whatever the mean divides by; bf16 has the exponent range and takes k = 0.  Rounding d to 16 bits costs each
// of its entries 2^-9 (bf16) or 2^-12 (f16) of itself, no more than the rounding of the gradients to the same type.
//
// At 8192 x 128256 x 4096 the three products run at 1355 to 1415 TFLOP/s, sustained under the card's power limit (a
// plain library product of these sizes: 1281 to 1500); the step takes 21.5 ms.
//
// Few tokens take the narrow side of the products: the weights fill the 256 rows of a tile and the tokens its columns, 16
// at least.  As rows, T tokens would still cost the tensor cores 256 rows: 1 x 128256 x 4096 is bound by reading W, but
// drew the full 1000 W doing so, which lowered the clock to 1.1 GHz and W to 4.1 TB/s.  The limits were measured,
// sustained, at 128256 x 4096 (us, few against many): scores of 32 tokens 172 and 224, of 64 185 and 246, of 96 212 and
// 223 (a step's three products then gain nothing); dH of 64 tokens 197 and 234, of 128 219 and 238, of 192 249 and 258
// (but a whole step of 190 tokens 903 and 837).
//
// A label equal to `ignore` does not count: nll 0, d 0.  A label outside the vocabulary makes the token's nll and its
// d NaN; no memory is read for it.
#include <algorithm>
#include <cmath>
#include <cuda_bf16.h>
#include "umma.cuh"

namespace mpq {
namespace xent {

using namespace tc;

// A tile is 256 x 256, computed by a pair of CTAs: each holds 128 rows of A, 128 of B and 128 rows of the accumulator.
constexpr int kEpiWarps = 8, kThreads = 64 + 32 * kEpiWarps;
constexpr int kBM = 256, kBN = 256, kGroup = 16;
constexpr uint32_t kRingBytes = 192 * 1024;
constexpr int kMostStages = 11;  // of 16 KB of one operand and 1 KB of the other
constexpr int kFewScored = 64, kFewGrads = 128;
// k-blocks that the forward pass accumulates before it adds in FP32.  Over drawn sizes the scores were off by at most
// 7e-7 of themselves in bf16 at 8; in f16, whose products have more bits to lose, by 1.1e-6 at 8 and 6e-7 at 4 (time of
// 2047 x 151936 x 1024: 475 us at 8, 520 at 4, 575 at 2).
constexpr int kChunkBf16 = 8, kChunkF16 = 4;
constexpr float kLog2e = 1.4426950408889634f;

enum { kLse = 0, kGrad = 1, kOut = 2 };

constexpr int kTimedOut = 20;  // added to the code of a wait that ran out: whose it was

struct Args {
  int M, N, K, mt, nt;      // C[M, N] over K; mt x nt tiles
  int splits;               // parts of K; more than one only with `acc`
  int tile_out;             // the result's rows are aligned for tile stores
  int a_rows, b_rows;       // rows of A and of B that a CTA loads
  int tile_n;               // columns of a tile (256, or the tokens' 16 .. 128)
  int stages;               // of the ring, each (a_rows + b_rows) x 128 bytes
  int chunk;                // kLse: k-blocks to an accumulator
  int f16;                  // 1: f16 operands, 0: bf16
  int* status;
  // kLse, kGrad
  const int64_t* labels;
  int64_t ignore;
  int vocab;                // labels in [0, vocab) count
  int v0;                   // first column's vocabulary index
  float2* part;             // kLse: [tokens, parts] (max, sum of exp(l - max)) of 128 columns each, 32 if few
  int parts;
  float* tgt;               // kLse: [M] the label's logit; kGrad: its score
  uint16_t* keep;           // kLse: distances of the columns below keep_cols (a multiple of 256, or V), [tokens, ldk]
  int64_t ldk;
  int keep_cols;
  const float* lse;         // kGrad: [M]
  const float* gout;        // kGrad: upstream gradient, gout[t * gstride]
  int gstride;
  const float* count;       // kGrad: divides g where given (the mean's number of labels)
  const float* gmax;        // kGrad, kOut: largest finite |g| of the counted tokens; null: all share g
  // kGrad, kOut
  void* out;
  int64_t ldo;
  float* acc;               // kOut: FP32 planes [splits, M, N], one for each part of K; null: C goes straight to `out`
};

// MN-major operand in the 128B-swizzled layout: 64 elements of the row dimension to a 128-byte line, one line for each
// k, eight lines to a 1024-byte atom (SBO: next eight k), 64-element groups 8192 bytes apart (LBO).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ uint32_t idesc16(int f16, bool a_mn, bool b_mn, int m, int n) {
  const uint32_t fmt = f16 ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A token's factor in d, in units of unit_of(), and that unit.
__device__ __forceinline__ float factor_of(bool inside, const float* gout, int64_t at, const float* count,
                                           const float* gmax, int f16) {
  const float top = f16 ? 32768.f : 1.f;
  if (!inside) return __int_as_float(0x7fc00000);
  if (!gmax) return top;
  const float g = count ? gout[at] / *count : gout[at];
  return *gmax == 0.f && g == 0.f ? 0.f : g / *gmax * top;
}
__device__ __forceinline__ float unit_of(const float* gout, const float* count, const float* gmax, int f16) {
  const float u = gmax ? *gmax : (count ? (*count > 0.f ? *gout / *count : 0.f) : *gout);
  return f16 ? u * (1.f / 32768.f) : u;
}

// Unit u -> its tile and range of k-blocks.  The raster walks kGroup row tiles down before it takes the next column
// tile: the tiles in flight share a few row tiles (kept in L2) and stream the columns once for each group.
__device__ __forceinline__ void unit_at(int u, const Args& p, int kblocks, int& mb, int& nb, int& k0, int& k1) {
  int t = u, s = 0;
  k0 = 0;
  k1 = kblocks;
  if (p.splits > 1) {
    t = u / p.splits;
    s = u - t * p.splits;
    k0 = (int)((int64_t)kblocks * s / p.splits);
    k1 = (int)((int64_t)kblocks * (s + 1) / p.splits);
  }
  const int per = kGroup * p.nt, g = t / per, r = t - g * per;
  const int rows = min(kGroup, p.mt - g * kGroup);
  nb = r / rows;
  mb = g * kGroup + r - nb * rows;
}

// 64 16-bit values (32 words) of each of a warp's rows from (row0, col) on, `lim` columns wanted: as a tile, or row by
// row where the result's rows are not aligned.
__device__ __forceinline__ void store_half_rows(const Args& p, const CUtensorMap* map, unsigned char* buf, int lane,
                                                int row0, int col, uint16_t* out, int64_t ld, const uint32_t (&w)[32],
                                                int lim) {
  if (lim <= 0 || row0 >= p.M) return;  // the same for the warp
  chunk_put(buf, lane, w);
  if (p.tile_out)
    chunk_send(buf, lane, map, col, row0, 0);
  else
    chunk_rows<2>(buf, lane, out + row0 * ld + col, ld * 2, p.M - row0, lim);
}

// 2^t in one instruction (denormal results become 0, 2^-22 relative)
__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// Largest of a warp's values, NaN if one is: order-preserving whole numbers for the integer reduction.
__device__ __forceinline__ float warp_max(float v) {
  const int b = __float_as_int(v);
  const int m = __reduce_max_sync(0xffffffffu, b ^ ((b >> 31) & 0x7fffffff));
  return __int_as_float(m ^ ((m >> 31) & 0x7fffffff));
}

// Kept distances of t = l - max <= 0, in steps of 1 / kStep log2 units.  The sum with 2^23 rounds to a whole number, whose
// bits end the mantissa.  Maxima stay in the logits' own units: t is exactly 0 for the maximum itself and never above it
// (the difference to a maximum rounded in log2 units was, by 2^-24 of it), and no logit is too large for log2 units.
constexpr float kStep = 2048.f;
__device__ __forceinline__ uint32_t distance_bits(float t) {
  return __float_as_uint(fminf(fmaf(t, -kStep * kLog2e, 8388608.f), 8388608.f + 65535.f));
}

// C[M, N] = A B with an epilogue.  A K-major: [M, K] rows; A_MN: [K, M] rows.  B likewise ([N, K] or [K, N] rows).
// 16-bit operands, FP32 accumulation in TMEM.  Persistent pairs of CTAs walk the 256 x 256 tiles (or, with `splits`,
// a K range of a tile); in each CTA warp 0 loads its halves of the operands by TMA into a ring, warps 2..9 are the
// epilogue, a row and 128 columns to a thread; warp 1 of the first CTA issues the MMAs of both (M = 256, N = 256,
// tcgen05 cta_group::2), so that each CTA's shared memory feeds 128 columns of B instead of 256.  Two accumulators let
// the epilogue overlap the next tile's MMAs.  (A tile of 512 columns, which halves A's loads but fills TMEM, gained
// nothing once the MMAs were issued fast enough: 6075 us against 6970 for dH at 8192 x 128256 x 4096.)
//
// With at most 128 rows of A only those are loaded: a tile load takes two to three cycles a 128-byte row, and 128 rows of
// zeros would cost as much as the columns of B that bound such a product (1 x 128256 x 4096: 263 us with them, 209
// without), and the ring takes more stages for it.  What the other rows' shared memory holds stays in their rows of
// the accumulator.
//
// The tensor core's FP32 accumulator truncates, and a score is a small difference of sums of H products; so the
// forward pass (kLse) accumulates p.chunk k-blocks at a time and adds these to nearest in registers.
//
// FEW: A is the weights' side and B the tokens', one tile of p.tile_n columns; a thread holds a vocabulary row (kLse) or
// a column of dH (kOut) for half of the tokens.
template <int EPI, bool A_MN, bool B_MN, bool FEW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_xent_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_o, const Args p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* out_buf = ring + kRingBytes;  // 4 KB to an epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(out_buf + kEpiWarps * 4096);
  uint64_t* empty = full + kMostStages;
  uint64_t* acc_full = empty + kMostStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // the full operand of a stage comes first: what the MMA reads beyond a short A belongs to this kernel's memory
  const uint32_t stage = (p.a_rows + p.b_rows) * 128;
  const uint32_t lead_a = FEW ? 0 : p.b_rows * 128, lead_b = FEW ? p.a_rows * 128 : 0;
  auto s_b = [&](int s) { return ring + s * stage + lead_b; };
  auto s_a = [&](int s) { return ring + s * stage + lead_a; };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), pairs = gridDim.x >> 1;
  const int kblocks = (p.K + 63) / 64, units = p.mt * p.nt * p.splits;
  allow_behind();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before any is signalled
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  wait_before();  // operands, scalars and workspaces may be those of the kernel before

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t bar0 = mapa(smem_u32(full), 0);
      int64_t it = 0;
      Ring r(p.stages);
      bool ok = true;
      for (int u = blockIdx.x >> 1; u < units && ok; u += pairs) {
        int mb, nb, k0, k1;
        unit_at(u, p, kblocks, mb, nb, k0, k1);
        const int row_a = mb * kBM + rank * 128, row_b = nb * kBN + rank * p.b_rows;
        for (int kb = k0; kb < k1; ++kb, ++it, r.next()) {
          if (!mbar_wait_cluster(&empty[r.s], r.ph ^ 1u) || *abort_flag) {
            ok = false;
            break;
          }
          // both CTAs' bytes count on the first one's barrier (a peer's copy may land before the expectation)
          if (rank == 0) mbar_expect_tx(&full[r.s], 2 * stage);
          const uint32_t bar = bar0 + r.s * 8;
          if constexpr (A_MN) {
            tma_load_2d_pair(s_a(r.s), &map_a, bar, row_a, kb * 64);
            tma_load_2d_pair(s_a(r.s) + 8192, &map_a, bar, row_a + 64, kb * 64);
          } else {
            tma_load_2d_pair(s_a(r.s), &map_a, bar, kb * 64, row_a);
          }
          if constexpr (B_MN) {
            tma_load_2d_pair(s_b(r.s), &map_b, bar, row_b, kb * 64);
            tma_load_2d_pair(s_b(r.s) + 8192, &map_b, bar, row_b + 64, kb * 64);
          } else {
            tma_load_2d_pair(s_b(r.s), &map_b, bar, kb * 64, row_b);
          }
        }
      }
      if (!ok) {  // drain the copies in flight (each wait bounded); the peer leaves only after the cluster barrier
        *abort_flag = 1;
        for (int i = 0; rank == 0 && i < p.stages && i < it; ++i) {
          r.back();
          mbar_wait_cluster(&full[r.s], r.ph);
        }
        atomicCAS(p.status, 0, kTimedOut + 2);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool lead = elect_one();
      const uint32_t idesc = idesc16(p.f16, A_MN, B_MN, kBM, p.tile_n);
      const uint64_t da0 = A_MN ? smem_desc_mn_sw128(smem_u32(s_a(0))) : smem_desc_k_sw128(smem_u32(s_a(0)));
      const uint64_t db0 = B_MN ? smem_desc_mn_sw128(smem_u32(s_b(0))) : smem_desc_k_sw128(smem_u32(s_b(0)));
      constexpr uint32_t kStepA = A_MN ? 2048 : 32, kStepB = B_MN ? 2048 : 32;  // K = 16: 16 lines, or 32 bytes of a line
      const int chunk = EPI == kLse ? p.chunk : kblocks;
      Ring r(p.stages);
      bool ok = true;
      int n = 0;  // accumulators handed over
      for (int u = blockIdx.x >> 1; u < units && ok; u += pairs) {
        int mb, nb, k0, k1;
        unit_at(u, p, kblocks, mb, nb, k0, k1);
        for (int kc = k0; kc < k1 && ok; kc += chunk, ++n) {
          const int ke = min(k1, kc + chunk), b = n & 1;
          if (!warp_agrees(mbar_wait_cluster(&acc_empty[b], ((uint32_t)(n >> 1) & 1u) ^ 1u))) {
            ok = false;
            break;
          }
          for (int kb = kc; kb < ke; ++kb, r.next()) {
            if (!warp_agrees(mbar_wait_cluster(&full[r.s], r.ph) && !*abort_flag)) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t da = desc_add(da0, r.s * stage), db = desc_add(db0, r.s * stage);
            const uint32_t add = kb > kc;
            if (lead) {
              #pragma unroll
              for (int j = 0; j < 4; ++j)
                asm volatile(
                    "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem + b * kBN),
                    "l"(desc_add(da, j * kStepA)), "l"(desc_add(db, j * kStepB)), "r"(idesc), "r"(j > 0 ? 1u : add)
                    : "memory");
              commit_pair(&empty[r.s]);
              if (kb == ke - 1) commit_pair(&acc_full[b]);
            }
            __syncwarp();
          }
        }
      }
      if (!ok && lead) {
        *abort_flag = 1;
        atomicCAS(p.status, 0, kTimedOut + 3);
      }
    }
  } else {
    // a warp reads the TMEM lanes of its quadrant (warp % 4); warps 2..5 take columns 0..127, warps 6..9 the others
    const int quad = warp & 3, half = (warp - 2) >> 2;
    unsigned char* buf = out_buf + (warp - 2) * 4096;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * 128);
    int n = 0;
    int token_label = -1;  // FEW: lane i holds the label of this warp's token i, -1 where it does not count
    if constexpr (FEW && EPI == kLse) {
      const int cw = p.tile_n >> 1, t = half * cw + lane;
      const int64_t y = lane < cw && t < p.N ? p.labels[t] : -1;
      if (y >= 0 && y < p.vocab && y != p.ignore) token_label = (int)y;
    }
    const float alpha = EPI == kOut ? unit_of(p.gout, p.count, p.gmax, p.f16) : 1.f;
    // the next accumulator in TMEM, false after a time-out
    auto take = [&]() {
      const bool ready = !*abort_flag && mbar_wait_cluster(&acc_full[n & 1], (uint32_t)(n >> 1) & 1u);
      if (!__all_sync(0xffffffffu, ready) || *abort_flag) {
        if (!*abort_flag) atomicCAS(p.status, 0, kTimedOut + 4);
        *abort_flag = 1;
        return false;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return true;
    };
    auto release = [&]() {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(&acc_empty[n & 1]), 0));
      ++n;
    };
    for (int u = blockIdx.x >> 1; u < units; u += pairs) {
      int mb, nb, k0, k1;
      unit_at(u, p, kblocks, mb, nb, k0, k1);
      if constexpr (FEW) {
        const int cw = p.tile_n >> 1, t0 = half * cw;  // this warp's tokens
        const int col = mb * kBM + rank * 128 + quad * 32 + lane;  // vocabulary index, or column of dH
        const bool inside = col < p.M;
        const uint32_t at0 = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)t0;
        constexpr int kMost = (EPI == kLse ? kFewScored : kFewGrads) / 2;
        float x[kMost];
        bool good = true;
        const int chunk = EPI == kLse ? p.chunk : kblocks;
        for (int kc = k0; kc < k1; kc += chunk) {
          if (!(good = take())) break;
          #pragma unroll
          for (int c = 0; c < kMost; c += 8) {
            if (c < cw) {
              float v[8];
              tmem_ld8(at0 + (uint32_t)((n & 1) * kBN + c), v);
              #pragma unroll
              for (int i = 0; i < 8; ++i) x[c + i] = kc == k0 ? v[i] : x[c + i] + v[i];
            }
          }
          release();
        }
        if (!good) break;
        if constexpr (EPI == kLse) {
          const int first = col - lane;
          #pragma unroll
          for (int j = 0; j < kMost; j += 4) {
            if (j >= cw || t0 + j >= p.N) break;
            float e[4], most = 0.f;  // lane i keeps token j + i's maximum
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int t = t0 + j + i;
              const bool own = __shfl_sync(0xffffffffu, token_label, j + i) == col;
              if (own && t < p.N) p.tgt[t] = x[j + i];
              const float v = inside && !own ? x[j + i] : -INFINITY, m = warp_max(v);
              e[i] = v - (m == -INFINITY ? 0.f : m);
              if (lane == i) most = m;
              if (col < p.keep_cols && t < p.N) p.keep[t * p.ldk + col] = (uint16_t)(distance_bits(e[i]) & 0xffffu);
              e[i] = ex2(e[i] * kLog2e);
            }
            const float sum = warp_sum4(e, lane);  // lane i: token j + i
            const int t = t0 + j + lane;
            if (lane < 4 && t < p.N && first < p.M) p.part[(int64_t)t * p.parts + (first >> 5)] = make_float2(most, sum);
          }
        } else if (inside) {
          #pragma unroll
          for (int j = 0; j < kMost; ++j) {
            const int t = t0 + j;
            if (j >= cw || t >= p.N) break;
            const float v = alpha * x[j];
            if (p.acc) p.acc[((int64_t)(u % p.splits) * p.N + t) * p.M + col] = v;
            else reinterpret_cast<uint16_t*>(p.out)[t * p.ldo + col] = (uint16_t)pack16(v, 0.f, p.f16);
          }
        }
        continue;
      }
      const int row0 = mb * kBM + rank * 128 + quad * 32, row = row0 + lane;
      const bool live = row < p.M;
      const int n0 = nb * kBN + half * 128;
      int label = -1;  // the label's column among this thread's 128, if it is one of them
      float g = 0.f, lse = 0.f, own_d = 0.f;
      if constexpr (EPI != kOut) {
        if (live) {
          const int64_t y = p.labels[row];
          const bool inside = y >= 0 && y < p.vocab;
          if (inside && y != p.ignore) label = (int)y - (p.v0 + n0);
          if constexpr (EPI == kGrad) {
            if (y != p.ignore) {
              g = factor_of(inside, p.gout, (int64_t)row * p.gstride, p.count, p.gmax, p.f16);
              lse = p.lse[row];
              own_d = expm1f(-p.tgt[row]);
            }
          }
        }
      }
      if constexpr (EPI == kLse) {
        float x[128];
        if (!take()) break;
        tmem_ld128(lanes + (uint32_t)((n & 1) * kBN), x);
        release();
        bool good = true;
        #pragma unroll 1
        for (int kc = k0 + p.chunk; kc < k1; kc += p.chunk) {
          if (!(good = take())) break;
          #pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(lanes + (uint32_t)((n & 1) * kBN + c0), v);
            #pragma unroll
            for (int i = 0; i < 16; ++i) x[c0 + i] += __uint_as_float(v[i]);
          }
          release();
        }
        if (!good) break;
        const int lim = p.N - n0;
        if (lim < 128) {
          #pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = i < lim ? x[i] : -INFINITY;
        }
        if (__any_sync(0xffffffffu, label >= 0 && label < 128)) {  // few of the warps' tiles hold a label
          float own = 0.f;
          #pragma unroll
          for (int i = 0; i < 128; ++i) {
            own = label == i ? x[i] : own;
            x[i] = label == i ? -INFINITY : x[i];
          }
          if (label >= 0 && label < 128) p.tgt[row] = own;
        }
        float m = x[0];
        #pragma unroll
        for (int i = 1; i < 128; ++i) m = fmaxf(m, x[i]);
        const float base = m == -INFINITY ? 0.f : m;
        if (n0 < p.keep_cols && row0 < p.M) {
          #pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 64) {
            if (lim <= c0) break;
            chunk_begin(lane);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {  // 16 bytes at a time: the sums leave no registers for more
              uint32_t w[4];
              #pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int c = c0 + 8 * j + 2 * i;
                w[i] = __byte_perm(distance_bits(x[c] - base), distance_bits(x[c + 1] - base), 0x5410);
              }
              chunk_unit(buf, lane, j, make_uint4(w[0], w[1], w[2], w[3]));
            }
            chunk_send(buf, lane, &map_o, n0 + c0, row0, 0);
          }
        }
        float sum0 = 0.f, sum1 = 0.f;
        #pragma unroll
        for (int i = 0; i < 128; i += 2) {
          sum0 += ex2((x[i] - base) * kLog2e);
          sum1 += ex2((x[i + 1] - base) * kLog2e);
        }
        if (live) p.part[(int64_t)row * p.parts + 2 * nb + half] = make_float2(m, sum0 + sum1);
      } else {
        if (!take()) break;
        float x[128];
        tmem_ld128(lanes + (uint32_t)((n & 1) * kBN), x);
        release();
        if (EPI == kOut && p.acc) {
          float* acc = p.acc + (int64_t)(u % p.splits) * p.M * p.N;
          #pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 32) {
            const int lim = p.N - (n0 + c0);
            if (lim <= 0 || row0 >= p.M) break;
            chunk_begin(lane);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float* e = x + c0 + 4 * j;
              chunk_unit(buf, lane, j, make_uint4(__float_as_uint(alpha * e[0]), __float_as_uint(alpha * e[1]),
                                                  __float_as_uint(alpha * e[2]), __float_as_uint(alpha * e[3])));
            }
            if (p.tile_out)
              chunk_send(buf, lane, &map_o, n0 + c0, row0, u % p.splits);
            else
              chunk_rows<4>(buf, lane, acc + (int64_t)row0 * p.N + n0 + c0, (int64_t)p.N * 4, p.M - row0, lim);
          }
        } else {
          #pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 64) {
            uint32_t w[32];
            #pragma unroll
            for (int i = 0; i < 64; i += 2) {
              float a = x[c0 + i], b = x[c0 + i + 1];
              if constexpr (EPI == kGrad) {
                a = label == c0 + i ? own_d : ex2((a - lse) * kLog2e);
                b = label == c0 + i + 1 ? own_d : ex2((b - lse) * kLog2e);
                a = g == 0.f ? 0.f : g * a;
                b = g == 0.f ? 0.f : g * b;
              } else {
                a *= alpha;
                b *= alpha;
              }
              w[i / 2] = pack16(a, b, p.f16);
            }
            store_half_rows(p, &map_o, buf, lane, row0, n0 + c0, reinterpret_cast<uint16_t*>(p.out), p.ldo, w,
                            p.N - (n0 + c0));
          }
        }
      }
    }
    chunk_drain(lane);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other's loads, MMAs or arrivals may touch its shared memory
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// d of the kept columns, in place of their distances q below the maximum m of their part of the columns (2^shift of
// them): g (exp(l - lse) - [v = y]) = g (exp(m - lse) 2^-q - ..); the label's own entry comes from its score.  A row
// to blockIdx.y, eight columns to a thread and step, so that a row's scalars are read once for the columns of a CTA.  It
// moves memory: 4 bytes an entry (511 x 32003: 12 us, 5.4 TB/s).
__global__ void __launch_bounds__(256) k_xent_kept(uint16_t* __restrict__ d, int64_t ldk, int T, int cols,
                                                   const float2* __restrict__ part, int parts, int shift,
                                                   const float* __restrict__ score, const float* __restrict__ lse,
                                                   const int64_t* __restrict__ labels, int64_t ignore, int vocab,
                                                   const float* __restrict__ gout, int gstride,
                                                   const float* __restrict__ count, const float* __restrict__ gmax,
                                                   int f16) {
  allow_behind();
  wait_before();
  for (int row = blockIdx.y; row < T; row += gridDim.y) {
    const int64_t y = labels[row];
    const bool inside = y >= 0 && y < vocab;
    const float of_all = lse[row];
    float g = 0.f, own = 0.f;
    if (y != ignore) {
      g = factor_of(inside, gout, (int64_t)row * gstride, count, gmax, f16);
      if (inside) own = g * expm1f(-score[row]);
    }
    const int label = inside && y != ignore ? (int)y : -1;
    // log2 units above lse of a column; beyond the distances' range (2^-32 of the part's largest) there is none
    auto above = [](float up, uint32_t q) { return up + (q == 0xffffu ? -INFINITY : (float)q * (-1.f / kStep)); };
    #pragma unroll 4
    for (int c0 = (blockIdx.x * 256 + threadIdx.x) * 8; c0 < cols; c0 += gridDim.x * 2048) {
      uint4* at = reinterpret_cast<uint4*>(d + row * ldk + c0);
      uint4 raw = __ldcs(at);
      const float up = (part[(int64_t)row * parts + (c0 >> shift)].x - of_all) * kLog2e;
      uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = g * ex2(above(up, w[i] & 0xffffu));
        float b = g * ex2(above(up, w[i] >> 16));
        if (label == c0 + 2 * i) a = own;
        if (label == c0 + 2 * i + 1) b = own;
        w[i] = g == 0.f ? 0u : pack16(a, b, f16);
      }
      *at = raw;
    }
  }
}

// out (16 bits, ldo) or sum (FP32, contiguous) = (add ? sum : 0) + the planes in order.  W columns to a thread: 4 where
// the rows are aligned for it, else 1; rows to blockIdx.y.
template <int W>
__global__ void __launch_bounds__(256) k_xent_planes(const float* __restrict__ planes, int splits, int M, int N, float* sum,
                                                     int add, uint16_t* __restrict__ out, int64_t ldo, int f16) {
  allow_behind();
  wait_before();
  const int c = (blockIdx.x * 256 + threadIdx.x) * W;
  if (c >= N) return;
  const int64_t total = (int64_t)M * N;
  for (int row = blockIdx.y; row < M; row += gridDim.y) {
    const int64_t at = (int64_t)row * N + c;
    float a[W];
    auto load = [&](const float* from, float (&v)[W]) {
      if constexpr (W == 4) {
        const float4 f = *reinterpret_cast<const float4*>(from);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
      } else {
        v[0] = *from;
      }
    };
    #pragma unroll
    for (int i = 0; i < W; ++i) a[i] = 0.f;
    if (add) load(sum + at, a);
    #pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      float v[W];
      load(planes + s * total + at, v);
      #pragma unroll
      for (int i = 0; i < W; ++i) a[i] += v[i];
    }
    if constexpr (W == 4) {
      if (out)
        *reinterpret_cast<uint2*>(out + row * ldo + c) = make_uint2(pack16(a[0], a[1], f16), pack16(a[2], a[3], f16));
      else
        *reinterpret_cast<float4*>(sum + at) = make_float4(a[0], a[1], a[2], a[3]);
    } else {
      if (out) out[row * ldo + c] = (uint16_t)pack16(a[0], 0.f, f16);
      else sum[at] = a[0];
    }
  }
}

// Joins a token's parts, which leave the label out, with the label's logit: lse and nll; one CTA a token, fixed order.  A
// thread's first kHeld parts stay in registers between the two passes: all of them up to kHeld parts a thread.
constexpr int kHeld = 8;
__global__ void __launch_bounds__(1024) k_xent_join(const float2* __restrict__ part, int ld, int nt,
                                                    float* __restrict__ tgt, const int64_t* __restrict__ labels,
                                                    int64_t ignore, int vocab, float* __restrict__ lse,
                                                    float* __restrict__ nll) {
  __shared__ float red[32];
  __shared__ float top_s;
  allow_behind();
  wait_before();
  const int64_t t = blockIdx.x;
  const float2* row = part + t * ld;
  float2 v[kHeld];
  #pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    v[j] = i < nt ? row[i] : make_float2(-INFINITY, 0.f);
  }
  float m = -INFINITY;
  #pragma unroll
  for (int j = 0; j < kHeld; ++j) m = fmaxf(m, v[j].x);
  for (int i = threadIdx.x + kHeld * blockDim.x; i < nt; i += blockDim.x) m = fmaxf(m, row[i].x);
  m = block_max(m, red, -INFINITY);  // logits may all be negative
  if (threadIdx.x == 0) top_s = m;
  __syncthreads();
  const float top = top_s, base = top == -INFINITY ? 0.f : top;
  float s = 0.f;
  #pragma unroll
  for (int j = 0; j < kHeld; ++j) s += v[j].y * expf(v[j].x - base);
  for (int i = threadIdx.x + kHeld * blockDim.x; i < nt; i += blockDim.x) s += row[i].y * expf(row[i].x - base);
  s = block_sum(s, red);
  if (threadIdx.x == 0) {
    const int64_t y = labels[t];
    const bool inside = y >= 0 && y < vocab;
    if (y == ignore || !inside) {  // the parts hold every column
      lse[t] = base + logf(s);
      nll[t] = tgt[t] = y == ignore ? 0.f : __int_as_float(0x7fc00000);
    } else {
      const float l = tgt[t], all = fmaxf(top, l);
      const float e = all + logf(s * expf(top - all) + expf(l - all));
      const float d = top - l;  // the others' maximum above the label
      lse[t] = e;
      // beyond e^44 the label's share of the sum is none
      const float n = !isfinite(l) ? e - l : (d < 44.f ? log1pf(s * expf(d)) : d + logf(s));
      nll[t] = tgt[t] = n;
    }
  }
}

// loss = sum_t nll_t (divided by the number of counted labels for the mean); count = that number.  One CTA.
__global__ void __launch_bounds__(1024) k_xent_reduce(const float* __restrict__ nll, const int64_t* __restrict__ labels,
                                                      int64_t ignore, int T, int mean, float* __restrict__ loss,
                                                      float* __restrict__ count) {
  __shared__ float red[32];
  allow_behind();
  wait_before();
  float s = 0.f, c = 0.f;
  for (int t = threadIdx.x; t < T; t += 1024) {
    s += nll[t];
    c += labels[t] != ignore ? 1.f : 0.f;  // exact: T < 2^24
  }
  s = block_sum(s, red);
  c = block_sum(c, red);
  if (threadIdx.x == 0) {
    *loss = mean ? s / c : s;
    *count = c;
  }
}

// gmax = max |g_t| over the tokens that count and whose g_t is finite, g_t = gout[t gstride] (/ count): one that is not
// spoils its own token's gradient only.  One CTA.
__global__ void __launch_bounds__(1024) k_xent_gmax(const float* __restrict__ gout, int gstride,
                                                    const int64_t* __restrict__ labels, int64_t ignore, int vocab, int T,
                                                    const float* __restrict__ count, float* __restrict__ gmax) {
  __shared__ float red[32];
  allow_behind();
  float m = 0.f;
  for (int t = threadIdx.x; t < T; t += 1024) {
    const int64_t y = labels[t];
    const float g = fabsf(gout[(int64_t)t * gstride]);
    if (y != ignore && y >= 0 && y < vocab && g < INFINITY) m = fmaxf(m, g);
  }
  m = block_max(m, red);
  if (threadIdx.x == 0) *gmax = count && m > 0.f ? m / *count : m;
}

// 16-bit row-major matrix [rows, cols] (leading dimension ld): box of 64 columns (one swizzle line) x `box` rows.
static int map16(CUtensorMap* m, const void* p, int rows, int cols, int64_t ld, int box, int f16) {
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t boxes[2] = {64, (cuuint32_t)box};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                              const_cast<void*>(p), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("mpq_xent: cuTensorMapEncodeTiled failed (%d) rows=%d cols=%d ld=%lld", (int)r, rows, cols,
                   (long long)ld);
    return MPQ_ERR_ARG;
  }
  return MPQ_OK;
}

// One operand of a product: [rows, k] K-major or [k, rows] MN-major; `box`: rows of a CTA's half tile.
static int operand(CUtensorMap* m, bool mn, const void* p, int rows, int k, int64_t ld, int box, int f16) {
  return mn ? map16(m, p, k, rows, ld, 64, f16) : map16(m, p, rows, k, ld, box, f16);
}

static int num_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = n > 1 ? n : 148;
  }
  return cached[dev];
}

// Parts of K for an M x N product: the number with the least estimated cycles.  A unit takes 512 a k-block and 2000 for
// its start and end; parts add FP32 planes, written and read once at 3600 bytes a cycle (the memory's rate), and the
// launch that sums them.  Every part has at least 16 k-blocks.  (dH at 511 x 32003 x 2048, us: 1 part 190, 2 96, 4 65,
// 8 73; at 8192 x 128256 x 4096: 1 part 6075, 2 7600.)
static int splits_for(int M, int N, int K) {
  const int pairs = num_sms() / 2, kblocks = (K + 63) / 64;
  const double tiles = (double)((M + kBM - 1) / kBM) * ((N + kBN - 1) / kBN);
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= 32 && (s == 1 || s * 16 <= kblocks); ++s) {
    const double planes = s > 1 ? 8.0 * M * N * s / 3600.0 + 5000.0 : 0.0;
    const double t = std::ceil(tiles * s / pairs) * (std::ceil((double)kblocks / s) * 512 + 2000) + planes;
    if (t < 0.98 * least) {
      least = t;
      best = s;
    }
  }
  return best;
}

template <int EPI, bool A_MN, bool B_MN, bool FEW = false>
static int product(const void* A, int64_t lda, const void* B, int64_t ldb, Args p, bool behind, cudaStream_t st) {
  CUtensorMap ma, mb, mo{};
  p.tile_n = FEW ? (p.N + 15) / 16 * 16 : kBN;
  p.a_rows = A_MN || FEW ? 128 : std::min((p.M + 7) / 8 * 8, 128);
  p.b_rows = p.tile_n / 2;
  p.chunk = p.f16 ? kChunkF16 : kChunkBf16;
  p.stages = std::min<int>(kMostStages, kRingBytes / ((p.a_rows + p.b_rows) * 128));
  int r = operand(&ma, A_MN, A, p.M, p.K, lda, p.a_rows, p.f16);
  if (r) return r;
  if ((r = operand(&mb, B_MN, B, p.N, p.K, ldb, p.b_rows, p.f16))) return r;
  p.mt = (p.M + kBM - 1) / kBM;
  p.nt = (p.N + kBN - 1) / kBN;
  p.splits = std::max(p.splits, 1);
  const int type = p.f16 ? 2 : 1;
  if (FEW) {
    // the threads store: a warp's 32 columns of a token are neighbours
  } else if (EPI == kLse) {
    MPQ_CHECK_ARG(p.keep_cols == 0 || result_map(&mo, p.keep, type, 1, p.M, p.keep_cols, p.ldk, true),
                  "mpq_xent_forward: no tensor map for %d kept columns", p.keep_cols);
  } else if (p.acc) {
    p.tile_out = result_map(&mo, p.acc, 0, p.splits, p.M, p.N, p.N, false);
  } else {
    p.tile_out = result_map(&mo, p.out, type, 1, p.M, p.N, p.ldo, EPI == kGrad);  // d's rows are workspace
  }
  const size_t smem = 1024 + kRingBytes + kEpiWarps * 4096 + 256;
  const int grid = 2 * std::min(p.mt * p.nt * p.splits, num_sms() / 2);
  return launch("mpq_xent product", k_xent_gemm<EPI, A_MN, B_MN, FEW>, grid, kThreads, smem, 0, behind, st, ma, mb, mo,
                p);
}

// Width of the piece that starts at column v0.
static int piece_at(int v0, int V, int piece, int keep_cols) {
  return v0 < keep_cols ? keep_cols : std::min(piece, V - v0);
}

static bool operand_ok(const void* p, int64_t ld, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld >= cols;
}

}  // namespace xent
}  // namespace mpq

using namespace mpq;

// Parts of the vocabulary in the forward pass: `part` holds T x this many float2.
MPQ_API int mpq_xent_tiles(int T, int V) {
  return T > 0 && V > 0 ? (T <= xent::kFewScored ? 8 : 2) * (int)(((int64_t)V + xent::kBN - 1) / xent::kBN) : 0;
}

// FP32 planes of T x H that the backward pass needs for dhidden (0: none): one for each part of K of its largest
// piece, and the running sum of several pieces.
MPQ_API int mpq_xent_planes(int T, int V, int H, int piece, int keep_cols) {
  if (T <= 0 || V <= 0 || H <= 0 || piece <= 0 || keep_cols < 0 || keep_cols > V) return 0;
  const int rest = V - keep_cols, pieces = (keep_cols > 0) + (rest + piece - 1) / piece;
  int most = 1;  // over the widths that occur: the kept columns, whole pieces and the last one
  for (int w : {keep_cols, std::min(piece, rest), rest % piece})
    if (w > 0) most = std::max(most, xent::splits_for(T, H, w));
  return pieces > 1 ? most + 1 : (most > 1 ? most : 0);
}

MPQ_API int mpq_xent_forward(int T, int V, int H, int dtype, const void* hidden, int64_t ldh, const void* weight,
                             int64_t ldw, const int64_t* labels, int64_t ignore, float* part, int64_t part_floats,
                             float* tgt, float* lse, float* nll, int reduction, float* loss,
                             float* count, void* keep, int64_t ldk, int keep_cols, int* status, void* stream) {
  MPQ_CHECK_ARG(reduction >= 0 && reduction <= 2 && (reduction == 0 || (loss && count)),
                "mpq_xent_forward: reduction must be 0 (none), 1 (sum) or 2 (mean); the last two need loss and count");
  MPQ_CHECK_ARG(dtype == 1 || dtype == 2, "mpq_xent_forward: dtype must be 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(T >= 0 && V >= 1 && H >= 1 && T <= (1 << 24) && V <= (1 << 30),
                "mpq_xent_forward: bad shape %d x %d x %d", T, V, H);
  if (T == 0 && reduction == 0) return MPQ_OK;
  if (T == 0) {
    xent::k_xent_reduce<<<1, 1024, 0, (cudaStream_t)stream>>>(nullptr, nullptr, ignore, 0, reduction == 2, loss, count);
    return launch_status("mpq_xent_forward (reduce)");
  }
  MPQ_CHECK_ARG(hidden && weight && labels && part && tgt && lse && nll && status, "mpq_xent_forward: null pointer");
  MPQ_CHECK_ARG(xent::operand_ok(hidden, ldh, H) && xent::operand_ok(weight, ldw, H),
                "mpq_xent_forward: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  MPQ_CHECK_ARG(part_floats >= 2ll * T * mpq_xent_tiles(T, V) && (reinterpret_cast<uintptr_t>(part) & 7) == 0,
                "mpq_xent_forward: the workspace needs %lld floats", 2ll * T * mpq_xent_tiles(T, V));
  MPQ_CHECK_ARG(keep_cols == 0 || (keep && (keep_cols == V || (keep_cols > 0 && keep_cols < V && keep_cols % 256 == 0)) &&
                                   xent::operand_ok(keep, ldk, keep_cols)),
                "mpq_xent_forward: keep_cols must be V or a multiple of 256 below it, kept in rows like the operands");
  MPQ_CHECK_ARG((int64_t)((T + 255) / 256) * mpq_xent_tiles(T, V) < (1ll << 31), "mpq_xent_forward: too many tiles");
  cudaStream_t cs = (cudaStream_t)stream;
  int st = tc::get_encoder();
  if (st) return st;
  xent::Args p{};
  p.K = H;
  p.f16 = dtype == 2;
  p.status = status;
  p.labels = labels; p.ignore = ignore; p.vocab = V;
  p.part = reinterpret_cast<float2*>(part);
  p.parts = mpq_xent_tiles(T, V);
  p.tgt = tgt;
  p.keep = reinterpret_cast<uint16_t*>(keep); p.ldk = ldk; p.keep_cols = keep_cols;
  if (T <= xent::kFewScored) {
    p.M = V; p.N = T;
    st = xent::product<xent::kLse, false, false, true>(weight, ldw, hidden, ldh, p, false, cs);
  } else {
    p.M = T; p.N = V;
    st = xent::product<xent::kLse, false, false>(hidden, ldh, weight, ldw, p, false, cs);
  }
  if (st) return st;
  const int live = T <= xent::kFewScored ? (V + 31) / 32 : p.parts;  // parts that hold columns
  // threads for a token: kHeld parts each, as far as a CTA goes
  const int threads = live <= 1024 ? 128 : (live <= 2048 ? 256 : (live <= 4096 ? 512 : 1024));
  st = tc::launch("mpq_xent_forward (join)", xent::k_xent_join, T, threads, 0, 0, true, cs, (const float2*)p.part, p.parts,
                  live, tgt, labels, ignore, V, lse, nll);
  if (st || reduction == 0) return st;
  return tc::launch("mpq_xent_forward (reduce)", xent::k_xent_reduce, 1, 1024, 0, 0, true, cs, (const float*)nll, labels,
                    ignore, T, (int)(reduction == 2), loss, count);
}

MPQ_API int mpq_xent_backward(int T, int V, int H, int dtype, const void* hidden, int64_t ldh, const void* weight,
                              int64_t ldw, const int64_t* labels, int64_t ignore, const float* lse, const float* gout,
                              int gstride, const float* count, const float* part, const float* tgt, void* keep,
                              int64_t ldk, int keep_cols, float* gmax, void* d, int piece, float* acc, void* dhidden,
                              int64_t lddh, void* dweight, int64_t lddw, int* status, void* stream) {
  MPQ_CHECK_ARG(dtype == 1 || dtype == 2, "mpq_xent_backward: dtype must be 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(T >= 0 && V >= 1 && H >= 1 && T <= (1 << 24) && V <= (1 << 30),
                "mpq_xent_backward: bad shape %d x %d x %d", T, V, H);
  MPQ_CHECK_ARG(piece >= 256 && piece % 256 == 0, "mpq_xent_backward: the piece must be a multiple of 256 columns");
  MPQ_CHECK_ARG(keep_cols == 0 || keep_cols == V || (keep_cols > 0 && keep_cols < V && keep_cols % 256 == 0),
                "mpq_xent_backward: keep_cols must be V or a multiple of 256 below it");
  if (T == 0) return MPQ_OK;
  MPQ_CHECK_ARG(hidden && weight && labels && lse && gout && (gmax || gstride == 0) && status,
                "mpq_xent_backward: null pointer");
  MPQ_CHECK_ARG(xent::operand_ok(hidden, ldh, H) && xent::operand_ok(weight, ldw, H),
                "mpq_xent_backward: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  MPQ_CHECK_ARG(tgt && (keep_cols == 0 || (keep && part && xent::operand_ok(keep, ldk, keep_cols))),
                "mpq_xent_backward: the gradient needs tgt, the kept columns their rows and part");
  MPQ_CHECK_ARG(keep_cols == V || (d && xent::operand_ok(d, piece, 0)), "mpq_xent_backward: a piece needs its workspace");
  MPQ_CHECK_ARG(!dhidden || lddh >= H, "mpq_xent_backward: lddh < H");
  MPQ_CHECK_ARG(!dweight || lddw >= H, "mpq_xent_backward: lddw < H");
  const int planes = mpq_xent_planes(T, V, H, piece, keep_cols);
  MPQ_CHECK_ARG(!dhidden || planes == 0 || acc, "mpq_xent_backward: dhidden needs %d planes of workspace", planes);
  cudaStream_t cs = (cudaStream_t)stream;
  int st = tc::get_encoder();
  if (st) return st;
  const int f16 = dtype == 2;
  bool behind = false;  // a kernel of this call came before
  if (gstride == 0) {
    gmax = nullptr;
  } else {
    xent::k_xent_gmax<<<1, 1024, 0, cs>>>(gout, gstride, labels, ignore, V, T, count, gmax);
    if ((st = launch_status("mpq_xent_backward (scale)"))) return st;
    behind = true;
  }
  for (int v0 = 0, w; v0 < V; v0 += w) {
    w = xent::piece_at(v0, V, piece, keep_cols);
    const uint16_t* W = reinterpret_cast<const uint16_t*>(weight) + (int64_t)v0 * ldw;
    const void* dv = d;
    int64_t ldd = piece;
    xent::Args p{};
    p.f16 = f16;
    p.status = status;
    p.gout = gout; p.gstride = gstride; p.count = count; p.gmax = gmax;
    if (v0 < keep_cols) {
      dim3 grid(std::min((keep_cols + 2047) / 2048, 4), std::min(T, 32768));
      st = tc::launch("mpq_xent_backward (kept)", xent::k_xent_kept, grid, 256, 0, 0, behind, cs, (uint16_t*)keep, ldk, T,
                      keep_cols, (const float2*)part, mpq_xent_tiles(T, V), T <= xent::kFewScored ? 5 : 7, tgt, lse, labels,
                      ignore, V, gout, gstride, count, (const float*)gmax, f16);
      if (st) return st;
      dv = keep;
      ldd = ldk;
    } else {
      p.M = T; p.N = w; p.K = H;
      p.labels = labels; p.ignore = ignore; p.vocab = V; p.v0 = v0;
      p.lse = lse;
      p.tgt = const_cast<float*>(tgt);
      p.out = d; p.ldo = piece;
      if ((st = xent::product<xent::kGrad, false, false>(hidden, ldh, W, ldw, p, behind, cs))) return st;
    }
    behind = true;
    if (dhidden) {
      p.K = w;
      p.out = dhidden; p.ldo = lddh;
      p.acc = planes ? acc : nullptr;
      p.splits = xent::splits_for(T, H, w);  // no more for a narrower last piece
      if (T <= xent::kFewGrads) {
        p.M = H; p.N = T;
        st = xent::product<xent::kOut, true, false, true>(W, ldw, dv, ldd, p, true, cs);
      } else {
        p.M = T; p.N = H;
        st = xent::product<xent::kOut, false, true>(dv, ldd, W, ldw, p, true, cs);
      }
      if (st) return st;
      if (planes) {
        const int64_t n = (int64_t)T * H;
        float* sum = acc + (planes - 1) * n;
        uint16_t* out = v0 + w == V ? (uint16_t*)dhidden : nullptr;
        const bool wide = H % 4 == 0 && lddh % 4 == 0 && (reinterpret_cast<uintptr_t>(acc) & 15) == 0 &&
                          (reinterpret_cast<uintptr_t>(dhidden) & 7) == 0;
        const dim3 grid(wide ? (H / 4 + 255) / 256 : (H + 255) / 256, std::min(T, 65535));
        st = tc::launch("mpq_xent_backward (planes)", wide ? xent::k_xent_planes<4> : xent::k_xent_planes<1>, grid, 256,
                        0, 0, true, cs, (const float*)acc, p.splits, T, H, sum, (int)(v0 > 0), out, lddh, f16);
        if (st) return st;
      }
    }
    if (dweight) {
      p.M = w; p.N = H; p.K = T;
      p.out = reinterpret_cast<uint16_t*>(dweight) + (int64_t)v0 * lddw; p.ldo = lddw;
      p.acc = nullptr;
      p.splits = 1;
      if ((st = xent::product<xent::kOut, true, true>(dv, ldd, hidden, ldh, p, true, cs))) return st;
    }
  }
  return MPQ_OK;
}
