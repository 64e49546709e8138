// Softmax cross entropy of an output head over its whole vocabulary, from the hidden states, with its gradients.
//
//   l[t, v] = h_t . w_v,   lse_t = log sum_v exp l[t, v],   nll_t = lse_t - l[t, y_t]
//   d[t, v] = g_t (exp(l[t, v] - lse_t) - [v = y_t]),   dH = d W,   dW = d^T H
//
// The logits are never stored.  The forward product reduces each 256-column tile of a token's logits to (max, sum of
// exp) in its epilogue and picks the label's logit out on the way; a second kernel joins the tiles in order.  The
// backward pass takes the vocabulary in pieces: it computes a piece's logits again, turns them into d in 16 bits in the
// epilogue, and multiplies d with the piece of W (dH, summed over the pieces in FP32) and with H (dW's rows of the
// piece).  Every sum runs in a fixed order, so results repeat bit for bit.
//
// d is held as 2^k d / max|g|, in units of its largest possible magnitude, and the products take the factor back in
// FP32: in f16 (k = 15) probabilities down to 2^-39 then stay normal numbers, whatever the mean divides by; bf16 has
// the exponent range and takes k = 0.  Rounding d to 16 bits costs each of its entries 2^-9 (bf16) or 2^-12 (f16) of
// itself, no more than the rounding of the gradients to the same type.
//
// A label equal to `ignore` does not count: nll 0, d 0.  A label outside the vocabulary makes the token's nll and its
// d NaN; no memory is read for it.
#include <algorithm>
#include <cuda_bf16.h>
#include "umma.cuh"

namespace mpq {
namespace xent {

using namespace tc;

constexpr int kThreads = 192;
constexpr int kBM = 128, kBN = 256, kStages = 4, kGroup = 16;
constexpr uint32_t kStageA = kBM * 128, kStageB = kBN * 128;
constexpr float kLog2e = 1.4426950408889634f;

enum { kLse = 0, kGrad = 1, kOut = 2 };

struct Args {
  int M, N, K, mt, nt;      // C[M, N] over K; tiles of 128 x 256
  int f16;                  // 1: f16 operands, 0: bf16
  int* status;
  // kLse, kGrad
  const int64_t* labels;
  int64_t ignore;
  int vocab;                // labels in [0, vocab) count
  int v0;                   // first column's vocabulary index
  float2* part;             // kLse: [M, nt] (max in log2 units, sum of exp2)
  float* tgt;               // kLse: [M] the label's logit
  const float* lse;         // kGrad: [M]
  const float* gout;        // kGrad: upstream gradient, gout[t * gstride]
  int gstride;
  const float* count;       // kGrad: divides g where given (the mean's number of labels)
  const float* gmax;        // kGrad, kOut: largest |g| of the counted tokens
  // kGrad, kOut
  void* out;
  int64_t ldo;
  float* acc;               // kOut: FP32 running sum [M, N], contiguous; null: C goes straight to `out`
  int first, last;          // kOut with acc: start the sum / round it to `out`
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

// Tile t of a raster that walks kGroup row tiles down before it takes the next column tile: the tiles in flight share
// a few row tiles (kept in L2) and stream the columns once for each group.
__device__ __forceinline__ void tile_at(int t, int mt, int nt, int& mb, int& nb) {
  const int per = kGroup * nt, g = t / per, r = t - g * per;
  const int rows = min(kGroup, mt - g * kGroup);
  mb = g * kGroup + r % rows;
  nb = r / rows;
}

// 32 consecutive 16-bit results of one row.
__device__ __forceinline__ void store16(void* out, int64_t at, const float (&o)[32], int lim, int f16) {
  uint16_t* dst = reinterpret_cast<uint16_t*>(out) + at;
  uint32_t w[16];
  #pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack16(o[2 * i], o[2 * i + 1], f16);
  if (lim >= 32 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
    #pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  } else {
    #pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < lim) dst[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
}

// C[M, N] = A B with an epilogue.  A K-major: [M, K] rows; A_MN: [K, M] rows.  B likewise ([N, K] or [K, N] rows).
// 16-bit operands, FP32 accumulation in TMEM; persistent over the tiles, two accumulators.  Warp 0 loads (TMA), warp 1
// issues the MMAs, warps 2..5 are the epilogue, one row to a thread.
template <int EPI, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1)
    k_xent_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Args p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * (kStageA + kStageB));
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto s_a = [&](int s) { return ring + s * kStageA; };
  auto s_b = [&](int s) { return ring + kStages * kStageA + s * kStageB; };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkb = (p.K + 63) / 64, tiles = p.mt * p.nt;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int64_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        int mb, nb;
        tile_at(t, p.mt, p.nt, mb, nb);
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = (int)(it % kStages);
          if (*abort_flag || !mbar_wait(&empty[s], ((uint32_t)(it / kStages) & 1u) ^ 1u)) {
            ok = false;
            break;
          }
          mbar_expect_tx(&full[s], kStageA + kStageB);
          if constexpr (A_MN) {
            #pragma unroll
            for (int i = 0; i < kBM / 64; ++i)
              tma_load_2d(s_a(s) + i * 8192, &map_a, &full[s], mb * kBM + i * 64, kb * 64);
          } else {
            tma_load_2d(s_a(s), &map_a, &full[s], kb * 64, mb * kBM);
          }
          if constexpr (B_MN) {
            #pragma unroll
            for (int i = 0; i < kBN / 64; ++i)
              tma_load_2d(s_b(s) + i * 8192, &map_b, &full[s], nb * kBN + i * 64, kb * 64);
          } else {
            tma_load_2d(s_b(s), &map_b, &full[s], kb * 64, nb * kBN);
          }
        }
      }
      if (!ok) {  // drain the copies in flight (each wait bounded) before the CTA may end
        *abort_flag = 1;
        for (int64_t k = it < kStages ? 0 : it - kStages; k < it; ++k)
          mbar_wait(&full[k % kStages], (uint32_t)(k / kStages) & 1u);
        atomicCAS(p.status, 0, 2);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc16(p.f16, A_MN, B_MN, kBM, kBN);
      int64_t it = 0;
      bool ok = true;
      int n = 0;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++n) {
        const int b = n & 1;
        if (*abort_flag || !mbar_wait(&acc_empty[b], ((uint32_t)(n >> 1) & 1u) ^ 1u)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = (int)(it % kStages);
          if (*abort_flag || !mbar_wait(&full[s], (uint32_t)(it / kStages) & 1u)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a0 = smem_u32(s_a(s)), b0 = smem_u32(s_b(s));
          #pragma unroll
          for (int j = 0; j < 4; ++j) {  // K = 16: 32 bytes along a K-major line, 16 lines of an MN-major operand
            const uint64_t da = A_MN ? smem_desc_mn_sw128(a0 + j * 2048) : smem_desc_k_sw128(a0 + j * 32);
            const uint64_t db = B_MN ? smem_desc_mn_sw128(b0 + j * 2048) : smem_desc_k_sw128(b0 + j * 32);
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem + b * kBN),
                "l"(da), "l"(db), "r"(idesc), "r"((kb > 0 || j > 0) ? 1u : 0u)
                : "memory");
          }
          asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                           smem_u32(&empty[s]))
                       : "memory");
        }
        // the accumulator is complete (or, after an abort, the issued MMAs have retired)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                         smem_u32(&acc_full[b]))
                     : "memory");
      }
      if (!ok) {
        *abort_flag = 1;
        atomicCAS(p.status, 0, 3);
      }
    }
  } else {
    const int quad = warp & 3;
    int n = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
      const int b = n & 1;
      int mb, nb;
      tile_at(t, p.mt, p.nt, mb, nb);
      const bool ready = !*abort_flag && mbar_wait(&acc_full[b], (uint32_t)(n >> 1) & 1u);
      if (!__all_sync(0xffffffffu, ready) || *abort_flag) {
        if (!*abort_flag) atomicCAS(p.status, 0, 4);
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int row = mb * kBM + quad * 32 + lane;
      const bool live = row < p.M;
      const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kBN);
      const int n0 = nb * kBN;
      int64_t label = -1;
      float g = 0.f, lse2 = 0.f, alpha = 1.f;
      if constexpr (EPI == kOut) alpha = *p.gmax * (p.f16 ? 1.f / 32768.f : 1.f);
      if constexpr (EPI != kOut) {
        if (live) label = p.labels[row];
        if constexpr (EPI == kGrad) {
          if (live && label != p.ignore) {
            g = label >= 0 && label < p.vocab ? p.gout[(int64_t)row * p.gstride] : __int_as_float(0x7fc00000);
            if (p.count) g /= *p.count;
            const float top = *p.gmax;
            g = top == 0.f && g == 0.f ? 0.f : g / top * (p.f16 ? 32768.f : 1.f);
            lse2 = p.lse[row] * kLog2e;
          }
        }
        if (label == p.ignore || label < 0 || label >= p.vocab) label = -1;
        else label -= p.v0 + n0;  // the label's column in this tile, if it is in [0, 256)
      }
      float m = -INFINITY, sum = 0.f;
      #pragma unroll 1
      for (int c0 = 0; c0 < kBN; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(trow + c0, v);
        const int lim = p.N - (n0 + c0);
        if (lim <= 0) continue;
        if constexpr (EPI == kLse) {
          float x[32], top = -INFINITY;
          #pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (label == c0 + i && live) p.tgt[row] = __uint_as_float(v[i]);
            x[i] = i < lim ? __uint_as_float(v[i]) * kLog2e : -INFINITY;
            top = fmaxf(top, x[i]);
          }
          const float mn = fmaxf(m, top);
          const float base = mn == -INFINITY ? 0.f : mn;
          sum *= exp2f(m - base);
          #pragma unroll
          for (int i = 0; i < 32; ++i) sum += exp2f(x[i] - base);
          m = mn;
        } else if constexpr (EPI == kGrad) {
          float o[32];
          #pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float e = exp2f(fmaf(__uint_as_float(v[i]), kLog2e, -lse2)) - (label == c0 + i ? 1.f : 0.f);
            o[i] = g == 0.f ? 0.f : g * e;
          }
          if (live) store16(p.out, (int64_t)row * p.ldo + n0 + c0, o, lim, p.f16);
        } else {
          float o[32];
          float* acc = p.acc ? p.acc + (int64_t)row * p.N + n0 + c0 : nullptr;
          #pragma unroll
          for (int i = 0; i < 32; ++i) {
            o[i] = alpha * __uint_as_float(v[i]);
            if (acc && !p.first && live && i < lim) o[i] += acc[i];
          }
          if (live) {
            if (!acc || p.last) {
              store16(p.out, (int64_t)row * p.ldo + n0 + c0, o, lim, p.f16);
            } else {
              #pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i < lim) acc[i] = o[i];
            }
          }
        }
      }
      if constexpr (EPI == kLse) {
        if (live) p.part[(int64_t)row * p.nt + nb] = make_float2(m, sum);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Joins a token's tiles: lse = log2-domain maximum and sum -> natural log; one CTA a token, fixed order.
__global__ void __launch_bounds__(128) k_xent_join(const float2* __restrict__ part, int nt, const float* __restrict__ tgt,
                                                   const int64_t* __restrict__ labels, int64_t ignore, int vocab,
                                                   float* __restrict__ lse, float* __restrict__ nll) {
  __shared__ float red[4];
  __shared__ float top_s;
  const int64_t t = blockIdx.x;
  const float2* row = part + t * nt;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < nt; i += 128) m = fmaxf(m, row[i].x);
  m = block_max(m, red);
  if (threadIdx.x == 0) top_s = m;
  __syncthreads();
  const float top = top_s, base = top == -INFINITY ? 0.f : top;
  float s = 0.f;
  for (int i = threadIdx.x; i < nt; i += 128) s += row[i].y * exp2f(row[i].x - base);
  s = block_sum(s, red);
  if (threadIdx.x == 0) {
    const float l = (base + log2f(s)) * 0.69314718055994531f;
    const int64_t y = labels[t];
    lse[t] = l;
    nll[t] = y == ignore ? 0.f : (y >= 0 && y < vocab ? l - tgt[t] : __int_as_float(0x7fc00000));
  }
}

// loss = sum_t nll_t (divided by the number of counted labels for the mean); count = that number.  One CTA.
__global__ void __launch_bounds__(1024) k_xent_reduce(const float* __restrict__ nll, const int64_t* __restrict__ labels,
                                                      int64_t ignore, int T, int mean, float* __restrict__ loss,
                                                      float* __restrict__ count) {
  __shared__ float red[32];
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

// gmax = max |g_t| over the tokens that count, g_t = gout[t gstride] (/ count).  One CTA.
__global__ void __launch_bounds__(1024) k_xent_gmax(const float* __restrict__ gout, int gstride,
                                                    const int64_t* __restrict__ labels, int64_t ignore, int vocab, int T,
                                                    const float* __restrict__ count, float* __restrict__ gmax) {
  __shared__ float red[32];
  float m = 0.f;
  for (int t = threadIdx.x; t < T; t += 1024) {
    const int64_t y = labels[t];
    if (y != ignore && y >= 0 && y < vocab) m = fmaxf(m, fabsf(gout[(int64_t)t * gstride]));
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

// One operand of a product: [rows, k] K-major or [k, rows] MN-major; `box`: rows of the CTA's tile.
static int operand(CUtensorMap* m, bool mn, const void* p, int rows, int k, int64_t ld, int box, int f16) {
  return mn ? map16(m, p, k, rows, ld, 64, f16) : map16(m, p, rows, k, ld, box, f16);
}

template <int EPI, bool A_MN, bool B_MN>
static int product(const void* A, int64_t lda, const void* B, int64_t ldb, Args p, cudaStream_t st) {
  CUtensorMap ma, mb;
  int r = operand(&ma, A_MN, A, p.M, p.K, lda, kBM, p.f16);
  if (r) return r;
  if ((r = operand(&mb, B_MN, B, p.N, p.K, ldb, kBN, p.f16))) return r;
  p.mt = (p.M + kBM - 1) / kBM;
  p.nt = (p.N + kBN - 1) / kBN;
  const size_t smem = 1024 + kStages * (kStageA + kStageB) + 256;
  if ((r = smem_opt_in((const void*)k_xent_gemm<EPI, A_MN, B_MN>, smem, "mpq_xent"))) return r;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  k_xent_gemm<EPI, A_MN, B_MN><<<std::min(p.mt * p.nt, sms), kThreads, smem, st>>>(ma, mb, p);
  return launch_status("mpq_xent product");
}

static bool operand_ok(const void* p, int64_t ld, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld >= cols;
}

}  // namespace xent
}  // namespace mpq

using namespace mpq;

// Vocabulary tiles of the forward pass: `part` holds T x this many float2.
MPQ_API int mpq_xent_tiles(int V) { return V > 0 ? (int)(((int64_t)V + xent::kBN - 1) / xent::kBN) : 0; }

MPQ_API int mpq_xent_forward(int T, int V, int H, int dtype, const void* hidden, int64_t ldh, const void* weight,
                             int64_t ldw, const int64_t* labels, int64_t ignore, float* part, int64_t part_floats,
                             float* tgt, float* lse, float* nll, int* status, void* stream) {
  MPQ_CHECK_ARG(dtype == 1 || dtype == 2, "mpq_xent_forward: dtype must be 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(T >= 0 && V >= 1 && H >= 1 && T <= (1 << 24) && V <= (1 << 30), "mpq_xent_forward: bad shape %d x %d x %d", T, V, H);
  if (T == 0) return MPQ_OK;
  MPQ_CHECK_ARG(hidden && weight && labels && part && tgt && lse && nll && status, "mpq_xent_forward: null pointer");
  MPQ_CHECK_ARG(xent::operand_ok(hidden, ldh, H) && xent::operand_ok(weight, ldw, H),
                "mpq_xent_forward: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  MPQ_CHECK_ARG(part_floats >= 2ll * T * mpq_xent_tiles(V) && (reinterpret_cast<uintptr_t>(part) & 7) == 0,
                "mpq_xent_forward: the workspace needs %lld floats", 2ll * T * mpq_xent_tiles(V));
  MPQ_CHECK_ARG((int64_t)((T + 127) / 128) * mpq_xent_tiles(V) < (1ll << 31), "mpq_xent_forward: too many tiles");
  int st = tc::get_encoder();
  if (st) return st;
  xent::Args p{};
  p.M = T; p.N = V; p.K = H;
  p.f16 = dtype == 2;
  p.status = status;
  p.labels = labels; p.ignore = ignore; p.vocab = V;
  p.part = reinterpret_cast<float2*>(part);
  p.tgt = tgt;
  st = xent::product<xent::kLse, false, false>(hidden, ldh, weight, ldw, p, (cudaStream_t)stream);
  if (st) return st;
  xent::k_xent_join<<<T, 128, 0, (cudaStream_t)stream>>>(p.part, (int)mpq_xent_tiles(V), tgt, labels, ignore, V, lse, nll);
  return launch_status("mpq_xent_forward (join)");
}

MPQ_API int mpq_xent_reduce(int T, const float* nll, const int64_t* labels, int64_t ignore, int mean, float* loss,
                            float* count, void* stream) {
  MPQ_CHECK_ARG(T >= 0 && T <= (1 << 24), "mpq_xent_reduce: bad shape");
  MPQ_CHECK_ARG(loss && count && (T == 0 || (nll && labels)), "mpq_xent_reduce: null pointer");
  xent::k_xent_reduce<<<1, 1024, 0, (cudaStream_t)stream>>>(nll, labels, ignore, T, mean, loss, count);
  return launch_status("mpq_xent_reduce");
}

MPQ_API int mpq_xent_backward(int T, int V, int H, int dtype, const void* hidden, int64_t ldh, const void* weight,
                              int64_t ldw, const int64_t* labels, int64_t ignore, const float* lse, const float* gout,
                              int gstride, const float* count, float* gmax, void* d, int piece, float* acc,
                              void* dhidden, int64_t lddh, void* dweight, int64_t lddw, int* status, void* stream) {
  MPQ_CHECK_ARG(dtype == 1 || dtype == 2, "mpq_xent_backward: dtype must be 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(T >= 0 && V >= 1 && H >= 1 && T <= (1 << 24) && V <= (1 << 30), "mpq_xent_backward: bad shape %d x %d x %d", T, V, H);
  MPQ_CHECK_ARG(piece >= 256 && piece % 256 == 0, "mpq_xent_backward: the piece must be a multiple of 256 columns");
  if (T == 0) return MPQ_OK;
  MPQ_CHECK_ARG(hidden && weight && labels && lse && gout && gmax && d && status, "mpq_xent_backward: null pointer");
  MPQ_CHECK_ARG(xent::operand_ok(hidden, ldh, H) && xent::operand_ok(weight, ldw, H) && xent::operand_ok(d, piece, 0),
                "mpq_xent_backward: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  MPQ_CHECK_ARG(!dhidden || lddh >= H, "mpq_xent_backward: lddh < H");
  MPQ_CHECK_ARG(!dweight || lddw >= H, "mpq_xent_backward: lddw < H");
  MPQ_CHECK_ARG(!dhidden || V <= piece || acc, "mpq_xent_backward: several pieces need the FP32 sum of dhidden");
  int st = tc::get_encoder();
  if (st) return st;
  xent::k_xent_gmax<<<1, 1024, 0, (cudaStream_t)stream>>>(gout, gstride, labels, ignore, V, T, count, gmax);
  if ((st = launch_status("mpq_xent_backward (scale)"))) return st;
  for (int v0 = 0; v0 < V; v0 += piece) {
    const int w = std::min(piece, V - v0);
    const uint16_t* W = reinterpret_cast<const uint16_t*>(weight) + (int64_t)v0 * ldw;
    xent::Args p{};
    p.f16 = dtype == 2;
    p.status = status;
    p.M = T; p.N = w; p.K = H;
    p.labels = labels; p.ignore = ignore; p.vocab = V; p.v0 = v0;
    p.lse = lse; p.gout = gout; p.gstride = gstride; p.count = count; p.gmax = gmax;
    p.out = d; p.ldo = piece;
    if ((st = xent::product<xent::kGrad, false, false>(hidden, ldh, W, ldw, p, (cudaStream_t)stream))) return st;
    if (dhidden) {
      p.M = T; p.N = H; p.K = w;
      p.out = dhidden; p.ldo = lddh;
      p.acc = V > piece ? acc : nullptr;
      p.first = v0 == 0; p.last = v0 + w == V;
      if ((st = xent::product<xent::kOut, false, true>(d, piece, W, ldw, p, (cudaStream_t)stream))) return st;
    }
    if (dweight) {
      p.M = w; p.N = H; p.K = T;
      p.out = reinterpret_cast<uint16_t*>(dweight) + (int64_t)v0 * lddw; p.ldo = lddw;
      p.acc = nullptr;
      if ((st = xent::product<xent::kOut, true, true>(d, piece, hidden, ldh, p, (cudaStream_t)stream))) return st;
    }
  }
  return MPQ_OK;
}
