// Microscaled 4-bit floating point (MX4): quantisation, reading back, and the product of two quantised matrices.
//
// A row is cut into blocks of 32 consecutive elements.  A block holds 32 E2M1 elements q (values 0, 0.5, 1, 1.5, 2, 3,
// 4, 6 and their negatives) and one E8M0 scale code c, and stands for q 2^(c - 127).  With E the biased exponent of
// the block's largest magnitude, c = max(E - 2, 0): the largest magnitude lands in [4, 8) and what rounds above 6
// saturates.  The scaling is a power of two, so x 2^(127 - c) is exact in FP32 and the rounding to E2M1 (nearest, ties
// to even) is the only one.  A block that holds an infinity or a NaN gets c = 255, which reads back as NaN.
//
// Stored form: codes, two to a byte (the even column in the low half), ldc = 16 ceil(cols / 32) bytes a row; scales in
// tiles of 128 rows x 4 blocks, 512 bytes each, [row tile][block tile][512] with byte (r % 32) 16 + (r / 32) 4 + b % 4.
// That is the layout in which the tensor cores take scales (32 lanes x 16 bytes), so a tile moves from memory to TMEM
// as it is.  Blocks and rows that pad a tile carry c = 0.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp4.h>
#include "umma.cuh"

namespace mpq {
namespace mx4 {

using namespace tc;

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

// ------------------------------------------------------------------------------------------------------------------
// Elements
// ------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// 2^(c - 127), NaN for c = 255 (2^-127 is a denormal)
__device__ __forceinline__ float scale_value(uint32_t c) {
  return __uint_as_float(c == 0 ? 0x00400000u : (c == 255 ? 0x7fc00000u : c << 23));
}
// 2^(127 - c) for c < 254 (the largest code of finite data is 252)
__device__ __forceinline__ float scale_inverse(uint32_t c) { return __uint_as_float((254u - c) << 23); }

// The scale code of a block whose largest magnitude has these bits (sign cleared); a NaN's bits exceed infinity's.
__device__ __forceinline__ uint32_t scale_code(uint32_t mag) {
  const uint32_t e = mag >> 23;
  return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

// Eight elements -> eight codes, element i in bits [4 i, 4 i + 4): round to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
  uint32_t r = 0;
  #pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_E2M1, cudaRoundNearest) << (8 * i);
  return r;
}

// Eight codes -> four f16 pairs, exactly.
__device__ __forceinline__ void decode8(uint32_t codes, __half2 (&h)[4]) {
  #pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(codes >> (8 * i)), __NV_E2M1));
}

// Byte of the scale of (row, block) inside the tiled scales of a matrix with kt tiles along its blocks.
__device__ __forceinline__ int64_t scale_at(int64_t row, int block, int kt) {
  return ((row >> 7) * kt + (block >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3);
}

// Eight consecutive elements from column c on, zeros beyond `cols`; 16-byte loads where `vec` allows.
template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c, int cols, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    constexpr int kPer = 16 / sizeof(T);
    #pragma unroll
    for (int i = 0; i < 8; i += kPer) {
      const uint4 raw = *reinterpret_cast<const uint4*>(row + c + i);
      const T* e = reinterpret_cast<const T*>(&raw);
      #pragma unroll
      for (int j = 0; j < kPer; ++j) v[i + j] = to_f32(e[j]);
    }
  } else {
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f32(row[c + i]) : 0.f;
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Quantisation: four lanes to a block, eight elements to a lane
// ------------------------------------------------------------------------------------------------------------------

template <class T>
__global__ void __launch_bounds__(256) k_mx4_quantize(const T* __restrict__ x, int64_t ldx, int rows, int cols, bool vec,
                                                      uint8_t* __restrict__ codes, int64_t ldc,
                                                      uint8_t* __restrict__ scales, int kt) {
  const int nb = (cols + 31) >> 5, rows_pad = (rows + 127) & ~127;
  const int q = blockIdx.x * 256 + threadIdx.x;  // quarter block along the row; kt tiles hold 16 of them
  const int block = q >> 2;
  const bool any = block < 4 * kt;  // whole warps agree: 16 kt quarters and 256 threads are multiples of 16, the
                                    // shuffles below stay inside groups of four
  for (int64_t row = blockIdx.y; row < rows_pad; row += gridDim.y) {
    const bool real = any && row < rows && block < nb;
    float v[8];
    uint32_t mag = 0;
    if (real) {
      load8(x + row * ldx, q * 8, cols, vec, v);
      #pragma unroll
      for (int i = 0; i < 8; ++i) mag = max(mag, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
    mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
    const uint32_t c = scale_code(mag);
    const float inv = c == 255 ? 0.f : scale_inverse(c);
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = real && c != 255 ? v[i] * inv : 0.f;
    const uint32_t word = encode8(v);
    if (real) *reinterpret_cast<uint32_t*>(codes + row * ldc + q * 4) = word;
    if (any && (q & 3) == 0) scales[scale_at(row, block, kt)] = real ? (uint8_t)c : 0;
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Reading back: eight elements to a thread
// ------------------------------------------------------------------------------------------------------------------

template <class T>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* __restrict__ codes, int64_t ldc,
                                                        const uint8_t* __restrict__ scales, int kt, int rows, int cols,
                                                        bool vec, T* __restrict__ out, int64_t ldo) {
  const int c0 = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (c0 >= cols) return;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + row * ldc + c0 / 2);
    const float s = scale_value(scales[scale_at(row, c0 >> 5, kt)]);
    __half2 h[4];
    decode8(w, h);
    alignas(16) T v[8];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = from_f32<T>(f.x * s);
      v[2 * i + 1] = from_f32<T>(f.y * s);
    }
    T* dst = out + row * ldo + c0;
    if (vec && c0 + 8 <= cols) {
      #pragma unroll
      for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
    } else {
      #pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < cols) dst[i] = v[i];
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Product: y[t, n] = sum_k A[t, k] B[n, k] (+ bias[n]), A and B in the stored form, on the block-scaled tensor cores
// ------------------------------------------------------------------------------------------------------------------
//
// One CTA per SM walks 128 x 128 output tiles.  A k-block is one 128-byte swizzle row per operand row = 256 codes, with
// two 512-byte scale tiles for each operand.  Warp 0 fills a ring of stages by TMA; warp 1's elected thread copies the
// stage's scales from shared memory to TMEM (tcgen05.cp, replicated to the four lane quadrants) and issues four MMAs
// of K = 64; warps 2..5 read the FP32 accumulator, add the bias, round once and store.  Two accumulators let the
// epilogue overlap the next tile.  Scale columns in TMEM belong to the stage, so they are not rewritten before the
// MMAs that read them are done.

constexpr int kThreads = 192;
constexpr int kBM = 128, kBN = 128, kStages = 6;
constexpr uint32_t kOperand = 128 * 128, kScale = 1024, kStage = 2 * kOperand + 2 * kScale;
constexpr uint32_t kScaleCols = 256, kStageCols = 16;  // TMEM: accumulators [0, 256), 16 scale columns a stage above

// kind::mxf4 with E8M0 scales of 32 elements: A = B = E2M1, K-major, D = F32, M = m, N = n; `sf`: which half of the
// four scales of a 128-element tile this K = 64 step takes (0 or 2, the same for A and B).
__device__ __forceinline__ uint32_t idesc_mxf4(int m, int n, int sf) {
  return ((uint32_t)sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
         ((uint32_t)(m >> 7) << 27) | ((uint32_t)sf << 29);
}

// Unswizzled descriptor of a 512-byte scale tile: 32 rows of 16 bytes, eight rows to 128 bytes.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) |
         ((uint64_t)1 << 46);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

struct GemmArgs {
  const uint8_t *sfa, *sfb;
  const void* bias;
  void* out;
  int64_t ldo;
  int M, N, kt, mt, nt;
  int* status;
};

template <class T>
__global__ void __launch_bounds__(kThreads, 1)
    k_mx4_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * kStage);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // a stage: A codes, B codes (1024-byte aligned), then the scales of all stages behind the operands of all stages
  auto s_a = [&](int s) { return ring + s * 2 * kOperand; };
  auto s_b = [&](int s) { return ring + s * 2 * kOperand + kOperand; };
  auto s_sf = [&](int s) { return ring + kStages * 2 * kOperand + s * 2 * kScale; };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkb = (p.kt + 1) / 2, tiles = p.mt * p.nt;
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
        const int mb = t % p.mt, nb = t / p.mt;
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = (int)(it % kStages);
          if (*abort_flag || !mbar_wait(&empty[s], ((uint32_t)(it / kStages) & 1u) ^ 1u)) {
            ok = false;
            break;
          }
          const uint32_t sf_bytes = 512u * min(2, p.kt - 2 * kb);
          mbar_expect_tx(&full[s], 2 * kOperand + 2 * sf_bytes);
          tma_load_2d(s_a(s), &map_a, &full[s], kb * 128, mb * kBM);
          tma_load_2d(s_b(s), &map_b, &full[s], kb * 128, nb * kBN);
          bulk_load(s_sf(s), p.sfa + ((int64_t)mb * p.kt + 2 * kb) * 512, sf_bytes, &full[s]);
          bulk_load(s_sf(s) + kScale, p.sfb + ((int64_t)nb * p.kt + 2 * kb) * 512, sf_bytes, &full[s]);
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
          const uint32_t sf = tmem + kScaleCols + s * kStageCols;
          const int ktiles = min(2, p.kt - 2 * kb);
          for (int j = 0; j < ktiles; ++j) {
            asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(sf + j * 4),
                         "l"(scale_desc(smem_u32(s_sf(s)) + j * 512))
                         : "memory");
            asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(sf + 8 + j * 4),
                         "l"(scale_desc(smem_u32(s_sf(s)) + kScale + j * 512))
                         : "memory");
          }
          const uint32_t a0 = smem_u32(s_a(s)), b0 = smem_u32(s_b(s));
          for (int j = 0; j < 2 * ktiles; ++j) {  // steps beyond the last scale tile hold no elements
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "setp.ne.b32 p, %6, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
                    tmem + b * kBN),
                "l"(smem_desc_k_sw128(a0 + j * 32)), "l"(smem_desc_k_sw128(b0 + j * 32)),
                "r"(idesc_mxf4(kBM, kBN, (j & 1) * 2)), "r"(sf + (j >> 1) * 4), "r"(sf + 8 + (j >> 1) * 4),
                "r"((kb > 0 || j > 0) ? 1u : 0u)
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
      const int b = n & 1, mb = t % p.mt, nb = t / p.mt;
      const bool ready = !*abort_flag && mbar_wait(&acc_full[b], (uint32_t)(n >> 1) & 1u);
      if (!__all_sync(0xffffffffu, ready) || *abort_flag) {
        if (!*abort_flag) atomicCAS(p.status, 0, 4);
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int row = mb * kBM + quad * 32 + lane;
      #pragma unroll 1
      for (int c0 = 0; c0 < kBN; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kBN + c0), v);
        const int col = nb * kBN + c0;
        if (row < p.M && col < p.N) {
          T* dst = reinterpret_cast<T*>(p.out) + (int64_t)row * p.ldo + col;
          const T* bias = reinterpret_cast<const T*>(p.bias);
          const int lim = min(32, p.N - col);
          alignas(16) T o[32];
          #pragma unroll
          for (int i = 0; i < 32; ++i) {
            float f = __uint_as_float(v[i]);
            if (bias && i < lim) f += to_f32(bias[col + i]);
            o[i] = from_f32<T>(f);
          }
          if (lim == 32 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
            #pragma unroll
            for (int i = 0; i < (int)(32 * sizeof(T) / 16); ++i)
              reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(o)[i];
          } else {
            #pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < lim) dst[i] = o[i];
          }
        }
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

// Codes as rows of bytes: box = 128 bytes x 128 rows, 128B swizzle, zeros (codes of 0) beyond the matrix.
static int code_map(CUtensorMap* m, const void* p, int rows, int64_t ldc) {
  cuuint64_t dims[2] = {(cuuint64_t)ldc, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ldc};
  cuuint32_t box[2] = {128, 128};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("mpq_mx4_gemm: cuTensorMapEncodeTiled failed (%d) rows=%d ldc=%lld", (int)r, rows, (long long)ldc);
    return MPQ_ERR_ARG;
  }
  return MPQ_OK;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class T>
static int quantize(const void* x, int64_t ldx, int rows, int cols, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  const int nb = (cols + 31) / 32, kt = (nb + 3) / 4;
  const bool vec = aligned16(x) && (ldx * (int64_t)sizeof(T)) % 16 == 0;
  dim3 grid((16 * kt + 255) / 256, std::min((rows + 127) / 128 * 128, 65535));
  k_mx4_quantize<T><<<grid, 256, 0, st>>>((const T*)x, ldx, rows, cols, vec, codes, 16 * (int64_t)nb, scales, kt);
  return launch_status("mpq_mx4_quantize");
}

template <class T>
static int dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int cols, void* out, int64_t ldo,
                      cudaStream_t st) {
  const int nb = (cols + 31) / 32, kt = (nb + 3) / 4;
  const bool vec = aligned16(out) && (ldo * (int64_t)sizeof(T)) % 16 == 0;
  dim3 grid((cols + 2047) / 2048, std::min(rows, 65535));
  k_mx4_dequantize<T><<<grid, 256, 0, st>>>(codes, 16 * (int64_t)nb, scales, kt, rows, cols, vec, (T*)out, ldo);
  return launch_status("mpq_mx4_dequantize");
}

template <class T>
static int gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& p, cudaStream_t st) {
  const size_t smem = 1024 + kStages * kStage + 256;
  const int ast = smem_opt_in((const void*)k_mx4_gemm<T>, smem, "mpq_mx4_gemm");
  if (ast) return ast;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int grid = std::min(p.mt * p.nt, sms);
  k_mx4_gemm<T><<<grid, kThreads, smem, st>>>(a, b, p);
  return launch_status("mpq_mx4_gemm");
}

}  // namespace mx4
}  // namespace mpq

using namespace mpq;

#define MX4_BY_TYPE(dtype, fn, ...)                         \
  ((dtype) == mx4::kF32    ? mx4::fn<float>(__VA_ARGS__)    \
   : (dtype) == mx4::kBF16 ? mx4::fn<__nv_bfloat16>(__VA_ARGS__) \
                           : mx4::fn<__half>(__VA_ARGS__))

MPQ_API int mpq_mx4_quantize(const void* x, int dtype, int64_t ldx, int rows, int cols, uint8_t* codes, uint8_t* scales,
                             void* stream) {
  MPQ_CHECK_ARG(dtype >= 0 && dtype <= 2, "mpq_mx4_quantize: dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(rows >= 0 && cols >= 0 && rows <= 0x7fffff00 && cols <= 0x7fffff00 && ldx >= cols,
                "mpq_mx4_quantize: bad shape %d x %d (ld %lld)", rows, cols, (long long)ldx);
  if (rows == 0 || cols == 0) return MPQ_OK;
  MPQ_CHECK_ARG(x && codes && scales, "mpq_mx4_quantize: null pointer");
  MPQ_CHECK_ARG(mx4::aligned16(codes) && mx4::aligned16(scales), "mpq_mx4_quantize: codes and scales must be 16-byte aligned");
  return MX4_BY_TYPE(dtype, quantize, x, ldx, rows, cols, codes, scales, (cudaStream_t)stream);
}

MPQ_API int mpq_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int cols, void* out, int dtype,
                               int64_t ldo, void* stream) {
  MPQ_CHECK_ARG(dtype >= 0 && dtype <= 2, "mpq_mx4_dequantize: dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(rows >= 0 && cols >= 0 && rows <= 0x7fffff00 && cols <= 0x7fffff00 && ldo >= cols,
                "mpq_mx4_dequantize: bad shape %d x %d (ld %lld)", rows, cols, (long long)ldo);
  if (rows == 0 || cols == 0) return MPQ_OK;
  MPQ_CHECK_ARG(codes && scales && out, "mpq_mx4_dequantize: null pointer");
  MPQ_CHECK_ARG(mx4::aligned16(codes) && mx4::aligned16(scales),
                "mpq_mx4_dequantize: codes and scales must be 16-byte aligned");
  return MX4_BY_TYPE(dtype, dequantize, codes, scales, rows, cols, out, ldo, (cudaStream_t)stream);
}

MPQ_API int mpq_mx4_gemm(int M, int N, int K, const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                         const uint8_t* b_scales, const void* bias, void* out, int dtype, int64_t ldo, int* status,
                         void* stream) {
  MPQ_CHECK_ARG(dtype >= 0 && dtype <= 2, "mpq_mx4_gemm: dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && K <= 0x7fffff00 && ldo >= N, "mpq_mx4_gemm: bad shape %d x %d x %d", M, N, K);
  if (M == 0 || N == 0) return MPQ_OK;
  MPQ_CHECK_ARG(a_codes && a_scales && b_codes && b_scales && out && status, "mpq_mx4_gemm: null pointer");
  MPQ_CHECK_ARG(mx4::aligned16(a_codes) && mx4::aligned16(a_scales) && mx4::aligned16(b_codes) && mx4::aligned16(b_scales),
                "mpq_mx4_gemm: codes and scales must be 16-byte aligned");
  int st = tc::get_encoder();
  if (st) return st;
  const int nb = (K + 31) / 32;
  mx4::GemmArgs p{a_scales, b_scales, bias, out, ldo, M, N, (nb + 3) / 4, (M + 127) / 128, (N + 127) / 128, status};
  MPQ_CHECK_ARG((int64_t)p.mt * p.nt <= 0x7fffffff, "mpq_mx4_gemm: too many tiles");
  CUtensorMap ma, mb;
  if ((st = mx4::code_map(&ma, a_codes, M, 16 * (int64_t)nb))) return st;
  if ((st = mx4::code_map(&mb, b_codes, N, 16 * (int64_t)nb))) return st;
  return MX4_BY_TYPE(dtype, gemm, ma, mb, p, (cudaStream_t)stream);
}
