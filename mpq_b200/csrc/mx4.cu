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
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp4.h>
#include "umma.cuh"

namespace mpq {
namespace mx4 {

using namespace tc;

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

constexpr int kTimedOut = 10;  // added to the code of a wait that ran out: whose it was

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

template <class T>
constexpr int type_code() { return sizeof(T) == 4 ? kF32 : (std::is_same<T, __half>::value ? kF16 : kBF16); }

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
// The same with one instruction a pair, each taking its byte out of the word by itself, where the function above adds a
// shift and a mask.  Only for code that a warp runs together: in code that diverges, ptxas 12.9.86 has lost the
// operands of this form (seen in reading back and, with the opposite conversion, in quantisation; the cause is not known).
// The use below is checked code by code, at every place of a block, in slices of K and rounds of rows.
__device__ __forceinline__ void decode8_together(uint32_t codes, __half2 (&h)[4]) {
  uint32_t r[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(codes));
  #pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2*>(&r[i]);
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
// Quantisation and reading back
// ------------------------------------------------------------------------------------------------------------------
//
// Both move memory: 4 or 2 bytes in and 17/32 out for an element, or the reverse, which at the memory's rate leaves some
// ten instructions an element.  Quantisation gives half a block to a thread: its partner's maximum is one shuffle away,
// and for 16-bit types the maximum is taken two elements at a time.  (With a quarter block to a thread and every
// element in 32 bits it ran 17 instructions an element, 2.5 TB/s.)  Reading back gives 16 bytes of the result to a
// thread.  A thread issues its kRows rows' loads before it uses the first, and a CTA of 256 threads covers as many rows
// side by side as a narrow matrix leaves room for.

constexpr int kRows = 2;

// Sixteen elements of a row as they are stored.
template <class T>
struct Half {
  static constexpr int kWords = 16 * sizeof(T) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* __restrict__ row, int c, int cols, bool vec) {
    if (vec && c + 16 <= cols) {
      #pragma unroll
      for (int i = 0; i < kWords / 4; ++i)
        *reinterpret_cast<uint4*>(w + 4 * i) = __ldcs(reinterpret_cast<const uint4*>(row + c) + i);
    } else {
      #pragma unroll
      for (int i = 0; i < 16; ++i) reinterpret_cast<T*>(w)[i] = c + i < cols ? row[c + i] : T(0.f);
    }
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(reinterpret_cast<const T*>(w)[i]); }
  // the largest magnitude's FP32 bits
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
      #pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
      #pragma unroll
      for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = max(m & 0xffffu, m >> 16);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
      else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
  }
};

template <class T>
__global__ void __launch_bounds__(256) k_mx4_quantize(const T* __restrict__ x, int64_t ldx, int rows, int cols, bool vec,
                                                      uint8_t* __restrict__ codes, int64_t ldc,
                                                      uint8_t* __restrict__ scales, int kt) {
  allow_behind();  // a product launched behind may set itself up
  // blockDim.x is a multiple of 8 (a scale tile's width in half blocks): partners sit in one warp
  const int nb = (cols + 31) >> 5, rows_pad = (rows + 127) & ~127;
  const int q = blockIdx.y * blockDim.x + threadIdx.x, block = q >> 1;
  const int row0 = (blockIdx.x * blockDim.y + threadIdx.y) * kRows;
  const uint32_t two = 3u << ((threadIdx.y * blockDim.x + threadIdx.x) & 30);  // the block's lanes
  if (block >= 4 * kt) return;
  Half<T> h[kRows];
  #pragma unroll
  for (int r = 0; r < kRows; ++r) {
    #pragma unroll
    for (int i = 0; i < Half<T>::kWords; ++i) h[r].w[i] = 0;
    if (row0 + r < rows && block < nb) h[r].load(x + (int64_t)(row0 + r) * ldx, q * 16, cols, vec);
  }
  uint8_t* code = codes + (int64_t)row0 * ldc + q * 8;
  #pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int row = row0 + r;
    uint32_t mag = h[r].largest();
    mag = max(mag, __shfl_xor_sync(two, mag, 1));
    const uint32_t c = scale_code(mag);
    const float inv = c == 255 ? 0.f : scale_inverse(c);  // a block that is not finite reads back as NaN anyway
    uint2 word;
    #pragma unroll
    for (int k = 0; k < 2; ++k) {
      float v[8];
      #pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = h[r].at(8 * k + i) * inv;
      (k ? word.y : word.x) = encode8(v);
    }
    if (row < rows && block < nb) *reinterpret_cast<uint2*>(code + r * ldc) = word;
    if (row < rows_pad && (q & 1) == 0) scales[scale_at(row, block, kt)] = (uint8_t)c;
  }
}

template <class T>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* __restrict__ codes, int64_t ldc,
                                                        const uint8_t* __restrict__ scales, int kt, int rows, int cols,
                                                        bool vec, T* __restrict__ out, int64_t ldo) {
  constexpr int kPer = 16 / sizeof(T);  // elements of a thread and row
  const int c0 = (blockIdx.y * blockDim.x + threadIdx.x) * kPer;
  const int row0 = (blockIdx.x * blockDim.y + threadIdx.y) * kRows * 2;
  if (c0 >= cols) return;
  uint32_t w[kRows * 2], c[kRows * 2];
  #pragma unroll
  for (int r = 0; r < kRows * 2; ++r) {
    const int row = min(row0 + r, rows - 1);
    const uint8_t* at = codes + (int64_t)row * ldc + c0 / 2;
    w[r] = kPer == 8 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
    c[r] = scales[scale_at(row, c0 >> 5, kt)];
  }
  #pragma unroll
  for (int r = 0; r < kRows * 2; ++r) {
    if (row0 + r >= rows) break;
    const float s = scale_value(c[r]);
    __half2 h[4];
    decode8(w[r], h);
    alignas(16) T v[kPer];
    #pragma unroll
    for (int i = 0; i < kPer / 2; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = from_f32<T>(f.x * s);
      v[2 * i + 1] = from_f32<T>(f.y * s);
    }
    T* dst = out + (int64_t)(row0 + r) * ldo + c0;
    if (vec && c0 + kPer <= cols) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
    } else {
      #pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (c0 + i < cols) dst[i] = v[i];
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Product for one or two tokens: y[t, n] = sum_k Q(x)[t, k] W[n, k] (+ bias[n]), x quantised in the same launch
// ------------------------------------------------------------------------------------------------------------------
//
// W is read once (17 bytes for 32 weights), and the arithmetic has to keep up with that: a block of a row takes 16
// conversions of two codes to an f16 pair and 16 f16 products a token.  The products are exact: they are multiples of
// 1/4 up to 36, and the eight that a half of an accumulator adds stay below 2^11 quarters; a block's four sums are
// added in FP32 and scaled by 2^(cx + cw - 254) once.  1 x 4096 x 14336 takes 9.9 us, 3.2 TB/s (13.0 with a shift and a
// mask to every conversion; 14.1 with byte permutations and dp4a, twice the instructions).
// The scales apply one after the other, W's first: their product may lie outside FP32 where the result does not (x
// holding its type's lowest value, and a 0 in W for it).  So that no step overflows by itself, x's f16 values carry 2^-10
// of its block's scale: a sum is then at most 1.125, times 2^127 at most.  Where x's scale has no room for the 2^10 in
// return, its values keep as much more, and what overflows is the result.
// Every CTA quantises x for itself into shared memory (f16 values in four planes of 16 bytes a block, so that a warp's
// reads are free of conflicts) while its first weights are on their way.  A warp takes kFewRows rows of W and one of
// `slices` parts of K (so that all warps have work whatever N is), a lane every 32nd block; the next blocks are loaded
// before the last are used.  (With a deeper ring in shared memory it took 15.0 us instead of 13.0: the arithmetic bounds
// it, not the latency.)

constexpr int kFewRows = 4, kFewThreads = 256, kFewWarps = kFewThreads / 32;

template <class T, int TOK>
__global__ void __launch_bounds__(kFewThreads, 3)
    k_mx4_few(const T* __restrict__ x, int64_t ldx, int tokens, int N, int K, bool vec, const uint8_t* __restrict__ codes,
              const uint8_t* __restrict__ scales, const T* __restrict__ bias, T* __restrict__ out, int64_t ldo,
              int slices) {
  extern __shared__ __align__(16) unsigned char sm[];
  __shared__ float part[2][kFewWarps][kFewRows * TOK];
  const int nb = (K + 31) >> 5, kt = (nb + 3) >> 2;
  uint4* xb = reinterpret_cast<uint4*>(sm);                        // [TOK][4][nb]
  float* xs = reinterpret_cast<float*>(xb + (size_t)TOK * 4 * nb);  // [TOK][nb]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = warp % slices, wide = kFewWarps / slices;  // a CTA takes `wide` groups of rows at a time
  const int iters = (nb + 31) >> 5, i0 = iters * slice / slices, i1 = iters * (slice + 1) / slices;
  const int groups = (N + kFewRows - 1) / kFewRows, rounds = (groups + wide - 1) / wide;

  uint4 raw[kFewRows];
  uint32_t sc[kFewRows];
  auto load = [&](int n0, int i) {  // n0 is a multiple of 4: a group's rows are neighbours in their scale tile
    const int b = lane + 32 * i;
    #pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
      raw[r] = make_uint4(0, 0, 0, 0);
      sc[r] = 0;
    }
    if (b < nb) {
      const uint4* at = reinterpret_cast<const uint4*>(codes) + (int64_t)n0 * nb + b;
      const uint8_t* s = scales + scale_at(n0, b, kt);
      #pragma unroll
      for (int r = 0; r < kFewRows; ++r) {
        raw[r] = __ldcs(at + min(r, N - 1 - n0) * nb);
        sc[r] = s[r * 16];
      }
    }
  };
  int round = blockIdx.x;
  int n0 = (round * wide + warp / slices) * kFewRows;
  if (n0 < N) load(n0, i0);

  for (int i = threadIdx.x; i < TOK * 16 * kt; i += kFewThreads) {  // quarter blocks; 16 kt of them to a token
    const int t = i / (16 * kt), q = i - t * 16 * kt, block = q >> 2;
    const bool real = t < tokens && block < nb;
    float v[8];
    #pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (real) load8(x + t * ldx, q * 8, K, vec, v);
    uint32_t mag = 0;
    #pragma unroll
    for (int j = 0; j < 8; ++j) mag = max(mag, __float_as_uint(v[j]) & 0x7fffffffu);
    const uint32_t four = 0xfu << (lane & ~3);  // the block's lanes: a warp's last pass may be partial
    mag = max(mag, __shfl_xor_sync(four, mag, 1));
    mag = max(mag, __shfl_xor_sync(four, mag, 2));
    const uint32_t c = scale_code(mag);
    const float inv = c == 255 ? 0.f : scale_inverse(c);
    #pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * inv;
    __half2 h[4];
    decode8(encode8(v), h);
    const uint32_t kept = c > 244 ? min(c - 244, 10u) : 0;  // the values take 2^(kept - 10) of the scale, a normal number
    const __half2 part = __half2half2(__ushort_as_half((unsigned short)((kept + 5) << 10)));
    #pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __hmul2(h[j], part);
    if (block < nb) {
      xb[((size_t)t * 4 + (q & 3)) * nb + block] = *reinterpret_cast<const uint4*>(h);
      if ((q & 3) == 0) xs[t * nb + block] = c == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((c + 10 - kept) << 23);
    }
  }
  __syncthreads();

  for (int turn = 0; round < rounds; round += gridDim.x, turn ^= 1) {
    float acc[TOK][kFewRows];
    #pragma unroll
    for (int t = 0; t < TOK; ++t)
      #pragma unroll
      for (int r = 0; r < kFewRows; ++r) acc[t][r] = 0.f;
    const int next = ((round + gridDim.x) * wide + warp / slices) * kFewRows;
    if (n0 < N) {
      #pragma unroll 1
      for (int i = i0; i < i1; ++i) {
        const int b = min(lane + 32 * i, nb - 1);  // beyond the last block the weights are zeros
        uint4 w[kFewRows];
        float sw[kFewRows];
        #pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
          w[r] = raw[r];
          sw[r] = scale_value(sc[r]);
        }
        if (i + 1 < i1) load(n0, i + 1);
        else if (next < N) load(next, i0);
        __half2 lo[TOK][kFewRows], hi[TOK][kFewRows];  // sums of the block's first and last 16 products
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
          __half2 xv[TOK][4];
          #pragma unroll
          for (int t = 0; t < TOK; ++t) *reinterpret_cast<uint4*>(xv[t]) = xb[((size_t)t * 4 + q) * nb + b];
          #pragma unroll
          for (int r = 0; r < kFewRows; ++r) {
            __half2 h[4];
            decode8_together(q == 0 ? w[r].x : (q == 1 ? w[r].y : (q == 2 ? w[r].z : w[r].w)), h);
            #pragma unroll
            for (int t = 0; t < TOK; ++t) {
              __half2& sum = q < 2 ? lo[t][r] : hi[t][r];
              sum = (q & 1) ? __hfma2(h[0], xv[t][0], sum) : __hmul2(h[0], xv[t][0]);
              #pragma unroll
              for (int j = 1; j < 4; ++j) sum = __hfma2(h[j], xv[t][j], sum);
            }
          }
        }
        #pragma unroll
        for (int t = 0; t < TOK; ++t) {
          const float s = xs[t * nb + b];
          #pragma unroll
          for (int r = 0; r < kFewRows; ++r) {
            const float2 f = __half22float2(lo[t][r]), g = __half22float2(hi[t][r]);
            acc[t][r] = fmaf(((f.x + f.y) + (g.x + g.y)) * sw[r], s, acc[t][r]);
          }
        }
      }
    }
    #pragma unroll
    for (int t = 0; t < TOK; ++t) {
      const float y = warp_sum4(acc[t], lane);  // lane r: row r
      if (slices > 1) {
        if (lane < kFewRows) part[turn][warp][t * kFewRows + lane] = y;
      } else if (lane < kFewRows && n0 + lane < N && t < tokens) {
        const int n = n0 + lane;
        out[(int64_t)t * ldo + n] = from_f32<T>(bias ? y + to_f32(bias[n]) : y);
      }
    }
    if (slices > 1) {  // the parts in order; the other buffer takes the next round's, so one barrier is enough
      __syncthreads();
      for (int j = threadIdx.x; j < wide * kFewRows * TOK; j += kFewThreads) {
        const int g = j / (kFewRows * TOK), e = j - g * kFewRows * TOK;
        const int n = (round * wide + g) * kFewRows + e % kFewRows, t = e / kFewRows;
        if (n < N && t < tokens) {
          float y = 0.f;
          for (int k = 0; k < slices; ++k) y += part[turn][g * slices + k][e];
          out[(int64_t)t * ldo + n] = from_f32<T>(bias ? y + to_f32(bias[n]) : y);
        }
      }
    }
    n0 = next;
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Product: y[t, n] = sum_k A[t, k] B[n, k] (+ bias[n]), A and B in the stored form, on the block-scaled tensor cores
// ------------------------------------------------------------------------------------------------------------------
//
// Two kernels.  k_mx4_tile, for few rows of A: one CTA per SM walks 128 x BN output tiles (BN = 64 or 128: narrow tiles
// spread few tokens' work over more SMs; a narrower one's scales would start at an odd TMEM column, which is not an
// address that the MMA takes).  A k-block is one 128-byte swizzle row per operand row = 256 codes, with two 512-byte
// scale tiles for each operand.  Warp 0 fills a ring of stages by TMA; warp 6 copies the stages' scales from shared memory
// to TMEM (tcgen05.cp, replicated to the four lane quadrants); warp 1's elected thread issues four MMAs of K = 64 a
// stage; warps 2..5 read the FP32 accumulator, add the bias, round once and store.  Two accumulators let the epilogue
// overlap the next tile.  Scale columns in TMEM belong to the stage, so they are not rewritten before the MMAs that read
// them are done.
//
// With at most 128 rows of A only those are loaded (a tile load takes two to three cycles a 128-byte row; what the
// others' shared memory holds stays in their rows of the accumulator) and the ring takes the more stages for it.  A
// cluster of up to four CTAs may share a tile, each with a part of K: they leave their FP32 sums in shared memory, and
// each adds the parts of its share of the columns, in order.  7 x 14336 x 4096 takes 14 us, of which the tensor cores'
// steps are 5 and the weights at the memory's rate 5; the rest is the quantisation before it, filling the ring and the
// sum over the cluster, one after the other.  (With the scale copies issued by the MMAs' thread a k-block took 740
// cycles: 8 x 4096 x 14336 13.4 us instead of 11.8; with x quantised here, by every CTA, 19.6.)

constexpr int kThreads = 224;
constexpr int kBM = 128, kMostStages = 16;
constexpr uint32_t kTileRing = 204 * 1024;
constexpr uint32_t kOperand = 128 * 128, kScale = 1024;
constexpr uint32_t kScaleCols = 256, kStageCols = 16;   // TMEM: accumulators [0, 256), 16 scale columns a stage above

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

template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// What this thread has issued -> one arrival on a barrier of its CTA.
template <int CTAS>
__device__ __forceinline__ void commit_one(uint64_t* bar) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t add) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(add)
        : "memory");
}

struct GemmArgs {
  const uint8_t *sfa, *sfb;
  const void* bias;
  void* out;
  int64_t ldo;
  int M, N, kt, mt, nt;  // kt: scale tiles along K; mt x nt output tiles
  int a_rows;            // k_mx4_tile: rows of A that a tile loads
  int stages;            // k_mx4_tile: of the ring
  int tile_out;          // the result's rows are aligned for tile stores
  int* status;
};

// kCols<T> columns of the accumulator are 128 bytes of a row.  Columns col.. of a warp's 32 rows from row0 on (`lane`:
// the thread's row): bias, one rounding, and off as a tile, or row by row where the result's rows are not aligned.
template <class T>
constexpr int kCols = 128 / sizeof(T);

// 128 bytes of a row, rounded two at a time.
template <class T>
__device__ __forceinline__ void pack_row(const float* v, uint32_t (&w)[32]) {
  #pragma unroll
  for (int i = 0; i < 32; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}

template <class T>
__device__ __forceinline__ void store_rows(const GemmArgs& p, const CUtensorMap* map, unsigned char* buf, int lane,
                                           int row0, int col, const float* v) {
  const int lim = p.N - col;
  if (lim <= 0 || row0 >= p.M) return;  // the same for the warp
  uint32_t w[32];
  if (p.bias) {  // a lane's columns, passed around the warp
    const T* bias = reinterpret_cast<const T*>(p.bias) + col;
    float own[kCols<T> / 32], f[kCols<T>];
    #pragma unroll
    for (int i = 0; i < kCols<T> / 32; ++i) own[i] = lane + 32 * i < lim ? to_f32(bias[lane + 32 * i]) : 0.f;
    #pragma unroll
    for (int i = 0; i < kCols<T>; ++i) f[i] = v[i] + __shfl_sync(0xffffffffu, own[i >> 5], i & 31);
    pack_row<T>(f, w);
  } else {
    pack_row<T>(v, w);
  }
  chunk_put(buf, lane, w);
  if (p.tile_out)
    chunk_send(buf, lane, map, col, row0, 0);
  else
    chunk_rows<sizeof(T)>(buf, lane, reinterpret_cast<T*>(p.out) + (int64_t)row0 * p.ldo + col, p.ldo * sizeof(T),
                          p.M - row0, lim);
}

// kCols<T> columns of TMEM
template <int C>
__device__ __forceinline__ void tmem_cols(uint32_t at, float (&v)[C]) {
  #pragma unroll
  for (int c = 0; c < C; c += 32) {
    uint32_t t[32];
    tmem_ld32(at + c, t);
    #pragma unroll
    for (int i = 0; i < 32; ++i) v[c + i] = __uint_as_float(t[i]);
  }
}

template <class T, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    k_mx4_tile(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfb,
               const __grid_constant__ CUtensorMap map_o, const GemmArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t kOperandB = BN * 128;
  const uint32_t stage = kOperandB + p.a_rows * 128;
  // ring: B then A of each stage (1024-byte aligned), then the scales of all stages (A's, B's)
  unsigned char* out_buf = ring + kTileRing;  // 4 KB to an epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(out_buf + 4 * 4096);
  uint64_t* empty = full + kMostStages;
  uint64_t* acc_full = empty + kMostStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* sf_full = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_full + kMostStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto s_b = [&](int s) { return ring + s * stage; };
  auto s_a = [&](int s) { return ring + s * stage + kOperandB; };
  auto s_sf = [&](int s) { return ring + p.stages * stage + s * 2 * kScale; };
  float* part_sum = reinterpret_cast<float*>(ring);  // [BN][128] at the end of a part of K

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a cluster of `parts` CTAs shares a tile (more than one only where the grid holds every tile once)
  const int rank = (int)cluster_rank(), parts = (int)cluster_size();
  const int nkb = (p.kt + 1) / 2, kb0 = nkb * rank / parts, kb1 = nkb * (rank + 1) / parts;
  const int tiles = p.mt * p.nt, first_tile = blockIdx.x / parts, stride = gridDim.x / parts;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&sf_full[s], 1);
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
      const uint32_t bytes = stage + 2 * kScale;
      int64_t it = 0;
      Ring r(p.stages);
      bool ok = true;
      // The first tile's first weights, which no kernel before has made; A may come from one, so its loads wait for
      // that kernel's end.
      const int ahead = first_tile < tiles ? min(p.stages, kb1 - kb0) : 0, nb0 = first_tile / p.mt;
      for (int i = 0; i < ahead; ++i) {
        mbar_expect_tx(&full[i], bytes);
        tma_load_2d(s_b(i), &map_b, &full[i], (kb0 + i) * 128, nb0 * BN);
        tma_load_2d(s_sf(i) + kScale, &map_sfb, &full[i], (kb0 + i) * 256, nb0 * BN >> 7);
      }
      wait_before();
      for (int t = first_tile; t < tiles && ok; t += stride) {
        const int mb = t % p.mt, nb = t / p.mt;
        for (int kb = kb0; kb < kb1; ++kb, ++it, r.next()) {
          uint64_t* bar = &full[r.s];
          if (it >= ahead) {
            if (!mbar_wait_fast(&empty[r.s], r.ph ^ 1u) || *abort_flag) {
              ok = false;
              break;
            }
            mbar_expect_tx(bar, bytes);
            tma_load_2d(s_b(r.s), &map_b, bar, kb * 128, nb * BN);
            tma_load_2d(s_sf(r.s) + kScale, &map_sfb, bar, kb * 256, nb * BN >> 7);
          }
          tma_load_2d(s_a(r.s), &map_a, bar, kb * 128, mb * kBM);
          tma_load_2d(s_sf(r.s), &map_sfa, bar, kb * 256, mb);
        }
      }
      if (!ok) {  // drain the copies in flight (each wait bounded) before the CTA may end
        *abort_flag = 1;
        for (int i = 0; i < p.stages && i < it; ++i) {
          r.back();
          mbar_wait_fast(&full[r.s], r.ph);
        }
        atomicCAS(p.status, 0, kTimedOut + 2);
      }
    }
  } else if (warp == 1) {
    const bool lead = elect_one();
    const uint64_t da0 = smem_desc_k_sw128(smem_u32(s_a(0))), db0 = smem_desc_k_sw128(smem_u32(s_b(0)));
    const uint32_t i0 = idesc_mxf4(kBM, BN, 0), i2 = idesc_mxf4(kBM, BN, 2);
    Ring r(p.stages);
    bool ok = true;
    int n = 0;
    for (int t = first_tile; t < tiles && ok; t += stride, ++n) {
      const uint32_t acc = tmem + (n & 1) * BN;
      if (!warp_agrees(mbar_wait_fast(&acc_empty[n & 1], ((uint32_t)(n >> 1) & 1u) ^ 1u) && !*abort_flag)) {
        ok = false;
        break;
      }
      const uint32_t part = (uint32_t)((t / p.mt) * BN & 127) >> 5;  // the tile's column in its scale tile
      for (int kb = kb0; kb < kb1; ++kb, r.next()) {
        if (!warp_agrees(mbar_wait_fast(&sf_full[r.s], r.ph))) {  // the step's operands and scales are in place
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sf = tmem + kScaleCols + r.s * kStageCols;  // A's 2 x 4 columns, then B's
        const uint64_t da = desc_add(da0, r.s * stage), db = desc_add(db0, r.s * stage);
        const uint32_t add = kb > kb0;
        if (lead) {  // scales beyond the matrix are zeros, as are its codes
          #pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_mxf4<1>(acc, desc_add(da, j * 32), desc_add(db, j * 32), j & 1 ? i2 : i0, sf + (j >> 1) * 4,
                        sf + 8 + (j >> 1) * 4 + part, j ? 1u : add);
          commit_one<1>(&empty[r.s]);
        }
        __syncwarp();
      }
      // the accumulator is complete (or, after an abort, the issued MMAs have retired)
      if (lead) commit_one<1>(&acc_full[n & 1]);
      __syncwarp();
    }
    if (!ok && lead) {
      *abort_flag = 1;
      atomicCAS(p.status, 0, kTimedOut + 3);
    }
  } else if (warp == 6) {
    const bool lead = elect_one();
    const uint64_t ds0 = scale_desc(smem_u32(s_sf(0)));
    Ring c(p.stages);
    const int64_t steps = first_tile < tiles ? (int64_t)((tiles - first_tile + stride - 1) / stride) * (kb1 - kb0) : 0;
    bool ok = true;
    for (int64_t i = 0; i < steps; ++i, c.next()) {
      // a stage is filled again once its MMAs are done, which frees its scale columns in TMEM as well
      if (!warp_agrees(mbar_wait_fast(&full[c.s], c.ph) && !*abort_flag)) {
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t sf = tmem + kScaleCols + c.s * kStageCols;
      const uint64_t ds = desc_add(ds0, c.s * 2 * kScale);
      if (lead) {
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          copy_scales<1>(sf + j * 4, desc_add(ds, j * 512));
          copy_scales<1>(sf + 8 + j * 4, desc_add(ds, kScale + j * 512));
        }
        commit_one<1>(&sf_full[c.s]);
      }
      __syncwarp();
    }
    if (!ok && lead) {
      *abort_flag = 1;
      atomicCAS(p.status, 0, kTimedOut + 5);
    }
  } else {
    const int quad = warp & 3;
    int n = 0;
    for (int t = first_tile; t < tiles; t += stride, ++n) {
      const int b = n & 1, mb = t % p.mt, nb = t / p.mt;
      const bool ready = !*abort_flag && mbar_wait_fast(&acc_full[b], (uint32_t)(n >> 1) & 1u);
      if (!__all_sync(0xffffffffu, ready) || *abort_flag) {
        if (!*abort_flag) atomicCAS(p.status, 0, kTimedOut + 4);
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * BN);
      #pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += kCols<T>) {
        float v[kCols<T>];
        tmem_cols(at + c0, v);
        if (parts > 1) {  // every load of the ring has been consumed: it holds this part, column by column
          if (quad * 32 < p.M) {
            #pragma unroll
            for (int i = 0; i < kCols<T>; ++i) part_sum[(c0 + i) * kBM + quad * 32 + lane] = v[i];
          }
        } else {
          store_rows<T>(p, &map_o, out_buf + quad * 4096, lane, mb * kBM + quad * 32, nb * BN + c0, v);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
  }
  if (warp >= 2 && parts == 1) chunk_drain(lane);
  __syncwarp();
  if (parts > 1) {
    cluster_sync();  // the parts are complete
    const int quad = warp & 3, row = quad * 32 + lane;  // one row tile
    if (warp >= 2 && warp < 6 && quad * 32 < p.M && !*abort_flag) {
      // each CTA adds the parts of its share of the columns, in order
      #pragma unroll 1
      for (int c0 = rank * kCols<T>; c0 < BN; c0 += parts * kCols<T>) {
        float v[kCols<T>];
        #pragma unroll
        for (int i = 0; i < kCols<T>; ++i) v[i] = 0.f;
        for (int r = 0; r < parts; ++r) {
          const uint32_t at = mapa(smem_u32(part_sum + c0 * kBM + row), r);
          #pragma unroll
          for (int i = 0; i < kCols<T>; ++i) {
            float f;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(at + i * kBM * 4));
            v[i] += f;
          }
        }
        store_rows<T>(p, &map_o, out_buf + quad * 4096, lane, quad * 32, first_tile * BN + c0, v);
      }
      chunk_drain(lane);
    }
    __syncwarp();
    cluster_sync();  // the parts have been read
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// k_mx4_pair, for many rows of A: a pair of CTAs computes 256 x 256 tiles (tcgen05 cta_group::2, M = N = 256), each CTA
// loading 128 rows of A and of B a k-block.  An MMA takes 128 cycles whatever its N, so N is the full 256.  What bounds
// the rate is the thread that issues the MMAs: a step's four take it 200 cycles, their commit 95 and a wait 140, out of
// 512; so the six scale copies of a step are another warp's, which runs up to a ring ahead (in one warp with them a step
// took 680 to 760 cycles).  TMEM holds one accumulator and the scales of 5 stages (24 columns each: 8 of A's 128 rows,
// 16 of B's 256, the latter in both CTAs); the epilogue takes the accumulator into registers at once, so that the next
// tile's MMAs wait for the reading only.  16384 x 4096 x 14336: 380 us, 5.1 PFLOP/s, and 440 under the power limit that
// a longer run reaches; 300 without the result's stores (470 MB).

constexpr int kPairWarps = 8, kPairThreads = 96 + 32 * kPairWarps, kPairStages = 5, kPairGroup = 8;
constexpr int kPM = 256, kPN = 256;
constexpr uint32_t kPairOps = 2 * kOperand, kPairSf = 3 * kScale;
constexpr uint32_t kPairCols = 24;  // TMEM columns of a stage's scales, above the accumulator's 256

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    k_mx4_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfb,
               const __grid_constant__ CUtensorMap map_o, const GemmArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* out_buf = ring + kPairStages * (kPairOps + kPairSf);  // 4 KB to an epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(out_buf + kPairWarps * 4096);
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* sf_full = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_full + kPairStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto s_a = [&](int s) { return ring + s * kPairOps; };
  auto s_b = [&](int s) { return ring + s * kPairOps + kOperand; };
  auto s_sf = [&](int s) { return ring + kPairStages * kPairOps + s * kPairSf; };  // A's tile pair, then B's two

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;
  const int nkb = (p.kt + 1) / 2, tiles = p.mt * p.nt;
  auto tile_at = [&](int t, int& mb, int& nb) {  // kPairGroup row tiles down, then the next column tile
    const int per = kPairGroup * p.nt, g = t / per, r = t - g * per;
    const int rows = min(kPairGroup, p.mt - g * kPairGroup);
    mb = g * kPairGroup + r % rows;
    nb = r / rows;
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&sf_full[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * kPairWarps);
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

  if (warp == 0) {
    if (lane == 0) {
      wait_before();  // A may come from the kernel before
      const uint32_t bar0 = mapa(smem_u32(full), 0);
      int64_t it = 0;
      Ring r(kPairStages);
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int mb, nb;
        tile_at(t, mb, nb);
        const int row_a = mb * kPM + rank * 128, row_b = nb * kPN + rank * 128, tile_a = mb * 2 + rank, tile_b = nb * 2;
        for (int kb = 0; kb < nkb; ++kb, ++it, r.next()) {
          if (!mbar_wait_cluster(&empty[r.s], r.ph ^ 1u) || *abort_flag) {
            ok = false;
            break;
          }
          // both CTAs' bytes count on the first one's barrier (a peer's copy may land before the expectation)
          if (rank == 0) mbar_expect_tx(&full[r.s], 2 * (kPairOps + kPairSf));
          const uint32_t bar = bar0 + r.s * 8;
          tma_load_2d_pair(s_a(r.s), &map_a, bar, kb * 128, row_a);
          tma_load_2d_pair(s_b(r.s), &map_b, bar, kb * 128, row_b);
          tma_load_2d_pair(s_sf(r.s), &map_sfa, bar, kb * 256, tile_a);
          tma_load_2d_pair(s_sf(r.s) + kScale, &map_sfb, bar, kb * 256, tile_b);
        }
      }
      if (!ok) {  // drain the copies in flight (each wait bounded); the peer leaves only after the cluster barrier
        *abort_flag = 1;
        for (int i = 0; rank == 0 && i < kPairStages && i < it; ++i) {
          r.back();
          mbar_wait_cluster(&full[r.s], r.ph);
        }
        atomicCAS(p.status, 0, kTimedOut + 2);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool lead = elect_one();
      const uint64_t da0 = smem_desc_k_sw128(smem_u32(s_a(0)));
      const uint32_t i0 = idesc_mxf4(kPM, kPN, 0), i2 = idesc_mxf4(kPM, kPN, 2);
      Ring r(kPairStages);
      bool ok = true;
      uint32_t n = 0;  // tiles
      for (int t = pair; t < tiles && ok; t += pairs, ++n) {
        if (!warp_agrees(mbar_wait_cluster(acc_empty, (n & 1u) ^ 1u) && !*abort_flag)) {
          ok = false;
          break;
        }
        for (int kb = 0; kb < nkb; ++kb, r.next()) {
          if (!warp_agrees(mbar_wait_fast(&sf_full[r.s], r.ph))) {  // the step's operands and scales are in place
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sf = tmem + kPN + r.s * kPairCols;  // A's 2 x 4 columns, then B's 2 x 8
          const uint64_t da = desc_add(da0, r.s * kPairOps), db = desc_add(da, kOperand);
          const uint32_t add = kb > 0;
          if (lead) {  // scales beyond the matrix are zeros, as are its codes
            #pragma unroll
            for (int j = 0; j < 4; ++j)
              mma_mxf4<2>(tmem, desc_add(da, j * 32), desc_add(db, j * 32), j & 1 ? i2 : i0, sf + (j >> 1) * 4,
                          sf + 8 + (j >> 1) * 8, j ? 1u : add);
            commit_pair(&empty[r.s]);
            if (kb == nkb - 1) commit_pair(acc_full);
          }
          __syncwarp();
        }
      }
      if (!ok && lead) {
        *abort_flag = 1;
        atomicCAS(p.status, 0, kTimedOut + 3);
      }
    }
  } else if (warp == 2 + kPairWarps) {
    if (rank == 0) {
      const bool lead = elect_one();
      const uint64_t ds0 = scale_desc(smem_u32(s_sf(0)));
      Ring c(kPairStages);
      const int64_t steps = pair < tiles ? (int64_t)((tiles - pair + pairs - 1) / pairs) * nkb : 0;
      bool ok = true;
      for (int64_t i = 0; i < steps; ++i, c.next()) {
        // a stage is filled again once its MMAs are done, which frees its scale columns in TMEM as well
        if (!warp_agrees(mbar_wait_cluster(&full[c.s], c.ph) && !*abort_flag)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sf = tmem + kPN + c.s * kPairCols;
        const uint64_t ds = desc_add(ds0, c.s * kPairSf);
        if (lead) {
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            copy_scales<2>(sf + j * 4, desc_add(ds, j * 512));
            #pragma unroll
            for (int h = 0; h < 2; ++h)
              copy_scales<2>(sf + 8 + j * 8 + h * 4, desc_add(ds, kScale * (1 + h) + j * 512));
          }
          commit_one<2>(&sf_full[c.s]);
        }
        __syncwarp();
      }
      if (!ok && lead) {
        *abort_flag = 1;
        atomicCAS(p.status, 0, kTimedOut + 5);
      }
    }
  } else {
    // a warp reads the TMEM lanes of its quadrant (warp % 4); warps 2..5 take columns 0..127, warps 6..9 the others
    const int quad = warp & 3, half = (warp - 2) >> 2;
    unsigned char* buf = out_buf + (warp - 2) * 4096;
    uint32_t n = 0;
    for (int t = pair; t < tiles; t += pairs, ++n) {
      int mb, nb;
      tile_at(t, mb, nb);
      const bool ready = !*abort_flag && mbar_wait_cluster(acc_full, n & 1u);
      if (!__all_sync(0xffffffffu, ready) || *abort_flag) {
        if (!*abort_flag) atomicCAS(p.status, 0, kTimedOut + 4);
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float x[128];
      tmem_ld128(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * 128), x);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(acc_empty), 0));
      #pragma unroll
      for (int c0 = 0; c0 < 128; c0 += kCols<T>)
        store_rows<T>(p, &map_o, buf, lane, mb * kPM + rank * 128 + quad * 32, nb * kPN + half * 128 + c0, x + c0);
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

// Codes as rows of bytes: box = 128 bytes x box_rows, 128B swizzle, zeros (codes of 0) beyond the matrix.
static int code_map(CUtensorMap* m, const void* p, int rows, int64_t ldc, int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)ldc, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ldc};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
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

static int num_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = n > 0 ? n : 148;
  }
  return cached[dev];
}

// CTAs of 256 threads: `wide` threads along a row (all of a narrow one), the others on further rows.
static void shape_of(int wide, int rows, int rows_each, dim3* grid, dim3* block) {
  const int bx = std::min(wide, 256), by = 256 / bx;
  *block = dim3(bx, by);
  *grid = dim3((rows + by * rows_each - 1) / (by * rows_each), (wide + bx - 1) / bx);
}

template <class T>
static int quantize(const void* x, int64_t ldx, int rows, int cols, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  const int nb = (cols + 31) / 32, kt = (nb + 3) / 4;
  const bool vec = aligned16(x) && (ldx * (int64_t)sizeof(T)) % 16 == 0;
  dim3 grid, block;
  shape_of(8 * kt, (rows + 127) / 128 * 128, kRows, &grid, &block);
  MPQ_CHECK_ARG(grid.y <= 65535, "mpq_mx4_quantize: %d columns are too many", cols);
  k_mx4_quantize<T><<<grid, block, 0, st>>>((const T*)x, ldx, rows, cols, vec, codes, 16 * (int64_t)nb, scales, kt);
  return launch_status("mpq_mx4_quantize");
}

template <class T>
static int dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int cols, void* out, int64_t ldo,
                      cudaStream_t st) {
  const int nb = (cols + 31) / 32, kt = (nb + 3) / 4;
  const bool vec = aligned16(out) && (ldo * (int64_t)sizeof(T)) % 16 == 0;
  dim3 grid, block;
  shape_of((int)((cols * sizeof(T) + 15) / 16), rows, 2 * kRows, &grid, &block);
  MPQ_CHECK_ARG(grid.y <= 65535, "mpq_mx4_dequantize: %d columns are too many", cols);
  k_mx4_dequantize<T><<<grid, block, 0, st>>>(codes, 16 * (int64_t)nb, scales, kt, rows, cols, vec, (T*)out, ldo);
  return launch_status("mpq_mx4_dequantize");
}

// Scales as rows of tiles: box = `rows` row tiles x two block tiles (1024 bytes), zeros beyond the matrix.
static int scale_map(CUtensorMap* m, const void* p, int row_tiles, int kt, int rows) {
  cuuint64_t dims[2] = {(cuuint64_t)kt * 128, (cuuint64_t)row_tiles};
  cuuint64_t strides[1] = {(cuuint64_t)kt * 512};
  cuuint32_t box[2] = {256, (cuuint32_t)rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(p), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("mpq_mx4_gemm: cuTensorMapEncodeTiled failed (%d) for scales, tiles %d x %d", (int)r, row_tiles, kt);
    return MPQ_ERR_ARG;
  }
  return MPQ_OK;
}

template <class T, int BN>
static int gemm_tile(const uint8_t* a_codes, const uint8_t* b_codes, int64_t ldc, GemmArgs p, int parts, bool behind,
                     cudaStream_t st) {
  p.a_rows = std::min((p.M + 7) / 8 * 8, kBM);
  CUtensorMap a, b;
  int r = code_map(&a, a_codes, p.M, ldc, p.a_rows);
  if (r) return r;
  if ((r = code_map(&b, b_codes, p.N, ldc, BN))) return r;
  CUtensorMap sa, sb;
  if ((r = scale_map(&sa, p.sfa, (p.M + 127) / 128, p.kt, 1))) return r;
  if ((r = scale_map(&sb, p.sfb, (p.N + 127) / 128, p.kt, 1))) return r;
  p.mt = (p.M + kBM - 1) / kBM;
  p.nt = (p.N + BN - 1) / BN;
  MPQ_CHECK_ARG((int64_t)p.mt * p.nt <= 0x1fffffff, "mpq_mx4_gemm: too many tiles");
  CUtensorMap o{};
  p.tile_out = result_map(&o, p.out, type_code<T>(), 1, p.M, p.N, p.ldo, false);
  p.stages = std::min<int>(kMostStages, kTileRing / (BN * 128 + p.a_rows * 128 + 2 * kScale));
  const size_t smem = 1024 + kTileRing + 4 * 4096 + 512;
  const int grid = parts > 1 ? p.mt * p.nt * parts : std::min(p.mt * p.nt, num_sms());
  return launch("mpq_mx4_gemm", k_mx4_tile<T, BN>, grid, kThreads, smem, parts, behind, st, a, b, sa, sb, o, p);
}

template <class T>
static int gemm_pair(const uint8_t* a_codes, const uint8_t* b_codes, int64_t ldc, GemmArgs p, bool behind,
                     cudaStream_t st) {
  CUtensorMap a, b, sa, sb;
  int r = code_map(&a, a_codes, p.M, ldc, 128);
  if (r) return r;
  if ((r = code_map(&b, b_codes, p.N, ldc, 128))) return r;
  if ((r = scale_map(&sa, p.sfa, (p.M + 127) / 128, p.kt, 1))) return r;
  if ((r = scale_map(&sb, p.sfb, (p.N + 127) / 128, p.kt, 2))) return r;
  p.mt = (p.M + kPM - 1) / kPM;
  p.nt = (p.N + kPN - 1) / kPN;
  MPQ_CHECK_ARG((int64_t)p.mt * p.nt <= 0x7fffffff, "mpq_mx4_gemm: too many tiles");
  CUtensorMap o{};
  p.tile_out = result_map(&o, p.out, type_code<T>(), 1, p.M, p.N, p.ldo, false);
  const size_t smem = 1024 + kPairStages * (kPairOps + kPairSf) + kPairWarps * 4096 + 256;
  return launch("mpq_mx4_gemm", k_mx4_pair<T>, 2 * std::min(p.mt * p.nt, num_sms() / 2), kPairThreads, smem, 0, behind,
                st, a, b, sa, sb, o, p);
}

// The kernel with the shortest estimate in cycles, from measured parts: a k-block takes 680 in k_mx4_tile, whatever the
// tile's width, and 700 in k_mx4_pair; a round of tiles 1000, the pair's launch 3000 more; a cluster's sum of two parts
// of K 3500, of four 6200, and more for each of its rows.  (Fitted to whole launches: the MMAs' own 512 cycles of a
// k-block are not reached, see above.  us, 512 x 4096 x 4096: 128 columns 11.9, 64 16.9, pair 13.7;
// 8 x 14336 x 4096: 128 columns in 4 parts 14.5, 2 parts 16.2, whole 24.0; 128 x 4096 x 4096: 64 columns in 2 parts 9.8,
// whole 10.2, 128 columns in 4 parts 12.6.)
template <class T>
static int gemm(const uint8_t* a_codes, const uint8_t* b_codes, const GemmArgs& p, int K, bool behind, cudaStream_t st) {
  const int64_t ldc = 16 * (int64_t)((K + 31) / 32);
  const int sms = num_sms(), nkb = (p.kt + 1) / 2;
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  int bn = 0, parts = 1;  // 0: pairs
  double least = (double)up(up(p.M, kPM) * up(p.N, kPN), sms / 2) * (nkb * 700.0 + 1000.0) + 3000.0;
  for (int w : {128, 64})
    for (int s : {1, 2, 4}) {
      const int64_t tiles = up(p.M, kBM) * up(p.N, w);
      if (s > 1 && (p.M > kBM || tiles * s > sms || nkb < s)) break;
      const double join = s == 1 ? 0.0 : (s == 2 ? 3500.0 + 12.0 * p.M : 6200.0 + 0.4 * w * p.M);
      const double t = (double)up(tiles, s > 1 ? tiles : sms) * (up(nkb, s) * 680.0 + 1000.0) + join + w;
      if (t < least) {
        least = t;
        bn = w;
        parts = s;
      }
    }
  return bn == 0     ? gemm_pair<T>(a_codes, b_codes, ldc, p, behind, st)
         : bn == 128 ? gemm_tile<T, 128>(a_codes, b_codes, ldc, p, parts, behind, st)
                     : gemm_tile<T, 64>(a_codes, b_codes, ldc, p, parts, behind, st);
}

template <class T, int TOK>
static int few_tokens(const void* x, int64_t ldx, int M, int N, int K, const uint8_t* codes, const uint8_t* scales,
                      const void* bias, void* out, int64_t ldo, cudaStream_t st) {
  const int nb = (K + 31) / 32, iters = (nb + 31) / 32, groups = (N + kFewRows - 1) / kFewRows;
  const size_t smem = (size_t)TOK * nb * 68;
  const bool vec = aligned16(x) && (ldx * (int64_t)sizeof(T)) % 16 == 0;
  const int ctas = num_sms() * (smem <= 70 * 1024 ? 3 : 1);
  // the parts of K with the fewest steps for the busiest warp; a round's sum counts as half of one
  int slices = 1, least = 1 << 30;
  for (int s = 1; s <= kFewWarps && s <= iters; s *= 2) {
    const int rounds = (groups * s + ctas * kFewWarps - 1) / (ctas * kFewWarps);
    const int steps = rounds * (2 * ((iters + s - 1) / s) + 1);
    if (steps < least) {
      least = steps;
      slices = s;
    }
  }
  const int wide = kFewWarps / slices, grid = std::min((groups + wide - 1) / wide, ctas);
  return launch("mpq_mx4_linear (few tokens)", k_mx4_few<T, TOK>, grid, kFewThreads, smem, 0, false, st, (const T*)x, ldx, M,
                N, K, vec, codes, scales, (const T*)bias, (T*)out, ldo, slices);
}

// x has to fit in shared memory; a second token's arithmetic costs more than k_mx4_tile's start from 30 M weights on
// (us, few against tile: 4096 x 4096 7.6 and 8.5, 14336 x 4096 15.1 and 11.8; one token 9.9 and 11.8, 4096 x 14336 13.2
// and 14.1).
static bool takes_few(int M, int N, int K) {
  return M <= 2 && M * ((K + 31ll) / 32) * 68 <= 200 * 1024 && (M == 1 || (int64_t)N * K <= 30000000);
}

template <class T>
static int linear(const void* x, int dtype, int64_t ldx, int M, int N, int K, const uint8_t* codes, const uint8_t* scales,
                  const void* bias, uint8_t* work, void* out, int64_t ldo, int* status, cudaStream_t st) {
  if (takes_few(M, N, K)) {
    return M == 1 ? few_tokens<T, 1>(x, ldx, M, N, K, codes, scales, bias, out, ldo, st)
                  : few_tokens<T, 2>(x, ldx, M, N, K, codes, scales, bias, out, ldo, st);
  }
  const int nb = (K + 31) / 32;
  uint8_t* x_scales = work + 16 * (int64_t)nb * M;
  const int r = quantize<T>(x, ldx, M, K, work, x_scales, st);
  if (r) return r;
  const GemmArgs args{x_scales, scales, bias, out, ldo, M, N, (nb + 3) / 4, 0, 0, 0, 0, 0, status};
  return gemm<T>(work, codes, args, K, true, st);
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
  const int st = tc::get_encoder();
  if (st) return st;
  const mx4::GemmArgs p{a_scales, b_scales, bias, out, ldo, M, N, ((K + 31) / 32 + 3) / 4, 0, 0, 0, 0, 0, status};
  return MX4_BY_TYPE(dtype, gemm, a_codes, b_codes, p, K, false, (cudaStream_t)stream);
}

// Bytes of workspace that mpq_mx4_linear needs: the quantised x, or none.
MPQ_API int64_t mpq_mx4_linear_work(int M, int K) {
  if (M <= 0 || K <= 0 || (M == 1 && mx4::takes_few(M, 1, K))) return 0;
  const int64_t nb = ((int64_t)K + 31) / 32;
  return 16 * nb * M + (M + 127ll) / 128 * ((nb + 3) / 4) * 512;
}

MPQ_API int mpq_mx4_linear(const void* x, int dtype, int64_t ldx, int M, int N, int K, const uint8_t* w_codes,
                           const uint8_t* w_scales, const void* bias, uint8_t* work, void* out, int64_t ldo, int* status,
                           void* stream) {
  MPQ_CHECK_ARG(dtype >= 0 && dtype <= 2, "mpq_mx4_linear: dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  MPQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && K <= 0x7fffff00 && M <= 0x7fffff00 && ldx >= K && ldo >= N,
                "mpq_mx4_linear: bad shape %d x %d x %d", M, N, K);
  if (M == 0 || N == 0) return MPQ_OK;
  MPQ_CHECK_ARG(x && w_codes && w_scales && out && status, "mpq_mx4_linear: null pointer");
  MPQ_CHECK_ARG(mpq_mx4_linear_work(M, K) == 0 || work, "mpq_mx4_linear: the workspace is missing");
  MPQ_CHECK_ARG(mx4::aligned16(w_codes) && mx4::aligned16(w_scales) && mx4::aligned16(work),
                "mpq_mx4_linear: codes, scales and workspace must be 16-byte aligned");
  const int st = tc::get_encoder();
  if (st) return st;
  return MX4_BY_TYPE(dtype, linear, x, dtype, ldx, M, N, K, w_codes, w_scales, bias, work, out, ldo, status,
                     (cudaStream_t)stream);
}
