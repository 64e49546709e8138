// Building blocks of the tcgen05 kernels (sm_100a): mbarriers with bounded waits, TMA tile loads, shared-memory
// operand descriptors, TMEM reads, and the tensor-map encoder.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace mpq {
namespace tc {

constexpr uint64_t kWaitNs = 2000000000ull;  // 2 s per wait

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ uint64_t globaltimer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait: false when the deadline passes first.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - t0 > kWaitNs) return false;
  }
  return true;
}

// The same wait with the clock read only once the first try has failed: %globaltimer takes hundreds of cycles, which a
// pipeline with short steps would pay at each.
__device__ __forceinline__ bool mbar_wait_fast(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait(bar, parity);
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// UMMA shared-memory descriptor, K-major operand in the 128B-swizzled canonical layout:
// rows of 128 B, 8-row swizzle atoms 1024 B apart (SBO), version 1, layout type 2 (SWIZZLE_128B).
__device__ __forceinline__ uint64_t smem_desc_k_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(16 >> 4) << 16;    // LBO (unused for swizzled K-major)
  d |= (uint64_t)(1024 >> 4) << 32;  // SBO: 8 rows x 128 B
  d |= (uint64_t)1 << 46;            // descriptor version (sm_100)
  d |= (uint64_t)2 << 61;            // SWIZZLE_128B
  return d;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Sums of four values over a warp: lane l gets the total of value l & 3.
__device__ __forceinline__ float warp_sum4(const float (&v)[4], int lane) {
  const bool odd = lane & 1, high = lane & 2;
  float a = odd ? v[1] : v[0], b = odd ? v[3] : v[2];
  a += __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1);
  b += __shfl_xor_sync(0xffffffffu, odd ? v[2] : v[3], 1);
  float c = high ? b : a;
  c += __shfl_xor_sync(0xffffffffu, high ? a : b, 2);
  #pragma unroll
  for (int o = 4; o < 32; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  return c;
}

// ---- CTA pairs (clusters of two whose tensor cores work on one tile) ----

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of the same shared-memory object in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Arrival on a barrier of either CTA by a thread that has read TMEM, after its tcgen05.wait::ld and
// tcgen05.fence::before_thread_sync, which order those reads; nothing in memory is handed over, so it is relaxed.  (A
// release at cluster scope waits for all of the thread's stores: 1550 cycles a tile in which no MMA ran, against 330.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait for arrivals from both CTAs of the pair; the clock is read only once the first try has failed.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (globaltimer() - t0 > kWaitNs) return false;
  }
  return true;
}
// Tile load of one CTA of a pair, its bytes counted on a barrier of either (`bar`: a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// All MMAs that this thread has issued for the pair -> one arrival on `bar` in each of its CTAs.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// 128 columns at once, one wait for all of them.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&x)[128]) {
  #pragma unroll
  for (int c = 0; c < 128; c += 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(x[c + 0]), "=f"(x[c + 1]), "=f"(x[c + 2]), "=f"(x[c + 3]),
          "=f"(x[c + 4]), "=f"(x[c + 5]), "=f"(x[c + 6]), "=f"(x[c + 7]),
          "=f"(x[c + 8]), "=f"(x[c + 9]), "=f"(x[c + 10]), "=f"(x[c + 11]),
          "=f"(x[c + 12]), "=f"(x[c + 13]), "=f"(x[c + 14]), "=f"(x[c + 15]),
          "=f"(x[c + 16]), "=f"(x[c + 17]), "=f"(x[c + 18]), "=f"(x[c + 19]),
          "=f"(x[c + 20]), "=f"(x[c + 21]), "=f"(x[c + 22]), "=f"(x[c + 23]),
          "=f"(x[c + 24]), "=f"(x[c + 25]), "=f"(x[c + 26]), "=f"(x[c + 27]),
          "=f"(x[c + 28]), "=f"(x[c + 29]), "=f"(x[c + 30]), "=f"(x[c + 31])
        : "r"(taddr + c));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ---- results: a warp's 32 rows x 128 bytes through shared memory ----
//
// A thread holds a row of the accumulator; stored as it is, each 16 bytes of a warp go to 32 different lines, and the
// stores, not the products, bound a kernel (measured on a 4-bit product: 418 us of stores, 231 us without).  So a warp
// lays 128 bytes of each of its rows out in a 4 KB buffer of its own, swizzled as a tile load would (no bank is hit
// twice), and one lane sends them off as a tile.

__device__ __forceinline__ void chunk_begin(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last chunk has left the buffer
  __syncwarp();
}
// 16 bytes of the lane's row, j = 0..7
__device__ __forceinline__ void chunk_unit(unsigned char* buf, int lane, int j, uint4 w) {
  *reinterpret_cast<uint4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) = w;
}
__device__ __forceinline__ void chunk_put(unsigned char* buf, int lane, const uint32_t (&w)[32]) {
  chunk_begin(lane);
  #pragma unroll
  for (int j = 0; j < 8; ++j) chunk_unit(buf, lane, j, make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]));
}
// x: first column, y: first row, z: plane.  Rows and columns beyond the map's are not written.
__device__ __forceinline__ void chunk_send(const unsigned char* buf, int lane, const CUtensorMap* map, int x, int y, int z) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(buf)), "r"(x), "r"(y), "r"(z)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// The same chunk where the result's rows do not start on 16 bytes: the lanes go along the rows, E bytes an element.
template <int E>
__device__ __forceinline__ void chunk_rows(const unsigned char* buf, int lane, void* dst, int64_t ld_bytes, int rows,
                                           int cols) {
  __syncwarp();
  for (int r = 0; r < rows && r < 32; ++r) {
    #pragma unroll
    for (int b = lane * E; b < 128; b += 32 * E) {
      if (b >= cols * E) break;
      const unsigned char* at = buf + r * 128 + ((((b >> 4) ^ (r & 7)) << 4) | (b & 15));
      unsigned char* to = reinterpret_cast<unsigned char*>(dst) + r * ld_bytes + b;
      if constexpr (E == 2) *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(at);
      else *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(at);
    }
  }
  __syncwarp();
}
// Before the buffer's CTA ends.
__device__ __forceinline__ void chunk_drain(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  __syncwarp();
}

// ---- issue ----
//
// One thread issues the MMAs, but the whole warp walks its loop: the loop's values stay uniform, and what is left to the
// elected thread is straight-line.  (In a loop of lane 0 alone, with descriptors made for each MMA, an MMA of 96 tensor
// cycles took 233 to issue.)

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// A wait's outcome, the same for all lanes (they leave a loop together).
__device__ __forceinline__ bool warp_agrees(bool ok) { return __all_sync(0xffffffffu, ok); }
// K-major / MN-major descriptors advance by their low word: (byte offset) / 16.
__device__ __forceinline__ uint64_t desc_add(uint64_t d, uint32_t bytes) { return d + (bytes >> 4); }

// Position in a ring of n stages: slot and phase parity.
struct Ring {
  int n, s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ explicit Ring(int stages) : n(stages) {}
  __device__ __forceinline__ void next() {
    if (++s == n) {
      s = 0;
      ph ^= 1u;
    }
  }
  __device__ __forceinline__ void back() {
    if (s-- == 0) {
      s = n - 1;
      ph ^= 1u;
    }
  }
};

// ---- host: tensor maps through the driver entry point (no libcuda link dependency) ----
// One variable for the library: the inline functions below are one function each, whichever file's copy the linker keeps.
inline PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

inline int get_encoder() {
  if (g_encode) return MPQ_OK;
  cudaDriverEntryPointQueryResult q;
  void* fn = nullptr;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
  if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) {
    set_last_error("cuTensorMapEncodeTiled unavailable (%s)", cudaGetErrorString(e));
    return MPQ_ERR_UNSUPPORTED;
  }
  g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  return MPQ_OK;
}

// Map of a result [planes, rows, cols] (leading dimension ld, planes contiguous) for chunk_send: type 0 f32, 1 bf16, 2
// f16.  False where a tile store cannot take it: rows that do not start on 16 bytes, or, unless `pads` (what lies
// between a row's columns and its leading dimension is the kernel's own), rows that do not end on 16 bytes: a tile
// store writes zeros up to there.
inline bool result_map(CUtensorMap* m, void* p, int type, int64_t planes, int64_t rows, int64_t cols, int64_t ld,
                       bool pads) {
  const int size = type == 0 ? 4 : 2;
  if (!pads && (cols * size) % 16) return false;
  if ((reinterpret_cast<uintptr_t>(p) & 15) || (ld * size) % 16 || (ld * size * rows) >> 40) return false;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * size), (cuuint64_t)(ld * size * rows)};
  cuuint32_t box[3] = {(cuuint32_t)(128 / size), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType t = type == 0   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : type == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return g_encode(m, t, 3, p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Launch of a kernel: `cluster` CTAs to a cluster (0: the kernel says).  `behind`: it may start while the kernel before
// it on the stream still runs (where that one allows it), and waits for its end by wait_before().
template <class... P, class... A>
static int launch(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, bool behind,
                  cudaStream_t st, A... args) {
  int r = MPQ_OK;
  if (smem > 40 * 1024 && (r = smem_opt_in((const void*)kernel, smem, what))) return r;  // 48 KB with the static part
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  if (cluster) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (behind) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_error("%s: %s", what, cudaGetErrorString(e));
    return (int)e;
  }
  return MPQ_OK;
}

// The kernel behind this one may be started once all of this grid's CTAs are here; and: wait for the kernel before.
__device__ __forceinline__ void allow_behind() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace tc
}  // namespace mpq
