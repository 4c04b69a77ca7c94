// What the attention kernels on the 5th-generation tensor cores share: the
// shape of their tiles, tensor memory and TMA primitives, the key blocks that a
// range of positions sees.
#pragma once

#include <cudaTypedefs.h>

#include "paged.cuh"

namespace nkimoe {

constexpr int kPfBlock = 128;                  // key positions per block
constexpr int kPfRows = 128;                   // MMA rows per tile
constexpr uint32_t kPfTileBytes = kPfRows * kHeadDim * 2;    // 32 KB: a Q tile
constexpr uint32_t kPfTileHalf = kPfTileBytes / 2;           // one 64-column half (128 rows x 128 bytes)
constexpr uint32_t kPfBlockBytes = kPfBlock * kHeadDim * 2;  // 32 KB: a K block or a V block
constexpr uint32_t kPfBlockHalf = kPfBlockBytes / 2;
constexpr float kPfLog2e = 1.4426950408889634f;
constexpr float kPfSlack = 8.f;                // log2 by which a block may exceed the running maximum
// tensor memory columns: S of tile t at 128 t (P over its first half), O at 256 + 128 t
constexpr uint32_t kPfTmemO = 256;

// The key blocks of queries at positions [lo, hi]: those of the first `sinks`
// positions, then from the first block of lo's window on.
struct Blocks {
  int sink, first, n;
  __device__ __forceinline__ int at(int i) const { return i < sink ? i : i - sink + first; }
};
__device__ __forceinline__ Blocks blocks_of(int lo, int hi, int window, int sinks) {
  Blocks r;
  const int start = window && lo >= window ? lo - window + 1 : 0;
  r.first = start / kPfBlock;
  r.sink = start > 0 ? min((min(sinks, start) + kPfBlock - 1) / kPfBlock, r.first) : 0;
  r.n = r.sink + hi / kPfBlock - r.first + 1;
  return r;
}

// ------------------------------------------------------------------ tensor memory, MMA with A from tensor memory
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D += A B with A (bf16 pairs, one row per lane) in tensor memory
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Descriptor of a 128-byte-swizzled MN-major operand: blocks of 64 columns
// (leading byte offset: the distance of two blocks), 8 rows of K every 1024 bytes.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The lowest n bits (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// ------------------------------------------------------------------ tensor maps
// Packed query rows [T, nq, 128], row_stride elements apart: boxes of 64 columns,
// the grp heads of a kv head, tpt rows.
inline bool tmap_of_rows(PFN_cuTensorMapEncodeTiled_v12000 encode, CUtensorMap* map, const __nv_bfloat16* q, int nq,
                         long long T, long long row_stride, int grp, int tpt) {
  const cuuint64_t dims[3] = {kHeadDim, static_cast<cuuint64_t>(nq), static_cast<cuuint64_t>(T)};
  const cuuint64_t strides[2] = {kHeadDim * 2, static_cast<cuuint64_t>(row_stride) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(grp), static_cast<cuuint32_t>(tpt)};
  const cuuint32_t one[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(q), dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A pool of pages (keys, or values): boxes of 64 columns and a page's rows, a
// block's at most, of one kv head.
inline bool tmap_of_pages(PFN_cuTensorMapEncodeTiled_v12000 encode, CUtensorMap* map, const PagedCache& c, bool values) {
  const int page = 1 << c.page_shift;
  const cuuint64_t dims[4] = {kHeadDim, static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(c.nkv),
                              static_cast<cuuint64_t>(c.num_pages)};
  const cuuint64_t strides[3] = {kHeadDim * 2, static_cast<cuuint64_t>(page) * kHeadDim * 2,
                                 static_cast<cuuint64_t>(values ? c.v_stride : c.k_stride) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page < kPfBlock ? page : kPfBlock), 1, 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, values ? c.v : c.k, dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace nkimoe
