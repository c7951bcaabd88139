// Microscaled 4-bit numbers: the layout that the quantisers (quant_fp4.cu) write and the products
// (gemm_fp4.cu) read.
//
// Codes: e2m1, two per byte, the even column in the low half. Scales: one byte per block of 16 columns (nvfp4,
// e4m3) or 32 (mxfp4, e8m0), in tiles of 128 rows by four blocks, 512 bytes each: byte
// (r % 32) * 16 + (r / 32) * 4 + b is row r's block b. That is the order in which one tcgen05.cp of
// 32 x 128 bits puts a tile into four columns of tensor memory, 32 rows a column, as the product
// expects them; a tile of rows' scales for one step of the product is then consecutive memory.
#pragma once

#include "ptx.cuh"

namespace ab200 {

constexpr int kFp4ScaleTile = 512;
constexpr int kFp4TileRows = 128;

enum Fp4Format : int { kNvfp4 = 0, kMxfp4 = 1 };

__host__ __device__ constexpr int fp4_block(bool mx) { return mx ? 32 : 16; }
__host__ __device__ __forceinline__ int fp4_k_tiles(int K, bool mx) {
  return (K / fp4_block(mx) + 3) / 4;
}
__device__ __forceinline__ int fp4_scale_byte(int row_in_tile) {
  return (row_in_tile & 31) * 16 + (row_in_tile >> 5) * 4;
}

// 2^e for e >= -127
__device__ __forceinline__ float fp4_pow2(int e) {
  return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 1u << 22);
}

// ------------------------------- block-scaled products ----------------------------
// kind::mxf4nvf4 / mxf4, fp32 accumulation. Both operands e2m1; sf_id: which byte of a scale column the
// instruction's first block has (a 64-wide step of mxf4 uses two of the four).
__host__ __device__ constexpr uint32_t make_idesc_fp4(uint32_t m, uint32_t n, bool mx, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((mx ? 1u : 0u) << 23) | ((m >> 4) << 24) |
         (sf_id << 29);
}

template <bool MX, bool PAIR>
__device__ __forceinline__ void umma_fp4_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define AB200_UMMA_FP4(GROUP, KIND)                                                              \
  asm volatile(                                                                                  \
      "{\n\t"                                                                                    \
      ".reg .pred p;\n\t"                                                                        \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t"     \
      "}\n" ::"r"(d_tmem),                                                                       \
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                  \
      : "memory")
  if (MX) {
    if (PAIR) AB200_UMMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
    else AB200_UMMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
  } else {
    if (PAIR) AB200_UMMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else AB200_UMMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
  }
#undef AB200_UMMA_FP4
}

// One tile of scales (32 pieces of 16 consecutive bytes) from shared memory into four columns, the same in all four
// lane quadrants. Groups of eight pieces are 128 bytes apart; no swizzle. In a pair each CTA copies its own.
__device__ __forceinline__ uint64_t make_desc_scales(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}
template <bool PAIR>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// TMEM -> registers in the layout of 8 x 8 matrix fragments: 16 lanes (the address says which half of the warp's 32)
// by 32 columns. r[4 j + 0, 1]: lane l / 4, columns 8 j + 2 (l % 4) and the next; r[4 j + 2, 3]: eight lanes further.
__device__ __forceinline__ void tmem_ld_frag_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Transposed 8 x 8 matrices of 16-bit numbers between registers and shared memory; lane l gives the address of row
// l % 8 of matrix l / 8.
__device__ __forceinline__ void stmatrix_t4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void stmatrix_t2(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_t4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

}  // namespace ab200
