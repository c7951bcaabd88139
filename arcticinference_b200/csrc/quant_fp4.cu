// Quantisation to microscaled 4-bit numbers, alone and behind the operations that produce the rows of a
// linear layer, and back:
//
//   quant_fp4        x bf16 [M, K]
//   rmsnorm_fp4      RMSNorm(x (+ residual, updated in place))
//   silu_mul_fp4     SiLU(gate) * up of fused blocks
//   dequant_fp4      codes and scales -> bf16
//
// nvfp4, blocks of 16:  g = 2^ceil(log2(max_k |x_k| / 2688)), one per row, at least 2^-126 (1 for a row of zeros);
//                       s = round_e4m3(max_block |x_k| / (6 g));  q = round_e2m1(x / (g s)), 0 where s = 0
// mxfp4, blocks of 32:  s = 2^(floor(log2(max_block |x_k|)) - 2), at least 2^-127;  q = round_e2m1(x / s)
// both rounding to nearest, ties to even, q saturated at 6. 2688 = 6 * 448, the largest product of the two types.
// A value that is no number: nvfp4 gives its row the factor NaN, mxfp4 its block the scale NaN; codes are zero.
//
// With g a power of two every step but the two roundings that the formulas name is exact, so that the result is a
// function of the real numbers, whatever computes it. x / (g s) against a border of e2m1 compares an integer of
// at most 8 bits with one of at most 7: a quotient that is no tie is at least 2^-8 away from it, relatively. It is
// computed as x' * (1 / s) and rounded to a multiple of 2^-13 by adding and subtracting 1.5 * 2^10: the product's
// error of 2^-22 vanishes, ties are met exactly, and all else stays on its side (a border is at least 1/4). (Which of
// its two codes a zero gets says nothing.)
//
// One CTA per row, the row in registers between the maximum and the rounding: one pass over memory. Eight columns
// per thread and step: 16-byte loads, 4-byte stores of codes; the lanes of a block share its maximum by shuffles and
// four blocks' scales leave as one word. The values are the bf16 numbers that the unfused kernel would have
// stored (same order of the norm's sum), so fused and unfused paths agree bit for bit.

#include <cuda_fp8.h>
#include <math.h>

#include "api.h"
#include "common/fp4.cuh"
#include "common/pdl.cuh"

namespace ab200 {

typedef __nv_bfloat16 bf16;

enum Fp4Source : int { kFp4Plain = 0, kFp4Norm = 1, kFp4Silu = 2 };

struct QuantFp4Args {
  const bf16* x;
  long long ldx;
  bf16* residual;       // norm: contiguous rows
  const bf16* weight;
  float eps;
  int inter, nblk;      // silu: nblk blocks of (gate | up), inter wide
  int K;                // columns of the result
  uint8_t* q;
  long long ldq;        // bytes
  uint8_t* scale;       // tiles [row tile][k_tiles][512]
  float* row_scale;     // nvfp4
  int k_tiles;
  const int4* tiles;    // optional: rows lie in these tiles (group, first row, rows), the scales by tile
  const int* num_tiles;
};

__device__ __forceinline__ void fq_unpack8(const uint4& q, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 fq_pack8(const float (&f)[8]) {
  uint4 q;
  q.x = pack_bf16x2(f[0], f[1]);
  q.y = pack_bf16x2(f[2], f[3]);
  q.z = pack_bf16x2(f[4], f[5]);
  q.w = pack_bf16x2(f[6], f[7]);
  return q;
}
// The largest magnitude of eight bf16 numbers, as bits: infinities and NaN are above all numbers.
__device__ __forceinline__ uint32_t fq_top8(const uint4& q) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t t = __vmaxu2(__vmaxu2(q.x & m, q.y & m), __vmaxu2(q.z & m, q.w & m));
  return max(t & 0xffffu, t >> 16);
}
__device__ __forceinline__ float fq_block_sum(float v, float* red) {
  v = warp_sum(v);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nwarps = (blockDim.x + 31) >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nwarps ? red[lane] : 0.f);
}
__device__ __forceinline__ uint32_t fq_block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nwarps = (blockDim.x + 31) >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < nwarps ? red[lane] : 0u);
}
// Eight numbers times `up` (a power of two) times `inv` -> eight codes
__device__ __forceinline__ uint32_t fq_codes8(const uint4& raw, float up, float inv) {
  float v[8];
  fq_unpack8(raw, v);
  const float2 u = make_float2(up, up), r = make_float2(inv, inv);
  const float2 big = make_float2(1536.f, 1536.f), neg = make_float2(-1536.f, -1536.f);   // 1.5 * 2^10
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = add_x2(fma_x2(mul_x2(make_float2(v[2 * i], v[2 * i + 1]), u), r, big), neg);
    v[2 * i] = t.x;
    v[2 * i + 1] = t.y;
  }
  uint32_t w;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}\n"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// The place of a row's scales: the row itself, or by the tile that holds it (-1: none does).
__device__ __forceinline__ int fq_slot(const QuantFp4Args& p, int row, int* found) {
  if (p.tiles == nullptr) return row;
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  const int n = *p.num_tiles;
  for (int t = threadIdx.x; t < n; t += blockDim.x) {
    const int4 w = p.tiles[t];
    if (row >= w.y && row < w.y + w.z) *found = t * kFp4TileRows + row - w.y;
  }
  __syncthreads();
  return *found;
}

template <int SRC, bool MX, int VPT>
__global__ void __launch_bounds__(512) quant_fp4_kernel(const QuantFp4Args p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[32];
  __shared__ int found;
  constexpr int kBlockVecs = MX ? 4 : 2;          // lanes of a block
  constexpr int kTileVecs = 4 * kBlockVecs;       // lanes of a word of scales
  const int row = blockIdx.x;
  const int nvec = p.K / 8, all = p.k_tiles * kTileVecs;
  uint4 raw[VPT];
  if (SRC == kFp4Silu) {
    const int per = p.inter / 8;
    const bf16* xr = p.x + row * p.ldx;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x + j * blockDim.x;
      raw[j] = make_uint4(0, 0, 0, 0);
      if (i < nvec) {
        const int b = p.nblk == 1 ? 0 : i / per;
        const uint4* blk = reinterpret_cast<const uint4*>(xr + (long long)b * 2 * p.inter);
        float g[8], u[8];
        fq_unpack8(blk[i - b * per], g);
        fq_unpack8(blk[per + i - b * per], u);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = __fdividef(g[k], 1.f + __expf(-g[k])) * u[k];
        raw[j] = fq_pack8(g);
      }
    }
  } else {
    const uint4* xr = reinterpret_cast<const uint4*>(p.x + row * p.ldx);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x + j * blockDim.x;
      raw[j] = i < nvec ? xr[i] : make_uint4(0, 0, 0, 0);
    }
  }
  if (SRC == kFp4Norm) {
    uint4* rr = p.residual ? reinterpret_cast<uint4*>(p.residual + (long long)row * p.K) : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x + j * blockDim.x;
      if (i < nvec) {
        float v[8];
        fq_unpack8(raw[j], v);
        if (rr) {
          float r[8];
          fq_unpack8(rr[i], r);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += r[k];
          raw[j] = fq_pack8(v);
          rr[i] = raw[j];
          fq_unpack8(raw[j], v);   // normalise the value that was stored
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += v[k] * v[k];
      }
    }
    ss = fq_block_sum(ss, reinterpret_cast<float*>(red));
    const float inv_rms = rsqrtf(ss / (float)p.K + p.eps);
    const uint4* wr = reinterpret_cast<const uint4*>(p.weight);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x + j * blockDim.x;
      if (i < nvec) {
        float v[8], w[8];
        fq_unpack8(raw[j], v);
        fq_unpack8(wr[i], w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] * inv_rms * w[k];
        raw[j] = fq_pack8(v);
      }
    }
  }
  const int slot = fq_slot(p, row, &found);
  uint32_t top[VPT], most = 0;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    uint32_t t = fq_top8(raw[j]);
    t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
    if (MX) t = max(t, __shfl_xor_sync(0xffffffffu, t, 2));
    top[j] = t;
    most = max(most, t);
  }
  float up = 1.f;
  if (!MX) {
    most = fq_block_max(most, red);
    // 2688 = 1.3125 * 2^11
    const uint32_t bits = most << 16;
    int e = (int)(bits >> 23) - 127 - 11 + ((bits & 0x7fffffu) > 0x280000u ? 1 : 0);
    e = most == 0 ? 0 : max(e, -126);
    const bool fine = most < 0x7f80u;
    up = fine ? fp4_pow2(-e) : 0.f;
    if (threadIdx.x == 0 && slot >= 0) p.row_scale[row] = fine ? fp4_pow2(e) : __uint_as_float(0x7fffffffu);
  }
  if (slot < 0) return;
  uint32_t* qr = reinterpret_cast<uint32_t*>(p.q + row * p.ldq);
  uint8_t* sr = p.scale + (long long)(slot / kFp4TileRows) * p.k_tiles * kFp4ScaleTile +
                fp4_scale_byte(slot % kFp4TileRows);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    uint32_t byte;
    float scaled = up, inv;
    uint4 v = raw[j];
    if (MX) {
      const int e = max((int)(top[j] >> 7) - 2, 0);      // the exponent's field
      byte = (uint32_t)e;
      inv = 1.f;
      scaled = fp4_pow2(127 - e);
      if (top[j] >= 0x7f80u) {
        byte = 0xffu;
        v = make_uint4(0, 0, 0, 0);
      }
    } else {
      const float t = __fdiv_rn(__uint_as_float(top[j] << 16) * up, 6.f);
      byte = most < 0x7f80u ? (uint32_t)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3) : 0u;
      inv = byte ? __frcp_rn(e4m3_value(byte)) : 0.f;
      if (byte == 0u) v = make_uint4(0, 0, 0, 0);
    }
    if (i < nvec) qr[i] = fq_codes8(v, scaled, inv);
    // the scales of four blocks in one word; blocks behind the row's end have the scale zero
    if (i >= nvec) byte = 0u;
    const uint32_t b1 = __shfl_down_sync(0xffffffffu, byte, kBlockVecs);
    const uint32_t two = byte | (b1 << 8);
    const uint32_t four = two | (__shfl_down_sync(0xffffffffu, two, 2 * kBlockVecs) << 16);
    if (i < all && (i % kTileVecs) == 0)
      *reinterpret_cast<uint32_t*>(sr + (long long)(i / kTileVecs) * kFp4ScaleTile) = four;
  }
}

// One thread per eight numbers. Rows of a weight of several groups: each group's scale tiles begin anew.
template <bool MX>
__global__ void __launch_bounds__(256)
dequant_fp4_kernel(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ scale,
                   const float* __restrict__ row_scale, bf16* __restrict__ out, long long ldo, long long rows,
                   int K, int k_tiles, int group_rows, const int4* __restrict__ tiles,
                   const int* __restrict__ num_tiles) {
  pdl_wait();
  pdl_trigger();
  constexpr int kBlockVecs = MX ? 4 : 2;
  const int nvec = K / 8;
  auto row_of = [&](long long row, long long slot) {
    const float g = row_scale != nullptr ? row_scale[row] : 1.f;
    const uint8_t* sr = scale + slot / kFp4TileRows * k_tiles * kFp4ScaleTile +
                        fp4_scale_byte((int)(slot % kFp4TileRows));
    const uint32_t* qr = reinterpret_cast<const uint32_t*>(q + row * ldq);
    uint4* o = reinterpret_cast<uint4*>(out + row * ldo);
    for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
      const int b = i / kBlockVecs;
      const uint32_t byte = sr[(long long)(b / 4) * kFp4ScaleTile + b % 4], w = qr[i];
      float s;
      if (MX) s = byte == 0xffu ? __uint_as_float(0x7fffffffu) : fp4_pow2((int)byte - 127);
      else s = e4m3_value(byte);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t c = w >> (4 * k);
        // value of the code: (1 + m / 2) 2^(e - 1), m / 2 where e = 0
        const int e = (int)(c >> 1) & 3;
        const float mag = e == 0 ? 0.5f * (float)(c & 1u) : (float)(2u + (c & 1u)) * 0.25f * (float)(1 << e);
        v[k] = ((c & 8u) ? -mag : mag) * s * g;
      }
      o[i] = fq_pack8(v);
    }
  };
  if (tiles != nullptr) {
    const int n = *num_tiles;
    for (int t = blockIdx.x; t < n * kFp4TileRows; t += gridDim.x) {
      const int4 w = tiles[t / kFp4TileRows];
      const int r = t % kFp4TileRows;
      if (r < w.z) row_of(w.y + r, t);
    }
    return;
  }
  const int padded = (group_rows + kFp4TileRows - 1) / kFp4TileRows * kFp4TileRows;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x)
    row_of(row, row / group_rows * padded + row % group_rows);
}

template <int SRC, bool MX>
static int launch_quant_fp4(const QuantFp4Args& a, long long M, cudaStream_t stream) {
  const int vecs = a.k_tiles * (MX ? 16 : 8);
  // Two steps per thread keep enough loads in flight and enough threads per row; wider rows take more. (The norm's
  // sum has the order of the unfused kernel's: 256 threads.)
  int vpt = 1, threads = 256;
  if (SRC == kFp4Norm) {
    while (vpt * 256 < vecs) vpt *= 2;
  } else {
    while (vpt < 2 && vecs > 32 * vpt) vpt *= 2;
    while (vecs > 512 * vpt) vpt *= 2;
    threads = ((vecs + vpt - 1) / vpt + 31) / 32 * 32;
  }
  if (vpt > 8 || M > 0x7fffffff) return -6;
  cudaError_t e;
  const dim3 grid((unsigned)M), block((unsigned)threads);
  switch (vpt) {
    case 1: e = launch_pdl(quant_fp4_kernel<SRC, MX, 1>, grid, block, 0, stream, a); break;
    case 2: e = launch_pdl(quant_fp4_kernel<SRC, MX, 2>, grid, block, 0, stream, a); break;
    case 4: e = launch_pdl(quant_fp4_kernel<SRC, MX, 4>, grid, block, 0, stream, a); break;
    default: e = launch_pdl(quant_fp4_kernel<SRC, MX, 8>, grid, block, 0, stream, a); break;
  }
  return e == cudaSuccess ? 0 : -5;
}

}  // namespace ab200

using namespace ab200;

static bool fp4_misaligned(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0;
}

extern "C" {

// x bf16 [M, K], rows ldx apart -> codes [M, K / 2] (rows ldq bytes apart), scale tiles [row tiles][k_tiles][512]
// with k_tiles = ceil(K / (4 * block)), and for nvfp4 (fmt 0; mxfp4: 1) row_scale fp32 [M]. K: a multiple of 32, at
// most 32768. With `tiles` (int32 x 4: group, first row, rows; *num_tiles of them) a row's scales lie in
// the row tile of its tile, and rows that no tile holds are left out.
int ab200_quant_fp4(const void* x, long long ldx, void* q, long long ldq, void* scale, void* row_scale, long long M,
                    int K, int fmt, const void* tiles, const void* num_tiles, cudaStream_t stream) {
  if (M <= 0 || K <= 0) return 0;
  if ((K % 32) || K > 32768 || (ldx % 8) || (ldq % 16) || fp4_misaligned(x, q) || fmt < 0 || fmt > 1 ||
      (fmt == kNvfp4 && row_scale == nullptr) || (tiles != nullptr && num_tiles == nullptr))
    return -2;
  QuantFp4Args a = {};
  a.x = reinterpret_cast<const bf16*>(x);
  a.ldx = ldx;
  a.K = K;
  a.q = reinterpret_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scale = reinterpret_cast<uint8_t*>(scale);
  a.row_scale = reinterpret_cast<float*>(row_scale);
  a.k_tiles = fp4_k_tiles(K, fmt == kMxfp4);
  a.tiles = reinterpret_cast<const int4*>(tiles);
  a.num_tiles = reinterpret_cast<const int*>(num_tiles);
  return fmt == kMxfp4 ? launch_quant_fp4<kFp4Plain, true>(a, M, stream)
                       : launch_quant_fp4<kFp4Plain, false>(a, M, stream);
}

// The same of RMSNorm(x (+ residual)) * weight; residual (contiguous rows) is updated in place. K at most 16384.
int ab200_rmsnorm_fp4(const void* x, long long ldx, void* residual, const void* weight, void* q, long long ldq,
                      void* scale, void* row_scale, long long M, int K, float eps, int fmt, cudaStream_t stream) {
  if (M <= 0 || K <= 0) return 0;
  if ((K % 32) || K > 16384 || (ldx % 8) || (ldq % 16) || fp4_misaligned(x, q) ||
      fp4_misaligned(residual, weight) || fmt < 0 || fmt > 1 || (fmt == kNvfp4 && row_scale == nullptr))
    return -2;
  QuantFp4Args a = {};
  a.x = reinterpret_cast<const bf16*>(x);
  a.ldx = ldx;
  a.residual = reinterpret_cast<bf16*>(residual);
  a.weight = reinterpret_cast<const bf16*>(weight);
  a.eps = eps;
  a.K = K;
  a.q = reinterpret_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scale = reinterpret_cast<uint8_t*>(scale);
  a.row_scale = reinterpret_cast<float*>(row_scale);
  a.k_tiles = fp4_k_tiles(K, fmt == kMxfp4);
  return fmt == kMxfp4 ? launch_quant_fp4<kFp4Norm, true>(a, M, stream)
                       : launch_quant_fp4<kFp4Norm, false>(a, M, stream);
}

// The same of SiLU(gate) * up: x has rows of nblk blocks of (gate | up), each `inter` wide; K = nblk * inter.
int ab200_silu_mul_fp4(const void* x, long long ldx, void* q, long long ldq, void* scale, void* row_scale,
                       long long M, int inter, int nblk, int fmt, cudaStream_t stream) {
  if (M <= 0 || inter <= 0) return 0;
  if (nblk < 1 || inter > 32768 / nblk) return -2;
  const int K = nblk * inter;
  if ((K % 32) || (inter % 8) || (ldx % 8) || (ldq % 16) || fp4_misaligned(x, q) || fmt < 0 || fmt > 1 ||
      (fmt == kNvfp4 && row_scale == nullptr))
    return -2;
  QuantFp4Args a = {};
  a.x = reinterpret_cast<const bf16*>(x);
  a.ldx = ldx;
  a.inter = inter;
  a.nblk = nblk;
  a.K = K;
  a.q = reinterpret_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scale = reinterpret_cast<uint8_t*>(scale);
  a.row_scale = reinterpret_cast<float*>(row_scale);
  a.k_tiles = fp4_k_tiles(K, fmt == kMxfp4);
  return fmt == kMxfp4 ? launch_quant_fp4<kFp4Silu, true>(a, M, stream)
                       : launch_quant_fp4<kFp4Silu, false>(a, M, stream);
}

// Back: out bf16 [rows, K] (rows ldo apart). `group_rows`: rows per group of a weight of several matrices (the
// whole of it otherwise); `tiles`: as in ab200_quant_fp4. row_scale null: no factors.
int ab200_dequant_fp4(const void* q, long long ldq, const void* scale, const void* row_scale, void* out,
                      long long ldo, long long rows, int K, int group_rows, int fmt, const void* tiles,
                      const void* num_tiles, cudaStream_t stream) {
  if (rows <= 0 || K <= 0) return 0;
  if ((K % 32) || (ldq % 4) || (ldo % 8) || fp4_misaligned(out, nullptr) || group_rows <= 0 || fmt < 0 || fmt > 1 ||
      (reinterpret_cast<uintptr_t>(q) & 3) || (tiles != nullptr && num_tiles == nullptr))
    return -2;
  const int nvec = K / 8;
  const unsigned threads = nvec >= 256 ? 256u : (unsigned)((nvec + 31) / 32 * 32);
  const long long want = rows < 148ll * 16 ? rows : 148ll * 16;
  const dim3 grid((unsigned)(tiles != nullptr ? 148 * 8 : want));
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, grid, dim3(threads), 0, stream, reinterpret_cast<const uint8_t*>(q), ldq,
                      reinterpret_cast<const uint8_t*>(scale), reinterpret_cast<const float*>(row_scale),
                      reinterpret_cast<bf16*>(out), ldo, rows, K, fp4_k_tiles(K, fmt == kMxfp4), group_rows,
                      reinterpret_cast<const int4*>(tiles), reinterpret_cast<const int*>(num_tiles));
  };
  const cudaError_t e = fmt == kMxfp4 ? go(dequant_fp4_kernel<true>) : go(dequant_fp4_kernel<false>);
  return e == cudaSuccess ? 0 : -5;
}

}  // extern "C"
