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
// error of 2^-20 vanishes, ties are met exactly, and all else stays on its side (a border is at least 1/4). In the same
// way max / 6 against a border of e4m3 (five bits) is rounded to fp16 first, which meets the ties and keeps the rest on
// its side. Divisions rounded to the last bit gave the same results in twice the time. (Which of
// its two codes a zero gets says nothing.)
//
// One CTA (or warp) per row, the row in registers between the maximum and the rounding: one pass over memory. 16-byte
// loads, 4 or 8-byte stores of codes; the lanes of a block share its maximum by shuffles and four blocks' scales leave as
// one word. The values are the bf16 numbers that the unfused kernel would have
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
  int max_tiles;        // what the list and the scales have room for, whatever *num_tiles says
  int M;
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
// Eight numbers times r -> eight codes. EXACT: the products are (r is a power of two).
template <bool EXACT>
__device__ __forceinline__ uint32_t fq_codes8(const uint4& raw, float r) {
  float v[8];
  fq_unpack8(raw, v);
  const float2 rr = make_float2(r, r), big = make_float2(1536.f, 1536.f), neg = make_float2(-1536.f, -1536.f);   // 1.5 * 2^10
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = make_float2(v[2 * i], v[2 * i + 1]);
    const float2 t = EXACT ? mul_x2(x, rr) : add_x2(fma_x2(x, rr, big), neg);
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
// Eight codes' values
__device__ __forceinline__ void fq_values8(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = t.x;
    v[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// The place of a row's scales: the row itself, or by the tile that holds it (-1: none does). A warp looks: among 32
// tiles spread over the list, then among those from the last one that does not begin behind the row. (A tile
// without rows fills its expert's list up to an even number and begins where the one before it ends.)
__device__ __forceinline__ int fq_slot(const QuantFp4Args& p, int row, int lane) {
  if (p.tiles == nullptr) return row;
  const int n = min(*p.num_tiles, p.max_tiles), step = (n + 31) / 32;
  bool before = false;
  if (lane * step < n) {
    const int4 t = p.tiles[lane * step];
    int first = t.y;
    if (t.z <= 0 && lane > 0) {
      const int4 u = p.tiles[lane * step - 1];
      first = u.y + u.z;
    }
    before = first <= row;
  }
  const uint32_t some = __ballot_sync(0xffffffffu, before);
  if (some == 0u) return -1;
  const int from = (31 - __clz((int)some)) * step;
  for (int i = 0; i < step; i += 32) {
    const int at = from + i + lane;
    int in = -1;
    if (i + lane < step && at < n) {
      const int4 t = p.tiles[at];
      if (row >= t.y && row < t.y + min(t.z, kFp4TileRows)) in = row - t.y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, in >= 0);
    if (hit != 0u) {
      const int who = __ffs((int)hit) - 1;
      return (from + i + who) * kFp4TileRows + __shfl_sync(0xffffffffu, in, who);
    }
  }
  return -1;
}

// WARP: a warp per row and no barrier, for rows that 32 threads hold; otherwise a block per row. A thread takes pieces
// of 16 columns, whose one scale (nvfp4) it then computes alone: 8192 x 4096 took 16.1 us with pieces of 8, and the
// instructions bound it; with pieces of 16 it takes 14.5 (5.9 TB/s; mxfp4 13.3, 6.4). (The norm keeps
// pieces of 8, in which the unfused kernel adds; both lanes of an nvfp4 block then compute its scale. That order binds the
// sum only, and pieces of 16 behind it have not been tried: 4096 x 4096 17.8 us, 2.4 TB/s, an instruction issued in 78 % of
// the cycles. SiLU, 4096 x 14336: 58 us, 4.6 TB/s, 67 %.)
template <int SRC, bool MX, int VPT, bool WARP>
__global__ void __launch_bounds__(512) quant_fp4_kernel(const QuantFp4Args p) {
  static_assert(!(WARP && SRC == kFp4Norm), "a norm's sum is the block's");
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[32];
  __shared__ int block_slot;
  constexpr int kPer = SRC == kFp4Norm || VPT == 1 ? 1 : 2;        // eight columns each in a piece
  constexpr int kPieces = VPT / kPer;
  constexpr int kBlockLanes = (MX ? 4 : 2) / kPer;                 // lanes of a block
  constexpr int kTileLanes = 4 * kBlockLanes;                      // lanes of a word of scales
  const int lane = threadIdx.x & 31;
  const int tid = WARP ? lane : (int)threadIdx.x, threads = WARP ? 32 : (int)blockDim.x;
  const int row = WARP ? (int)(blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) : (int)blockIdx.x;
  if (WARP && row >= p.M) return;
  const int nvec = p.K / 8, pieces = nvec / kPer, all = p.k_tiles * kTileLanes;
  auto vec_of = [&](int j) { return (tid + j / kPer * threads) * kPer + j % kPer; };
  // everything that is read is requested first
  uint4 raw[VPT], other[SRC == kFp4Plain ? 1 : VPT], wraw[SRC == kFp4Norm ? VPT : 1];
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + (long long)row * p.ldx);
  uint4* rr = SRC == kFp4Norm && p.residual != nullptr ? reinterpret_cast<uint4*>(p.residual + (long long)row * p.K)
                                                       : nullptr;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int i = vec_of(j);
    raw[j] = make_uint4(0, 0, 0, 0);
    if (SRC != kFp4Plain) other[j] = make_uint4(0, 0, 0, 0);
    if (SRC == kFp4Norm) wraw[j] = make_uint4(0, 0, 0, 0);
    if (i < nvec) {
      if (SRC == kFp4Silu) {
        const int per = p.inter / 8, b = p.nblk == 1 ? 0 : i / per;
        raw[j] = xr[i + b * per];
        other[j] = xr[i + (b + 1) * per];
      } else {
        raw[j] = xr[i];
        if (SRC == kFp4Norm && rr != nullptr) other[j] = rr[i];
        if (SRC == kFp4Norm) wraw[j] = reinterpret_cast<const uint4*>(p.weight)[i];
      }
    }
  }
  int slot = row;
  if (SRC == kFp4Plain) {
    if (WARP) {
      slot = fq_slot(p, row, lane);
    } else if (p.tiles != nullptr) {
      if (threadIdx.x < 32) {
        slot = fq_slot(p, row, lane);
        if (lane == 0) block_slot = slot;
      }
      __syncthreads();
      slot = block_slot;
    }
  }
  if (SRC == kFp4Silu) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      float g[8], u[8];
      fq_unpack8(raw[j], g);
      fq_unpack8(other[j], u);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = __fdividef(g[k], 1.f + __expf(-g[k])) * u[k];
      raw[j] = fq_pack8(g);
    }
  }
  if (SRC == kFp4Norm) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = vec_of(j);
      float v[8];
      fq_unpack8(raw[j], v);
      if (rr != nullptr) {
        float a[8];
        fq_unpack8(other[j], a);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += a[k];
        raw[j] = fq_pack8(v);
        if (i < nvec) rr[i] = raw[j];
        fq_unpack8(raw[j], v);   // normalise the value that was stored
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) ss += v[k] * v[k];
    }
    ss = fq_block_sum(ss, reinterpret_cast<float*>(red));
    const float inv_rms = rsqrtf(ss / (float)p.K + p.eps);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      float v[8], f[8];
      fq_unpack8(raw[j], v);
      fq_unpack8(wraw[j], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = v[k] * inv_rms * f[k];
      raw[j] = fq_pack8(v);
    }
  }
  uint32_t top[kPieces], most = 0;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    uint32_t t = fq_top8(raw[kPer * j]);
    if (kPer == 2) t = max(t, fq_top8(raw[kPer * j + kPer - 1]));
    if (kBlockLanes >= 2) t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
    if (kBlockLanes >= 4) t = max(t, __shfl_xor_sync(0xffffffffu, t, 2));
    top[j] = t;
    most = max(most, t);
  }
  float up = 1.f;
  if (!MX) {
    most = WARP ? __reduce_max_sync(0xffffffffu, most) : fq_block_max(most, red);
    // 2688 = 1.3125 * 2^11
    const uint32_t bits = most << 16;
    int e = (int)(bits >> 23) - 127 - 11 + ((bits & 0x7fffffu) > 0x280000u ? 1 : 0);
    e = most == 0 ? 0 : max(e, -126);
    const bool fine = most < 0x7f80u;
    up = fine ? fp4_pow2(-e) : 0.f;
    if (tid == 0 && slot >= 0) p.row_scale[row] = fine ? fp4_pow2(e) : __uint_as_float(0x7fffffffu);
    if (up > 0x1p+110f) {
      // 1 / (g s) would pass the range: the row's numbers, all below 2^-98, are enlarged first (exactly)
      up *= 0x1p-60f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float v[8];
        fq_unpack8(raw[j], v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= 0x1p+60f;
        raw[j] = fq_pack8(v);
      }
#pragma unroll
      for (int j = 0; j < kPieces; ++j) top[j] = __float_as_uint(__uint_as_float(top[j] << 16) * 0x1p+60f) >> 16;
    }
  }
  if (slot < 0) return;
  uint32_t* qr = reinterpret_cast<uint32_t*>(p.q + (long long)row * p.ldq);
  uint8_t* sr = p.scale + (long long)(slot / kFp4TileRows) * p.k_tiles * kFp4ScaleTile +
                fp4_scale_byte(slot % kFp4TileRows);
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int i = tid + j * threads;
    uint32_t byte, code[kPer];
    float r;
    bool some;
    if (MX) {
      const int e = max((int)(top[j] >> 7) - 2, 0);      // the exponent's field
      some = top[j] < 0x7f80u;
      byte = some ? (uint32_t)e : 0xffu;
      r = fp4_pow2(127 - e);
    } else {
      const __half t = __float2half_rn(__uint_as_float(top[j] << 16) * up * (1.f / 6.f));
      byte = most < 0x7f80u ? (uint32_t)__nv_cvt_halfraw_to_fp8(t, __NV_SATFINITE, __NV_E4M3) : 0u;
      some = byte != 0u;
      r = up * rcp_approx(e4m3_value(byte));
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const uint32_t c = fq_codes8<MX>(raw[kPer * j + e], r);
      code[e] = some ? c : 0u;
    }
    if (i < pieces) {
      if (kPer == 2) *reinterpret_cast<uint2*>(qr + 2 * i) = make_uint2(code[0], code[kPer - 1]);
      else qr[i] = code[0];
    }
    // the scales of four blocks in one word; blocks behind the row's end have the scale zero
    if (i >= pieces) byte = 0u;
    const uint32_t b1 = __shfl_down_sync(0xffffffffu, byte, kBlockLanes);
    const uint32_t two = byte | (b1 << 8);
    const uint32_t four = two | (__shfl_down_sync(0xffffffffu, two, 2 * kBlockLanes) << 16);
    if (i < all && (i % kTileLanes) == 0)
      *reinterpret_cast<uint32_t*>(sr + (long long)(i / kTileLanes) * kFp4ScaleTile) = four;
  }
}

// Eight numbers per thread and step, four steps on their way together; threadIdx.y: rows of a block. Rows of a weight of
// several groups: each group's scale tiles begin anew. (16 numbers a thread would halve the work on scales, but a store
// instruction then leaves half of every sector to the next one: 20.6 instead of 15.0 us for 8192 x 4096.)
template <bool MX>
__global__ void __launch_bounds__(256)
dequant_fp4_kernel(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ scale,
                   const float* __restrict__ row_scale, bf16* __restrict__ out, long long ldo, long long rows,
                   int K, int k_tiles, int group_rows, const int4* __restrict__ tiles,
                   const int* __restrict__ num_tiles, int max_tiles) {
  pdl_wait();
  pdl_trigger();
  constexpr int kBlockVecs = MX ? 4 : 2;
  const int nvec = K / 8;
  const int padded = (group_rows + kFp4TileRows - 1) / kFp4TileRows * kFp4TileRows;
  const long long items = tiles != nullptr ? (long long)min(*num_tiles, max_tiles) * kFp4TileRows : rows;
  // (blockIdx.y: a part of the row)
  for (long long item = (long long)blockIdx.x * blockDim.y + threadIdx.y; item < items;
       item += (long long)gridDim.x * blockDim.y) {
    long long row = item, slot;
    if (tiles != nullptr) {
      const int4 t = tiles[item / kFp4TileRows];
      const int in = (int)(item % kFp4TileRows);
      row = t.y + in;
      if (in >= t.z || row < 0 || row >= rows) continue;
      slot = item;
    } else {
      slot = row / group_rows * padded + row % group_rows;
    }
    const float g = row_scale != nullptr ? row_scale[row] : 1.f;
    const uint8_t* sr = scale + slot / kFp4TileRows * k_tiles * kFp4ScaleTile +
                        fp4_scale_byte((int)(slot % kFp4TileRows));
    const uint32_t* qr = reinterpret_cast<const uint32_t*>(q + row * ldq);
    uint4* o = reinterpret_cast<uint4*>(out + row * ldo);
    for (int i0 = threadIdx.x + 4 * blockDim.x * blockIdx.y; i0 < nvec; i0 += 4 * blockDim.x * gridDim.y) {
      uint32_t byte[4], w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * blockDim.x, b = i / kBlockVecs;
        byte[j] = i < nvec ? sr[(long long)(b / 4) * kFp4ScaleTile + b % 4] : 0u;
        w[j] = i < nvec ? qr[i] : 0u;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * blockDim.x;
        float s;
        if (MX) s = byte[j] == 0xffu ? __uint_as_float(0x7fffffffu) : fp4_pow2((int)byte[j] - 127);
        else s = e4m3_value(byte[j]);
        const float2 f = make_float2(s * g, s * g);
        float v[8];
        fq_values8(w[j], v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 t = mul_x2(make_float2(v[2 * k], v[2 * k + 1]), f);
          v[2 * k] = t.x;
          v[2 * k + 1] = t.y;
        }
        if (i < nvec) o[i] = fq_pack8(v);
      }
    }
  }
}

template <int SRC, bool MX>
static int launch_quant_fp4(const QuantFp4Args& a, long long M, cudaStream_t stream) {
  const int vecs = a.k_tiles * (MX ? 16 : 8);
  if (M > 0x7fffffff) return -6;
  QuantFp4Args args = a;
  args.M = (int)M;
  auto go = [&](auto kernel, long long blocks, int threads) {
    return launch_pdl(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), 0, stream, args) == cudaSuccess ? 0 : -5;
  };
  if constexpr (SRC == kFp4Norm) {   // 256 threads: the norm's sum has the order of the unfused kernel's
    if (vecs <= 256) return go(quant_fp4_kernel<SRC, MX, 1, false>, M, 256);
    if (vecs <= 512) return go(quant_fp4_kernel<SRC, MX, 2, false>, M, 256);
    if (vecs <= 1024) return go(quant_fp4_kernel<SRC, MX, 4, false>, M, 256);
    return vecs <= 2048 ? go(quant_fp4_kernel<SRC, MX, 8, false>, M, 256) : -6;
  } else {
    // Few rows want many threads each, many rows much in flight per thread (4096 columns, nvfp4, us for 2, 4 and 8
    // steps: 128 rows 1.75, 1.89, 2.35; 8192 rows 20.2, 17.1, 16.0). The activation holds both factors: 4096 rows
    // of 14336 62.3 with 4 steps and 110 with 8.
    const bool many = M >= 148 * 8;
    if (vecs <= 64) return go(quant_fp4_kernel<SRC, MX, 2, true>, (M + 3) / 4, 128);
    if (vecs <= 128 && many) return go(quant_fp4_kernel<SRC, MX, 4, true>, (M + 3) / 4, 128);
    if constexpr (SRC == kFp4Plain)
      if (vecs <= 256 && many) return go(quant_fp4_kernel<SRC, MX, 8, true>, (M + 3) / 4, 128);
    int vpt = !many ? 2 : SRC == kFp4Silu ? 4 : 8;
    while (vecs > 512 * vpt) vpt *= 2;
    const int threads = ((vecs + vpt - 1) / vpt + 31) / 32 * 32;
    if (vpt == 2) return go(quant_fp4_kernel<SRC, MX, 2, false>, M, threads);
    if (vpt == 4) return go(quant_fp4_kernel<SRC, MX, 4, false>, M, threads);
    return vpt == 8 ? go(quant_fp4_kernel<SRC, MX, 8, false>, M, threads) : -6;
  }
}

}  // namespace ab200

using namespace ab200;

static bool fp4_misaligned(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0;
}

extern "C" {

// x bf16 [M, K], rows ldx apart -> codes [M, K / 2] (rows ldq bytes apart), scale tiles [row tiles][k_tiles][512]
// with k_tiles = ceil(K / (4 * block)), and for nvfp4 (fmt 0; mxfp4: 1) row_scale fp32 [M]. K: a multiple of 32, at
// most 32768. With `tiles` (int32 x 4: group, first row, rows; *num_tiles of them, at most max_tiles, in
// the order of their rows) a row's scales lie in
// the row tile of its tile, and rows that no tile holds are left out.
int ab200_quant_fp4(const void* x, long long ldx, void* q, long long ldq, void* scale, void* row_scale, long long M,
                    int K, int fmt, const void* tiles, const void* num_tiles, int max_tiles, cudaStream_t stream) {
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
  a.max_tiles = max_tiles;
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
                      const void* num_tiles, int max_tiles, cudaStream_t stream) {
  if (rows <= 0 || K <= 0) return 0;
  if ((K % 32) || (ldq % 4) || (ldo % 8) || fp4_misaligned(out, nullptr) || group_rows <= 0 || fmt < 0 || fmt > 1 ||
      (reinterpret_cast<uintptr_t>(q) & 3) || (tiles != nullptr && num_tiles == nullptr))
    return -2;
  const int nvec = K / 8;
  const int across = nvec >= 1024 ? 256 : (((nvec + 3) / 4 + 31) / 32 * 32), down = 256 / across;
  const long long blocks = (rows + down - 1) / down;
  const dim3 grid((unsigned)(tiles != nullptr ? 148 * 8 : blocks < 148ll * 256 ? blocks : 148ll * 256),
                  (unsigned)((nvec + 4 * across - 1) / (4 * across)));
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, grid, dim3(across, down), 0, stream, reinterpret_cast<const uint8_t*>(q), ldq,
                      reinterpret_cast<const uint8_t*>(scale), reinterpret_cast<const float*>(row_scale),
                      reinterpret_cast<bf16*>(out), ldo, rows, K, fp4_k_tiles(K, fmt == kMxfp4), group_rows,
                      reinterpret_cast<const int4*>(tiles), reinterpret_cast<const int*>(num_tiles), max_tiles);
  };
  const cudaError_t e = fmt == kMxfp4 ? go(dequant_fp4_kernel<true>) : go(dequant_fp4_kernel<false>);
  return e == cudaSuccess ? 0 : -5;
}

}  // extern "C"
