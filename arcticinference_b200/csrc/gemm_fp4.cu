// Products of microscaled 4-bit operands for sm_100a: out[m, n] = act(g_m h_n sum_b s_mb t_nb sum_{k in b} q_mk p_nk
// + bias_n) + residual_mn, tokens m, features n, blocks b of 16 (nvfp4) or 32 (mxfp4) columns; one matrix, or each row
// with its expert's (rows sorted by expert, the list of row tiles made on the device by the router).
//
// tcgen05.mma kind::mxf4nvf4 / mxf4 takes the blocks' scales from tensor memory and multiplies e2m1 codes at twice the
// rate of fp8; the fp32 accumulator needs no rescaling, only the factors of rows and features at the end.
//
// Features are the tensor core's M side (128 per CTA), tokens its N side: a step's instruction is as wide as
// there are tokens, so a single token or a ragged group costs what it has. One thread feeds a ring of stages by TMA:
// 256 columns of both operands (128 bytes a row, 128-byte swizzle) and their scale tiles. One warp copies a stage's
// scales to tensor memory (sets used in turn) and issues the products into one of two accumulators;
// eight warps drain the other one.
//
// One B200, nvfp4: 8192 x 28672 x 4096 375 to 383 us (5.0 to 5.1 PFLOP/s; mxfp4 354 to 366, 5.3 to 5.4), bound by shared memory
// (608 cycles of copies and operands per 512 of products); 49152 rows of 64 experts, 2 x 1408 from 2048, 148 to 153 us, bound
// by the boundaries of tiles of eight steps; 768 rows 39 us, the weights at 5.4 TB/s. (Lists run in pairs from 640 rows an
// expert on, a border that the router took from bf16 products; in 4 bits the two forms have not been compared.)

#include <string.h>

#include "api.h"
#include "common/elem.cuh"
#include "common/fp4.cuh"
#include "common/pdl.cuh"
#include "common/tensormap.h"

namespace ab200 {

typedef __nv_bfloat16 bf16;

constexpr int kF4EpilogueWarps = 8;
constexpr int kF4Threads = (2 + kF4EpilogueWarps) * 32;
constexpr int kF4MaxStages = 10;
constexpr int kF4StoreBytes = 32 * 64;                 // a warp's staging tile
constexpr int kF4StepCols = 256;                       // columns of a stage: 128 bytes of codes
constexpr uint32_t kF4ABytes = 128 * 128;
// Tensor memory: columns 0 - 383 for two accumulators, then sets of scales. An accumulator of more than 128 tokens
// takes columns 0 - 255 or 128 - 383: the middle ones belong to both, are drained first and handed on at once.
constexpr uint32_t kF4Middle = 128, kF4ScaleAt = 384;

struct Fp4GemmArgs {
  int N, M, kblocks, n_tiles, m_tiles;
  int bn;                  // tokens of a tile
  int stages;
  uint32_t b_bytes, sfa_bytes, sfb_bytes;
  int sfb_tiles;           // row tiles that the scales of a tile's tokens lie in
  int w_row_tiles;         // row tiles of scales per matrix
  int groups;
  int list_tiles;          // tiles of the list that are taken together: two where groups have an even number
  int act;
  GateParams gate;
  const int4* tiles;
  const int* num_tiles;
  const float* x_scale;    // nvfp4: factor per token, null: 1
  const float* w_scale;    // factor per feature [groups][N], null: 1
  const bf16* bias;
  const bf16* residual;
  long long ldr;
  bf16* out;
  long long ldo;
  int* status;
};

struct F4Work {
  int nt;                  // feature tile
  int group, row0, nrows;  // matrix, first token, tokens
  int slot;                // row tile of the tokens' scales
  int shift;               // first token's place in it, in columns of 32
};

__device__ __forceinline__ F4Work f4_work(const Fp4GemmArgs& p, int w) {
  F4Work r;
  if (p.tiles != nullptr) {
    r.nt = w % p.n_tiles;
    const int mt = w / p.n_tiles * p.list_tiles;
    const int4 t = p.tiles[mt];
    r.group = t.x;
    r.row0 = t.y;
    r.nrows = t.z;
    if (p.list_tiles == 2) r.nrows += p.tiles[mt + 1].z;
    // (a list made for other rows or experts reaches beyond neither)
    r.nrows = min(min(r.nrows, p.bn), p.M - r.row0);
    if ((unsigned)r.group >= (unsigned)p.groups || r.row0 < 0) {
      r.group = 0;
      r.row0 = 0;
      r.nrows = 0;
    }
    r.slot = mt;
    r.shift = 0;
    return r;
  }
  // groups of eight feature tiles: what the resident CTAs read stays in L2
  const int per = 8 * p.m_tiles, first = w / per * 8;
  const int wide = min(8, p.n_tiles - first), in = w % per;
  r.nt = first + in % wide;
  const int mt = in / wide;
  r.group = 0;
  r.row0 = mt * p.bn;
  r.nrows = min(p.bn, p.M - r.row0);
  r.slot = r.row0 / kFp4TileRows;
  r.shift = r.row0 % kFp4TileRows / 32;
  return r;
}

// Columns of the instruction: what a tile has, in steps of 16
__device__ __forceinline__ int f4_width(int nrows) { return (nrows + 15) & ~15; }

// First column of an accumulator: side columns 0 - 127 or 256 - 383 with the middle ones between them
__device__ __forceinline__ uint32_t f4_accumulator(int acc, int nrows) {
  return acc == 0 ? 0u : nrows > (int)kF4Middle ? kF4Middle : 2u * kF4Middle;
}

__device__ __forceinline__ float gelu_exact(float x) { return 0.5f * x * (1.f + erff(x * 0.70710678118654752f)); }

template <int ACT>
__device__ __forceinline__ float f4_gated(const GateParams& p, float g, float u) {
  float t;   // g * sigmoid(t)
  if (ACT == kActClampedSwish) {
    g = fminf(g, p.limit);
    u = fminf(fmaxf(u, -p.limit), p.limit) + 1.f;
    t = p.alpha * g;
  } else {   // gelu_tanh(z) = z * sigmoid(2 sqrt(2/pi) (...))
    t = ACT == kActSilu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  }
  return __fdividef(g, 1.f + __expf(-t)) * u;
}

// The factors and biases of a lane's four features of a warp's 32: l / 4 and every eighth after it.
struct F4Features {
  float h[4], bias[4];
};

// A warp's staging tile: [32 tokens][32 features] bf16, the 16-byte pieces of a token's 64 bytes permuted so that eight
// tokens' equal pieces (a matrix fragment) lie in different banks
__device__ __forceinline__ uint32_t f4_piece(int token, int piece) {
  return (uint32_t)(token * 64 + ((piece ^ (token >> 1)) & 3) * 16);
}

// The factor of token c of a tile
__device__ __forceinline__ float f4_token(const float* x_scale, int row0, int c, int nrows) {
  return x_scale == nullptr || c >= nrows ? 1.f : x_scale[row0 + c];
}

// Whether a factor lies outside of 2^-63 .. 2^63. The others are multiplied with each other first, which stays within
// 2^-126 .. 2^126: one operation less per number than a sum times both. (A factor that is no number gives none either way,
// and should not move its neighbours, whose bias is added to an unrounded product, to the other.)
__device__ __forceinline__ bool f4_far(float factor) {
  return (__float_as_uint(factor) & 0x7fffffffu) - 0x20000000u > 0x3f000000u && factor == factor;
}
// v g h for any factors (rows near 2^-126 or 2^127, whose factor and a feature's may have a product outside of fp32): a sum of
// at least 1 takes the smaller factor first, one below 1 the larger, so that what overflows or vanishes on the way does so
// in the end.
__device__ __forceinline__ float f4_scaled(float v, float g, float h) {
  const bool swap = fabsf(g) > fabsf(h);
  const float less = swap ? h : g, more = swap ? g : h;
  return fabsf(v) < 1.f ? v * more * less : v * less * more;
}
// Every other 32 tokens of a warp's 32 features, from `first` on, multiplied by both factors where they lie in tensor memory
// (rare, and small: the epilogues have to stay in the instruction cache)
__device__ __noinline__ void f4_rescale(uint32_t t_addr, int first, int row0, int nrows, const float* x_scale, float h) {
  __syncwarp();
#pragma unroll 1
  for (int c = first; c < nrows; c += (c & 24) == 24 ? 40 : 8) {
    uint32_t r[8];
    tmem_ld_x8(t_addr + (uint32_t)c, r);
    tmem_ld_wait_dep(r);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      r[t] = __float_as_uint(f4_scaled(__uint_as_float(r[t]), f4_token(x_scale, row0, c + t, nrows), h));
    tmem_st_x8(t_addr + (uint32_t)c, r);
  }
  tmem_st_wait();
}

// 16 gate rows (lo) and the 16 up rows they belong to (hi), joined into the staging tile
template <int ACT>
__device__ __forceinline__ void f4_join(const Fp4GemmArgs& p, const uint32_t (&lo)[16], const uint32_t (&hi)[16],
                                        const float2 (&g)[4], const F4Features& ft, uint32_t frag, int c0, int nrows) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c0 + 8 * j >= nrows) break;
    uint32_t q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float a = f4_gated<ACT>(p.gate, __uint_as_float(lo[4 * j + 2 * i]) * (g[j].x * ft.h[i]),
                                    __uint_as_float(hi[4 * j + 2 * i]) * (g[j].x * ft.h[2 + i]));
      const float b = f4_gated<ACT>(p.gate, __uint_as_float(lo[4 * j + 2 * i + 1]) * (g[j].y * ft.h[i]),
                                    __uint_as_float(hi[4 * j + 2 * i + 1]) * (g[j].y * ft.h[2 + i]));
      q[i] = pack_bf16x2(a, b);
    }
    stmatrix_t2(frag + 512u * j, q[0], q[1]);
  }
}

// What an epilogue does, known when it is compiled: the code of all options together does not stay in the instruction
// cache (a tile of 128 x 256 took 6200 cycles to store, more than the products of a K of 1408).
enum F4Epilogue : int { kF4Plain = 0, kF4Any = 1, kF4Gate = 2 };   // factors and bias; GELU and residual too; gate / up

// Tokens c0 .. c0 + 31 of a finished tile: lo, hi the warp's first and last 16 features (tmem_ld_frag_x4), gx the factor
// of token c0 + lane. Fragments
// are transposed through the staging tile, so that a store has 64 consecutive bytes of eight tokens. Moving them by
// shuffles, four by four, cost three times the shared-memory cycles, which the products are short of.
template <int EPI>
__device__ __forceinline__ void f4_store32(const Fp4GemmArgs& p, const uint32_t (&lo)[16], const uint32_t (&hi)[16],
                                           uint8_t* stage, int c0, int row0, int nrows, int feature0,
                                           const F4Features& ft, float gx, int lane) {
  const uint32_t at = smem_u32(stage);
  float2 g[4];
  float* cols = reinterpret_cast<float*>(stage);
  __syncwarp();   // (the tile's last readers are done)
  cols[lane] = gx;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = *reinterpret_cast<const float2*>(cols + 8 * j + 2 * (lane & 3));
  __syncwarp();
  const uint32_t frag = at + f4_piece(lane & 7, lane >> 3);   // + 512 per eight tokens
  if (EPI == kF4Gate) {
    if (p.act == kActSilu) f4_join<kActSilu>(p, lo, hi, g, ft, frag, c0, nrows);
    else if (p.act == kActGeluTanh) f4_join<kActGeluTanh>(p, lo, hi, g, ft, frag, c0, nrows);
    else f4_join<kActClampedSwish>(p, lo, hi, g, ft, frag, c0, nrows);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 16 * i + (lane >> 1), f = (feature0 >> 1) + 8 * (lane & 1);
      if (c0 + t < nrows)
        *reinterpret_cast<uint4*>(p.out + (long long)(row0 + c0 + t) * p.ldo + f) =
            *reinterpret_cast<const uint4*>(stage + f4_piece(t, lane & 1));
    }
    return;
  }
  const int f = feature0 + 8 * (lane & 3);
  if (EPI == kF4Any && p.residual != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 8 * i + (lane >> 2);
      if (c0 + t < nrows && f < p.N)
        *reinterpret_cast<uint4*>(stage + f4_piece(t, lane & 3)) =
            *reinterpret_cast<const uint4*>(p.residual + (long long)(row0 + c0 + t) * p.ldr + f);
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c0 + 8 * j >= nrows) break;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t* r = (i < 2 ? lo : hi) + 4 * j + 2 * (i & 1);
      v[2 * i] = __uint_as_float(r[0]) * (g[j].x * ft.h[i]) + ft.bias[i];
      v[2 * i + 1] = __uint_as_float(r[1]) * (g[j].y * ft.h[i]) + ft.bias[i];
    }
    if (EPI == kF4Any && p.act == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = gelu_exact(v[i]);
    }
    if (EPI == kF4Any && p.residual != nullptr) {
      uint32_t r[4];
      ldmatrix_t4(frag + 512u * j, r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r[i]));
        v[2 * i] += a.x;
        v[2 * i + 1] += a.y;
      }
    }
    stmatrix_t4(frag + 512u * j, pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                pack_bf16x2(v[6], v[7]));
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 8 * i + (lane >> 2);
    if (c0 + t < nrows && f < p.N)
      *reinterpret_cast<uint4*>(p.out + (long long)(row0 + c0 + t) * p.ldo + f) =
          *reinterpret_cast<const uint4*>(stage + f4_piece(t, lane & 3));
  }
}

// Without pairs (experts with few rows) two CTAs share an SM: a tile has few steps, each of which costs some 0.3 us of
// waits and issue whatever it moves, and one CTA's accumulator is drained beside the other's products. 64 experts of
// 2 x 1408, mxfp4, gate / up and down in us, one CTA an SM and two: 768 rows 36.9 + 22.0 and 36.2 + 23.6, 6144 rows 50.6
// + 32.8 and 47.7 + 30.6, 20000 rows 105 + 63 and 88 + 56.
template <bool MX, bool PAIR, int SFB, int EPI>
__global__ void __launch_bounds__(kF4Threads, PAIR ? 1 : 2)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                const __grid_constant__ CUtensorMap tmap_sw, const __grid_constant__ CUtensorMap tmap_sx,
                const __grid_constant__ CUtensorMap tmap_x32, const Fp4GemmArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023u) {  // swizzled tiles need 1024-byte alignment
    pdl_trigger();
    pdl_wait();
    if (threadIdx.x == 0) report_error(p.status, kErrBadArgument, 1500, (int)(smem_u32(smem) & 1023u));
    return;
  }
  constexpr int kTiles = MX ? 2 : 4;      // scale tiles of a step
  constexpr int kCtas = PAIR ? 2 : 1;
  constexpr int kAccs = PAIR ? 2 : 1;
  constexpr uint32_t kColumns = PAIR ? 512 : 256, kScaleAt = PAIR ? kF4ScaleAt : 128u;
  const uint32_t stage_bytes = kF4ABytes + p.b_bytes + p.sfa_bytes + p.sfb_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)p.stages * stage_bytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kF4MaxStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* store_stage = reinterpret_cast<uint8_t*>(bars) + 256;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bars_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bars_base + 8u * s; };
  auto empty_bar = [&](int s) { return bars_base + 8u * (kF4MaxStages + s); };
  auto tfull_bar = [&](int a) { return bars_base + 8u * (2 * kF4MaxStages + a); };
  auto side_bar = [&](int a) { return bars_base + 8u * (2 * kF4MaxStages + 2 + a); };
  const uint32_t middle_bar = bars_base + 8u * (2 * kF4MaxStages + 4);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(side_bar(a), kCtas * kF4EpilogueWarps);   // (the even CTA's: both CTAs drain)
    }
    mbar_init(middle_bar, kCtas * kF4EpilogueWarps);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_x);
    prefetch_tensormap(&tmap_sw);
    prefetch_tensormap(&tmap_sx);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), kColumns);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), kColumns);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();   // the other CTA's barriers are ready for this one's copies and arrivals
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();   // (tensor memory is owned)
  pdl_wait();
  const int total_work =
      (p.tiles != nullptr ? min(*p.num_tiles, p.m_tiles) / p.list_tiles : p.m_tiles) * p.n_tiles;
  const int first_work = (int)blockIdx.x / kCtas, work_step = (int)gridDim.x / kCtas;
  auto work = [&](int w) {
    F4Work none = {};
    return w < total_work ? f4_work(p, w) : none;
  };

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      F4Work t = work(first_work);
      for (int w = first_work; w < total_work && ok; w += work_step) {
        const F4Work after = work(w + work_step);     // (a list's next entry is on its way meanwhile)
        const F4Work now = t;
        t = after;
        if (now.nrows <= 0) continue;
        const int slice = kCtas * now.nt + rank;       // 128 features
        const int row = now.row0 + rank * (f4_width(now.nrows) / 2);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 1500 + stage, kb)) {
            ok = false;
            break;
          }
          // (pairs: one barrier, the even CTA's, collects the copies of both)
          const bool few = !PAIR && now.nrows <= 32;     // (an expert's few rows: a quarter of the box)
          if (rank == 0)
            mbar_arrive_expect_tx(full_bar(stage), few ? stage_bytes - p.b_bytes + 32u * 128u : kCtas * stage_bytes);
          const uint32_t full = PAIR ? map_to_cta(full_bar(stage), 0) : full_bar(stage);
          const uint32_t dst = smem_base + (uint32_t)stage * stage_bytes;
          const uint32_t sfa = dst + kF4ABytes + p.b_bytes;
          if (PAIR) {
            tma_load_3d_pair(dst, &tmap_w, full, kb * 128, slice * 128, now.group);
            tma_load_2d_pair(dst + kF4ABytes, &tmap_x, full, kb * 128, row);
            tma_load_3d_pair(sfa, &tmap_sw, full, 0, kb * kTiles, now.group * p.w_row_tiles + slice);
            tma_load_3d_pair(sfa + p.sfa_bytes, &tmap_sx, full, 0, kb * kTiles, now.slot);
          } else {
            tma_load_3d(dst, &tmap_w, full, kb * 128, slice * 128, now.group);
            tma_load_2d(dst + kF4ABytes, few ? &tmap_x32 : &tmap_x, full, kb * 128, row);
            tma_load_3d(sfa, &tmap_sw, full, 0, kb * kTiles, now.group * p.w_row_tiles + slice);
            tma_load_3d(sfa + p.sfa_bytes, &tmap_sx, full, 0, kb * kTiles, now.slot);
          }
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {   // copies already issued, by either CTA, get a short time to land
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 20000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer -------------------------------
    // (uniform control and one elected lane, see gemm_bf16.cu)
    if (rank == 0) {
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint64_t a0 = make_desc_kmajor_sw128(smem_base);
      const uint64_t s0 = make_desc_scales(smem_base + kF4ABytes + p.b_bytes);
      const uint64_t stage_step = stage_bytes / 16;
      constexpr uint32_t kSfaBytes = kTiles * kFp4ScaleTile;
      int stage = 0, acc = 0;
      uint32_t phase = 0, side_phase = 0, middle_phase = 0;
      // A step's scales go to one of two or four sets in turn: the products that read the set last must be done.
      constexpr int kSets = SFB == 1 ? 4 : 2;
      constexpr uint32_t kSetColumns = 128u / kSets;
      uint32_t set = 0;
      int steps = 0;
      bool ok = true;
      F4Work coming = work(first_work);
      for (int w = first_work; w < total_work && ok; w += work_step) {
        const F4Work t = coming;
        coming = work(w + work_step);
        if (t.nrows <= 0) continue;
        if (!__all_sync(0xffffffffu, mbar_wait(side_bar(acc), side_phase ^ 1u, abort_flag, p.status, 1600 + acc, w)))
          break;
        if (t.nrows > (int)kF4Middle) {
          if (!__all_sync(0xffffffffu, mbar_wait(middle_bar, middle_phase ^ 1u, abort_flag, p.status, 1610, w))) break;
          middle_phase ^= 1u;
        }
        tc_fence_after();
        // (from the list: the same in all lanes, which the compiler cannot know)
        const uint32_t n = __shfl_sync(0xffffffffu, (uint32_t)f4_width(t.nrows), 0);
        const uint32_t shift = __shfl_sync(0xffffffffu, (uint32_t)t.shift, 0);
        const uint32_t idesc = make_idesc_fp4(128 * kCtas, n, MX, 0), idesc_hi = make_idesc_fp4(128 * kCtas, n, MX, 2);
        const uint32_t d_tmem = __shfl_sync(0xffffffffu, tm + f4_accumulator(acc, t.nrows), 0);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          // (a ring of no more stages than sets: the stage's own wait says so)
          if (steps >= kSets && p.stages > kSets) {
            const bool wrapped = stage < kSets;
            if (!__all_sync(0xffffffffu, mbar_wait(empty_bar(stage - kSets + (wrapped ? p.stages : 0)),
                                                   phase ^ (wrapped ? 1u : 0u), abort_flag, p.status, 1620 + stage, kb))) {
              ok = false;
              break;
            }
          }
          if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag, p.status, 1640 + stage, kb))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_desc = a0 + (uint64_t)stage * stage_step;
          const uint64_t b_desc = a_desc + (uint64_t)(kF4ABytes / 16);
          const uint64_t sa_desc = s0 + (uint64_t)stage * stage_step;
          const uint64_t sb_desc = sa_desc + (uint64_t)(kSfaBytes / 16);
          const uint32_t sfa = tm + kScaleAt + set * kSetColumns, sfb = sfa + 16u;
          const uint32_t sfb_first = sfb + shift;
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              tmem_copy_scales<PAIR>(sfa + 4u * j, sa_desc + (uint64_t)(j * (kFp4ScaleTile / 16)));
#pragma unroll
              for (int i = 0; i < SFB; ++i)
                tmem_copy_scales<PAIR>(sfb + 4u * (SFB * j + i),
                                       sb_desc + (uint64_t)((i * kTiles + j) * (kFp4ScaleTile / 16)));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = MX ? k / 2 : k;
              umma_fp4_ss<MX, PAIR>(d_tmem, a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k),
                                    MX && (k & 1) ? idesc_hi : idesc, sfa + 4u * j,
                                    sfb_first + 4u * SFB * j, (kb > 0 || k > 0) ? 1u : 0u);
            }
            if (PAIR) {
              tc_commit_pair(empty_bar(stage));
              if (kb == p.kblocks - 1) tc_commit_pair(tfull_bar(acc));
            } else {
              tc_commit(empty_bar(stage));
              if (kb == p.kblocks - 1) tc_commit(tfull_bar(acc));
            }
          }
          __syncwarp();
          set = set + 1u == (uint32_t)kSets ? 0u : set + 1u;
          ++steps;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (++acc == kAccs) {
          acc = 0;
          side_phase ^= 1u;
        }
      }
    }
  } else {
    // --------------------------------- epilogue --------------------------------
    const int quad = warp & 3;            // TMEM lane quadrant this warp may read
    const int half = (warp - 2) >> 2;     // which of the quadrant's two warps this is
    uint8_t* my_stage = store_stage + (warp - 2) * kF4StoreBytes;
    auto hand_back = [&](uint32_t bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(map_to_cta(bar, 0));
        else mbar_arrive(bar);
      }
    };
    int acc = 0;
    uint32_t acc_phase = 0;
    // A tile's factors (and a list's entries) are requested a tile ahead: one after the other they cost a short K more
    // than its products.
    struct Factors {
      F4Features ft;
      float gx[4];
    };
    auto fetch = [&](const F4Work& t) {
      Factors r;
      const int feature0 = (kCtas * t.nt + rank) * 128 + quad * 32;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = min(feature0 + 8 * i + (lane >> 2), p.N - 1);
        r.ft.h[i] = p.w_scale != nullptr ? p.w_scale[(long long)t.group * p.N + f] : 1.f;
        r.ft.bias[i] = p.bias != nullptr ? __bfloat162float(p.bias[f]) : 0.f;
        r.gx[i] = f4_token(p.x_scale, t.row0, 32 * half + 64 * i + lane, t.nrows);
      }
      return r;
    };
    F4Work coming = work(first_work);
    Factors coming_factors = fetch(coming);
    for (int w = first_work; w < total_work; w += work_step) {
      const F4Work t = coming;
      Factors fc = coming_factors;
      coming = work(w + work_step);
      if (t.nrows <= 0) {
        coming_factors = fetch(coming);
        continue;
      }
      const int feature0 = (kCtas * t.nt + rank) * 128 + quad * 32;
      bool far = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) far |= f4_far(fc.ft.h[i]) | (PAIR || i < 2 ? f4_far(fc.gx[i]) : false);
      far = __any_sync(0xffffffffu, far);
      if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.status, 1700 + acc, w)))
        break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + f4_accumulator(acc, t.nrows) + ((uint32_t)(quad * 32) << 16);
      if (__builtin_expect(far, 0)) {
        const int f = min(feature0 + lane, p.N - 1);
        f4_rescale(t_addr, 32 * half, t.row0, t.nrows, p.x_scale,
                   p.w_scale != nullptr ? p.w_scale[(long long)t.group * p.N + f] : 1.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) fc.ft.h[i] = fc.gx[i] = 1.f;
      }
      if (!PAIR) {
        // (half the registers: 32 tokens at a time)
        coming_factors = fetch(coming);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int c0 = 32 * half + 64 * q;
          const bool any = c0 < t.nrows && feature0 < p.N;
          uint32_t r[2][16];
          __syncwarp();
          if (any) {
            tmem_ld_frag_x4(t_addr + (uint32_t)c0, r[0]);
            tmem_ld_frag_x4(t_addr + (uint32_t)c0 + (16u << 16), r[1]);
            tmem_ld_wait_dep(r[0]);
            tmem_ld_wait_dep(r[1]);
          }
          if (q == 1) hand_back(side_bar(acc));
          if (any) f4_store32<EPI>(p, r[0], r[1], my_stage, c0, t.row0, t.nrows, feature0, fc.ft, fc.gx[q], lane);
        }
      } else {
        // 128 tokens at a time, alternate groups of 32 for the quadrant's two warps. The middle columns first, and
        // both handed back as soon as they are in registers.
        const bool wide = t.nrows > (int)kF4Middle;
        const int first = wide && acc == 0 ? 128 : 0;
        for (int part = 0; part < (wide ? 2 : 1); ++part) {
          const int c0 = (part == 0 ? first : 128 - first) + 32 * half;
          const bool any0 = c0 < t.nrows && feature0 < p.N, any1 = c0 + 64 < t.nrows && feature0 < p.N;
          uint32_t r[4][16];
          __syncwarp();
          if (any0) {
            tmem_ld_frag_x4(t_addr + (uint32_t)c0, r[0]);
            tmem_ld_frag_x4(t_addr + (uint32_t)c0 + (16u << 16), r[1]);
          }
          if (any1) {
            tmem_ld_frag_x4(t_addr + (uint32_t)c0 + 64u, r[2]);
            tmem_ld_frag_x4(t_addr + (uint32_t)c0 + 64u + (16u << 16), r[3]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < 2 ? any0 : any1) tmem_ld_wait_dep(r[i]);
          hand_back(wide && part == 0 ? middle_bar : side_bar(acc));
          if (part == 0) coming_factors = fetch(coming);
          const bool upper = c0 >= 128;
          if (any0) f4_store32<EPI>(p, r[0], r[1], my_stage, c0, t.row0, t.nrows, feature0, fc.ft, upper ? fc.gx[2] : fc.gx[0], lane);
          if (any1)
            f4_store32<EPI>(p, r[2], r[3], my_stage, c0 + 64, t.row0, t.nrows, feature0, fc.ft, upper ? fc.gx[3] : fc.gx[1], lane);
        }
      }
      if (++acc == kAccs) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();   // neither CTA leaves while the other may still signal it
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, kColumns);
    else tmem_dealloc(tmem_base, kColumns);
  }
}

// ------------------------------------------------------------------------------------------
// Few tokens (at most 128): the weights are streamed once, which bounds it. A CTA has 128 features and, where these
// tiles are fewer than the SMs, a part of K: the CTAs of a cluster that share a tile send each other their fp32 sums,
// slices of 16 features, and each adds those of its own slices in the order of K and stores them. The sums go into
// the sender's shared memory first and from there as bulk copies that complete on a barrier of the receiver; stores
// into another CTA's memory, eight bytes a lane, and a cluster barrier on either side took 5.5 us for 128 tokens. The
// weights' first steps are requested into L2 before the wait for the kernel ahead, whose tail (the rows' quantisation)
// they cover: a prefetch changes no value, whoever has written them. One token, nvfp4: 28672 x 4096 13.0 us (5.1 TB/s),
// 4096 x 14336 10.6 us (3.1; 25.4 before K was split), 4096 x 4096 5.5 us; 128 tokens 15.5, 12.9 and 8.1 us.
struct Fp4FewArgs {
  int N, M, kblocks, splits, per_split, stages;
  uint32_t b_bytes, columns, scale_at, recv_at;
  int act;
  const float* x_scale;
  const float* w_scale;
  const bf16* bias;
  const bf16* residual;
  long long ldr;
  bf16* out;
  long long ldo;
  int* status;
};

constexpr int kFewSlice = 16;                    // features of an exchanged slice
constexpr uint32_t kFewHeader = 1024;            // barriers in front of the stages
// Tensor memory: the accumulator, then a set of scales per stage, so that a stage's wait covers its set too. (A CTA of a
// cluster takes at most 256 columns: fp4_few_plan.)
constexpr uint32_t kFewScaleSet = 32;
constexpr int kFewTokens = 128;

__device__ __forceinline__ void tma_prefetch_3d(const void* tmap, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// `bytes` (a multiple of 16) of this CTA's shared memory into another CTA's, completing on a barrier of that CTA
__device__ __forceinline__ void bulk_to_cta(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "r"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <bool MX, int EPI>
__global__ void __launch_bounds__(kF4Threads, 2)
fp4_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
               const __grid_constant__ CUtensorMap tmap_sw, const __grid_constant__ CUtensorMap tmap_sx,
               const Fp4FewArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023u) {  // swizzled tiles need 1024-byte alignment
    pdl_trigger();
    pdl_wait();
    if (threadIdx.x == 0) report_error(p.status, kErrBadArgument, 1800, (int)(smem_u32(smem) & 1023u));
    return;
  }
  constexpr int kTiles = MX ? 2 : 4;
  constexpr uint32_t kSfaBytes = kTiles * kFp4ScaleTile;
  const uint32_t stage_bytes = kF4ABytes + p.b_bytes + 2 * kSfaBytes;
  const uint32_t base = smem_u32(smem);
  const uint32_t stages0 = base + kFewHeader;
  auto full_bar = [&](int s) { return base + 8u * s; };
  auto empty_bar = [&](int s) { return base + 8u * (kF4MaxStages + s); };
  const uint32_t done_bar = base + 8u * (2 * kF4MaxStages);
  const uint32_t recv_bar = done_bar + 8u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 8 * (2 * kF4MaxStages + 2));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* ring = smem + kFewHeader;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / p.splits, split = (int)blockIdx.x % p.splits;
  // sums: [slice][16 features][tokens] floats, sent from where the stages were to a place of their own behind them
  const int pitch = ((p.M + 31) & ~31) + 8, mine = 8 / p.splits;
  const uint32_t slice_bytes = (uint32_t)(kFewSlice * pitch) * 4u, source_bytes = slice_bytes * (uint32_t)mine;
  const int k0 = split * p.per_split, n = min(p.per_split, p.kblocks - k0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    mbar_init(recv_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    if (p.splits > 1) mbar_arrive_expect_tx(recv_bar, (uint32_t)(p.splits - 1) * source_bytes);
    const int ahead = min(n, 2 * p.stages);
    for (int i = 0; i < ahead; ++i) {
      tma_prefetch_3d(&tmap_w, (k0 + i) * 128, tile * 128, 0);
      tma_prefetch_3d(&tmap_sw, 0, (k0 + i) * kTiles, tile);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), p.columns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();   // (tensor memory is owned)
  if (p.splits > 1) cluster_arrive();   // (this CTA's receiving barrier is ready)
  pdl_wait();
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1;
      for (int i = 0; i < n; ++i) {
        if (!mbar_wait(empty_bar(stage), phase, abort_flag, p.status, 1800 + stage, i)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(full_bar(stage), stage_bytes);
        const uint32_t dst = stages0 + (uint32_t)stage * stage_bytes;
        const uint32_t sfa = dst + kF4ABytes + p.b_bytes;
        tma_load_3d(dst, &tmap_w, full_bar(stage), (k0 + i) * 128, tile * 128, 0);
        tma_load_3d(sfa, &tmap_sw, full_bar(stage), 0, (k0 + i) * kTiles, tile);
        tma_load_2d(dst + kF4ABytes, &tmap_x, full_bar(stage), (k0 + i) * 128, 0);
        tma_load_3d(sfa + kSfaBytes, &tmap_sx, full_bar(stage), 0, (k0 + i) * kTiles, 0);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {   // copies already issued get a short time to land
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 20000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem_base, 0);
    const uint64_t a0 = make_desc_kmajor_sw128(stages0);
    const uint64_t s0 = make_desc_scales(stages0 + kF4ABytes + p.b_bytes);
    const uint64_t stage_step = stage_bytes / 16;
    const uint32_t width = (uint32_t)f4_width(p.M);
    const uint32_t idesc = make_idesc_fp4(128, width, MX, 0), idesc_hi = make_idesc_fp4(128, width, MX, 2);
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag, p.status, 1840 + stage, i))) break;
      tc_fence_after();
      const uint64_t a_desc = a0 + (uint64_t)stage * stage_step;
      const uint64_t b_desc = a_desc + (uint64_t)(kF4ABytes / 16);
      const uint64_t sa_desc = s0 + (uint64_t)stage * stage_step;
      const uint64_t sb_desc = sa_desc + (uint64_t)(kSfaBytes / 16);
      const uint32_t sfa = tm + p.scale_at + (uint32_t)stage * kFewScaleSet, sfb = sfa + 16u;
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          tmem_copy_scales<false>(sfa + 4u * j, sa_desc + (uint64_t)(j * (kFp4ScaleTile / 16)));
          tmem_copy_scales<false>(sfb + 4u * j, sb_desc + (uint64_t)(j * (kFp4ScaleTile / 16)));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = MX ? k / 2 : k;
          umma_fp4_ss<MX, false>(tm, a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k),
                                 MX && (k & 1) ? idesc_hi : idesc, sfa + 4u * j, sfb + 4u * j,
                                 (i > 0 || k > 0) ? 1u : 0u);
        }
        tc_commit(empty_bar(stage));
        if (i == n - 1) tc_commit(done_bar);
      }
      __syncwarp();
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
  const int quad = warp & 3, half = (warp - 2) >> 2;
  const uint32_t t_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
  if (p.splits == 1) {
    if (warp >= 2) {
      const int feature0 = tile * 128 + quad * 32;
      F4Features ft;
      Fp4GemmArgs g = {};
      g.N = p.N;
      g.act = p.act;
      g.x_scale = p.x_scale;
      g.residual = p.residual;
      g.ldr = p.ldr;
      g.out = p.out;
      g.ldo = p.ldo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = min(feature0 + 8 * i + (lane >> 2), p.N - 1);
        ft.h[i] = p.w_scale != nullptr ? p.w_scale[f] : 1.f;
        ft.bias[i] = p.bias != nullptr ? __bfloat162float(p.bias[f]) : 0.f;
      }
      float gx = f4_token(p.x_scale, 0, 32 * half + lane, p.M);
      ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag, p.status, 1900, n));
      tc_fence_after();
      const float* x_scale = p.x_scale;
      bool far = f4_far(gx) | f4_far(f4_token(x_scale, 0, 32 * half + 64 + lane, p.M));
#pragma unroll
      for (int i = 0; i < 4; ++i) far |= f4_far(ft.h[i]);
      if (ok && __any_sync(0xffffffffu, far)) {
        const int f = min(feature0 + lane, p.N - 1);
        f4_rescale(t_addr, 32 * half, 0, p.M, x_scale, p.w_scale != nullptr ? p.w_scale[f] : 1.f);
        x_scale = nullptr;
        gx = 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ft.h[i] = 1.f;
      }
      if (ok && feature0 < p.N)
        for (int c0 = 32 * half; c0 < p.M; c0 += 64) {
          const float next = f4_token(x_scale, 0, c0 + 64 + lane, p.M);
          uint32_t lo[16], hi[16];
          __syncwarp();
          tmem_ld_frag_x4(t_addr + (uint32_t)c0, lo);
          tmem_ld_frag_x4(t_addr + (uint32_t)c0 + (16u << 16), hi);
          tmem_ld_wait_dep(lo);
          tmem_ld_wait_dep(hi);
          f4_store32<EPI>(g, lo, hi, ring + (warp - 2) * kF4StoreBytes, c0, 0, p.M, feature0, ft, gx, lane);
          gx = next;
        }
    }
  } else {
    const uint32_t my = cluster_ctarank();
    // A thread finishes eight features of every `across`-th token; what it needs beside the sums is requested before
    // they arrive.
    const int tid = (int)threadIdx.x - 64, across = kF4EpilogueWarps * 32 / (2 * mine);
    const int part = tid / across, first = tid % across;
    const int f = tile * 128 + (int)my * mine * kFewSlice + 8 * part;
    const bool mine_too = warp >= 2 && warp < 2 + kF4EpilogueWarps && f < p.N;
    float h[8], bias[8], gx = 1.f;
    uint4 rq = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = 1.f;
      bias[e] = 0.f;
    }
    if (mine_too) {
      if (p.w_scale != nullptr) {   // (on any 4-byte boundary)
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = p.w_scale[f + e];
      }
      if (p.bias != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = __bfloat162float(p.bias[f + e]);
      }
      if (first < p.M) {
        gx = f4_token(p.x_scale, 0, first, p.M);
        if (EPI == kF4Any && p.residual != nullptr)
          rq = *reinterpret_cast<const uint4*>(p.residual + (long long)first * p.ldr + f);
      }
    }
    if (warp >= 2 && warp < 2 + kF4EpilogueWarps) {
      ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag, p.status, 1900, n));
      tc_fence_after();
      if (ok)
        for (int c0 = 32 * half; c0 < p.M; c0 += 64) {
          uint32_t r[2][16];
          __syncwarp();
          tmem_ld_frag_x4(t_addr + (uint32_t)c0, r[0]);
          tmem_ld_frag_x4(t_addr + (uint32_t)c0 + (16u << 16), r[1]);
          tmem_ld_wait_dep(r[0]);
          tmem_ld_wait_dep(r[1]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float* to = reinterpret_cast<float*>(ring + (uint32_t)(2 * quad + q) * slice_bytes) +
                        (lane >> 2) * pitch + c0 + 2 * (lane & 3);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              *reinterpret_cast<uint2*>(to + 8 * j) = make_uint2(r[q][4 * j], r[q][4 * j + 1]);
              *reinterpret_cast<uint2*>(to + 8 * j + 8 * pitch) = make_uint2(r[q][4 * j + 2], r[q][4 * j + 3]);
            }
          }
        }
      fence_proxy_async_smem();
    }
    __syncthreads();
    cluster_wait();   // every receiver is ready
    if (warp == 2 && lane < p.splits && lane != (int)my) {
      const uint32_t place = (uint32_t)((int)my < lane ? (int)my : (int)my - 1) * source_bytes;
      bulk_to_cta(map_to_cta(base + p.recv_at + place, (uint32_t)lane), stages0 + (uint32_t)lane * source_bytes,
                  source_bytes, map_to_cta(recv_bar, (uint32_t)lane));
    }
    __syncwarp();
    if (warp >= 2 && warp < 2 + kF4EpilogueWarps)
      ok = __all_sync(0xffffffffu, mbar_wait(recv_bar, 0, abort_flag, p.status, 1910, n)) && ok;
    __syncwarp();
    cluster_arrive();   // (nobody leaves before its sums have been received)
    if (mine_too && ok) {
      bool far = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) far |= f4_far(h[e]);
      const float* own = reinterpret_cast<const float*>(ring + my * source_bytes) + (size_t)(8 * part) * pitch;
      const float* others = reinterpret_cast<const float*>(smem + p.recv_at) + (size_t)(8 * part) * pitch;
      for (int m = first; m < p.M; m += across) {
        const int after = m + across;
        float next_gx = 1.f;
        uint4 next_rq = make_uint4(0, 0, 0, 0);
        if (after < p.M) {
          next_gx = f4_token(p.x_scale, 0, after, p.M);
          if (EPI == kF4Any && p.residual != nullptr)
            next_rq = *reinterpret_cast<const uint4*>(p.residual + (long long)after * p.ldr + f);
        }
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int src = 0; src < p.splits; ++src) {
          const float* a = (src == (int)my ? own
                                           : others + (size_t)(src < (int)my ? src : src - 1) * (source_bytes / 4)) + m;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += a[e * pitch];
        }
        if (far || f4_far(gx)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = f4_scaled(v[e], gx, h[e]) + bias[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * (gx * h[e]) + bias[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (EPI == kF4Any && p.act == 1) v[e] = gelu_exact(v[e]);
        }
        if (EPI == kF4Any && p.residual != nullptr) {
          const __nv_bfloat162* rp = reinterpret_cast<const __nv_bfloat162*>(&rq);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 t = __bfloat1622float2(rp[e]);
            v[2 * e] += t.x;
            v[2 * e + 1] += t.y;
          }
        }
        *reinterpret_cast<uint4*>(p.out + (long long)m * p.ldo + f) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
        gx = next_gx;
        rq = next_rq;
      }
    }
    __syncwarp();
    cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, p.columns);
  }
}

struct Fp4FewPlan {
  int x_rows, splits, per_split, stages, columns, scale_at;
  uint64_t recv_at, smem;
};

// Parts of K, stages and memory of a product of M tokens, at most kFewTokens.
static Fp4FewPlan fp4_few_plan(int M, int N, int K, bool mx, int sms) {
  Fp4FewPlan f;
  const int step_tiles = mx ? 2 : 4, kblocks = (K + kF4StepCols - 1) / kF4StepCols, w_row_tiles = (N + 127) / 128;
  f.x_rows = (M + 15) / 16 * 16;
  const uint64_t stage = kF4ABytes + (uint64_t)f.x_rows * 128 + 2ull * step_tiles * kFp4ScaleTile;
  // More tiles than SMs: two CTAs on each, with half of its shared and tensor memory. Fewer: a tile's steps are
  // split.
  const int per_sm = w_row_tiles > sms ? 2 : 1;
  // (0.31 us a step; the exchange 1.0 to 2.0 us between two CTAs, 1.8 to 3.7 between four, by the tokens: 4096 x 4096,
  // 1, 64 and 128 tokens 7.2, 7.5, 8.5 us unsplit, 5.7, 6.5, 7.8 with two parts, 5.2, 6.6, 8.4 with four; eight never paid)
  f.splits = 1;
  double least = 0.31 * kblocks;
  for (int parts = 2; parts <= 4 && w_row_tiles * parts <= sms; parts *= 2) {
    const double t = 0.31 * kblocks / parts + (parts == 2 ? 1.0 + 0.008 * M : 1.8 + 0.015 * M);
    if (t < least) {
      least = t;
      f.splits = parts;
    }
  }
  f.per_split = (kblocks + f.splits - 1) / f.splits;
  while (f.splits > 1 && f.per_split * (f.splits - 1) >= kblocks) {   // every CTA of a cluster has work
    f.splits /= 2;
    f.per_split = (kblocks + f.splits - 1) / f.splits;
  }
  const uint64_t slice = (uint64_t)kFewSlice * (((M + 31) & ~31) + 8) * 4;
  const uint64_t send = f.splits > 1 ? 8 * slice : kF4EpilogueWarps * kF4StoreBytes;
  const uint64_t receive = f.splits > 1 ? (uint64_t)(f.splits - 1) * (8 / f.splits) * slice : 0;
  // A CTA of a cluster holds its tensor memory while it waits for the others, and these wait for theirs without a limit.
  // What two such CTAs hold (more do not fit on an SM: 320 threads of over 68 registers) must fit together, or two
  // clusters of two streams could each hold what the other wants. The other kernels of that kind (gemm_few.cuh) hold at
  // most 128 columns where they leave shared memory for another CTA.
  f.columns = per_sm == 2 || f.splits > 1 ? 256 : 512;
  f.scale_at = M <= 64 ? 64 : 128;
  const int sets = (f.columns - f.scale_at) / (int)kFewScaleSet;
  f.stages = (int)((227 * 1024 / per_sm - 1024 * (per_sm - 1) - kFewHeader - receive) / stage);
  if (f.stages > kF4MaxStages) f.stages = kF4MaxStages;
  if (f.stages > sets) f.stages = sets;
  if (f.stages > f.per_split) f.stages = f.per_split;
  uint64_t body = f.stages * stage;
  if (body < send) body = send;
  f.recv_at = kFewHeader + body;
  f.smem = kFewHeader + body + receive;
  return f;
}

}  // namespace ab200

using namespace ab200;

extern "C" {

// How a product of M <= 128 tokens runs on `sms` SMs: CTAs of a cluster, columns of tensor memory and bytes of shared
// memory of each. -2: not by that kernel.
int ab200_linear_fp4_plan(long long M, int N, int K, int fmt, int sms, int* splits, int* columns, long long* smem) {
  if (M <= 0 || M > kFewTokens || N <= 0 || K <= 0 || (K % 32) || (N % 8) || fmt < 0 || fmt > 1 || sms <= 0) return -2;
  const Fp4FewPlan f = fp4_few_plan((int)M, N, K, fmt == kMxfp4, sms);
  *splits = f.splits;
  *columns = f.columns;
  *smem = (long long)f.smem;
  return 0;
}

// x: codes [M, K / 2] (rows ldx bytes apart), scale tiles sx [row tiles][k_tiles][512], factors gx fp32 [M] or null;
// w: codes [groups][N][K / 2] (w_gstride and ldw bytes), scale tiles sw [groups][ceil(N / 128)][k_tiles][512], factors
// gw fp32 [groups][N] or null; out bf16. K a multiple of 32, N of 8 (of 32 with a gate), strides of codes multiples of
// 16 bytes, ldo and ldr of 8 elements. fmt: 0 nvfp4, 1 mxfp4. act: 0, 1 (GELU); gate: 0, 1 (silu), 2 (gelu_tanh), 3
// (clamped swish): rows of w alternate 16 gate and 16 up rows and out has N / 2 columns; only with `tiles`. With `tiles` (int32 x 4:
// group, first row, rows; *num_tiles of them, at most max_tiles) row tile i's scales are sx's i-th row tile; even: every
// group has an even number of tiles, all but the last two full, of which the last may be empty.
int ab200_linear_fp4(const void* x, long long ldx, const void* sx, const void* gx, const void* w, long long ldw,
                     long long w_gstride, const void* sw, const void* gw, void* out, long long ldo, long long M,
                     int N, int K, int groups, int fmt, const void* bias, const void* residual, long long ldr, int act,
                     int gate, float gate_limit, float gate_alpha, const void* tiles, const void* num_tiles,
                     int max_tiles, int even, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || groups <= 0 || (tiles != nullptr && max_tiles <= 0)) return 0;
  auto odd = [](const void* q, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(q) & mask) != 0; };
  if ((K % 32) || (N % 8) || (gate != 0 && N % 32) || gate < 0 || gate > 3 || act < 0 || act > 1 || fmt < 0 || fmt > 1 ||
      (ldx % 16) || (ldw % 16) || (w_gstride % 16) || (ldo % 8) || (ldr % 8) || odd(x, 15) || odd(w, 15) ||
      odd(sx, 15) || odd(sw, 15) || odd(out, 15) || odd(residual, 15) || M > 0x7fffff00ll ||
      (gate != 0 && (tiles == nullptr || act != 0 || bias != nullptr || residual != nullptr)) ||
      (tiles == nullptr ? groups != 1 : num_tiles == nullptr || bias != nullptr || residual != nullptr))
    return -2;
  const bool mx = fmt == kMxfp4;
  static bool attr_set[64] = {false};
  static int sm_count[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return -3;
  if (!attr_set[dev]) {
    auto large = [](auto kernel) {
      return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess;
    };
    auto both = [&](auto a, auto b) { return large(a) || large(b); };
    if (both(fp4_gemm_kernel<false, false, 1, kF4Plain>, fp4_gemm_kernel<true, false, 1, kF4Plain>) ||
        both(fp4_gemm_kernel<false, false, 1, kF4Gate>, fp4_gemm_kernel<true, false, 1, kF4Gate>) ||
        both(fp4_gemm_kernel<false, true, 1, kF4Plain>, fp4_gemm_kernel<true, true, 1, kF4Plain>) ||
        both(fp4_gemm_kernel<false, true, 1, kF4Any>, fp4_gemm_kernel<true, true, 1, kF4Any>) ||
        both(fp4_gemm_kernel<false, true, 2, kF4Plain>, fp4_gemm_kernel<true, true, 2, kF4Plain>) ||
        both(fp4_gemm_kernel<false, true, 2, kF4Any>, fp4_gemm_kernel<true, true, 2, kF4Any>) ||
        both(fp4_gemm_kernel<false, true, 2, kF4Gate>, fp4_gemm_kernel<true, true, 2, kF4Gate>) ||
        both(fp4_few_kernel<false, kF4Plain>, fp4_few_kernel<true, kF4Plain>) ||
        both(fp4_few_kernel<false, kF4Any>, fp4_few_kernel<true, kF4Any>) ||
        cudaDeviceGetAttribute(&sm_count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return -3;
    attr_set[dev] = true;
  }
  const int sms = sm_count[dev];
  const bool plain = act == 0 && residual == nullptr;
  const int step_tiles = mx ? 2 : 4, kblocks = (K + kF4StepCols - 1) / kF4StepCols;
  const int w_row_tiles = (N + 127) / 128, k_tiles = fp4_k_tiles(K, mx);
  CUtensorMap tw, tx, tsw, tsx, tx32;
  // tokens of a tile (their rows of codes per CTA), row tiles that their scales lie in
  auto make_maps = [&](int x_rows, int sfb_tiles) {
    const uint64_t dims[3] = {(uint64_t)K / 2, (uint64_t)N, (uint64_t)groups};
    const uint64_t strides[2] = {(uint64_t)ldw, (uint64_t)(groups > 1 ? w_gstride : ldw)};
    const uint32_t box[3] = {128, 128, 1};
    auto scales = [&](CUtensorMap* map, const void* base, uint64_t row_tiles, uint32_t box_tiles) {
      const uint64_t sdims[3] = {kFp4ScaleTile / 4, (uint64_t)k_tiles, row_tiles};
      const uint64_t sstrides[2] = {kFp4ScaleTile, (uint64_t)k_tiles * kFp4ScaleTile};
      const uint32_t sbox[3] = {kFp4ScaleTile / 4, (uint32_t)step_tiles, box_tiles};
      return make_tmap_nd(map, base, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, sdims, sstrides, sbox,
                          CU_TENSOR_MAP_SWIZZLE_NONE);
    };
    return make_tmap_nd(&tw, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, dims, strides, box) == 0 &&
           make_tmap_2d(&tx, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)M, (uint64_t)K / 2, (uint64_t)ldx,
                        (uint32_t)x_rows, 128) == 0 &&
           scales(&tsw, sw, (uint64_t)groups * w_row_tiles, 1) == 0 &&
           scales(&tsx, sx, (uint64_t)(tiles != nullptr ? max_tiles : (M + 127) / 128), (uint32_t)sfb_tiles) == 0;
  };

  if (tiles == nullptr && M <= kFewTokens) {
    const Fp4FewPlan plan = fp4_few_plan((int)M, N, K, mx, sms);
    Fp4FewArgs f;
    memset(&f, 0, sizeof(f));
    f.N = N;
    f.M = (int)M;
    f.kblocks = kblocks;
    f.splits = plan.splits;
    f.per_split = plan.per_split;
    f.stages = plan.stages;
    f.b_bytes = (uint32_t)plan.x_rows * 128;
    f.columns = (uint32_t)plan.columns;
    f.scale_at = (uint32_t)plan.scale_at;
    f.recv_at = (uint32_t)plan.recv_at;
    f.act = act;
    f.x_scale = reinterpret_cast<const float*>(gx);
    f.w_scale = reinterpret_cast<const float*>(gw);
    f.bias = reinterpret_cast<const bf16*>(bias);
    f.residual = reinterpret_cast<const bf16*>(residual);
    f.ldr = ldr;
    f.out = reinterpret_cast<bf16*>(out);
    f.ldo = ldo;
    f.status = status;
    if (!make_maps(plan.x_rows, 1)) return -4;
    auto go = [&](auto kernel) {
      return launch_pdl_cluster(kernel, dim3((unsigned)(w_row_tiles * f.splits)), dim3(kF4Threads),
                                (size_t)plan.smem, stream, (unsigned)f.splits, tw, tx, tsw, tsx, f);
    };
    auto by_format = [&](auto nv, auto mxf) { return mx ? go(mxf) : go(nv); };
    const cudaError_t e = plain ? by_format(fp4_few_kernel<false, kF4Plain>, fp4_few_kernel<true, kF4Plain>)
                                : by_format(fp4_few_kernel<false, kF4Any>, fp4_few_kernel<true, kF4Any>);
    return e == cudaSuccess ? 0 : -5;
  }

  Fp4GemmArgs a;
  memset(&a, 0, sizeof(a));
  a.N = N;
  a.M = (int)M;
  a.kblocks = kblocks;
  // Lists whose groups have an even number of tiles have many rows per group: pairs of CTAs on two tiles at a time.
  const bool pair = tiles == nullptr || even != 0;
  a.n_tiles = (N + (pair ? 255 : 127)) / (pair ? 256 : 128);
  a.list_tiles = even != 0 ? 2 : 1;
  a.bn = 128 * a.list_tiles;
  if (tiles == nullptr) {
    // Width of the token tiles: waves of pairs times what 16 steps of a tile take (measured with N = 28672, M = 1500: 75,
    // 85, 110 and 203 us for 256, 192, 128 and 64; M = 300, N = 4096: 11.0, 10.4, 9.6, 13.8).
    const int width[4] = {256, 192, 128, 64};
    const double us[4] = {7.7, 6.7, 5.9, 5.6};
    double best = 1e30;
    for (int i = 0; i < 4; ++i) {
      const long long items = (M + width[i] - 1) / width[i] * a.n_tiles, pairs = sms / 2;
      const double t = (double)((items + pairs - 1) / pairs) * us[i];
      if (t < best) {
        best = t;
        a.bn = width[i];
      }
    }
  }
  a.m_tiles = tiles != nullptr ? max_tiles : (int)((M + a.bn - 1) / a.bn);
  a.sfb_tiles = a.bn > 128 ? 2 : 1;
  a.b_bytes = (uint32_t)(pair ? a.bn / 2 : a.bn) * 128;
  a.sfa_bytes = (uint32_t)step_tiles * kFp4ScaleTile;
  a.sfb_bytes = a.sfa_bytes * (uint32_t)a.sfb_tiles;
  a.w_row_tiles = w_row_tiles;
  a.groups = groups;
  a.act = gate != 0 ? gate : act;
  a.gate.limit = gate_limit;
  a.gate.alpha = gate_alpha;
  a.tiles = reinterpret_cast<const int4*>(tiles);
  a.num_tiles = reinterpret_cast<const int*>(num_tiles);
  a.x_scale = reinterpret_cast<const float*>(gx);
  a.w_scale = reinterpret_cast<const float*>(gw);
  a.bias = reinterpret_cast<const bf16*>(bias);
  a.residual = reinterpret_cast<const bf16*>(residual);
  a.ldr = ldr;
  a.out = reinterpret_cast<bf16*>(out);
  a.ldo = ldo;
  a.status = status;
  const uint64_t stage = kF4ABytes + a.b_bytes + a.sfa_bytes + a.sfb_bytes;
  const uint64_t header = 256 + kF4EpilogueWarps * kF4StoreBytes;
  const int per_sm = pair ? 1 : 2;
  a.stages = (int)((227 * 1024 / per_sm - 1024 * (per_sm - 1) - header) / stage);
  if (a.stages > kF4MaxStages) a.stages = kF4MaxStages;
  const long long total = (long long)a.m_tiles * a.n_tiles;
  if (total > 0x7fffffff) return -6;

  if (!make_maps(pair ? a.bn / 2 : a.bn, a.sfb_tiles) ||
      make_tmap_2d(&tx32, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)M, (uint64_t)K / 2, (uint64_t)ldx, 32, 128) != 0)
    return -4;
  const size_t smem = (size_t)(a.stages * stage + header);
  const long long most = pair ? sms / 2 : 2 * sms;
  const dim3 grid((unsigned)((total < most ? total : most) * (pair ? 2 : 1)));
  auto go = [&](auto kernel) {
    return launch_pdl_cluster(kernel, grid, dim3(kF4Threads), smem, stream, pair ? 2u : 1u, tw, tx, tsw, tsx, tx32,
                              a);
  };
  auto by_format = [&](auto nv, auto mxf) { return mx ? go(mxf) : go(nv); };
  cudaError_t e;
  if (!pair)
    e = gate != 0 ? by_format(fp4_gemm_kernel<false, false, 1, kF4Gate>, fp4_gemm_kernel<true, false, 1, kF4Gate>)
                  : by_format(fp4_gemm_kernel<false, false, 1, kF4Plain>, fp4_gemm_kernel<true, false, 1, kF4Plain>);
  else if (a.sfb_tiles == 1)
    e = plain ? by_format(fp4_gemm_kernel<false, true, 1, kF4Plain>, fp4_gemm_kernel<true, true, 1, kF4Plain>)
              : by_format(fp4_gemm_kernel<false, true, 1, kF4Any>, fp4_gemm_kernel<true, true, 1, kF4Any>);
  else if (gate != 0)
    e = by_format(fp4_gemm_kernel<false, true, 2, kF4Gate>, fp4_gemm_kernel<true, true, 2, kF4Gate>);
  else
    e = plain ? by_format(fp4_gemm_kernel<false, true, 2, kF4Plain>, fp4_gemm_kernel<true, true, 2, kF4Plain>)
              : by_format(fp4_gemm_kernel<false, true, 2, kF4Any>, fp4_gemm_kernel<true, true, 2, kF4Any>);
  return e == cudaSuccess ? 0 : -5;
}

}  // extern "C"
