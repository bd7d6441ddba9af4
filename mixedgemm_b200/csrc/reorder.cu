// Reorder-and-quantise kernels for sm_100a.
//
// One kernel template serves activations (FP4 / FP6 / FP8 by K segment) and weights
// (FP4 in all three segments).  It produces byte-for-byte what MixedGemm's
// reorder_bf16_mixed_kernel / reorder_bf16_fp4_kernel write (src/reorder.cu:94-432 of that
// project), but is organised for an HBM-bound B200:
//   * one persistent CTA per SM; a producer warp streams whole rows into a ring of
//     shared-memory stages with 1-D bulk copies (cp.async.bulk + mbarrier), R rows per stage,
//     while 16 consumer warps quantise the previous stage - loads, math and stores overlap;
//   * the reorder index stays in shared memory for the life of the CTA, pre-multiplied to
//     byte offsets;
//   * a thread owns one (row, 32-element group): lanes of a warp walk the R rows of the same
//     group, and rows are skewed by 16 bytes, so the channel gather hits distinct banks; tasks
//     are dealt round-robin to all threads, so every warp sees the same mix of formats;
//   * the group maximum, the E8M0 scale (exponent arithmetic, no log2) and the codes are
//     computed in registers: round-half-away-from-zero is a fused multiply-add against a magic
//     constant (FMA pipe) and the codes come from cvt.rn.satfinite.{e2m1x2,e3m2x2,e4m3x2}.f32;
//     codes leave as 16/8-byte vector stores.
// Waits on mbarriers are bounded (see mg_wait.cuh): on expiry a code goes to the device status word, and a role
// whose wait failed issues no copy, stores nothing and arrives nowhere any more, so the stage it waited for stays
// closed to the others, whose waits then fail as well.
#include <cuda_bf16.h>
#include <cuda_fp4.h>
#include <cuda_fp6.h>
#include <cuda_fp8.h>

#include <atomic>

#include "mg_common.h"
#include "mg_wait.cuh"
#include "overlap.h"
#include "ptx_sm100.cuh"

namespace {

constexpr int kConsumerWarps = 16;
constexpr int kConsumers = kConsumerWarps * 32;
constexpr int kThreads = kConsumers + 32;  // + one producer warp
constexpr int kNormWarps = 8;              // of the kernel with a norm
constexpr int kNormThreads = kThreads + kNormWarps * 32;
constexpr int kMostStages = 8;
constexpr int kNormBarriers = 3 * kMostStages + 4;  // full, normed, empty; full, empty of the residual's two stages
constexpr size_t kStaticSmem = 256;        // of the kernel with a norm: the rows' partial sums
constexpr int kRowSkew = 16;               // bytes added to the shared-memory row pitch

struct SegOut {
  uint8_t* codes;  // packed codes of this segment
  uint8_t* sf;     // swizzled scale bytes
  int katoms;      // ceil(kseg / 128)
  int pitch;       // bytes per row of `codes`
};

struct ReorderParams {
  const uint16_t* X;
  const int16_t* idx;
  int rows, K;
  int g4, g46;  // groups in segment 0, in segments 0+1
  SegOut seg[3];
  int num_tiles;
  int stages;
  long long wait_cycles;
  int* status;
  int skip_load;  // fault injection for the bounded-wait test: the first CTA withholds its n-th stage load (0 = off)
};

// A wait of a whole warp (see mg_wait.cuh): all lanes go on or none does.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* stop, int* status, long long limit,
                                          int code) {
  return __all_sync(0xffffffffu, mg::wait_parity(bar, parity, stop, status, limit, code));
}

// E8M0 byte of the smallest power of two 2^e with maxv <= fmt_max * 2^e, from the bf16
// bit pattern of maxv (fmt_max = 1.5 * 2^2, 1.75 * 2^4, 1.75 * 2^8).
__device__ __forceinline__ int scale_byte(float maxv, int fmt) {
  unsigned a = __float_as_uint(maxv) >> 16;
  int E = (int)(a >> 7), m = (int)(a & 0x7F);
  int sh = fmt == 0 ? 2 : fmt == 1 ? 4 : 8;
  int thr = fmt == 0 ? 64 : 96;
  int sf = E - sh + (m > thr ? 1 : 0);
  sf = max(0, min(254, sf));
  return a == 0 ? 126 : sf;
}

__device__ __forceinline__ unsigned lds_u16(uint32_t addr) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 lds_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// What a thread keeps for its row across the groups it quantises in one stage.
struct RowCtx {
  uint32_t smem_row;    // shared address of the staged row
  uint32_t sf_row;      // row part of the scale offset: (row%32)*16 + (row/32%4)*4
  uint32_t row_blk;     // row / 128
  uint32_t row;
};

// Two fp32 operations in one instruction, each lane rounded as the scalar form rounds it.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// round(x * 2^e) to the nearest integer, halves away from zero, sign of x kept on a zero result.
// `rs` is 2^e * (1 + 2^-12): the fused multiply-add forms x * rs + 1.5 * 2^23 exactly and rounds it
// once, to nearest even, which leaves the wanted integer in the low mantissa bits.  The factor
// (1 + 2^-12) pushes an exact .5 just past the tie and is too small to move anything else across
// one (x has 8 significant bits, so every other product is at least x * 2^-8 away from a tie).
// Subtracting the constant gives the integer back as a float, and or-ing the sign of x restores
// "-0".  All three run on the FMA / ALU pipes; the conversion unit, which a round-to-integer
// instruction would occupy for sixteen cycles per warp, stays free for the code conversions.
// Two values at a time.
__device__ __forceinline__ void scale_round(float& x, float& y, uint64_t rs2) {
  const uint64_t magic = f2(12582912.0f, 12582912.0f), unmagic = f2(-12582912.0f, -12582912.0f);
  float a, b;
  un2(add2(fma2(f2(x, y), rs2, magic), unmagic), a, b);
  x = __uint_as_float(__float_as_uint(a) | (__float_as_uint(x) & 0x80000000u));
  y = __uint_as_float(__float_as_uint(b) | (__float_as_uint(y) & 0x80000000u));
}

// The 32 values of group g (already gathered) and their largest magnitude: scale, quantise, pack, store.
// nan: the scale is NaN, whatever the values.
template <bool WEIGHTS>
__device__ __forceinline__ void emit_group(const ReorderParams& p, const RowCtx& rc, int g, float (&x)[32], float maxv,
                                           bool nan) {
  const int seg = g < p.g4 ? 0 : (g < p.g46 ? 1 : 2);
  const int gs = g - (seg == 0 ? 0 : (seg == 1 ? p.g4 : p.g46));
  const int fmt = WEIGHTS ? 0 : seg;
  const SegOut so = seg == 0 ? p.seg[0] : (seg == 1 ? p.seg[1] : p.seg[2]);

  const int sf = scale_byte(maxv, fmt);
  so.sf[rc.sf_row + (gs & 3) + (size_t)(gs >> 2) * 512 + (size_t)rc.row_blk * 512 * so.katoms] = (uint8_t)(nan ? 255 : sf);
  const float rs = __uint_as_float(((unsigned)(254 - sf) << 23) | 0x800u);  // 2^(127-sf) * (1 + 2^-12)

  const uint64_t rs2 = f2(rs, rs);
#pragma unroll
  for (int i = 0; i < 32; i += 2) scale_round(x[i], x[i + 1], rs2);

  uint8_t* out = so.codes + (size_t)rc.row * so.pitch;
  if (fmt == 0) {
    unsigned wds[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // four cvt.rn.satfinite.e2m1x2.f32 (first source -> high nibble) packed into one word
      asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
          "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
          "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
          "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
          "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
          "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
          : "=r"(wds[q])
          : "f"(x[q * 8]), "f"(x[q * 8 + 1]), "f"(x[q * 8 + 2]), "f"(x[q * 8 + 3]), "f"(x[q * 8 + 4]),
            "f"(x[q * 8 + 5]), "f"(x[q * 8 + 6]), "f"(x[q * 8 + 7]));
    }
    *reinterpret_cast<uint4*>(out + (size_t)gs * 16) = make_uint4(wds[0], wds[1], wds[2], wds[3]);
  } else if (fmt == 1) {
    unsigned w24[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      unsigned p01 = __nv_cvt_float2_to_fp6x2(make_float2(x[q * 4], x[q * 4 + 1]), __NV_E3M2, cudaRoundNearest);
      unsigned p23 = __nv_cvt_float2_to_fp6x2(make_float2(x[q * 4 + 2], x[q * 4 + 3]), __NV_E3M2, cudaRoundNearest);
      w24[q] = (p01 & 0x3Fu) | ((p01 >> 2) & 0xFC0u) | ((p23 & 0x3Fu) << 12) | ((p23 & 0x3F00u) << 10);
    }
    unsigned ow[6];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned a = w24[h * 4], b = w24[h * 4 + 1], c = w24[h * 4 + 2], d = w24[h * 4 + 3];
      ow[h * 3] = a | (b << 24);
      ow[h * 3 + 1] = (b >> 8) | (c << 16);
      ow[h * 3 + 2] = (c >> 16) | (d << 8);
    }
    uint2* o8 = reinterpret_cast<uint2*>(out + (size_t)gs * 24);
    o8[0] = make_uint2(ow[0], ow[1]);
    o8[1] = make_uint2(ow[2], ow[3]);
    o8[2] = make_uint2(ow[4], ow[5]);
  } else {
    unsigned wds[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      unsigned wd = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // the reference rounds the integer to bf16 before the E4M3 conversion
        float a = __bfloat162float(__float2bfloat16_rn(x[q * 4 + j * 2]));
        float b = __bfloat162float(__float2bfloat16_rn(x[q * 4 + j * 2 + 1]));
        unsigned h = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        wd |= (h & 0xFFFFu) << (16 * j);
      }
      wds[q] = wd;
    }
    uint4* o16 = reinterpret_cast<uint4*>(out + (size_t)gs * 32);
    o16[0] = make_uint4(wds[0], wds[1], wds[2], wds[3]);
    o16[1] = make_uint4(wds[4], wds[5], wds[6], wds[7]);
  }
}

// One (row, group): gather, scale, quantise, pack, store.
// NORM: the row may hold values that are not finite; the group's scale is then NaN.
template <bool WEIGHTS, bool NORM = false>
__device__ __forceinline__ void quantise_group(const ReorderParams& p, const RowCtx& rc, uint32_t idx2_addr, int g) {
  float x[32];
  float maxv = 0.f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 iv = lds_v4(idx2_addr + g * 64 + q * 16);
    const unsigned o[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned lo = lds_u16(rc.smem_row + (o[j] & 0xFFFFu));
      const unsigned hi = lds_u16(rc.smem_row + (o[j] >> 16));
      x[q * 8 + j * 2] = __uint_as_float(lo << 16);
      x[q * 8 + j * 2 + 1] = __uint_as_float(hi << 16);
      if constexpr (NORM)
        asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(maxv) : "f"(maxv), "f"(x[q * 8 + j * 2]), "f"(x[q * 8 + j * 2 + 1]));
      else
        maxv = fmaxf(maxv, fmaxf(fabsf(x[q * 8 + j * 2]), fabsf(x[q * 8 + j * 2 + 1])));
    }
  }
  emit_group<WEIGHTS>(p, rc, g, x, maxv, NORM && !(maxv <= 3.4028235e38f));
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// bf16(fp32(a) + fp32(b)) of both halves.  Rounded once here; going through fp32 gives the same bits, since its 24
// significant bits are more than twice the 8 of the result and two.
__device__ __forceinline__ uint32_t add_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// What a norm in front of the quantiser adds to a problem.
struct NormPart {
  const uint16_t* R;  // residual, or null
  uint16_t* U;        // the stream after the addition (with R only)
  const uint16_t* W;
  size_t px, pr, pu;  // row pitches in elements
  float eps, inv_k;
  int stages;         // of the residual's ring; 0: its rows are read from memory
};

// The consumers bring the index in while the producer's first rows are already in flight:
// 16-byte loads, four in flight per thread: element-wise loads through a pointer the compiler must
// assume may alias shared memory ran one after the other, 8 to 28 L2 round trips (4 to 15 us)
// before the first row could be touched.
__device__ __forceinline__ void load_index(const ReorderParams& p, uint16_t* idx2, int tid) {
  const int K = p.K;
  const int16_t* idx = ptx::written_before(p.idx);
  if ((reinterpret_cast<uintptr_t>(idx) & 15) == 0) {
    const uint4* src = reinterpret_cast<const uint4*>(idx);
    uint4* dst = reinterpret_cast<uint4*>(idx2);
    const int nv = K >> 3;
    const unsigned kmax = (unsigned)(K - 1);
    for (int base = 0; base < nv; base += 4 * kConsumers) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = base + u * kConsumers + tid;
        if (j < nv) v[u] = ptx::ldg_v4(src + j);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = base + u * kConsumers + tid;
        if (j < nv) {
          unsigned w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = (min(w[k] & 0xFFFFu, kmax) * 2u) | ((min(w[k] >> 16, kmax) * 2u) << 16);
          dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  } else {
    for (int i = tid; i < K; i += kConsumers) {
      unsigned v = (uint16_t)idx[i];
      v = min(v, (unsigned)(K - 1));
      idx2[i] = (uint16_t)(v * 2);
    }
  }
}

// One CTA's work: block `blk` of the `nblk` blocks that share the rows of problem p.
template <int R, bool WEIGHTS>
__device__ __forceinline__ void reorder_quantize_cta(const ReorderParams& p, int blk, int nblk) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int K = p.K;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.stages;
  const int pitch = 2 * K + kRowSkew;
  uint16_t* idx2 = reinterpret_cast<uint16_t*>(smem);
  uint8_t* tiles = smem + ((2 * K + 15) & ~15);
  const int stage_bytes = R * pitch;
  uint8_t* tail = tiles + (size_t)S * stage_bytes;  // barriers: full[8], empty[8], then the stop flag
  const uint32_t bar0 = ptx::smem_u32(tail);
  volatile int* stop = reinterpret_cast<volatile int*>(tail + 16 * 8);

  ptx::grid_dep_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(bar0 + 8 * s, 1);                     // full: one expect_tx arrival + bytes
      ptx::mbar_init(bar0 + 8 * (8 + s), kConsumerWarps);  // empty: one arrival per consumer warp
    }
    *stop = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  ptx::grid_dep_wait();  // nothing before this line reads or writes global memory

  // This CTA's contiguous share of the rows, walked in stages of up to R rows.
  const int row_begin = (int)((long long)p.rows * blk / nblk);
  const int row_end = (int)((long long)p.rows * (blk + 1) / nblk);
  const int nstage = (row_end - row_begin + R - 1) / R;

  const int G = K >> 5;
  if (warp == kConsumerWarps) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      int skip = blockIdx.x == 0 ? p.skip_load : 0;
      for (int it = 0; it < nstage; ++it, s = s + 1 == S ? 0 : s + 1, ph ^= (s == 0)) {
        if (!mg::wait_parity(bar0 + 8 * (8 + s), ph ^ 1u, stop, p.status, p.wait_cycles, 16)) break;
        if (skip > 0 && --skip == 0) continue;
        const int row0 = row_begin + it * R;
        const int nrows = min(R, row_end - row0);
        const uint32_t fb = bar0 + 8 * s;
        const uint32_t dst = ptx::smem_u32(tiles + (size_t)s * stage_bytes);
        ptx::mbar_expect_tx(fb, (uint32_t)nrows * 2u * K);
        for (int r = 0; r < nrows; ++r)
          ptx::bulk_load_1d(dst + r * pitch, p.X + (size_t)(row0 + r) * K, 2u * K, fb);
      }
    }
  } else {
    // ---------------------------------------------------------------- consumers
    load_index(p, idx2, tid);
    ptx::named_barrier_sync(1, kConsumers);
    // a thread keeps its row
    constexpr int kGStep = kConsumers / R;
    const bool worker = tid < R * kGStep;
    const int r = tid % R;
    const int g0 = tid / R;
    const uint32_t idx2_addr = ptx::smem_u32(idx2);
    int s = 0;
    uint32_t ph = 0;
    for (int it = 0; it < nstage; ++it, s = s + 1 == S ? 0 : s + 1, ph ^= (s == 0)) {
      if (!warp_wait(bar0 + 8 * s, ph, stop, p.status, p.wait_cycles, 32)) break;
      const int row = row_begin + it * R + r;
      if (worker && row < row_end) {
        RowCtx rc;
        rc.smem_row = ptx::smem_u32(tiles + (size_t)s * stage_bytes) + r * pitch;
        rc.sf_row = (uint32_t)(row & 31) * 16 + (uint32_t)((row >> 5) & 3) * 4;
        rc.row_blk = (uint32_t)row >> 7;
        rc.row = (uint32_t)row;
        for (int g = g0; g < G; g += kGStep) quantise_group<WEIGHTS>(p, rc, idx2_addr, g);
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar0 + 8 * (8 + s));
    }
  }
  __syncthreads();
  if (*stop) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land
  }
}

template <int R, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, 1) reorder_quantize_kernel(const __grid_constant__ ReorderParams p) {
  reorder_quantize_cta<R, WEIGHTS>(p, (int)blockIdx.x, (int)gridDim.x);
}

// Several independent problems (own input, index, K split and outputs) in one launch: the CTAs are
// dealt out to the problems in proportion to their bytes, so that a step's activations are quantised
// in one wave instead of one launch - and one partly filled wave - each.
constexpr int kMaxQuant = 8;
struct ReorderMulti {
  int nprob;
  int cta_end[kMaxQuant];  // problem j owns CTAs [cta_end[j-1], cta_end[j])
  int rows_per_stage[kMaxQuant];
  ReorderParams prob[kMaxQuant];
};

template <bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, 1) reorder_quantize_multi_kernel(const __grid_constant__ ReorderMulti mp) {
  int j = 0, first = 0;
  while (j + 1 < mp.nprob && (int)blockIdx.x >= mp.cta_end[j]) first = mp.cta_end[j++];
  const ReorderParams& p = mp.prob[j];
  const int blk = (int)blockIdx.x - first, nblk = mp.cta_end[j] - first;
  switch (mp.rows_per_stage[j]) {
    case 8: reorder_quantize_cta<8, WEIGHTS>(p, blk, nblk); break;
    case 4: reorder_quantize_cta<4, WEIGHTS>(p, blk, nblk); break;
    case 2: reorder_quantize_cta<2, WEIGHTS>(p, blk, nblk); break;
    default: reorder_quantize_cta<1, WEIGHTS>(p, blk, nblk); break;
  }
}

enum Residual { kNoResidual, kStagedResidual, kResidualInMemory };

// B vectors of a staged row, kStep apart: all are read before the first is written back (one after the other, each
// would wait for shared memory by itself).
template <int B, int kStep, Residual RES>
__device__ __forceinline__ uint64_t sum_squares_of(uint32_t xs, uint32_t rs, const uint4* rg, uint4* ug, int i, uint64_t sum2) {
  uint4 a[B], b[B];
#pragma unroll
  for (int t = 0; t < B; ++t) {
    a[t] = lds_v4(xs + (i + t * kStep) * 16);
    if (RES == kStagedResidual) b[t] = lds_v4(rs + (i + t * kStep) * 16);
    if (RES == kResidualInMemory) b[t] = rg[i + t * kStep];
  }
#pragma unroll
  for (int t = 0; t < B; ++t) {
    if (RES != kNoResidual) {
      a[t] = make_uint4(add_pair(a[t].x, b[t].x), add_pair(a[t].y, b[t].y), add_pair(a[t].z, b[t].z), add_pair(a[t].w, b[t].w));
      ug[i + t * kStep] = a[t];
      ptx::sts_v4(xs + (i + t * kStep) * 16, a[t].x, a[t].y, a[t].z, a[t].w);
    }
    const uint32_t u[4] = {a[t].x, a[t].y, a[t].z, a[t].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t u2 = f2(bf16_lo(u[k]), bf16_hi(u[k]));
      sum2 = fma2(u2, u2, sum2);
    }
  }
  return sum2;
}

template <int kStep, Residual RES>
__device__ __forceinline__ uint64_t sum_squares(uint32_t xs, uint32_t rs, const uint4* rg, uint4* ug, int first, int nv) {
  constexpr int B = RES == kNoResidual ? 4 : 2;
  uint64_t sum2 = 0;  // two zeros
  int i = first;
  for (; i + (B - 1) * kStep < nv; i += B * kStep) sum2 = sum_squares_of<B, kStep, RES>(xs, rs, rg, ug, i, sum2);
  for (; i < nv; i += kStep) sum2 = sum_squares_of<1, kStep, RES>(xs, rs, rg, ug, i, sum2);
  return sum2;
}

// h = bf16((u w) v) in the place of u.
template <int B, int kStep>
__device__ __forceinline__ void normalise_some(uint32_t xs, uint32_t wts, uint64_t v2, int i) {
  uint4 a[B], b[B];
#pragma unroll
  for (int t = 0; t < B; ++t) a[t] = lds_v4(xs + (i + t * kStep) * 16), b[t] = lds_v4(wts + (i + t * kStep) * 16);
#pragma unroll
  for (int t = 0; t < B; ++t) {
    const uint32_t u[4] = {a[t].x, a[t].y, a[t].z, a[t].w}, w[4] = {b[t].x, b[t].y, b[t].z, b[t].w};
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float lo, hi;
      un2(mul2(mul2(f2(bf16_lo(u[k]), bf16_hi(u[k])), f2(bf16_lo(w[k]), bf16_hi(w[k]))), v2), lo, hi);
      h[k] = bf16_pair(lo, hi);
    }
    ptx::sts_v4(xs + (i + t * kStep) * 16, h[0], h[1], h[2], h[3]);
  }
}

template <int kStep>
__device__ __forceinline__ void normalise(uint32_t xs, uint32_t wts, float v, int first, int nv) {
  const uint64_t v2 = f2(v, v);
  int i = first;
  for (; i + kStep < nv; i += 2 * kStep) normalise_some<2, kStep>(xs, wts, v2, i);
  if (i < nv) normalise_some<1, kStep>(xs, wts, v2, i);
}

// Root-mean-square norm in front of the quantiser: three kinds of warps, each one stage behind the one before.
//   * the producer copies rows of x, and of the residual into a ring of their own;
//   * kNormWarps / R warps share a row: they read it in 16-byte vectors, add the residual (u goes to the stream
//     and back to the staged row), add up u^2, and then write h = bf16((u w) v) over u;
//   * the quantising warps gather from h as they do from x.  A stage of fewer groups than threads goes on where
//     the one before left off, so that all warps get their share.
// The sum over a row is the only thing that threads wait for one another for, and only those of the row.  (With
// the norm as a phase of the quantising warps and two barriers of all of them in a stage: 8192 x 8192 with a
// residual 99 us, now 88; 2048 x 14336 57.7, now 48.7; 8 x 4096 4.2, now 3.8; but 512 x 4096, one stage to a CTA,
// 6.8, now 7.1.)  Bound: shared memory, whose pipe is 73 % busy; of its wavefronts 55 % are the gather's, three
// quarters of those because the lanes' channels meet in a bank.
template <int R>
__global__ void __launch_bounds__(kNormThreads, 1) norm_reorder_quantize_kernel(const __grid_constant__ ReorderParams p,
                                                                                const __grid_constant__ NormPart np) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_sum[2][kNormWarps];
  const int K = p.K, G = K >> 5;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.stages, SR = np.stages;
  const int pitch = 2 * K + kRowSkew;
  const int stage_bytes = R * pitch;
  uint16_t* idx2 = reinterpret_cast<uint16_t*>(smem);
  const uint32_t wts = ptx::smem_u32(smem) + 2 * K;
  const uint32_t tiles = wts + 2 * K, rtiles = tiles + S * stage_bytes, bar0 = rtiles + SR * stage_bytes;
  volatile int* stop = reinterpret_cast<volatile int*>(smem + (bar0 - ptx::smem_u32(smem)) + kNormBarriers * 8);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto normed = [&](int s) { return bar0 + 8u * (kMostStages + s); };
  auto empty = [&](int s) { return bar0 + 8u * (2 * kMostStages + s); };
  auto rfull = [&](int s) { return bar0 + 8u * (3 * kMostStages + s); };
  auto rempty = [&](int s) { return bar0 + 8u * (3 * kMostStages + 2 + s); };

  ptx::grid_dep_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full(s), 1);  // one expect_tx arrival + bytes
      ptx::mbar_init(normed(s), kNormWarps);
      ptx::mbar_init(empty(s), kConsumerWarps);
    }
    for (int s = 0; s < SR; ++s) {
      ptx::mbar_init(rfull(s), 1);
      ptx::mbar_init(rempty(s), kNormWarps);
    }
    *stop = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  ptx::grid_dep_wait();  // nothing before this line reads or writes global memory

  const int row_begin = (int)((long long)p.rows * blockIdx.x / gridDim.x);
  const int row_end = (int)((long long)p.rows * (blockIdx.x + 1) / gridDim.x);
  const int nstage = (row_end - row_begin + R - 1) / R;
  int s = 0, sr = 0;
  uint32_t ph = 0, phr = 0;
  auto next = [&] {
    if (++s == S) { s = 0; ph ^= 1u; }
    if (++sr >= SR) { sr = 0; phr ^= 1u; }
  };

  if (warp == kConsumerWarps + kNormWarps) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int skip = blockIdx.x == 0 ? p.skip_load : 0;
      for (int it = 0; it < nstage; ++it, next()) {
        const int row0 = row_begin + it * R, nrows = min(R, row_end - row0);
        if (!mg::wait_parity(empty(s), ph ^ 1u, stop, p.status, p.wait_cycles, 16)) break;
        if (skip > 0 && --skip == 0) continue;
        ptx::mbar_expect_tx(full(s), (uint32_t)nrows * 2u * K);
        for (int r = 0; r < nrows; ++r)
          ptx::bulk_load_1d(tiles + s * stage_bytes + r * pitch, p.X + (size_t)(row0 + r) * np.px, 2u * K, full(s));
        if (SR > 0) {
          if (!mg::wait_parity(rempty(sr), phr ^ 1u, stop, p.status, p.wait_cycles, 16)) break;
          ptx::mbar_expect_tx(rfull(sr), (uint32_t)nrows * 2u * K);
          for (int r = 0; r < nrows; ++r)
            ptx::bulk_load_1d(rtiles + sr * stage_bytes + r * pitch, np.R + (size_t)(row0 + r) * np.pr, 2u * K, rfull(sr));
        }
      }
    }
  } else if (warp >= kConsumerWarps) {
    // ---------------------------------------------------------------- norm
    const int ntid = tid - kConsumers, nwarp = warp - kConsumerWarps;
    constexpr int kWarpsPerRow = kNormWarps / R, kStep = kWarpsPerRow * 32;
    const int nr = nwarp / kWarpsPerRow, first = ntid % kStep;
    const int nv = K >> 3;
    {
      uint16_t* w = reinterpret_cast<uint16_t*>(smem + 2 * K);
      const uint16_t* W = ptx::written_before(np.W);
      if ((reinterpret_cast<uintptr_t>(W) & 15) == 0) {
#pragma unroll 4
        for (int j = ntid; j < nv; j += kNormWarps * 32) reinterpret_cast<uint4*>(w)[j] = ptx::ldg_v4(W + j * 8);
      } else {
        for (int j = ntid; j < K; j += kNormWarps * 32) w[j] = ptx::ldg(W + j);
      }
      ptx::named_barrier_sync(2, kNormWarps * 32);
    }
    bool live = true;  // (a warp whose wait failed still comes to the barriers of its rows)
    for (int it = 0; it < nstage; ++it, next()) {
      live = live && warp_wait(full(s), ph, stop, p.status, p.wait_cycles, 32) &&
             (SR == 0 || warp_wait(rfull(sr), phr, stop, p.status, p.wait_cycles, 32));
      const int row = row_begin + it * R + nr;
      const bool work = live && row < row_end;
      const uint32_t xs = tiles + s * stage_bytes + nr * pitch, rs = rtiles + sr * stage_bytes + nr * pitch;
      uint64_t sum2 = 0;  // two zeros
      if (work) {
        const uint4* rg = reinterpret_cast<const uint4*>(np.R + (size_t)row * np.pr);
        uint4* ug = reinterpret_cast<uint4*>(np.U + (size_t)row * np.pu);
        if (np.R == nullptr) sum2 = sum_squares<kStep, kNoResidual>(xs, rs, rg, ug, first, nv);
        else if (SR > 0) sum2 = sum_squares<kStep, kStagedResidual>(xs, rs, rg, ug, first, nv);
        else sum2 = sum_squares<kStep, kResidualInMemory>(xs, rs, rg, ug, first, nv);
      }
      float sum, sum_hi;
      un2(sum2, sum, sum_hi);
      sum += sum_hi;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (SR > 0 && live && lane == 0) ptx::mbar_arrive(rempty(sr));  // (behind the shuffles: the whole warp has read its part)
      if constexpr (kWarpsPerRow > 1) {  // every thread of the row comes here, also after a wait that gave up
        if (lane == 0) s_sum[it & 1][nwarp] = sum;  // (the other half may still be read)
        __syncwarp();
        ptx::named_barrier_sync(3 + nr, kStep);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < kWarpsPerRow; ++i) sum += s_sum[it & 1][nr * kWarpsPerRow + i];
      }
      if (work) {
        // a row whose sum is not finite: all of h is NaN
        const float v = sum <= 3.4028235e38f ? rsqrtf(fmaf(sum, np.inv_k, np.eps)) : __uint_as_float(0x7fc00000u);
        normalise<kStep>(xs, wts, v, first, nv);
      }
      ptx::fence_proxy_async_smem();  // (the next copy into the stage overwrites what was written here)
      __syncwarp();
      if (live && lane == 0) ptx::mbar_arrive(normed(s));
    }
  } else {
    // ---------------------------------------------------------------- quantisers
    load_index(p, idx2, tid);
    ptx::named_barrier_sync(1, kConsumers);
    constexpr int kGStep = kConsumers / R;
    const uint32_t idx2_addr = ptx::smem_u32(idx2);
    const int taken = (R * G + 31) >> 5;  // warps' worth of groups in a stage
    int turn = warp;
    for (int it = 0; it < nstage; ++it, next(), turn -= taken) {
      if (!warp_wait(normed(s), ph, stop, p.status, p.wait_cycles, 32)) break;
      const int t = (turn & (kConsumerWarps - 1)) * 32 + lane;
      const int r = t % R, row = row_begin + it * R + r;
      if (row < row_end) {
        RowCtx rc;
        rc.smem_row = tiles + s * stage_bytes + r * pitch;
        rc.sf_row = (uint32_t)(row & 31) * 16 + (uint32_t)((row >> 5) & 3) * 4;
        rc.row_blk = (uint32_t)row >> 7;
        rc.row = (uint32_t)row;
        for (int g = t / R; g < G; g += kGStep) quantise_group<false, true>(p, rc, idx2_addr, g);
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(empty(s));
    }
  }
  __syncthreads();
  if (*stop) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land
  }
}

size_t smem_bytes(int K, int R, int S) {
  return (size_t)((2 * K + 15) & ~15) + (size_t)S * R * (2 * K + kRowSkew) + 16 * 8 + 16;
}

template <int R, bool WEIGHTS>
int launch(const ReorderParams& p, int grid, size_t smem, cudaStream_t st) {
  auto kern = reorder_quantize_kernel<R, WEIGHTS>;
  if (smem > 48 * 1024) MG_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  MG_CUDA_TRY(mg::launch_kernel(kern, dim3(grid), dim3(kThreads), smem, st, p));
  return MG_OK;
}

// Checks one problem and fills its kernel parameters (everything but the status word and the stage shape, which
// depends on how many CTAs the problem gets).  MG_OK with p->rows == 0 means "nothing to do".
int fill_params(bool weights, const void* X, int rows, int K, const int16_t* idx, int KN, int KS, int KO, uint8_t* o4,
                uint8_t* o6, uint8_t* o8, const size_t* pitches, uint8_t* s4, uint8_t* s6, uint8_t* s8,
                ReorderParams* out) {
  out->rows = 0;
  if (rows < 0 || K <= 0 || KN < 0 || KS < 0 || KO < 0 || KN + KS + KO != K) return MG_ERR_SHAPE;
  if ((KN | KS | KO) & 31) return MG_ERR_SHAPE;
  if (K > 32736) return MG_ERR_SHAPE;  // int16 index
  if (rows == 0) return MG_OK;
  if (!X || !idx) return MG_ERR_NULL;
  if ((KN && (!o4 || !s4)) || (KS && (!o6 || !s6)) || (KO && (!o8 || !s8))) return MG_ERR_NULL;
  if (!mg::aligned(X, 16)) return MG_ERR_ALIGN;
  if (!mg::aligned(o4, 16) || !mg::aligned(o6, 8) || !mg::aligned(o8, 16)) return MG_ERR_ALIGN;

  ReorderParams& p = *out;
  p.X = static_cast<const uint16_t*>(X);
  p.idx = idx;
  p.rows = rows;
  p.K = K;
  p.g4 = KN / 32;
  p.g46 = (KN + KS) / 32;
  const size_t dense[3] = {(size_t)KN / 2, (size_t)(weights ? KS / 2 : KS / 4 * 3), (size_t)(weights ? KO / 2 : KO)};
  const size_t align[3] = {16, (size_t)(weights ? 16 : 8), 16};
  size_t pitch[3];
  for (int i = 0; i < 3; ++i) {
    pitch[i] = pitches && pitches[i] ? pitches[i] : dense[i];
    if (pitch[i] < dense[i] || pitch[i] > 0x7fffffffu) return MG_ERR_SHAPE;
    if (pitch[i] % align[i]) return MG_ERR_ALIGN;
  }
  p.seg[0] = {o4, s4, (KN + 127) / 128, (int)pitch[0]};
  p.seg[1] = {o6, s6, (KS + 127) / 128, (int)pitch[1]};
  p.seg[2] = {o8, s8, (KO + 127) / 128, (int)pitch[2]};
  p.wait_cycles = mg::wait_limit_cycles();
  p.skip_load = mg::options().fault_skip_load;
  return MG_OK;
}

// Rows per stage and stage count of a problem whose rows are shared by `grid` CTAs; returns the
// shared memory a CTA needs, or 0 when the problem does not fit.
size_t stage_shape(ReorderParams* p, int grid, size_t smem_optin, int* rows_per_stage) {
  const int K = p->K, rows = p->rows;
  const size_t budget = smem_optin - 1024;
  const int rows_per_cta = rows / grid;
  static const int kRs[] = {8, 4, 2, 1};
  int R = 1;
  for (int cand : kRs)
    if (smem_bytes(K, cand, 2) <= budget && (2 * cand <= rows_per_cta || cand == 1)) { R = cand; break; }
  int S = 2;
  while (S < 4 && smem_bytes(K, R, S + 1) <= budget) ++S;
  if (smem_bytes(K, R, 2) > budget) S = 1;
  const size_t smem = smem_bytes(K, R, S);
  if (smem > smem_optin) return 0;
  p->num_tiles = (rows + R - 1) / R;
  p->stages = S;
  *rows_per_stage = R;
  return smem;
}

int reorder_quantize(bool weights, const void* X, int rows, int K, const int16_t* idx, int KN, int KS,
                     int KO, uint8_t* o4, uint8_t* o6, uint8_t* o8, const size_t* pitches, uint8_t* s4, uint8_t* s6,
                     uint8_t* s8, void* stream) {
  ReorderParams p;
  int rc = fill_params(weights, X, rows, K, idx, KN, KS, KO, o4, o6, o8, pitches, s4, s6, s8, &p);
  if (rc != MG_OK || p.rows == 0) return rc;
  mg::DeviceInfo di;
  if ((rc = mg::device_info(&di)) != MG_OK || (rc = mg::device_status_word(&p.status)) != MG_OK) return rc;

  // Rows per stage (8, 4, 2 or 1): as many as fit twice (double buffering) beside the index, but no more than
  // half of a CTA's share so that its last stage is not mostly empty.  Then as many stages as
  // fit, up to 4.
  int grid = rows < di.sm_count ? rows : di.sm_count;  // rows are dealt out evenly, at least one per CTA
  const int cap = mg::options().reorder_ctas;  // a caller that runs another kernel beside this one may cap the grid
  if (cap > 0 && grid > cap) grid = cap;
  int R = 1;
  const size_t smem = stage_shape(&p, grid, (size_t)di.smem_optin, &R);
  if (smem == 0) return MG_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

#define MG_LAUNCH_R(RR)                                                            \
  case RR:                                                                         \
    return weights ? launch<RR, true>(p, grid, smem, st) : launch<RR, false>(p, grid, smem, st);
  switch (R) {
    MG_LAUNCH_R(8)
    MG_LAUNCH_R(4)
    MG_LAUNCH_R(2)
    MG_LAUNCH_R(1)
  }
#undef MG_LAUNCH_R
  return MG_ERR_SHAPE;
}

template <bool WEIGHTS>
int launch_multi(const ReorderMulti& mp, int grid, size_t smem, cudaStream_t st) {
  auto kern = reorder_quantize_multi_kernel<WEIGHTS>;
  if (smem > 48 * 1024) MG_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  MG_CUDA_TRY(mg::launch_kernel(kern, dim3(grid), dim3(kThreads), smem, st, mp));
  return MG_OK;
}

}  // namespace

extern "C" int mg_reorder_quantize_multi(int weights, int nprob, const mg_quant_problem_t* probs, void* stream) {
  if (nprob < 0 || nprob > kMaxQuant) return MG_ERR_SHAPE;
  if (nprob == 0) return MG_OK;
  if (!probs) return MG_ERR_NULL;
  mg::DeviceInfo di;
  int rc = mg::device_info(&di);
  if (rc != MG_OK) return rc;
  ReorderMulti mp;
  int n = 0;
  double bytes[kMaxQuant], total = 0;
  for (int j = 0; j < nprob; ++j) {
    const mg_quant_problem_t& q = probs[j];
    ReorderParams& p = mp.prob[n];
    rc = fill_params(weights != 0, q.X, q.rows, q.K, q.idx, q.KN, q.KS, q.KO, q.C4, q.C6, q.C8, q.pitch, q.SF4, q.SF6,
                     q.SF8, &p);
    if (rc != MG_OK) return rc;
    if (p.rows == 0) continue;
    if ((rc = mg::device_status_word(&p.status)) != MG_OK) return rc;
    // Cost of a problem = its elements, weighted by how well its rows pipeline: a row must be whole
    // in shared memory (the index may gather from anywhere in it), so a large K leaves room for only
    // one or two rows per stage and two or three stages, and a CTA then moves 1.5x / 1.3x fewer bytes
    // per second than with four or more rows per stage (measured per CTA with all SMs busy).
    int r_fit = 1;
    for (int cand : {8, 4, 2})
      if (smem_bytes(p.K, cand, 2) <= (size_t)di.smem_optin - 1024) { r_fit = cand; break; }
    bytes[n] = (double)p.rows * p.K * (r_fit == 1 ? 1.48 : r_fit == 2 ? 1.3 : 1.0);
    total += bytes[n];
    ++n;
  }
  if (n == 0) return MG_OK;
  // CTAs in proportion to the cost, at least one and at most one per row; one CTA per SM in all
  int sms = di.sm_count;
  const int cap = mg::options().reorder_ctas;
  if (cap > 0 && sms > cap) sms = cap;
  if (sms < n) sms = n;
  int share[kMaxQuant], used = 0;
  for (int j = 0; j < n; ++j) {
    int g = (int)(sms * bytes[j] / total);
    if (g < 1) g = 1;
    if (g > mp.prob[j].rows) g = mp.prob[j].rows;
    share[j] = g;
    used += g;
  }
  // what rounding down left over goes, one CTA at a time, to the problem whose CTAs carry the most
  while (used < sms) {
    int best = -1;
    for (int j = 0; j < n; ++j)
      if (share[j] < mp.prob[j].rows && (best < 0 || bytes[j] / share[j] > bytes[best] / share[best])) best = j;
    if (best < 0) break;
    ++share[best];
    ++used;
  }
  int grid = 0;
  size_t smem = 0;
  for (int j = 0; j < n; ++j) {
    const int g = share[j];
    const size_t sm = stage_shape(&mp.prob[j], g, (size_t)di.smem_optin, &mp.rows_per_stage[j]);
    if (sm == 0) return MG_ERR_SHAPE;
    if (sm > smem) smem = sm;
    grid += g;
    mp.cta_end[j] = grid;
  }
  for (int j = n; j < kMaxQuant; ++j) { mp.cta_end[j] = grid; mp.rows_per_stage[j] = 1; }
  mp.nprob = n;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return weights ? launch_multi<true>(mp, grid, smem, st) : launch_multi<false>(mp, grid, smem, st);
}

extern "C" int mg_reorder_quantize_x(const void* X, int M, int K, const int16_t* idx, int KN, int KS, int KO,
                                     uint8_t* AN, uint8_t* AS, uint8_t* AO, uint8_t* SFAN, uint8_t* SFAS,
                                     uint8_t* SFAO, void* stream) {
  return reorder_quantize(false, X, M, K, idx, KN, KS, KO, AN, AS, AO, nullptr, SFAN, SFAS, SFAO, stream);
}

extern "C" int mg_reorder_quantize_w(const void* W, int N, int K, const int16_t* idx, int KN, int KS, int KO,
                                     uint8_t* BN, uint8_t* BS, uint8_t* BO, uint8_t* SFBN, uint8_t* SFBS,
                                     uint8_t* SFBO, void* stream) {
  return reorder_quantize(true, W, N, K, idx, KN, KS, KO, BN, BS, BO, nullptr, SFBN, SFBS, SFBO, stream);
}

extern "C" int mg_reorder_quantize_pitched(int weights, const void* X, int rows, int K, const int16_t* idx, int KN,
                                           int KS, int KO, uint8_t* C4, uint8_t* C6, uint8_t* C8,
                                           const size_t* pitches, uint8_t* SF4, uint8_t* SF6, uint8_t* SF8,
                                           void* stream) {
  return reorder_quantize(weights != 0, X, rows, K, idx, KN, KS, KO, C4, C6, C8, pitches, SF4, SF6, SF8, stream);
}

extern "C" size_t mg_code_pitch(int weights, int segment, int kseg) {
  const int kp = (kseg + 127) / 128 * 128;
  if (segment == 0 || weights) return (size_t)kp / 2;
  return segment == 1 ? (size_t)kp / 4 * 3 : (size_t)kp;
}

namespace {

// Rows per stage and stages of x and of the residual, for rows shared by `grid` CTAs; returns the shared memory a CTA
// needs, or 0 when a row does not fit.  A stage costs 0.6 us beside what it holds, so it gets as many rows as
// fit (8192 x 4096 without a residual: 29.6 us with eight rows, 34.5 with four, 43.2 with two).
size_t norm_shape(ReorderParams* p, NormPart* np, int grid, size_t room, int* rows_per_stage) {
  const int K = p->K, most = (p->rows + grid - 1) / grid;
  const size_t row = 2 * (size_t)K + kRowSkew, fixed = 4 * (size_t)K + kNormBarriers * 8 + 16;
  auto fits = [&](int R, int S, int SR) { return fixed + (size_t)R * (S + SR) * row <= room; };
  int R = 1, S = 3, SR = np->R ? 2 : 0;
  for (int cand : {8, 4, 2, 1})
    if (cand <= most && fits(cand, S, SR)) { R = cand; break; }
  if (!fits(R, S, SR)) S = 2, SR = SR ? 1 : 0;
  if (!fits(R, S, SR)) SR = 0;
  if (!fits(R, S, SR)) S = 1;
  if (!fits(R, S, SR)) return 0;
  while (S < kMostStages && S * R < most && fits(R, S + 1, SR)) ++S;
  p->num_tiles = (p->rows + R - 1) / R;
  p->stages = S;
  np->stages = SR;
  *rows_per_stage = R;
  return fixed + (size_t)R * (S + SR) * row;
}

template <int R>
int launch_norm(const ReorderParams& p, const NormPart& np, int grid, size_t smem, const mg::DeviceInfo& di, cudaStream_t st) {
  auto kern = norm_reorder_quantize_kernel<R>;
  static std::atomic<unsigned long long> allowed;
  MG_CUDA_TRY(mg::allow_smem(kern, (size_t)di.smem_optin - kStaticSmem, di.device, allowed));
  MG_CUDA_TRY(mg::launch_kernel(kern, dim3(grid), dim3(kNormThreads), smem, st, p, np));
  return MG_OK;
}

}  // namespace

extern "C" int mg_rms_norm_reorder_quantize(const void* X, size_t ldx, const void* R, size_t ldr, const void* W, float eps,
                                            void* U, size_t ldu, int M, int K, const int16_t* idx, int KN, int KS, int KO,
                                            uint8_t* C4, uint8_t* C6, uint8_t* C8, const size_t* pitches, uint8_t* SF4,
                                            uint8_t* SF6, uint8_t* SF8, void* stream) {
  ReorderParams p;
  NormPart np{};
  if (!(eps >= 0.f && eps <= 3.4028235e38f)) return MG_ERR_SHAPE;
  if (M > 0) {
    if (!W || (R != nullptr) != (U != nullptr)) return MG_ERR_NULL;
    if (M == 1) ldx = ldr = ldu = (size_t)(K > 0 ? K : 0);  // one row has no pitch
    if (ldx < (size_t)K || (R && (ldr < (size_t)K || ldu < (size_t)K))) return MG_ERR_SHAPE;
    if (!mg::aligned(W, 2) || !mg::aligned(R, 16) || !mg::aligned(U, 16)) return MG_ERR_ALIGN;
    if (ldx % 8 || (R && (ldr % 8 || ldu % 8))) return MG_ERR_ALIGN;
  }
  int rc = fill_params(false, X, M, K, idx, KN, KS, KO, C4, C6, C8, pitches, SF4, SF6, SF8, &p);
  if (rc != MG_OK || p.rows == 0) return rc;
  const size_t m = (size_t)M, bytes = (size_t)K * 2;
  const mg::Span x(X, m, bytes, ldx * 2), r(R, m, bytes, ldr * 2), u(U, m, bytes, ldu * 2), w(W, bytes), index(idx, bytes);
  if (mg::any_overlap({mg::Span(C4, m, (size_t)KN / 2, (size_t)p.seg[0].pitch), mg::Span(C6, m, (size_t)KS / 4 * 3, (size_t)p.seg[1].pitch),
                       mg::Span(C8, m, (size_t)KO, (size_t)p.seg[2].pitch), mg::Span(SF4, mg_sf_bytes(M, KN)),
                       mg::Span(SF6, mg_sf_bytes(M, KS)), mg::Span(SF8, mg_sf_bytes(M, KO))},
                      {x, r, w, index, u}))
    return MG_ERR_OVERLAP;
  if (U && (mg::any_overlap({u}, {w, index}) || (mg::overlap(u, x) && !mg::same(u, x)) || (mg::overlap(u, r) && !mg::same(u, r))))
    return MG_ERR_OVERLAP;
  np.R = static_cast<const uint16_t*>(R);
  np.U = static_cast<uint16_t*>(U);
  np.W = static_cast<const uint16_t*>(W);
  np.px = ldx;
  np.pr = ldr;
  np.pu = ldu;
  np.eps = eps;
  np.inv_k = 1.0f / (float)K;
  mg::DeviceInfo di;
  if ((rc = mg::device_info(&di)) != MG_OK || (rc = mg::device_status_word(&p.status)) != MG_OK) return rc;
  int grid = M < di.sm_count ? M : di.sm_count;
  const int cap = mg::options().reorder_ctas;
  if (cap > 0 && grid > cap) grid = cap;
  int rows = 1;
  const size_t smem = norm_shape(&p, &np, grid, (size_t)di.smem_optin - kStaticSmem, &rows);
  if (smem == 0) return MG_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (rows) {
    case 8: return launch_norm<8>(p, np, grid, smem, di, st);
    case 4: return launch_norm<4>(p, np, grid, smem, di, st);
    case 2: return launch_norm<2>(p, np, grid, smem, di, st);
    default: return launch_norm<1>(p, np, grid, smem, di, st);
  }
}

