// Product of 8-bit integers with a scale per token and per channel, for sm_100a:
//
//   D[m,n] = (sum_k A[m,k] B[n,k]) * sa[m] * sb[n] + bias[n]
//
// The sum runs on the tensor cores (tcgen05.mma kind::i8) in 32-bit integers held in tensor memory,
// so it is exact and does not depend on the order or on how K is split.  The channels are the MMA's
// 128-row operand and the tokens its column operand: a thread of the epilogue then owns one channel
// (its scale and bias are two registers), a warp stores 32 consecutive channels of one token, and no
// alignment of D is needed; a tile carries only as many tokens as there are.  Rows beyond M or N and
// bytes beyond K are filled with zeros by the tensor-map loads.
//
//   warp 0      producer: one 128-byte slice of K per stage for both operands (tiled tensor maps,
//               128-byte swizzle)
//   warp 1      MMA issuer: four K = 32 instructions per stage; owns the tensor memory
//   warps 2-    epilogue: four or eight
//
// All waits are bounded (see mg_wait.cuh); a kernel that gives up stores nothing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>

#include "mg_common.h"
#include "mg_wait.cuh"
#include "overlap.h"
#include "ptx_sm100.cuh"
#include "tensor_map.h"

namespace {

using mg::wait_parity;
using mg::wait_parity_cluster;

constexpr int kRows = 128;      // channels of a CTA's tile
constexpr int kMaxSplit = 8;
constexpr size_t kSmemLimit = 227 * 1024;  // of a CTA
constexpr int kMostRows = 0x7ffffe00;  // a tile that starts below still ends in 31 bits

struct Int8Params {
  int M, N;
  int stages;  // 128-byte slices of K
  const float* sa;
  const float* sb;
  const float* bias;
  void* D;
  size_t ldd;
  int* status;
  long long wait_cycles;
  int skip_load;  // fault injection for the bounded-wait test: the first CTA withholds its n-th stage load (0 = off)
};

// Instruction descriptor: 32-bit integer accumulator, signed 8-bit operands, both K-major.
template <int MMA_M, int MMA_N>
constexpr uint32_t kIdescI8 =
    (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(MMA_N >> 3) << 17) | ((uint32_t)(MMA_M >> 4) << 24);

// Tile order: token tiles in groups of eight, all channel tiles of a group before the next group, so
// that the tiles that run at one time share operands in L2.
__device__ __forceinline__ void raster(int t, int tiles_m, int tiles_n, int& m_tile, int& n_tile) {
  constexpr int kGroup = 8;
  const int g = t / (kGroup * tiles_n), r = t - g * kGroup * tiles_n;
  const int rows = min(kGroup, tiles_m - g * kGroup);
  m_tile = g * kGroup + r % rows;
  n_tile = r / rows;
}

template <typename T>
__device__ __forceinline__ T round_to(float f);
template <>
__device__ __forceinline__ __nv_bfloat16 round_to(float f) {
  return __float2bfloat16_rn(f);
}
template <>
__device__ __forceinline__ __half round_to(float f) {
  return __float2half_rn(f);
}
template <>
__device__ __forceinline__ float round_to(float f) {
  return f;
}

// What a warp of the epilogue keeps for its 32 channels (one per lane).
template <typename T>
struct Channel {
  float sb, bias;
  bool real;
  T* out;  // this channel's column of D, at the tile's first token

  __device__ __forceinline__ Channel(const Int8Params& p, int n, int m0)
      : sb(0.f), bias(0.f), real(n < p.N), out(static_cast<T*>(p.D) + (size_t)m0 * p.ldd + n) {
    if (real) {
      sb = p.sb[n];
      if (p.bias) bias = p.bias[n];
    }
  }
};

// Scales, rounds and stores the sums of NC tokens (from token `c` of the tile, `left` of them real) of
// this lane's channel.  `scales` holds the tile's token scales in shared memory.  All loads come before
// all stores: one column after the other, a load behind a store that may alias it, took 75 cycles a
// column, 10 us for a tile of 256 tokens.
template <int NC, typename T>
__device__ __forceinline__ void finish(const int* sum, uint32_t scales, int c, int left, const Channel<T>& ch, size_t ldd) {
  constexpr int kStep = NC < 8 ? NC : 8;
  T v[NC];
#pragma unroll
  for (int i = 0; i < NC; i += 4) {
    const uint4 sv = ptx::lds_v4(scales + (uint32_t)(c + i) * 4u);
    const uint32_t sa[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[i + k] = round_to<T>(__fmaf_rn(__fmul_rn((float)sum[i + k], __uint_as_float(sa[k])), ch.sb, ch.bias));
  }
  T* out = ch.out + (size_t)c * ldd;
  if (left >= NC) {
#pragma unroll
    for (int i = 0; i < NC; ++i) out[(size_t)i * ldd] = v[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < NC; i += kStep) {
    if (left >= i + kStep) {
#pragma unroll
      for (int k = 0; k < kStep; ++k) out[(size_t)(i + k) * ldd] = v[i + k];
    } else if (left > i) {
#pragma unroll
      for (int k = 0; k < kStep; ++k)
        if (i + k < left) out[(size_t)(i + k) * ldd] = v[i + k];
    }
  }
}

// The token scales of a tile into a warp's part of shared memory.
template <int BT>
__device__ __forceinline__ void stage_scales(float* dst, const Int8Params& p, int m0, int lane) {
#pragma unroll
  for (int c = 0; c < BT; c += 32) dst[c + lane] = m0 + c + lane < p.M ? p.sa[m0 + c + lane] : 0.f;
  __syncwarp();
}

// A tile of 128 channels x BT tokens per cluster; the CTAs of the cluster (gridDim.z of them, along z)
// share its K and add their sums through distributed shared memory.  Up to 64 tokens a stage holds two slices of
// 128 bytes of K, so that barriers and commits are paid once for both: along K a slice takes 0.135 us in place of
// 0.165 (32 tokens) and 0.145 in place of 0.18 (64).  With 128 tokens the ring holds too few stages of two slices
// to keep up with memory along a long K: 128 x 4096 x 14336 took 17.3 us in place of 15.7 (a shorter one gained:
// 2048 x 1024 x 4096 9.7 in place of 10.1).
template <int BT>
struct SmallCfg {
  static constexpr int SLICES = BT <= 64 ? 2 : 1;
  static constexpr uint32_t W_BYTES = kRows * 128;  // of a slice
  static constexpr uint32_t T_BYTES = BT * 128;
  static constexpr uint32_t STAGE_BYTES = SLICES * (W_BYTES + T_BYTES);
  static constexpr int MOST_STAGES = 8;
  // sums received from the other CTAs: this CTA's BT / splits columns from splits - 1 senders
  static constexpr uint32_t recv_bytes(int splits) { return (uint32_t)(splits - 1) * kRows * (BT / splits) * 4; }
  // one epilogue warp to a quadrant of the tensor-memory lanes, two from 64 tokens on (half of them each)
  static constexpr int SIDE = BT >= 64 ? 2 : 1, EPILOGUE = 4 * SIDE, COLS = BT / SIDE, THREADS = (2 + EPILOGUE) * 32;
  static constexpr uint32_t SCALE_BYTES = 4 * BT * 4;  // the tile's token scales, once per quadrant
  static constexpr size_t smem(int splits, int ring) {
    return 1024 + (size_t)ring * STAGE_BYTES + 256 + SCALE_BYTES + recv_bytes(splits);
  }
  static constexpr int ring(int splits) {  // stages that fit
    int n = 1;
    while (n < MOST_STAGES && smem(splits, n + 1) <= kSmemLimit) ++n;
    return n;
  }
};

template <int BT, typename T>
__global__ void __launch_bounds__(SmallCfg<BT>::THREADS) int8_gemm_kernel(
    const Int8Params p, int ring, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmT) {
  using C = SmallCfg<BT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + (uint32_t)ring * C::STAGE_BYTES;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (C::MOST_STAGES + s); };
  const uint32_t done_bar = bar0 + 8u * (2 * C::MOST_STAGES);
  volatile uint32_t* tmem_holder =
      reinterpret_cast<volatile uint32_t*>(gbase + (bar0 - base) + 8 * (2 * C::MOST_STAGES + 1));
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const uint32_t scales = bar0 + 256u;
  const uint32_t recv = scales + C::SCALE_BYTES;  // [sender][column / 4][channel][4] sums

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = gridDim.z, rank = blockIdx.z;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ring; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(done_bar, 1);
    *stop = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmW);
    ptx::prefetch_tmap(&tmT);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_holder)), BT);
    ptx::tmem_relinquish();
  }
  ptx::grid_dep_launch_dependents();
  ptx::tc_fence_before();
  __syncthreads();
  if (splits > 1) ptx::cluster_arrive();  // (waited for below, before anyone stores into another CTA)
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  ptx::grid_dep_wait();  // the prologue above touched no global memory

  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * BT;
  const int quad = warp & 3, row = quad * 32 + lane;  // an epilogue warp's tensor-memory lanes = channels of the tile
  const Channel<T> chan(p, warp >= 2 ? n0 + row : p.N, m0);
  const int side = (warp - 2) >> 2;  // an epilogue warp's share of the tokens
  const uint32_t my_scales = scales + (uint32_t)((warp - 2) & 3) * (BT * 4);
  const int left = p.M - m0;     // tokens of this tile and beyond
  const int cols = BT / splits;  // columns this CTA finishes
  const uint32_t per_sender = (uint32_t)kRows * cols * 4;
  const int stages = (p.stages + C::SLICES - 1) / C::SLICES;
  const int s0 = (int)((long long)stages * rank / splits), s1 = (int)((long long)stages * (rank + 1) / splits);

  if (warp == 0) {
    const bool leader = ptx::elect_one();
    int slot = 0;
    uint32_t phase = 0;
    int skip = (blockIdx.x | blockIdx.y | blockIdx.z) == 0 ? p.skip_load : 0;
    for (int s = s0; s < s1; ++s) {
      if (!wait_parity(empty_bar(slot), phase ^ 1u, stop, p.status, p.wait_cycles, 1)) break;
      if (leader && !(skip > 0 && --skip == 0)) {
        const uint32_t sbase = base + slot * C::STAGE_BYTES, fb = full_bar(slot);
        ptx::mbar_expect_tx(fb, C::STAGE_BYTES);
#pragma unroll
        for (int i = 0; i < C::SLICES; ++i) {  // (a slice beyond K reads as zeros)
          const int k = (s * C::SLICES + i) * 128;
          ptx::tma_load_2d(sbase + i * C::W_BYTES, &tmW, k, n0, fb);
          ptx::tma_load_2d(sbase + C::SLICES * C::W_BYTES + i * C::T_BYTES, &tmT, k, m0, fb);
        }
      }
      if (++slot == ring) { slot = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    const bool leader = ptx::elect_one();
    constexpr uint32_t kIdesc = kIdescI8<kRows, BT>;
    int slot = 0;
    uint32_t phase = 0, accumulate = 0;
    bool live = true;
    for (int s = s0; s < s1; ++s) {
      if (!wait_parity(full_bar(slot), phase, stop, p.status, p.wait_cycles, 2)) { live = false; break; }
      ptx::tc_fence_after();
      const uint32_t sbase = base + slot * C::STAGE_BYTES;
      const uint32_t w_lo = ptx::desc_lo(sbase), t_lo = ptx::desc_lo(sbase + C::SLICES * C::W_BYTES);
      if (leader) {
#pragma unroll
        for (int j = 0; j < 4 * C::SLICES; ++j) {
          ptx::mma_i8(tmem, w_lo + (j >> 2) * (C::W_BYTES >> 4) + (j & 3) * 2, t_lo + (j >> 2) * (C::T_BYTES >> 4) + (j & 3) * 2,
                      ptx::kDescHiSw128, kIdesc, accumulate);
          accumulate = 1;
        }
        ptx::tc_commit(empty_bar(slot));
      }
      if (++slot == ring) { slot = 0; phase ^= 1u; }
    }
    if (leader && live) ptx::tc_commit(done_bar);
  } else {
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
    stage_scales<BT>(reinterpret_cast<float*>(gbase + (my_scales - base)), p, m0, lane);  // (the same values from either side)
    const bool store = wait_parity(done_bar, 0, stop, p.status, p.wait_cycles, 8) && chan.real && !*stop;
    __syncwarp();
    ptx::tc_fence_after();
    if (splits == 1) {
#pragma unroll 1
      for (int c = side * C::COLS; c < (side + 1) * C::COLS && c < left; c += 32) {
        uint32_t r[32];
        ptx::tmem_ld_32x32(taddr + c, r);
        ptx::tmem_ld_wait();
        if (store) finish<32>(reinterpret_cast<const int*>(r), my_scales, c, left - c, chan, p.ldd);
      }
    } else {
      // Column group g of this tile (BT / splits columns) is finished by CTA g: the others send it
      // theirs, 16 bytes (four columns of a channel) at a time.
      ptx::cluster_wait();  // every CTA of the cluster runs
#pragma unroll 1
      for (int c = side * C::COLS; c < (side + 1) * C::COLS && c < left; c += 32) {
        uint32_t r[32];
        ptx::tmem_ld_32x32(taddr + c, r);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          const int col = c + v * 4, g = col / cols;
          if (g != rank && col < left) {
            const uint32_t dst = recv + (uint32_t)(rank - (rank > g)) * per_sender +
                                 (uint32_t)((col - g * cols) >> 2) * (kRows * 16u) + (uint32_t)row * 16u;
            ptx::st_cluster_v4(ptx::map_to_cta(dst, (uint32_t)g), r[v * 4], r[v * 4 + 1], r[v * 4 + 2], r[v * 4 + 3]);
          }
        }
      }
    }
  }

  if (splits > 1) {
    __syncwarp();
    if (warp < 2) ptx::cluster_wait();
    // every wait above is bounded, so every thread of the cluster arrives here; a CTA that gave up
    // tells the others first, so that nobody adds sums that were never sent
    __syncthreads();
    if (threadIdx.x == 0 && *stop)
      for (int g = 0; g < splits; ++g) ptx::st_cluster_u32(ptx::map_to_cta(ptx::smem_u32(const_cast<int*>(stop)), (uint32_t)g), 1u);
    ptx::cluster_sync();
    if (warp >= 2 && !*stop) {
      const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
      const int first = rank * cols;
      for (int c = side * 4; c < cols && first + c < left; c += 4 * C::SIDE) {
        uint32_t r[4];
        ptx::tmem_ld_32x4(taddr + first + c, r);
        ptx::tmem_ld_wait();
        int sum[4] = {(int)r[0], (int)r[1], (int)r[2], (int)r[3]};
        for (int s = 0; s < splits - 1; ++s) {
          const uint4 a = ptx::lds_v4(recv + (uint32_t)s * per_sender + (uint32_t)(c >> 2) * (kRows * 16u) +
                                         (uint32_t)row * 16u);
          sum[0] += (int)a.x;
          sum[1] += (int)a.y;
          sum[2] += (int)a.z;
          sum[3] += (int)a.w;
        }
        if (chan.real) finish<4>(sum, my_scales, first + c, left - first - c, chan, p.ldd);
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (*stop) {
    // give copies and MMAs that are still in flight time to land before the CTA goes away
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) ptx::tmem_dealloc(tmem, BT);
}

// ---------------------------------------------------------------- single tokens
// One or two tokens: the weights are read once, straight into registers, and multiplied with dp4a.  The
// product is bound by their bytes, and what the tensor-core form adds to reading them (staging, the MMA's
// and the cluster's hand-overs) shows: 1 x 4096 x 4096 5.0 us here against 6.5 there, 1 x 6144 x 4096 6.7 / 8.4,
// 1 x 4096 x 14336 11.4 / 12.8, 2 x 14336 x 4096 11.5 / 13.3.  With four tokens dp4a and the tokens' bytes are
// the bound (4096 x 14336: 13.4 / 12.7).  A warp takes four channels, so that the tokens' bytes, which all warps
// share through L1, serve four rows (two rows: 13.9 us at 1 x 14336 x 4096, four: 11.4); `parts` warps of a
// CTA share them when there are too few channels to keep the memory busy.
constexpr int kFewWarps = 4, kFewRows = 4, kFewUnroll = 4, kFewTokens = 2;

template <int MT, typename T>
__global__ void __launch_bounds__(kFewWarps * 32) int8_few_tokens_kernel(const Int8Params p, const int8_t* A,
                                                                         size_t lda, const int8_t* B, size_t ldb,
                                                                         int K, int parts) {
  __shared__ int s_sum[kFewWarps][kFewRows * MT];
  ptx::grid_dep_launch_dependents();
  ptx::grid_dep_wait();
  A = ptx::written_before(A);
  B = ptx::written_before(B);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / parts, part = warp - group * parts;
  const int n0 = (int)(blockIdx.x * (kFewWarps / parts) + group) * kFewRows;
  // rows beyond the last channel or token stand for the last one; nothing of them is stored
  const int8_t* w[kFewRows];
  const int8_t* x[MT];
#pragma unroll
  for (int r = 0; r < kFewRows; ++r) w[r] = B + (size_t)min(n0 + r, p.N - 1) * ldb;
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = A + (size_t)min(m, p.M - 1) * lda;

  int sum[kFewRows][MT] = {};
  const int chunks = K >> 4;  // whole 16-byte vectors
  const int c1 = (int)((long long)chunks * (part + 1) / parts);
  for (int c = (int)((long long)chunks * part / parts) + lane; c < c1; c += 32 * kFewUnroll) {
    uint4 wv[kFewRows][kFewUnroll];
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u)
#pragma unroll
      for (int r = 0; r < kFewRows; ++r)
        wv[r][u] = c + 32 * u < c1 ? ptx::ldg_v4_once(w[r] + (size_t)(c + 32 * u) * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint4 xv = make_uint4(0, 0, 0, 0);
        if (c + 32 * u < c1) xv = ptx::ldg_v4(x[m] + (size_t)(c + 32 * u) * 16);
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
          sum[r][m] = __dp4a((int)wv[r][u].x, (int)xv.x, sum[r][m]);
          sum[r][m] = __dp4a((int)wv[r][u].y, (int)xv.y, sum[r][m]);
          sum[r][m] = __dp4a((int)wv[r][u].z, (int)xv.z, sum[r][m]);
          sum[r][m] = __dp4a((int)wv[r][u].w, (int)xv.w, sum[r][m]);
        }
      }
    }
  }
  // the last K % 16 bytes of a row, one a lane
  if (part == parts - 1 && lane < (K & 15)) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < kFewRows; ++r) sum[r][m] += (int)w[r][chunks * 16 + lane] * (int)x[m][chunks * 16 + lane];
  }
#pragma unroll
  for (int r = 0; r < kFewRows; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m) sum[r][m] = __reduce_add_sync(0xffffffffu, sum[r][m]);
  if (parts > 1) {
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < kFewRows; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) s_sum[warp][r * MT + m] = sum[r][m];
    }
    __syncthreads();
    if (part != 0) return;
  }
  // lane r * MT + m finishes channel n0 + r of token m
  int total = 0;
#pragma unroll
  for (int r = 0; r < kFewRows; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (lane == r * MT + m) total = sum[r][m];
  const int n = n0 + lane / MT, m = lane % MT;
  if (lane < kFewRows * MT && n < p.N && m < p.M) {
    for (int i = 1; i < parts; ++i) total += s_sum[warp + i][lane];
    const float bias = p.bias ? p.bias[n] : 0.f;
    static_cast<T*>(p.D)[(size_t)m * p.ldd + n] = round_to<T>(__fmaf_rn(__fmul_rn((float)total, p.sa[m]), p.sb[n], bias));
  }
}

template <int MT, typename T>
int launch_few(const Int8Params& p, const int8_t* A, size_t lda, const int8_t* B, size_t ldb, int K, int sms, cudaStream_t st) {
  const int groups = (p.N + kFewRows - 1) / kFewRows;
  // 16 warps an SM at least, but no part of a row shorter than a 16-byte vector for every lane
  int parts = 1;
  while (parts < kFewWarps && (long long)groups * parts < 16ll * sms && K >= parts * 2 * 32 * 16) parts *= 2;
  const int per_cta = kFewWarps / parts;
  MG_CUDA_TRY(mg::launch_kernel(int8_few_tokens_kernel<MT, T>, dim3((groups + per_cta - 1) / per_cta), dim3(kFewWarps * 32), 0, st, p,
                                A, lda, B, ldb, K, parts));
  return MG_OK;
}

// ---------------------------------------------------------------- CTA-pair form
// Two CTAs of a cluster compute 256 channels x 256 tokens with tcgen05.mma.cta_group::2: each stages
// its own 128 channels and half of the tokens, and one instruction of the leader drives both tensor
// cores.  The loads of both CTAs are counted on the leader's barrier.  Two accumulators alternate, so
// the epilogue of a tile runs under the products of the next.  Persistent: cluster c takes tiles
// c, c + clusters, ... for as many whole rounds as there are; the tiles that are left over (4 of the 448 of
// 2048 x 14336 on 74 clusters would take a round of their own) are cut into two or four parts of 128 or 64
// tokens, as long as every cluster gets at most one.
struct PairCfg {
  static constexpr int BT = 256, STAGES = 6;
  static constexpr uint32_t W_BYTES = 128 * 128;
  static constexpr uint32_t T_BYTES = BT / 2 * 128;
  static constexpr uint32_t STAGE_BYTES = W_BYTES + T_BYTES;
  // Eight epilogue warps, two to a quadrant of the tensor-memory lanes, each with half of the tokens: 2048 x
  // 14336 x 512 takes 21.8 us with them and 24.9 with four; from K = 4096 on it makes no difference.
  static constexpr int SIDE = 2, EPILOGUE = 4 * SIDE, COLS = BT / SIDE, THREADS = (2 + EPILOGUE) * 32;
  static constexpr uint32_t SCALE_BYTES = EPILOGUE * COLS * 4;  // each warp's token scales
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + SCALE_BYTES + 256;
};

// rounds: whole rounds of tiles;  cut: parts of a tile that is left over (1, 2, 4), tmPart: their load of tokens
template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::THREADS, 1)
int8_gemm_pair_kernel(const Int8Params p, int rounds, int cut, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmT, const __grid_constant__ CUtensorMap tmPart) {
  using C = PairCfg;
  constexpr int BT = C::BT;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t scales = base + C::STAGES * C::STAGE_BYTES;
  const uint32_t bar0 = scales + C::SCALE_BYTES;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (C::STAGES + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * C::STAGES + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * C::STAGES + 2 + a); };
  volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(gbase + C::STAGES * C::STAGE_BYTES + C::SCALE_BYTES +
                                                                        8 * (2 * C::STAGES + 4));
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);  // (used in the leader only)
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(tfull_bar(a), 1);
      ptx::mbar_init(tempty_bar(a), 2 * C::EPILOGUE);  // the epilogue warps of both CTAs (used in the leader only)
    }
    *stop = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmW);
    ptx::prefetch_tmap(&tmT);
  }
  ptx::cluster_sync();  // both CTAs' barriers exist before anything arrives on them
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_u32(const_cast<uint32_t*>(tmem_holder)), 2 * BT);
    ptx::tmem_relinquish_pair();
  }
  ptx::grid_dep_launch_dependents();
  ptx::tc_fence_before();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  ptx::grid_dep_wait();  // the prologue above touched no global memory

  const int tiles_n = (p.N + 255) / 256, tiles_m = (p.M + BT - 1) / BT;
  const int first = (int)ptx::cluster_id_x(), step = (int)ptx::nclusters_x();
  // item i of this cluster: its first channel and token, and how many tokens it has
  auto locate = [&](int i, int& n0, int& m0, int& width) {
    const bool whole = i < rounds;
    int m_tile, n_tile;
    raster(whole ? first + i * step : rounds * step + first / cut, tiles_m, tiles_n, m_tile, n_tile);
    width = whole ? BT : BT / cut;
    n0 = n_tile * 256 + (int)rank * 128;
    m0 = m_tile * BT + (whole ? 0 : first % cut * width);
  };
  int count = rounds;
  if (rounds * step + first / cut < tiles_n * tiles_m) {
    int n0, m0, width;
    locate(rounds, n0, m0, width);
    if (m0 < p.M) ++count;  // (a part may lie wholly beyond the last token)
  }

  if (warp == 0) {
    const bool leader = ptx::elect_one();
    int slot = 0;
    uint32_t phase = 0;
    bool live = true;
    int skip = blockIdx.x == 0 ? p.skip_load : 0;
    for (int i = 0; i < count && live; ++i) {
      int n0, m0, width;
      locate(i, n0, m0, width);
      m0 += (int)rank * (width / 2);
      const CUtensorMap* tokens = width == BT ? &tmT : &tmPart;
      const uint32_t tx = 2 * (C::W_BYTES + (uint32_t)width / 2 * 128);
#pragma unroll 1
      for (int s = 0; s < p.stages; ++s) {
        if (!wait_parity(empty_bar(slot), phase ^ 1u, stop, p.status, p.wait_cycles, 1)) { live = false; break; }
        if (leader && !(skip > 0 && --skip == 0)) {
          const uint32_t sbase = base + slot * C::STAGE_BYTES;
          const uint32_t fb = ptx::map_to_cta(full_bar(slot), 0);
          if (rank == 0) ptx::mbar_expect_tx(full_bar(slot), tx);
          ptx::tma_load_2d_pair(sbase, &tmW, s * 128, n0, fb);
          ptx::tma_load_2d_pair(sbase + C::W_BYTES, tokens, s * 128, m0, fb);
        }
        if (++slot == C::STAGES) { slot = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = ptx::elect_one();
      int slot = 0;
      uint32_t phase = 0;
      bool live = true;
      for (int i = 0; i < count && live; ++i) {
        const int acc = i & 1;
        if (!wait_parity_cluster(tempty_bar(acc), (((uint32_t)i >> 1) & 1u) ^ 1u, stop, p.status, p.wait_cycles, 4)) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + (uint32_t)acc * BT;
        const uint32_t idesc = i < rounds ? kIdescI8<256, BT> : cut == 1 ? kIdescI8<256, BT> : cut == 2 ? kIdescI8<256, BT / 2> : kIdescI8<256, BT / 4>;
        uint32_t accumulate = 0;
#pragma unroll 1
        for (int s = 0; s < p.stages; ++s) {
          if (!wait_parity_cluster(full_bar(slot), phase, stop, p.status, p.wait_cycles, 2)) { live = false; break; }
          ptx::tc_fence_after();
          const uint32_t sbase = base + slot * C::STAGE_BYTES;
          const uint32_t w_lo = ptx::desc_lo(sbase), t_lo = ptx::desc_lo(sbase + C::W_BYTES);
          if (leader) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              ptx::mma_i8_pair(d, w_lo + j * 2, t_lo + j * 2, ptx::kDescHiSw128, idesc, accumulate);
              accumulate = 1;
            }
            ptx::tc_commit_pair(empty_bar(slot), 3);  // frees the stage in both CTAs
          }
          if (++slot == C::STAGES) { slot = 0; phase ^= 1u; }
        }
        if (leader && live) ptx::tc_commit_pair(tfull_bar(acc), 3);
      }
    }
  } else {
    const int quad = warp & 3;  // tensor-memory lanes this warp may read
    const uint32_t my_scales = scales + (uint32_t)(warp - 2) * (C::COLS * 4);
    float* g_scales = reinterpret_cast<float*>(gbase + (my_scales - base));
    for (int i = 0; i < count; ++i) {
      int n0, m0, width;
      locate(i, n0, m0, width);
      const int c0 = ((warp - 2) >> 2) * (width / C::SIDE);  // this warp's tokens of the tile
      m0 += c0;
      const int acc = i & 1;
      const Channel<T> chan(p, n0 + quad * 32 + lane, m0);
      stage_scales<C::COLS>(g_scales, p, m0, lane);
      const bool store = wait_parity(tfull_bar(acc), ((uint32_t)i >> 1) & 1u, stop, p.status, p.wait_cycles, 8) &&
                         chan.real && !*stop;
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BT + c0);
      const int left = min(p.M - m0, width / C::SIDE);
      if (left <= 0) {  // none of this warp's tokens is real
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(tempty_bar(acc), 0));
      }
#pragma unroll 1
      for (int c = 0; c < left; c += 64) {
        uint32_t r[2][32];
        ptx::tmem_ld_32x32(taddr + c, r[0]);
        ptx::tmem_ld_32x32(taddr + c + 32, r[1]);
        ptx::tmem_ld_wait();
        if (c + 64 >= left) {  // the accumulator is in registers: hand it back
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(tempty_bar(acc), 0));
        }
        if (store) {
          finish<32>(reinterpret_cast<const int*>(r[0]), my_scales, c, left - c, chan, p.ldd);
          finish<32>(reinterpret_cast<const int*>(r[1]), my_scales, c + 32, left - c - 32, chan, p.ldd);
        }
      }
      __syncwarp();  // the scales have been read
    }
  }

  ptx::tc_fence_before();
  // A CTA that gave up tells its peer (which is still here: it cannot pass the barrier below before
  // this CTA arrives), so that both take the same path through the second barrier.
  __syncthreads();
  if (threadIdx.x == 0 && *stop) ptx::st_cluster_u32(ptx::map_to_cta(ptx::smem_u32(const_cast<int*>(stop)), rank ^ 1u), 1u);
  ptx::cluster_sync();
  ptx::tc_fence_after();
  if (*stop) {
    // give copies and MMAs that are still in flight time to land before either CTA goes away
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    ptx::cluster_sync();
  }
  if (warp == 1) ptx::tmem_dealloc_pair(tmem, 2 * BT);
}

// How the tiles of a problem are dealt out to `most` clusters.
struct PairPlan {
  int clusters, rounds, cut;
};
PairPlan plan_pair(double tiles, int most) {
  PairPlan pl;
  pl.rounds = (int)(tiles / most);
  const int rest = (int)(tiles - (double)pl.rounds * most);
  pl.cut = rest == 0 || rest * 2 > most ? 1 : rest * 4 > most ? 2 : 4;
  pl.clusters = pl.rounds > 0 ? most : rest * pl.cut;
  return pl;
}

template <typename T>
int launch_pair(const Int8Params& p, const int8_t* A, size_t lda, int K, const CUtensorMap& w, const mg::DeviceInfo& di,
                cudaStream_t st) {
  using C = PairCfg;
  auto kern = int8_gemm_pair_kernel<T>;
  static std::atomic<unsigned long long> allowed;
  MG_CUDA_TRY(mg::allow_smem(kern, C::SMEM, di.device, allowed));
  const PairPlan pl = plan_pair(std::ceil(p.N / 256.0) * std::ceil(p.M / (double)C::BT), di.sm_count / 2);
  CUtensorMap t, part;
  int rc;
  if ((rc = mg::make_map(&t, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, K, p.M, lda, 128, C::BT / 2))) return rc;
  if ((rc = mg::make_map(&part, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, K, p.M, lda, 128, C::BT / 2 / pl.cut))) return rc;
  MG_CUDA_TRY(mg::launch_kernel(kern, dim3(pl.clusters * 2), dim3(C::THREADS), C::SMEM, st, p, pl.rounds, pl.cut, w, t, part));
  return MG_OK;
}

template <int BT, typename T>
int launch_small(const Int8Params& p, const CUtensorMap& w, const CUtensorMap& t, int splits, const mg::DeviceInfo& di,
                 cudaStream_t st) {
  using C = SmallCfg<BT>;
  auto kern = int8_gemm_kernel<BT, T>;
  const int ring = C::ring(splits);
  const size_t smem = C::smem(splits, ring);
  static std::atomic<unsigned long long> allowed;
  MG_CUDA_TRY(mg::allow_smem(kern, kSmemLimit, di.device, allowed));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + kRows - 1) / kRows, (p.M + BT - 1) / BT, splits);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = splits;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = mg::pdl_enabled() ? 2 : 1;
  MG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, ring, w, t));
  return MG_OK;
}

// How many clusters of `splits` such CTAs the device holds at one time (asked once per device and shape;
// 0 where it holds none).
template <int BT, typename T>
int small_capacity(int splits, const mg::DeviceInfo& di) {
  if (splits == 1) return di.sm_count;
  static std::atomic<int> known[64][3];
  std::atomic<int>& slot = known[di.device][splits == 2 ? 0 : splits == 4 ? 1 : 2];
  int k = slot.load();
  if (k == 0) {
    using C = SmallCfg<BT>;
    auto kern = int8_gemm_kernel<BT, T>;
    int n = 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, 1, splits);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::smem(splits, C::ring(splits));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = splits;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool ok = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess && n >= 1;
    if (!ok) (void)cudaGetLastError();  // the question is allowed to fail; the answer is then "none"
    k = ok ? n : -1;
    slot.store(k);
  }
  return k > 0 ? k : 0;
}

// Which form takes the problem: the one with the least of
//   T = fixed + wave * waves + sqrt(compute^2 + bytes^2)   in us,
// compute = waves * 128-byte slices of K of a CTA * stage (a part of a tile in the pair form's last round: kCutStage;
// a stage of the small form that is half empty, an odd slice at 32 or 64 tokens, counts as one slice, in the fit too),
// bytes = those of the operands and the result / 6.5 MB per us, waves = tiles / (clusters that run at one time).
// The constants are fitted to 137 problems (8 to 2048 tokens, N and K = 1024, 4096, 14336, and 32 to 8192 tokens
// with K = 128 and 512; bf16 results, cold weights) run with every form: over them the choice is 0.4 % slower than
// the best form on average and 14 % at most.  What they say: a stage of the pair form runs at the tensor cores'
// rate (0.29 us for 256 x 256 x 128), one of the small form at the rate of its loads and barriers; a pair costs two
// microseconds more to set up, every further wave one or two; adding sums across a cluster costs 1.4 us.  For
// example 2048 x 4096 x 4096: pair 25 us, small 128 39; 256 x 4096 x 4096: pair 10.9, small 64 8.5;
// 64 x 4096 x 4096: small 64 with four splits 7.3, one split 8.2; 128 x 4096 x 14336: small 128 with four splits
// 15.6, two 19.6.
struct FormCost {
  double fixed, wave, stage;
};
constexpr FormCost kPair = {3.26, 0.99, 0.286};
constexpr double kCutStage[5] = {0, kPair.stage, 0.186, 0, 0.169};  // of a tile in one, two, four parts
constexpr FormCost kSmall32 = {1.26, 1.08, 0.145}, kSmall64 = {1.14, 1.41, 0.169}, kSmall128 = {1.09, 1.98, 0.225};
constexpr double kSplitCost = 1.44, kBytesPerUs = 6.5e6;

struct Form {
  bool pair;
  int tokens, splits;
};

template <typename T>
Form choose_form(int M, int N, int K, const mg::DeviceInfo& di, const mg::Options& opt) {
  const int sms = di.sm_count;
  const double stages = (K + 127) / 128;
  const double bytes = ((double)N * K + (double)M * K + (double)sizeof(T) * M * N) / kBytesPerUs;
  Form best = {true, 0, 1};
  double least = 1e300;
  auto offer = [&](const Form& f, const FormCost& c, double tiles, int capacity, double extra) {
    const double waves = std::ceil(tiles / capacity), compute = waves * std::ceil(stages / f.splits) * c.stage;
    const double t = c.fixed + extra + waves * c.wave + std::sqrt(compute * compute + bytes * bytes);
    if (t < least) {
      least = t;
      best = f;
    }
  };
  auto tiles = [&](int channels, int tokens) { return std::ceil((double)N / channels) * std::ceil((double)M / tokens); };
  if (opt.int8_pair != 0) {
    const double all = tiles(256, 256);
    const PairPlan pl = plan_pair(all, sms / 2);
    const bool rest = (double)pl.rounds * pl.clusters < all;
    const double compute = stages * (pl.rounds * kPair.stage + (rest ? kCutStage[pl.cut] : 0));
    least = kPair.fixed + (pl.rounds + rest) * kPair.wave + std::sqrt(compute * compute + bytes * bytes);
  }
  if (opt.int8_pair <= 0) {
    const double most_splits = std::ceil(stages / 2);  // (a stage may hold two slices)
    for (int splits = 1; splits <= kMaxSplit && splits <= most_splits; splits *= 2) {
      if (opt.int8_split > 0 && opt.int8_split != splits && !(opt.int8_split > splits && splits * 2 > most_splits)) continue;
      for (int tokens = 32; tokens <= 128; tokens *= 2) {
        if (opt.int8_tokens > 0 && opt.int8_tokens != tokens) continue;
        if ((double)M / tokens > 65535) continue;  // (the grid's second dimension)
        const int capacity = tokens == 32   ? small_capacity<32, T>(splits, di)
                             : tokens == 64 ? small_capacity<64, T>(splits, di)
                                            : small_capacity<128, T>(splits, di);
        if (capacity < 1) continue;
        const FormCost& c = tokens == 32 ? kSmall32 : tokens == 64 ? kSmall64 : kSmall128;
        offer({false, tokens, splits}, c, tiles(kRows, tokens), capacity, splits > 1 ? kSplitCost : 0);
      }
    }
  }
  return best;
}

template <typename T>
int launch_int8(const Int8Params& p, const int8_t* A, size_t lda, const int8_t* B, size_t ldb, int K,
                const mg::DeviceInfo& di, cudaStream_t st) {
  const mg::Options opt = mg::options();
  if (opt.int8_few != 0 && p.M <= kFewTokens)
    return p.M == 1 ? launch_few<1, T>(p, A, lda, B, ldb, K, di.sm_count, st) : launch_few<2, T>(p, A, lda, B, ldb, K, di.sm_count, st);
  const Form f = choose_form<T>(p.M, p.N, K, di, opt);
  CUtensorMap w, t;
  int rc;
  if ((rc = mg::make_map(&w, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, K, p.N, ldb, 128, 128))) return rc;
  if (f.pair) return launch_pair<T>(p, A, lda, K, w, di, st);
  if ((rc = mg::make_map(&t, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, K, p.M, lda, 128, f.tokens))) return rc;
  if (f.tokens == 32) return launch_small<32, T>(p, w, t, f.splits, di, st);
  if (f.tokens == 64) return launch_small<64, T>(p, w, t, f.splits, di, st);
  return launch_small<128, T>(p, w, t, f.splits, di, st);
}

}  // namespace

extern "C" int mg_matmul_int8(const int8_t* A, size_t lda, const int8_t* B, size_t ldb, const float* scale_a,
                              const float* scale_b, const float* bias, int M, int N, int K, void* D, int dtype,
                              size_t ldd, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || K > MG_INT8_MAX_K || dtype < 0 || dtype > 2) return MG_ERR_SHAPE;
  if (M > kMostRows || N > kMostRows) return MG_ERR_SHAPE;
  // one row has no pitch: any value stands for the smallest that a tensor map takes
  const size_t dense = ((size_t)K + 15) / 16 * 16;
  if (M <= 1) lda = dense;
  if (N <= 1) ldb = dense;
  if (M <= 1) ldd = (size_t)N;
  if (lda < (size_t)K || ldb < (size_t)K || ldd < (size_t)N) return MG_ERR_SHAPE;
  if (lda % 16 || ldb % 16) return MG_ERR_ALIGN;
  if (lda >= (1ull << 40) || ldb >= (1ull << 40)) return MG_ERR_SHAPE;
  if (M == 0 || N == 0) return MG_OK;
  if (!A || !B || !scale_a || !scale_b || !D) return MG_ERR_NULL;
  if (!mg::aligned(A, 16) || !mg::aligned(B, 16) || !mg::aligned(scale_a, 4) || !mg::aligned(scale_b, 4) ||
      !mg::aligned(bias, 4) || !mg::aligned(D, dtype == MG_FP32 ? 4 : 2))
    return MG_ERR_ALIGN;
  const size_t e = dtype == MG_FP32 ? 4 : 2;
  if (mg::any_overlap({mg::Span(D, (size_t)M, (size_t)N * e, ldd * e)},
                      {mg::Span(A, (size_t)M, (size_t)K, lda), mg::Span(B, (size_t)N, (size_t)K, ldb), mg::Span(scale_a, (size_t)M * 4),
                       mg::Span(scale_b, (size_t)N * 4), mg::Span(bias, (size_t)N * 4)}))
    return MG_ERR_OVERLAP;
  mg::DeviceInfo di;
  int rc = mg::device_info(&di);
  if (rc != MG_OK) return rc;
  Int8Params p{};
  p.M = M;
  p.N = N;
  p.stages = (K + 127) / 128;
  p.sa = scale_a;
  p.sb = scale_b;
  p.bias = bias;
  p.D = D;
  p.ldd = ldd;
  p.wait_cycles = mg::wait_limit_cycles();
  p.skip_load = mg::options().fault_skip_load;
  if ((rc = mg::device_status_word(&p.status)) != MG_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MG_BF16) return launch_int8<__nv_bfloat16>(p, A, lda, B, ldb, K, di, st);
  if (dtype == MG_FP16) return launch_int8<__half>(p, A, lda, B, ldb, K, di, st);
  return launch_int8<float>(p, A, lda, B, ldb, K, di, st);
}
