// Rows in 8 bits with one scale each: plain (quantize_int8) and behind a root-mean-square norm with
// the residual's addition (rms_norm_int8).
//
//   plain   a = max |x|                  s = a / 127            q = rint(x * (127 / a))
//   norm    u = T(x + r)                 v = rsqrt(sum u^2 / K + eps)
//           h = (u w) v                  then as above with h for x
//
// v is one factor for the whole row, so max |h| = v max |u w|: the sum of squares and the largest
// magnitude come out of the same pass, one reduction gives both, and the row is read once and kept
// in registers between the statistics and the codes.  The maximum is one that hands NaN on, so a value
// that is not finite is seen; such a row, and one whose sum of squares leaves the fp32 range, gets the
// scale NaN and codes 0: a product with it is NaN in that row and in no other.  a counts as 2^-100 at
// least, which keeps 127 / a finite and gives a row of zeros the codes 0 and a small positive scale.
// Everything between the loads and the codes is fp32; u is rounded to T once, because it is the
// stream that later layers read.
//
// Bound: bytes, 2 + 1 per element plain in 16 bits, 6 + 1 with a residual.  14336 x 4096 bf16: plain 29.4 us
// (6.0 TB/s), with norm and residual 63.8 us (6.5 TB/s), norm alone 34.0 us (5.2 TB/s: one CTA to an SM, whose
// reduction shows).  A call has a fixed part beside its bytes: 4096 elements take 2.6 us plus 1.86 us per 1000 rows
// plain (6.6 TB/s) and 2.9 plus 2.20 behind a norm (5.6 TB/s), so 2048 rows take 6.8 and 7.1.  Rows without 16-byte
// alignment are moved element by element: 4096 x 1931 8.5 us plain (2.8 TB/s), 17.3 us with norm and residual
// (3.2 TB/s).  Aligned 16-bit rows beyond 16384 elements are read twice: 2048 x 28672 plain 55.5 us (bytes 27).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "mg_common.h"
#include "overlap.h"
#include "ptx_sm100.cuh"

namespace {

constexpr float kTiny = 0x1p-100f;
constexpr float kMaxFloat = 3.4028235e38f;

struct RowQuantParams {
  const void* X;
  const void* R;  // residual, or null
  void* U;        // x + r rounded to T (with R only)
  const void* W;  // norm weight
  int8_t* Q;
  float* S;
  int M, K;
  size_t px, pr, pu;  // row pitches in elements of T
  size_t pq;          // row pitch of the codes in bytes
  float eps, inv_k;
};

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float up(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t down(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
  using Raw = uint16_t;
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float up(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ uint16_t down(float f) { return __half_as_ushort(__float2half_rn(f)); }
  using Raw = uint16_t;
};
template <>
struct Elem<float> {
  static __device__ __forceinline__ float up(uint32_t v) { return __uint_as_float(v); }
  static __device__ __forceinline__ uint32_t down(float f) { return __float_as_uint(f); }
  using Raw = uint32_t;
};

template <typename T, bool ALIGNED>
constexpr int kChunk = ALIGNED ? 16 / (int)sizeof(typename Elem<T>::Raw) : 4;

// A chunk of a row as it lies in memory: a whole 16-byte vector, or four elements that are moved one by
// one.  `n` elements are left in the row: what lies beyond reads as zero and is not written, so that the
// arithmetic in between needs no branches.
template <typename T, bool ALIGNED>
struct Chunk {
  using Raw = typename Elem<T>::Raw;
  static constexpr int CH = kChunk<T, ALIGNED>;
  union {
    uint4 v;
    Raw e[16 / sizeof(Raw)];
  };

  __device__ __forceinline__ void load(const Raw* row, int e0, int n) {
    if constexpr (ALIGNED) {
      v = make_uint4(0, 0, 0, 0);
      if (n > 0) v = *reinterpret_cast<const uint4*>(row + e0);
    } else {
#pragma unroll
      for (int j = 0; j < CH; ++j) e[j] = j < n ? row[e0 + j] : (Raw)0;
    }
  }
  __device__ __forceinline__ void load_const(const Raw* row, int e0, int n) {  // not written by this grid (see ptx::ldg_v4)
    if constexpr (ALIGNED) {
      v = make_uint4(0, 0, 0, 0);
      if (n > 0) v = ptx::ldg_v4(row + e0);
    } else {
#pragma unroll
      for (int j = 0; j < CH; ++j) e[j] = j < n ? ptx::ldg(row + e0 + j) : (Raw)0;
    }
  }
  __device__ __forceinline__ void store(Raw* row, int e0, int n) const {
    if constexpr (ALIGNED) {
      if (n > 0) *reinterpret_cast<uint4*>(row + e0) = v;
    } else {
#pragma unroll
      for (int j = 0; j < CH; ++j)
        if (j < n) row[e0 + j] = e[j];
    }
  }
  __device__ __forceinline__ float at(int j) const { return Elem<T>::up(e[j]); }
  __device__ __forceinline__ void add(const Chunk& r) {  // the one rounding of the stream
#pragma unroll
    for (int j = 0; j < CH; ++j) e[j] = Elem<T>::down(at(j) + r.at(j));
  }
};

// The code of p f in the low byte: adding 1.5 * 2^23 leaves the integer, rounded to nearest even, in the low
// mantissa bits.  The plain form rounds the product first, which is its definition; behind a norm p f
// is not more exact than that rounding, and one instruction does both.
template <bool NORM>
__device__ __forceinline__ uint32_t code(float p, float f) {
  const float kMagic = 12582912.0f;
  return __float_as_uint(NORM ? __fmaf_rn(p, f, kMagic) : __fadd_rn(__fmul_rn(p, f), kMagic));
}
template <bool NORM>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float f) {
  return __byte_perm(__byte_perm(code<NORM>(a, f), code<NORM>(b, f), 0x0040),
                     __byte_perm(code<NORM>(c, f), code<NORM>(d, f), 0x0040), 0x5410);
}

// max(top, |a|, |b|), NaN when one of them is.
__device__ __forceinline__ float max_abs(float top, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <bool NORM, bool ALIGNED, int CH>
__device__ __forceinline__ void store_codes(int8_t* q, int n, const float (&p)[CH], float f, bool bad) {
  uint32_t w[CH / 4];
#pragma unroll
  for (int j = 0; j < CH / 4; ++j)
    w[j] = bad ? 0u : codes4<NORM>(p[j * 4], p[j * 4 + 1], p[j * 4 + 2], p[j * 4 + 3], f);
  if constexpr (CH == 8) {
    if (n > 0) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  } else if constexpr (ALIGNED) {
    if (n > 0) *reinterpret_cast<uint32_t*>(q) = w[0];
  } else {
    if (n >= 4 && (reinterpret_cast<uintptr_t>(q) & 3) == 0) {
      *reinterpret_cast<uint32_t*>(q) = w[0];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) q[j] = (int8_t)(w[0] >> (8 * j));
    }
  }
}

// Sum and maximum over the threads of a row: blockDim.x lanes, one or more whole warps.  The
// caller alternates between two sets of shared words, so that one barrier per row is enough.
struct RowShared {
  float2 part[32];
};

__device__ __forceinline__ void reduce_row(float& sum, float& top, int warps, RowShared& sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh.part[warp] = make_float2(sum, top);
  __syncthreads();
  const float2 part = lane < warps ? sh.part[lane] : make_float2(0.f, 0.f);
  sum = part.x;
  top = part.y;
  int o = 1;
  for (; o < warps; o *= 2) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (o < 32) {  // the other lanes hold the sums of nothing
    sum = __shfl_sync(0xffffffffu, sum, 0);
    top = __shfl_sync(0xffffffffu, top, 0);
  }
}

// What a row's statistics make of it: codes = rint(u w f), scale = a / 127.
struct RowScale {
  float f, a;
  bool bad;
};

template <bool NORM>
__device__ __forceinline__ RowScale row_scale(float sum, float top, const RowQuantParams& p) {
  float v = 1.f, a = top;
  bool bad = !(top <= kMaxFloat);
  if constexpr (NORM) {
    bad = bad || !(sum <= kMaxFloat);
    v = rsqrtf(fmaf(sum, p.inv_k, p.eps));
    a *= v;
    bad = bad || !(a <= kMaxFloat);
  }
  a = fmaxf(a, kTiny);
  return {fminf(v * (127.0f / a), kMaxFloat), a, bad};  // (finite, so that 0 stays 0 under a floor that is far away)
}

// Persistent: blockDim.x threads take a row at a time (blockDim.y rows side by side in a CTA when a row is
// one warp's).  A thread's CPT chunks stay in registers from the statistics to the codes, and the next row's
// are on their way while the row is reduced.
// CPT = 0 is the form for rows that do not fit: it reads them twice.
// Plain rows of four chunks a thread run two CTAs to an SM: 8192 x 16384 62 us, with one 74.  That leaves 64 registers;
// the 16-bit aligned form is 12 bytes over, which costs 1 % at 14336 x 4096.
constexpr int max_threads(int cpt) { return cpt >= 4 ? 512 : 1024; }  // (registers)

// MODE: plain, norm, or norm behind the residual's addition
enum { kPlain = 0, kNorm = 1, kNormAdd = 2 };

template <typename T, int MODE, bool ALIGNED, int CPT>
__global__ void __launch_bounds__(max_threads(CPT), MODE == kPlain && CPT == 4 ? 2 : 1) row_quant_kernel(const RowQuantParams p) {
  constexpr bool NORM = MODE != kPlain, ADD = MODE == kNormAdd;
  constexpr bool RAW = !NORM && ALIGNED;  // a plain row is kept as it lies in memory: half the registers
  // The norm's weight is loaded wherever that suits the compiler, but in the order of the source where a thread
  // holds 32 elements and a weight loaded early takes registers that they need (fp32 with a residual 4141 x 15768
  // 203 us, in order 151; fp32 unaligned 2856 x 10477 57 and 48; bf16 aligned 8192 x 16384 with a residual 143.7 and
  // 141.9, 16 x 14336 without 2.57 and 2.46).  The other way round: fp32 aligned without a residual (4141 x 15768 55,
  // in order 78) and 16-bit unaligned rows (2856 x 10477 with a residual 88 and 107).
  constexpr bool kWeightInOrder =
      CPT * Chunk<T, ALIGNED>::CH >= 32 && (sizeof(typename Chunk<T, ALIGNED>::Raw) == 4 ? ADD || !ALIGNED : ALIGNED);
  using Ck = Chunk<T, ALIGNED>;
  using Raw = typename Ck::Raw;
  constexpr int CH = Ck::CH;
  __shared__ RowShared sh[2];
  ptx::grid_dep_launch_dependents();
  ptx::grid_dep_wait();
  const int K = p.K, nt = blockDim.x, warps = nt >> 5, chunks = (K + CH - 1) / CH;
  const unsigned rows = (unsigned)p.M, step = gridDim.x * blockDim.y;
  const Raw* W = ptx::written_before(static_cast<const Raw*>(p.W));
  auto x_row = [&](unsigned row) { return static_cast<const Raw*>(p.X) + (size_t)row * p.px; };
  auto r_row = [&](unsigned row) { return static_cast<const Raw*>(p.R) + (size_t)row * p.pr; };
  auto u_row = [&](unsigned row) { return static_cast<Raw*>(p.U) + (size_t)row * p.pu; };

  // u w (or x) of a chunk in fp32, counted into the statistics when asked for
  float sum, top;
  auto values = [&](const Ck& c, int i, bool count, float (&f)[CH]) {
    if constexpr (NORM) {
      Ck w;
      if constexpr (kWeightInOrder) w.load(W, i * CH, K - i * CH);
      else w.load_const(W, i * CH, K - i * CH);
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        const float u = c.at(j);
        if (count) sum = fmaf(u, u, sum);
        f[j] = u * w.at(j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < CH; ++j) f[j] = c.at(j);
    }
    if (count) {
#pragma unroll
      for (int j = 0; j < CH; j += 2) top = max_abs(top, f[j], f[j + 1]);
    }
  };

  unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  if constexpr (CPT > 0) {
    Ck next[CPT], next_r[ADD ? CPT : 1];
    auto fetch = [&](unsigned at) {
      const Raw* x = x_row(at);
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        const int e0 = (i * nt + (int)threadIdx.x) * CH;
        next[i].load(x, e0, K - e0);
      }
      if constexpr (ADD) {
        const Raw* r = r_row(at);
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          const int e0 = (i * nt + (int)threadIdx.x) * CH;
          next_r[i].load(r, e0, K - e0);
        }
      }
    };
    if (row < rows) fetch(row);
    for (int turn = 0; row < rows; row += step, turn ^= 1) {
      Ck cur[RAW ? CPT : 1];
      float f[RAW ? 1 : CPT][CH];
      sum = top = 0.f;
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        const int c = i * nt + (int)threadIdx.x;
        if constexpr (ADD) {
          next[i].add(next_r[i]);
          next[i].store(u_row(row), c * CH, K - c * CH);
        }
        if constexpr (RAW) cur[i] = next[i];
        values(next[i], c, true, f[RAW ? 0 : i]);
      }
      if (row + step < rows) fetch(row + step);
      reduce_row(sum, top, warps, sh[turn]);
      const RowScale rs = row_scale<NORM>(sum, top, p);
      if (threadIdx.x == 0) p.S[row] = rs.bad ? __uint_as_float(0x7fc00000u) : rs.a / 127.0f;
      int8_t* q = p.Q + (size_t)row * p.pq;
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        const int c = i * nt + (int)threadIdx.x;
        if constexpr (RAW) values(cur[i], c, false, f[0]);
        store_codes<NORM, ALIGNED, CH>(q + c * CH, K - c * CH, f[RAW ? 0 : i], rs.f, rs.bad);
      }
    }
  } else {
    for (int turn = 0; row < rows; row += step, turn ^= 1) {
      const Raw* x = x_row(row);
      auto take = [&](int c) {
        Ck v;
        v.load(x, c * CH, K - c * CH);
        if constexpr (ADD) {
          Ck r;
          r.load(r_row(row), c * CH, K - c * CH);
          v.add(r);
        }
        return v;
      };
      sum = top = 0.f;
      float f[CH];
      for (int c = threadIdx.x; c < chunks; c += nt) values(take(c), c, true, f);
      reduce_row(sum, top, warps, sh[turn]);
      const RowScale rs = row_scale<NORM>(sum, top, p);
      if (threadIdx.x == 0) p.S[row] = rs.bad ? __uint_as_float(0x7fc00000u) : rs.a / 127.0f;
      int8_t* q = p.Q + (size_t)row * p.pq;
      for (int c = threadIdx.x; c < chunks; c += nt) {
        const Ck v = take(c);  // (U may be X or R: every thread writes what it alone reads, after its last read)
        if constexpr (ADD) v.store(u_row(row), c * CH, K - c * CH);
        values(v, c, false, f);
        store_codes<NORM, ALIGNED, CH>(q + c * CH, K - c * CH, f, rs.f, rs.bad);
      }
    }
  }
}

// CTAs of `nt` threads of this kernel that an SM holds (asked once per device and size).
template <typename T, int MODE, bool ALIGNED, int CPT>
int resident(int nt, int device) {
  static std::atomic<int> known[64][33];
  std::atomic<int>& slot = known[device][nt / 32];
  int k = slot.load(std::memory_order_relaxed);
  if (k == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&k, row_quant_kernel<T, MODE, ALIGNED, CPT>, nt, 0) != cudaSuccess || k < 1) {
      (void)cudaGetLastError();
      k = 1;
    }
    slot.store(k, std::memory_order_relaxed);
  }
  return k;
}

template <typename T, int MODE, bool ALIGNED, int CPT>
int launch_form(const RowQuantParams& p, int nt, int side, const mg::DeviceInfo& di, cudaStream_t st) {
  const unsigned ctas = ((unsigned)p.M + side - 1) / side;
  const unsigned most = (unsigned)di.sm_count * resident<T, MODE, ALIGNED, CPT>(nt * side, di.device);
  MG_CUDA_TRY(mg::launch_kernel(row_quant_kernel<T, MODE, ALIGNED, CPT>, dim3(ctas < most ? ctas : most), dim3(nt, side), 0, st, p));
  return MG_OK;
}

template <typename T, int MODE, bool ALIGNED>
int launch_rows(const RowQuantParams& p, const mg::DeviceInfo& di, cudaStream_t st) {
  const int chunks = (p.K + kChunk<T, ALIGNED> - 1) / kChunk<T, ALIGNED>;
  auto threads = [&](int cpt) { return ((chunks + cpt - 1) / cpt + 31) / 32 * 32; };
  // A warp to a row, four rows to a CTA, when two chunks per thread hold one; few rows want many threads
  // (latency: 64 x 4096 1.7 us with one chunk per thread, 1.8 with two), many rows many bytes in flight per
  // thread (14336 x 4096: 28.4 us with four, 36.5 with two, 44 with one, 61 read twice).
  if (chunks <= 64 && p.M > di.sm_count) return launch_form<T, MODE, ALIGNED, 2>(p, 32, 4, di, st);
  if (p.M <= 2 * di.sm_count && threads(1) <= 1024) return launch_form<T, MODE, ALIGNED, 1>(p, threads(1), 1, di, st);
  if (threads(4) <= 512) return launch_form<T, MODE, ALIGNED, 4>(p, threads(4), 1, di, st);
  // Eight chunks of four elements (2856 x 10477 bf16 plain 28.7 us, read twice 65; 4141 x 15768 fp32 51, 115), also
  // where the registers fall a little short (16-bit unaligned with a residual, 32 to 40 bytes spilled: 2856 x 10477
  // 88 us, read twice 110; fp32 aligned with one, 16 bytes: 4141 x 15768 151), but not for fp32 without alignment and
  // with a residual (2856 x 10477: 201 us, read twice 146).
  if constexpr (kChunk<T, ALIGNED> == 4 && (ALIGNED || MODE != kNormAdd || sizeof(typename Elem<T>::Raw) == 2)) {
    if (threads(8) <= 512) return launch_form<T, MODE, ALIGNED, 8>(p, threads(8), 1, di, st);
  }
  return launch_form<T, MODE, ALIGNED, 0>(p, 1024, 1, di, st);
}

template <typename T, bool NORM>
int launch_type(const RowQuantParams& p, bool vec, const mg::DeviceInfo& di, cudaStream_t st) {
  if constexpr (NORM) {
    if (p.R) return vec ? launch_rows<T, kNormAdd, true>(p, di, st) : launch_rows<T, kNormAdd, false>(p, di, st);
    return vec ? launch_rows<T, kNorm, true>(p, di, st) : launch_rows<T, kNorm, false>(p, di, st);
  } else {
    return vec ? launch_rows<T, kPlain, true>(p, di, st) : launch_rows<T, kPlain, false>(p, di, st);
  }
}

// dtype: 0 bf16, 1 fp16, 2 fp32 (MG_BF16, MG_FP16, MG_FP32)
template <bool NORM>
int row_quant(const RowQuantParams& p, int dtype, void* stream) {
  if (p.M < 0 || p.K <= 0 || p.K > MG_INT8_MAX_K || dtype < 0 || dtype > 2) return MG_ERR_SHAPE;
  if (NORM && !(p.eps >= 0.f && p.eps <= kMaxFloat)) return MG_ERR_SHAPE;
  if (p.M > 1 && (p.px < (size_t)p.K || p.pq < (size_t)p.K)) return MG_ERR_SHAPE;
  if (p.M > 1 && p.R && (p.pr < (size_t)p.K || p.pu < (size_t)p.K)) return MG_ERR_SHAPE;
  if (p.M == 0) return MG_OK;
  if (!p.X || !p.Q || !p.S || (NORM && !p.W) || (p.R != nullptr) != (p.U != nullptr)) return MG_ERR_NULL;
  const size_t e = dtype == 2 ? 4 : 2;
  if (!mg::aligned(p.X, e) || !mg::aligned(p.S, 4) || (NORM && !mg::aligned(p.W, e)) || !mg::aligned(p.R, e) ||
      !mg::aligned(p.U, e))
    return MG_ERR_ALIGN;
  // a row's codes and scale are written while other rows, and in the form that reads twice its own, are still read
  const size_t M = (size_t)p.M, bytes = (size_t)p.K * e;
  const mg::Span x(p.X, M, bytes, p.px * e), r(p.R, M, bytes, p.pr * e), u(p.U, M, bytes, p.pu * e), w(NORM ? p.W : nullptr, bytes);
  if (mg::any_overlap({mg::Span(p.Q, M, (size_t)p.K, p.pq), mg::Span(p.S, M * 4)}, {x, r, w, u})) return MG_ERR_OVERLAP;
  if (p.U && (mg::overlap(u, w) || (mg::overlap(u, x) && !mg::same(u, x)) || (mg::overlap(u, r) && !mg::same(u, r))))
    return MG_ERR_OVERLAP;
  mg::DeviceInfo di;
  const int rc = mg::device_info(&di);
  if (rc != MG_OK) return rc;
  // the vector form: every row of every tensor starts on a 16-byte boundary (codes: on a chunk's)
  const size_t ch = 16 / e;
  const bool one = p.M == 1;
  bool vec = p.K % ch == 0 && mg::aligned(p.X, 16) && (one || p.px % ch == 0) && mg::aligned(p.Q, ch) &&
             (one || p.pq % ch == 0);
  if (NORM) {
    vec = vec && mg::aligned(p.W, 16);
    if (p.R) vec = vec && mg::aligned(p.R, 16) && mg::aligned(p.U, 16) && (one || (p.pr % ch == 0 && p.pu % ch == 0));
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MG_BF16) return launch_type<__nv_bfloat16, NORM>(p, vec, di, st);
  if (dtype == MG_FP16) return launch_type<__half, NORM>(p, vec, di, st);
  return launch_type<float, NORM>(p, vec, di, st);
}

}  // namespace

extern "C" int mg_quantize_int8(const void* X, int dtype, int M, int K, size_t ldx, int8_t* Q, size_t ldq, float* scale,
                                void* stream) {
  RowQuantParams p{};
  p.X = X;
  p.Q = Q;
  p.S = scale;
  p.M = M;
  p.K = K;
  p.px = ldx;
  p.pq = ldq;
  return row_quant<false>(p, dtype, stream);
}

extern "C" int mg_rms_norm_int8(const void* X, const void* R, const void* W, float eps, int dtype, int M, int K,
                                size_t ldx, size_t ldr, void* U, size_t ldu, int8_t* Q, size_t ldq, float* scale,
                                void* stream) {
  RowQuantParams p{};
  p.X = X;
  p.R = R;
  p.U = U;
  p.W = W;
  p.Q = Q;
  p.S = scale;
  p.M = M;
  p.K = K;
  p.px = ldx;
  p.pr = ldr;
  p.pu = ldu;
  p.pq = ldq;
  p.eps = eps;
  p.inv_k = 1.0f / (float)K;
  return row_quant<true>(p, dtype, stream);
}
