// Rows in 8 bits with one scale each: plain (quantize_int8) and behind a root-mean-square norm with
// the residual's addition (rms_norm_int8).
//
//   plain   a = max |x|                  s = a / 127            q = rint(x * (127 / a))
//   norm    u = T(x + r)                 v = rsqrt(sum u^2 / K + eps)
//           h = (u w) v                  then as above with h for x
//
// v is one factor for the whole row, so max |h| = v max |u w|: the sum of squares and the largest
// magnitude come out of the same pass, one reduction gives both, and the row is read once and kept
// in registers between the statistics and the codes.  Magnitudes are compared as integers (the sign
// bit cleared, fp32 order is integer order and NaN is above infinity), so a value that is not finite
// is seen; such a row, and one whose sum of squares leaves the fp32 range, gets the scale NaN and
// codes 0: a product with it is NaN in that row and in no other.  a counts as 2^-100 at least, which
// keeps 127 / a finite and gives a row of zeros the codes 0 and a small positive scale.
// Everything between the loads and the codes is fp32; u is rounded to T once, because it is the
// stream that later layers read.
//
// Bound: bytes.  2 + 1 per element plain in 16 bits, 6 + 1 with a residual; about ten instructions
// per element are needed, sixteen would fit under the copy bandwidth.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mg_common.h"
#include "ptx_sm100.cuh"

namespace {

constexpr float kTiny = 0x1p-100f;

// Most threads of a CTA whose threads hold `held` values in registers.
constexpr int max_threads(int held) { return held >= 64 ? 512 : 1024; }

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
  float eps;
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

// CH elements of one chunk <-> fp32.  Aligned chunks are whole 16-byte vectors; the others hold four
// elements that are moved one by one, those beyond `n` reading as zero.
template <typename T, bool ALIGNED, int CH>
__device__ __forceinline__ void load_chunk(const void* row, int e0, int n, float (&f)[CH]) {
  using Raw = typename Elem<T>::Raw;
  if constexpr (ALIGNED) {
    static_assert(CH * sizeof(Raw) == 16, "a chunk is one vector");
    union {
      uint4 v;
      Raw e[CH];
    } u;
    u.v = *reinterpret_cast<const uint4*>(static_cast<const Raw*>(row) + e0);
#pragma unroll
    for (int j = 0; j < CH; ++j) f[j] = Elem<T>::up(u.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < CH; ++j) f[j] = j < n ? Elem<T>::up(static_cast<const Raw*>(row)[e0 + j]) : 0.f;
  }
}

template <typename T, bool ALIGNED, int CH>
__device__ __forceinline__ void store_chunk(void* row, int e0, int n, const float (&f)[CH]) {
  using Raw = typename Elem<T>::Raw;
  if constexpr (ALIGNED) {
    union {
      uint4 v;
      Raw e[CH];
    } u;
#pragma unroll
    for (int j = 0; j < CH; ++j) u.e[j] = Elem<T>::down(f[j]);
    *reinterpret_cast<uint4*>(static_cast<Raw*>(row) + e0) = u.v;
  } else {
#pragma unroll
    for (int j = 0; j < CH; ++j)
      if (j < n) static_cast<Raw*>(row)[e0 + j] = Elem<T>::down(f[j]);
  }
}

// rint(fl(p * f)) of four values as the four bytes of a word: adding 1.5 * 2^23 leaves the integer,
// rounded to nearest even, in the low mantissa bits.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float f) {
  const float kMagic = 12582912.0f;
  const uint32_t ia = __float_as_uint(__fadd_rn(__fmul_rn(a, f), kMagic));
  const uint32_t ib = __float_as_uint(__fadd_rn(__fmul_rn(b, f), kMagic));
  const uint32_t ic = __float_as_uint(__fadd_rn(__fmul_rn(c, f), kMagic));
  const uint32_t id = __float_as_uint(__fadd_rn(__fmul_rn(d, f), kMagic));
  return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}

template <bool ALIGNED, int CH>
__device__ __forceinline__ void store_codes(int8_t* q, int n, const float (&p)[CH], float f, bool bad) {
  uint32_t w[CH / 4];
#pragma unroll
  for (int j = 0; j < CH / 4; ++j)
    w[j] = bad ? 0u : codes4(p[j * 4], p[j * 4 + 1], p[j * 4 + 2], p[j * 4 + 3], f);
  if constexpr (CH == 8) {
    *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  } else {
    if (ALIGNED || (n >= 4 && (reinterpret_cast<uintptr_t>(q) & 3) == 0)) {
      *reinterpret_cast<uint32_t*>(q) = w[0];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) q[j] = (int8_t)(w[0] >> (8 * j));
    }
  }
}

// Sum and integer maximum over the threads of a row: blockDim.x lanes, one or more whole warps.
__device__ __forceinline__ void reduce_row(float& sum, uint32_t& top, int warps, float* s_sum, uint32_t* s_top) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    s_sum[warp] = sum;
    s_top[warp] = top;
  }
  __syncthreads();
  sum = lane < warps ? s_sum[lane] : 0.f;
  top = lane < warps ? s_top[lane] : 0u;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
}

// One row for blockDim.x threads (blockDim.y rows per CTA when a row is one warp's).  CPT chunks per
// thread stay in registers; CPT = 0 is the form for rows that do not fit, which reads them twice.
template <typename T, bool ALIGNED>
constexpr int kChunk = ALIGNED ? 16 / (int)sizeof(typename Elem<T>::Raw) : 4;

template <typename T, bool NORM, bool ALIGNED, int CPT>
__global__ void __launch_bounds__(max_threads(CPT * kChunk<T, ALIGNED>)) row_quant_kernel(const RowQuantParams p) {
  constexpr int CH = kChunk<T, ALIGNED>;
  using Raw = typename Elem<T>::Raw;
  __shared__ float s_sum[32];
  __shared__ uint32_t s_top[32];
  ptx::grid_dep_launch_dependents();
  ptx::grid_dep_wait();
  const int row = (int)(blockIdx.x * blockDim.y + threadIdx.y);
  if (row >= p.M) return;  // whole warps; with several warps to a row blockDim.y is 1
  const int K = p.K, nt = blockDim.x, warps = nt >> 5;
  const Raw* x = static_cast<const Raw*>(p.X) + (size_t)row * p.px;
  const Raw* r = p.R ? static_cast<const Raw*>(p.R) + (size_t)row * p.pr : nullptr;
  Raw* u = p.R ? static_cast<Raw*>(p.U) + (size_t)row * p.pu : nullptr;
  int8_t* q = p.Q + (size_t)row * p.pq;
  const int chunks = (K + CH - 1) / CH;

  float sum = 0.f;
  uint32_t top = 0;
  // one chunk: read, add, keep u w (or x) in f, and count it in
  auto take = [&](int c, float (&f)[CH], bool count) {
    const int e0 = c * CH, n = K - e0;
    load_chunk<T, ALIGNED, CH>(x, e0, n, f);
    if constexpr (NORM) {
      if (r) {
        float g[CH];
        load_chunk<T, ALIGNED, CH>(r, e0, n, g);
#pragma unroll
        for (int j = 0; j < CH; ++j) f[j] = Elem<T>::up(Elem<T>::down(f[j] + g[j]));
        if (!count || CPT > 0) store_chunk<T, ALIGNED, CH>(u, e0, n, f);
      }
      float w[CH];
      load_chunk<T, ALIGNED, CH>(p.W, e0, n, w);
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        if (count) sum = fmaf(f[j], f[j], sum);
        f[j] *= w[j];
      }
    }
    if (count) {
#pragma unroll
      for (int j = 0; j < CH; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
    }
  };

  float keep[CPT > 0 ? CPT : 1][CH];
  if constexpr (CPT > 0) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = i * nt + (int)threadIdx.x;
      if (c < chunks) take(c, keep[i], true);
    }
  } else {
    for (int c = threadIdx.x; c < chunks; c += nt) take(c, keep[0], true);
  }
  reduce_row(sum, top, warps, s_sum, s_top);

  float v = 1.f, a = __uint_as_float(top);
  bool bad = top >= 0x7f800000u;
  if constexpr (NORM) {
    bad = bad || !(sum <= 3.4028235e38f);
    v = rsqrtf(sum / (float)K + p.eps);
    a *= v;
    bad = bad || !(a <= 3.4028235e38f);
  }
  a = fmaxf(a, kTiny);
  const float f = v * (127.0f / a);
  if (threadIdx.x == 0) p.S[row] = bad ? __uint_as_float(0x7fc00000u) : a / 127.0f;
  if constexpr (CPT > 0) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = i * nt + (int)threadIdx.x;
      if (c < chunks) store_codes<ALIGNED, CH>(q + c * CH, K - c * CH, keep[i], f, bad);
    }
  } else {
    for (int c = threadIdx.x; c < chunks; c += nt) {
      take(c, keep[0], false);
      store_codes<ALIGNED, CH>(q + c * CH, K - c * CH, keep[0], f, bad);
    }
  }
}

template <typename T, bool NORM, bool ALIGNED>
int launch_rows(const RowQuantParams& p, int sms, cudaStream_t st) {
  constexpr int CH = kChunk<T, ALIGNED>;
  const int chunks = (p.K + CH - 1) / CH;
  int cpt, nt, rows = 1;
  if (chunks <= 128 && p.M > 1) {  // a warp to a row, four rows to a CTA
    cpt = chunks <= 64 ? 2 : 4;
    nt = 32;
    rows = 4;
  } else {
    // few rows want many threads (latency), many rows want many chunks in flight per thread
    const int most = p.M <= sms ? 1024 : 256;
    cpt = 2;
    while (cpt < 8 && (chunks + cpt - 1) / cpt > most) cpt *= 2;
    nt = ((chunks + cpt - 1) / cpt + 31) / 32 * 32;
    if (nt > max_threads(cpt * CH)) {
      nt = 1024;
      cpt = 0;
    }
  }
  auto kern = cpt == 0   ? row_quant_kernel<T, NORM, ALIGNED, 0>
              : cpt == 2 ? row_quant_kernel<T, NORM, ALIGNED, 2>
              : cpt == 4 ? row_quant_kernel<T, NORM, ALIGNED, 4>
                         : row_quant_kernel<T, NORM, ALIGNED, 8>;
  MG_CUDA_TRY(mg::launch_kernel(kern, dim3((p.M + rows - 1) / rows), dim3(nt, rows), 0, st, p));
  return MG_OK;
}

// dtype: 0 bf16, 1 fp16, 2 fp32 (MG_BF16, MG_FP16, MG_FP32)
template <bool NORM>
int row_quant(const RowQuantParams& p, int dtype, void* stream) {
  if (p.M < 0 || p.K <= 0 || p.K > MG_INT8_MAX_K || dtype < 0 || dtype > 2) return MG_ERR_SHAPE;
  if (NORM && !(p.eps >= 0.f && p.eps <= 3.4028235e38f)) return MG_ERR_SHAPE;
  if (p.M > 1 && (p.px < (size_t)p.K || p.pq < (size_t)p.K)) return MG_ERR_SHAPE;
  if (p.M > 1 && p.R && (p.pr < (size_t)p.K || p.pu < (size_t)p.K)) return MG_ERR_SHAPE;
  if (p.M == 0) return MG_OK;
  if (!p.X || !p.Q || !p.S || (NORM && !p.W) || (p.R != nullptr) != (p.U != nullptr)) return MG_ERR_NULL;
  const size_t e = dtype == 2 ? 4 : 2;
  if (!mg::aligned(p.X, e) || !mg::aligned(p.S, 4) || (NORM && !mg::aligned(p.W, e)) || !mg::aligned(p.R, e) ||
      !mg::aligned(p.U, e))
    return MG_ERR_ALIGN;
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
  if (dtype == MG_BF16)
    return vec ? launch_rows<__nv_bfloat16, NORM, true>(p, di.sm_count, st)
               : launch_rows<__nv_bfloat16, NORM, false>(p, di.sm_count, st);
  if (dtype == MG_FP16)
    return vec ? launch_rows<__half, NORM, true>(p, di.sm_count, st) : launch_rows<__half, NORM, false>(p, di.sm_count, st);
  return vec ? launch_rows<float, NORM, true>(p, di.sm_count, st) : launch_rows<float, NORM, false>(p, di.sm_count, st);
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
  return row_quant<true>(p, dtype, stream);
}
