// Layer norm for B200 (sm_100a): y = n w + b with n = (x - mean) rstd, rstd = (var + eps)^(-1/2)
// over the last dimension; forward, and backward with the weight's and bias's gradients:
//   dx = rstd (dy w - mean(dy w) - n mean(dy w n)),  dw = sum_rows dy n,  db = sum_rows dy.
//
// Both directions read every activation once: a row lives in the registers of one warp, or of one
// CTA where it is wider, as NV vectors of VEC elements a thread (16 bytes where width, strides and
// bases allow it, else single elements). The statistics are exact two-step ones: each warp's mean,
// then its squared deviations about that mean, joined over the warps with one barrier by
//   mean = sum n_i mean_i / n,  M = sum M_i + n_i (mean_i - mean)^2,
// so no sum of squares about zero cancels. CTAs walk the rows; in the backward a thread keeps the
// sums of dw and db of its own columns in registers, each CTA writes one row of partial sums, and
// a second kernel adds those rows in a fixed order (bitwise reproducible). Rows wider than the
// registers hold go to kernels that read them again from cache.
#include <algorithm>

#include "common.cuh"
#include "sparc_b200.h"
#include "timing.cuh"

namespace sparc {

struct LnParams {
  const void* x;
  const void* dy;     // backward
  void* out;          // y, or dx
  const float* w;
  const float* b;     // forward: or null
  float* mean;        // [R] (forward: out or null)
  float* rstd;
  float* part;        // backward: [gridDim.x, 2, W] partial sums of dw and db
  long long R, sx, sdy;  // rows; row strides in elements (out is dense)
  int W;
  float eps;
};

// ---------------------------------------------------------------- vectors of VEC elements
template <typename T, int VEC> struct LnVec;
template <> struct LnVec<float, 1> {
  using type = float;
  static __device__ __forceinline__ void get(float v, float* f) { f[0] = v; }
  static __device__ __forceinline__ float make(const float* f) { return f[0]; }
};
template <> struct LnVec<float, 4> {
  using type = float4;
  static __device__ __forceinline__ void get(float4 v, float* f) { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
  static __device__ __forceinline__ float4 make(const float* f) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct LnVec<__nv_bfloat16, 1> {
  using type = unsigned short;
  static __device__ __forceinline__ void get(unsigned short v, float* f) { f[0] = __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned short make(const float* f) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
  }
};
template <> struct LnVec<__nv_bfloat16, 8> {
  using type = uint4;
  static __device__ __forceinline__ void pair(unsigned v, float* f) {
    f[0] = __uint_as_float(v << 16), f[1] = __uint_as_float(v & 0xffff0000u);
  }
  static __device__ __forceinline__ unsigned pack(const float* f) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const unsigned*>(&v);
  }
  static __device__ __forceinline__ void get(uint4 v, float* f) {
    pair(v.x, f), pair(v.y, f + 2), pair(v.z, f + 4), pair(v.w, f + 6);
  }
  static __device__ __forceinline__ uint4 make(const float* f) {
    return make_uint4(pack(f), pack(f + 2), pack(f + 4), pack(f + 6));
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Threads per row = 32 WARPS; with WARPS == 1 a CTA's kLnRows warps take a row each.
constexpr int kLnRows = 8;
template <int WARPS> constexpr int kLnThreads = WARPS == 1 ? 32 * kLnRows : 32 * WARPS;

// Column of element e of vector j of thread i of a row: (j * 32 * WARPS + i) * VEC + e.
template <typename T, int VEC, int NV, int WARPS>
__global__ void __launch_bounds__(kLnThreads<WARPS>) ln_fwd_kernel(const LnParams p) {
  using V = LnVec<T, VEC>;
  __shared__ float2 s_stat[2][WARPS];
  const int i = WARPS == 1 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long first = WARPS == 1 ? (long long)blockIdx.x * kLnRows + wp : blockIdx.x;
  const long long step = WARPS == 1 ? (long long)gridDim.x * kLnRows : gridDim.x;
  const float inv_w = 1.0f / (float)p.W;
  // this warp's elements of a row
  int count = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c0 = (j * 32 * WARPS + (i - lane)) * VEC;
    count += max(0, min(32 * VEC, p.W - c0));
  }
  const float inv_count = count > 0 ? 1.0f / (float)count : 0.0f;
  int par = 0;
  for (long long r = first; r < p.R; r += step, par ^= 1) {
    float x[NV][VEC];
    float sum = 0.0f;
    typename V::type raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
      if (c < p.W) raw[j] = __ldg(reinterpret_cast<const typename V::type*>(static_cast<const T*>(p.x) + r * p.sx + c));
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
      V::get(raw[j], x[j]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += c < p.W ? x[j][e] : 0.0f;
    }
    float mean = warp_sum(sum) * inv_count, m2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = x[j][e] - mean;
        m2 += c < p.W ? d * d : 0.0f;
      }
    }
    m2 = warp_sum(m2);
    if constexpr (WARPS > 1) {
      if (lane == 0) s_stat[par][wp] = make_float2(mean, m2);
      __syncthreads();
      float all = 0.0f;
      m2 = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) n += max(0, min(32 * VEC, p.W - (j * 32 * WARPS + k * 32) * VEC));
        all = fmaf((float)n, s_stat[par][k].x, all);
      }
      mean = all * inv_w;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) n += max(0, min(32 * VEC, p.W - (j * 32 * WARPS + k * 32) * VEC));
        const float d = s_stat[par][k].x - mean;
        m2 += n > 0 ? fmaf((float)n * d, d, s_stat[par][k].y) : 0.0f;
      }
    }
    const float rstd = 1.0f / sqrtf(fmaf(m2, inv_w, p.eps));
    if (i == 0 && p.mean != nullptr) p.mean[r] = mean, p.rstd[r] = rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
      if (c < p.W) {
        float y[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float n = (x[j][e] - mean) * rstd;
          y[e] = p.b != nullptr ? fmaf(n, __ldg(p.w + c + e), __ldg(p.b + c + e)) : n * __ldg(p.w + c + e);
        }
        *reinterpret_cast<typename V::type*>(static_cast<T*>(p.out) + r * p.W + c) = V::make(y);
      }
    }
  }
}

template <typename T, int VEC, int NV, int WARPS>
__global__ void __launch_bounds__(kLnThreads<WARPS>) ln_bwd_kernel(const LnParams p) {
  using V = LnVec<T, VEC>;
  constexpr int E = NV * VEC;
  __shared__ float2 s_sum[2][WARPS];
  extern __shared__ float s_part[];  // WARPS == 1: [kLnRows][2][W]
  const int i = WARPS == 1 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long first = WARPS == 1 ? (long long)blockIdx.x * kLnRows + wp : blockIdx.x;
  const long long step = WARPS == 1 ? (long long)gridDim.x * kLnRows : gridDim.x;
  const float inv_w = 1.0f / (float)p.W;
  float w[E], dw[E], db[E];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * 32 * WARPS + i) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[j * VEC + e] = c < p.W ? __ldg(p.w + c + e) : 0.0f;
      dw[j * VEC + e] = db[j * VEC + e] = 0.0f;
    }
  }
  int par = 0;
  for (long long r = first; r < p.R; r += step, par ^= 1) {
    typename V::type rx[NV], rd[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
      if (c < p.W) {
        rx[j] = __ldg(reinterpret_cast<const typename V::type*>(static_cast<const T*>(p.x) + r * p.sx + c));
        rd[j] = __ldg(reinterpret_cast<const typename V::type*>(static_cast<const T*>(p.dy) + r * p.sdy + c));
      }
    }
    const float mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
    float n[E], d[E], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool on = (j * 32 * WARPS + i) * VEC < p.W;
      V::get(rx[j], n + j * VEC);
      V::get(rd[j], d + j * VEC);
#pragma unroll
      for (int k = j * VEC; k < (j + 1) * VEC; ++k) {
        n[k] = on ? (n[k] - mean) * rstd : 0.0f;
        d[k] = on ? d[k] : 0.0f;
        dw[k] = fmaf(d[k], n[k], dw[k]);
        db[k] += d[k];
        d[k] *= w[k];
        s1 += d[k];
        s2 = fmaf(d[k], n[k], s2);
      }
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (WARPS > 1) {
      if (lane == 0) s_sum[par][wp] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) s1 += s_sum[par][k].x, s2 += s_sum[par][k].y;
    }
    s1 *= inv_w;
    s2 *= inv_w;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
      if (c < p.W) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = rstd * (d[j * VEC + e] - s1 - n[j * VEC + e] * s2);
        *reinterpret_cast<typename V::type*>(static_cast<T*>(p.out) + r * p.W + c) = V::make(o);
      }
    }
  }
  if (p.part == nullptr) return;
  float* part = p.part + (long long)blockIdx.x * 2 * p.W;
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * WARPS + i) * VEC;
      if (c < p.W) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[c + e] = dw[j * VEC + e], part[p.W + c + e] = db[j * VEC + e];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 + lane) * VEC;
      if (c < p.W) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s_part[wp * 2 * p.W + c + e] = dw[j * VEC + e];
          s_part[wp * 2 * p.W + p.W + c + e] = db[j * VEC + e];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.W; c += kLnThreads<WARPS>) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kLnRows; ++k) s += s_part[k * 2 * p.W + c];
      part[c] = s;
    }
  }
}

// Rows wider than the registers hold: one CTA per row, three passes (mean, deviations, output),
// the later ones from cache.
constexpr int kLnWide = 1024;

__device__ __forceinline__ float block_sum(float v, float* s) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int k = 0; k < kLnWide / 32; ++k) v += s[k];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kLnWide) ln_wide_fwd_kernel(const LnParams p) {
  __shared__ float s[kLnWide / 32];
  const float inv_w = 1.0f / (float)p.W;
  for (long long r = blockIdx.x; r < p.R; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.sx;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < p.W; c += kLnWide) sum += Io<T>::load(x + c);
    float mean = block_sum(sum, s) * inv_w;
    float m2 = 0.0f, m1 = 0.0f;
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float d = Io<T>::load(x + c) - mean;
      m1 += d;
      m2 = fmaf(d, d, m2);
    }
    // the deviations' own mean is what rounding left of the mean
    const float off = block_sum(m1, s) * inv_w;
    const float var = block_sum(m2, s) * inv_w - off * off, rstd = 1.0f / sqrtf(var + p.eps);
    mean += off;
    if (threadIdx.x == 0 && p.mean != nullptr) p.mean[r] = mean, p.rstd[r] = rstd;
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float n = (Io<T>::load(x + c) - mean) * rstd;
      Io<T>::store(static_cast<T*>(p.out) + r * p.W + c, p.b != nullptr ? fmaf(n, p.w[c], p.b[c]) : n * p.w[c]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLnWide) ln_wide_bwd_kernel(const LnParams p) {
  __shared__ float s[kLnWide / 32];
  const float inv_w = 1.0f / (float)p.W;
  for (long long r = blockIdx.x; r < p.R; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.sx;
    const T* dy = static_cast<const T*>(p.dy) + r * p.sdy;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float d = Io<T>::load(dy + c) * p.w[c];
      s1 += d;
      s2 = fmaf(d, (Io<T>::load(x + c) - mean) * rstd, s2);
    }
    s1 = block_sum(s1, s) * inv_w;
    s2 = block_sum(s2, s) * inv_w;
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float n = (Io<T>::load(x + c) - mean) * rstd;
      Io<T>::store(static_cast<T*>(p.out) + r * p.W + c, rstd * (Io<T>::load(dy + c) * p.w[c] - s1 - n * s2));
    }
  }
}

// Partial sums of dw and db over a span of rows per CTA row, a thread per column.
template <typename T>
__global__ void __launch_bounds__(256) ln_wide_cols_kernel(const LnParams p) {
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= p.W) return;
  float dw = 0.0f, db = 0.0f;
  for (long long r = blockIdx.x; r < p.R; r += gridDim.x) {
    const float d = Io<T>::load(static_cast<const T*>(p.dy) + r * p.sdy + c);
    dw = fmaf(d, (Io<T>::load(static_cast<const T*>(p.x) + r * p.sx + c) - p.mean[r]) * p.rstd[r], dw);
    db += d;
  }
  p.part[(long long)blockIdx.x * 2 * p.W + c] = dw;
  p.part[(long long)blockIdx.x * 2 * p.W + p.W + c] = db;
}

// dw, db from the partial rows: a block owns 32 of the 2 W columns, its warps every 8th row, in
// float64 and in order.
__global__ void __launch_bounds__(256) ln_reduce_kernel(const float* part, float* dw, float* db, int rows, int W) {
  __shared__ double s[8][32];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  double t = 0.0;
  if (c < 2LL * W)
    for (int r = wp; r < rows; r += 8) t += (double)part[(long long)r * 2 * W + c];
  s[wp][lane] = t;
  __syncthreads();
  if (wp == 0 && c < 2LL * W) {
    for (int k = 1; k < 8; ++k) t += s[k][lane];
    if (c < W) {
      if (dw != nullptr) dw[c] = (float)t;
    } else if (db != nullptr) {
      db[c - W] = (float)t;
    }
  }
}

// ---------------------------------------------------------------- host
constexpr int kLnMaxGrid = 148 * 8;  // the most CTAs that walk the rows, and rows of partial sums

struct LnPlan {
  int vec, nv, warps;  // warps == 0: the wide kernels
};

// The narrowest of the instances that holds a row; vectors where `vectors` (16-byte aligned rows).
static LnPlan ln_plan(int W, bool vectors, int size) {
  const int vec = vectors ? 16 / size : 1;
  const int small = vec == 8 ? 1 : vec == 4 ? 2 : 4, big = vec == 8 ? 2 : vec == 4 ? 4 : 16;
  for (int warps : {1, 4, 8, 16})
    for (int nv : {small, big})
      if ((long long)32 * warps * vec * nv >= W) return LnPlan{vec, nv, warps};
  return LnPlan{1, 0, 0};
}

static int ln_rows_per_cta(const LnPlan& pl) { return pl.warps == 1 ? kLnRows : 1; }

static int ln_grid(long long R, const LnPlan& pl) {
  const int per = ln_rows_per_cta(pl);
  return (int)std::min<long long>((R + per - 1) / per, kLnMaxGrid);
}

static int ln_check_shape(long long R, long long W) {
  if (R <= 0 || W <= 0) return fail(SPARC_ERR_SHAPE, "rows and width must be positive");
  if (W > (1LL << 24) || R > (1LL << 40) || (double)R * (double)W > 4.0e18)
    return fail(SPARC_ERR_SHAPE, "shape beyond the launch grid (width <= 2^24)");
  return SPARC_OK;
}

static size_t ln_ws_bytes(long long R, long long W) {
  return (size_t)std::min<long long>(R, kLnMaxGrid) * 2 * (size_t)W * sizeof(float);
}

template <typename T, int VEC, int NV, int WARPS>
static cudaError_t ln_launch(const LnParams& p, int grid, bool backward, cudaStream_t s) {
  TimedLaunch tl(backward ? kTimeLnBwd : kTimeLnFwd, s);
  if (backward) {
    const size_t smem = WARPS == 1 ? (size_t)kLnRows * 2 * p.W * sizeof(float) : 0;
    ln_bwd_kernel<T, VEC, NV, WARPS><<<grid, kLnThreads<WARPS>, smem, s>>>(p);
  } else {
    ln_fwd_kernel<T, VEC, NV, WARPS><<<grid, kLnThreads<WARPS>, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename T, int VEC, int NV>
static cudaError_t ln_warps(const LnParams& p, const LnPlan& pl, int grid, bool backward, cudaStream_t s) {
  switch (pl.warps) {
    case 1: return ln_launch<T, VEC, NV, 1>(p, grid, backward, s);
    case 4: return ln_launch<T, VEC, NV, 4>(p, grid, backward, s);
    case 8: return ln_launch<T, VEC, NV, 8>(p, grid, backward, s);
    default: return ln_launch<T, VEC, NV, 16>(p, grid, backward, s);
  }
}

template <typename T>
static cudaError_t ln_dispatch(const LnParams& p, const LnPlan& pl, bool backward, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int grid = ln_grid(p.R, pl);
  if (pl.warps == 0) {
    TimedLaunch tl(backward ? kTimeLnBwd : kTimeLnFwd, s);
    if (!backward) {
      ln_wide_fwd_kernel<T><<<grid, kLnWide, 0, s>>>(p);
    } else {
      ln_wide_bwd_kernel<T><<<grid, kLnWide, 0, s>>>(p);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
      if (p.part != nullptr) ln_wide_cols_kernel<T><<<dim3(grid, (p.W + 255) / 256), 256, 0, s>>>(p);
    }
    return cudaGetLastError();
  }
  if (pl.vec == 1) {
    return pl.nv == 4 ? ln_warps<T, 1, 4>(p, pl, grid, backward, s) : ln_warps<T, 1, 16>(p, pl, grid, backward, s);
  }
  if constexpr (V == 8) {
    return pl.nv == 1 ? ln_warps<T, 8, 1>(p, pl, grid, backward, s) : ln_warps<T, 8, 2>(p, pl, grid, backward, s);
  } else {
    return pl.nv == 2 ? ln_warps<T, 4, 2>(p, pl, grid, backward, s) : ln_warps<T, 4, 4>(p, pl, grid, backward, s);
  }
}

static bool ln_aligned(const void* q, long long stride, long long R, int size) {
  return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (R <= 1 || (stride * size) % 16 == 0);
}

}  // namespace sparc

using namespace sparc;

extern "C" {

size_t sparc_layer_norm_workspace_bytes(long long rows, long long width) {
  if (ln_check_shape(rows, width) != SPARC_OK) return 0;
  return ln_ws_bytes(rows, width);
}

int sparc_layer_norm_forward(const SparcLayerNormFwdArgs* a, void* stream) {
  NvtxRange nvtx(__func__);
  if (a == nullptr) return fail(SPARC_ERR_ARG, "null args");
  if (!a->x || !a->y || !a->weight) return fail(SPARC_ERR_ARG, "null tensor pointer");
  if ((a->mean == nullptr) != (a->rstd == nullptr)) return fail(SPARC_ERR_ARG, "mean and rstd go together");
  const int rc = ln_check_shape(a->rows, a->width);
  if (rc != SPARC_OK) return rc;
  if (a->dtype != SPARC_DTYPE_F32 && a->dtype != SPARC_DTYPE_BF16) return fail(SPARC_ERR_DTYPE, "unsupported dtype");
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  for (const void* q : {a->x, (const void*)a->y})
    if (reinterpret_cast<uintptr_t>(q) % size != 0) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
  LnParams p = {};
  p.x = a->x;
  p.out = a->y;
  p.w = a->weight;
  p.b = a->bias;
  p.mean = a->mean;
  p.rstd = a->rstd;
  p.R = a->rows;
  p.sx = a->x_row_stride;
  p.W = (int)a->width;
  p.eps = a->eps;
  const bool vectors = p.W * size % 16 == 0 && ln_aligned(a->x, p.sx, p.R, size) && ln_aligned(a->y, p.W, p.R, size);
  const LnPlan pl = ln_plan(p.W, vectors, size);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == SPARC_DTYPE_BF16 ? ln_dispatch<__nv_bfloat16>(p, pl, false, s)
                                                     : ln_dispatch<float>(p, pl, false, s);
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

int sparc_layer_norm_backward(const SparcLayerNormBwdArgs* a, void* stream) {
  NvtxRange nvtx(__func__);
  if (a == nullptr) return fail(SPARC_ERR_ARG, "null args");
  if (!a->x || !a->dy || !a->dx || !a->weight || !a->mean || !a->rstd) return fail(SPARC_ERR_ARG, "null tensor pointer");
  const int rc = ln_check_shape(a->rows, a->width);
  if (rc != SPARC_OK) return rc;
  if (a->dtype != SPARC_DTYPE_F32 && a->dtype != SPARC_DTYPE_BF16) return fail(SPARC_ERR_DTYPE, "unsupported dtype");
  const bool sums = a->grad_weight != nullptr || a->grad_bias != nullptr;
  if (sums && (a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 4 != 0 ||
               a->workspace_bytes < ln_ws_bytes(a->rows, a->width)))
    return fail(SPARC_ERR_WORKSPACE, "workspace missing, too small or not 4-byte aligned");
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  for (const void* q : {a->x, a->dy, (const void*)a->dx})
    if (reinterpret_cast<uintptr_t>(q) % size != 0) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
  LnParams p = {};
  p.x = a->x;
  p.dy = a->dy;
  p.out = a->dx;
  p.w = a->weight;
  p.mean = const_cast<float*>(a->mean);
  p.rstd = const_cast<float*>(a->rstd);
  p.part = sums ? static_cast<float*>(a->workspace) : nullptr;
  p.R = a->rows;
  p.sx = a->x_row_stride;
  p.sdy = a->dy_row_stride;
  p.W = (int)a->width;
  const bool vectors = p.W * size % 16 == 0 && ln_aligned(a->x, p.sx, p.R, size) &&
                       ln_aligned(a->dy, p.sdy, p.R, size) && ln_aligned(a->dx, p.W, p.R, size);
  const LnPlan pl = ln_plan(p.W, vectors, size);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = a->dtype == SPARC_DTYPE_BF16 ? ln_dispatch<__nv_bfloat16>(p, pl, true, s)
                                               : ln_dispatch<float>(p, pl, true, s);
  if (e == cudaSuccess && sums) {
    TimedLaunch tl(kTimeLnReduce, s);
    ln_reduce_kernel<<<(2 * p.W + 31) / 32, 256, 0, s>>>(p.part, a->grad_weight, a->grad_bias, ln_grid(p.R, pl), p.W);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

}  // extern "C"
