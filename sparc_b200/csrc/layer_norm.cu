// Layer norm for B200 (sm_100a): y = n w + b with n = (x - mean) rstd, rstd = (var + eps)^(-1/2)
// over the last dimension; forward, and backward with the weight's and bias's gradients:
//   dx = rstd (dy w - mean(dy w) - n mean(dy w n)),  dw = sum_rows dy n,  db = sum_rows dy.
//
// Both directions read every activation once: a row lives in the registers of one warp, or of one
// CTA where it is wider, as NV vectors of VEC elements a thread (16 bytes where width, strides and
// bases allow it, else pairs, else single elements). CTAs walk the rows and keep the next few on the way into
// shared memory by asynchronous copies (two rows in registers leave HBM a third idle): of 16-byte
// vectors each thread copies and waits for its own; rows that begin anywhere come in the aligned
// 16-byte pieces that hold them, and every thread takes its elements once all pieces are there. The
// statistics take two steps: each warp's mean,
// then its squared deviations about that mean, joined over the warps with one barrier by
//   mean = sum n_i mean_i / n,  M = sum M_i + n_i (mean_i - mean)^2,
// so no sum of squares about zero cancels. (The mean keeps its own sum's rounding, which the wide kernels
// take out: at 16384 x 512 float32 y is 6e-8 from 64 bits, the weight's gradient 9e-8.) In the backward
// a thread keeps the sums of dw and db of its own columns in registers, each CTA writes one row of partial sums, and
// a second kernel adds those rows in a fixed order (bitwise reproducible). Rows wider than the
// registers hold go to kernels that read them again from cache.
//
// Measured on a B200 (131072 x 2048 bfloat16): forward 190 us = 5.6 TB/s (86% of what a copy reaches),
// backward 284 us = 5.7 TB/s (86%) and 5 us of reduction; bound by HBM, and by a row's chain of
// reductions where rows are narrow or not 16-byte aligned (138996 x 1374: 212 us = 3.6 TB/s). 16384 x 512
// float32: 13, 17 and 4 us, of floors 10 and 15.
#include <algorithm>
#include <initializer_list>

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
template <> struct LnVec<float, 2> {
  using type = float2;
  static __device__ __forceinline__ void get(float2 v, float* f) { f[0] = v.x, f[1] = v.y; }
  static __device__ __forceinline__ float2 make(const float* f) { return make_float2(f[0], f[1]); }
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
template <> struct LnVec<__nv_bfloat16, 2> {
  using type = unsigned;
  static __device__ __forceinline__ void get(unsigned v, float* f) {
    f[0] = __uint_as_float(v << 16), f[1] = __uint_as_float(v & 0xffff0000u);
  }
  static __device__ __forceinline__ unsigned make(const float* f) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const unsigned*>(&v);
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
constexpr int kLnHeld = 16;  // a thread's columns whose parameters it holds in registers
template <int WARPS> constexpr int kLnThreads = WARPS == 1 ? 32 * kLnRows : 32 * WARPS;

// A thread's share of a row: element e of its vector j is column (j * 32 WARPS + i) VEC + e, i the
// thread's number among the row's.
template <typename T, int VEC, int NV, int WARPS>
struct LnRow {
  using V = LnVec<T, VEC>;
  static constexpr int kStep = 32 * WARPS * VEC;  // columns from a vector to the next
  // `f` <- the row's values, zeros beyond it
  static __device__ __forceinline__ void get(const typename V::type (&raw)[NV], int c0, int W, float (&f)[NV * VEC]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      V::get(raw[j], f + j * VEC);
      if (c0 + j * kStep >= W) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[j * VEC + e] = 0.0f;
      }
    }
  }
  static __device__ __forceinline__ void put(void* base, long long row, int c0, int W, const float (&f)[NV * VEC]) {
    T* q = static_cast<T*>(base) + row + c0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * kStep < W) *reinterpret_cast<typename V::type*>(q + j * kStep) = V::make(f + j * VEC);
  }
  // float32 parameters of the same columns (zeros beyond the row, or where there are none)
  static __device__ __forceinline__ void params(const float* w, int c0, int W, float (&f)[NV * VEC]) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = c0 + j * kStep + e;
        f[j * VEC + e] = w != nullptr && c < W ? __ldg(w + c) : 0.0f;
      }
  }
};

// The next rows of NT tensors on their way into shared memory, slot by slot: up to kLnRing of them, as
// far as kLnRingBytes a CTA go. Rows are asked for in order, one for each that is taken.
constexpr int kLnRing = 4, kLnRingBytes = 96 * 1024;
template <typename T, int VEC, int NV, int WARPS, int NT>
struct LnAhead {
  using Row = LnRow<T, VEC, NV, WARPS>;
  using R = typename LnVec<T, VEC>::type;
  static constexpr bool kVectors = VEC * sizeof(T) == 16;
  static constexpr int kRows = WARPS == 1 ? kLnRows : 1;  // of a CTA at a time
  // of one tensor's row in a slot: the threads' vectors, or the row with the rest of its outer pieces
  static constexpr int kTensorBytes = 32 * WARPS * NV * VEC * (int)sizeof(T) + (kVectors ? 0 : 16);
  static constexpr int kSlotBytes = NT * kTensorBytes;
  static constexpr int kDepth = std::min(kLnRing, kLnRingBytes / (kSlotBytes * kRows));
  static constexpr int kBytes = kDepth * kSlotBytes * kRows;
  static_assert(kDepth >= 1);
  unsigned char* mine;  // [slot][tensor], of this thread's row
  int i, slot;          // the thread's number among the row's; the slot asked for next

  __device__ __forceinline__ explicit LnAhead(unsigned char* ring)
      : mine(ring + (WARPS == 1 ? (threadIdx.x >> 5) * kDepth * kSlotBytes : 0)),
        i(WARPS == 1 ? (int)(threadIdx.x & 31) : (int)threadIdx.x), slot(0) {}

  // tensor n's row at `q`
  __device__ __forceinline__ void ask(int n, const T* q, int W) {
    unsigned char* to = mine + slot * kSlotBytes + n * kTensorBytes;
    if constexpr (kVectors) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (i * VEC + j * Row::kStep < W) copy(to + (j * 32 * WARPS + i) * 16, q + i * VEC + j * Row::kStep);
    } else {
      const char* a = reinterpret_cast<const char*>(q);
      const int off = (int)(reinterpret_cast<unsigned long long>(a) & 15u), end = off + W * (int)sizeof(T);
      for (int at = i * 16; at < end; at += 32 * WARPS * 16) copy(to + at, a - off + at);
    }
  }
  static __device__ __forceinline__ void copy(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(from) : "memory");
  }
  __device__ __forceinline__ void asked() {  // the row's tensors are complete
    asm volatile("cp.async.commit_group;" ::: "memory");
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  }
  // with kDepth rows asked for and not taken, the first of them has come (its slot is the next one asked for)
  __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    if constexpr (!kVectors) {
      if constexpr (WARPS == 1) __syncwarp();
      else __syncthreads();
    }
  }
  __device__ __forceinline__ void take(int n, const T* q, int W, float (&f)[NV * VEC]) {
    const unsigned char* from = mine + slot * kSlotBytes + n * kTensorBytes;
    if constexpr (kVectors) {
      R v[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) v[j] = reinterpret_cast<const R*>(from)[j * 32 * WARPS + i];
      Row::get(v, i * VEC, W, f);
    } else {
      const R* e = reinterpret_cast<const R*>(from + (reinterpret_cast<unsigned long long>(q) & 15u)) + i;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if ((j * 32 * WARPS + i) * VEC < W) {
          LnVec<T, VEC>::get(e[j * 32 * WARPS], f + j * VEC);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) f[j * VEC + k] = 0.0f;
        }
      }
    }
  }
  // Between a row's last take and the next ask, which writes its slot: every thread has taken it. (With
  // several warps a row, the barrier of the row's sums stands between the two.)
  __device__ __forceinline__ void taken() {
    if constexpr (!kVectors && WARPS == 1) __syncwarp();
  }
};

// Elements of a row that warp k of its WARPS holds.
template <int VEC, int NV, int WARPS>
__device__ __forceinline__ int ln_count(int k, int W) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) n += max(0, min(32 * VEC, W - (j * 32 * WARPS + k * 32) * VEC));
  return n;
}

template <typename T, int VEC, int NV, int WARPS>
__global__ void __launch_bounds__(kLnThreads<WARPS>) ln_fwd_kernel(const LnParams p) {
  using Row = LnRow<T, VEC, NV, WARPS>;
  constexpr int E = NV * VEC;
  __shared__ float4 s_stat[2][WARPS];  // mean, squared deviations, count
  const int i = WARPS == 1 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31, c0 = i * VEC;
  const long long first = WARPS == 1 ? (long long)blockIdx.x * kLnRows + wp : blockIdx.x;
  const long long step = WARPS == 1 ? (long long)gridDim.x * kLnRows : gridDim.x;
  const float inv_w = 1.0f / (float)p.W;
  const float count = (float)ln_count<VEC, NV, WARPS>(WARPS == 1 ? 0 : wp, p.W);
  const float inv_count = count > 0.0f ? 1.0f / count : 0.0f;
  extern __shared__ __align__(16) unsigned char s_ring[];
  using Ahead = LnAhead<T, VEC, NV, WARPS, 1>;
  Ahead ahead(s_ring);
  auto ask = [&](long long r) {
    if (r < p.R) ahead.ask(0, static_cast<const T*>(p.x) + r * p.sx, p.W);
    ahead.asked();
  };
#pragma unroll
  for (int k = 0; k < Ahead::kDepth; ++k) ask(first + k * step);
  constexpr bool kHeld = E <= kLnHeld;  // the parameters of the thread's columns in registers, else in shared memory
  float w[kHeld ? E : 1], b[kHeld ? E : 1];
  constexpr int kColumns = 32 * WARPS * E;
  float* s_w = reinterpret_cast<float*>(s_ring + Ahead::kBytes);  // [2][kColumns]
  if constexpr (kHeld) {
    Row::params(p.w, c0, p.W, w);
    Row::params(p.b, c0, p.W, b);
  } else {
    for (int c = threadIdx.x; c < kColumns; c += kLnThreads<WARPS>) {
      s_w[c] = c < p.W ? __ldg(p.w + c) : 0.0f;
      s_w[kColumns + c] = p.b != nullptr && c < p.W ? __ldg(p.b + c) : 0.0f;
    }
    __syncthreads();
  }
  int par = 0;
  for (long long r = first; r < p.R; r += step, par ^= 1) {
    float x[E], sum = 0.0f, m2 = 0.0f;
    ahead.wait();
    ahead.take(0, static_cast<const T*>(p.x) + r * p.sx, p.W, x);
    ahead.taken();
    if (Ahead::kVectors || WARPS == 1) ask(r + Ahead::kDepth * step);
#pragma unroll
    for (int k = 0; k < E; ++k) sum += x[k];
    float mean = warp_sum(sum) * inv_count;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * Row::kStep < p.W) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = x[j * VEC + e] - mean;
          m2 = fmaf(d, d, m2);
        }
      }
    m2 = warp_sum(m2);
    if constexpr (WARPS > 1) {
      if (lane == 0) s_stat[par][wp] = make_float4(mean, m2, count, 0.0f);
      __syncthreads();
      if (!Ahead::kVectors) ask(r + Ahead::kDepth * step);
      float all = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) all = fmaf(s_stat[par][k].z, s_stat[par][k].x, all);
      mean = all * inv_w;
      m2 = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float4 q = s_stat[par][k];
        const float d = q.x - mean;
        m2 += q.z > 0.0f ? fmaf(q.z * d, d, q.y) : 0.0f;
      }
    }
    const float rstd = 1.0f / sqrtf(fmaf(m2, inv_w, p.eps));
    if (i == 0 && p.mean != nullptr) p.mean[r] = mean, p.rstd[r] = rstd;
    // (without a bias b = 0: fmaf(n, w, 0) is n w but for the sign of a zero)
    if constexpr (kHeld) {
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = fmaf((x[k] - mean) * rstd, w[k], b[k]);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const float* q = s_w + c0 + j * Row::kStep;
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[j * VEC + e] = fmaf((x[j * VEC + e] - mean) * rstd, q[e], q[kColumns + e]);
      }
    }
    Row::put(p.out, r * p.W, c0, p.W, x);
  }
}

template <typename T, int VEC, int NV, int WARPS>
__global__ void __launch_bounds__(kLnThreads<WARPS>) ln_bwd_kernel(const LnParams p) {
  using Row = LnRow<T, VEC, NV, WARPS>;
  constexpr int E = NV * VEC;
  __shared__ float2 s_sum[2][WARPS];
  const int i = WARPS == 1 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31, c0 = i * VEC;
  const long long first = WARPS == 1 ? (long long)blockIdx.x * kLnRows + wp : blockIdx.x;
  const long long step = WARPS == 1 ? (long long)gridDim.x * kLnRows : gridDim.x;
  const float inv_w = 1.0f / (float)p.W;
  extern __shared__ __align__(16) unsigned char s_ring[];
  using Ahead = LnAhead<T, VEC, NV, WARPS, 2>;
  Ahead ahead(s_ring);
  auto ask = [&](long long r) {
    if (r < p.R) {
      ahead.ask(0, static_cast<const T*>(p.x) + r * p.sx, p.W);
      ahead.ask(1, static_cast<const T*>(p.dy) + r * p.sdy, p.W);
    }
    ahead.asked();
  };
#pragma unroll
  for (int k = 0; k < Ahead::kDepth; ++k) ask(first + k * step);
  float mean = 0.0f, rstd = 0.0f, next_mean = 0.0f, next_rstd = 0.0f;
  if (first < p.R) next_mean = __ldg(p.mean + first), next_rstd = __ldg(p.rstd + first);
  float w[E], dw[E], db[E];
  Row::params(p.w, c0, p.W, w);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.0f;
  int par = 0;
  for (long long r = first; r < p.R; r += step, par ^= 1) {
    float n[E], d[E], s1 = 0.0f, s2 = 0.0f;
    ahead.wait();
    ahead.take(0, static_cast<const T*>(p.x) + r * p.sx, p.W, n);
    ahead.take(1, static_cast<const T*>(p.dy) + r * p.sdy, p.W, d);
    ahead.taken();
    if (Ahead::kVectors || WARPS == 1) ask(r + Ahead::kDepth * step);
    mean = next_mean;
    rstd = next_rstd;
    if (r + step < p.R) next_mean = __ldg(p.mean + r + step), next_rstd = __ldg(p.rstd + r + step);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      n[k] = (n[k] - mean) * rstd;  // (beyond the row d = 0, so n does not matter)
      dw[k] = fmaf(d[k], n[k], dw[k]);
      db[k] += d[k];
      d[k] *= w[k];
      s1 += d[k];
      s2 = fmaf(d[k], n[k], s2);
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (WARPS > 1) {
      if (lane == 0) s_sum[par][wp] = make_float2(s1, s2);
      __syncthreads();
      if (!Ahead::kVectors) ask(r + Ahead::kDepth * step);
      s1 = s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) s1 += s_sum[par][k].x, s2 += s_sum[par][k].y;
    }
    s1 *= inv_w * rstd;
    s2 *= inv_w * rstd;
#pragma unroll
    for (int k = 0; k < E; ++k) d[k] = fmaf(rstd, d[k], fmaf(-n[k], s2, -s1));
    Row::put(p.out, r * p.W, c0, p.W, d);
  }
  if (p.part == nullptr) return;
  float* part = p.part + (long long)blockIdx.x * 2 * p.W;
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * Row::kStep < p.W) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = c0 + j * Row::kStep + e;
          part[c] = dw[j * VEC + e], part[p.W + c] = db[j * VEC + e];
        }
      }
  } else {
    float* s_part = reinterpret_cast<float*>(s_ring);  // [kLnRows][2][W], once every warp is through with its rows
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * Row::kStep < p.W) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = c0 + j * Row::kStep + e;
          s_part[wp * 2 * p.W + c] = dw[j * VEC + e];
          s_part[wp * 2 * p.W + p.W + c] = db[j * VEC + e];
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

// The backward of rows whose column sums do not fit the registers beside them: a row in the registers of 32
// warps, weights and sums in shared memory (every thread its own columns), which leaves none for rows
// ahead: the next row is asked for into L2 while this one is worked on. (2690 x 14960 float32 100 us,
// 4000 x 16384 bfloat16 117 us, of floors 74 and 60; two reads of each row and a third for the sums took
// 199 and 259. One CTA an SM walks its rows without overlap of a row's loads and its stores.)
constexpr int kLnTallWarps = 32;
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(32 * kLnTallWarps) ln_tall_bwd_kernel(const LnParams p) {
  constexpr int WARPS = kLnTallWarps, E = NV * VEC, N = 32 * WARPS;
  using V = LnVec<T, VEC>;
  using Row = LnRow<T, VEC, NV, WARPS>;
  __shared__ float2 s_sum[2][WARPS];
  extern __shared__ float s_columns[];  // [w, dw, db][element of a thread][thread]
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31, c0 = threadIdx.x * VEC;
  const float inv_w = 1.0f / (float)p.W;
  const bool sums = p.part != nullptr;
  float *w = s_columns + threadIdx.x, *dw = w + E * N, *db = dw + E * N;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const int c = c0 + k / VEC * Row::kStep + k % VEC;
    w[k * N] = c < p.W ? __ldg(p.w + c) : 0.0f;
    if (sums) dw[k * N] = db[k * N] = 0.0f;
  }
  int par = 0;
  for (long long r = blockIdx.x; r < p.R; r += gridDim.x, par ^= 1) {
    const T *x = static_cast<const T*>(p.x) + r * p.sx, *dy = static_cast<const T*>(p.dy) + r * p.sdy;
    typename V::type rx[NV], rd[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * Row::kStep < p.W) {
        rx[j] = *reinterpret_cast<const typename V::type*>(x + c0 + j * Row::kStep);
        rd[j] = *reinterpret_cast<const typename V::type*>(dy + c0 + j * Row::kStep);
      }
    const float mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
    if (r + gridDim.x < p.R) {
      constexpr int kLine = 128 / (int)sizeof(T);
      for (int c = threadIdx.x * kLine; c < p.W; c += 32 * WARPS * kLine) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(x + gridDim.x * p.sx + c));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(dy + gridDim.x * p.sdy + c));
      }
    }
    float n[E], d[E], s1 = 0.0f, s2 = 0.0f;
    Row::get(rx, c0, p.W, n);
    Row::get(rd, c0, p.W, d);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      n[k] = (n[k] - mean) * rstd;  // (beyond the row d = 0, so n does not matter)
      if (sums) {
        dw[k * N] = fmaf(d[k], n[k], dw[k * N]);
        db[k * N] += d[k];
      }
      d[k] *= w[k * N];
      s1 += d[k];
      s2 = fmaf(d[k], n[k], s2);
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (lane == 0) s_sum[par][wp] = make_float2(s1, s2);
    __syncthreads();
    const float2 part = s_sum[par][lane];  // (a warp's sum a lane)
    s1 = warp_sum(part.x) * (inv_w * rstd);
    s2 = warp_sum(part.y) * (inv_w * rstd);
#pragma unroll
    for (int k = 0; k < E; ++k) d[k] = fmaf(rstd, d[k], fmaf(-n[k], s2, -s1));
    Row::put(p.out, r * p.W, c0, p.W, d);
  }
  if (!sums) return;
  float* out = p.part + (long long)blockIdx.x * 2 * p.W;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (c0 + j * Row::kStep < p.W) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = c0 + j * Row::kStep + e;
        out[c] = dw[(j * VEC + e) * N], out[p.W + c] = db[(j * VEC + e) * N];
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
#pragma unroll 4
    for (int c = threadIdx.x; c < p.W; c += kLnWide) sum += Io<T>::load(x + c);
    float mean = block_sum(sum, s) * inv_w;
    float m2 = 0.0f, m1 = 0.0f;
#pragma unroll 4
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float d = Io<T>::load(x + c) - mean;
      m1 += d;
      m2 = fmaf(d, d, m2);
    }
    // the deviations' own mean is what rounding left of the mean
    const float off = block_sum(m1, s) * inv_w;
    // (what is left of a row without variance may be below zero by rounding)
    float var = block_sum(m2, s) * inv_w - off * off;
    if (var < 0.0f) var = 0.0f;
    const float rstd = 1.0f / sqrtf(var + p.eps);
    mean += off;
    if (threadIdx.x == 0 && p.mean != nullptr) p.mean[r] = mean, p.rstd[r] = rstd;
#pragma unroll 4
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
#pragma unroll 4
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float d = Io<T>::load(dy + c) * p.w[c];
      s1 += d;
      s2 = fmaf(d, (Io<T>::load(x + c) - mean) * rstd, s2);
    }
    s1 = block_sum(s1, s) * inv_w;
    s2 = block_sum(s2, s) * inv_w;
#pragma unroll 4
    for (int c = threadIdx.x; c < p.W; c += kLnWide) {
      const float n = (Io<T>::load(x + c) - mean) * rstd;
      Io<T>::store(static_cast<T*>(p.out) + r * p.W + c, rstd * (Io<T>::load(dy + c) * p.w[c] - s1 - n * s2));
    }
  }
}

// Partial sums of dw and db over every gridDim.y-th row, a thread per column.
template <typename T>
__global__ void __launch_bounds__(256) ln_wide_cols_kernel(const LnParams p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.W) return;
  float dw = 0.0f, db = 0.0f;
#pragma unroll 4
  for (long long r = blockIdx.y; r < p.R; r += gridDim.y) {
    const float d = Io<T>::load(static_cast<const T*>(p.dy) + r * p.sdy + c);
    dw = fmaf(d, (Io<T>::load(static_cast<const T*>(p.x) + r * p.sx + c) - p.mean[r]) * p.rstd[r], dw);
    db += d;
  }
  p.part[(long long)blockIdx.y * 2 * p.W + c] = dw;
  p.part[(long long)blockIdx.y * 2 * p.W + p.W + c] = db;
}

// dw, db from the partial rows: a block owns 32 of the 2 W columns, its 32 warps every 32nd row, in
// float64 and in order. (The rows are read four at a time: the kernel is a chain of loads.)
__global__ void __launch_bounds__(1024) ln_reduce_kernel(const float* part, float* dw, float* db, int rows, int W) {
  __shared__ double s[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane, n = 2LL * W;
  double t = 0.0;
  if (c < n)
    for (int r = wp; r < rows; r += 128) {
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = r + 32 * u < rows ? part[(r + 32 * u) * n + c] : 0.0f;
      t += ((double)v[0] + (double)v[1]) + ((double)v[2] + (double)v[3]);
    }
  s[wp][lane] = t;
  __syncthreads();
  t = s[lane][wp];  // column wp of the block, row lane of its sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const long long out = (long long)blockIdx.x * 32 + wp;
  if (lane == 0 && out < n) {
    if (out < W) {
      if (dw != nullptr) dw[out] = (float)t;
    } else if (db != nullptr) {
      db[out - W] = (float)t;
    }
  }
}

// ---------------------------------------------------------------- host
constexpr int kLnSms = 148;
constexpr int kLnSumGrid = kLnSms * 8;  // the most CTAs that walk the rows

struct LnPlan {
  int vec, elements, warps;  // elements a thread; warps a row (0: the wide kernels)
};

// The narrowest of the instances that holds a row. The forward gives a row of up to 2048 to one warp,
// which needs no barrier, once there are rows enough to fill the SMs with such warps (131072 x 2048
// bf16: four warps a row 202 us, one 194; 138996 x 1374: 249, 216); with fewer, four warps are done
// sooner.
static LnPlan ln_plan(long long R, int W, int vec, bool backward) {
  if (W <= 256) return LnPlan{vec, 8, 1};
  if (W <= 512) return LnPlan{vec, 16, 1};
  if (!backward && R >= kLnSms * 16) {
    if (W <= 1024) return LnPlan{vec, 32, 1};
    if (W <= 2048) return LnPlan{vec, 64, 1};
  }
  if (W <= 1024) return LnPlan{vec, 8, 4};
  for (int warps : {4, 8, 16})
    if (W <= 32 * 16 * warps) return LnPlan{vec, 16, warps};
  if (W <= 32 * 32 * 16) return backward ? LnPlan{vec, 16, kLnTallWarps} : LnPlan{vec, 32, 16};
  return LnPlan{1, 0, 0};
}

static int ln_check_shape(long long R, long long W) {
  if (R <= 0 || W <= 0) return fail(SPARC_ERR_SHAPE, "rows and width must be positive");
  if (W > (1LL << 24) || R > (1LL << 40) || (double)R * (double)W > 4.0e18)
    return fail(SPARC_ERR_SHAPE, "shape beyond the launch grid (width <= 2^24)");
  return SPARC_OK;
}

static size_t ln_ws_bytes(long long R, long long W) {
  return (size_t)std::min<long long>(R, kLnSumGrid) * 2 * (size_t)W * sizeof(float);
}

// CTAs that walk the rows: as many as are resident at once, and in the backward write a row of partial
// sums each (kLnSumGrid of them at most).
template <typename T, int VEC, int NV, int WARPS>
static cudaError_t ln_launch(const LnParams& p, int* grid, bool backward, cudaStream_t s) {
  void (*kernel)(const LnParams) = ln_fwd_kernel<T, VEC, NV, WARPS>;
  if constexpr (VEC * NV <= kLnHeld) {  // (the backward's sums are in registers too)
    if (backward) kernel = ln_bwd_kernel<T, VEC, NV, WARPS>;
  }
  int ring = LnAhead<T, VEC, NV, WARPS, 1>::kBytes;
  if constexpr (VEC * NV <= kLnHeld) {
    if (backward) ring = LnAhead<T, VEC, NV, WARPS, 2>::kBytes;
  }
  // (one warp a row: the warps' sums meet in the same memory)
  int smem = backward && WARPS == 1 ? std::max(ring, kLnRows * 2 * 32 * VEC * NV * (int)sizeof(float)) : ring;
  if (!backward && VEC * NV > kLnHeld) smem += 2 * 32 * WARPS * VEC * NV * (int)sizeof(float);
  cudaError_t e = cudaSuccess;
  if (smem > 40 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  static int resident[2] = {0, 0};
  int per_sm = __atomic_load_n(&resident[backward], __ATOMIC_RELAXED);
  if (per_sm == 0) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kLnThreads<WARPS>, smem);
    if (e != cudaSuccess) return e;
    per_sm = std::max(1, std::min(per_sm, kLnSumGrid / kLnSms));
    __atomic_store_n(&resident[backward], per_sm, __ATOMIC_RELAXED);
  }
  const int rows = WARPS == 1 ? kLnRows : 1;
  *grid = (int)std::min<long long>((p.R + rows - 1) / rows, (long long)per_sm * kLnSms);
  TimedLaunch tl(backward ? kTimeLnBwd : kTimeLnFwd, s);
  kernel<<<*grid, kLnThreads<WARPS>, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int VEC>
static cudaError_t ln_tall_launch(const LnParams& p, int* grid, cudaStream_t s) {
  const auto kernel = ln_tall_bwd_kernel<T, VEC, 16 / VEC>;
  constexpr int kArray = 32 * kLnTallWarps * 16 * (int)sizeof(float);
  const int smem = (p.part != nullptr ? 3 : 1) * kArray;
  // (the limit is the kernel's, not the launch's: always the largest, as another thread may launch between)
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * kArray);
  if (e != cudaSuccess) return e;
  *grid = (int)std::min<long long>(p.R, kLnSms);
  TimedLaunch tl(kTimeLnBwd, s);
  kernel<<<*grid, 32 * kLnTallWarps, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int VEC>
static cudaError_t ln_instance(const LnParams& p, const LnPlan& pl, int* grid, bool backward, cudaStream_t s) {
  switch (pl.warps * 100 + pl.elements) {
    case 108: return ln_launch<T, VEC, 8 / VEC, 1>(p, grid, backward, s);
    case 116: return ln_launch<T, VEC, 16 / VEC, 1>(p, grid, backward, s);
    case 132: return ln_launch<T, VEC, 32 / VEC, 1>(p, grid, backward, s);
    case 164: return ln_launch<T, VEC, 64 / VEC, 1>(p, grid, backward, s);
    case 408: return ln_launch<T, VEC, 8 / VEC, 4>(p, grid, backward, s);
    case 416: return ln_launch<T, VEC, 16 / VEC, 4>(p, grid, backward, s);
    case 816: return ln_launch<T, VEC, 16 / VEC, 8>(p, grid, backward, s);
    case kLnTallWarps * 100 + 16: return ln_tall_launch<T, VEC>(p, grid, s);
    case 1632: return ln_launch<T, VEC, 32 / VEC, 16>(p, grid, backward, s);
    default: return ln_launch<T, VEC, 16 / VEC, 16>(p, grid, backward, s);
  }
}

template <typename T>
static cudaError_t ln_dispatch(const LnParams& p, const LnPlan& pl, int* grid, bool backward, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (pl.warps == 0) {
    // (fewer rows of column sums than rows: each is worth four rows at least)
    *grid = (int)std::min<long long>(backward ? (p.R + 3) / 4 : p.R, kLnSms * 2);
    TimedLaunch tl(backward ? kTimeLnBwd : kTimeLnFwd, s);
    if (!backward) {
      ln_wide_fwd_kernel<T><<<*grid, kLnWide, 0, s>>>(p);
    } else {
      ln_wide_bwd_kernel<T><<<*grid, kLnWide, 0, s>>>(p);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
      if (p.part != nullptr) ln_wide_cols_kernel<T><<<dim3((unsigned)(p.W + 255) / 256, (unsigned)*grid), 256, 0, s>>>(p);
    }
    return cudaGetLastError();
  }
  if (pl.vec == 1) return ln_instance<T, 1>(p, pl, grid, backward, s);
  if (pl.vec == 2) return ln_instance<T, 2>(p, pl, grid, backward, s);
  return ln_instance<T, V>(p, pl, grid, backward, s);
}

// Elements that width, bases and row strides let be read and written at once: 16 bytes, a pair, or one.
struct LnTensor {
  const void* p;
  long long stride;
};
static int ln_vec(long long R, int W, std::initializer_list<LnTensor> tensors, int size) {
  auto fits = [&](int bytes) {
    bool ok = (long long)W * size % bytes == 0;
    for (const LnTensor& t : tensors)
      ok = ok && reinterpret_cast<uintptr_t>(t.p) % bytes == 0 && (R <= 1 || t.stride * size % bytes == 0);
    return ok;
  };
  return fits(16) ? 16 / size : fits(2 * size) ? 2 : 1;
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
  const LnPlan pl = ln_plan(p.R, p.W, ln_vec(p.R, p.W, {{a->x, p.sx}, {a->y, p.W}}, size), false);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int grid = 0;
  const cudaError_t e = a->dtype == SPARC_DTYPE_BF16 ? ln_dispatch<__nv_bfloat16>(p, pl, &grid, false, s)
                                                     : ln_dispatch<float>(p, pl, &grid, false, s);
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
  const LnPlan pl = ln_plan(p.R, p.W, ln_vec(p.R, p.W, {{a->x, p.sx}, {a->dy, p.sdy}, {a->dx, p.W}}, size), true);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int grid = 0;
  cudaError_t e = a->dtype == SPARC_DTYPE_BF16 ? ln_dispatch<__nv_bfloat16>(p, pl, &grid, true, s)
                                               : ln_dispatch<float>(p, pl, &grid, true, s);
  if (e == cudaSuccess && sums) {
    TimedLaunch tl(kTimeLnReduce, s);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((2 * p.W + 31) / 32));
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, ln_reduce_kernel, (const float*)p.part, a->grad_weight, a->grad_bias, grid, p.W);
  }
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

}  // extern "C"
