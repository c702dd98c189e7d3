// Global gradient norm over many tensors, and clipping by it, for B200 (sm_100a):
//   norm = sqrt(sum_i g_i^2) over every element of every tensor,
//   out_i = g_i min(1, max_norm / (norm + eps)).
//
// Two launches whatever the number of tensors (up to kClipTensors each; more tensors take more
// launches): the tensors are cut into chunks of kClipChunk elements, the CTAs of a grid that fills
// the GPU walk the chunks of all tensors, and each writes one partial sum; every CTA of the second
// kernel adds the partial sums in the same fixed order (bitwise reproducible, no atomics), and
// scales its chunks, the last read first, so that it meets what the caches still hold. Where
// nothing is to be clipped and the gradients are updated in place nothing is written.
//
// Measured on a B200 (537 MB of float32 gradients in 56 tensors, four of 33 MB to a layer): norm 95 us =
// 5.7 TB/s (86% of what a copy reaches), scaling 165 us = 6.5 TB/s (99%): bound by HBM. Forty tensors
// of 1024 to 2049: 7 and 4 us, launches and one chain of loads each.
//
// Squares are summed in float32 over a thread's 16 or 32 elements at a time and then in float64. A
// group whose sum leaves [2^-100, 2^120] is summed again in float64, so neither a square that
// overflows nor one that underflows is lost: the norm is right for every finite float32 input.
#include <algorithm>
#include <exception>
#include <vector>

#include "common.cuh"
#include "sparc_b200.h"
#include "timing.cuh"

namespace sparc {

constexpr int kClipTensors = 256;   // tensors per launch
constexpr int kClipChunk = 8192;    // elements per chunk
constexpr int kClipThreads = 256;
constexpr int kClipGrid = 148 * 8;  // the most CTAs, and partial sums per launch
constexpr int kClipVecs = 4;        // 16-byte vectors a thread has on the way at once

struct ClipTensors {
  const void* in[kClipTensors];
  void* out[kClipTensors];
  long long count[kClipTensors];
  unsigned first[kClipTensors + 1];  // chunks before tensor i
  unsigned char bf16[kClipTensors];
  int n;
  int single;  // every tensor is one chunk: chunk i is tensor i, with no search
};

struct ClipScale {
  const double* part;
  int parts;       // over every launch of the norm
  float max_norm, eps;
  float* norm;     // written by the first CTA, or null
};

__device__ __forceinline__ int clip_find(const ClipTensors& t, unsigned chunk) {
  if (t.single) return (int)chunk;
  int lo = 0, hi = t.n;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 16 bytes of gradients: four float32 or eight bfloat16.
template <typename T> struct ClipVec;
template <> struct ClipVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 scaled(uint4 v, float k) {
    return make_uint4(__float_as_uint(__uint_as_float(v.x) * k), __float_as_uint(__uint_as_float(v.y) * k),
                      __float_as_uint(__uint_as_float(v.z) * k), __float_as_uint(__uint_as_float(v.w) * k));
  }
};
template <> struct ClipVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(uint4 v, float (&f)[8]) {
    const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) f[2 * k] = __uint_as_float(u[k] << 16), f[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
  }
  static __device__ __forceinline__ unsigned scaled(unsigned u, float k) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(u << 16) * k, __uint_as_float(u & 0xffff0000u) * k);
    return *reinterpret_cast<const unsigned*>(&b);
  }
  static __device__ __forceinline__ uint4 scaled(uint4 v, float k) {
    return make_uint4(scaled(v.x, k), scaled(v.y, k), scaled(v.z, k), scaled(v.w, k));
  }
};

// The squares of n elements from `g` on.
template <typename T>
__device__ __forceinline__ void clip_squares(const T* g, int n, bool wide, double& sum) {
  using V = ClipVec<T>;
  int done = 0;
  if (wide) {
    const uint4* gv = reinterpret_cast<const uint4*>(g);
    const int vecs = n / V::N;
    for (int k = threadIdx.x; k < vecs; k += kClipVecs * kClipThreads) {
      uint4 v[kClipVecs];
#pragma unroll
      for (int u = 0; u < kClipVecs; ++u)
        v[u] = k + u * kClipThreads < vecs ? __ldg(gv + k + u * kClipThreads) : make_uint4(0u, 0u, 0u, 0u);
      // sums of four squares, added in pairs: at most seven roundings
      constexpr int kParts = kClipVecs * V::N / 4;
      float f[kClipVecs][V::N], s[kParts];
#pragma unroll
      for (int u = 0; u < kClipVecs; ++u) V::get(v[u], f[u]);
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        const float* e = &f[q * 4 / V::N][q * 4 % V::N];
        s[q] = fmaf(e[3], e[3], fmaf(e[2], e[2], fmaf(e[1], e[1], e[0] * e[0])));
      }
#pragma unroll
      for (int d = 1; d < kParts; d *= 2)
#pragma unroll
        for (int q = 0; q + d < kParts; q += 2 * d) s[q] += s[q + d];
      if (s[0] >= 7.8886090522101181e-31f && s[0] <= 1.3292279957849159e36f) {
        sum += (double)s[0];
      } else {  // (also zeros, infinities and NaN)
#pragma unroll
        for (int u = 0; u < kClipVecs; ++u)
#pragma unroll
          for (int e = 0; e < V::N; ++e) sum = fma((double)f[u][e], (double)f[u][e], sum);
      }
    }
    done = vecs * V::N;
  }
  for (int k = done + threadIdx.x; k < n; k += kClipThreads) {
    const double v = (double)to_float(g[k]);
    sum = fma(v, v, sum);
  }
}

// out = g k for n elements.
template <typename T>
__device__ __forceinline__ void clip_scale(const T* g, T* o, int n, bool wide, float k0) {
  using V = ClipVec<T>;
  int done = 0;
  if (wide) {
    const uint4* gv = reinterpret_cast<const uint4*>(g);
    uint4* ov = reinterpret_cast<uint4*>(o);
    const int vecs = n / V::N;
    for (int k = threadIdx.x; k < vecs; k += kClipVecs * kClipThreads) {
      uint4 v[kClipVecs];
#pragma unroll
      for (int u = 0; u < kClipVecs; ++u)
        if (k + u * kClipThreads < vecs) v[u] = gv[k + u * kClipThreads];
#pragma unroll
      for (int u = 0; u < kClipVecs; ++u)
        if (k + u * kClipThreads < vecs) ov[k + u * kClipThreads] = V::scaled(v[u], k0);
    }
    done = vecs * V::N;
  }
  for (int k = done + threadIdx.x; k < n; k += kClipThreads) Io<T>::store(o + k, to_float(g[k]) * k0);
}

// The sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ double clip_block_sum(double v, double* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int k = 0; k < kClipThreads / 32; ++k) v += s[k];
  return v;
}

__global__ void __launch_bounds__(kClipThreads) grad_norm_kernel(const __grid_constant__ ClipTensors t, double* part) {
  __shared__ double s[kClipThreads / 32];
  double sum = 0.0;
  const unsigned chunks = t.first[t.n];
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = clip_find(t, c);
    const long long e0 = (long long)(c - t.first[i]) * kClipChunk;
    const int n = (int)min((long long)kClipChunk, t.count[i] - e0);
    const bool wide = reinterpret_cast<unsigned long long>(t.in[i]) % 16 == 0;
    if (t.bf16[i]) clip_squares(static_cast<const __nv_bfloat16*>(t.in[i]) + e0, n, wide, sum);
    else clip_squares(static_cast<const float*>(t.in[i]) + e0, n, wide, sum);
  }
  sum = clip_block_sum(sum, s);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

__device__ __forceinline__ double clip_norm(const ClipScale& c, double* s) {
  double sum = 0.0;
  for (int k = threadIdx.x; k < c.parts; k += kClipThreads) sum += c.part[k];
  return sqrt(clip_block_sum(sum, s));
}

__global__ void __launch_bounds__(kClipThreads) grad_norm_finish_kernel(const ClipScale c) {
  __shared__ double s[kClipThreads / 32];
  pdl_wait();
  const double norm = clip_norm(c, s);
  if (threadIdx.x == 0) *c.norm = (float)norm;
}

__global__ void __launch_bounds__(kClipThreads) grad_clip_kernel(const __grid_constant__ ClipTensors t,
                                                                 const __grid_constant__ ClipScale sc) {
  __shared__ double s[kClipThreads / 32];
  pdl_wait();
  const double norm = clip_norm(sc, s);
  if (sc.norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *sc.norm = (float)norm;
  const double limit = norm + (double)sc.eps;
  // (a norm that is NaN clips: every gradient becomes NaN, as the product says)
  const float k0 = (double)sc.max_norm >= limit ? 1.0f : (float)((double)sc.max_norm / limit);
  const unsigned chunks = t.first[t.n];
  if (blockIdx.x >= chunks) return;
  unsigned c = blockIdx.x + (chunks - 1 - blockIdx.x) / gridDim.x * gridDim.x;  // this CTA's last chunk
  for (;; c -= gridDim.x) {
    const int i = clip_find(t, c);
    const long long e0 = (long long)(c - t.first[i]) * kClipChunk;
    const int n = (int)min((long long)kClipChunk, t.count[i] - e0);
    const bool same = t.in[i] == t.out[i];
    if (!(same && k0 == 1.0f)) {
      const bool wide = (reinterpret_cast<unsigned long long>(t.in[i]) | reinterpret_cast<unsigned long long>(t.out[i])) % 16 == 0;
      if (t.bf16[i])
        clip_scale(static_cast<const __nv_bfloat16*>(t.in[i]) + e0, static_cast<__nv_bfloat16*>(t.out[i]) + e0, n, wide, k0);
      else
        clip_scale(static_cast<const float*>(t.in[i]) + e0, static_cast<float*>(t.out[i]) + e0, n, wide, k0);
    }
    if (c < gridDim.x) break;
  }
}

// A launch that may start while the kernel before it drains (it waits for that kernel's sums itself).
template <typename... P>
static cudaError_t clip_launch(void (*kernel)(P...), unsigned grid, cudaStream_t s, const P&... params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kClipThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, params...);
}

static int clip_launches(int tensors) { return std::max(1, (tensors + kClipTensors - 1) / kClipTensors); }

}  // namespace sparc

using namespace sparc;

extern "C" {

size_t sparc_grad_clip_workspace_bytes(int tensors) {
  return tensors < 0 ? 0 : (size_t)clip_launches(tensors) * kClipGrid * sizeof(double);
}

int sparc_grad_clip(const SparcGradClipArgs* a, void* stream) {
  NvtxRange nvtx(__func__);
  if (a == nullptr) return fail(SPARC_ERR_ARG, "null args");
  if (a->tensors <= 0) return fail(SPARC_ERR_SHAPE, "no tensors");
  if (!a->grads || !a->counts || !a->dtypes || !a->norm) return fail(SPARC_ERR_ARG, "null pointer");
  if (a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 8 != 0 ||
      a->workspace_bytes < sparc_grad_clip_workspace_bytes(a->tensors))
    return fail(SPARC_ERR_WORKSPACE, "workspace missing, too small or not 8-byte aligned");
  if (a->out != nullptr && !(a->max_norm >= 0.0f && a->eps >= 0.0f))
    return fail(SPARC_ERR_ARG, "max_norm and eps must not be negative");
  try {
    struct Span {
      uintptr_t begin, end;
      int tensor;
      bool out;
    };
    std::vector<Span> spans;
    long long total = 0;
    for (int i = 0; i < a->tensors; ++i) {
      const int dt = a->dtypes[i];
      if (dt != SPARC_DTYPE_F32 && dt != SPARC_DTYPE_BF16) return fail(SPARC_ERR_DTYPE, "unsupported dtype");
      const long long n = a->counts[i];
      const size_t size = dt == SPARC_DTYPE_BF16 ? 2 : 4;
      if (n < 0 || n > (1LL << 43) - total) return fail(SPARC_ERR_SHAPE, "element count out of range");  // 2^30 chunks
      if (n == 0) continue;
      total += n;
      const uintptr_t in = reinterpret_cast<uintptr_t>(a->grads[i]);
      const uintptr_t out = a->out != nullptr ? reinterpret_cast<uintptr_t>(a->out[i]) : in;
      if (in == 0 || out == 0) return fail(SPARC_ERR_ARG, "null tensor pointer");
      if (in % size != 0 || out % size != 0) return fail(SPARC_ERR_ARG, "misaligned tensor pointer");
      if (a->out != nullptr) {
        spans.push_back(Span{out, out + (uintptr_t)n * size, i, true});
        if (in != out) spans.push_back(Span{in, in + (uintptr_t)n * size, i, false});
      }
    }
    // an output may be its own gradient, but may overlap nothing else
    std::sort(spans.begin(), spans.end(), [](const Span& p, const Span& q) { return p.begin < q.begin; });
    uintptr_t end = 0, out_end = 0;
    for (const Span& s : spans) {
      if (s.begin < (s.out ? end : out_end)) return fail(SPARC_ERR_ARG, "an output overlaps another tensor");
      end = std::max(end, s.end);
      if (s.out) out_end = std::max(out_end, s.end);
    }
  } catch (const std::exception&) {
    return fail(SPARC_ERR_ARG, "out of host memory");
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  double* part = static_cast<double*>(a->workspace);
  ClipScale sc = {};
  sc.part = part;
  sc.max_norm = a->max_norm;
  sc.eps = a->eps;
  sc.norm = a->norm;
  // one launch's tensors, from tensor `from` on: those with elements, as many as fit
  auto fill = [&](ClipTensors* t, int from) {
    t->n = 0;
    t->first[0] = 0;
    int i = from;
    for (; i < a->tensors && t->n < kClipTensors; ++i) {
      if (a->counts[i] == 0) continue;
      const long long chunks = (a->counts[i] - 1) / kClipChunk + 1;
      t->in[t->n] = a->grads[i];
      t->out[t->n] = a->out != nullptr ? a->out[i] : nullptr;
      t->count[t->n] = a->counts[i];
      t->bf16[t->n] = a->dtypes[i] == SPARC_DTYPE_BF16;
      t->first[t->n + 1] = t->first[t->n] + (unsigned)chunks;
      ++t->n;
    }
    t->single = t->first[t->n] == (unsigned)t->n;
    return i;
  };
  cudaError_t e = cudaSuccess;
  ClipTensors t;
  for (int i = 0; i < a->tensors && e == cudaSuccess;) {
    i = fill(&t, i);
    if (t.n == 0) break;
    const unsigned grid = std::min<unsigned>(t.first[t.n], kClipGrid);
    TimedLaunch tl(kTimeGradNorm, s);
    grad_norm_kernel<<<grid, kClipThreads, 0, s>>>(t, part + sc.parts);
    sc.parts += (int)grid;
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && (a->out == nullptr || sc.parts == 0)) {
    TimedLaunch tl(kTimeGradClip, s);
    e = clip_launch(grad_norm_finish_kernel, 1, s, sc);
  } else {
    for (int i = 0; i < a->tensors && e == cudaSuccess;) {
      i = fill(&t, i);
      if (t.n == 0) break;
      TimedLaunch tl(kTimeGradClip, s);
      e = clip_launch(grad_clip_kernel, std::min<unsigned>(t.first[t.n], kClipGrid), s, t, sc);
      sc.norm = nullptr;
    }
  }
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

}  // extern "C"
