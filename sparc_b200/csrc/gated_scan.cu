// Gated linear recurrence for B200 (sm_100a): forward, backward and one decode step. Per batch row
// and channel, with s the logistic function, nu = e^{nu_log}:
//   u_t = -nu s(retention_t),  a_t = e^{u_t},  g_t = sqrt(1 - a_t^2) s(write_t),
//   h_t = c_t h_{t-1} + g_t x_t,  c_t = a_t, or 0 where token t starts a segment (segment_pos == 0).
// Backward for the adjoint lam_t = dy_t + c_{t+1} lam_{t+1} (lam_{T-1} also takes the gradient of
// the last state):
//   dx_t = lam_t g_t,  dwrite_t = lam_t g_t x_t (1 - s(write_t)),
//   du_t = lam_t (c_t h_{t-1} - x_t s(write_t) a_t^2 / sqrt(1 - a_t^2)),
//   dretention_t = du_t u_t (1 - s(retention_t)),  dnu_log = sum_{b,t} du_t u_t,  dh_0 = c_0 lam_0.
// u / sqrt(1 - a^2) stays finite as a -> 1 (it goes to -sqrt(-u/2)), so du u is formed from it.
//
// Decomposition: one launch each way, every tensor read once and written once. A lane owns VEC
// adjacent channels and a warp K consecutive tokens; a CTA's warps own consecutive spans of K
// tokens (a tile), and a thread-block cluster's CTAs consecutive tiles; the cluster walks the
// sequence. A thread turns its K tokens into an affine map (A, H): h_out = A h_in + H in
// registers, the maps of the CTA's warps are composed through shared memory, those of the
// cluster's CTAs through distributed shared memory (one cluster barrier per step, buffers of two
// parities), and the thread then replays its tokens from the state entering them. The backward
// does both directions in one step: the states from the forward's saved chunk carries (float32,
// one per kGatedChunk tokens, so that the states are not rounded to the activations' type), the
// adjoints from the step before. The cluster size grows as rows x channels shrink. All orders are
// fixed: results are bitwise reproducible.
//
// A segment start drops what came before it, infinities and NaN included: its factor is kept as
// -0 (a_t >= +0, so the sign marks it through products), and composing with it selects instead of
// multiplying.
#include <algorithm>

#include "common.cuh"
#include "sparc_b200.h"
#include "timing.cuh"

namespace sparc {

constexpr int kGatedChunk = 32;  // tokens per saved carry
constexpr int kGatedWarps = 8;   // warps per CTA
constexpr int kFwdK = 8;         // tokens per thread and step, forward
constexpr int kBwdK = 4;         // tokens per thread and step, backward (a chunk per CTA and step)
constexpr int kGatedMaxCluster = 8;
static_assert(kBwdK * kGatedWarps == kGatedChunk, "the backward's tile is one chunk");
static_assert(kGatedChunk % kFwdK == 0, "a carry is some thread's entering state");

struct GatedIn {
  const void* p;
  long long sb, st;  // batch and token strides in elements (channels adjacent)
};

struct GatedParams {
  GatedIn x, r, w, dy;
  void* y;             // [B, L, D] (forward)
  void *dx, *dr, *dw;  // [B, L, D] (backward)
  const float* nu_log; // [D]
  const float* h0;     // [B, D] or null
  float* last;         // [B, D] or null
  float* carry;        // [B, chunks, D]: the state entering each chunk, or null (forward)
  const float* grad_last;  // [B, D] or null
  float* grad_h0;      // [B, D] or null
  double* part;        // [rows, D] partial sums of dnu_log
  const void* pos;     // segment positions [B, L] or null
  int pos_bytes;
  long long B, L, chunks;
  int D, groups, cluster, rows;  // rows: clusters per channel group, each walking rows of the batch
};

// ---------------------------------------------------------------- VEC adjacent values
template <typename T, int VEC> struct Pack;
template <> struct Pack<float, 1> {
  using type = float;
  static __device__ __forceinline__ void get(float v, float* f) { f[0] = v; }
  static __device__ __forceinline__ float make(const float* f) { return f[0]; }
};
template <> struct Pack<float, 2> {
  using type = float2;
  static __device__ __forceinline__ void get(float2 v, float* f) { f[0] = v.x, f[1] = v.y; }
  static __device__ __forceinline__ float2 make(const float* f) { return make_float2(f[0], f[1]); }
};
template <> struct Pack<__nv_bfloat16, 1> {
  using type = unsigned short;
  static __device__ __forceinline__ void get(unsigned short v, float* f) { f[0] = __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned short make(const float* f) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
  }
};
template <> struct Pack<__nv_bfloat16, 2> {
  using type = unsigned;
  static __device__ __forceinline__ void get(unsigned v, float* f) {
    f[0] = __uint_as_float(v << 16);
    f[1] = __uint_as_float(v & 0xffff0000u);
  }
  static __device__ __forceinline__ unsigned make(const float* f) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const unsigned*>(&v);
  }
};

template <typename T, int VEC>
__device__ __forceinline__ typename Pack<T, VEC>::type gated_load(const GatedIn& in, long long b, long long t, int ch) {
  return __ldg(reinterpret_cast<const typename Pack<T, VEC>::type*>(static_cast<const T*>(in.p) + b * in.sb +
                                                                     t * in.st + ch));
}

__device__ __forceinline__ bool gated_starts(const void* pos, int bytes, long long i) {
  switch (bytes) {
    case 1: return __ldg(static_cast<const unsigned char*>(pos) + i) == 0;
    case 2: return __ldg(static_cast<const unsigned short*>(pos) + i) == 0;
    case 4: return __ldg(static_cast<const unsigned*>(pos) + i) == 0;
    default: return __ldg(static_cast<const unsigned long long*>(pos) + i) == 0;
  }
}

// ---------------------------------------------------------------- gates
__device__ __forceinline__ float min_nan(float a, float b) {  // min that keeps NaN
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// e^{-v}. float32: the product with log2 e is carried in two terms (its rounding alone would cost
// |v| 2^-24 in the result), with v held to +-88 so that both stay finite; 1 / (1 + e^88) flushes
// to the exact 0 that s(-inf) is.
template <typename T>
__device__ __forceinline__ float exp_neg(float v) {
  if constexpr (sizeof(T) == 2) {
    return ex2_approx(v * -kLog2e);
  } else {
    constexpr float kLog2eLo = 1.9259630e-8f;  // log2 e - kLog2e
    v = min_nan(max_nan(v, -88.0f), 88.0f);
    const float t = v * -kLog2e;
    const float lo = fmaf(v, -kLog2eLo, fmaf(v, -kLog2e, -t));
    const float e = ex2_approx(t);
    return fmaf(e, lo * 0.6931471805599453f, e);
  }
}

// a = e^u and a - 1 for u <= 0: above -1/2 from the series of e^u - 1 (through u^8 / 8!: the next
// term is below 2^-26 of the first), which keeps 1 - a^2 = -(a - 1)(2 + (a - 1)) exact to a few
// ulp where a is near 1 and holds the decay of long sequences; else the hardware exp2, which keeps
// a to a few ulp where it is small.
__device__ __forceinline__ float2 exp_expm1_neg(float u) {  // (a, a - 1)
  float p = 2.4801587301587302e-5f;             // 1/8!
  p = fmaf(p, u, 1.9841269841269841e-4f);       // 1/7!
  p = fmaf(p, u, 1.3888888888888889e-3f);       // 1/6!
  p = fmaf(p, u, 8.3333333333333333e-3f);       // 1/5!
  p = fmaf(p, u, 4.1666666666666667e-2f);       // 1/4!
  p = fmaf(p, u, 1.6666666666666667e-1f);       // 1/3!
  p = fmaf(p, u, 0.5f);
  const float small = fmaf(p * u, u, u);
  const float e = ex2_approx(u * kLog2e);
  const bool near = u > -0.5f;
  return make_float2(near ? 1.0f + small : e, near ? small : e - 1.0f);
}

// -nu of a channel, held finite so that nu s(retention) never meets 0 x infinity.
__device__ __forceinline__ float gated_minus_nu(float nu_log) { return -min_nan(expf(nu_log), 3.402823466e38f); }

template <typename T>
__device__ __forceinline__ void gated_ab(float x, float r, float w, float minus_nu, float* a, float* b) {
  const float sr = rcp_approx(1.0f + exp_neg<T>(r));
  const float sw = rcp_approx(1.0f + exp_neg<T>(w));
  const float2 e = exp_expm1_neg(minus_nu * sr);
  *a = e.x;
  *b = sqrt_approx(-e.y * (2.0f + e.y)) * sw * x;
}

// 1 - s(v) = e^{-v} s(v) without cancellation, given e = e^{-v} (which may be infinite).
__device__ __forceinline__ float one_minus_s(float e, float s) { return e > 8.5070592e37f ? 1.0f : e * s; }

// ---------------------------------------------------------------- affine maps
__device__ __forceinline__ bool dropped(float A) { return __float_as_int(A) < 0; }

// v <- A v + H
template <bool SEG>
__device__ __forceinline__ float through(float A, float H, float v) {
  const float o = fmaf(A, v, H);
  return SEG && dropped(A) ? H : o;
}
// (A1, H1) then (A2, H2)
template <bool SEG>
__device__ __forceinline__ void compose(float& A1, float& H1, float A2, float H2) {
  H1 = through<SEG>(A2, H2, H1);
  A1 = SEG && dropped(A2) ? A2 : A1 * A2;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster(unsigned addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// ---------------------------------------------------------------- forward
template <typename T, int VEC, bool SEG>
__global__ void __launch_bounds__(kGatedWarps * 32) gated_fwd_kernel(const __grid_constant__ GatedParams p) {
  using P = Pack<T, VEC>;
  constexpr int K = kFwdK, NW = kGatedWarps, TILE = K * NW;
  __shared__ float s_map[2][NW][2 * VEC][32];                 // (A, H) per warp, lane and channel
  __shared__ float s_cta[2][kGatedMaxCluster][2 * VEC][32];   // and per CTA of the cluster
  __shared__ float s_carry[2][VEC][32];                       // one CTA: the state leaving its tile
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int cs = p.cluster, rank = (int)(blockIdx.x % (unsigned)cs);
  const unsigned id = blockIdx.x / (unsigned)cs;
  const int ch = ((int)(id % (unsigned)p.groups) * 32 + lane) * VEC;
  const bool on = ch < p.D;
  const long long tiles = (p.L + TILE - 1) / TILE, steps = (tiles + cs - 1) / cs;
  float nu[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) nu[v] = on ? gated_minus_nu(p.nu_log[ch + v]) : 0.0f;
  if (cs > 1) cluster_barrier();  // every CTA of the cluster has started before its memory is written
  int par = 0;

  for (long long bt = id / (unsigned)p.groups; bt < p.B; bt += p.rows) {
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = on && p.h0 != nullptr ? p.h0[bt * p.D + ch + v] : 0.0f;
    if (cs == 1 && wp == NW - 1) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) s_carry[par ^ 1][v][lane] = carry[v];
    }
    typename P::type rx[K], rr[K], rw[K];
    unsigned seg = 0;  // bit k: token k starts a segment
    auto fetch = [&](long long step) {
      const long long t0 = (step * cs + rank) * TILE + wp * K;
      seg = 0;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const long long t = t0 + k;
        if (on && t < p.L) {
          rx[k] = gated_load<T, VEC>(p.x, bt, t, ch);
          rr[k] = gated_load<T, VEC>(p.r, bt, t, ch);
          rw[k] = gated_load<T, VEC>(p.w, bt, t, ch);
        }
        if (SEG && t < p.L && gated_starts(p.pos, p.pos_bytes, bt * p.L + t)) seg |= 1u << k;
      }
    };
    fetch(0);
    for (long long step = 0; step < steps; ++step, par ^= 1) {
      const long long t0 = (step * cs + rank) * TILE + wp * K;
      float a[K][VEC], b[K][VEC], A[VEC], H[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) A[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const bool live = on && t0 + k < p.L;
        float x[VEC], r[VEC], w[VEC];
        P::get(rx[k], x);
        P::get(rr[k], r);
        P::get(rw[k], w);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          gated_ab<T>(x[v], r[v], w[v], nu[v], &a[k][v], &b[k][v]);
          if (SEG && (seg >> k & 1u)) a[k][v] = -0.0f;
          if (!live) a[k][v] = 1.0f, b[k][v] = 0.0f;
          compose<SEG>(A[v], H[v], a[k][v], b[k][v]);
        }
      }
      if (step + 1 < steps) fetch(step + 1);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s_map[par][wp][2 * v][lane] = A[v];
        s_map[par][wp][2 * v + 1][lane] = H[v];
      }
      __syncthreads();
      float PA[VEC], PH[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) PA[v] = 1.0f, PH[v] = 0.0f;
      for (int j = 0; j < wp; ++j) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          compose<SEG>(PA[v], PH[v], s_map[par][j][2 * v][lane], s_map[par][j][2 * v + 1][lane]);
      }
      float in[VEC];  // the state entering this CTA's tile
      if (cs > 1) {
        if (wp == NW - 1) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            float TA = PA[v], TH = PH[v];
            compose<SEG>(TA, TH, A[v], H[v]);
            for (int q = 0; q < cs; ++q) {
              st_cluster(cluster_smem_addr(&s_cta[par][rank][2 * v][lane], q), TA);
              st_cluster(cluster_smem_addr(&s_cta[par][rank][2 * v + 1][lane], q), TH);
            }
          }
        }
        cluster_barrier();
#pragma unroll
        for (int v = 0; v < VEC; ++v) in[v] = carry[v];
        for (int q = 0; q < cs; ++q) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            if (q == rank) in[v] = carry[v];
            carry[v] = through<SEG>(s_cta[par][q][2 * v][lane], s_cta[par][q][2 * v + 1][lane], carry[v]);
          }
        }
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) in[v] = s_carry[par ^ 1][v][lane];
      }
      float h[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = through<SEG>(PA[v], PH[v], in[v]);
      if (p.carry != nullptr && on && t0 % kGatedChunk == 0 && t0 < p.L) {
        const long long c = (bt * p.chunks + t0 / kGatedChunk) * p.D + ch;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.carry[c + v] = h[v];
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = through<SEG>(a[k][v], b[k][v], h[v]);
        const long long t = t0 + k;
        if (on && t < p.L) {
          *reinterpret_cast<typename P::type*>(static_cast<T*>(p.y) + (bt * p.L + t) * p.D + ch) = P::make(h);
          if (t == p.L - 1 && p.last != nullptr) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) p.last[bt * p.D + ch + v] = h[v];
          }
        }
      }
      if (cs == 1 && wp == NW - 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) s_carry[par][v][lane] = h[v];
      }
    }
  }
}

// ---------------------------------------------------------------- backward
template <typename T, int VEC, bool SEG>
__global__ void __launch_bounds__(kGatedWarps * 32) gated_bwd_kernel(const __grid_constant__ GatedParams p) {
  using P = Pack<T, VEC>;
  constexpr int K = kBwdK, NW = kGatedWarps, TILE = K * NW;
  // per warp: A, H (states, forward) and G (adjoints, reverse: out = A in + G)
  __shared__ float s_map[2][NW][3 * VEC][32];
  __shared__ float s_cta[2][kGatedMaxCluster][2 * VEC][32];  // (A, G) per CTA of the cluster
  __shared__ float s_adj[2][VEC][32];                        // one CTA: the adjoint leaving its tile
  __shared__ double s_nu[NW][VEC][32];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int cs = p.cluster, rank = (int)(blockIdx.x % (unsigned)cs);
  const unsigned id = blockIdx.x / (unsigned)cs;
  const int ch = ((int)(id % (unsigned)p.groups) * 32 + lane) * VEC;
  const bool on = ch < p.D;
  const long long tiles = p.chunks, steps = (tiles + cs - 1) / cs;
  float nu[VEC];
  double dnu[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    nu[v] = on ? gated_minus_nu(p.nu_log[ch + v]) : 0.0f;
    dnu[v] = 0.0;
  }
  if (cs > 1) cluster_barrier();
  int par = 0;

  for (long long bt = id / (unsigned)p.groups; bt < p.B; bt += p.rows) {
    float adj[VEC];  // c_{t+1} lam_{t+1} entering the step's last token
#pragma unroll
    for (int v = 0; v < VEC; ++v) adj[v] = on && p.grad_last != nullptr ? p.grad_last[bt * p.D + ch + v] : 0.0f;
    if (cs == 1 && wp == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) s_adj[par ^ 1][v][lane] = adj[v];
    }
    typename P::type rx[K], rr[K], rw[K], rd[K];
    float hc[VEC];
    unsigned seg = 0;
    auto fetch = [&](long long step) {
      const long long tile = step * cs + rank, t0 = tile * TILE + wp * K;
      seg = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        hc[v] = on && tile < tiles ? p.carry[(bt * p.chunks + tile) * p.D + ch + v] : 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const long long t = t0 + k;
        if (on && t < p.L) {
          rx[k] = gated_load<T, VEC>(p.x, bt, t, ch);
          rr[k] = gated_load<T, VEC>(p.r, bt, t, ch);
          rw[k] = gated_load<T, VEC>(p.w, bt, t, ch);
          rd[k] = gated_load<T, VEC>(p.dy, bt, t, ch);
        }
        if (SEG && t < p.L && gated_starts(p.pos, p.pos_bytes, bt * p.L + t)) seg |= 1u << k;
      }
    };
    fetch(steps - 1);
    for (long long step = steps - 1; step >= 0; --step, par ^= 1) {
      const long long t0 = (step * cs + rank) * TILE + wp * K;
      // a; g; b = g x; bw = b (1 - s(write)); q1 = -a u; q2 = x s(write) a^2 u / sqrt(1 - a^2);
      // omr = 1 - s(retention); d = dy
      float a[K][VEC], g[K][VEC], b[K][VEC], bw[K][VEC], q1[K][VEC], q2[K][VEC], omr[K][VEC], d[K][VEC];
      float A[VEC], H[VEC], G[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) A[v] = 1.0f, H[v] = 0.0f, G[v] = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const bool live = on && t0 + k < p.L;
        float x[VEC], r[VEC], w[VEC];
        P::get(rx[k], x);
        P::get(rr[k], r);
        P::get(rw[k], w);
        P::get(rd[k], d[k]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float er = exp_neg<T>(r[v]), ew = exp_neg<T>(w[v]);
          const float sr = rcp_approx(1.0f + er), sw = rcp_approx(1.0f + ew);
          const float u = nu[v] * sr;
          const float2 e = exp_expm1_neg(u);
          const float av = e.x, m = -e.y * (2.0f + e.y);
          const float rs = rsqrt_approx(fmaxf(m, 1.17549435e-38f));
          const float xs = x[v] * sw;
          a[k][v] = av;
          g[k][v] = m * rs * sw;
          b[k][v] = m * rs * xs;
          bw[k][v] = b[k][v] * one_minus_s(ew, sw);
          q1[k][v] = av * -u;  // >= +0, as a
          q2[k][v] = xs * (av * av) * (u * rs);
          omr[k][v] = one_minus_s(er, sr);
          if (SEG && (seg >> k & 1u)) a[k][v] = -0.0f, q1[k][v] = -0.0f;
          if (!live) a[k][v] = 1.0f, b[k][v] = 0.0f, d[k][v] = 0.0f;
          compose<SEG>(A[v], H[v], a[k][v], b[k][v]);
        }
      }
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) G[v] = through<SEG>(a[k][v], 0.0f, d[k][v] + G[v]);
      }
      float h[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = hc[v];
      if (step > 0) fetch(step - 1);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s_map[par][wp][3 * v][lane] = A[v];
        s_map[par][wp][3 * v + 1][lane] = H[v];
        s_map[par][wp][3 * v + 2][lane] = G[v];
      }
      __syncthreads();
      // the state entering this warp's tokens, from the chunk's carry through the warps before
      for (int j = 0; j < wp; ++j) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          h[v] = through<SEG>(s_map[par][j][3 * v][lane], s_map[par][j][3 * v + 1][lane], h[v]);
      }
      // the map of the adjoint through the warps behind
      float PA[VEC], PG[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) PA[v] = 1.0f, PG[v] = 0.0f;
      for (int j = NW - 1; j > wp; --j) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          compose<SEG>(PA[v], PG[v], s_map[par][j][3 * v][lane], s_map[par][j][3 * v + 2][lane]);
      }
      float c[VEC];
      if (cs > 1) {
        if (wp == 0) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            float TA = PA[v], TG = PG[v];
            compose<SEG>(TA, TG, A[v], G[v]);
            for (int q = 0; q < cs; ++q) {
              st_cluster(cluster_smem_addr(&s_cta[par][rank][2 * v][lane], q), TA);
              st_cluster(cluster_smem_addr(&s_cta[par][rank][2 * v + 1][lane], q), TG);
            }
          }
        }
        cluster_barrier();
#pragma unroll
        for (int v = 0; v < VEC; ++v) c[v] = adj[v];
        for (int q = cs - 1; q >= 0; --q) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            if (q == rank) c[v] = adj[v];
            adj[v] = through<SEG>(s_cta[par][q][2 * v][lane], s_cta[par][q][2 * v + 1][lane], adj[v]);
          }
        }
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) c[v] = s_adj[par ^ 1][v][lane];
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) c[v] = through<SEG>(PA[v], PG[v], c[v]);
      // states forward: q1 <- q1 h_{t-1} + q2 = -du u / lam
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          q1[k][v] = through<SEG>(q1[k][v], q2[k][v], h[v]);
          h[v] = through<SEG>(a[k][v], b[k][v], h[v]);
        }
      }
      // adjoints in reverse
      float sum[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) sum[v] = 0.0f;
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
        const long long t = t0 + k;
        const bool live = on && t < p.L;
        float ox[VEC], orr[VEC], ow[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float lam = d[k][v] + c[v];
          const float du = -lam * q1[k][v];  // du u
          ox[v] = lam * g[k][v];
          ow[v] = lam * bw[k][v];
          orr[v] = du * omr[k][v];
          if (live) sum[v] += du;
          c[v] = through<SEG>(a[k][v], 0.0f, lam);
        }
        if (live) {
          const long long i = (bt * p.L + t) * p.D + ch;
          *reinterpret_cast<typename P::type*>(static_cast<T*>(p.dx) + i) = P::make(ox);
          *reinterpret_cast<typename P::type*>(static_cast<T*>(p.dr) + i) = P::make(orr);
          *reinterpret_cast<typename P::type*>(static_cast<T*>(p.dw) + i) = P::make(ow);
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) dnu[v] += (double)sum[v];
      if (wp == 0) {
        if (cs == 1) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) s_adj[par][v][lane] = c[v];
        }
        if (t0 == 0 && on && p.grad_h0 != nullptr) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) p.grad_h0[bt * p.D + ch + v] = c[v];
        }
      }
    }
  }
  // the CTA's sum of dnu_log per channel, over its warps in order
#pragma unroll
  for (int v = 0; v < VEC; ++v) s_nu[wp][v][lane] = dnu[v];
  __syncthreads();
  if (wp == 0 && on) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      double s = 0.0;
      for (int j = 0; j < NW; ++j) s += s_nu[j][v][lane];
      p.part[((long long)(id / (unsigned)p.groups) * cs + rank) * p.D + ch + v] = s;
    }
  }
}

// dnu_log[d] = the sum of the partial rows, in order: a warp's lanes own 32 channels, the block's
// warps every kGatedWarps-th row, then warp 0 adds the warps' sums.
__global__ void __launch_bounds__(kGatedWarps * 32) gated_reduce_kernel(const double* part, float* out, int rows, int D) {
  __shared__ double s[kGatedWarps][32];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  double t = 0.0;
  if (d < D)
    for (int r = wp; r < rows; r += kGatedWarps) t += part[(long long)r * D + d];
  s[wp][lane] = t;
  __syncthreads();
  if (wp == 0 && d < D) {
    for (int j = 1; j < kGatedWarps; ++j) t += s[j][lane];
    out[d] = (float)t;
  }
}

// ---------------------------------------------------------------- one decode step
struct GatedStepParams {
  const void *x, *r, *w;       // [B, D], row strides in elements
  long long sx, sr, sw;
  const float *nu_log, *state; // [D], [B, D]
  const void* pos;             // [B] or null
  int pos_bytes;
  void* y;                     // [B, D]
  float* new_state;            // [B, D]
  long long B;
  int D;
};

template <typename T>
__global__ void __launch_bounds__(128) gated_step_kernel(const GatedStepParams p) {
  const int d = blockIdx.x * 128 + threadIdx.x;
  if (d >= p.D) return;
  const float nu = gated_minus_nu(__ldg(p.nu_log + d));
  for (long long b = blockIdx.y; b < p.B; b += gridDim.y) {
    const float x = Io<T>::load(static_cast<const T*>(p.x) + b * p.sx + d);
    const float r = Io<T>::load(static_cast<const T*>(p.r) + b * p.sr + d);
    const float w = Io<T>::load(static_cast<const T*>(p.w) + b * p.sw + d);
    const float s = p.state[b * p.D + d];
    float a, c;
    gated_ab<T>(x, r, w, nu, &a, &c);
    const bool start = p.pos != nullptr && gated_starts(p.pos, p.pos_bytes, b);
    const float h = start ? c : fmaf(a, s, c);
    Io<T>::store(static_cast<T*>(p.y) + b * p.D + d, h);
    p.new_state[b * p.D + d] = h;
  }
}

// ---------------------------------------------------------------- host
struct GatedPlan {
  int vec, groups, cluster, rows;
};

// Channels two per lane where sizes and strides allow it. The cluster grows (to the portable 8
// CTAs, no further than the tiles reach) until rows x channel groups x cluster fills the SMs four
// CTAs each; more rows than a few waves of CTAs need are walked by the same clusters, which
// bounds the partial sums.
static GatedPlan gated_plan(long long B, long long L, long long D, bool pairs, int tile) {
  constexpr long long kFill = 148 * 4, kMost = kFill * 4;
  GatedPlan pl;
  pl.vec = pairs ? 2 : 1;
  pl.groups = (int)((D + 32 * pl.vec - 1) / (32 * pl.vec));
  const long long tiles = (L + tile - 1) / tile;
  pl.cluster = 1;
  while (pl.cluster < kGatedMaxCluster && pl.cluster * 2 <= tiles && B * pl.groups * pl.cluster < kFill) pl.cluster *= 2;
  const long long rows = std::max(1LL, kMost / ((long long)pl.groups * pl.cluster));
  pl.rows = (int)std::min(B, rows);
  return pl;
}

static bool gated_valid_dtype(int d) { return d == SPARC_DTYPE_F32 || d == SPARC_DTYPE_BF16; }

static int gated_check_shape(long long B, long long L, long long D) {
  if (B <= 0 || L <= 0 || D <= 0) return fail(SPARC_ERR_SHAPE, "batch, length and channels must be positive");
  if (D > (1LL << 24) || B > (1LL << 31) || L > (1LL << 40) || (double)B * (double)L * (double)D > 4.0e18)
    return fail(SPARC_ERR_SHAPE, "shape beyond the launch grid (channels <= 2^24, batch <= 2^31)");
  return SPARC_OK;
}

static bool gated_pos_ok(const void* pos, int bytes) {
  return pos == nullptr || bytes == 1 || bytes == 2 || bytes == 4 || bytes == 8;
}

static bool gated_pairs(const GatedIn& in, long long B, long long L, int size) {
  return reinterpret_cast<uintptr_t>(in.p) % (2 * size) == 0 && (B <= 1 || in.sb % 2 == 0) &&
         (L <= 1 || in.st % 2 == 0);
}
static bool gated_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T, int VEC, bool SEG>
static cudaError_t gated_launch(const GatedParams& p, bool backward, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.groups * (unsigned)p.rows * (unsigned)p.cluster);
  cfg.blockDim = dim3(kGatedWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  TimedLaunch tl(backward ? kTimeGatedBwd : kTimeGatedFwd, s);
  return backward ? cudaLaunchKernelEx(&cfg, gated_bwd_kernel<T, VEC, SEG>, p)
                  : cudaLaunchKernelEx(&cfg, gated_fwd_kernel<T, VEC, SEG>, p);
}

template <typename T>
static cudaError_t gated_dispatch(const GatedParams& p, int vec, bool backward, cudaStream_t s) {
  if (p.pos != nullptr)
    return vec == 2 ? gated_launch<T, 2, true>(p, backward, s) : gated_launch<T, 1, true>(p, backward, s);
  return vec == 2 ? gated_launch<T, 2, false>(p, backward, s) : gated_launch<T, 1, false>(p, backward, s);
}

static size_t gated_ws_bytes(long long B, long long L, long long D) {
  size_t rows = 0;  // whichever way the strides let the channels be read
  for (int pairs = 0; pairs < 2; ++pairs) {
    const GatedPlan pl = gated_plan(B, L, D, pairs != 0, kGatedChunk);
    rows = std::max(rows, (size_t)pl.rows * (size_t)pl.cluster);
  }
  return rows * (size_t)D * sizeof(double);
}

}  // namespace sparc

using namespace sparc;

extern "C" {

long long sparc_gated_chunk_tokens(void) { return kGatedChunk; }
long long sparc_gated_carry_chunks(long long length) {
  return length <= 0 ? 0 : (length - 1) / kGatedChunk + 1;
}

size_t sparc_gated_workspace_bytes(long long batch, long long length, long long channels) {
  if (gated_check_shape(batch, length, channels) != SPARC_OK) return 0;
  return gated_ws_bytes(batch, length, channels);
}

int sparc_gated_scan_forward(const SparcGatedFwdArgs* a, void* stream) {
  NvtxRange nvtx(__func__);
  if (a == nullptr) return fail(SPARC_ERR_ARG, "null args");
  if (!a->x || !a->retention_gate || !a->write_gate || !a->nu_log || !a->y)
    return fail(SPARC_ERR_ARG, "null tensor pointer");
  const int rc = gated_check_shape(a->batch, a->length, a->channels);
  if (rc != SPARC_OK) return rc;
  if (!gated_valid_dtype(a->dtype)) return fail(SPARC_ERR_DTYPE, "unsupported dtype");
  if (!gated_pos_ok(a->segment_pos, a->segment_pos_bytes))
    return fail(SPARC_ERR_ARG, "segment_pos_bytes must be 1, 2, 4 or 8");
  GatedParams p = {};
  p.x = GatedIn{a->x, a->x_batch_stride, a->x_token_stride};
  p.r = GatedIn{a->retention_gate, a->retention_batch_stride, a->retention_token_stride};
  p.w = GatedIn{a->write_gate, a->write_batch_stride, a->write_token_stride};
  p.y = a->y;
  p.nu_log = a->nu_log;
  p.h0 = a->h0;
  p.last = a->last;
  p.carry = a->carry;
  p.pos = a->segment_pos;
  p.pos_bytes = a->segment_pos_bytes;
  p.B = a->batch;
  p.L = a->length;
  p.D = (int)a->channels;
  p.chunks = sparc_gated_carry_chunks(a->length);
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  for (const void* q : {a->x, a->retention_gate, a->write_gate, (const void*)a->y})
    if (!gated_aligned(q, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
  const bool pairs = p.D % 2 == 0 && gated_pairs(p.x, p.B, p.L, size) && gated_pairs(p.r, p.B, p.L, size) &&
                     gated_pairs(p.w, p.B, p.L, size) && gated_aligned(p.y, 2 * size);
  const GatedPlan pl = gated_plan(p.B, p.L, p.D, pairs, kFwdK * kGatedWarps);
  p.groups = pl.groups;
  p.cluster = pl.cluster;
  p.rows = pl.rows;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == SPARC_DTYPE_BF16 ? gated_dispatch<__nv_bfloat16>(p, pl.vec, false, s)
                                                     : gated_dispatch<float>(p, pl.vec, false, s);
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

int sparc_gated_scan_backward(const SparcGatedBwdArgs* a, void* stream) {
  NvtxRange nvtx(__func__);
  if (a == nullptr) return fail(SPARC_ERR_ARG, "null args");
  if (!a->x || !a->retention_gate || !a->write_gate || !a->nu_log || !a->dy || !a->carry || !a->grad_x ||
      !a->grad_retention_gate || !a->grad_write_gate || !a->grad_nu_log)
    return fail(SPARC_ERR_ARG, "null tensor pointer");
  const int rc = gated_check_shape(a->batch, a->length, a->channels);
  if (rc != SPARC_OK) return rc;
  if (!gated_valid_dtype(a->dtype)) return fail(SPARC_ERR_DTYPE, "unsupported dtype");
  if (!gated_pos_ok(a->segment_pos, a->segment_pos_bytes))
    return fail(SPARC_ERR_ARG, "segment_pos_bytes must be 1, 2, 4 or 8");
  if (a->workspace == nullptr || !gated_aligned(a->workspace, 8) ||
      a->workspace_bytes < gated_ws_bytes(a->batch, a->length, a->channels))
    return fail(SPARC_ERR_WORKSPACE, "workspace missing, too small or not 8-byte aligned");
  GatedParams p = {};
  p.x = GatedIn{a->x, a->x_batch_stride, a->x_token_stride};
  p.r = GatedIn{a->retention_gate, a->retention_batch_stride, a->retention_token_stride};
  p.w = GatedIn{a->write_gate, a->write_batch_stride, a->write_token_stride};
  p.dy = GatedIn{a->dy, a->dy_batch_stride, a->dy_token_stride};
  p.dx = a->grad_x;
  p.dr = a->grad_retention_gate;
  p.dw = a->grad_write_gate;
  p.nu_log = a->nu_log;
  p.carry = const_cast<float*>(a->carry);
  p.grad_last = a->grad_last;
  p.grad_h0 = a->grad_h0;
  p.part = static_cast<double*>(a->workspace);
  p.pos = a->segment_pos;
  p.pos_bytes = a->segment_pos_bytes;
  p.B = a->batch;
  p.L = a->length;
  p.D = (int)a->channels;
  p.chunks = sparc_gated_carry_chunks(a->length);
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  bool pairs = p.D % 2 == 0;
  for (const GatedIn* in : {&p.x, &p.r, &p.w, &p.dy}) {
    if (!gated_aligned(in->p, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
    pairs = pairs && gated_pairs(*in, p.B, p.L, size);
  }
  for (const void* q : {p.dx, p.dr, p.dw}) {
    if (!gated_aligned(q, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
    pairs = pairs && gated_aligned(q, 2 * size);
  }
  const GatedPlan pl = gated_plan(p.B, p.L, p.D, pairs, kGatedChunk);
  p.groups = pl.groups;
  p.cluster = pl.cluster;
  p.rows = pl.rows;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = a->dtype == SPARC_DTYPE_BF16 ? gated_dispatch<__nv_bfloat16>(p, pl.vec, true, s)
                                               : gated_dispatch<float>(p, pl.vec, true, s);
  if (e == cudaSuccess) {
    TimedLaunch tl(kTimeGatedReduce, s);
    gated_reduce_kernel<<<(p.D + 31) / 32, kGatedWarps * 32, 0, s>>>(p.part, a->grad_nu_log, pl.rows * pl.cluster, p.D);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

int sparc_gated_step(const SparcGatedStepArgs* a, void* stream) {
  NvtxRange nvtx(__func__);
  if (a == nullptr) return fail(SPARC_ERR_ARG, "null args");
  if (!a->x || !a->retention_gate || !a->write_gate || !a->nu_log || !a->state || !a->y || !a->new_state)
    return fail(SPARC_ERR_ARG, "null tensor pointer");
  const int rc = gated_check_shape(a->batch, 1, a->channels);
  if (rc != SPARC_OK) return rc;
  if (!gated_valid_dtype(a->dtype)) return fail(SPARC_ERR_DTYPE, "unsupported dtype");
  if (!gated_pos_ok(a->segment_pos, a->segment_pos_bytes))
    return fail(SPARC_ERR_ARG, "segment_pos_bytes must be 1, 2, 4 or 8");
  GatedStepParams p = {};
  p.x = a->x;
  p.r = a->retention_gate;
  p.w = a->write_gate;
  p.sx = a->x_stride;
  p.sr = a->retention_stride;
  p.sw = a->write_stride;
  p.nu_log = a->nu_log;
  p.state = a->state;
  p.pos = a->segment_pos;
  p.pos_bytes = a->segment_pos_bytes;
  p.y = a->y;
  p.new_state = a->new_state;
  p.B = a->batch;
  p.D = (int)a->channels;
  const dim3 grid((unsigned)((p.D + 127) / 128), (unsigned)std::min<long long>(p.B, 32768));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  TimedLaunch tl(kTimeGatedStep, s);
  if (a->dtype == SPARC_DTYPE_BF16)
    gated_step_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else
    gated_step_kernel<float><<<grid, 128, 0, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

}  // extern "C"
