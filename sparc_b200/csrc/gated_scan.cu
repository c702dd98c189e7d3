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
// Decomposition: one launch each way, every tensor read once and written once. A lane owns two
// adjacent channels (packed f32x2 arithmetic) and a warp K consecutive tokens; a CTA's eight warps
// own consecutive spans of K tokens (a tile), and a thread-block cluster's CTAs consecutive tiles;
// the cluster walks the sequence. A thread turns its K tokens into an affine map (A, H): h_out =
// A h_in + H in registers; after one barrier every warp runs the state through the maps of the
// warps before it (and, over distributed shared memory, through those of the cluster's CTAs before
// its own), and replays its tokens from there. The backward does
// both directions in one step: the states from the forward's saved chunk carries (float32, one
// per kGatedChunk tokens, so that the states are not rounded to the activations' type), the
// adjoints from the step before. The cluster size grows as rows x channels shrink. All orders are
// fixed: results are bitwise reproducible. Each warp copies its own tokens to shared memory
// asynchronously, one or two steps ahead (into the place whose values it has just taken into registers),
// so nothing but the copies' own completion orders them.
//
// A segment start drops what came before it, infinities and NaN included: its factor is kept as
// -0 (a_t >= +0 or NaN, so the sign marks it; composing keeps the sign of either side), and passing
// through it selects instead of multiplying.
//
// Measured on a B200 (B=8 T=16384 D=2048 bfloat16, 268M channels x tokens): forward 480 us = 4.5 TB/s
// of its 8 bytes each (68% of what a copy reaches), backward 879 us = 4.3 TB/s of 14 bytes (65%). Neither
// bytes nor any one unit bounds them but the latency of a step's chain (gates, barrier, maps, replay), which
// the 7-16 warps an SM holds (128 and 162 registers) do not cover: their 34 and 60 thread-instructions an
// element issue on 53-55% of the cycles; more warps at fewer registers issue
// more instructions and were slower (backward with 128 registers: 1033 us with eight warps a CTA,
// 1298 us with four CTAs). A copy in the same pattern (128-byte pieces of a token) takes 330-350 and
// 650-680 us. float32 (B=8 T=2048 D=512): 30 and 46 us, of floors 20 and 36.
#include <algorithm>

#include "common.cuh"
#include "sparc_b200.h"
#include "timing.cuh"

namespace sparc {

constexpr int kGatedChunk = 32;       // tokens per saved carry
constexpr int kGatedMaxCluster = 16;  // (above 8 a kernel has to allow it)
constexpr unsigned kGatedSpin = 1u << 22;  // default bound of a wait's polls (each may sleep in hardware)
constexpr unsigned kGatedDrain = 1u << 12;  // and of the wait on the way out for stores that have been issued

// How a CTA cuts its tile: WARPS spans of K tokens; BLOCKS CTAs per SM that the registers are held to;
// STAGES steps of inputs on their way.
template <int K_, int WARPS_, int BLOCKS_, int STAGES_>
struct GatedCut {
  static constexpr int K = K_, WARPS = WARPS_, BLOCKS = BLOCKS_, STAGES = STAGES_, TILE = K * WARPS;
};
template <typename T> struct GatedFwdCut;
template <> struct GatedFwdCut<__nv_bfloat16> : GatedCut<16, 4, 4, 1> {};
template <> struct GatedFwdCut<float> : GatedCut<8, 8, 2, 1> {};
template <typename T> struct GatedBwdCut;
template <> struct GatedBwdCut<__nv_bfloat16> : GatedCut<8, 4, 3, 2> {};
template <> struct GatedBwdCut<float> : GatedCut<8, 4, 2, 2> {};
// some warp's tokens begin each chunk
template <typename C> constexpr bool kGatedWhole = C::TILE % kGatedChunk == 0 && kGatedChunk % C::K == 0;
static_assert(kGatedWhole<GatedFwdCut<float>> && kGatedWhole<GatedFwdCut<__nv_bfloat16>> &&
              kGatedWhole<GatedBwdCut<float>> && kGatedWhole<GatedBwdCut<__nv_bfloat16>>);

struct GatedIn {
  const void* p;
  long long sb, st;  // batch and token strides in elements (channels adjacent)
};

struct GatedParams {
  GatedIn in[4];       // x, retention gate, write gate; backward: dy
  void* y;             // [B, L, D] (forward)
  void *dx, *dr, *dw;  // [B, L, D] (backward)
  const float* nu_log; // [D]
  const float* h0;     // [B, D] or null
  float* last;         // [B, D] or null
  float* carry;        // [B, chunks, D]: the state entering each chunk, or null (forward)
  const float* grad_last;  // [B, D] or null
  float* grad_h0;      // [B, D] or null
  double* part;        // [rows * cluster, D] partial sums of dnu_log
  const void* pos;     // segment positions [B, L] or null
  int pos_bytes;
  long long B;
  int L, chunks;
  int D, groups, cluster, rows;  // rows: clusters per channel group, each walking rows of the batch
  unsigned max_spin;             // polls of a wait for the cluster's maps
  unsigned* status;              // or'ed with kStatusTimeout where one ran out, or null
  unsigned withhold;             // tests: the step (from 1) at which a cluster's last CTA pushes nothing, or 0
};

// ---------------------------------------------------------------- two adjacent channels
template <typename T> struct Duo;
template <> struct Duo<float> {
  using type = float2;
  static __device__ __forceinline__ float2 get(float2 v) { return v; }
  static __device__ __forceinline__ float2 make(float2 v) { return v; }
};
template <> struct Duo<__nv_bfloat16> {
  using type = unsigned;
  static __device__ __forceinline__ float2 get(unsigned v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ unsigned make(float2 v) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned*>(&b);
  }
};

__device__ __forceinline__ bool gated_starts(const void* pos, int bytes, long long i) {
  switch (bytes) {
    case 1: return __ldg(static_cast<const unsigned char*>(pos) + i) == 0;
    case 2: return __ldg(static_cast<const unsigned short*>(pos) + i) == 0;
    case 4: return __ldg(static_cast<const unsigned*>(pos) + i) == 0;
    default: return __ldg(static_cast<const unsigned long long*>(pos) + i) == 0;
  }
}

// How a warp reads its tokens, copied to shared memory ahead of their use: in pieces of 16 bytes, of
// one pair of channels, or (odd widths, strides or bases) in the aligned 16-byte pieces that hold the
// token's channels, from the middle of which the lanes then read.
enum GatedMode { kModeWide, kModePair, kModeSingle };

template <int BYTES>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {  // for all but the last N groups
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's reads of its next tokens: K of them a step, of NT tensors, into stage[tensor][token][lane].
// What lies beyond the sequence or the channels is not copied: those values are never used.
// Each lane owns pieces kRows tokens apart, and keeps a pointer per tensor that moves by a constant
// from step to step (with single elements the warp's pointers are of the tokens' first channel).
template <typename T, int MODE, int K, int NT, int S>
struct GatedReader {
  using R = typename Duo<T>::type;
  static constexpr int kBytes = MODE == kModeWide ? 16 : (int)sizeof(R);
  static constexpr int kPieces = 32 * (int)sizeof(R) / kBytes;  // of a token
  static constexpr int kRows = MODE == kModeSingle ? 1 : 32 / kPieces;
  static constexpr int kWindow = 64 * (int)sizeof(T) / 16 + 1;                      // aligned pieces of an odd token
  static constexpr int kRowBytes = MODE == kModeSingle ? kWindow * 16 : 32 * (int)sizeof(R);  // of a token in the stage
  const char* src[NT];
  long long row[NT], move[NT];  // bytes from a piece to the next, from a step to the next
  R* stage;
  unsigned dst;  // this lane's first piece in the stage
  int token;     // and its token of the step (none of this lane's where its channels are beyond D)
  int bytes;     // odd tokens: of the token's channels

  __device__ __forceinline__ GatedReader(const GatedParams& p, R* stage_, int ch0, int lane, int tokens) : stage(stage_) {
    const int chan = ch0 + lane % kPieces * (kBytes / (int)sizeof(T));
    token = chan < p.D ? lane / kPieces : K;
    bytes = min(64, p.D - ch0) * (int)sizeof(T);
    dst = smem_addr(stage) + (MODE == kModeSingle ? 0 : lane * kBytes);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      row[n] = kRows * p.in[n].st * (int)sizeof(T);
      move[n] = tokens * p.in[n].st * (int)sizeof(T);
    }
  }
  __device__ __forceinline__ void start(const GatedParams& p, long long bt, int t0, int ch0, int lane) {
    const int chan = MODE == kModeSingle ? ch0 : ch0 + lane % kPieces * (kBytes / (int)sizeof(T));
    const int t = MODE == kModeSingle ? t0 : t0 + lane / kPieces;
#pragma unroll
    for (int n = 0; n < NT; ++n)
      src[n] = reinterpret_cast<const char*>(static_cast<const T*>(p.in[n].p) + bt * p.in[n].sb + (long long)t * p.in[n].st + chan);
  }
  static constexpr int kStageBytes = NT * K * kRowBytes;

  // `left`: tokens of the sequence from this step's first on (none: an empty group, so that the groups count steps)
  __device__ __forceinline__ void copy(int slot, int left, int lane) {
    const unsigned to = dst + slot * kStageBytes;
    if constexpr (MODE == kModeSingle) {
      // (rolled: code that runs once is paid for in instruction fetches)
      const int some = min(K, left);
#pragma unroll 1
      for (int c = lane; c < some * kWindow; c += 32) {
        const int k = c / kWindow, at = c % kWindow * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const char* a = src[n] + k * row[n];
          const int off = (int)(reinterpret_cast<unsigned long long>(a) & 15u);
          if (at - off < bytes) copy_async<16>(to + n * K * kRowBytes + c * 16, a - off + at);
        }
      }
    } else if (left >= K) {
      if (token < K) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < K / kRows; ++i)
            copy_async<kBytes>(to + (n * K + i * kRows) * 32 * (int)sizeof(R), src[n] + i * row[n]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < K / kRows; ++i)
          if (token < K && token + i * kRows < left)
            copy_async<kBytes>(to + (n * K + i * kRows) * 32 * (int)sizeof(R), src[n] + i * row[n]);
    }
    copy_commit();
#pragma unroll
    for (int n = 0; n < NT; ++n) src[n] += move[n];
  }
  // tokens k0 .. k0 + N - 1 of tensor n of the step in `slot`, the first of the S that are on their way, once it has come
  template <int N>
  __device__ __forceinline__ void read(int slot, int n, int k0, int lane, R (&v)[N]) const {
    const char* q = reinterpret_cast<const char*>(stage) + slot * kStageBytes + (n * K + k0) * kRowBytes + lane * (int)sizeof(R);
    const unsigned step = (unsigned)row[n], first = (unsigned)reinterpret_cast<unsigned long long>(src[n] - S * move[n]) + k0 * step;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const char* w = q + k * kRowBytes;
      if constexpr (MODE != kModeSingle) {
        v[k] = *reinterpret_cast<const R*>(w);
      } else {
        const unsigned off = first + k * step & 15u;  // where the token begins in its first piece
        if constexpr (sizeof(T) == 2) {
          const unsigned* u = reinterpret_cast<const unsigned*>(w + (off & ~3u));
          v[k] = off & 2u ? __funnelshift_r(u[0], u[1], 16) : u[0];
        } else {
          const float* f = reinterpret_cast<const float*>(w + off);
          v[k] = make_float2(f[0], f[1]);
        }
      }
    }
  }
};

template <typename T, int MODE>
__device__ __forceinline__ void gated_store(T* o, int ch, int D, float2 v) {
  if constexpr (MODE != kModeSingle) {
    *reinterpret_cast<typename Duo<T>::type*>(o) = Duo<T>::make(v);
  } else {
    Io<T>::store(o, v.x);
    if (ch + 1 < D) Io<T>::store(o + 1, v.y);
  }
}

// float32 pairs of a [.., D] array
__device__ __forceinline__ float2 load_pair(const float* a, long long i, int ch, int D) {
  return make_float2(a != nullptr && ch < D ? a[i] : 0.0f, a != nullptr && ch + 1 < D ? a[i + 1] : 0.0f);
}
__device__ __forceinline__ void store_pair(float* a, long long i, int ch, int D, float2 v) {
  if (ch < D) a[i] = v.x;
  if (ch + 1 < D) a[i + 1] = v.y;
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
__device__ __forceinline__ float2 neg2(float2 v) { return make_float2(-v.x, -v.y); }

// The functions below take N tokens' pairs at once, an operation after the other over all of them:
// a constant of packed arithmetic is a pair of registers that two moves set, which N tokens share.

// e^{-v}. float32: the product with log2 e is carried in two terms (its rounding alone would cost
// |v| 2^-24 in the result), with v held to +-88 so that both stay finite; 1 / (1 + e^88) flushes
// to the exact 0 that s(-inf) is.
template <typename T, int N>
__device__ __forceinline__ void exp_neg(const float2 (&v)[N], float2 (&e)[N]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = mul2(v[k], bcast2(-kLog2e));
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = ex2_2(e[k]);
  } else {
    constexpr float kLog2eLo = 1.9259630e-8f;  // log2 e - kLog2e
    float2 lo[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float2 c = make_float2(min_nan(max_nan(v[k].x, -88.0f), 88.0f), min_nan(max_nan(v[k].y, -88.0f), 88.0f));
      const float2 t = mul2(c, bcast2(-kLog2e));
      lo[k] = mul2(fma2(c, bcast2(-kLog2eLo), fma2(c, bcast2(-kLog2e), neg2(t))), bcast2(0.6931471805599453f));
      e[k] = t;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = ex2_2(e[k]);
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = fma2(e[k], lo[k], e[k]);
  }
}
// s = 1 / (1 + e)
template <int N>
__device__ __forceinline__ void logistic_of(const float2 (&e)[N], float2 (&s)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = add2(e[k], bcast2(1.0f));
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = rcp_2(s[k]);
}

// For w = -u >= 0: a = e^{-w} and q = 1 - a. Below 1/2 from the series of q (through w^8 / 8!: the
// next term is below 2^-26 of the first), which keeps 1 - a^2 = q (1 + a) exact to a few ulp where
// a is near 1 and holds the decay of long sequences; else the hardware exp2 of w log2 e, rounded once: a's
// relative error grows with w, to about 1.2 w 2^-24 (at w = 40, where a = 4e-18, some 20 ulp). NEAR: nu <=
// 1/2 in every channel of the warp, so w never leaves the series.
constexpr float kGatedNear = 0.5f;
template <bool NEAR, int N>
__device__ __forceinline__ void decay(const float2 (&w)[N], float2 (&a)[N], float2 (&q)[N]) {
  constexpr float kSeries[6] = {1.9841269841269841e-4f,  -1.3888888888888889e-3f, 8.3333333333333333e-3f,
                                -4.1666666666666667e-2f, 1.6666666666666667e-1f,  -0.5f};  // 1/7! ... -1/2!
#pragma unroll
  for (int k = 0; k < N; ++k) q[k] = bcast2(-2.4801587301587302e-5f);  // -1/8!
#pragma unroll
  for (int i = 0; i < 6; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) q[k] = fma2(q[k], w[k], bcast2(kSeries[i]));
#pragma unroll
  for (int k = 0; k < N; ++k) q[k] = fma2(mul2(q[k], w[k]), w[k], w[k]);
#pragma unroll
  for (int k = 0; k < N; ++k) a[k] = sub2(bcast2(1.0f), q[k]);
  if constexpr (!NEAR) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float2 e = ex2_2(mul2(w[k], bcast2(-kLog2e))), f = sub2(bcast2(1.0f), e);
      const bool nx = w[k].x < kGatedNear, ny = w[k].y < kGatedNear;
      a[k] = make_float2(nx ? a[k].x : e.x, ny ? a[k].y : e.y);
      q[k] = make_float2(nx ? q[k].x : f.x, ny ? q[k].y : f.y);
    }
  }
}

// nu of a channel, held finite so that nu s(retention) never meets 0 x infinity.
__device__ __forceinline__ float gated_nu(float nu_log) { return min_nan(expf(nu_log), 3.402823466e38f); }

// 1 - s(v) = e^{-v} s(v) without cancellation, given e = e^{-v} (which may be infinite).
__device__ __forceinline__ float2 one_minus_s(float2 e, float2 s) {
  const float2 p = mul2(e, s);
  return make_float2(e.x > 8.5070592e37f ? 1.0f : p.x, e.y > 8.5070592e37f ? 1.0f : p.y);
}

template <int DEG, int N>
__device__ __forceinline__ void polynomial(const float (&c)[DEG + 1], const float2 (&x)[N], float2 (&y)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) y[k] = fma2(bcast2(c[DEG]), x[k], bcast2(c[DEG - 1]));
#pragma unroll
  for (int i = DEG - 2; i >= 0; --i)
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = fma2(y[k], x[k], bcast2(c[i]));
}

// What N tokens' gates give: a, beta = sqrt(1 - a^2), sw = s(write), and for the backward u = log a,
// kappa = -u a^2 / (1 - a^2), and 1 - s of the gates.
//
// In the bfloat16 kernels the special functions' units would bound the forward (five of their
// operations a channel and token take 16 a clock and SM: as long as the bytes), so with nu <= 1/2
// throughout the warp one of them goes: from rho = (1 + e^{-retention})^(-1/2) follow s(retention) =
// rho^2 and beta = sqrt(nu) rho S(w), w = nu rho^2 = -u, where S(w) = sqrt((1 - e^{-2w}) / w) is smooth. S,
// (1 - e^{-w}) / w and w / (e^{2w} - 1) are interpolated on [0, 1/2] by polynomials through the
// Chebyshev points (relative errors 1.4e-7, 8e-8 and 2e-8).
template <bool BWD, int N>
struct GatedGates {
  float2 a[N], beta[N], sw[N], u[BWD ? N : 1], kappa[BWD ? N : 1], om_r[BWD ? N : 1], om_w[BWD ? N : 1];
};
template <typename T, bool NEAR, bool BWD, int N>
__device__ __forceinline__ void gated_gates(const float2 (&r)[N], const float2 (&w)[N], float2 nu, float2 root_nu,
                                            GatedGates<BWD, N>& o) {
  float2 e[N], u[N];
  if constexpr (NEAR && sizeof(T) == 2) {
    constexpr float kDecay[5] = {0.999999929f, -0.499992883f, 0.166551928f, -0.0410132105f, 0.00678286256f};
    constexpr float kRoot[5] = {1.41421339f, -0.70709001f, 0.2943573f, -0.0868460191f, 0.0157274518f};
    float2 rho[N], y[N], v[N];
    exp_neg<T>(r, e);
#pragma unroll
    for (int k = 0; k < N; ++k) rho[k] = add2(e[k], bcast2(1.0f));
#pragma unroll
    for (int k = 0; k < N; ++k) rho[k] = make_float2(rsqrt_approx(rho[k].x), rsqrt_approx(rho[k].y));
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = mul2(rho[k], rho[k]);
    if constexpr (BWD) {
#pragma unroll
      for (int k = 0; k < N; ++k) o.om_r[k] = one_minus_s(e[k], y[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = mul2(nu, y[k]), u[k] = mul2(make_float2(-nu.x, -nu.y), y[k]);
    polynomial<4>(kDecay, v, y);
#pragma unroll
    for (int k = 0; k < N; ++k) o.a[k] = fma2(u[k], y[k], bcast2(1.0f));
    polynomial<4>(kRoot, v, y);
#pragma unroll
    for (int k = 0; k < N; ++k) o.beta[k] = mul2(y[k], mul2(rho[k], root_nu));
    if constexpr (BWD) {
      constexpr float kRatio[6] = {0.499999993f, -0.499998992f, 0.166643005f, 0.000204218905f, -0.0119145593f, 0.00147940113f};
      polynomial<5>(kRatio, v, o.kappa);
#pragma unroll
      for (int k = 0; k < N; ++k) o.u[k] = u[k];
    }
  } else {
    float2 s[N], q[N];
    exp_neg<T>(r, e);
    logistic_of(e, s);
    if constexpr (BWD) {
#pragma unroll
      for (int k = 0; k < N; ++k) o.om_r[k] = one_minus_s(e[k], s[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) u[k] = mul2(nu, s[k]);
    decay<NEAR>(u, o.a, q);
#pragma unroll
    for (int k = 0; k < N; ++k) q[k] = mul2(q[k], add2(o.a[k], bcast2(1.0f)));  // 1 - a^2
    if constexpr (BWD) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        // (1 - a^2 = 0 only with u = 0, or u too small for float32: the products with it and u are then 0)
        const float2 rs = make_float2(rsqrt_approx(fmaxf(q[k].x, 1.17549435e-38f)), rsqrt_approx(fmaxf(q[k].y, 1.17549435e-38f)));
        o.beta[k] = mul2(q[k], rs);
        o.kappa[k] = mul2(mul2(mul2(mul2(u[k], o.a[k]), o.a[k]), rs), rs);
        o.u[k] = make_float2(-u[k].x, -u[k].y);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) o.beta[k] = sqrt_2(q[k]);
    }
  }
  exp_neg<T>(w, e);
  logistic_of(e, o.sw);
  if constexpr (BWD) {
#pragma unroll
    for (int k = 0; k < N; ++k) o.om_w[k] = one_minus_s(e[k], o.sw[k]);
  }
}

template <typename T, bool NEAR, int N>
__device__ __forceinline__ void gated_ab(const float2 (&x)[N], const float2 (&r)[N], const float2 (&w)[N], float2 nu,
                                         float2 root_nu, float2 (&a)[N], float2 (&b)[N]) {
  GatedGates<false, N> g;
  gated_gates<T, NEAR, false, N>(r, w, nu, root_nu, g);
#pragma unroll
  for (int k = 0; k < N; ++k) a[k] = g.a[k], b[k] = mul2(mul2(g.beta[k], g.sw[k]), x[k]);
}

// ---------------------------------------------------------------- affine maps
__device__ __forceinline__ bool dropped(float A) { return __float_as_int(A) < 0; }
// A with the sign that says so where a or b has it
__device__ __forceinline__ float marked(float A, float a, float b) {
  return __int_as_float((__float_as_int(A) & 0x7fffffff) | ((__float_as_int(a) | __float_as_int(b)) & (int)0x80000000));
}

// A v + H
template <bool SEG>
__device__ __forceinline__ float2 through(float2 A, float2 H, float2 v) {
  const float2 o = fma2(A, v, H);
  if constexpr (!SEG) return o;
  return make_float2(dropped(A.x) ? H.x : o.x, dropped(A.y) ? H.y : o.y);
}
// (A1, H1) then (A2, H2). The mark of a start in either stays, also beside a factor that is NaN: the sign is
// put onto the product, whose own sign says nothing (a factor that is no start is +0, positive or NaN).
template <bool SEG>
__device__ __forceinline__ void compose(float2& A1, float2& H1, float2 A2, float2 H2) {
  H1 = through<SEG>(A2, H2, H1);
  const float2 A = mul2(A1, A2);
  A1 = SEG ? make_float2(marked(A.x, A1.x, A2.x), marked(A.y, A1.y, A2.y)) : A;
}
// A lam, nothing of it at a segment start
template <bool SEG>
__device__ __forceinline__ float2 through0(float2 A, float2 lam) {
  const float2 o = mul2(A, lam);
  if constexpr (!SEG) return o;
  return make_float2(dropped(A.x) ? 0.0f : o.x, dropped(A.y) ? 0.0f : o.y);
}

__device__ __forceinline__ float2 lo2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 cat4(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }

// The cluster's exchange, once a step: a warp of every CTA pushes the CTA's map to every CTA by
// asynchronous stores that count down the receiver's mbarrier, and every warp waits for its own
// CTA's. (A cluster barrier that releases the maps would wait for the warp's outputs on their way
// to global memory too.) Buffers and barriers are of two parities: a CTA pushes step n + 2 after it
// has step n + 1 from every CTA, which each pushed once all its warps were through with step n.
__host__ __device__ constexpr int gated_map_bytes(int cs) { return cs > 1 ? 2 * cs * 32 * 16 : 0; }

struct GatedExchange {
  float4* map;              // [2][CTAs of the cluster][32], at the same place in every CTA
  unsigned long long* bar;  // [2]
  int* late;                // [2]: a wait of the step ran out
  unsigned* pushed;         // [1 + CTAs of the cluster]: steps pushed, by this CTA and (on the way out) by each
  int cs;
  __device__ __forceinline__ float4* at(int par, int rank) const { return map + (par * cs + rank) * 32; }
};

__device__ __forceinline__ void exchange_init(const GatedExchange& x) {
  if (threadIdx.x == 0) {
    mbar_init(&x.bar[0], 1);
    mbar_init(&x.bar[1], 1);
    mbar_init_fence();
    x.late[0] = x.late[1] = 0;
    x.pushed[0] = 0;
  }
  // every CTA of the cluster has started, and its barriers stand, before anything is pushed
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void exchange_send(const GatedExchange& x, unsigned n, int rank, int lane, float4 v) {
  const int par = n & 1;
  if (lane == 0) mbar_arrive_expect_tx(&x.bar[par], (unsigned)x.cs * 32u * 16u);
  for (int q = 0; q < x.cs; ++q)
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                     cluster_smem_addr(x.at(par, rank) + lane, q)),
                 "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(cluster_smem_addr(&x.bar[par], q))
                 : "memory");
}
__device__ __forceinline__ void exchange_push(const GatedParams& p, const GatedExchange& x, unsigned n, int rank, int lane,
                                              float4 v) {
  if (p.withhold == n + 1 && rank == x.cs - 1) return;
  exchange_send(x, n, rank, lane, v);
  if (lane == 0) x.pushed[0] = n + 1;
}
// v through the maps of CTAs q0, q0 + d, ... up to before q1; they are read two ahead of their use
template <bool SEG>
__device__ __forceinline__ float2 exchange_through(const GatedExchange& x, int par, int q0, int q1, int d, int lane, float2 v) {
  for (; q0 != q1 && q0 + d != q1; q0 += 2 * d) {
    const float4 m = x.at(par, q0)[lane], n = x.at(par, q0 + d)[lane];
    v = through<SEG>(lo2(n), hi2(n), through<SEG>(lo2(m), hi2(m), v));
  }
  if (q0 != q1) v = through<SEG>(lo2(x.at(par, q0)[lane]), hi2(x.at(par, q0)[lane]), v);
  return v;
}
// A wait that runs out is marked, and the CTA leaves its loop at the next step, between the barrier that all its
// warps pass (so that all see the mark) and its push; its peers' waits then run out and they leave too.
__device__ __forceinline__ void exchange_wait(const GatedParams& p, const GatedExchange& x, unsigned n) {
  if (!mbar_wait_cluster(&x.bar[n & 1], n >> 1 & 1u, p.max_spin)) {
    x.late[n & 1] = 1;
    if (p.status != nullptr) atomicOr(p.status, kStatusTimeout);
  }
}
__device__ __forceinline__ bool exchange_late(const GatedExchange& x, unsigned n) {  // of the step before
  return *reinterpret_cast<volatile int*>(x.late + (n & 1 ^ 1)) != 0;
}

// The way out of the kernel, for every warp at once: no CTA exits while a push to it may be on its way. Every
// CTA comes to the barrier, and all pushes that the loops make have then been issued. A CTA none of whose
// waits ran out has every push, and may go. The others settle it (out of line and with the count of
// pushes in shared memory: in the kernel's body, or with the count in a register, the loops lose 2%). Where
// a CTA could go every step was pushed everywhere, so one that pushed every step itself waits for the last
// again. If that does not come, or not every step was pushed, no CTA can have gone, and they agree on the
// steps that were: a CTA pushes a step only if its wait for the one before did not run out, that is once
// every CTA had pushed that one, so their counts differ by one at most. Those behind push once more (no
// one reads it), which completes the last two phases everywhere, and each CTA waits until they have
// come. (These waits are for stores that have been issued, or are right behind the barrier: only a fault
// of the hardware could outlast their bound.)
__device__ __noinline__ void exchange_settle(const GatedExchange x, unsigned all) {
  const int lane = threadIdx.x & 31, rank = (int)(blockIdx.x % (unsigned)x.cs);
  auto come = [&](unsigned k) { return mbar_wait_cluster(&x.bar[k & 1], k >> 1 & 1u, kGatedDrain); };
  const unsigned pushed = x.pushed[0];
  if (pushed == all && __syncthreads_and(come(all - 1))) return;
  if (threadIdx.x < (unsigned)x.cs)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_smem_addr(x.pushed + 1 + rank, threadIdx.x)), "r"(pushed)
                 : "memory");
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  unsigned most = 0;
  for (int q = 1; q <= x.cs; ++q) most = max(most, *reinterpret_cast<volatile unsigned*>(x.pushed + q));
  if (threadIdx.x < 32 && pushed < most) exchange_send(x, pushed, rank, lane, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
  for (unsigned k = most < 2 ? 0 : most - 2; k < most; ++k) come(k);
}
// (behind a barrier of the CTA that follows its last wait)
__device__ __forceinline__ void exchange_leave(const GatedParams& p, const GatedExchange& x, int tile) {
  cluster_sync_relaxed();
  if ((x.late[0] | x.late[1]) == 0) return;
  const unsigned steps = (unsigned)(((p.L + tile - 1) / tile + x.cs - 1) / x.cs);
  const long long first = blockIdx.x / (unsigned)x.cs / (unsigned)p.groups;
  exchange_settle(x, (unsigned)((p.B - first + p.rows - 1) / p.rows) * steps);
}

// Which of a warp's K tokens from t0 on start a segment, as bits.
template <int K>
__device__ __forceinline__ unsigned gated_segments(const GatedParams& p, long long bt, int t0, int lane) {
  const int t = t0 + lane;
  return __ballot_sync(0xffffffffu, lane < K && t < p.L && gated_starts(p.pos, p.pos_bytes, bt * p.L + t));
}

// ---------------------------------------------------------------- forward
// A thread's tokens go through the gates eight at a time, in the backward four (more take too many registers).
template <typename T, bool NEAR, int K>
__device__ __forceinline__ void gated_fwd_tokens(const typename Duo<T>::type (&rx)[K], const typename Duo<T>::type (&rr)[K],
                                                 const typename Duo<T>::type (&rw)[K], float2 nu, float2 root_nu,
                                                 float2 (&a)[K], float2 (&b)[K]) {
  constexpr int N = 8;
#pragma unroll
  for (int k0 = 0; k0 < K; k0 += N) {
    float2 x[N], r[N], w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = Duo<T>::get(rx[k0 + k]), r[k] = Duo<T>::get(rr[k0 + k]), w[k] = Duo<T>::get(rw[k0 + k]);
    gated_ab<T, NEAR>(x, r, w, nu, root_nu, *reinterpret_cast<float2(*)[N]>(a + k0), *reinterpret_cast<float2(*)[N]>(b + k0));
  }
}

template <typename T, bool SEG, int MODE>
__global__ void __launch_bounds__(GatedFwdCut<T>::WARPS * 32, GatedFwdCut<T>::BLOCKS)
    gated_fwd_kernel(const __grid_constant__ GatedParams p) {
  using R = typename Duo<T>::type;
  using C = GatedFwdCut<T>;
  constexpr int K = C::K, NW = C::WARPS, TILE = C::TILE, S = C::STAGES, NT = 3;
  extern __shared__ __align__(16) unsigned char s_raw[];  // the cluster's maps, then [warp][tensor][token][lane]
  __shared__ float4 s_map[2][NW][32];                     // (A, H) of each warp
  __shared__ unsigned long long s_bar[2];
  __shared__ int s_late[2];
  __shared__ unsigned s_pushed[1 + kGatedMaxCluster];
  __shared__ float2 s_out[2][32];                         // one CTA: the state leaving its tile
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int cs = p.cluster, rank = (int)(blockIdx.x % (unsigned)cs);
  const unsigned id = blockIdx.x / (unsigned)cs;
  const int ch0 = (int)(id % (unsigned)p.groups) * 64, ch = ch0 + 2 * lane;
  const bool on = ch < p.D;
  const int stride = cs * TILE;  // tokens from a step to the next
  const GatedExchange peers{reinterpret_cast<float4*>(s_raw), s_bar, s_late, s_pushed, cs};  // (A, H) of each CTA
  R* stage = reinterpret_cast<R*>(s_raw + gated_map_bytes(cs)) + wp * S * (GatedReader<T, MODE, K, NT, S>::kStageBytes / (int)sizeof(R));
  const float2 nu = make_float2(on ? gated_nu(p.nu_log[ch]) : 0.0f, ch + 1 < p.D ? gated_nu(p.nu_log[ch + 1]) : 0.0f);
  const float2 root_nu = make_float2(sqrtf(nu.x), sqrtf(nu.y));
  const bool near = __all_sync(0xffffffffu, nu.x <= kGatedNear && nu.y <= kGatedNear);
  GatedReader<T, MODE, K, NT, S> reader(p, stage, ch0, lane, stride);
  if (cs > 1) exchange_init(peers);
  unsigned n = 0;  // steps so far

  for (long long bt = id / (unsigned)p.groups; bt < p.B; bt += p.rows) {
    int t0 = rank * TILE + wp * K;  // this warp's first token of the step
    float2 carry = load_pair(p.h0, bt * p.D + ch, ch, p.D);  // the state entering the step
    T* y = static_cast<T*>(p.y) + (bt * p.L + rank * TILE) * p.D;  // of the CTA's first token and channel
    reader.start(p, bt, t0, ch0, lane);
    int slot = 0;
#pragma unroll
    for (int k = 0; k < S; ++k) reader.copy(k, p.L - t0 - k * stride, lane);
    for (int first = 0; first < p.L; first += stride, t0 += stride, ++n) {
      const int par = n & 1;
      const unsigned seg = SEG ? gated_segments<K>(p, bt, t0, lane) : 0u;
      copy_wait<S - 1>();
      __syncwarp();
      float2 a[K], b[K], A = bcast2(1.0f), H = bcast2(0.0f);
      const int live = p.L - t0;  // tokens of the sequence from here on
      {
        R rx[K], rr[K], rw[K];
        reader.read(slot, 0, 0, lane, rx);
        reader.read(slot, 1, 0, lane, rr);
        reader.read(slot, 2, 0, lane, rw);
        __syncwarp();  // every lane has read its values
        reader.copy(slot, live - S * stride, lane);
        if (S > 1) slot = slot + 1 == S ? 0 : slot + 1;
        // (also of warps beyond the sequence: a condition here makes the others spill, and costs 8%)
        if (near) gated_fwd_tokens<T, true>(rx, rr, rw, nu, root_nu, a, b);
        else gated_fwd_tokens<T, false>(rx, rr, rw, nu, root_nu, a, b);
      }
      if (SEG && seg != 0) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (seg >> k & 1u) a[k] = bcast2(-0.0f);
      }
      if (live < K) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (k >= live) a[k] = bcast2(1.0f), b[k] = bcast2(0.0f);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) H = through<SEG>(a[k], b[k], H), A = mul2(A, a[k]);
      if (SEG && seg != 0) A = bcast2(-0.0f);  // (also where a later factor is NaN)
      s_map[par][wp][lane] = cat4(A, H);
      __syncthreads();
      float2 h;  // the state entering this CTA's tile, then this warp's tokens
      if (cs > 1) {
        if (exchange_late(peers, n)) goto leave;
        if (wp == NW - 1) {
          A = bcast2(1.0f), H = bcast2(0.0f);
#pragma unroll
          for (int j = 0; j < NW; ++j) compose<SEG>(A, H, lo2(s_map[par][j][lane]), hi2(s_map[par][j][lane]));
          exchange_push(p, peers, n, rank, lane, cat4(A, H));
        }
        exchange_wait(p, peers, n);
        h = exchange_through<SEG>(peers, par, 0, rank, 1, lane, carry);
        carry = exchange_through<SEG>(peers, par, rank, cs, 1, lane, h);
      } else {
        h = first == 0 ? carry : s_out[par ^ 1][lane];
      }
#pragma unroll
      for (int j = 0; j < NW - 1; ++j)
        if (j < wp) h = through<SEG>(lo2(s_map[par][j][lane]), hi2(s_map[par][j][lane]), h);
      if (p.carry != nullptr && wp * K % kGatedChunk == 0 && live > 0)
        store_pair(p.carry, (bt * p.chunks + t0 / kGatedChunk) * p.D + ch, ch, p.D, h);
      unsigned i = (unsigned)(wp * K) * (unsigned)p.D + (unsigned)ch;
      if (live >= K && on) {
#pragma unroll
        for (int k = 0; k < K; ++k, i += (unsigned)p.D) {
          h = through<SEG>(a[k], b[k], h);
          gated_store<T, MODE>(y + i, ch, p.D, h);
        }
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k, i += (unsigned)p.D) {
          h = through<SEG>(a[k], b[k], h);
          if (k < live && on) gated_store<T, MODE>(y + i, ch, p.D, h);
        }
      }
      y += (long long)stride * p.D;
      if (live <= K && live > 0 && p.last != nullptr) store_pair(p.last, bt * p.D + ch, ch, p.D, h);
      if (cs == 1 && wp == NW - 1) s_out[par][lane] = h;
    }
  }
leave:
  copy_wait<0>();
  if (cs > 1) {
    __syncthreads();
    exchange_leave(p, peers, TILE);
  }
}

// ---------------------------------------------------------------- backward
// Of a thread's tokens: f = a (-0 later where a segment starts); b = g x with g = sqrt(1 - a^2) s(write);
// q1 = a u and q2 = b kappa, so that q1 h_{t-1} + q2 = u du / lam; and, put by in shared memory until
// the adjoints are there, g, b (1 - s(write)) and 1 - s(retention).
template <typename T, bool NEAR, int K>
__device__ __forceinline__ void gated_bwd_tokens(const typename Duo<T>::type (&rx)[K], const typename Duo<T>::type (&rr)[K],
                                                 const typename Duo<T>::type (&rw)[K], float2 nu, float2 root_nu, int live,
                                                 float2* put, float2 (&f)[K], float2 (&b)[K], float2 (&q1)[K], float2 (&q2)[K]) {
  constexpr int N = 4;
#pragma unroll
  for (int k0 = 0; k0 < K; k0 += N) {
    if (k0 >= live) continue;
    float2 r[N], w[N];
    GatedGates<true, N> o;
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = Duo<T>::get(rr[k0 + k]), w[k] = Duo<T>::get(rw[k0 + k]);
    gated_gates<T, NEAR, true, N>(r, w, nu, root_nu, o);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float2 g = mul2(o.beta[k], o.sw[k]), bk = mul2(g, Duo<T>::get(rx[k0 + k]));
      put[(k0 + k) * 96] = g;
      put[(k0 + k) * 96 + 32] = mul2(bk, o.om_w[k]);
      put[(k0 + k) * 96 + 64] = o.om_r[k];
      f[k0 + k] = o.a[k];
      b[k0 + k] = bk;
      q1[k0 + k] = mul2(o.a[k], o.u[k]);
      q2[k0 + k] = mul2(bk, o.kappa[k]);
    }
  }
}

template <typename T, bool SEG, int MODE>
__global__ void __launch_bounds__(GatedBwdCut<T>::WARPS * 32, GatedBwdCut<T>::BLOCKS)
    gated_bwd_kernel(const __grid_constant__ GatedParams p) {
  using R = typename Duo<T>::type;
  using C = GatedBwdCut<T>;
  constexpr int K = C::K, NW = C::WARPS, TILE = C::TILE, S = C::STAGES, NT = 4;
  extern __shared__ __align__(16) unsigned char s_raw[];  // the cluster's maps, [warp][token][3][lane] put by, the inputs
  __shared__ float4 s_map[2][NW][32];                // (A, H) of each warp: states, forward
  __shared__ float2 s_adj[2][NW][32];                // G: adjoints, in reverse, out = A in + G
  __shared__ unsigned long long s_bar[2];
  __shared__ int s_late[2];
  __shared__ unsigned s_pushed[1 + kGatedMaxCluster];
  __shared__ float2 s_out[2][32];                    // one CTA: the adjoint leaving its tile
  __shared__ double2 s_nu[NW][32];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int cs = p.cluster, rank = (int)(blockIdx.x % (unsigned)cs);
  const unsigned id = blockIdx.x / (unsigned)cs;
  const int ch0 = (int)(id % (unsigned)p.groups) * 64, ch = ch0 + 2 * lane;
  const bool on = ch < p.D;
  const int stride = cs * TILE, steps = ((p.L + TILE - 1) / TILE + cs - 1) / cs;
  constexpr int kSpan = kGatedChunk / K;  // warps of a chunk
  const GatedExchange peers{reinterpret_cast<float4*>(s_raw), s_bar, s_late, s_pushed, cs};  // (A, G) of each CTA
  float2* put = reinterpret_cast<float2*>(s_raw + gated_map_bytes(cs)) + wp * K * 96 + lane;
  R* stage = reinterpret_cast<R*>(s_raw + gated_map_bytes(cs) + NW * K * 96 * sizeof(float2)) + wp * S * (GatedReader<T, MODE, K, NT, S>::kStageBytes / (int)sizeof(R));
  const float2 nu = make_float2(on ? gated_nu(p.nu_log[ch]) : 0.0f, ch + 1 < p.D ? gated_nu(p.nu_log[ch + 1]) : 0.0f);
  const float2 root_nu = make_float2(sqrtf(nu.x), sqrtf(nu.y));
  const bool near = __all_sync(0xffffffffu, nu.x <= kGatedNear && nu.y <= kGatedNear);
  GatedReader<T, MODE, K, NT, S> reader(p, stage, ch0, lane, -stride);
  if (cs > 1) exchange_init(peers);
  unsigned n = 0;  // steps so far
  double dnu_x = 0.0, dnu_y = 0.0;

  for (long long bt = id / (unsigned)p.groups; bt < p.B; bt += p.rows) {
    int tile = (steps - 1) * cs + rank, t0 = tile * TILE + wp * K;
    float2 carry = load_pair(p.grad_last, bt * p.D + ch, ch, p.D);  // c_{t+1} lam_{t+1} entering the step's last token
    long long base = (bt * p.L + (long long)tile * TILE) * p.D;     // of the CTA's first token and channel in the gradients
    reader.start(p, bt, t0, ch0, lane);
    int slot = 0;
#pragma unroll
    for (int k = 0; k < S; ++k) reader.copy(k, k < steps ? p.L - t0 + k * stride : 0, lane);
    for (int step = steps - 1; step >= 0; --step, tile -= cs, t0 -= stride, ++n) {
      const int par = n & 1;
      const unsigned seg = SEG ? gated_segments<K>(p, bt, t0, lane) : 0u;
      // the state entering this warp's chunk
      float2 h = load_pair(t0 < p.L ? p.carry : nullptr, (bt * p.chunks + t0 / kGatedChunk) * p.D + ch, ch, p.D);
      copy_wait<S - 1>();
      __syncwarp();
      const int live = p.L - t0;
      float2 f[K], b[K], q1[K], q2[K], A = bcast2(1.0f), H = bcast2(0.0f), G = bcast2(0.0f);
      R rd[K];
      {
        R rx[K], rr[K], rw[K];
        reader.read(slot, 0, 0, lane, rx);
        reader.read(slot, 1, 0, lane, rr);
        reader.read(slot, 2, 0, lane, rw);
        reader.read(slot, 3, 0, lane, rd);
        __syncwarp();
        reader.copy(slot, step >= S ? live + S * stride : 0, lane);
        if (S > 1) slot = slot + 1 == S ? 0 : slot + 1;
        if (near) gated_bwd_tokens<T, true>(rx, rr, rw, nu, root_nu, live, put, f, b, q1, q2);
        else gated_bwd_tokens<T, false>(rx, rr, rw, nu, root_nu, live, put, f, b, q1, q2);
      }
      if (SEG && seg != 0) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (seg >> k & 1u) f[k] = bcast2(-0.0f);
      }
      if (live < K) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (k >= live) f[k] = bcast2(1.0f), b[k] = bcast2(0.0f), rd[k] = Duo<T>::make(bcast2(0.0f));
      }
#pragma unroll
      for (int k = 0; k < K; ++k) H = through<SEG>(f[k], b[k], H), A = mul2(A, f[k]);
      if (SEG && seg != 0) A = bcast2(-0.0f);  // (also where a later factor is NaN)
#pragma unroll
      for (int k = K - 1; k >= 0; --k) G = through0<SEG>(f[k], add2(Duo<T>::get(rd[k]), G));
      s_map[par][wp][lane] = cat4(A, H);
      s_adj[par][wp][lane] = G;
      __syncthreads();
      if (cs > 1) {
        if (exchange_late(peers, n)) goto leave;
        if (wp == 0) {
#pragma unroll
          for (int i = NW - 1; i >= 0; --i) {
            if (i == NW - 1) A = lo2(s_map[par][i][lane]), G = s_adj[par][i][lane];
            else compose<SEG>(A, G, lo2(s_map[par][i][lane]), s_adj[par][i][lane]);
          }
          exchange_push(p, peers, n, rank, lane, cat4(A, G));
        }
      }
#pragma unroll
      for (int j = 0; j < NW - 1; ++j)
        if (j < wp && j >= wp / kSpan * kSpan) h = through<SEG>(lo2(s_map[par][j][lane]), hi2(s_map[par][j][lane]), h);
      // states forward: q1 <- q1 h_{t-1} + q2 (nothing of h_{t-1} at a segment start)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float2 v = fma2(q1[k], h, q2[k]);
        q1[k] = SEG ? make_float2(dropped(f[k].x) ? q2[k].x : v.x, dropped(f[k].y) ? q2[k].y : v.y) : v;
        h = through<SEG>(f[k], b[k], h);
      }
      float2 c;  // the adjoint entering this CTA's tile, then this warp's tokens
      if (cs > 1) {
        exchange_wait(p, peers, n);
        c = exchange_through<SEG>(peers, par, cs - 1, rank, -1, lane, carry);
        carry = exchange_through<SEG>(peers, par, rank, -1, -1, lane, c);
      } else {
        c = step == steps - 1 ? carry : s_out[par ^ 1][lane];
      }
#pragma unroll
      for (int j = NW - 1; j > 0; --j)
        if (j > wp) c = through<SEG>(lo2(s_map[par][j][lane]), s_adj[par][j][lane], c);
      // adjoints in reverse
      float2 sum = bcast2(0.0f);
      T *dx = static_cast<T*>(p.dx) + base, *dr = static_cast<T*>(p.dr) + base, *dw = static_cast<T*>(p.dw) + base;
      unsigned i = (unsigned)(wp * K + K - 1) * (unsigned)p.D + (unsigned)ch;
      auto token = [&](int k, bool store) {
        const float2 lam = add2(Duo<T>::get(rd[k]), c), du = mul2(lam, q1[k]);
        c = through0<SEG>(f[k], lam);
        if (store) {
          gated_store<T, MODE>(dx + i, ch, p.D, mul2(lam, put[k * 96]));
          gated_store<T, MODE>(dw + i, ch, p.D, mul2(lam, put[k * 96 + 32]));
          gated_store<T, MODE>(dr + i, ch, p.D, mul2(du, put[k * 96 + 64]));
          sum = add2(sum, du);
        }
        i -= (unsigned)p.D;
      };
      if (live >= K && on) {
#pragma unroll
        for (int k = K - 1; k >= 0; --k) token(k, true);
      } else {
#pragma unroll
        for (int k = K - 1; k >= 0; --k) token(k, k < live && on);
      }
      base -= (long long)stride * p.D;
      dnu_x += (double)sum.x;
      dnu_y += (double)sum.y;
      if (wp == 0) {
        if (cs == 1) s_out[par][lane] = c;
        if (tile == 0 && p.grad_h0 != nullptr) store_pair(p.grad_h0, bt * p.D + ch, ch, p.D, c);
      }
    }
  }
leave:
  copy_wait<0>();
  // the CTA's sum of dnu_log per channel, over its warps in order
  s_nu[wp][lane] = make_double2(dnu_x, dnu_y);
  __syncthreads();
  if (wp == 0) {
    double sx = 0.0, sy = 0.0;
    for (int j = 0; j < NW; ++j) sx += s_nu[j][lane].x, sy += s_nu[j][lane].y;
    double* part = p.part + ((long long)(id / (unsigned)p.groups) * cs + rank) * p.D;
    if (on) part[ch] = sx;
    if (ch + 1 < p.D) part[ch + 1] = sy;
  }
  if (cs > 1) {
    __syncwarp();
    exchange_leave(p, peers, TILE);
  }
}

// dnu_log[d] = the sum of the partial rows, in order: a warp's lanes own 32 channels, the block's
// warps every kReduceRows-th row, then warp 0 adds the warps' sums.
constexpr int kReduceRows = 8;
__global__ void __launch_bounds__(kReduceRows * 32) gated_reduce_kernel(const double* part, float* out, int rows, int D) {
  __shared__ double s[kReduceRows][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  double t = 0.0;
  if (d < D)
    for (int r = wp; r < rows; r += kReduceRows) t += part[(long long)r * D + d];
  s[wp][lane] = t;
  __syncthreads();
  if (wp == 0 && d < D) {
    for (int j = 1; j < kReduceRows; ++j) t += s[j][lane];
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

// A warp owns the 64 channels that a warp of the scan owns (two a lane), so that its arithmetic and
// its results are those of a scan of one token.
template <typename T, int MODE>
__global__ void __launch_bounds__(128) gated_step_kernel(const GatedStepParams p) {
  const int ch = (int)(blockIdx.x * 128 + threadIdx.x) * 2;
  const bool on = ch < p.D, both = ch + 1 < p.D;
  const float2 nu = make_float2(on ? gated_nu(__ldg(p.nu_log + ch)) : 0.0f, both ? gated_nu(__ldg(p.nu_log + ch + 1)) : 0.0f);
  const float2 root_nu = make_float2(sqrtf(nu.x), sqrtf(nu.y));
  const bool near = __all_sync(0xffffffffu, nu.x <= kGatedNear && nu.y <= kGatedNear);
  if (!on) return;
  auto load = [&](const void* base, long long i) {
    const T* q = static_cast<const T*>(base) + i + ch;
    if constexpr (MODE != kModeSingle) return Duo<T>::get(__ldg(reinterpret_cast<const typename Duo<T>::type*>(q)));
    return make_float2(Io<T>::load(q), both ? Io<T>::load(q + 1) : 0.0f);
  };
  for (long long b = blockIdx.y; b < p.B; b += gridDim.y) {
    const float2 x[1] = {load(p.x, b * p.sx)}, r[1] = {load(p.r, b * p.sr)}, w[1] = {load(p.w, b * p.sw)};
    const float2 s = load_pair(p.state, b * p.D + ch, ch, p.D);
    const bool start = p.pos != nullptr && gated_starts(p.pos, p.pos_bytes, b);
    float2 a[1], c[1];
    if (near) gated_ab<T, true>(x, r, w, nu, root_nu, a, c);
    else gated_ab<T, false>(x, r, w, nu, root_nu, a, c);
    const float2 h = start ? c[0] : fma2(a[0], s, c[0]);
    gated_store<T, MODE>(static_cast<T*>(p.y) + b * p.D + ch, ch, p.D, h);
    store_pair(p.new_state, b * p.D + ch, ch, p.D, h);
  }
}

// ---------------------------------------------------------------- host
__device__ unsigned g_gated_status;  // zero from the module's loading on: no stream orders its clearing

struct GatedPlan {
  int groups, cluster, rows;
};

// 64 channels a cluster. A CTA's throughput does not depend on how many others share its sequence,
// but their exchange costs (B=8 T=16384 D=2048 bf16, 256 rows x groups, backward: one CTA each 932 us,
// clusters of eight 1017 us), and an SM with one CTA waits most of the time (one row of the same,
// forward: clusters of one to eight 419, 249, 133, 95 us). So the cluster grows, no further than the
// tiles reach, until half the CTAs that are resident at once are there; to 16 CTAs only where eight
// would leave SMs without one (3 rows T=24864 D=90, six rows x groups: 144 -> 89 us and backward 200 ->
// 118 us; but the one row of 32 groups above 95 -> 121 us). More
// rows than a few waves of CTAs need are walked by the same clusters, which bounds the partial sums.
static GatedPlan gated_plan(long long B, long long L, long long D, bool backward, int dtype) {
  constexpr long long kSms = 148, kMost = kSms * 16;
  using bf16 = __nv_bfloat16;
  const bool half = dtype == SPARC_DTYPE_BF16;
  const int blocks = backward ? (half ? GatedBwdCut<bf16>::BLOCKS : GatedBwdCut<float>::BLOCKS)
                              : (half ? GatedFwdCut<bf16>::BLOCKS : GatedFwdCut<float>::BLOCKS);
  const int tile = backward ? (half ? GatedBwdCut<bf16>::TILE : GatedBwdCut<float>::TILE)
                            : (half ? GatedFwdCut<bf16>::TILE : GatedFwdCut<float>::TILE);
  GatedPlan pl;
  pl.groups = (int)((D + 63) / 64);
  const long long tiles = (L + tile - 1) / tile;
  pl.cluster = 1;
  while (pl.cluster < kGatedMaxCluster && pl.cluster * 2 <= tiles &&
         B * pl.groups * pl.cluster * 2 < (pl.cluster < 8 ? kSms * blocks : 2 * kSms))
    pl.cluster *= 2;
  const long long rows = std::max(1LL, kMost / ((long long)pl.groups * pl.cluster));
  pl.rows = (int)std::min(B, rows);
  return pl;
}

static bool gated_valid_dtype(int d) { return d == SPARC_DTYPE_F32 || d == SPARC_DTYPE_BF16; }

static int gated_check_shape(long long B, long long L, long long D) {
  if (B <= 0 || L <= 0 || D <= 0) return fail(SPARC_ERR_SHAPE, "batch, length and channels must be positive");
  if (D > (1LL << 22) || B > (1LL << 31) || L > (1LL << 30) || (double)B * (double)L * (double)D > 4.0e18)
    return fail(SPARC_ERR_SHAPE, "shape beyond the launch grid (channels <= 2^22, length <= 2^30, batch <= 2^31)");
  return SPARC_OK;
}

static bool gated_pos_ok(const void* pos, int bytes) {
  return pos == nullptr || bytes == 1 || bytes == 2 || bytes == 4 || bytes == 8;
}

static bool gated_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// The widest reads that the inputs' bases, strides and width allow.
static GatedMode gated_mode(const GatedParams& p, int inputs, int size) {
  auto fits = [&](int bytes) {
    bool ok = (long long)p.D * size % bytes == 0;
    for (int n = 0; n < inputs; ++n)
      ok = ok && gated_aligned(p.in[n].p, bytes) && (p.B <= 1 || p.in[n].sb * size % bytes == 0) &&
           (p.L <= 1 || p.in[n].st * size % bytes == 0);
    return ok;
  };
  return fits(16) ? kModeWide : fits(2 * size) ? kModePair : kModeSingle;
}

template <typename T, bool SEG, int MODE>
static cudaError_t gated_launch(const GatedParams& p, bool backward, cudaStream_t s) {
  using F = GatedFwdCut<T>;
  using W = GatedBwdCut<T>;
  constexpr int kFwdBytes = F::WARPS * F::STAGES * GatedReader<T, MODE, F::K, 3, F::STAGES>::kStageBytes;
  constexpr int kBwdBytes = W::WARPS * W::STAGES * GatedReader<T, MODE, W::K, 4, W::STAGES>::kStageBytes +
                            W::TILE * 96 * (int)sizeof(float2);
  const int smem = gated_map_bytes(p.cluster) + (backward ? kBwdBytes : kFwdBytes);
  // The limit belongs to the kernel, not to a launch: every call sets that of the largest cluster, as a
  // smaller one could come between another thread's setting and its launch.
  const int most = gated_map_bytes(kGatedMaxCluster) + (backward ? kBwdBytes : kFwdBytes);
  const auto kernel = backward ? gated_bwd_kernel<T, SEG, MODE> : gated_fwd_kernel<T, SEG, MODE>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return e;
  if (p.cluster > 8) {
    const cudaError_t wide = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (wide != cudaSuccess) return wide;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.groups * (unsigned)p.rows * (unsigned)p.cluster);
  cfg.blockDim = dim3((backward ? W::WARPS : F::WARPS) * 32);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  TimedLaunch tl(backward ? kTimeGatedBwd : kTimeGatedFwd, s);
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, bool SEG>
static cudaError_t gated_modes(const GatedParams& p, GatedMode mode, bool backward, cudaStream_t s) {
  switch (mode) {
    case kModeWide: return gated_launch<T, SEG, kModeWide>(p, backward, s);
    case kModePair: return gated_launch<T, SEG, kModePair>(p, backward, s);
    default: return gated_launch<T, SEG, kModeSingle>(p, backward, s);
  }
}

static cudaError_t gated_dispatch(const GatedParams& p, GatedMode mode, int dtype, bool backward, cudaStream_t s) {
  if (dtype == SPARC_DTYPE_BF16)
    return p.pos != nullptr ? gated_modes<__nv_bfloat16, true>(p, mode, backward, s)
                            : gated_modes<__nv_bfloat16, false>(p, mode, backward, s);
  return p.pos != nullptr ? gated_modes<float, true>(p, mode, backward, s)
                          : gated_modes<float, false>(p, mode, backward, s);
}

static size_t gated_ws_bytes(long long B, long long L, long long D) {
  size_t rows = 0;  // of either type
  for (int dtype : {SPARC_DTYPE_F32, SPARC_DTYPE_BF16}) {
    const GatedPlan pl = gated_plan(B, L, D, true, dtype);
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

int sparc_gated_status_word(unsigned** word) {
  if (word == nullptr) return fail(SPARC_ERR_ARG, "null pointer");
  void* p = nullptr;
  // (the first call on a device may load the module, also while the thread captures a graph)
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
  if (e == cudaSuccess) {
    e = cudaGetSymbolAddress(&p, g_gated_status);
    cudaThreadExchangeStreamCaptureMode(&mode);
  }
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  *word = static_cast<unsigned*>(p);
  return SPARC_OK;
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
  p.in[0] = GatedIn{a->x, a->x_batch_stride, a->x_token_stride};
  p.in[1] = GatedIn{a->retention_gate, a->retention_batch_stride, a->retention_token_stride};
  p.in[2] = GatedIn{a->write_gate, a->write_batch_stride, a->write_token_stride};
  p.y = a->y;
  p.nu_log = a->nu_log;
  p.h0 = a->h0;
  p.last = a->last;
  p.carry = a->carry;
  p.pos = a->segment_pos;
  p.pos_bytes = a->segment_pos_bytes;
  p.B = a->batch;
  p.L = (int)a->length;
  p.D = (int)a->channels;
  p.chunks = (int)sparc_gated_carry_chunks(a->length);
  p.max_spin = a->max_spin != 0 ? a->max_spin : kGatedSpin;
  p.status = a->status;
  p.withhold = a->inject_withhold_step;
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  for (const void* q : {a->x, a->retention_gate, a->write_gate, (const void*)a->y})
    if (!gated_aligned(q, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
  const GatedMode mode = gated_aligned(p.y, 2 * size) ? gated_mode(p, 3, size) : kModeSingle;
  const GatedPlan pl = gated_plan(p.B, p.L, p.D, false, a->dtype);
  p.groups = pl.groups;
  p.cluster = pl.cluster;
  p.rows = pl.rows;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = gated_dispatch(p, mode, a->dtype, false, s);
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
  p.in[0] = GatedIn{a->x, a->x_batch_stride, a->x_token_stride};
  p.in[1] = GatedIn{a->retention_gate, a->retention_batch_stride, a->retention_token_stride};
  p.in[2] = GatedIn{a->write_gate, a->write_batch_stride, a->write_token_stride};
  p.in[3] = GatedIn{a->dy, a->dy_batch_stride, a->dy_token_stride};
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
  p.L = (int)a->length;
  p.D = (int)a->channels;
  p.chunks = (int)sparc_gated_carry_chunks(a->length);
  p.max_spin = a->max_spin != 0 ? a->max_spin : kGatedSpin;
  p.status = a->status;
  p.withhold = a->inject_withhold_step;
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  for (const GatedIn& in : p.in)
    if (!gated_aligned(in.p, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
  bool pairs = true;
  for (const void* q : {p.dx, p.dr, p.dw}) {
    if (!gated_aligned(q, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
    pairs = pairs && gated_aligned(q, 2 * size);
  }
  const GatedMode mode = pairs ? gated_mode(p, 4, size) : kModeSingle;
  const GatedPlan pl = gated_plan(p.B, p.L, p.D, true, a->dtype);
  p.groups = pl.groups;
  p.cluster = pl.cluster;
  p.rows = pl.rows;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = gated_dispatch(p, mode, a->dtype, true, s);
  if (e == cudaSuccess) {
    TimedLaunch tl(kTimeGatedReduce, s);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.D + 31) / 32));
    cfg.blockDim = dim3(kReduceRows * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, gated_reduce_kernel, (const double*)p.part, a->grad_nu_log, pl.rows * pl.cluster, p.D);
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
  const int size = a->dtype == SPARC_DTYPE_BF16 ? 2 : 4;
  for (const void* q : {a->x, a->retention_gate, a->write_gate, (const void*)a->y})
    if (!gated_aligned(q, size)) return fail(SPARC_ERR_ARG, "misaligned activation pointer");
  bool pairs = p.D % 2 == 0 && gated_aligned(p.x, 2 * size) && gated_aligned(p.r, 2 * size) &&
               gated_aligned(p.w, 2 * size) && gated_aligned(p.y, 2 * size);
  if (p.B > 1) pairs = pairs && p.sx % 2 == 0 && p.sr % 2 == 0 && p.sw % 2 == 0;
  const dim3 grid((unsigned)((p.D + 255) / 256), (unsigned)std::min<long long>(p.B, 32768));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  TimedLaunch tl(kTimeGatedStep, s);
  if (a->dtype == SPARC_DTYPE_BF16) {
    if (pairs) gated_step_kernel<__nv_bfloat16, kModePair><<<grid, 128, 0, s>>>(p);
    else gated_step_kernel<__nv_bfloat16, kModeSingle><<<grid, 128, 0, s>>>(p);
  } else {
    if (pairs) gated_step_kernel<float, kModePair><<<grid, 128, 0, s>>>(p);
    else gated_step_kernel<float, kModeSingle><<<grid, 128, 0, s>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(SPARC_ERR_LAUNCH, cudaGetErrorString(e));
  return SPARC_OK;
}

}  // extern "C"
