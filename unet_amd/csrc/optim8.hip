// AdamW with its two moments held in 8 bits (the fp32 form is optim.hip), behind the same clip of the group's gradient norm:
//   m <- b1 m + (1-b1) g,   r <- sqrt(b2 r^2 + (1-b2) g^2),   p <- (1 - lr wd) p - lr/(1-b1^t) * m / (r / sqrt(1-b2^t) + eps)
// m and r = sqrt(v) are stored as e4m3 codes with one fp32 scale = max|.| / 448 per block of 256 elements of a tensor.  The
// ROOT of v is kept because codes with a 4-bit exponent cover 2^-15 of a block's largest root, that is 2^-30 of its largest v.
// A positive root never becomes zero (it is raised to the smallest code, 2^-9): a stored m over a vanished root would be
// divided by eps alone at the next step.  A block whose largest value is below 2^-100 is stored as zeros: 448 / max would
// overflow, and such moments are far below any eps.  An infinite or NaN gradient makes its block of 256 NaN; with a clip a NaN
// reaches every element through the norm, and an infinite norm takes all other gradients to zero.
// Stored values are rounded to nearest even; the step itself uses m and r before that rounding.
// Tensors the caller keeps in 32 bits (small ones: norms, biases) go through the same launches.
//
// HBM-bound: p, g and two codes read, p and two codes written = 16 bytes an element (the fp32 form: 28), plus 4 for the
// norm's pass over g when a clip needs it first.  Without a clip the squares are summed while the step runs.
// A wave owns ONE block of 256 elements, four a lane, so a block's maximum is a wave reduction and the many short waves hide each
// other's loads (with eight blocks a wave, four in flight, a model of 126 k parameters took 19 us instead of 5).  Parameters and
// codes are not needed again before the next step: their accesses are non-temporal, which leaves the caches to the gradient,
// read twice (at 42 M parameters the norm's pass 48 -> 32 us, this kernel 131 -> 113; at 446.6 M 335 -> 299 and 1363 -> 1203 us,
// 6.0 TB/s).
#include "common.h"

namespace {

constexpr int A8_THREADS = 256;
constexpr int A8_WAVES = A8_THREADS / 64;                          // blocks of 256 elements a workgroup
constexpr unsigned A8_WIDE = 0x80000000u;                        // slot flag: 32-bit moments
constexpr float A8_MAX = 448.f, A8_LEAST = 0.001953125f;         // largest and smallest positive e4m3 value
constexpr float A8_TINY = 7.888609052210118e-31f;                // 2^-100

struct GradPtrs { const float* g[UNET_OPT_MAX_TENSORS]; };

struct Adam8 {
  float* const* p;                 // [n] parameters
  const unsigned* start;           // [n + 1] first block of every tensor (of this batch; absolute numbers)
  const unsigned* numel;           // [n]
  const unsigned* slot;            // [n] first block in the code buffers, or A8_WIDE | first float4 in m32 / v32
  unsigned char *m8, *r8;
  float *sm, *sr, *m32, *v32;
  const float* coef;               // [0] clip, [4] lr
  const float2* bc;                // [n] (lr / (1 - b1^t), 1 / sqrt(1 - b2^t))
  float* partial;                  // sums of g^2 per workgroup, or null
  float beta1, beta2, grow1, grow2;   // grow = 1 - beta, rounded once from the caller's double
  float eps, weight_decay;
  int n;
};

// The update's roundings, one after the other and without contraction: what is stored is a rounding of these values, and a
// fused step would move a few of them across a code's border.
__device__ __forceinline__ void moments(float g, float& m, float& r, const Adam8& k) {
#pragma clang fp contract(off)
  m = m * k.beta1 + g * k.grow1;
  r = sqrtf(r * r * k.beta2 + g * k.grow2 * g);
}
__device__ __forceinline__ void move(float& p, float m, float r, float keep, float2 bc, float eps) {
  p = p * keep - bc.x * (m * __builtin_amdgcn_rcpf(fmaf(r, bc.y, eps)));
}

__device__ __forceinline__ void decode(unsigned w, float scale, float (&f)[4]) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  f[0] = lo[0] * scale; f[1] = lo[1] * scale; f[2] = hi[0] * scale; f[3] = hi[1] * scale;
}
__device__ __forceinline__ unsigned encode(const float (&y)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
// maximum that keeps a NaN
__device__ __forceinline__ float top4(const float (&x)[4]) {
  float t = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  return (x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3]) ? INFINITY : t;
}
// codes and scale of one block from a wave's values; ROOT: positive values stay positive
template <bool ROOT> __device__ __forceinline__ unsigned store_block(const float (&x)[4], float& scale) {
#pragma clang fp contract(off)
  const float top = wave_max(top4(x));
  const bool some = top >= A8_TINY;
  const float inv = some ? (1.f / top) * A8_MAX : 0.f;
  scale = some ? top * (1.f / A8_MAX) : 0.f;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = x[e] * inv;
    if (ROOT && some && x[e] > 0.f) y[e] = fmaxf(y[e], A8_LEAST);
  }
  return encode(y);
}

__device__ __forceinline__ int find_tensor(const unsigned* start, int n, unsigned b) {
  int lo = 0, hi = n;                       // start[lo] <= b < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

// Sums of g^2 in 64 bits, one a workgroup: with 32-bit sums the clip was now and then an ulp off the one of the exact norm, which
// moves some of 42 M codes across a border.  HBM-bound: NORM_BLOCKS loads of 16 bytes a lane in flight; 42 M elements 31 us.
constexpr int NORM_BLOCKS = 8;                                     // blocks of 256 elements a wave
__global__ __launch_bounds__(A8_THREADS) void adamw8_sqnorm_kernel(const GradPtrs gp, const unsigned* start, const unsigned* numel, int n,
                                                                   double* partial) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned first = start[0] + (blockIdx.x * A8_WAVES + wave) * NORM_BLOCKS;
  const unsigned end = min(first + NORM_BLOCKS, start[n]);
  double s = 0.0;
  if (first < end) {
    int t = find_tensor(start, n, first);
    const float* g0 = gp.g[t];
    // the usual case: whole blocks of one aligned tensor
    if (end == first + NORM_BLOCKS && end <= start[t + 1] && (end - start[t]) * 256u <= numel[t] && !(reinterpret_cast<uintptr_t>(g0) & 15)) {
      if (g0) {
        f32x4 v[NORM_BLOCKS];
#pragma unroll
        for (int u = 0; u < NORM_BLOCKS; ++u) v[u] = *reinterpret_cast<const f32x4*>(g0 + (first - start[t] + u) * 256u + lane * 4);
#pragma unroll
        for (int u = 0; u < NORM_BLOCKS; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) s = fma((double)v[u][e], (double)v[u][e], s);
      }
    } else {
      for (unsigned b = first; b < end; ++b) {
        while (b >= start[t + 1]) ++t;
        const float* g = gp.g[t];
        if (!g) continue;
        const unsigned i = (b - start[t]) * 256u + lane * 4, ne = numel[t];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < ne) s = fma((double)g[i + e], (double)g[i + e], s);
      }
    }
  }
  __shared__ double red[A8_WAVES];
#pragma unroll
  for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m, 64);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(A8_THREADS) void adamw8_apply_kernel(const Adam8 k, const GradPtrs gp) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned b = k.start[0] + blockIdx.x * A8_WAVES + wave;
  float sq = 0.f;
  const int t = b < k.start[k.n] ? find_tensor(k.start, k.n, b) : -1;
  const float* gt = t >= 0 ? gp.g[t] : nullptr;
  if (gt) {                                           // no gradient this step: the tensor and its moments stay as they are
    const float clip = k.coef[0], keep = 1.f - k.coef[4] * k.weight_decay;
    float* pt = k.p[t];
    const unsigned slot = k.slot[t], ne = k.numel[t], bo = b - k.start[t], i = bo * 256u + lane * 4;
    const float2 bc = k.bc[t];
    float g[4] = {0.f, 0.f, 0.f, 0.f}, p[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = (bo + 1) * 256u <= ne && !((reinterpret_cast<uintptr_t>(gt) | reinterpret_cast<uintptr_t>(pt)) & 15);
    const int cnt = i >= ne ? 0 : (ne - i < 4 ? (int)(ne - i) : 4);
    const bool wide = slot & A8_WIDE;
    const size_t cb = (size_t)slot + bo;
    unsigned* const mc = reinterpret_cast<unsigned*>(k.m8 + cb * 256 + lane * 4);
    unsigned* const rc = reinterpret_cast<unsigned*>(k.r8 + cb * 256 + lane * 4);
    unsigned mw = 0, rw = 0;
    float ms = 0.f, rs = 0.f;
    if (!wide) {
      mw = __builtin_nontemporal_load(mc);
      rw = __builtin_nontemporal_load(rc);
      ms = k.sm[cb];
      rs = k.sr[cb];
    }
    if (whole) {
      const f32x4 gv = *reinterpret_cast<const f32x4*>(gt + i);
      const f32x4 pv = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(pt + i));
#pragma unroll
      for (int e = 0; e < 4; ++e) { g[e] = gv[e]; p[e] = pv[e]; }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < cnt) { g[e] = gt[(size_t)i + e]; p[e] = pt[(size_t)i + e]; }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sq = fmaf(g[e], g[e], sq);
    if (wide) {
      const size_t at = (size_t)(slot & ~A8_WIDE) * 4 + i;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < cnt) {
          const float gc = g[e] * clip;
          const float m1 = k.beta1 * k.m32[at + e] + k.grow1 * gc;
          const float v1 = k.beta2 * k.v32[at + e] + k.grow2 * gc * gc;
          k.m32[at + e] = m1;
          k.v32[at + e] = v1;
          move(p[e], m1, sqrtf(v1), keep, bc, k.eps);
        }
    } else {
      decode(mw, ms, m);
      decode(rw, rs, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e < cnt) {
          moments(g[e] * clip, m[e], r[e], k);
          move(p[e], m[e], r[e], keep, bc, k.eps);
        } else m[e] = r[e] = 0.f;
      }
      float s1, s2;
      __builtin_nontemporal_store(store_block<false>(m, s1), mc);
      __builtin_nontemporal_store(store_block<true>(r, s2), rc);
      if (lane == 0) { k.sm[cb] = s1; k.sr[cb] = s2; }
    }
    if (whole) {
      __builtin_nontemporal_store(f32x4{p[0], p[1], p[2], p[3]}, reinterpret_cast<f32x4*>(pt + i));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < cnt) pt[(size_t)i + e] = p[e];
    }
  }
  if (k.partial) {
    __shared__ float red[A8_WAVES];
    sq = wave_sum(sq);
    if (lane == 0) red[wave] = sq;
    __syncthreads();
    if (threadIdx.x == 0) k.partial[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
  }
}

// One workgroup.  blocks > 0: ||g|| from the partial sums into coef[3], and the clip min(1, max_norm / (||g|| + 1e-6)) into
// coef[0]; otherwise coef[0] = 1.  Then lr into coef[4], and the tensors with a gradient count this step and get their bias corrections.
constexpr int PREP_THREADS = 1024;
template <typename T> __device__ __forceinline__ double prepare_sum(const T* partial, int blocks) {
  double a = 0.0;
  int i = threadIdx.x;
  for (; i + 3 * PREP_THREADS < blocks; i += 4 * PREP_THREADS)
    a += ((double)partial[i] + (double)partial[i + PREP_THREADS]) +
         ((double)partial[i + 2 * PREP_THREADS] + (double)partial[i + 3 * PREP_THREADS]);
  for (; i < blocks; i += PREP_THREADS) a += (double)partial[i];
  return a;
}
__global__ __launch_bounds__(PREP_THREADS) void adamw8_prepare_kernel(const GradPtrs gp, const void* partial, int blocks, int sums64,
                                                                      float max_norm, const float* lr, float* coef, float* step_t, int n,
                                                                      double beta1, double beta2, float2* bc) {
  const int t = threadIdx.x;
  if (bc && t < n) {
    if (gp.g[t]) step_t[t] += 1.f;
    const double st = (double)step_t[t];
    bc[t] = make_float2((float)((double)*lr / (1.0 - pow(beta1, st))), (float)(1.0 / sqrt(1.0 - pow(beta2, st))));
  }
  __shared__ double red[PREP_THREADS];
  red[t] = sums64 ? prepare_sum(static_cast<const double*>(partial), blocks) : prepare_sum(static_cast<const float*>(partial), blocks);
  __syncthreads();
  for (int s = PREP_THREADS / 2; s > 0; s >>= 1) {
    if (t < s) red[t] += red[t + s];
    __syncthreads();
  }
  if (t == 0) {
    float clip = 1.f;
    if (blocks > 0) {
      const float total = (float)sqrt(red[0]);
      coef[3] = total;
      if (max_norm > 0.f) {
        clip = max_norm * (1.f / (total + 1e-6f));      // rounded as clip_grad_norm_ does: an ulp of it moves codes
        clip = clip > 1.f ? 1.f : clip;                 // (a NaN norm reaches every tensor, as it does there)
      }
    }
    coef[0] = clip;
    coef[4] = *lr;
  }
}

}  // namespace

extern "C" int32_t unet_adamw8_blocks(int64_t blocks256) { return (int32_t)((blocks256 + A8_WAVES - 1) / A8_WAVES); }

extern "C" int32_t unet_adamw8_norm_blocks(int64_t blocks256) {
  return (int32_t)((blocks256 + A8_WAVES * NORM_BLOCKS - 1) / (A8_WAVES * NORM_BLOCKS));
}

extern "C" int unet_adamw8_sqnorm(const float* const* grads_host, int32_t n_tensors, const uint32_t* start256, const uint32_t* numel,
                                  int64_t blocks256, double* partial, void* stream) {
  UNET_REQUIRE(grads_host && start256 && numel && partial, "adamw8_sqnorm: null pointer");
  UNET_REQUIRE(n_tensors >= 1 && n_tensors <= UNET_OPT_MAX_TENSORS, "adamw8_sqnorm: 1..%d tensors per call, got %d",
               UNET_OPT_MAX_TENSORS, n_tensors);
  UNET_REQUIRE(blocks256 > 0 && blocks256 < (1ll << 31), "adamw8_sqnorm: %lld blocks", (long long)blocks256);
  GradPtrs gp;
  for (int i = 0; i < UNET_OPT_MAX_TENSORS; ++i) gp.g[i] = i < n_tensors ? grads_host[i] : nullptr;
  hipLaunchKernelGGL(adamw8_sqnorm_kernel, dim3(unet_adamw8_norm_blocks(blocks256)), dim3(A8_THREADS), 0, static_cast<hipStream_t>(stream),
                     gp, start256, numel, n_tensors, partial);
  UNET_LAUNCH_CHECK("adamw8_sqnorm");
  return 0;
}

extern "C" int unet_adamw8_prepare(const float* const* grads_host, int32_t n_tensors, const void* partial, int32_t n_partial,
                                   int32_t sums64, float max_norm, const float* lr, float* coef, float* step_t, double beta1,
                                   double beta2, float* bc, void* stream) {
  UNET_REQUIRE(lr && coef, "adamw8_prepare: null pointer");
  UNET_REQUIRE(n_tensors >= 0 && n_tensors <= UNET_OPT_MAX_TENSORS, "adamw8_prepare: at most %d tensors per call, got %d",
               UNET_OPT_MAX_TENSORS, n_tensors);
  UNET_REQUIRE(n_tensors == 0 || (grads_host && step_t && bc), "adamw8_prepare: null pointer");
  UNET_REQUIRE(n_partial >= 0 && (n_partial == 0 || partial), "adamw8_prepare: bad partial sums");
  UNET_REQUIRE(n_partial > 0 || !(max_norm > 0.f), "adamw8_prepare: a clip needs the partial sums");
  GradPtrs gp;
  for (int i = 0; i < UNET_OPT_MAX_TENSORS; ++i) gp.g[i] = i < n_tensors ? grads_host[i] : nullptr;
  hipLaunchKernelGGL(adamw8_prepare_kernel, dim3(1), dim3(PREP_THREADS), 0, static_cast<hipStream_t>(stream), gp, partial, n_partial, sums64,
                     max_norm, lr, coef, step_t, n_tensors, beta1, beta2,
                     n_tensors ? reinterpret_cast<float2*>(bc) : nullptr);
  UNET_LAUNCH_CHECK("adamw8_prepare");
  return 0;
}

extern "C" int unet_adamw8_apply(const float* const* grads_host, int32_t n_tensors, float* const* p_ptrs, const uint32_t* start256,
                                 const uint32_t* numel, const uint32_t* slot, int64_t blocks256, void* m8, void* r8, float* m_scale,
                                 float* r_scale, float* m32, float* v32, const float* coef, const float* bc, float* partial,
                                 double beta1, double beta2, float eps, float weight_decay, void* stream) {
  UNET_REQUIRE(grads_host && p_ptrs && start256 && numel && slot && m8 && r8 && m_scale && r_scale && m32 && v32 && coef && bc,
               "adamw8_apply: null pointer");
  UNET_REQUIRE(n_tensors >= 1 && n_tensors <= UNET_OPT_MAX_TENSORS, "adamw8_apply: 1..%d tensors per call, got %d",
               UNET_OPT_MAX_TENSORS, n_tensors);
  UNET_REQUIRE(blocks256 > 0 && blocks256 < (1ll << 31), "adamw8_apply: %lld blocks", (long long)blocks256);
  UNET_REQUIRE(!((reinterpret_cast<uintptr_t>(m8) | reinterpret_cast<uintptr_t>(r8)) & 3), "adamw8_apply: code buffers must be 4-byte aligned");
  Adam8 k = {};
  k.p = p_ptrs; k.start = start256; k.numel = numel; k.slot = slot;
  k.m8 = static_cast<unsigned char*>(m8); k.r8 = static_cast<unsigned char*>(r8);
  k.sm = m_scale; k.sr = r_scale; k.m32 = m32; k.v32 = v32; k.coef = coef; k.bc = reinterpret_cast<const float2*>(bc);
  k.partial = partial; k.beta1 = (float)beta1; k.beta2 = (float)beta2; k.grow1 = (float)(1.0 - beta1); k.grow2 = (float)(1.0 - beta2);
  k.eps = eps; k.weight_decay = weight_decay; k.n = n_tensors;
  GradPtrs gp;
  for (int i = 0; i < UNET_OPT_MAX_TENSORS; ++i) gp.g[i] = i < n_tensors ? grads_host[i] : nullptr;
  hipLaunchKernelGGL(adamw8_apply_kernel, dim3(unet_adamw8_blocks(blocks256)), dim3(A8_THREADS), 0, static_cast<hipStream_t>(stream),
                     k, gp);
  UNET_LAUNCH_CHECK("adamw8_apply");
  return 0;
}
