// The fp32 form of relattn.hip (parity runs): exact products on v_mfma_f32_16x16x4_f32 with the tiles of attn_f32.hip.  The bias is
// one LDS read per score; the sums of dS by offset go into a wave's own LDS array, the four lane groups (whose offsets overlap) one
// after the other, so the order of every sum is fixed.
//
// A workgroup's four waves own 16 rows each and share the tiles of the other side (32 rows a step).  Launches with few such
// workgroups (rel32_rows) are SPLIT: the four waves own the same 16 rows, take every fourth piece of 32 of the other side and add up
// at the end, so a wave walks a quarter of the length and four times the CUs work.  [3, 301, 160], 4 heads (60 workgroups or 228):
// forward 26.3 -> 14.2 us, dQ 38.1 -> 17.8, dK and dV 36.4 -> 16.8; a wave alone on its SIMD is bound by its chain of products.
#include "attn_f32_tiles.h"
#include "relattn.h"

namespace {

// Scores stay in the natural domain and lse is kept as two planes, the maximum and log2 of the sum: in P = exp(s - m) / l the
// difference of two scores is exact where one key dominates, so that P is as good there as an exp of 32 bits, and dP - delta keeps its
// digits (one rounded sum m + log2 l, in the log2 domain, cost up to 4 times the error of dQ and the table's gradient).
__device__ __forceinline__ float rel32_exp(float diff, float lg = 0.f) { return __builtin_amdgcn_exp2f(fmaf(diff, REL_LOG2E, -lg)); }

template <bool SPLIT> struct Shape {
  static constexpr int ROWS = SPLIT ? 16 : A32_ROWS;          // rows a workgroup owns
  static constexpr int STEP = SPLIT ? 4 * A32_BK : A32_BK;    // rows of the other side a step
};

struct Place { int head, n, len, tile; long long base, stat; };
template <int ROWS> __device__ __forceinline__ Place place(const RelK& p) {
  const int nt = (p.l + ROWS - 1) / ROWS;
  int wg = blockIdx.x;
  Place o;
  o.tile = wg % nt; wg /= nt;
  o.head = wg % p.nh;
  o.n = wg / p.nh;
  o.len = rel_length(p, o.n);
  o.base = (long long)o.n * p.l * p.c + o.head * p.hd;
  o.stat = ((long long)o.n * p.nh + o.head) * p.l;
  return o;
}

// load_tile of attn_f32_tiles.h in two halves: the next tile is fetched into registers while this one is worked on
template <int HDP, int ROWS> struct Fetch {
  static constexpr int CH = HDP / 4, TOTAL = ROWS * CH, N = (TOTAL + A32_THREADS - 1) / A32_THREADS;
  f32x4 v[N];
  __device__ __forceinline__ void get(const float* slab, int row0, int l, int ld, int hd, int tid) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = tid + k * A32_THREADS, r = i / CH, ch = i % CH;
      v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (i < TOTAL && row0 + r < l && ch * 4 < hd) v[k] = *reinterpret_cast<const f32x4*>(slab + (long long)(row0 + r) * ld + ch * 4);
    }
  }
  __device__ __forceinline__ void put(float* tile, int tid) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = tid + k * A32_THREADS;
      if (i < TOTAL) *reinterpret_cast<f32x4*>(tile + i / CH * (HDP + 4) + i % CH * 4) = v[k];
    }
  }
};

// SPLIT: the waves' accumulators meet in `buf` (free LDS, 64 HDP floats); add(dt, f) sums part dt, f[w] the factor of wave w's
template <int DT> struct Join {
  float* buf;
  __device__ __forceinline__ void put(const f32x4 (&acc)[DT], int wave, int lane) const {
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(buf + ((wave * DT + d) * 64 + lane) * 4) = acc[d];
  }
  __device__ __forceinline__ f32x4 add(int d, int lane, const float (&f)[4]) const {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) s += *reinterpret_cast<const f32x4*>(buf + ((w * DT + d) * 64 + lane) * 4) * f[w];
    return s;
  }
};

template <int HDP, bool SPLIT>
__global__ __launch_bounds__(A32_THREADS, 1) void rel32_fwd_kernel(const RelK p) {
  constexpr int LD = HDP + 4, DT = HDP / 16, ROWS = Shape<SPLIT>::ROWS, STEP = Shape<SPLIT>::STEP;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  float* kt = reinterpret_cast<float*>(smem_raw);
  float* vt = kt + STEP * LD;
  float* bias = vt + STEP * LD;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, g = lane >> 4;
  const Place o = place<ROWS>(p);
  const int qrow = o.tile * ROWS + (SPLIT ? 0 : wave * 16) + l15, mine = SPLIT ? wave * A32_BK : 0;    // the wave's piece of a step
  const bool row_ok = qrow < o.len;
  const float* kslab = static_cast<const float*>(p.k) + o.base;
  const float* vslab = static_cast<const float*>(p.v) + o.base;

  f32x4 qreg[DT], oacc[DT];
  load_rows<HDP>(qreg, static_cast<const float*>(p.q) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
#pragma unroll
  for (int d = 0; d < DT; ++d) oacc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  rel_fill(p, o.head, bias, tid, A32_THREADS, 1.f);
  float m = -INFINITY, lsum = 0.f;
  const int end = o.tile * ROWS < o.len ? o.len : 0;            // (uniform) nothing to do behind the window's length
  Fetch<HDP, STEP> fk, fv;
  fk.get(kslab, 0, end, p.c, p.hd, tid);
  fv.get(vslab, 0, end, p.c, p.hd, tid);
  for (int step = 0; step < end; step += STEP) {
    __syncthreads();
    fk.put(kt, tid);
    fv.put(vt, tid);
    __syncthreads();
    fk.get(kslab, step + STEP, end, p.c, p.hd, tid);
    fv.get(vslab, step + STEP, end, p.c, p.hd, tid);
    const int key0 = step + mine;
    f32x4 st[2];
    float mx = -INFINITY;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      st[s] = rows_dot<HDP>(kt, mine + 16 * s, qreg, l15, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * s + 4 * g + i;
        const float b = bias[max(-p.sat, min(key - qrow, p.sat)) + p.sat + REL_PAD];
        st[s][i] = key < o.len ? fmaf(st[s][i], p.scale, b) : -INFINITY;
        mx = fmaxf(mx, st[s][i]);
      }
    }
    mx = group_max(mx);
    const float m_new = fmaxf(m, mx), ref = m_new == -INFINITY ? 0.f : m_new;       // a row with nothing to see yet
    const float alpha = m == -INFINITY ? 0.f : rel32_exp(m - m_new);
    float ps = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) { st[s][i] = rel32_exp(st[s][i] - ref); ps += st[s][i]; }
    lsum = lsum * alpha + group_sum(ps);
    m = m_new;
#pragma unroll
    for (int d = 0; d < DT; ++d) oacc[d] *= alpha;
    rows_acc<HDP>(oacc, vt, mine, st[0], l15, g);
    rows_acc<HDP>(oacc, vt, mine + 16, st[1], l15, g);
  }
  float f[4] = {1.f, 0.f, 0.f, 0.f};
  const Join<DT> join{kt};
  if constexpr (SPLIT) {                                             // maxima, sums and accumulators of the four waves
    __syncthreads();
    join.put(oacc, wave, lane);
    if (g == 0) { vt[wave * 32 + l15] = m; vt[wave * 32 + 16 + l15] = lsum; }
    __syncthreads();
    m = fmaxf(fmaxf(vt[l15], vt[32 + l15]), fmaxf(vt[64 + l15], vt[96 + l15]));
    lsum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = vt[w * 32 + l15] == -INFINITY ? 0.f : rel32_exp(vt[w * 32 + l15] - m);
      lsum = fmaf(vt[w * 32 + 16 + l15], f[w], lsum);
    }
  }
  if (qrow < p.l) {
    const bool seen = row_ok && lsum > 0.f, spoiled = row_ok && lsum != lsum;
    const float inv = seen ? 1.f / lsum : spoiled ? lsum : 0.f;
    if (p.lse && g == 0 && (!SPLIT || wave == 0)) {
      p.lse[o.stat + qrow] = seen ? m : spoiled ? lsum : INFINITY;
      p.lse[rel_logs(p) + o.stat + qrow] = seen ? __builtin_amdgcn_logf(lsum) : 0.f;
    }
    float* yp = static_cast<float*>(p.out) + o.base + (long long)qrow * p.c;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (16 * d + 4 * g < p.hd && (!SPLIT || (d & 3) == wave)) {
        const f32x4 x = SPLIT ? join.add(d, lane, f) : oacc[d];
        *reinterpret_cast<f32x4*>(yp + 16 * d + 4 * g) = inv == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x * inv;
      }
  }
}

template <int HDP, bool SPLIT>
__global__ __launch_bounds__(A32_THREADS, 1) void rel32_dq_kernel(const RelK p) {
  constexpr int LD = HDP + 4, DT = HDP / 16, ROWS = Shape<SPLIT>::ROWS, STEP = Shape<SPLIT>::STEP;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  const int w = 2 * p.sat + 1;
  float* kt = reinterpret_cast<float*>(smem_raw);
  float* vt = kt + STEP * LD;
  float* bias = vt + STEP * LD;
  float* sums = bias + rel_width(p.sat);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, g = lane >> 4;
  const Place o = place<ROWS>(p);
  const int qrow = o.tile * ROWS + (SPLIT ? 0 : wave * 16) + l15, mine = SPLIT ? wave * A32_BK : 0;
  const bool row_ok = qrow < o.len;
  const float* kslab = static_cast<const float*>(p.k) + o.base;
  const float* vslab = static_cast<const float*>(p.v) + o.base;

  f32x4 qreg[DT], doreg[DT], acc[DT];
  load_rows<HDP>(qreg, static_cast<const float*>(p.q) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
  load_rows<HDP>(doreg, static_cast<const float*>(p.dout) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  rel_fill(p, o.head, bias, tid, A32_THREADS, 1.f);
  if (p.part)
    for (int i = tid; i < 4 * w; i += A32_THREADS) sums[i] = 0.f;
  auto add = [](float* at, float v) { __hip_atomic_fetch_add(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
  const float m = row_ok ? p.lse[o.stat + qrow] : INFINITY;            // rows past the end: p = 0
  const float lg = row_ok ? p.lse[rel_logs(p) + o.stat + qrow] : 0.f;
  float delta;                                                         // <dO, O>, kept for dK and dV
  {
    f32x4 oreg[DT];
    load_rows<HDP>(oreg, static_cast<const float*>(p.out) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
    double d = 0.0;                          // (its error stays in every dS of the row, where the sums of a bucket cancel)
#pragma unroll
    for (int u = 0; u < DT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) d = fma((double)doreg[u][e], (double)oreg[u][e], d);
    d += __shfl_xor(d, 16, 64);
    delta = (float)(d + __shfl_xor(d, 32, 64));
    if (g == 0 && row_ok && (!SPLIT || wave == 0)) p.delta[o.stat + qrow] = delta;
  }
  float fneg = 0.f, fpos = 0.f;                          // sums beyond the band
  const int end = o.tile * ROWS < o.len ? o.len : 0;
  Fetch<HDP, STEP> fk, fv;
  fk.get(kslab, 0, end, p.c, p.hd, tid);
  fv.get(vslab, 0, end, p.c, p.hd, tid);
  for (int step = 0; step < end; step += STEP) {
    __syncthreads();
    fk.put(kt, tid);
    fv.put(vt, tid);
    __syncthreads();
    fk.get(kslab, step + STEP, end, p.c, p.hd, tid);
    fv.get(vslab, step + STEP, end, p.c, p.hd, tid);
    const int key0 = step + mine;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 st = rows_dot<HDP>(kt, mine + 16 * s, qreg, l15, g);
      const f32x4 dp = rows_dot<HDP>(vt, mine + 16 * s, doreg, l15, g);
      int at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * s + 4 * g + i;
        at[i] = max(-p.sat, min(key - qrow, p.sat)) + p.sat;
        const float b = bias[at[i] + REL_PAD];
        const float pe = key < o.len ? rel32_exp(fmaf(st[i], p.scale, b) - m, lg) : 0.f;
        st[i] = pe * (dp[i] - delta);
      }
      if (p.part) {
        // inside the band the sixteen rows of a lane group have sixteen offsets; beyond it they share one: kept in a register
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int off = key0 + 16 * s + 4 * g + i - qrow;
          const bool neg = off <= -p.sat, pos = off >= p.sat;
          fneg += neg ? st[i] : 0.f;
          fpos += pos ? st[i] : 0.f;
          if (__any(!neg && !pos)) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (g == q && !neg && !pos) add(sums + wave * w + at[i], st[i]);
          }
        }
      }
      rows_acc<HDP>(acc, kt, mine + 16 * s, st, l15, g);
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f};
  const Join<DT> join{kt};
  if constexpr (SPLIT) {
    __syncthreads();
    join.put(acc, wave, lane);
    __syncthreads();
  }
  if (qrow < p.l) {
    float* yp = static_cast<float*>(p.dq) + o.base + (long long)qrow * p.c;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (16 * d + 4 * g < p.hd && (!SPLIT || (d & 3) == wave)) {
        const f32x4 x = SPLIT ? join.add(d, lane, one) : acc[d];
        *reinterpret_cast<f32x4*>(yp + 16 * d + 4 * g) = row_ok ? x * p.scale : f32x4{0.f, 0.f, 0.f, 0.f};
      }
  }
  if (p.part) {
    fneg = wave_sum(fneg);
    fpos = wave_sum(fpos);
    if (lane == 0) {
      add(sums + wave * w, fneg);
      add(sums + wave * w + w - 1, fpos);
    }
    __syncthreads();
    const int nt = (p.l + ROWS - 1) / ROWS;
    float* row = p.part + ((long long)o.head * p.parts + o.n * nt + o.tile) * w;
    for (int i = tid; i < w; i += A32_THREADS) row[i] = (sums[i] + sums[w + i]) + (sums[2 * w + i] + sums[3 * w + i]);
  }
}

template <int HDP, bool SPLIT>
__global__ __launch_bounds__(A32_THREADS, 1) void rel32_dkv_kernel(const RelK p) {
  constexpr int LD = HDP + 4, DT = HDP / 16, ROWS = Shape<SPLIT>::ROWS, STEP = Shape<SPLIT>::STEP;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  float* qtile = reinterpret_cast<float*>(smem_raw);
  float* dtile = qtile + STEP * LD;
  float* stats = dtile + STEP * LD;                     // [STEP] maxima, [STEP] log2 of the sums, [STEP] delta of the step's rows
  float* bias = stats + 3 * STEP;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, g = lane >> 4;
  const Place o = place<ROWS>(p);
  const int key = o.tile * ROWS + (SPLIT ? 0 : wave * 16) + l15, mine = SPLIT ? wave * A32_BK : 0;
  const bool key_ok = key < o.len;
  const long long kvo = o.base + (long long)key * p.c;
  const float* qslab = static_cast<const float*>(p.q) + o.base;
  const float* dslab = static_cast<const float*>(p.dout) + o.base;

  f32x4 kreg[DT], vreg[DT], dka[DT], dva[DT];
  load_rows<HDP>(kreg, static_cast<const float*>(p.k) + kvo, key_ok, g, p.hd);
  load_rows<HDP>(vreg, static_cast<const float*>(p.v) + kvo, key_ok, g, p.hd);
#pragma unroll
  for (int d = 0; d < DT; ++d) { dka[d] = f32x4{0.f, 0.f, 0.f, 0.f}; dva[d] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  rel_fill(p, o.head, bias, tid, A32_THREADS, 1.f);
  const int end = o.tile * ROWS < o.len ? o.len : 0;
  Fetch<HDP, STEP> fq, fd;
  constexpr int NS = (3 * STEP + A32_THREADS - 1) / A32_THREADS;
  float stat[NS];
  auto get = [&](int row0) {
    fq.get(qslab, row0, end, p.c, p.hd, tid);
    fd.get(dslab, row0, end, p.c, p.hd, tid);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int i = tid + k * A32_THREADS, which = i / STEP, r = row0 + i % STEP;
      stat[k] = which == 0 ? INFINITY : 0.f;
      if (which < 3 && r < end) stat[k] = which == 0 ? p.lse[o.stat + r] : which == 1 ? p.lse[rel_logs(p) + o.stat + r] : p.delta[o.stat + r];
    }
  };
  get(0);
  for (int step = 0; step < end; step += STEP) {
    __syncthreads();
    fq.put(qtile, tid);
    fd.put(dtile, tid);
#pragma unroll
    for (int k = 0; k < NS; ++k)
      if (tid + k * A32_THREADS < 3 * STEP) stats[tid + k * A32_THREADS] = stat[k];
    __syncthreads();
    get(step + STEP);
    const int row0 = step + mine;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 st = rows_dot<HDP>(qtile, mine + 16 * s, kreg, l15, g);
      f32x4 dp = rows_dot<HDP>(dtile, mine + 16 * s, vreg, l15, g);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int rl = 16 * s + 4 * g + r;
        const float b = bias[max(-p.sat, min(key - row0 - rl, p.sat)) + p.sat + REL_PAD];
        const float pe = rel32_exp(fmaf(st[r], p.scale, b) - stats[mine + rl], stats[STEP + mine + rl]);   // rows past the end: inf
        st[r] = pe;
        dp[r] = pe * (dp[r] - stats[2 * STEP + mine + rl]);
      }
      rows_acc<HDP>(dva, dtile, mine + 16 * s, st, l15, g);
      rows_acc<HDP>(dka, qtile, mine + 16 * s, dp, l15, g);
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f};
  const Join<DT> jk{qtile}, jv{dtile};
  if constexpr (SPLIT) {
    __syncthreads();
    jk.put(dka, wave, lane);
    jv.put(dva, wave, lane);
    __syncthreads();
  }
  if (key < p.l) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (16 * d + 4 * g < p.hd && (!SPLIT || (d & 3) == wave)) {
        const f32x4 xk = SPLIT ? jk.add(d, lane, one) : dka[d], xv = SPLIT ? jv.add(d, lane, one) : dva[d];
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.dk) + kvo + 16 * d + 4 * g) = key_ok ? xk * p.scale : zero;
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.dv) + kvo + 16 * d + 4 * g) = key_ok ? xv : zero;
      }
  }
}

template <typename K> int set_lds(K kernel, size_t bytes, const char* what) {
  if (bytes > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    UNET_REQUIRE(e == hipSuccess, "%s: hipFuncSetAttribute failed: %s", what, hipGetErrorString(e));
  }
  return 0;
}

template <int HDP, bool SPLIT> int launch_fwd32(const RelK& p, hipStream_t st) {
  typedef Shape<SPLIT> S;
  const size_t lds = sizeof(float) * ((size_t)2 * S::STEP * (HDP + 4) + rel_width(p.sat));
  if (set_lds(&rel32_fwd_kernel<HDP, SPLIT>, lds, "rel_attn_fwd (fp32)")) return -1;
  const dim3 grid((unsigned)(p.n * p.nh * cdiv(p.l, S::ROWS)));
  hipLaunchKernelGGL((rel32_fwd_kernel<HDP, SPLIT>), grid, dim3(A32_THREADS), lds, st, p);
  UNET_LAUNCH_CHECK("rel_attn_fwd (fp32)");
  return 0;
}

template <int HDP, bool SPLIT> int launch_bwd32(const RelK& p, hipStream_t st) {
  typedef Shape<SPLIT> S;
  const size_t tiles = (size_t)2 * S::STEP * (HDP + 4) + rel_width(p.sat);
  const size_t lds_q = sizeof(float) * (tiles + (p.part ? 4 * (2 * (size_t)p.sat + 1) : 0)), lds_kv = sizeof(float) * (tiles + 3 * S::STEP);
  if (set_lds(&rel32_dq_kernel<HDP, SPLIT>, lds_q, "rel_attn_bwd (fp32 dq)")) return -1;
  if (set_lds(&rel32_dkv_kernel<HDP, SPLIT>, lds_kv, "rel_attn_bwd (fp32 dk, dv)")) return -1;
  const dim3 grid((unsigned)(p.n * p.nh * cdiv(p.l, S::ROWS)));
  hipLaunchKernelGGL((rel32_dq_kernel<HDP, SPLIT>), grid, dim3(A32_THREADS), lds_q, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (fp32 dq)");
  hipLaunchKernelGGL((rel32_dkv_kernel<HDP, SPLIT>), grid, dim3(A32_THREADS), lds_kv, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (fp32 dk, dv)");
  return 0;
}

#define REL32_DISPATCH(fn, p, st)                                           \
  do {                                                                      \
    const bool split = rel32_rows((p).n, (p).l, (p).nh, (p).hd) < A32_ROWS; \
    if ((p).hd <= 16) return split ? fn<16, true>(p, st) : fn<16, false>(p, st);    \
    if ((p).hd <= 32) return split ? fn<32, true>(p, st) : fn<32, false>(p, st);    \
    if ((p).hd <= 64) return split ? fn<64, true>(p, st) : fn<64, false>(p, st);    \
    if ((p).hd <= 128) return split ? fn<128, true>(p, st) : fn<128, false>(p, st); \
    return fn<256, false>(p, st);                                           \
  } while (0)

}  // namespace

int unet_rel_attn_fwd_f32(const RelK& p, hipStream_t st) { REL32_DISPATCH(launch_fwd32, p, st); }

int unet_rel_attn_bwd_f32(const RelK& p, hipStream_t st) {
  REL32_DISPATCH(launch_bwd32, p, st);
}
