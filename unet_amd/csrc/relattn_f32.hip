// The fp32 form of relattn.hip (parity runs): exact products on v_mfma_f32_16x16x4_f32 with the tiles of attn_f32.hip, written
// for clarity.  The bias is one LDS read per score; the sums of dS by offset go into a wave's own LDS array, the four lane
// groups (whose offsets overlap) one after the other, so the order of every sum is fixed.
#include "attn_f32_tiles.h"
#include "relattn.h"

namespace {

struct Place { int head, n, len, tile; long long base, stat; };
__device__ __forceinline__ Place place(const RelK& p) {
  const int nt = (p.l + A32_ROWS - 1) / A32_ROWS;
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
template <int HDP> struct Fetch {
  static constexpr int CH = HDP / 4, TOTAL = A32_BK * CH, N = (TOTAL + A32_THREADS - 1) / A32_THREADS;
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

template <int HDP>
__global__ __launch_bounds__(A32_THREADS, 1) void rel32_fwd_kernel(const RelK p) {
  constexpr int LD = HDP + 4, DT = HDP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  float* kt = reinterpret_cast<float*>(smem_raw);
  float* vt = kt + A32_BK * LD;
  float* bias = vt + A32_BK * LD;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, g = lane >> 4;
  const Place o = place(p);
  const int q0w = o.tile * A32_ROWS + wave * 16, qrow = q0w + l15;
  const bool row_ok = qrow < o.len;
  const float* kslab = static_cast<const float*>(p.k) + o.base;
  const float* vslab = static_cast<const float*>(p.v) + o.base;

  f32x4 qreg[DT], oacc[DT];
  load_rows<HDP>(qreg, static_cast<const float*>(p.q) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
#pragma unroll
  for (int d = 0; d < DT; ++d) oacc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  rel_fill(p, o.head, bias, tid, A32_THREADS);
  float m = -INFINITY, lsum = 0.f;
  const int end = o.tile * A32_ROWS < o.len ? o.len : 0;            // (uniform) nothing to do behind the window's length
  Fetch<HDP> fk, fv;
  fk.get(kslab, 0, end, p.c, p.hd, tid);
  fv.get(vslab, 0, end, p.c, p.hd, tid);
  for (int key0 = 0; key0 < end; key0 += A32_BK) {
    __syncthreads();
    fk.put(kt, tid);
    fv.put(vt, tid);
    __syncthreads();
    fk.get(kslab, key0 + A32_BK, end, p.c, p.hd, tid);
    fv.get(vslab, key0 + A32_BK, end, p.c, p.hd, tid);
    f32x4 st[2];
    float mx = -INFINITY;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      st[s] = rows_dot<HDP>(kt, 16 * s, qreg, l15, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * s + 4 * g + i;
        const float b = bias[max(-p.sat, min(key - qrow, p.sat)) + p.sat + REL_PAD];
        st[s][i] = key < o.len ? fmaf(st[s][i], p.scale_log2, b) : -INFINITY;
        mx = fmaxf(mx, st[s][i]);
      }
    }
    mx = group_max(mx);
    const float m_new = fmaxf(m, mx), ref = m_new == -INFINITY ? 0.f : m_new;       // a row with nothing to see yet
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    float ps = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) { st[s][i] = __builtin_amdgcn_exp2f(st[s][i] - ref); ps += st[s][i]; }
    lsum = lsum * alpha + group_sum(ps);
    m = m_new;
#pragma unroll
    for (int d = 0; d < DT; ++d) oacc[d] *= alpha;
    rows_acc<HDP>(oacc, vt, 0, st[0], l15, g);
    rows_acc<HDP>(oacc, vt, 16, st[1], l15, g);
  }
  if (qrow < p.l) {
    const bool seen = row_ok && lsum > 0.f, spoiled = row_ok && lsum != lsum;
    const float inv = seen ? 1.f / lsum : spoiled ? lsum : 0.f;
    if (p.lse && g == 0) p.lse[o.stat + qrow] = seen ? m + __builtin_amdgcn_logf(lsum) : spoiled ? lsum : INFINITY;
    float* yp = static_cast<float*>(p.out) + o.base + (long long)qrow * p.c;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (16 * d + 4 * g < p.hd) *reinterpret_cast<f32x4*>(yp + 16 * d + 4 * g) = inv == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : oacc[d] * inv;
  }
}

__global__ __launch_bounds__(A32_THREADS) void rel32_rowdot_kernel(const RelK p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.y, len = rel_length(p, n), row = blockIdx.x * 4 + wave;
  if (row >= p.l) return;
  const float* dop = static_cast<const float*>(p.dout) + ((long long)n * p.l + row) * p.c;
  const float* op = static_cast<const float*>(p.out) + ((long long)n * p.l + row) * p.c;
  for (int head = 0; head < p.nh; ++head) {
    float acc = 0.f;
    if (row < len)
      for (int d = lane; d < p.hd; d += 64) acc = fmaf(dop[head * p.hd + d], op[head * p.hd + d], acc);
    acc = wave_sum(acc);
    if (lane == 0) p.delta[((long long)n * p.nh + head) * p.l + row] = acc;
  }
}

template <int HDP>
__global__ __launch_bounds__(A32_THREADS, 1) void rel32_dq_kernel(const RelK p) {
  constexpr int LD = HDP + 4, DT = HDP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  const int w = 2 * p.sat + 1;
  float* kt = reinterpret_cast<float*>(smem_raw);
  float* vt = kt + A32_BK * LD;
  float* bias = vt + A32_BK * LD;
  float* sums = bias + rel_width(p.sat);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, g = lane >> 4;
  const Place o = place(p);
  const int qrow = o.tile * A32_ROWS + wave * 16 + l15;
  const bool row_ok = qrow < o.len;
  const float* kslab = static_cast<const float*>(p.k) + o.base;
  const float* vslab = static_cast<const float*>(p.v) + o.base;

  f32x4 qreg[DT], doreg[DT], acc[DT];
  load_rows<HDP>(qreg, static_cast<const float*>(p.q) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
  load_rows<HDP>(doreg, static_cast<const float*>(p.dout) + o.base + (long long)qrow * p.c, row_ok, g, p.hd);
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  rel_fill(p, o.head, bias, tid, A32_THREADS);
  if (p.part)
    for (int i = tid; i < 4 * w; i += A32_THREADS) sums[i] = 0.f;
  auto add = [](float* at, float v) { __hip_atomic_fetch_add(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
  const float lse = row_ok ? p.lse[o.stat + qrow] : INFINITY;          // rows past the end: p = 0
  const float delta = row_ok ? p.delta[o.stat + qrow] : 0.f;
  float fneg = 0.f, fpos = 0.f;                          // sums beyond the band
  const int end = o.tile * A32_ROWS < o.len ? o.len : 0;
  Fetch<HDP> fk, fv;
  fk.get(kslab, 0, end, p.c, p.hd, tid);
  fv.get(vslab, 0, end, p.c, p.hd, tid);
  for (int key0 = 0; key0 < end; key0 += A32_BK) {
    __syncthreads();
    fk.put(kt, tid);
    fv.put(vt, tid);
    __syncthreads();
    fk.get(kslab, key0 + A32_BK, end, p.c, p.hd, tid);
    fv.get(vslab, key0 + A32_BK, end, p.c, p.hd, tid);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 st = rows_dot<HDP>(kt, 16 * s, qreg, l15, g);
      const f32x4 dp = rows_dot<HDP>(vt, 16 * s, doreg, l15, g);
      int at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * s + 4 * g + i;
        at[i] = max(-p.sat, min(key - qrow, p.sat)) + p.sat;
        const float b = bias[at[i] + REL_PAD];
        const float pe = key < o.len ? __builtin_amdgcn_exp2f(fmaf(st[i], p.scale_log2, b - lse)) : 0.f;
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
      rows_acc<HDP>(acc, kt, 16 * s, st, l15, g);
    }
  }
  if (qrow < p.l) {
    float* yp = static_cast<float*>(p.dq) + o.base + (long long)qrow * p.c;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (16 * d + 4 * g < p.hd) *reinterpret_cast<f32x4*>(yp + 16 * d + 4 * g) = row_ok ? acc[d] * p.scale : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (p.part) {
    fneg = wave_sum(fneg);
    fpos = wave_sum(fpos);
    if (lane == 0) {
      add(sums + wave * w, fneg);
      add(sums + wave * w + w - 1, fpos);
    }
    __syncthreads();
    const int nt = (p.l + A32_ROWS - 1) / A32_ROWS;
    float* row = p.part + ((long long)o.head * p.parts + o.n * nt + o.tile) * w;
    for (int i = tid; i < w; i += A32_THREADS) row[i] = (sums[i] + sums[w + i]) + (sums[2 * w + i] + sums[3 * w + i]);
  }
}

template <int HDP>
__global__ __launch_bounds__(A32_THREADS, 1) void rel32_dkv_kernel(const RelK p) {
  constexpr int LD = HDP + 4, DT = HDP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  float* qtile = reinterpret_cast<float*>(smem_raw);
  float* dtile = qtile + A32_BK * LD;
  float* stats = dtile + A32_BK * LD;                   // [0..31] lse, [32..63] delta of the tile's rows
  float* bias = stats + 2 * A32_BK;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, g = lane >> 4;
  const Place o = place(p);
  const int key = o.tile * A32_ROWS + wave * 16 + l15;
  const bool key_ok = key < o.len;
  const long long kvo = o.base + (long long)key * p.c;
  const float* qslab = static_cast<const float*>(p.q) + o.base;
  const float* dslab = static_cast<const float*>(p.dout) + o.base;

  f32x4 kreg[DT], vreg[DT], dka[DT], dva[DT];
  load_rows<HDP>(kreg, static_cast<const float*>(p.k) + kvo, key_ok, g, p.hd);
  load_rows<HDP>(vreg, static_cast<const float*>(p.v) + kvo, key_ok, g, p.hd);
#pragma unroll
  for (int d = 0; d < DT; ++d) { dka[d] = f32x4{0.f, 0.f, 0.f, 0.f}; dva[d] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  rel_fill(p, o.head, bias, tid, A32_THREADS);
  const int end = o.tile * A32_ROWS < o.len ? o.len : 0;
  Fetch<HDP> fq, fd;
  float stat = 0.f;
  auto get = [&](int row0) {
    fq.get(qslab, row0, end, p.c, p.hd, tid);
    fd.get(dslab, row0, end, p.c, p.hd, tid);
    if (tid < 2 * A32_BK) {
      const int r = row0 + (tid & (A32_BK - 1));
      stat = r < end ? (tid < A32_BK ? p.lse[o.stat + r] : p.delta[o.stat + r]) : (tid < A32_BK ? INFINITY : 0.f);
    }
  };
  get(0);
  for (int row0 = 0; row0 < end; row0 += A32_BK) {
    __syncthreads();
    fq.put(qtile, tid);
    fd.put(dtile, tid);
    if (tid < 2 * A32_BK) stats[tid] = stat;
    __syncthreads();
    get(row0 + A32_BK);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 st = rows_dot<HDP>(qtile, 16 * s, kreg, l15, g);
      f32x4 dp = rows_dot<HDP>(dtile, 16 * s, vreg, l15, g);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int rl = 16 * s + 4 * g + r;
        const float b = bias[max(-p.sat, min(key - row0 - rl, p.sat)) + p.sat + REL_PAD];
        const float pe = __builtin_amdgcn_exp2f(fmaf(st[r], p.scale_log2, b - stats[rl]));   // rows past the end: lse = inf
        st[r] = pe;
        dp[r] = pe * (dp[r] - stats[A32_BK + rl]);
      }
      rows_acc<HDP>(dva, dtile, 16 * s, st, l15, g);
      rows_acc<HDP>(dka, qtile, 16 * s, dp, l15, g);
    }
  }
  if (key < p.l) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (16 * d + 4 * g < p.hd) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.dk) + kvo + 16 * d + 4 * g) = key_ok ? dka[d] * p.scale : zero;
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.dv) + kvo + 16 * d + 4 * g) = key_ok ? dva[d] : zero;
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

template <int HDP> int launch_fwd32(const RelK& p, hipStream_t st) {
  const size_t lds = sizeof(float) * ((size_t)2 * A32_BK * (HDP + 4) + rel_width(p.sat));
  if (set_lds(&rel32_fwd_kernel<HDP>, lds, "rel_attn_fwd (fp32)")) return -1;
  hipLaunchKernelGGL(rel32_fwd_kernel<HDP>, dim3((unsigned)(p.n * p.nh * cdiv(p.l, A32_ROWS))), dim3(A32_THREADS), lds, st, p);
  UNET_LAUNCH_CHECK("rel_attn_fwd (fp32)");
  return 0;
}

template <int HDP> int launch_bwd32(const RelK& p, hipStream_t st) {
  const size_t tiles = (size_t)2 * A32_BK * (HDP + 4) + rel_width(p.sat);
  const size_t lds_q = sizeof(float) * (tiles + (p.part ? 4 * (2 * (size_t)p.sat + 1) : 0)), lds_kv = sizeof(float) * (tiles + 2 * A32_BK);
  if (set_lds(&rel32_dq_kernel<HDP>, lds_q, "rel_attn_bwd (fp32 dq)")) return -1;
  if (set_lds(&rel32_dkv_kernel<HDP>, lds_kv, "rel_attn_bwd (fp32 dk, dv)")) return -1;
  const dim3 grid((unsigned)(p.n * p.nh * cdiv(p.l, A32_ROWS)));
  hipLaunchKernelGGL(rel32_dq_kernel<HDP>, grid, dim3(A32_THREADS), lds_q, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (fp32 dq)");
  hipLaunchKernelGGL(rel32_dkv_kernel<HDP>, grid, dim3(A32_THREADS), lds_kv, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (fp32 dk, dv)");
  return 0;
}

#define REL32_DISPATCH(fn, p, st)             \
  do {                                        \
    if ((p).hd <= 16) return fn<16>(p, st);   \
    if ((p).hd <= 32) return fn<32>(p, st);   \
    if ((p).hd <= 64) return fn<64>(p, st);   \
    if ((p).hd <= 128) return fn<128>(p, st); \
    return fn<256>(p, st);                    \
  } while (0)

}  // namespace

int unet_rel_attn_fwd_f32(const RelK& p, hipStream_t st) { REL32_DISPATCH(launch_fwd32, p, st); }

int unet_rel_attn_bwd_f32(const RelK& p, hipStream_t st) {
  hipLaunchKernelGGL(rel32_rowdot_kernel, dim3(cdiv(p.l, 4), p.n), dim3(A32_THREADS), 0, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (fp32 rowdot)");
  REL32_DISPATCH(launch_bwd32, p, st);
}
