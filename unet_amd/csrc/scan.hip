// Gated linear recurrence along the row axis of channels-last tensors, forward, backward and one row at a time:
//   f_t = sigmoid(g_t),   h_t = f_t h_{t-1} + (1 - f_t) x_t          (per window and channel; reverse: from the last row)
// Backward, with the adjoint lam_t = dh_t + f_{t+1} lam_{t+1}:
//   dx_t = (1 - f_t) lam_t,   dg_t = lam_t (h_{t-1} - x_t) f_t (1 - f_t),   dh_0 = f_1 lam_1
//
// A span of rows acts on the state as h -> A h + B, and two spans compose as (A2 A1, A2 B1 + B2): the recurrence is a scan
// of such pairs.  A workgroup owns CL * V channels of one window and walks the rows in tiles of 64: a thread holds R = 64 /
// groups consecutive rows of V channels in registers, reduces them to (A, B), the groups exchange their pairs through LDS,
// and every thread replays its rows from the state in front of them.  Each input is read once and each output written
// once; the next tile's loads are issued before this tile's exchange.  LDS is double-buffered: one barrier a tile.
// Backward walks the tiles from the last to the first.  It does not read h: the forward pass leaves the fp32 state in front
// of every tile ([n][tiles][c], 1/64 of a value a row) and the tile's states are recomputed from it, so h_{t-1} has not been
// rounded to the storage type.  With mu_t = f_t lam_t a span acts on mu as mu -> A mu + Bm with the SAME A.
//
// Few windows with many rows cannot fill 256 CUs that way.  Their rows are split into segments: a first launch reduces each
// segment to its pair (reads two of the inputs a second time), and a segment's workgroup composes the pairs in front of it.
//
// Everything between loads and stores is fp32.  sigmoid: with t = exp(-|g|), small = t / (1 + t), big = 1 - small; both sides
// keep full relative precision where 1 - f would cancel.
#include "common.h"

namespace {

constexpr int SC_THREADS = 512;
constexpr int SC_TILE = 64;      // rows of a tile, and the distance of the kept states
constexpr float LOG2E = 1.4426950408889634f;

struct ScanK {
  const void *x, *g, *dh;        // [n][l][ld]
  void *h, *dx, *dg;             // [n][l][c]
  const float *h0, *dlast;       // [n][c] or null
  float *last, *dh0;             // [n][c] or null
  float* states;                 // [n][tiles][c] or null: state in front of every tile
  float2* agg;                   // [n][segs][c] pairs, or null (one segment)
  long long x_ns, x_ld, g_ns, g_ld, dh_ns, dh_ld;
  int n, l, c, tiles, segs, seg_tiles, ncb, reverse;
};

// V consecutive values of a row
template <typename T, int V> struct Raw;
template <> struct Raw<float, 1> { typedef float type; };
template <> struct Raw<float, 2> { typedef f32x2 type; };
template <> struct Raw<__bf16, 1> { typedef unsigned short type; };
template <> struct Raw<__bf16, 2> { typedef unsigned int type; };
template <> struct Raw<__bf16, 4> { typedef u32x2 type; };

template <typename T, int V> __device__ __forceinline__ void unpack(const typename Raw<T, V>::type& r, float (&f)[V]) {
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (V == 1) f[0] = r;
    else { f[0] = r[0]; f[1] = r[1]; }
  } else {
    if constexpr (V == 1) f[0] = __builtin_bit_cast(float, (unsigned)r << 16);
    else if constexpr (V == 2) {
      f[0] = __builtin_bit_cast(float, r << 16);
      f[1] = __builtin_bit_cast(float, r & 0xffff0000u);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[2 * i] = __builtin_bit_cast(float, r[i] << 16);
        f[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xffff0000u);
      }
    }
  }
}
template <typename T, int V> __device__ __forceinline__ void put(T* p, const float (&f)[V]) {
  typedef __attribute__((ext_vector_type(V))) T vec;
  if constexpr (V == 1) *p = (T)f[0];
  else {
    vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)f[i];
    *reinterpret_cast<vec*>(p) = v;
  }
}

__device__ __forceinline__ void gate(float g, float& f, float& keep) {     // f = sigmoid(g), keep = 1 - f
  const float t = __builtin_amdgcn_exp2f(-fabsf(g) * LOG2E);
  const float small = t * __builtin_amdgcn_rcpf(1.f + t);
  const float big = 1.f - small;
  f = g >= 0.f ? big : small;
  keep = g >= 0.f ? small : big;
  if (g != g) f = keep = g;
}

// one thread's rows of a tile: raw values, loaded a tile ahead
template <typename T, int V, int R> struct Rows {
  typedef typename Raw<T, V>::type raw;
  raw r[R];
  // rows t0 .. t0+R-1 (walk order); rows at or past l are not read
  __device__ __forceinline__ void load(const T* base, long long ld, int t0, int l, int reverse) {
    if (t0 + R <= l) {
      const T* p = base + (long long)(reverse ? l - 1 - t0 : t0) * ld;
      const long long step = reverse ? -ld : ld;
#pragma unroll
      for (int i = 0; i < R; ++i) r[i] = *reinterpret_cast<const raw*>(p + i * step);
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        r[i] = raw{};
        if (t0 + i < l) r[i] = *reinterpret_cast<const raw*>(base + (long long)(reverse ? l - 1 - t0 - i : t0 + i) * ld);
      }
    }
  }
};

// start value of segment `seg`: the pairs of the segments before it (walk order DIR) applied to `s`
template <int V, int DIR>
__device__ __forceinline__ void compose(const ScanK& p, int n, int c, int seg, bool ok, float (&s)[V]) {
  if (!p.agg || !ok) return;
  const float2* a = p.agg + (long long)n * p.segs * p.c + c;
  if (DIR > 0) {
    for (int k = 0; k < seg; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) { const float2 ab = a[(long long)k * p.c + v]; s[v] = fmaf(ab.x, s[v], ab.y); }
  } else {
    for (int k = p.segs - 1; k > seg; --k)
#pragma unroll
      for (int v = 0; v < V; ++v) { const float2 ab = a[(long long)k * p.c + v]; s[v] = fmaf(ab.x, s[v], ab.y); }
  }
}

template <typename T, int V, int CL>
__global__ __launch_bounds__(SC_THREADS) void scan_fwd_kernel(const ScanK p) {
  constexpr int G = SC_THREADS / CL, R = SC_TILE / G;
  __shared__ float sa[2][G][CL * V], sb[2][G][CL * V];
  const int cl = threadIdx.x % CL, grp = threadIdx.x / CL;
  const int n = blockIdx.x / p.ncb, c = (blockIdx.x % p.ncb) * CL * V + cl * V;
  const int seg = blockIdx.y;
  const bool ok = c < p.c;                         // c % V == 0 and p.c % V == 0: a thread's channels are all in or all out
  const int cc = ok ? c : 0;
  const T* x = static_cast<const T*>(p.x) + n * p.x_ns + cc;
  const T* g = static_cast<const T*>(p.g) + n * p.g_ns + cc;
  T* h = static_cast<T*>(p.h) + (long long)n * p.l * p.c + cc;

  float s[V];                                      // state in front of the tile (the same in every group)
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = p.h0 ? p.h0[(long long)n * p.c + cc + v] : 0.f;
  compose<V, 1>(p, n, cc, seg, ok, s);

  const int first = seg * p.seg_tiles, end = min(p.tiles, first + p.seg_tiles);
  Rows<T, V, R> rx, rg;
  rx.load(x, p.x_ld, first * SC_TILE + grp * R, p.l, p.reverse);
  rg.load(g, p.g_ld, first * SC_TILE + grp * R, p.l, p.reverse);
  for (int tile = first; tile < end; ++tile) {
    const int t0 = tile * SC_TILE + grp * R, buf = tile & 1;
    float f[R][V], b[R][V], A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float xv[V], gv[V];
      unpack<T, V>(rx.r[i], xv);
      unpack<T, V>(rg.r[i], gv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float keep;
        gate(gv[v], f[i][v], keep);
        b[i][v] = keep * xv[v];
        if (t0 + i >= p.l) { f[i][v] = 1.f; b[i][v] = 0.f; }
        A[v] *= f[i][v];
        B[v] = fmaf(f[i][v], B[v], b[i][v]);
      }
    }
    if (tile + 1 < end) {
      rx.load(x, p.x_ld, t0 + SC_TILE, p.l, p.reverse);
      rg.load(g, p.g_ld, t0 + SC_TILE, p.l, p.reverse);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { sa[buf][grp][cl * V + v] = A[v]; sb[buf][grp][cl * V + v] = B[v]; }
    if (p.states && grp == 0 && ok) {
      float* st = p.states + ((long long)n * p.tiles + tile) * p.c + c;
#pragma unroll
      for (int v = 0; v < V; ++v) st[v] = s[v];
    }
    __syncthreads();
    float mine[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mine[v] = s[v];
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k == grp) mine[v] = s[v];
        s[v] = fmaf(sa[buf][k][cl * V + v], s[v], sb[buf][k][cl * V + v]);
      }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) mine[v] = fmaf(f[i][v], mine[v], b[i][v]);
      if (ok && t0 + i < p.l) put<T, V>(h + (long long)(p.reverse ? p.l - 1 - t0 - i : t0 + i) * p.c, mine);
    }
  }
  if (p.last && seg == p.segs - 1 && grp == 0 && ok) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.last[(long long)n * p.c + c + v] = s[v];
  }
}

template <typename T, int V, int CL>
__global__ __launch_bounds__(SC_THREADS) void scan_bwd_kernel(const ScanK p) {
  constexpr int G = SC_THREADS / CL, R = SC_TILE / G;
  __shared__ float sa[2][G][CL * V], sb[2][G][CL * V], sm[2][G][CL * V];
  const int cl = threadIdx.x % CL, grp = threadIdx.x / CL;
  const int n = blockIdx.x / p.ncb, c = (blockIdx.x % p.ncb) * CL * V + cl * V;
  const int seg = blockIdx.y;
  const bool ok = c < p.c;
  const int cc = ok ? c : 0;
  const T* x = static_cast<const T*>(p.x) + n * p.x_ns + cc;
  const T* g = static_cast<const T*>(p.g) + n * p.g_ns + cc;
  const T* dh = static_cast<const T*>(p.dh) + n * p.dh_ns + cc;
  T* dx = static_cast<T*>(p.dx) + (long long)n * p.l * p.c + cc;
  T* dg = static_cast<T*>(p.dg) + (long long)n * p.l * p.c + cc;
  const float* st = p.states + (long long)n * p.tiles * p.c + cc;

  float mu[V];                                     // f lam of the row behind the tile
#pragma unroll
  for (int v = 0; v < V; ++v) mu[v] = p.dlast ? p.dlast[(long long)n * p.c + cc + v] : 0.f;
  compose<V, -1>(p, n, cc, seg, ok, mu);

  const int first = seg * p.seg_tiles, end = min(p.tiles, first + p.seg_tiles);
  Rows<T, V, R> rx, rg, rd;
  float s0[V];
  auto load = [&](int tile) {
    const int t0 = tile * SC_TILE + grp * R;
    rx.load(x, p.x_ld, t0, p.l, p.reverse);
    rg.load(g, p.g_ld, t0, p.l, p.reverse);
    rd.load(dh, p.dh_ld, t0, p.l, p.reverse);
#pragma unroll
    for (int v = 0; v < V; ++v) s0[v] = st[(long long)tile * p.c + v];
  };
  load(end - 1);
  for (int tile = end - 1; tile >= first; --tile) {
    const int t0 = tile * SC_TILE + grp * R, buf = tile & 1;
    float f[R][V], keep[R][V], xv[R][V], d[R][V], A[V], B[V], M[V], s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; M[v] = 0.f; s[v] = s0[v]; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float gv[V];
      unpack<T, V>(rx.r[i], xv[i]);
      unpack<T, V>(rg.r[i], gv);
      unpack<T, V>(rd.r[i], d[i]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        gate(gv[v], f[i][v], keep[i][v]);
        if (t0 + i >= p.l) { f[i][v] = 1.f; keep[i][v] = 0.f; }          // (x and dh read as zero there)
        A[v] *= f[i][v];
        B[v] = fmaf(f[i][v], B[v], keep[i][v] * xv[i][v]);
      }
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i)
#pragma unroll
      for (int v = 0; v < V; ++v) M[v] = f[i][v] * (M[v] + d[i][v]);
    if (tile > first) load(tile - 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sa[buf][grp][cl * V + v] = A[v];
      sb[buf][grp][cl * V + v] = B[v];
      sm[buf][grp][cl * V + v] = M[v];
    }
    __syncthreads();
    float m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = mu[v];
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k < grp) s[v] = fmaf(sa[buf][k][cl * V + v], s[v], sb[buf][k][cl * V + v]);
      }
#pragma unroll
    for (int k = G - 1; k >= 0; --k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k == grp) m[v] = mu[v];
        mu[v] = fmaf(sa[buf][k][cl * V + v], mu[v], sm[buf][k][cl * V + v]);
      }
    // forward through the rows: h_{t-1} - x_t takes the place of x_t
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float before = s[v];
        s[v] = fmaf(f[i][v], s[v], keep[i][v] * xv[i][v]);
        xv[i][v] = before - xv[i][v];
      }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      float ox[V], og[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float lam = d[i][v] + m[v];
        ox[v] = keep[i][v] * lam;
        og[v] = ox[v] * f[i][v] * xv[i][v];
        m[v] = f[i][v] * lam;
      }
      if (ok && t0 + i < p.l) {
        const long long at = (long long)(p.reverse ? p.l - 1 - t0 - i : t0 + i) * p.c;
        put<T, V>(dx + at, ox);
        put<T, V>(dg + at, og);
      }
    }
  }
  if (p.dh0 && seg == 0 && grp == 0 && ok) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.dh0[(long long)n * p.c + c + v] = mu[v];
  }
}

// The pair of every segment: forward (A, B) from g and x, backward (A, Bm) from g and dh.  A group takes a contiguous part of
// the segment's rows, so the groups meet in LDS once.
template <typename T, int V, int CL, bool BWD>
__global__ __launch_bounds__(SC_THREADS) void scan_segment_kernel(const ScanK p) {
  constexpr int G = SC_THREADS / CL, R = 8;
  __shared__ float sa[G][CL * V], sb[G][CL * V];
  const int cl = threadIdx.x % CL, grp = threadIdx.x / CL;
  const int n = blockIdx.x / p.ncb, c = (blockIdx.x % p.ncb) * CL * V + cl * V;
  const int seg = blockIdx.y;
  const bool ok = c < p.c;
  const int cc = ok ? c : 0;
  const T* g = static_cast<const T*>(p.g) + n * p.g_ns + cc;
  const T* y = BWD ? static_cast<const T*>(p.dh) + n * p.dh_ns + cc : static_cast<const T*>(p.x) + n * p.x_ns + cc;
  const long long y_ld = BWD ? p.dh_ld : p.x_ld;
  const int row0 = seg * p.seg_tiles * SC_TILE, row1 = min(p.l, row0 + p.seg_tiles * SC_TILE);
  const int per = ((row1 - row0 + G - 1) / G + R - 1) / R * R;
  const int lo = min(row1, row0 + grp * per), hi = min(row1, lo + per);
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
  for (int k = 0; k < per; k += R) {
    const int t0 = BWD ? lo + per - R - k : lo + k;           // batches of R rows, backward from the last
    if (t0 >= hi) continue;
    Rows<T, V, R> ry, rg;
    rg.load(g, p.g_ld, t0, p.l, p.reverse);
    ry.load(y, y_ld, t0, p.l, p.reverse);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int i = BWD ? R - 1 - j : j;
      float gv[V], yv[V];
      unpack<T, V>(rg.r[i], gv);
      unpack<T, V>(ry.r[i], yv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f, keep;
        gate(gv[v], f, keep);
        if (t0 + i < hi) {
          A[v] *= f;
          B[v] = BWD ? f * (B[v] + yv[v]) : fmaf(f, B[v], keep * yv[v]);
        }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) { sa[grp][cl * V + v] = A[v]; sb[grp][cl * V + v] = B[v]; }
  __syncthreads();
  if (grp == 0 && ok) {
    float2* out = p.agg + ((long long)n * p.segs + seg) * p.c + c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = 1.f, b = 0.f;
      for (int k = 0; k < G; ++k) {
        const int q = BWD ? G - 1 - k : k;
        a *= sa[q][cl * V + v];
        b = fmaf(sa[q][cl * V + v], b, sb[q][cl * V + v]);
      }
      out[v] = make_float2(a, b);
    }
  }
}

// one row: h = f state + (1 - f) x, the state moves on in place
template <typename T>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* x, long long x_ld, const T* g, long long g_ld, float* state, T* h,
                                                        int c, long long total) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const long long n = i / c;
  const int ch = (int)(i - n * c);
  float f, keep;
  gate(to_f32(g[n * g_ld + ch]), f, keep);
  const float s = fmaf(f, state[i], keep * to_f32(x[n * x_ld + ch]));
  state[i] = s;
  h[i] = from_f32<T>(s);
}

// Workgroups of one segment a window; segments so that the launch has about 512 of them (two a CU), each at least
// SC_MIN_TILES tiles long.
constexpr int SC_FILL = 512, SC_MIN_TILES = 4;

struct Plan { int v, cl, ncb, tiles, segs, seg_tiles; };

Plan make_plan(int dtype, int n, int l, int c, bool even) {
  Plan q;
  q.v = dtype == UNET_BF16 && even ? 2 : 1;
  q.cl = 64;
  q.ncb = cdiv(c, q.cl * q.v);
  q.tiles = cdiv(l, SC_TILE);
  const long long wgs = (long long)n * q.ncb;
  int segs = 1;
  if (wgs < SC_FILL / 2) {
    segs = (int)(SC_FILL / wgs);
    segs = segs < q.tiles / SC_MIN_TILES ? segs : q.tiles / SC_MIN_TILES;
    if (segs < 1) segs = 1;
  }
  q.seg_tiles = cdiv(q.tiles, segs);
  q.segs = cdiv(q.tiles, q.seg_tiles);
  return q;
}

int check_scan(const char* what, int32_t dtype, int64_t n, int64_t l, int64_t c) {
  UNET_REQUIRE(dtype == UNET_BF16 || dtype == UNET_F32, "%s: bad dtype %d", what, dtype);
  UNET_REQUIRE(n > 0 && l > 0 && c > 0 && l <= 0x7fffffff - 4096 && n * ((c + 63) / 64) < (1ll << 31), "%s: bad shape n=%lld l=%lld c=%lld",
               what, (long long)n, (long long)l, (long long)c);
  return 0;
}

template <typename T, int V> int launch_fwd(const ScanK& p, hipStream_t st) {
  const dim3 grid((unsigned)p.n * p.ncb, p.segs);
  if (p.segs > 1) hipLaunchKernelGGL((scan_segment_kernel<T, V, 64, false>), grid, dim3(SC_THREADS), 0, st, p);
  hipLaunchKernelGGL((scan_fwd_kernel<T, V, 64>), grid, dim3(SC_THREADS), 0, st, p);
  UNET_LAUNCH_CHECK("gated_scan_fwd");
  return 0;
}
template <typename T, int V> int launch_bwd(const ScanK& p, hipStream_t st) {
  const dim3 grid((unsigned)p.n * p.ncb, p.segs);
  if (p.segs > 1) hipLaunchKernelGGL((scan_segment_kernel<T, V, 64, true>), grid, dim3(SC_THREADS), 0, st, p);
  hipLaunchKernelGGL((scan_bwd_kernel<T, V, 64>), grid, dim3(SC_THREADS), 0, st, p);
  UNET_LAUNCH_CHECK("gated_scan_bwd");
  return 0;
}

bool even4(const void* p, int64_t ns, int64_t ld) { return !((reinterpret_cast<uintptr_t>(p) & 3) || (ns & 1) || (ld & 1)); }

}  // namespace

extern "C" int32_t unet_gated_scan_tile(void) { return SC_TILE; }

extern "C" size_t unet_gated_scan_workspace_bytes(int32_t dtype, int32_t n, int32_t l, int32_t c) {
  if (n <= 0 || l <= 0 || c <= 0) return 0;
  size_t most = 0;
  for (int even = 0; even < 2; ++even) {
    const Plan q = make_plan(dtype, n, l, c, even != 0);
    const size_t b = q.segs > 1 ? (size_t)n * q.segs * c * sizeof(float2) : 0;
    most = b > most ? b : most;
  }
  return most;
}

extern "C" int unet_gated_scan_fwd(int32_t dtype, const void* x, int64_t x_ns, int64_t x_ld, const void* g, int64_t g_ns,
                                   int64_t g_ld, const float* h0, int32_t reverse, int32_t n, int32_t l, int32_t c, void* h,
                                   float* last, float* states, void* workspace, size_t ws_bytes, void* stream) {
  if (check_scan("gated_scan_fwd", dtype, n, l, c)) return -1;
  UNET_REQUIRE(x && g && h, "gated_scan_fwd: null pointer");
  const bool even = c % 2 == 0 && even4(x, x_ns, x_ld) && even4(g, g_ns, g_ld) && even4(h, 0, 0);
  const Plan q = make_plan(dtype, n, l, c, even);
  UNET_REQUIRE(q.segs == 1 || (workspace && ws_bytes >= (size_t)n * q.segs * c * sizeof(float2)),
               "gated_scan_fwd: workspace of %zu bytes, %zu needed", ws_bytes, (size_t)n * q.segs * c * sizeof(float2));
  ScanK p = {};
  p.x = x; p.g = g; p.h = h; p.h0 = h0; p.last = last; p.states = states;
  p.agg = q.segs > 1 ? static_cast<float2*>(workspace) : nullptr;
  p.x_ns = x_ns; p.x_ld = x_ld; p.g_ns = g_ns; p.g_ld = g_ld;
  p.n = n; p.l = l; p.c = c; p.reverse = reverse != 0;
  p.tiles = q.tiles; p.segs = q.segs; p.seg_tiles = q.seg_tiles; p.ncb = q.ncb;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UNET_F32) return launch_fwd<float, 1>(p, st);
  return q.v == 2 ? launch_fwd<__bf16, 2>(p, st) : launch_fwd<__bf16, 1>(p, st);
}

extern "C" int unet_gated_scan_bwd(int32_t dtype, const void* x, int64_t x_ns, int64_t x_ld, const void* g, int64_t g_ns,
                                   int64_t g_ld, const float* states, const void* dh, int64_t dh_ns, int64_t dh_ld,
                                   const float* dlast, int32_t reverse, int32_t n, int32_t l, int32_t c, void* dx, void* dg,
                                   float* dh0, void* workspace, size_t ws_bytes, void* stream) {
  if (check_scan("gated_scan_bwd", dtype, n, l, c)) return -1;
  UNET_REQUIRE(x && g && states && dh && dx && dg, "gated_scan_bwd: null pointer");
  const bool even = c % 2 == 0 && even4(x, x_ns, x_ld) && even4(g, g_ns, g_ld) && even4(dh, dh_ns, dh_ld) && even4(dx, 0, 0) &&
                    even4(dg, 0, 0);
  const Plan q = make_plan(dtype, n, l, c, even);
  UNET_REQUIRE(q.segs == 1 || (workspace && ws_bytes >= (size_t)n * q.segs * c * sizeof(float2)),
               "gated_scan_bwd: workspace of %zu bytes, %zu needed", ws_bytes, (size_t)n * q.segs * c * sizeof(float2));
  ScanK p = {};
  p.x = x; p.g = g; p.dh = dh; p.dx = dx; p.dg = dg; p.dlast = dlast; p.dh0 = dh0; p.states = const_cast<float*>(states);
  p.agg = q.segs > 1 ? static_cast<float2*>(workspace) : nullptr;
  p.x_ns = x_ns; p.x_ld = x_ld; p.g_ns = g_ns; p.g_ld = g_ld; p.dh_ns = dh_ns; p.dh_ld = dh_ld;
  p.n = n; p.l = l; p.c = c; p.reverse = reverse != 0;
  p.tiles = q.tiles; p.segs = q.segs; p.seg_tiles = q.seg_tiles; p.ncb = q.ncb;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UNET_F32) return launch_bwd<float, 1>(p, st);
  return q.v == 2 ? launch_bwd<__bf16, 2>(p, st) : launch_bwd<__bf16, 1>(p, st);
}

extern "C" int unet_gated_scan_step(int32_t dtype, const void* x, int64_t x_ld, const void* g, int64_t g_ld, float* state, void* h,
                                    int32_t n, int32_t c, void* stream) {
  if (check_scan("gated_scan_step", dtype, n, 1, c)) return -1;
  UNET_REQUIRE(x && g && state && h, "gated_scan_step: null pointer");
  const long long total = (long long)n * c;
  const dim3 grid((unsigned)((total + 255) / 256));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UNET_F32)
    hipLaunchKernelGGL((scan_step_kernel<float>), grid, dim3(256), 0, st, (const float*)x, x_ld, (const float*)g, g_ld, state,
                       (float*)h, c, total);
  else
    hipLaunchKernelGGL((scan_step_kernel<__bf16>), grid, dim3(256), 0, st, (const __bf16*)x, x_ld, (const __bf16*)g, g_ld, state,
                       (__bf16*)h, c, total);
  UNET_LAUNCH_CHECK("gated_scan_step");
  return 0;
}
