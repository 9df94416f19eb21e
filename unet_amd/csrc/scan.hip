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
// HBM-bound.  Inputs and outputs are touched once and are larger than the caches where it matters: their accesses are
// non-temporal (forward at [64, 1024, 1024] bf16 83 -> 71 us, and a kernel that reads h afterwards does not lose it).  Measured
// there, medians under the profiler: forward 74 us (403 MB, 5.4 TB/s), backward 132 us (671 MB, 5.1 TB/s); [1, 75000, 1024] forward 65 us
// for the segments and 83 for the walk (307 and 461 MB; 137 us for both in a row of calls).
//
// Everything between loads and stores is fp32.  sigmoid: with t = exp(-|g|), small = t / (1 + t), big = 1 - small; keep = 1 - f
// has full relative precision on both sides.  A long memory lives in 1 - f, which fp32 rounds to multiples of 2^-24 next to 1: 1 - f
// would be 0.07 % off at g = 10 and nothing at g = 17.4, so that a state would settle beside its input or never forget.  So the
// complement C = 1 - A of a span is summed beside A, C + A keep a row; where it is below a half, A is 1 - C and the rest that this
// rounding left, and h = A h + (rest h + B) rounds once.  Within eight rows, whose errors end with their span, f is used as it is.
// (A rest in every row took 86 and 146 us forward and backward, one across spans 72..75 and 129, none 72 and 126.)
#include "common.h"
#include <cfloat>

namespace {

constexpr int SC_THREADS = 512;
constexpr int SC_TILE = 64;      // rows of a tile, and the distance of the kept states
constexpr int NT = 2;            // buffer accesses: non-temporal
constexpr float LOG2E = 1.4426950408889634f;

struct Pair;

struct ScanK {
  const void *x, *g, *dh;        // [n][l][ld]
  void *h, *dx, *dg;             // [n][l][c]
  const float *h0, *dlast;       // [n][c] or null
  float *last, *dh0;             // [n][c] or null
  float* states;                 // [n][tiles][c] or null: state in front of every tile
  Pair* agg;                     // [n][segs][c], or null (one segment)
  long long x_ns, x_ld, g_ns, g_ld, dh_ns, dh_ld;
  int n, l, c, tiles, segs, seg_tiles, ncb, reverse;
};

// V consecutive values of a row: one fp32 or bf16, or two bf16
template <typename T, int V> struct Raw;
template <> struct Raw<float, 1> { typedef float type; };
template <> struct Raw<__bf16, 1> { typedef unsigned short type; };
template <> struct Raw<__bf16, 2> { typedef unsigned int type; };

template <typename T, int V> __device__ __forceinline__ void unpack(const typename Raw<T, V>::type& r, float (&f)[V]) {
  if constexpr (std::is_same<T, float>::value) f[0] = r;
  else {
    f[0] = __builtin_bit_cast(float, (unsigned)r << 16);
    if constexpr (V == 2) f[1] = __builtin_bit_cast(float, r & 0xffff0000u);
  }
}
template <typename T, int V> __device__ __forceinline__ typename Raw<T, V>::type pack(const float (&f)[V]) {
  typedef __attribute__((ext_vector_type(V))) T vec;
  vec v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (T)f[i];
  return __builtin_bit_cast(typename Raw<T, V>::type, v);
}

__device__ __forceinline__ void gate(float g, float& f, float& keep) {     // f = sigmoid(g), keep = 1 - f
  const float t = __builtin_amdgcn_exp2f(-fabsf(g) * LOG2E);
  const float small = t * __builtin_amdgcn_rcpf(1.f + t);
  const float big = 1.f - small;
  f = g >= 0.f ? big : small;
  keep = g >= 0.f ? small : big;
}

// h -> (a + rest) h + b.  a is rounded down, so that an infinite h meets a positive rest and stays as it is.
struct Pair { float a, rest, b; };
__device__ __forceinline__ float apply(const Pair& p, float h) { return fmaf(p.a, h, fmaf(p.rest, h, p.b)); }
// 1 - c (c at most a half) as a + rest
__device__ __forceinline__ void complement(float c, float& a, float& rest) {
  a = 1.f - (c + 0x1p-25f);
  rest = fmaxf((1.f - a) - c, FLT_MIN);
}
// A span as it grows in walk order: A, its complement, B
template <int V> struct Span {
  float a[V], c[V], b[V];
  __device__ __forceinline__ Span() {
#pragma unroll
    for (int v = 0; v < V; ++v) { a[v] = 1.f; c[v] = 0.f; b[v] = 0.f; }
  }
  __device__ __forceinline__ void grow(int v, float f, float keep) {
    c[v] = fmaf(keep, a[v], c[v]);
    a[v] *= f;
  }
  __device__ __forceinline__ void then(int v, const Pair& q) {          // a span behind this one
    grow(v, q.a, (1.f - q.a) - q.rest);
    b[v] = apply(q, b[v]);
  }
  __device__ __forceinline__ Pair pair(int v) const {
    Pair q = {a[v], FLT_MIN, b[v]};
    if (c[v] < 0.5f) complement(c[v], q.a, q.rest);
    return q;
  }
};

// One tensor [l][ld] of a window, as a thread walks it: R rows at `row` (a multiple of R inside the tile) of V channels.  Whole
// tiles go through buffer instructions: the tile's base and the rows' offsets are scalars, a lane holds one 32-bit offset.
template <typename T, int V, int R> struct Rows {
  typedef typename Raw<T, V>::type raw;
  const T* base;                  // the window's row 0, channel 0 (uniform)
  long long ld;
  int l, reverse, c;
  unsigned voff;
  __device__ __forceinline__ void init(const void* window, long long ld_, int l_, int reverse_, int row, int c_) {
    base = static_cast<const T*>(window);
    ld = ld_; l = l_; reverse = reverse_; c = c_;
    voff = (unsigned)(((reverse ? SC_TILE - R - row : row) * ld + c) * sizeof(T));
  }
  __device__ __forceinline__ auto rsrc(int tile) const {
    const int lo = reverse ? l - (tile + 1) * SC_TILE : tile * SC_TILE;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + lo * ld), 0, 0x80000000u, 0x00020000);
  }
  __device__ __forceinline__ int soff(int i) const { return (int)((reverse ? R - 1 - i : i) * ld * sizeof(T)); }
  __device__ __forceinline__ void load(raw (&r)[R], int tile) const {
    const auto d = rsrc(tile);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if constexpr (sizeof(raw) == 2) r[i] = (raw)__builtin_amdgcn_raw_buffer_load_b16(d, voff, soff(i), NT);
      else r[i] = __builtin_bit_cast(raw, __builtin_amdgcn_raw_buffer_load_b32(d, voff, soff(i), NT));
    }
  }
  __device__ __forceinline__ const T* at(int t) const { return base + (long long)(reverse ? l - 1 - t : t) * ld + c; }
  // rows t .. t+R-1 of a tile that the window's end cuts: rows at or past l read as zero
  __device__ __forceinline__ void load_cut(raw (&r)[R], int t) const {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      r[i] = raw{};
      if (t + i < l) r[i] = *reinterpret_cast<const raw*>(at(t + i));
    }
  }
  __device__ __forceinline__ void store(int tile, int i, const float (&f)[V]) const {
    const raw w = pack<T, V>(f);
    const auto d = rsrc(tile);
    if constexpr (sizeof(raw) == 2) __builtin_amdgcn_raw_buffer_store_b16(w, d, voff, soff(i), NT);
    else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, w), d, voff, soff(i), NT);
  }
  __device__ __forceinline__ void store_cut(int t, const float (&f)[V]) const {
    if (t < l) *reinterpret_cast<raw*>(const_cast<T*>(at(t))) = pack<T, V>(f);
  }
};

// R rows anywhere, by their addresses
template <typename T, int V, int R> struct Walk {
  typename Raw<T, V>::type r[R];
  const T* p;
  long long step;
  __device__ __forceinline__ void start(const T* base, long long ld, int t0, int l, int reverse) {
    step = reverse ? -ld : ld;
    p = base + (long long)(reverse ? l - 1 : 0) * ld + (long long)t0 * step;
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < R; ++i) r[i] = *reinterpret_cast<const typename Raw<T, V>::type*>(p + i * step);
  }
  __device__ __forceinline__ void load(int rows) {         // the first `rows` of them; the others read as zero
#pragma unroll
    for (int i = 0; i < R; ++i) {
      r[i] = typename Raw<T, V>::type{};
      if (i < rows) r[i] = *reinterpret_cast<const typename Raw<T, V>::type*>(p + i * step);
    }
  }
};

// Start value of segment `seg`: the pairs of the segments before it (walk order DIR) applied to `s`.  Each group composes a
// contiguous share of them, the groups' pairs meet in LDS (`sp`, free again after the call).
template <int V, int CL, int DIR>
__device__ __forceinline__ void compose(const ScanK& p, int n, int c, int seg, int grp, Pair (*sp)[CL * V], float (&s)[V]) {
  constexpr int G = SC_THREADS / CL;
  if (!p.agg) return;                              // uniform
  const int cl = threadIdx.x % CL, before = DIR > 0 ? seg : p.segs - 1 - seg, share = (before + G - 1) / G;
  const int lo = min(before, grp * share), hi = min(before, lo + share);
  const Pair* q = p.agg + ((long long)n * p.segs + (DIR > 0 ? 0 : p.segs - 1)) * p.c + c;       // k-th pair in walk order: q[DIR * k * c]
  Span<V> span;
#pragma unroll 4
  for (int k = lo; k < hi; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) span.then(v, q[(long long)DIR * k * p.c + v]);
#pragma unroll
  for (int v = 0; v < V; ++v) sp[grp][cl * V + v] = span.pair(v);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < G; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = apply(sp[k][cl * V + v], s[v]);
  __syncthreads();
}

template <typename T, int V, int CL>
__global__ __launch_bounds__(SC_THREADS) void scan_fwd_kernel(const ScanK p) {
  constexpr int G = SC_THREADS / CL, R = SC_TILE / G;
  __shared__ Pair sp[2][G][CL * V];
  const int cl = threadIdx.x % CL, grp = threadIdx.x / CL;
  const int n = blockIdx.x / p.ncb, c = (blockIdx.x % p.ncb) * CL * V + cl * V;
  const int seg = blockIdx.y;
  const bool ok = c < p.c;                         // c % V == 0 and p.c % V == 0: a thread's channels are all in or all out
  const int cc = ok ? c : 0;
  const int first = seg * p.seg_tiles, end = min(p.tiles, first + p.seg_tiles);
  const int full = min(end, p.l / SC_TILE);        // tiles whose rows all exist
  Rows<T, V, R> rx, rg, rh;
  rx.init(static_cast<const T*>(p.x) + n * p.x_ns, p.x_ld, p.l, p.reverse, grp * R, cc);
  rg.init(static_cast<const T*>(p.g) + n * p.g_ns, p.g_ld, p.l, p.reverse, grp * R, cc);
  rh.init(static_cast<const T*>(p.h) + (long long)n * p.l * p.c, p.c, p.l, p.reverse, grp * R, cc);
  typename Rows<T, V, R>::raw qx[R], qg[R];
  if (first < full) { rx.load(qx, first); rg.load(qg, first); }
  float s[V];                                      // state in front of the tile (the same in every group)
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = p.h0 ? p.h0[(long long)n * p.c + cc + v] : 0.f;
  compose<V, CL, 1>(p, n, cc, seg, grp, sp[0], s);

  auto work = [&](int tile, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int buf = tile & 1, t0 = tile * SC_TILE + grp * R;
    float f[R][V], b[R][V];
    Span<V> span;
    if (!WHOLE) { rx.load_cut(qx, t0); rg.load_cut(qg, t0); }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float xv[V], gv[V];
      unpack<T, V>(qx[i], xv);
      unpack<T, V>(qg[i], gv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float keep;
        gate(gv[v], f[i][v], keep);
        b[i][v] = keep * xv[v];
        if (!WHOLE && t0 + i >= p.l) { f[i][v] = 1.f; keep = b[i][v] = 0.f; }
        span.grow(v, f[i][v], keep);
        span.b[v] = fmaf(f[i][v], span.b[v], b[i][v]);
      }
    }
    if (WHOLE && tile + 1 < full) { rx.load(qx, tile + 1); rg.load(qg, tile + 1); }
#pragma unroll
    for (int v = 0; v < V; ++v) sp[buf][grp][cl * V + v] = span.pair(v);
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
        s[v] = apply(sp[buf][k][cl * V + v], s[v]);
      }
    if (ok) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int v = 0; v < V; ++v) mine[v] = fmaf(f[i][v], mine[v], b[i][v]);
        if (WHOLE) rh.store(tile, i, mine);
        else rh.store_cut(t0 + i, mine);
      }
    }
  };
  for (int tile = first; tile < full; ++tile) work(tile, std::true_type{});
  if (full < end) work(full, std::false_type{});
  if (p.last && seg == p.segs - 1 && grp == 0 && ok) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.last[(long long)n * p.c + c + v] = s[v];
  }
}

template <typename T, int V, int CL>
__global__ __launch_bounds__(SC_THREADS, 2) void scan_bwd_kernel(const ScanK p) {
  constexpr int G = SC_THREADS / CL, R = SC_TILE / G;
  __shared__ Pair sp[2][G][CL * V];
  __shared__ float sm[2][G][CL * V];
  const int cl = threadIdx.x % CL, grp = threadIdx.x / CL;
  const int n = blockIdx.x / p.ncb, c = (blockIdx.x % p.ncb) * CL * V + cl * V;
  const int seg = blockIdx.y;
  const bool ok = c < p.c;
  const int cc = ok ? c : 0;
  const int first = seg * p.seg_tiles, end = min(p.tiles, first + p.seg_tiles);
  Rows<T, V, R> rx, rg, rd, ox_, og_;
  rx.init(static_cast<const T*>(p.x) + n * p.x_ns, p.x_ld, p.l, p.reverse, grp * R, cc);
  rg.init(static_cast<const T*>(p.g) + n * p.g_ns, p.g_ld, p.l, p.reverse, grp * R, cc);
  rd.init(static_cast<const T*>(p.dh) + n * p.dh_ns, p.dh_ld, p.l, p.reverse, grp * R, cc);
  ox_.init(static_cast<const T*>(p.dx) + (long long)n * p.l * p.c, p.c, p.l, p.reverse, grp * R, cc);
  og_.init(static_cast<const T*>(p.dg) + (long long)n * p.l * p.c, p.c, p.l, p.reverse, grp * R, cc);
  const float* st = p.states + (long long)n * p.tiles * p.c + cc;
  typename Rows<T, V, R>::raw qx[R], qg[R], qd[R];
  float s0[V];
  auto load = [&](int tile) {
    rx.load(qx, tile); rg.load(qg, tile); rd.load(qd, tile);
#pragma unroll
    for (int v = 0; v < V; ++v) s0[v] = st[(long long)tile * p.c + v];
  };
  const bool cut = end * SC_TILE > p.l;            // the segment's last tile is not whole
  if (!cut) load(end - 1);
  float mu[V];                                     // f lam of the row behind the tile
#pragma unroll
  for (int v = 0; v < V; ++v) mu[v] = p.dlast ? p.dlast[(long long)n * p.c + cc + v] : 0.f;
  compose<V, CL, -1>(p, n, cc, seg, grp, sp[0], mu);

  auto work = [&](int tile, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int buf = tile & 1, t0 = tile * SC_TILE + grp * R;
    float f[R][V], keep[R][V], xv[R][V], d[R][V], M[V], s[V];
    Span<V> span;
    if (!WHOLE) {
      rx.load_cut(qx, t0); rg.load_cut(qg, t0); rd.load_cut(qd, t0);
#pragma unroll
      for (int v = 0; v < V; ++v) s0[v] = st[(long long)tile * p.c + v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { M[v] = 0.f; s[v] = s0[v]; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float gv[V];
      unpack<T, V>(qx[i], xv[i]);
      unpack<T, V>(qg[i], gv);
      unpack<T, V>(qd[i], d[i]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        gate(gv[v], f[i][v], keep[i][v]);
        if (!WHOLE && t0 + i >= p.l) { f[i][v] = 1.f; keep[i][v] = 0.f; }          // (x and dh read as zero there)
        span.grow(v, f[i][v], keep[i][v]);
        span.b[v] = fmaf(f[i][v], span.b[v], keep[i][v] * xv[i][v]);
      }
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i)
#pragma unroll
      for (int v = 0; v < V; ++v) M[v] = f[i][v] * (M[v] + d[i][v]);
    if (tile > first) load(tile - 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sp[buf][grp][cl * V + v] = span.pair(v);
      sm[buf][grp][cl * V + v] = M[v];
    }
    __syncthreads();
    float m[V], run[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { m[v] = mu[v]; run[v] = s[v]; }
#pragma unroll
    for (int k = 0; k < G - 1; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        run[v] = apply(sp[buf][k][cl * V + v], run[v]);
        if (k + 1 == grp) s[v] = run[v];
      }
#pragma unroll
    for (int k = G - 1; k >= 0; --k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k == grp) m[v] = mu[v];
        const Pair q = sp[buf][k][cl * V + v];
        mu[v] = apply({q.a, q.rest, sm[buf][k][cl * V + v]}, mu[v]);
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
    if (ok) {
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
        if (WHOLE) {
          ox_.store(tile, i, ox);
          og_.store(tile, i, og);
        } else {
          ox_.store_cut(t0 + i, ox);
          og_.store_cut(t0 + i, og);
        }
      }
    }
  };
  int tile = end - 1;
  if (cut) work(tile--, std::false_type{});
  for (; tile >= first; --tile) work(tile, std::true_type{});
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
  __shared__ Pair sp[G][CL * V];
  const int cl = threadIdx.x % CL, grp = threadIdx.x / CL;
  const int n = blockIdx.x / p.ncb, c = (blockIdx.x % p.ncb) * CL * V + cl * V;
  const int seg = blockIdx.y;
  const bool ok = c < p.c;
  const int cc = ok ? c : 0;
  const T* g = static_cast<const T*>(p.g) + n * p.g_ns + cc;
  const T* y = BWD ? static_cast<const T*>(p.dh) + n * p.dh_ns + cc : static_cast<const T*>(p.x) + n * p.x_ns + cc;
  const long long y_ld = BWD ? p.dh_ld : p.x_ld;
  const int row0 = seg * p.seg_tiles * SC_TILE, row1 = row0 + min(p.l - row0, p.seg_tiles * SC_TILE);
  const int per = ((row1 - row0 + G - 1) / G + R - 1) / R * R;
  const int lo = min(row1, row0 + grp * per), hi = min(row1, lo + per);
  Span<V> span;
  Walk<T, V, R> ry[2], rg[2];
  auto take = [&](int slot, int rows, auto whole) {              // `rows` of the batch exist
    constexpr bool WHOLE = decltype(whole)::value;
    Span<V> batch;                                               // R rows, then part of the span
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int i = BWD ? R - 1 - j : j;
      float gv[V], yv[V];
      unpack<T, V>(rg[slot].r[i], gv);
      unpack<T, V>(ry[slot].r[i], yv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f, keep;
        gate(gv[v], f, keep);
        if (WHOLE || i < rows) {
          batch.grow(v, f, keep);
          batch.b[v] = BWD ? f * (batch.b[v] + yv[v]) : fmaf(f, batch.b[v], keep * yv[v]);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) span.then(v, batch.pair(v));
  };
  // batches of R rows, in walk order or (backward) from the last; the short one is the last in walk order
  const int batches = (hi - lo) / R, rest = (hi - lo) - batches * R;
  auto at = [&](int slot, int t0) {
    rg[slot].start(g, p.g_ld, t0, p.l, p.reverse);
    ry[slot].start(y, y_ld, t0, p.l, p.reverse);
  };
  if (BWD && rest > 0) {
    at(0, lo + batches * R);
    rg[0].load(rest);
    ry[0].load(rest);
    take(0, rest, std::false_type{});
  }
  if (batches > 0) {
    at(0, BWD ? lo + (batches - 1) * R : lo);
    rg[0].load();
    ry[0].load();
    for (int k = 0; k < batches; k += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (k + u < batches) {
          if (k + u + 1 < batches) {
            at(u ^ 1, BWD ? lo + (batches - 2 - k - u) * R : lo + (k + u + 1) * R);
            rg[u ^ 1].load();
            ry[u ^ 1].load();
          }
          take(u, R, std::true_type{});
        }
      }
    }
  }
  if (!BWD && rest > 0) {
    at(0, lo + batches * R);
    rg[0].load(rest);
    ry[0].load(rest);
    take(0, rest, std::false_type{});
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sp[grp][cl * V + v] = span.pair(v);
  __syncthreads();
  if (grp == 0 && ok) {
    Pair* out = p.agg + ((long long)n * p.segs + seg) * p.c + c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Span<1> all;
      for (int k = 0; k < G; ++k) all.then(0, sp[BWD ? G - 1 - k : k][cl * V + v]);
      out[v] = all.pair(0);
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
  float keep;
  Pair row = {0.f, FLT_MIN, 0.f};
  gate(to_f32(g[n * g_ld + ch]), row.a, keep);
  if (keep < 0.5f) complement(keep, row.a, row.rest);
  row.b = keep * to_f32(x[n * x_ld + ch]);
  const float s = apply(row, state[i]);
  state[i] = s;
  h[i] = from_f32<T>(s);
}

// Enough workgroups to fill the chip: about two a CU.  Half of that or more without segments: one launch.  Otherwise as many
// segments as fill it, down to one tile each (against segments of at least four tiles, forward: [1, 1024, 1024] 15.6 -> 8.4 us,
// [1, 4096, 256] 16.3 -> 9.4, [4, 4096, 512] 19.7 -> 20.0; unsplit: 28, 105 and 106 us).  Two tiles gain nothing from a second
// launch.
constexpr int SC_FILL = 512;

struct Plan { int v, cl, ncb, tiles, segs, seg_tiles; };

Plan make_plan(int dtype, int n, int l, int c, bool even) {
  Plan q;
  q.v = dtype == UNET_BF16 && even ? 2 : 1;
  q.cl = 64;
  q.ncb = cdiv(c, q.cl * q.v);
  q.tiles = cdiv(l, SC_TILE);
  const long long wgs = (long long)n * q.ncb;
  int segs = 1;
  if (wgs < SC_FILL / 2 && q.tiles > 2) {
    segs = (int)(SC_FILL / wgs);
    segs = segs < q.tiles ? segs : q.tiles;
  }
  q.seg_tiles = cdiv(q.tiles, segs);
  q.segs = cdiv(q.tiles, q.seg_tiles);
  return q;
}

int check_scan(const char* what, int32_t dtype, int64_t n, int64_t l, int64_t c) {
  UNET_REQUIRE(dtype == UNET_BF16 || dtype == UNET_F32, "%s: bad dtype %d", what, dtype);
  UNET_REQUIRE(n > 0 && l > 0 && c > 0 && l <= 0x7fffffff - 4096 && n * ((c + 63) / 64) < (1ll << 31) && c <= (1 << 22), "%s: bad shape n=%lld l=%lld c=%lld",
               what, (long long)n, (long long)l, (long long)c);
  return 0;
}

// threads of a launch are counted in 32 bits
int check_grid(const char* what, long long workgroups, int threads) {
  UNET_REQUIRE(workgroups * threads < (1ll << 32), "%s: %lld workgroups of %d threads, at most 2^32 threads in all", what, workgroups, threads);
  return 0;
}

// a tile's rows lie within one buffer descriptor's 31 bits
int check_pitch(const char* what, int64_t ld) {
  UNET_REQUIRE(ld >= 0 && ld <= (1ll << 22), "%s: row pitch %lld, must be 0 .. 2^22 elements", what, (long long)ld);
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
    const size_t b = q.segs > 1 ? (size_t)n * q.segs * c * sizeof(Pair) : 0;
    most = b > most ? b : most;
  }
  return most;
}

extern "C" int unet_gated_scan_fwd(int32_t dtype, const void* x, int64_t x_ns, int64_t x_ld, const void* g, int64_t g_ns,
                                   int64_t g_ld, const float* h0, int32_t reverse, int32_t n, int32_t l, int32_t c, void* h,
                                   float* last, float* states, void* workspace, size_t ws_bytes, void* stream) {
  if (check_scan("gated_scan_fwd", dtype, n, l, c)) return -1;
  UNET_REQUIRE(x && g && h, "gated_scan_fwd: null pointer");
  if (check_pitch("gated_scan_fwd", x_ld) || check_pitch("gated_scan_fwd", g_ld)) return -1;
  const bool even = c % 2 == 0 && even4(x, x_ns, x_ld) && even4(g, g_ns, g_ld) && even4(h, 0, 0);
  const Plan q = make_plan(dtype, n, l, c, even);
  if (check_grid("gated_scan_fwd", (long long)n * q.ncb, SC_THREADS)) return -1;
  UNET_REQUIRE(q.segs == 1 || (workspace && ws_bytes >= (size_t)n * q.segs * c * sizeof(Pair)),
               "gated_scan_fwd: workspace of %zu bytes, %zu needed", ws_bytes, (size_t)n * q.segs * c * sizeof(Pair));
  ScanK p = {};
  p.x = x; p.g = g; p.h = h; p.h0 = h0; p.last = last; p.states = states;
  p.agg = q.segs > 1 ? static_cast<Pair*>(workspace) : nullptr;
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
  if (check_pitch("gated_scan_bwd", x_ld) || check_pitch("gated_scan_bwd", g_ld) || check_pitch("gated_scan_bwd", dh_ld)) return -1;
  const bool even = c % 2 == 0 && even4(x, x_ns, x_ld) && even4(g, g_ns, g_ld) && even4(dh, dh_ns, dh_ld) && even4(dx, 0, 0) &&
                    even4(dg, 0, 0);
  const Plan q = make_plan(dtype, n, l, c, even);
  if (check_grid("gated_scan_bwd", (long long)n * q.ncb, SC_THREADS)) return -1;
  UNET_REQUIRE(q.segs == 1 || (workspace && ws_bytes >= (size_t)n * q.segs * c * sizeof(Pair)),
               "gated_scan_bwd: workspace of %zu bytes, %zu needed", ws_bytes, (size_t)n * q.segs * c * sizeof(Pair));
  ScanK p = {};
  p.x = x; p.g = g; p.dh = dh; p.dx = dx; p.dg = dg; p.dlast = dlast; p.dh0 = dh0; p.states = const_cast<float*>(states);
  p.agg = q.segs > 1 ? static_cast<Pair*>(workspace) : nullptr;
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
  if (check_grid("gated_scan_step", (total + 255) / 256, 256)) return -1;
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
