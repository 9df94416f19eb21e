// Attention with a learned relative-position bias, bf16 MFMA, forward and backward:
//   S[i, j] = scale <q_i, k_j> + table[bucket(j - i), head],   P = softmax_j S,   O = P V
// The bias depends on the offset j - i alone: one value per offset up to the last bucket's start `sat`, constant beyond it on
// either side.  A workgroup keeps its head's values in LDS; a tile whose offsets all lie beyond +-sat adds one scalar (folded
// into the exponential's fma, so most of a long sequence pays nothing), the others read LDS once per score, conflict-free
// because neighbouring lanes are neighbouring offsets.  A far bucket of -inf is never walked: attention to a local band costs
// what the band costs.
//
// Forward and the two backward walks are the flash kernels of attn.hip for one band (128 query rows a workgroup, K / V tiles of
// 64 keys double-buffered in LDS, S^T = K Q^T so that P is the next product's operand as it stands).  delta_i = <dO_i, O_i>,
// dS = P o (dO V^T - delta); dV = P^T dO, dK = scale dS^T Q, dQ = scale dS K.
//   d table[b, h] = sum of dS over the pairs of bucket b
// is taken where dS is in registers anyway, in the dQ walk: far tiles add into one register a side, the others into a wave's
// own LDS array by offset, one diagonal of the tile a lane.  Workgroups write their sums by offset, a last launch adds them in a
// fixed order: no atomics, the same bits every time.  A few rows in a long window split the walked axis (rel_splits).
//
// At [32, 1024, 1024], 8 heads of 128 (69 GFLOP a product; a large matrix product of this card runs at 1247 TFLOP/s), medians
// under the profiler: forward 0.243 ms in front of a backward pass (0.17 for inference), dQ 0.311, dK and dV 0.369, table 0.014: 0.66 to
// 0.85 PFLOP/s in each walk.  Two waves a SIMD share the matrix pipe (busy 47, 35 and 38 % of the cycles) and the vector pipe (issuing in
// 52, 40 and 33 %); neither is full, what is left is one wave waiting for its own scores between the products.
#include "attn_tiles.h"
#include "relattn.h"

namespace {

// Up to this head size two workgroups share a CU: 256 registers a lane, which also keeps the accumulators out of AGPRs.
// Together with tile loops that have no branch around the accumulators: forward 286 -> 197 us, dK and dV 842 -> 389 us at
// [32, 1024, 1024], heads of 128.  Heads of 256 need the registers of a whole CU.
constexpr int REL_OCC2 = 128;

// What a tile adds to its scores: biases by offset (NEAR), or one constant (BEYOND, FLAT).  A constant is folded into the exponential's
// fma (BEYOND) while it is small.  A large one (a mask of the type's lowest value, -1e9) absorbs the scores it is added to; the
// difference of two such constants would bring them back, so the complete score is formed first and the row's maximum and the log2 of
// its sum are taken off one after the other, as in NEAR tiles: forward and backward then see the same P (FLAT).
enum Kind { NEAR, BEYOND, FLAT };
typedef std::integral_constant<Kind, NEAR> Near;
typedef std::integral_constant<Kind, BEYOND> Beyond;
typedef std::integral_constant<Kind, FLAT> Flat;
constexpr float REL_FOLD = 1024.f;      // folded up to here (log2 domain): its rounding, 2^-14, is below those of a P in bf16

__device__ __forceinline__ bool rel_folds(float beyond) {
  return __builtin_amdgcn_readfirstlane(!(fabsf(beyond) > REL_FOLD) || beyond == -INFINITY);
}

// Streamed tiles [lo, hi) of T rows against the 32 rows a wave holds from `own` on: [lo, n0) lie wholly beyond one edge of the
// band ([lo, f0) of them fold their constant, all or none), [n0, n1) touch it, [n1, hi) lie beyond the other edge ([n1, f1) fold).
// The runs are loops of their own (a wave's own bounds: every tile has one barrier, whichever loop it is in), so the accumulators
// pass no branch.
struct Runs { int f0, n0, n1, f1; };
template <int T> __device__ __forceinline__ Runs rel_runs(int lo, int hi, int own, int sat, float before, float behind) {
  const int left = own - sat - (T - 1), right = own + 31 + sat;           // first tile that starts behind `left` / at or behind `right`
  Runs r;
  r.n0 = max(lo, min(hi, left >= 0 ? left / T + 1 : 0));
  r.n1 = max(r.n0, min(hi, (right + T - 1) / T));
  r.f0 = rel_folds(before) ? r.n0 : lo;
  r.f1 = rel_folds(behind) ? hi : r.n1;
  return r;
}

// A lane's fragments of its own row of a [L][C] slab, from `t` at element `row` (a row that exists; zeros unless `ok`).  No branches:
// all loads leave at once.
template <int HDP> __device__ __forceinline__ void own_row(bf16x8 (&f)[Cfg<HDP>::KS], const void* t, long long row, bool ok, int h, int hd) {
#pragma unroll
  for (int s = 0; s < Cfg<HDP>::KS; ++s) {
    const int ch = (2 * s + h) * 8;
    f[s] = *reinterpret_cast<const bf16x8*>(static_cast<const __bf16*>(t) + row + (ch < hd ? ch : 0));
  }
#pragma unroll
  for (int s = 0; s < Cfg<HDP>::KS; ++s) {
    const bool in = ok && (2 * s + h) * 8 < hd;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[s][e] = in ? f[s][e] : (__bf16)0.f;
  }
}

// share `split` of the walked axis, cut in p.splits pieces of whole tiles of T rows, within [lo, hi)
__device__ __forceinline__ void rel_share(const RelK& p, int split, int T, int& lo, int& hi) {
  const int tiles = (p.l + T - 1) / T, per = (tiles + p.splits - 1) / p.splits;
  lo = max(lo, split * per);
  hi = min(hi, (split + 1) * per);
}
__device__ __forceinline__ float2* rel_split_stats(const RelK& p) {
  return reinterpret_cast<float2*>(p.split + (long long)p.splits * p.n * p.l * p.c);
}

// TileLoader of attn_tiles.h for tiles of ROWS rows (the same LDS image)
template <int HDP, int ROWS> struct RowLoader {
  static constexpr int BYTES = ROWS * HDP * 2, PIECES = BYTES / 1024, PPW = (PIECES + 3) / 4;
  unsigned voff[PPW];
  __device__ __forceinline__ void setup(int wave, int lane, int c, int hd) {
#pragma unroll
    for (int k = 0; k < PPW; ++k) {
      const int lin = (wave * PPW + k) * 1024 + lane * 16;
      const int row = lin / Cfg<HDP>::ROWB;
      const int ch = ((lin % Cfg<HDP>::ROWB) >> 4) ^ (xv(row) & Cfg<HDP>::XM);
      voff[k] = ch * 8 < hd ? (unsigned)((row * c + ch * 8) * 2) : AT_OOB;
    }
  }
  // rows row0 .. row0+ROWS-1 of the slab behind `base`; rows at or past l arrive as zeros
  __device__ __forceinline__ void issue(const __bf16* base, int l, int c, int hd, char* tile, unsigned row0, int wave) const {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (unsigned)((((long long)l - 1) * c + hd) * 2), 0x00020000);
#pragma unroll
    for (int k = 0; k < PPW; ++k)
      if (wave * PPW + k < PIECES)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (__attribute__((address_space(3))) void*)(tile + (wave * PPW + k) * 1024), 16, voff[k] + row0 * c * 2, 0, 0, 0);
  }
};

// What rounding to bf16 took from registers 8s..8s+7: x = pack8 + rest8 to 2^-16
__device__ __forceinline__ bf16x8 rest8(const f32x16& x, int s, const bf16x8& rounded) {
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = (__bf16)(x[8 * s + j] - (float)rounded[j]);
  return o;
}

template <int HDP, bool FINE>
__global__ __launch_bounds__(AT_THREADS, HDP <= REL_OCC2 ? 2 : 1) void rel_attn_fwd_kernel(const RelK p) {
  typedef Cfg<HDP> G;
  extern __shared__ __attribute__((aligned(16))) char smem[];   // [2 buffers][K tile | V tile], biases
  float* const bias = reinterpret_cast<float*>(smem + 4 * G::TILE);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;

  int wg = xcd_remap(blockIdx.x, gridDim.x);
  const int nqt = (p.l + AT_BQ - 1) / AT_BQ;
  const int qt = wg % nqt; wg /= nqt;
  const int split = wg % p.splits; wg /= p.splits;
  const int head = wg % p.nh;
  const int n = wg / p.nh;
  const int len = rel_length(p, n);
  const int hoff = head * p.hd;
  const long long base = (long long)n * p.l * p.c + hoff;
  const int q0 = qt * AT_BQ, qrow = q0 + wave * 32 + r;
  const bool row_ok = qrow < len;
  __bf16* const op = static_cast<__bf16*>(p.out) + base + (long long)qrow * p.c;
  float* const lse = p.lse ? p.lse + ((long long)n * p.nh + head) * p.l + qrow : nullptr;

  f32x16 acc[G::DT];
#pragma unroll
  for (int d = 0; d < G::DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
  float m = -INFINITY, lsum = 0.f, mtrue = -INFINITY;

  const float cneg = rel_bias(p, head, -p.sat), cpos = rel_bias(p, head, p.sat);
  // key tiles that any row of the workgroup can see, and of them the workgroup's share
  const int nkb = (len + AT_BK - 1) / AT_BK;
  int kb_lo = cneg == -INFINITY ? max(0, q0 - p.sat + 1) / AT_BK : 0;
  int kb_hi = cpos == -INFINITY ? min(nkb, (q0 + AT_BQ - 2 + p.sat) / AT_BK + 1) : nkb;
  rel_share(p, split, AT_BK, kb_lo, kb_hi);
  if (q0 < len && kb_lo < kb_hi) {                       // (uniform over the workgroup)
    TileLoader<HDP> ld;
    ld.setup(wave, lane, p.c, p.hd);
    const int a0 = row_read_base<HDP>(lane);
    const int vb0 = tr_read_base<HDP>(lane, 0), vb1 = tr_read_base<HDP>(lane, 1);
    const Runs runs = rel_runs<AT_BK>(kb_lo, kb_hi, q0 + wave * 32, p.sat, cneg, cpos);
    const unsigned tile_step = (unsigned)AT_BK * p.c * 2;
    auto issue = [&](int kb, int buf) {
      char* at = smem + buf * 2 * G::TILE;
      ld.issue(static_cast<const __bf16*>(p.k), base, len, p.c, p.hd, at, (unsigned)kb * tile_step, wave);
      ld.issue(static_cast<const __bf16*>(p.v), base, len, p.c, p.hd, at + G::TILE, (unsigned)kb * tile_step, wave);
    };
    issue(kb_lo, 0);
    bf16x8 qf[G::KS];
    own_row<HDP>(qf, p.q, base + (long long)min(qrow, len - 1) * p.c, row_ok, h, p.hd);
    rel_fill(p, head, bias, tid, AT_THREADS);
    // m: the row maximum of the first tile with anything to see, then fixed (scores up to 2^32 above it stay inside fp32);
    // a row that exceeds the margin sends the workgroup through a second walk with the true maxima
    int bad = 0, buf = 0;
    while (true) {
      auto tile = [&](int kb, auto kind, float beyond) {
        constexpr Kind KIND = decltype(kind)::value;
        __syncthreads();
        if (kb + 1 < kb_hi) issue(kb + 1, buf ^ 1);
        const char* kt = smem + buf * 2 * G::TILE;
        const char* vt = kt + G::TILE;
        buf ^= 1;
        const int key0 = kb * AT_BK;

        f32x16 st[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) st[t][e] = 0.f;
        __builtin_amdgcn_s_setprio(1);       // matrix instructions go before the other waves' exponentials
        bf16x8 fk[2][G::SB][2];
        auto load_k = [&](int b, int slot) {
#pragma unroll
          for (int s4 = 0; s4 < G::SB; ++s4)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              fk[slot][s4][t] = *reinterpret_cast<const bf16x8*>(kt + ((a0 ^ ((b * G::SB + s4) << 5)) + t * 32 * G::ROWB));
        };
        load_k(0, 0);
#pragma unroll
        for (int b = 0; b < G::KS / G::SB; ++b) {
          if (b + 1 < G::KS / G::SB) load_k(b + 1, (b + 1) & 1);
#pragma unroll
          for (int s4 = 0; s4 < G::SB; ++s4)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              st[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fk[b & 1][s4][t], qf[b * G::SB + s4], st[t], 0, 0, 0);
        }
        bf16x8 fv[2][G::DT];
        auto load_v = [&](int g, int slot) {
          const int rowoff = (32 * (g >> 1) + 16 * (g & 1)) * G::ROWB;
#pragma unroll
          for (int d = 0; d < G::DT; ++d)
            fv[slot][d] = tr_pair(vt + ((vb0 ^ (d << 6)) + rowoff), vt + ((vb1 ^ (d << 6)) + rowoff));
        };
        load_v(0, 0);
        __builtin_amdgcn_s_setprio(0);

        // score in the log2 domain = st * mul + add
        const float mul = KIND == BEYOND ? p.scale_log2 : 1.f, add = KIND == BEYOND ? beyond : 0.f;
        if constexpr (KIND != BEYOND) {
          const float* bl = bias + (key0 + 4 * h - qrow + p.sat + REL_PAD);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              st[t][e] = fmaf(st[t][e], p.scale_log2, KIND == NEAR ? bl[32 * t + (e & 3) + 8 * (e >> 2)] : beyond);
        }
        if (key0 + AT_BK > len) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (key0 + 32 * t + (e & 3) + 8 * (e >> 2) + 4 * h >= len) st[t][e] = -INFINITY;
        }
        float mx = st[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, st[t][e]);
        mx = fmaf(fmaxf(mx, __shfl_xor(mx, 32, 64)), mul, add);
        mtrue = fmaxf(mtrue, mx);
        m = m == -INFINITY ? mx : m;
        bad |= mx > m + 32.f;
        const float shift = add - (m == -INFINITY ? 0.f : m);
        auto exp_one = [&](int t, int e) {
          const float pe = __builtin_amdgcn_exp2f(KIND == BEYOND ? fmaf(st[t][e], mul, shift) : st[t][e] + shift);
          st[t][e] = pe;
          lsum += pe;
        };
#pragma unroll
        for (int e = 0; e < 8; ++e) exp_one(0, e);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int t = g >> 1, s = g & 1, tn = (g + 1) >> 1, sn = (g + 1) & 1;
          const bf16x8 pb = pack8(st[t], s);
          bf16x8 pl;
          if constexpr (FINE) pl = rest8(st[t], s, pb);
          if (g < 3) load_v(g + 1, (g + 1) & 1);
#pragma unroll
          for (int d = 0; d < G::DT; ++d) {
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv[g & 1][d], pb, acc[d], 0, 0, 0);
            if (g < 3) {
#pragma unroll
              for (int x = d * 8 / G::DT; x < (d + 1) * 8 / G::DT; ++x) exp_one(tn, 8 * sn + x);
            }
          }
          if constexpr (FINE) {
#pragma unroll
            for (int d = 0; d < G::DT; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv[g & 1][d], pl, acc[d], 0, 0, 0);
          }
        }
        __builtin_amdgcn_s_setprio(0);
      };
      int kb = kb_lo;
      for (; kb < runs.f0; ++kb) tile(kb, Beyond{}, cneg);
      for (; kb < runs.n0; ++kb) tile(kb, Flat{}, cneg);
      for (; kb < runs.n1; ++kb) tile(kb, Near{}, 0.f);
      for (; kb < runs.f1; ++kb) tile(kb, Beyond{}, cpos);
      for (; kb < kb_hi; ++kb) tile(kb, Flat{}, cpos);
      if (!(kb_hi - kb_lo > 1 && __syncthreads_or(bad))) break;
      issue(kb_lo, buf);
      m = mtrue;
      lsum = 0.f;
      bad = 0;
#pragma unroll
      for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
    }
  }

  // rows without a single visible key, and rows behind the window's length, give zeros
  const float lt = lsum + __shfl_xor(lsum, 32, 64);
  if (p.splits > 1) {                                    // rel_attn_join_fwd_kernel puts the shares together
    const long long slab = (long long)split * p.n + n;
    if (row_ok) {
      if (h == 0) rel_split_stats(p)[(slab * p.nh + head) * p.l + qrow] = make_float2(m, lt);
      float* sp = p.split + (slab * p.l + qrow) * p.c + hoff;
#pragma unroll
      for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int dd = 32 * d + 8 * e4 + 4 * h;
          if (dd < p.hd) *reinterpret_cast<f32x4*>(sp + dd) = f32x4{acc[d][4 * e4], acc[d][4 * e4 + 1], acc[d][4 * e4 + 2], acc[d][4 * e4 + 3]};
        }
    }
    return;
  }
  const bool seen = row_ok && lt > 0.f;
  const bool spoiled = row_ok && lt != lt;
  const float inv = seen ? 1.f / lt : spoiled ? lt : 0.f;
  if (qrow < p.l) {
    if (lse && h == 0) {
      lse[0] = seen ? m : spoiled ? lt : INFINITY;
      lse[rel_logs(p)] = seen ? __builtin_amdgcn_logf(lt) : 0.f;
    }
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = 32 * d + 8 * e4 + 4 * h;
        if (dd < p.hd) {
          bf16x4 o, rest;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = inv == 0.f ? 0.f : acc[d][4 * e4 + e] * inv;
            o[e] = (__bf16)x;
            rest[e] = (__bf16)(x - (float)o[e]);
          }
          *reinterpret_cast<bf16x4*>(op + dd) = o;
          if (p.rest) *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.rest) + base + (long long)qrow * p.c + dd) = rest;
        }
      }
  }
}

// The shares of a forward pass split over the keys: out = sum_s acc_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).  Four channels a thread.
__global__ __launch_bounds__(AT_THREADS) void rel_attn_join_fwd_kernel(const RelK p) {
  const int c4 = p.c >> 2;
  const long long i = (long long)blockIdx.x * AT_THREADS + threadIdx.x;
  const long long at = i / c4;                           // window and row
  if (at >= (long long)p.n * p.l) return;
  const int n = (int)(at / p.l), row = (int)(at - (long long)n * p.l), ch = (int)(i - at * c4) * 4, head = ch / p.hd;
  const float2* ml = rel_split_stats(p) + ((long long)n * p.nh + head) * p.l + row;
  const long long step = (long long)p.n * p.nh * p.l;
  const bool row_ok = row < rel_length(p, n);
  float m = -INFINITY, lt = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (row_ok) {
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[s * step].x);
    for (int s = 0; s < p.splits; ++s) {
      const float2 a = ml[s * step];
      const float f = a.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a.x - m);
      lt = fmaf(a.y, f, lt);
      acc += *reinterpret_cast<const f32x4*>(p.split + ((long long)s * p.n * p.l + at) * p.c + ch) * f;
    }
  }
  const bool seen = lt > 0.f, spoiled = lt != lt;
  const float inv = seen ? 1.f / lt : spoiled ? lt : 0.f;
  if (p.lse && ch == head * p.hd) {
    float* lse = p.lse + ((long long)n * p.nh + head) * p.l + row;
    lse[0] = seen ? m : spoiled ? lt : INFINITY;
    lse[rel_logs(p)] = seen ? __builtin_amdgcn_logf(lt) : 0.f;
  }
  bf16x4 o, rest;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = inv == 0.f ? 0.f : acc[e] * inv;
    o[e] = (__bf16)x;
    rest[e] = (__bf16)(x - (float)o[e]);
  }
  *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.out) + at * p.c + ch) = o;
  if (p.rest) *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.rest) + at * p.c + ch) = rest;
}

// The shares of a backward pass: dQ and dK (times scale), dV.  Four channels a thread, blockIdx.y the tensor.
__global__ __launch_bounds__(AT_THREADS) void rel_attn_join_bwd_kernel(const RelK p) {
  const long long total = (long long)p.n * p.l * p.c, i = ((long long)blockIdx.x * AT_THREADS + threadIdx.x) * 4;
  if (i >= total) return;
  const int which = blockIdx.y;
  const float* src = p.split + (long long)which * p.splits * total + i;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.splits; ++s) acc += *reinterpret_cast<const f32x4*>(src + s * total);
  if (which < 2) acc *= p.scale;
  bf16x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (__bf16)acc[e];
  void* dst = which == 0 ? p.dq : which == 1 ? p.dk : p.dv;
  *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(dst) + i) = o;
}

// ---------------------------------------------------------------------------------------------
// backward 1/3: delta = <dO, O> (dO is in registers here; dK and dV read it), dQ = scale dS K, and the sums of dS by offset.  Steps of
// 32 keys: 16 scores and 16 dP a lane, so that everything fits the 256 registers of two workgroups a CU.
//
// Sums by offset inside the band: a wave's [32 rows][32 keys] of dS go to its own LDS array with a row pitch of 68 words, 36 of
// them zero; lane d then adds the 32 words of diagonal d (stride 69) and keeps the sum with one read and one write.  Words outside
// the tile fall into the zeros, so nothing is masked; all accesses are conflict-free.  (LDS float atomics, one per score, took
// 85 cycles an instruction: 0.28 of this kernel's 0.74 ms at [32, 1024, 1024].)
// ---------------------------------------------------------------------------------------------
constexpr int BW_ROWS = 32;                         // rows of a streamed tile
constexpr int DG_ZERO = 36, DG_PITCH = DG_ZERO + 32, DG_WORDS = 33 * DG_PITCH;

template <int HDP, bool FINE>
__global__ __launch_bounds__(AT_THREADS, HDP <= REL_OCC2 ? 2 : 1) void rel_attn_dq_kernel(const RelK p) {
  typedef Cfg<HDP> G;
  constexpr int TILE = BW_ROWS * G::ROWB;
  extern __shared__ __attribute__((aligned(16))) char smem[];   // [2 buffers][K tile | V tile], biases, [4 waves] sums, diagonals
  const int w = rel_width(p.sat);
  float* const bias = reinterpret_cast<float*>(smem + 4 * TILE);
  float* const sums = bias + w;
  float* const diag = sums + 4 * w;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;

  int wg = xcd_remap(blockIdx.x, gridDim.x);
  const int nqt = (p.l + AT_BQ - 1) / AT_BQ;
  const int qt = wg % nqt; wg /= nqt;
  const int split = wg % p.splits; wg /= p.splits;
  const int head = wg % p.nh;
  const int n = wg / p.nh;
  const int len = rel_length(p, n);
  const long long base = (long long)n * p.l * p.c + head * p.hd;
  const int q0 = qt * AT_BQ, q0w = q0 + wave * 32, qrow = q0w + r;
  const bool row_ok = qrow < len;

  f32x16 acc[G::DT];
#pragma unroll
  for (int d = 0; d < G::DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
  if (p.part) {
    for (int i = tid; i < 4 * w; i += AT_THREADS) sums[i] = 0.f;
    for (int i = tid; i < 4 * DG_WORDS; i += AT_THREADS) diag[i] = 0.f;
  }
  float fneg = 0.f, fpos = 0.f;

  const float cneg = rel_bias(p, head, -p.sat), cpos = rel_bias(p, head, p.sat);
  const int nkb = (len + BW_ROWS - 1) / BW_ROWS;
  int kb_lo = cneg == -INFINITY ? max(0, q0 - p.sat + 1) / BW_ROWS : 0;
  int kb_hi = cpos == -INFINITY ? min(nkb, (q0 + AT_BQ - 2 + p.sat) / BW_ROWS + 1) : nkb;
  rel_share(p, split, BW_ROWS, kb_lo, kb_hi);
  const bool walks = kb_lo < kb_hi;
  if (q0 < len && (walks || split == 0)) {
    RowLoader<HDP, BW_ROWS> ld;
    ld.setup(wave, lane, p.c, p.hd);
    const __bf16* kbase = static_cast<const __bf16*>(p.k) + base;
    const __bf16* vbase = static_cast<const __bf16*>(p.v) + base;
    const int a0 = row_read_base<HDP>(lane);
    const int vb0 = tr_read_base<HDP>(lane, 0), vb1 = tr_read_base<HDP>(lane, 1);
    auto issue = [&](int kb, int buf) {
      char* at = smem + buf * 2 * TILE;
      ld.issue(kbase, len, p.c, p.hd, at, (unsigned)kb * BW_ROWS, wave);
      ld.issue(vbase, len, p.c, p.hd, at + TILE, (unsigned)kb * BW_ROWS, wave);
    };
    if (walks) issue(kb_lo, 0);
    bf16x8 qf[G::KS], dof[G::KS], of[G::KS], rest[G::KS];
    const long long at = base + (long long)min(qrow, len - 1) * p.c, si = ((long long)n * p.nh + head) * p.l + min(qrow, len - 1);
    own_row<HDP>(dof, p.dout, at, row_ok, h, p.hd);
    own_row<HDP>(of, p.out, at, row_ok, h, p.hd);
    own_row<HDP>(rest, p.rest, at, row_ok, h, p.hd);
    own_row<HDP>(qf, p.q, at, row_ok, h, p.hd);
    const float stat = p.lse[si], logs = p.lse[rel_logs(p) + si];
    const float m = row_ok ? stat : INFINITY, lg = row_ok ? logs : 0.f, lse = m + lg;       // rows past the end: p = 0
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < G::KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)dof[s][e], (float)of[s][e] + (float)rest[s][e], delta);
    delta += __shfl_xor(delta, 32, 64);
    if (split == 0 && h == 0 && row_ok) p.delta[si] = delta;
    rel_fill(p, head, bias, tid, AT_THREADS);
    float* const dg = diag + wave * DG_WORDS;
    int buf = 0;
    auto tile = [&](int kb, auto kind, float beyond, float& fsum) {
      constexpr Kind KIND = decltype(kind)::value;
      __syncthreads();
      if (kb + 1 < kb_hi) issue(kb + 1, buf ^ 1);
      const char* kt = smem + buf * 2 * TILE;
      const char* vt = kt + TILE;
      buf ^= 1;
      const int key0 = kb * BW_ROWS;

      f32x16 st, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) { st[e] = 0.f; dp[e] = 0.f; }
      bf16x8 fk[2], fw[2];
      auto load_kv = [&](int s, int slot) {
        fk[slot] = *reinterpret_cast<const bf16x8*>(kt + (a0 ^ (s << 5)));
        fw[slot] = *reinterpret_cast<const bf16x8*>(vt + (a0 ^ (s << 5)));
      };
      load_kv(0, 0);
#pragma unroll
      for (int s = 0; s < G::KS; ++s) {
        if (s + 1 < G::KS) load_kv(s + 1, (s + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fk[s & 1], qf[s], st, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw[s & 1], dof[s], dp, 0, 0, 0);
      }
      bf16x8 ft[2][G::DT];
      auto load_t = [&](int g, int slot) {
#pragma unroll
        for (int d = 0; d < G::DT; ++d)
          ft[slot][d] = tr_pair(kt + ((vb0 ^ (d << 6)) + 16 * g * G::ROWB), kt + ((vb1 ^ (d << 6)) + 16 * g * G::ROWB));
      };
      load_t(0, 0);
      __builtin_amdgcn_sched_barrier(0);
      const float* bl = bias + (key0 + 4 * h - qrow + p.sat + REL_PAD);
      const float shift = beyond - lse;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if constexpr (KIND == BEYOND) st[e] = __builtin_amdgcn_exp2f(fmaf(st[e], p.scale_log2, shift));
        else st[e] = __builtin_amdgcn_exp2f((fmaf(st[e], p.scale_log2, KIND == NEAR ? bl[(e & 3) + 8 * (e >> 2)] : beyond) - m) - lg);
      }
      if (key0 + BW_ROWS > len) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + (e & 3) + 8 * (e >> 2) + 4 * h >= len) st[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) st[e] *= dp[e] - delta;
      if (p.part) {
        if constexpr (KIND != NEAR) {
#pragma unroll
          for (int e = 0; e < 16; ++e) fsum += st[e];
        } else {
          float* row = dg + r * DG_PITCH + DG_ZERO + 4 * h;
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4)
            *reinterpret_cast<f32x4*>(row + 8 * e4) = f32x4{st[4 * e4], st[4 * e4 + 1], st[4 * e4 + 2], st[4 * e4 + 3]};
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
          const int d = lane < 63 ? lane : 62;                 // diagonal d: key - row = key0 - q0w + d - 31
          const float* src = dg + DG_ZERO - 31 + d;
          float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            s0 += src[(DG_PITCH + 1) * i];
            s1 += src[(DG_PITCH + 1) * (i + 1)];
            s2 += src[(DG_PITCH + 1) * (i + 2)];
            s3 += src[(DG_PITCH + 1) * (i + 3)];
          }
          float* sum = sums + wave * w + (key0 - q0w - 31 + d + p.sat + REL_PAD);
          if (lane < 63) *sum += (s0 + s1) + (s2 + s3);
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const bf16x8 db = pack8(st, g);
        if (g < 1) load_t(1, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < G::DT; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ft[g][d], db, acc[d], 0, 0, 0);
        if constexpr (FINE) {
          const bf16x8 dl = rest8(st, g, db);
#pragma unroll
          for (int d = 0; d < G::DT; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ft[g][d], dl, acc[d], 0, 0, 0);
        }
      }
    };
    const Runs runs = rel_runs<BW_ROWS>(kb_lo, kb_hi, q0w, p.sat, cneg, cpos);
    int kb = kb_lo;
    for (; kb < runs.f0; ++kb) tile(kb, Beyond{}, cneg, fneg);
    for (; kb < runs.n0; ++kb) tile(kb, Flat{}, cneg, fneg);
    for (; kb < runs.n1; ++kb) tile(kb, Near{}, 0.f, fneg);
    for (; kb < runs.f1; ++kb) tile(kb, Beyond{}, cpos, fpos);
    for (; kb < kb_hi; ++kb) tile(kb, Flat{}, cpos, fpos);
  }

  if (p.splits > 1 && qrow < p.l) {
    float* sp = p.split + (((long long)split * p.n + n) * p.l + qrow) * p.c + head * p.hd;
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = 32 * d + 8 * e4 + 4 * h;
        f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = row_ok ? acc[d][4 * e4 + e] : 0.f;
        if (dd < p.hd) *reinterpret_cast<f32x4*>(sp + dd) = o;
      }
  } else if (qrow < p.l) {
    __bf16* yp = static_cast<__bf16*>(p.dq) + base + (long long)qrow * p.c;
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = 32 * d + 8 * e4 + 4 * h;
        if (dd < p.hd) {
          bf16x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (__bf16)(row_ok ? acc[d][4 * e4 + e] * p.scale : 0.f);
          *reinterpret_cast<bf16x4*>(yp + dd) = o;
        }
      }
  }
  if (p.part) {
    __syncthreads();
    fneg = wave_sum(fneg);
    fpos = wave_sum(fpos);
    if (lane == 0) {
      sums[wave * w] += fneg;
      sums[wave * w + w - 1] += fpos;
    }
    __syncthreads();
    float* row = p.part + ((long long)head * p.parts + (n * nqt + qt) * p.splits + split) * (2 * p.sat + 1);
    for (int i = tid; i < 2 * p.sat + 1; i += AT_THREADS) {
      float s = 0.f;
      const int lo = i == 0 ? 0 : i + REL_PAD, hi = i == 2 * p.sat ? w - 1 : i + REL_PAD;      // the flat ends belong to +-sat
      for (int x = lo; x <= hi; ++x)
#pragma unroll
        for (int v = 0; v < 4; ++v) s += sums[v * w + x];
      row[i] = s;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// backward 2/3: dK = scale dS^T Q, dV = P^T dO.  A workgroup owns 128 keys, 32 a wave, and walks the query rows 32 at a time (Q and
// dO tiles, double-buffered).  X = Q K^T has the key on the lane and the rows in the registers, so P and dS are the next products'
// B operands as they stand: dV^T += dO^T P, dK^T += Q^T dS (transposed reads of the tiles).  The accumulators take 128 registers
// at head size 128; the keys' K rows are read from LDS, their V rows stay in registers, and two workgroups fit a CU.  At that size the
// kernel fills its 256 registers and keeps 4 more in scratch (20 with P and dS in 16 bits).
// ---------------------------------------------------------------------------------------------
constexpr int KV_KEYS = 128;
constexpr int KV_STATS = 4 * BW_ROWS;               // of a tile's rows: maximum, log2 of the sum, delta, and the first two added up

template <int HDP, bool FINE>
__global__ __launch_bounds__(AT_THREADS, HDP <= REL_OCC2 ? 2 : 1) void rel_attn_dkv_kernel(const RelK p) {
  typedef Cfg<HDP> G;
  constexpr int TILE = BW_ROWS * G::ROWB;
  extern __shared__ __attribute__((aligned(16))) char smem[];   // [2 buffers][Q tile | dO tile], K rows, [2][4][32] row stats, biases
  char* const krows = smem + 4 * TILE;
  float* const stats = reinterpret_cast<float*>(krows + KV_KEYS * G::ROWB);
  float* const bias = stats + 2 * KV_STATS;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;

  int wg = xcd_remap(blockIdx.x, gridDim.x);
  const int nkt = (p.l + KV_KEYS - 1) / KV_KEYS;
  const int ktl = wg % nkt; wg /= nkt;
  const int split = wg % p.splits; wg /= p.splits;
  const int head = wg % p.nh;
  const int n = wg / p.nh;
  const int len = rel_length(p, n);
  const long long base = (long long)n * p.l * p.c + head * p.hd;
  const int key0 = ktl * KV_KEYS, key0w = key0 + wave * 32, key = key0w + r;
  const bool key_ok = key < len;

  f32x16 dka[G::DT], dva[G::DT];
#pragma unroll
  for (int d = 0; d < G::DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) { dka[d][e] = 0.f; dva[d][e] = 0.f; }

  const float cneg = rel_bias(p, head, -p.sat), cpos = rel_bias(p, head, p.sat);
  // row tiles that can see any of the keys: row - key < sat if the left side is closed, key - row < sat if the right one is
  const int nqb = (len + BW_ROWS - 1) / BW_ROWS;
  int qb_lo = cpos == -INFINITY ? max(0, key0 - p.sat + 1) / BW_ROWS : 0;
  int qb_hi = cneg == -INFINITY ? min(nqb, (key0 + KV_KEYS - 2 + p.sat) / BW_ROWS + 1) : nqb;
  rel_share(p, split, BW_ROWS, qb_lo, qb_hi);
  if (key0 < len && qb_lo < qb_hi) {
    {
      RowLoader<HDP, KV_KEYS> lk;
      lk.setup(wave, lane, p.c, p.hd);
      lk.issue(static_cast<const __bf16*>(p.k) + base, len, p.c, p.hd, krows, (unsigned)key0, wave);
    }
    RowLoader<HDP, BW_ROWS> ld;
    ld.setup(wave, lane, p.c, p.hd);
    const __bf16* qbase = static_cast<const __bf16*>(p.q) + base;
    const __bf16* dbase = static_cast<const __bf16*>(p.dout) + base;
    const int a0 = row_read_base<HDP>(lane);
    const char* const kw = krows + wave * 32 * G::ROWB;
    const int vb0 = tr_read_base<HDP>(lane, 0), vb1 = tr_read_base<HDP>(lane, 1);
    auto issue = [&](int qb, int buf) {
      char* at = smem + buf * 2 * TILE;
      ld.issue(qbase, len, p.c, p.hd, at, (unsigned)qb * BW_ROWS, wave);
      ld.issue(dbase, len, p.c, p.hd, at + TILE, (unsigned)qb * BW_ROWS, wave);
    };
    const long long sbase = ((long long)n * p.nh + head) * p.l;
    auto load_stat = [&](int qb) {                   // 32 threads a kind
      const int which = tid / BW_ROWS, row = qb * BW_ROWS + (tid & (BW_ROWS - 1));
      float v = which == 0 || which == 3 ? INFINITY : 0.f;      // rows past the end: p = 0, delta = 0
      if (which < 4 && row < len) {
        v = which == 2 ? p.delta[sbase + row] : p.lse[(which == 1 ? rel_logs(p) : 0) + sbase + row];
        if (which == 3) v += p.lse[rel_logs(p) + sbase + row];
      }
      return v;
    };
    issue(qb_lo, 0);
    bf16x8 vf[G::KS];
    own_row<HDP>(vf, p.v, base + (long long)min(key, len - 1) * p.c, key_ok, h, p.hd);
    rel_fill(p, head, bias, tid, AT_THREADS);
    if (tid < KV_STATS) stats[tid] = load_stat(qb_lo);
    int buf = 0;
    auto tile = [&](int qb, auto kind, float beyond) {
      constexpr Kind KIND = decltype(kind)::value;
      __syncthreads();   // the tile and its stats are in LDS; every wave is done with the other buffer
      float stat_next = 0.f;
      if (qb + 1 < qb_hi) {
        issue(qb + 1, buf ^ 1);
        stat_next = load_stat(qb + 1);
      }
      const char* qtile = smem + buf * 2 * TILE;
      const char* dtile = qtile + TILE;
      const float* st_in = stats + buf * KV_STATS;
      const int row0 = qb * BW_ROWS;
      f32x16 st, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) { st[e] = 0.f; dp[e] = 0.f; }
      bf16x8 fq[2], fd[2], fk[2];
      auto load_qd = [&](int s, int slot) {
        fq[slot] = *reinterpret_cast<const bf16x8*>(qtile + (a0 ^ (s << 5)));
        fk[slot] = *reinterpret_cast<const bf16x8*>(kw + (a0 ^ (s << 5)));
        fd[slot] = *reinterpret_cast<const bf16x8*>(dtile + (a0 ^ (s << 5)));
      };
      load_qd(0, 0);
#pragma unroll
      for (int s = 0; s < G::KS; ++s) {
        if (s + 1 < G::KS) load_qd(s + 1, (s + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fq[s & 1], fk[s & 1], st, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fd[s & 1], vf[s], dp, 0, 0, 0);
      }
      constexpr int NTB = 2 * G::DT;               // batches over (k-step s, d)
      bf16x8 tq[2], td[2];
      auto load_tt = [&](int b, int slot) {
        const int s = b / G::DT, d0 = b % G::DT;
        const int o0 = (vb0 ^ (d0 << 6)) + 16 * s * G::ROWB, o1 = (vb1 ^ (d0 << 6)) + 16 * s * G::ROWB;
        td[slot] = tr_pair(dtile + o0, dtile + o1);
        tq[slot] = tr_pair(qtile + o0, qtile + o1);
      };
      load_tt(0, 0);
      __builtin_amdgcn_sched_barrier(0);
      const float* bl = bias + (key - row0 - 4 * h - 27 + p.sat + REL_PAD);     // bl[27 - x]: local row x + 4h
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        auto stat = [&](int which) { return *reinterpret_cast<const f32x4*>(st_in + which * BW_ROWS + 8 * e4 + 4 * h); };
        const f32x4 ls = stat(KIND == BEYOND ? 3 : 0), de = stat(2);
        f32x4 lg;
        if constexpr (KIND != BEYOND) lg = stat(1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float pe;
          if constexpr (KIND == BEYOND) pe = __builtin_amdgcn_exp2f(fmaf(st[4 * e4 + e], p.scale_log2, beyond - ls[e]));
          else pe = __builtin_amdgcn_exp2f((fmaf(st[4 * e4 + e], p.scale_log2, KIND == NEAR ? bl[27 - 8 * e4 - e] : beyond) - ls[e]) - lg[e]);
          st[4 * e4 + e] = pe;
          dp[4 * e4 + e] = pe * (dp[4 * e4 + e] - de[e]);
        }
      }
#pragma unroll
      for (int b = 0; b < NTB; ++b) {
        const int s = b / G::DT, d0 = b % G::DT;
        const bf16x8 pb = pack8(st, s), db = pack8(dp, s);
        if (b + 1 < NTB) load_tt(b + 1, (b + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
        dva[d0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(td[b & 1], pb, dva[d0], 0, 0, 0);
        dka[d0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tq[b & 1], db, dka[d0], 0, 0, 0);
        if constexpr (FINE) {
          dva[d0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(td[b & 1], rest8(st, s, pb), dva[d0], 0, 0, 0);
          dka[d0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tq[b & 1], rest8(dp, s, db), dka[d0], 0, 0, 0);
        }
      }
      if (qb + 1 < qb_hi && tid < KV_STATS) stats[(buf ^ 1) * KV_STATS + tid] = stat_next;
      buf ^= 1;
    };
    const Runs runs = rel_runs<BW_ROWS>(qb_lo, qb_hi, key0w, p.sat, cpos, cneg);       // rows in front of the keys: key - row > 0
    int qb = qb_lo;
    for (; qb < runs.f0; ++qb) tile(qb, Beyond{}, cpos);
    for (; qb < runs.n0; ++qb) tile(qb, Flat{}, cpos);
    for (; qb < runs.n1; ++qb) tile(qb, Near{}, 0.f);
    for (; qb < runs.f1; ++qb) tile(qb, Beyond{}, cneg);
    for (; qb < qb_hi; ++qb) tile(qb, Flat{}, cneg);
  }

  if (p.splits > 1 && key < p.l) {
    const long long total = (long long)p.n * p.l * p.c;
    float* sk = p.split + (p.splits + split) * total + base + (long long)key * p.c;
    float* sv = sk + p.splits * total;
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = 32 * d + 8 * e4 + 4 * h;
        f32x4 ok, ov;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ok[e] = key_ok ? dka[d][4 * e4 + e] : 0.f;
          ov[e] = key_ok ? dva[d][4 * e4 + e] : 0.f;
        }
        if (dd < p.hd) {
          *reinterpret_cast<f32x4*>(sk + dd) = ok;
          *reinterpret_cast<f32x4*>(sv + dd) = ov;
        }
      }
  } else if (key < p.l) {
    __bf16* dk = static_cast<__bf16*>(p.dk) + base + (long long)key * p.c;
    __bf16* dv = static_cast<__bf16*>(p.dv) + base + (long long)key * p.c;
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = 32 * d + 8 * e4 + 4 * h;
        if (dd < p.hd) {
          bf16x4 ok, ov;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ok[e] = (__bf16)(key_ok ? dka[d][4 * e4 + e] * p.scale : 0.f);
            ov[e] = (__bf16)(key_ok ? dva[d][4 * e4 + e] : 0.f);
          }
          *reinterpret_cast<bf16x4*>(dk + dd) = ok;
          *reinterpret_cast<bf16x4*>(dv + dd) = ov;
        }
      }
  }
}

// ---------------------------------------------------------------------------------------------
// backward 3/3: d table[b][head] = the sums of dS over the offsets of bucket b, added up over the dQ kernel's workgroups
// ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(AT_THREADS) void rel_attn_dtable_kernel(const RelK p, void* dtable) {
  __shared__ int range[2];
  __shared__ double wsum[4];
  const int b = blockIdx.x, head = blockIdx.y, side = p.buckets >> 1, tid = threadIdx.x;
  const int local = b < side ? b : b - side;
  if (tid == 0) { range[0] = p.sat + 1; range[1] = -1; }
  __syncthreads();
  for (int a = tid; a <= p.sat; a += AT_THREADS)
    if (p.bucket[a] == local && !(a == 0 && b >= side)) { atomicMin(&range[0], a); atomicMax(&range[1], a); }
  __syncthreads();
  const int a0 = range[0], cnt = range[1] - range[0] + 1;      // distances a0 .. a0+cnt-1; none: cnt <= 0
  double s = 0.0;                                 // (the sums of a bucket cancel)
  if (cnt > 0) {
    const float* src = p.part + (long long)head * p.parts * (2 * p.sat + 1);
    const int first = b < side ? p.sat - (a0 + cnt - 1) : p.sat + a0;
    const long long total = (long long)p.parts * cnt;
    for (long long i = tid; i < total; i += AT_THREADS) {
      const long long row = i / cnt;
      s += (double)src[row * (2 * p.sat + 1) + first + (int)(i - row * cnt)];
    }
  }
  for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((tid & 63) == 0) wsum[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    const float t = (float)((wsum[0] + wsum[1]) + (wsum[2] + wsum[3]));
    if (p.table_f32) static_cast<float*>(dtable)[b * p.nh + head] = t;
    else static_cast<__bf16*>(dtable)[b * p.nh + head] = (__bf16)t;
  }
}

#define REL_INSTANTIATE(HDP, FINE)                                     \
  template __global__ void rel_attn_fwd_kernel<HDP, FINE>(const RelK); \
  template __global__ void rel_attn_dkv_kernel<HDP, FINE>(const RelK);
REL_INSTANTIATE(32, false)
REL_INSTANTIATE(64, false)
REL_INSTANTIATE(128, false)
REL_INSTANTIATE(256, false)
REL_INSTANTIATE(32, true)
REL_INSTANTIATE(64, true)
REL_INSTANTIATE(128, true)
REL_INSTANTIATE(256, true)
#undef REL_INSTANTIATE
template __global__ void rel_attn_dq_kernel<32, true>(const RelK);
template __global__ void rel_attn_dq_kernel<64, false>(const RelK);
template __global__ void rel_attn_dq_kernel<64, true>(const RelK);
template __global__ void rel_attn_dq_kernel<128, false>(const RelK);
template __global__ void rel_attn_dq_kernel<128, true>(const RelK);
template __global__ void rel_attn_dq_kernel<256, false>(const RelK);
template __global__ void rel_attn_dq_kernel<256, true>(const RelK);

size_t bias_bytes(int sat, int copies) { return (size_t)rel_width(sat) * sizeof(float) * copies; }

template <typename K> int set_lds(K kernel, size_t bytes, const char* what) {
  if (bytes > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    UNET_REQUIRE(e == hipSuccess, "%s: hipFuncSetAttribute failed: %s", what, hipGetErrorString(e));
  }
  return 0;
}

template <int HDP, bool FINE> int launch_fwd(const RelK& p, hipStream_t st) {
  const size_t lds = 4 * (size_t)Cfg<HDP>::TILE + bias_bytes(p.sat, 1);
  if (set_lds(&rel_attn_fwd_kernel<HDP, FINE>, lds, "rel_attn_fwd")) return -1;
  hipLaunchKernelGGL((rel_attn_fwd_kernel<HDP, FINE>), dim3((unsigned)(p.n * p.nh * cdiv(p.l, AT_BQ) * p.splits)), dim3(AT_THREADS), lds, st, p);
  UNET_LAUNCH_CHECK("rel_attn_fwd");
  return 0;
}

template <int HDP, bool FINE> int launch_dq(const RelK& p, hipStream_t st) {
  const size_t lds = 4 * (size_t)BW_ROWS * Cfg<HDP>::ROWB + bias_bytes(p.sat, 1) +
                     (p.part ? bias_bytes(p.sat, 4) + 4 * DG_WORDS * sizeof(float) : 0);
  constexpr bool F = FINE || HDP <= 32;
  if (set_lds(&rel_attn_dq_kernel<HDP, F>, lds, "rel_attn_bwd (dq)")) return -1;
  hipLaunchKernelGGL((rel_attn_dq_kernel<HDP, F>), dim3((unsigned)(p.n * p.nh * cdiv(p.l, AT_BQ) * p.splits)), dim3(AT_THREADS), lds, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (dq)");
  return 0;
}

template <int HDP, bool FINE> int launch_dkv(const RelK& p, hipStream_t st) {
  const size_t lds = (4 * (size_t)BW_ROWS + KV_KEYS) * Cfg<HDP>::ROWB + 2 * KV_STATS * sizeof(float) + bias_bytes(p.sat, 1);
  if (set_lds(&rel_attn_dkv_kernel<HDP, FINE>, lds, "rel_attn_bwd (dk, dv)")) return -1;
  hipLaunchKernelGGL((rel_attn_dkv_kernel<HDP, FINE>), dim3((unsigned)(p.n * p.nh * cdiv(p.l, KV_KEYS) * p.splits)), dim3(AT_THREADS), lds, st, p);
  UNET_LAUNCH_CHECK("rel_attn_bwd (dk, dv)");
  return 0;
}

// Where P and dS are carried to 16 bits (FINE: the rounded value and its rest, two matrix products).  Rounded to bf16 once, their
// error is that of one more rounding of the result: 1.41 times the error of the final rounding alone, averaged over many rows.
//  - Forward in front of a backward pass: delta = <dO, O> must match the fp32 P that backward recomputes, or dP - delta loses its
//    leading digits where one key dominates (dQ, dK and the table's gradient had up to 7 times the error of a 32-bit form).
//    [32, 1024, 1024]: forward 171 -> 233 us, of a training pass of 0.85 ms; at [32, 1024], 8 heads of 32, 64 -> 90.
//  - Windows of one row tile, whose few rows average nothing: [32, 128], 8 heads of 128, forward 12.1 -> 12.6 us, backward 76 us
//    either way.
//  - dQ of heads up to 32, where the sum of dS K cancels most (1.6 times at heads of 8): backward of [32, 1024], 8 heads of 32,
//    246 -> 265 us.  dK and dV do not need it (1.41 there too).
bool one_tile(const RelK& p) { return p.l <= AT_BQ; }

#define REL_DISPATCH(fn, fine, p, st)                                              \
  do {                                                                             \
    if ((p).hd <= 32) return (fine) ? fn<32, true>(p, st) : fn<32, false>(p, st);    \
    if ((p).hd <= 64) return (fine) ? fn<64, true>(p, st) : fn<64, false>(p, st);    \
    if ((p).hd <= 128) return (fine) ? fn<128, true>(p, st) : fn<128, false>(p, st); \
    return (fine) ? fn<256, true>(p, st) : fn<256, false>(p, st);                    \
  } while (0)
int launch_fwd_bf16(const RelK& p, hipStream_t st) { REL_DISPATCH(launch_fwd, p.lse || one_tile(p), p, st); }
int launch_dq_bf16(const RelK& p, hipStream_t st) { REL_DISPATCH(launch_dq, p.hd <= 32 || one_tile(p), p, st); }
int launch_dkv_bf16(const RelK& p, hipStream_t st) { REL_DISPATCH(launch_dkv, one_tile(p), p, st); }

// Few rows in a long window: workgroups of 128 rows would leave CUs idle while each walks the whole window.  The walked axis is
// then cut into shares of at least 512 rows, up to two workgroups a CU, and a further launch adds up their fp32 sums.  Unsplit
// against split, one window, 2 heads, forward and backward of a training pass: [2048] heads of 128 51 and 28, 154 and 85 us; heads of
// 256 92 and 42, 271 and 120; [8192] heads of 64 121 and 68, 444 and 186.  [1024] gains nothing (22 and 24, 82 and 88), and
// shares of 256 are no faster.
int rel_splits(int dtype, int n, int l, int nh) {
  const long long wgs = (long long)n * nh * cdiv(l, AT_BQ);
  if (dtype != UNET_BF16 || wgs > 128) return 1;
  const int most = l / 512, want = (int)(512 / wgs);
  return most < 3 ? 1 : want < most ? want : most;
}

// argument checks shared by the entry points; fills everything of RelK but the tensors
int make_rel(const char* what, RelK& p, int32_t dtype, int32_t n, int32_t l, int32_t c, int32_t nh, float scale, const void* table,
             int32_t table_f32, int32_t buckets, const int32_t* starts_host, const int32_t* lengths) {
  UNET_REQUIRE(dtype == UNET_BF16 || dtype == UNET_F32, "%s: bad dtype %d", what, dtype);
  UNET_REQUIRE(table && starts_host, "%s: null pointer", what);
  UNET_REQUIRE(n > 0 && l > 0 && c > 0 && nh > 0 && nh <= 256 && n <= 65535, "%s: bad shape n=%d l=%d c=%d heads=%d", what, n, l, c, nh);
  const int unit = dtype == UNET_BF16 ? 8 : 4;
  UNET_REQUIRE(c % nh == 0 && (c / nh) % unit == 0 && c / nh <= 256,
               "%s: head_dim %d must be a multiple of %d and at most 256 (c=%d heads=%d)", what, c / nh, unit, c, nh);
  UNET_REQUIRE((long long)l * c * (dtype == UNET_BF16 ? 2 : 4) < (1ll << 31), "%s: one [L, C] slab of %lld bytes exceeds a buffer descriptor",
               what, (long long)l * c * (dtype == UNET_BF16 ? 2 : 4));
  UNET_REQUIRE((long long)n * nh * cdiv(l, dtype == UNET_BF16 ? AT_BQ : 64) < (1ll << 24),      // 256 threads each, counted in 32 bits
               "%s: n=%d windows of l=%d rows with %d heads take 2^24 workgroups or more", what, n, l, nh);
  UNET_REQUIRE(scale > 0.f && scale * REL_LOG2E < INFINITY, "%s: scale must be positive and finite (also times log2 e), got %g", what,
               (double)scale);
  UNET_REQUIRE(buckets >= 4 && buckets % 2 == 0 && buckets <= 2 * UNET_REL_MAX_SIDE, "%s: %d buckets, must be even and 4 .. %d", what,
               buckets, 2 * UNET_REL_MAX_SIDE);
  const int side = buckets / 2;
  UNET_REQUIRE(starts_host[0] == 0, "%s: the first bucket must start at distance 0", what);
  for (int i = 1; i < side; ++i)
    UNET_REQUIRE(starts_host[i] >= starts_host[i - 1], "%s: bucket starts must not decrease", what);
  const int sat = starts_host[side - 1];
  UNET_REQUIRE(sat >= 1 && sat <= UNET_REL_MAX_DISTANCE, "%s: the last bucket must start at distance 1 .. %d, got %d", what,
               UNET_REL_MAX_DISTANCE, sat);
  p.splits = rel_splits(dtype, n, l, nh);
  p.n = n; p.l = l; p.c = c; p.nh = nh; p.hd = c / nh; p.buckets = buckets; p.sat = sat;
  p.table = table; p.table_f32 = table_f32; p.lengths = lengths;
  p.scale = scale; p.scale_log2 = scale * REL_LOG2E;
  for (int a = 0, b = 0; a <= sat; ++a) {
    while (b + 1 < side && starts_host[b + 1] <= a) ++b;
    p.bucket[a] = (unsigned char)b;
  }
  return 0;
}

size_t workspace_bytes(int splits, int n, int l, int c, int nh, int backward) {
  if (splits < 2) return 0;
  const size_t rows = (size_t)splits * n * l;
  return rows * (backward ? 3 * (size_t)c : (size_t)c + 2 * (size_t)nh) * sizeof(float);
}
int take_workspace(const char* what, RelK& p, void* workspace, size_t bytes, int backward) {
  const size_t need = workspace_bytes(p.splits, p.n, p.l, p.c, p.nh, backward);
  UNET_REQUIRE(workspace && bytes >= need && aligned16(workspace), "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, bytes, need);
  p.split = static_cast<float*>(workspace);
  return 0;
}

// rows of partial sums: one a workgroup of the dQ kernel
int rel_parts(int dtype, int n, int l, int nh, int hd) {
  return dtype == UNET_BF16 ? n * cdiv(l, AT_BQ) * rel_splits(dtype, n, l, nh) : n * cdiv(l, rel32_rows(n, l, nh, hd));
}

}  // namespace

extern "C" int unet_rel_attn_fwd(int32_t dtype, const void* q, const void* k, const void* v, const void* table, int32_t table_f32,
                                 int32_t buckets, const int32_t* starts_host, const int32_t* lengths, int32_t n, int32_t l, int32_t c,
                                 int32_t n_heads, float scale, void* out, void* out_rest, float* lse, void* workspace,
                                 size_t ws_bytes, void* stream) {
  RelK p = {};
  UNET_REQUIRE(q && k && v && out, "rel_attn_fwd: null pointer");
  UNET_REQUIRE(dtype != UNET_BF16 || !lse == !out_rest, "rel_attn_fwd: a bf16 backward pass needs lse and out_rest, inference neither");
  if (make_rel("rel_attn_fwd", p, dtype, n, l, c, n_heads, scale, table, table_f32, buckets, starts_host, lengths)) return -1;
  UNET_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out_rest), "rel_attn_fwd: pointers must be 16-byte aligned");
  p.q = q; p.k = k; p.v = v; p.out = out; p.rest = out_rest; p.lse = lse;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == UNET_F32) return unet_rel_attn_fwd_f32(p, st);
  if (p.splits == 1) return launch_fwd_bf16(p, st);
  if (take_workspace("rel_attn_fwd", p, workspace, ws_bytes, 0) || launch_fwd_bf16(p, st)) return -1;
  hipLaunchKernelGGL(rel_attn_join_fwd_kernel, dim3((unsigned)(((long long)n * l * (c / 4) + AT_THREADS - 1) / AT_THREADS)),
                     dim3(AT_THREADS), 0, st, p);
  UNET_LAUNCH_CHECK("rel_attn_fwd (join)");
  return 0;
}

extern "C" size_t unet_rel_attn_workspace_bytes(int32_t dtype, int32_t n, int32_t l, int32_t c, int32_t n_heads, int32_t backward) {
  if (n <= 0 || l <= 0 || c <= 0 || n_heads <= 0) return 0;
  return workspace_bytes(rel_splits(dtype, n, l, n_heads), n, l, c, n_heads, backward);
}

extern "C" size_t unet_rel_attn_bwd_partials(int32_t dtype, int32_t n, int32_t l, int32_t n_heads, int32_t last_start) {
  if (n <= 0 || l <= 0 || n_heads <= 0 || last_start < 0) return 0;
  return (size_t)n_heads * rel_parts(dtype, n, l, n_heads, 1) * (2 * (size_t)last_start + 1);
}

extern "C" int unet_rel_attn_bwd(int32_t dtype, const void* q, const void* k, const void* v, const void* table, int32_t table_f32,
                                 int32_t buckets, const int32_t* starts_host, const int32_t* lengths, const void* out, const void* out_rest,
                                 const float* lse, const void* dout, int32_t n, int32_t l, int32_t c, int32_t n_heads, float scale, void* dq, void* dk,
                                 void* dv, void* dtable, float* partials, float* delta, void* workspace, size_t ws_bytes,
                                 void* stream) {
  RelK p = {};
  UNET_REQUIRE(q && k && v && out && lse && dout && dq && dk && dv && delta, "rel_attn_bwd: null pointer");
  UNET_REQUIRE(dtype != UNET_BF16 || out_rest, "rel_attn_bwd: null pointer (out_rest)");
  UNET_REQUIRE(!dtable || partials, "rel_attn_bwd: the table's gradient needs the partial sums");
  if (make_rel("rel_attn_bwd", p, dtype, n, l, c, n_heads, scale, table, table_f32, buckets, starts_host, lengths)) return -1;
  UNET_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out_rest) && aligned16(dout) && aligned16(dq) && aligned16(dk) &&
                   aligned16(dv), "rel_attn_bwd: pointers must be 16-byte aligned");
  p.q = q; p.k = k; p.v = v; p.out = const_cast<void*>(out); p.rest = const_cast<void*>(out_rest);
  p.lse = const_cast<float*>(lse); p.dout = dout;
  p.dq = dq; p.dk = dk; p.dv = dv; p.delta = delta; p.part = dtable ? partials : nullptr; p.parts = rel_parts(dtype, n, l, n_heads, p.hd);
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc;
  if (dtype == UNET_F32) rc = unet_rel_attn_bwd_f32(p, st);
  else {
    if (p.splits > 1 && take_workspace("rel_attn_bwd", p, workspace, ws_bytes, 1)) return -1;
    rc = launch_dq_bf16(p, st);
    if (!rc) rc = launch_dkv_bf16(p, st);
    if (!rc && p.splits > 1) {
      hipLaunchKernelGGL(rel_attn_join_bwd_kernel, dim3((unsigned)(((long long)n * l * (c / 4) + AT_THREADS - 1) / AT_THREADS), 3),
                         dim3(AT_THREADS), 0, st, p);
      UNET_LAUNCH_CHECK("rel_attn_bwd (join)");
    }
  }
  if (rc || !dtable) return rc;
  hipLaunchKernelGGL(rel_attn_dtable_kernel, dim3(buckets, n_heads), dim3(AT_THREADS), 0, st, p, dtable);
  UNET_LAUNCH_CHECK("rel_attn_bwd (dtable)");
  return 0;
}
