// What the bf16 and fp32 kernels of relative-bias attention share: arguments, the bias of an offset, the sums of its gradient.
#pragma once
#include "common.h"

struct RelK {
  const void *q, *k, *v;       // [N][L][C], head h in columns h*hd .. h*hd+hd-1
  void* out;                   // [N][L][C]
  void* rest;                  // [N][L][C] or null (bf16 with a backward pass): what rounding took from out
  float* lse;                  // [2][N][nh][L] or null: a reference m of the row's scores (bf16: in the log2 domain; +inf: nothing to
                               // see) and the log2 of the sum over m.  Two planes, p = exp2((s - m) - log): a score that a large finite bias
                               // absorbed differs from m by nothing, and log2 of the sum is not lost beside such an m
  const void* dout;            // [N][L][C]
  float* delta;                // [N][nh][L]: <dO, O> of a row and head
  void *dq, *dk, *dv;          // [N][L][C]
  const void* table;           // [buckets][nh], fp32 or bf16
  float* part;                 // [nh][parts][2*sat+1] sums of dS by offset, one row per workgroup of the dQ kernel, or null
  const int* lengths;          // [N] valid positions, or null
  float* split;                // bf16, few rows: [splits][N][L][C] sums of a workgroup's share of the walked axis (backward: three of
                               // them, dQ | dK | dV); behind them, forward, [splits][N][nh][L] (maximum, sum)
  int n, l, c, nh, hd, buckets, sat, parts, table_f32, splits;
  float scale, scale_log2;
  unsigned char bucket[UNET_REL_MAX_DISTANCE + 1];   // of |offset| = 0 .. sat within its side; sat: start of the last one
};

int unet_rel_attn_fwd_f32(const RelK& p, hipStream_t st);
int unet_rel_attn_bwd_f32(const RelK& p, hipStream_t st);

namespace {

// Rows a workgroup of the fp32 kernels owns: 16 where workgroups of 64 would take at most half of the CUs, 64 otherwise.  Forward,
// 64 against 16, heads of 64 at [2, 512] 39.7 and 17.2 us, [4, 512] (128 workgroups) 40.5 and 23.3, [7, 512] (224) 41.1 and 41.5; heads
// of 128 at [2, 500] 62 and 27, [7, 510] 66 and 103.  Heads of more than 128 stay at 64: the 128 rows of the other side that a
// workgroup of 16 takes a step would not fit the LDS.
__host__ __forceinline__ int rel32_rows(int n, int l, int nh, int hd) { return hd <= 128 && (long long)n * nh * cdiv(l, 64) <= 128 ? 16 : 64; }

constexpr float REL_LOG2E = 1.4426950408889634f;
constexpr float REL_LOWEST = -1e30f;    // finite biases stop here and at 1e30: the type's lowest and highest values, or sums with them,
                                        // must not become infinite
// LDS copy of a head's biases by offset: index REL_PAD + sat + offset, flat beyond +-sat for REL_PAD entries each way, so a
// tile that touches the band between -sat and sat reads it without clamping
constexpr int REL_PAD = 96;
__device__ __host__ __forceinline__ int rel_width(int sat) { return (2 * sat + 1 + 2 * REL_PAD + 3) & ~3; }      // 16-byte multiple

// Bias of key j seen from query i, off = j - i, times `unit`: log2(e) for scores in the log2 domain (bf16), 1 for natural ones
// (fp32).  An infinite entry or a NaN stays what it is; a finite one is held within +-1e30 (the type's lowest value times log2(e), or
// with a score added, would be -inf, which means "never"; its highest +inf, which makes NaN).
__device__ __forceinline__ float rel_bias(const RelK& p, int head, int off, float unit = REL_LOG2E) {
  const int a = min(abs(off), p.sat);
  const int b = p.bucket[a] + (off > 0 ? p.buckets >> 1 : 0);
  const float v = p.table_f32 ? static_cast<const float*>(p.table)[b * p.nh + head]
                              : (float)static_cast<const __bf16*>(p.table)[b * p.nh + head];
  return fabsf(v) < INFINITY ? fminf(fmaxf(v * unit, REL_LOWEST), -REL_LOWEST) : v;
}

__device__ __forceinline__ long long rel_logs(const RelK& p) { return (long long)p.n * p.nh * p.l; }      // lse: start of the logs

__device__ __forceinline__ int rel_length(const RelK& p, int n) {
  return p.lengths ? max(0, min(p.lengths[n], p.l)) : p.l;
}

__device__ __forceinline__ void rel_fill(const RelK& p, int head, float* bias, int tid, int threads, float unit = REL_LOG2E) {
  const int w = rel_width(p.sat);
  for (int i = tid; i < w; i += threads) {
    const int off = i - REL_PAD - p.sat;
    bias[i] = rel_bias(p, head, max(-p.sat, min(off, p.sat)), unit);
  }
}

}  // namespace
