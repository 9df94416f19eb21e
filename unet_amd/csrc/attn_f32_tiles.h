// Tile primitives of the exact-fp32 attention kernels (attn_f32.hip, relattn_f32.hip); attn_f32.hip's header explains the
// operand layout.
#pragma once
#include "common.h"

namespace {

constexpr int A32_THREADS = 256;
constexpr int A32_ROWS = 64;     // rows owned by a workgroup (16 per wave)
constexpr int A32_BK = 32;       // rows of a streamed tile

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// [rows][HDP] tile of a [L][C] slab (head columns hoff .. hoff+hd) -> LDS with row pitch HDP+4; rows past the end and
// columns past hd arrive as zeros
template <int HDP, int ROWS>
__device__ __forceinline__ void load_tile(float* tile, const float* slab, int row0, int l, int ld, int hd, int tid) {
  constexpr int LD = HDP + 4, CH = HDP / 4;
  for (int i = tid; i < ROWS * CH; i += A32_THREADS) {
    const int r = i / CH, ch = i - r * CH;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (row0 + r < l && ch * 4 < hd) v = *reinterpret_cast<const f32x4*>(slab + (long long)(row0 + r) * ld + ch * 4);
    *reinterpret_cast<f32x4*>(tile + r * LD + ch * 4) = v;
  }
}

// the wave's 16 operand rows as float4 chunks (see the header): reg[u] = row[16u + 4g .. +3]
template <int HDP>
__device__ __forceinline__ void load_rows(f32x4 (&reg)[HDP / 16], const float* rowp, bool ok, int g, int hd) {
#pragma unroll
  for (int u = 0; u < HDP / 16; ++u) {
    const int col = 16 * u + 4 * g;
    reg[u] = (ok && col < hd) ? *reinterpret_cast<const f32x4*>(rowp + col) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// C[row 4g+i][col l15] (+)= sum_k A[row][k] B[col][k]: A rows from an LDS tile (16 rows starting at `arow`), B rows from
// the register chunks
template <int HDP>
__device__ __forceinline__ f32x4 rows_dot(const float* tile, int arow, const f32x4 (&breg)[HDP / 16], int l15, int g) {
  constexpr int LD = HDP + 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < HDP / 16; ++u) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(tile + (arow + l15) * LD + 16 * u + 4 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = mfma4(a[e], breg[u][e], acc);
  }
  return acc;
}

// acc^T[d = 16dt + 4g + i][col l15] += sum over the 16 rows (arow ..) of  tile[row][d] * b[row][col], where b is an
// accumulator in the C layout (rows 4g+i): register t <-> k index g of step t
template <int HDP>
__device__ __forceinline__ void rows_acc(f32x4 (&acc)[HDP / 16], const float* tile, int arow, const f32x4& b, int l15, int g) {
  constexpr int LD = HDP + 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float* rp = tile + (arow + 4 * g + t) * LD + l15;
#pragma unroll
    for (int dt = 0; dt < HDP / 16; ++dt) acc[dt] = mfma4(rp[16 * dt], b[t], acc[dt]);
  }
}

__device__ __forceinline__ float group_max(float v) {      // over the 4 lane groups that share (l & 15)
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

}  // namespace
