// Tile primitives of the bf16 flash-attention kernels (attn.hip, relattn.hip): the LDS image of a [64][HDP] tile, its two
// kinds of fragment reads, and the loads that fill it.
#pragma once
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) short s16x8;

constexpr int AT_THREADS = 256;
constexpr int AT_BQ = 128;   // rows owned by a workgroup (32 per wave)
constexpr int AT_BK = 64;    // rows of a streamed tile
constexpr unsigned AT_OOB = 0x80000000u;

template <int HDP> struct Cfg {
  static constexpr int ROWB = HDP * 2;                 // bytes per tile row
  static constexpr int CPR = HDP / 8;                  // 16-byte chunks per row
  static constexpr int XM = CPR >= 16 ? 15 : CPR - 1;  // swizzle mask
  static constexpr int KS = HDP / 16;                  // k-steps over the head dim
  static constexpr int DT = HDP / 32;                  // 32-wide tiles over the head dim
  static constexpr int TILE = AT_BK * ROWB;            // bytes of a [64][HDP] tile
  static constexpr int PPW = TILE / 1024 / 4;          // 1 KiB pieces per wave
  static constexpr int SB = KS < 4 ? KS : 4;           // k-steps per batch of row-read fragments
};

// chunk swizzle of the LDS images: rows that differ in their low two bits land in different 64-byte groups
// (transposed reads), 16 rows of a ds_read_b128 lane group land on 16 different chunks
__device__ __forceinline__ int xv(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

__device__ __forceinline__ bf16x8 tr_pair(const char* lo, const char* hi) {
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi);
  const s16x8 t = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, t);
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& x, int s) {   // registers 8s..8s+7 -> bf16 fragment of k-step s
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = (__bf16)x[8 * s + j];
  return o;
}

// ---- streamed [64][HDP] tile: global -> LDS by buffer_load ... lds ---------------------------
template <int HDP> struct TileLoader {
  unsigned voff[Cfg<HDP>::PPW];
  __device__ __forceinline__ void setup(int wave, int lane, int c, int hd) {
#pragma unroll
    for (int k = 0; k < Cfg<HDP>::PPW; ++k) {
      const int lin = (wave * Cfg<HDP>::PPW + k) * 1024 + lane * 16;
      const int row = lin / Cfg<HDP>::ROWB;
      const int phys = (lin % Cfg<HDP>::ROWB) >> 4;
      const int ch = phys ^ (xv(row) & Cfg<HDP>::XM);
      voff[k] = ch * 8 < hd ? (unsigned)((row * c + ch * 8) * 2) : AT_OOB;
    }
  }
  // rows row0 .. row0+63 of the slab behind rsrc (rows past its end arrive as zeros)
  __device__ __forceinline__ void issue(const __bf16* base, long long elem_off, int l, int c, int hd, char* tile,
                                        unsigned row0_bytes, int wave) const {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(base + elem_off), 0,
                                                        (unsigned)((((long long)l - 1) * c + hd) * 2), 0x00020000);
#pragma unroll
    for (int k = 0; k < Cfg<HDP>::PPW; ++k)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(tile + (wave * Cfg<HDP>::PPW + k) * 1024), 16,
          voff[k] + row0_bytes, 0, 0, 0);
  }
};

// per-lane LDS byte offsets of the two kinds of reads (see the header comment)
template <int HDP> __device__ __forceinline__ int row_read_base(int lane) {   // + (s << 5) by xor, + 32*t*ROWB
  const int r = lane & 31, h = lane >> 5;
  return r * Cfg<HDP>::ROWB + ((h ^ (xv(r) & Cfg<HDP>::XM)) << 4);
}
template <int HDP> __device__ __forceinline__ int tr_read_base(int lane, int u) {   // ^ (dt << 6), + (32t + 16s)*ROWB
  const int g = lane >> 4, qq = (lane >> 2) & 3, pp = lane & 3;
  const int row = 8 * u + 4 * (g >> 1) + qq;
  const int c_lo = 2 * (g & 1) + (pp >> 1);
  return row * Cfg<HDP>::ROWB + ((c_lo ^ (xv(row) & Cfg<HDP>::XM)) << 4) + 8 * (pp & 1);
}

}  // namespace
