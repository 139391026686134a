// Warp-level tensor-core helpers shared by the decode kernels (sm_100a): ldmatrix, the
// m16n8k16 f16 MMA with f32 accumulation, movmatrix, f16 packing, the exact int8 -> f16 code
// conversion and the 128-byte swizzle address of a TMA-written tile.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace bg {

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}

constexpr uint32_t kSelLo = 0x4140, kSelHi = 0x4342, kSelEven = 0x4240, kSelOdd = 0x4341;

// Biased form without the subtraction: (code + 1152) as exact f16x2, from a word already xored
// with 0x80808080.  The kernels remove the +1152 inside the MMA instead (accumulator seed for K,
// an extra MMA with a constant -1152 operand for V).
__device__ __forceinline__ uint32_t i8pair_biased(uint32_t wx, uint32_t sel) {
  return __byte_perm(wx, 0x64646464u, sel);
}
__device__ __forceinline__ uint32_t kNeg1152x2() {
  __half2 h = __half2(__float2half_rn(-1152.f), __float2half_rn(-1152.f));
  return *reinterpret_cast<uint32_t *>(&h);
}

// Weights p * block scale as one f16, whatever the scales' magnitude: a warp keeps each 32-channel block's output
// divided by a power of two, so that scales (p is at most 1) times inv[block] stay below 2^15 / 127.  above() says
// whether a tile's would not (one vote for all blocks, each lane looks at its two rows' blocks of its place in the
// quad); admit() then lets `down` scale the block's output so far to the next power.  ya, yb: a lane's rows of scales.
template <int NB>
struct BlockPow {
  float inv[NB];       // the inverse power over 127
  float lim[NB / 4];   // scales that are too large, of blocks lane % 4, + 4
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int b = 0; b < NB; ++b) inv[b] = 0x1p126f * (1.0f / 127.0f);
#pragma unroll
    for (int q = 0; q < NB / 4; ++q) lim[q] = 0x1p-111f;
  }
  // The power's inverse itself (inv is 2^(k - 7) times 1.00..).
  __device__ __forceinline__ float exact(int b) const {
    return __uint_as_float((__float_as_uint(inv[b]) & 0x7f800000u) + (7u << 23));
  }
  __device__ __forceinline__ bool above(const float *ya, const float *yb, uint32_t lane) const {
    bool is = false;
#pragma unroll
    for (int q = 0; q < NB / 4; ++q) {
      const int b = 4 * q + (lane & 3);
      is |= fmaxf(fabsf(ya[b]), fabsf(yb[b])) >= lim[q];
    }
    return is;
  }
  template <typename F>
  __device__ __forceinline__ void admit(const float *ya, const float *yb, uint32_t lane, F down) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(ya[b]), fabsf(yb[b]))));
      const float was = exact(b);
      if (__uint_as_float(bits) * was < 32768.f) continue;
      const float now = pow2_inv(pow2_of(bits));
      down(b, now * pow2_inv(was));
      inv[b] = now * (1.0f / 127.0f);
      lim[b / 4] = (lane & 3) == (b & 3) ? 32768.f * pow2_inv(now) : lim[b / 4];
    }
    __syncwarp();
  }
  __device__ __forceinline__ float back(int b) const { return pow2_inv(exact(b)); }
};

// Shared-memory byte address of 16-byte chunk `gc` of tile row `row` (128B-swizzled column blocks
// of TP rows each, the layout TMA writes with CU_TENSOR_MAP_SWIZZLE_128B).
template <int TP>
__device__ __forceinline__ uint32_t swz(uint32_t base, int row, int gc) {
  return base + (gc >> 3) * (TP * 128) + row * 128 + (((gc & 7) ^ (row & 7)) << 4);
}

}  // namespace bg
