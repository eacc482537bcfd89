// Pieces that the attention kernels share: MFMA and packing by element type,
// global -> LDS copies, operand reads from swizzled LDS tiles.
#pragma once
#include "common.h"

namespace fs {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

template <typename T> struct MfmaOps;
template <> struct MfmaOps<bf16_t> {
  using V8 = bf16x8_t;
  static __device__ __forceinline__ f32x16_t mma(V8 a, V8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ V8 pack(const float* x) {
    V8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)x[i];
    return r;
  }
  static __device__ __forceinline__ uint16_t bits(float x) {
    __bf16 b = (__bf16)x;
    return __builtin_bit_cast(uint16_t, b);
  }
  // acc + sum of the 8 elements (v_dot2_f32_bf16 against ones)
  static __device__ __forceinline__ float sum8(V8 p, float acc) {
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
    const x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_fdot2_f32_bf16(x2{p[2 * i], p[2 * i + 1]}, one, acc, false);
    return acc;
  }
};
template <> struct MfmaOps<f16_t> {
  using V8 = f16x8_t;
  static __device__ __forceinline__ f32x16_t mma(V8 a, V8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ V8 pack(const float* x) {
    V8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)x[i];
    return r;
  }
  static __device__ __forceinline__ uint16_t bits(float x) {
    _Float16 b = (_Float16)x;
    return __builtin_bit_cast(uint16_t, b);
  }
  static __device__ __forceinline__ float sum8(V8 p, float acc) {
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
    const x2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_fdot2(x2{p[2 * i], p[2 * i + 1]}, one, acc, false);
    return acc;
  }
};

// the 8 elements of two transposing LDS reads (V read as it is stored)
__device__ __forceinline__ uint4 join8(i16x4_t a, i16x4_t b) {
  return __builtin_bit_cast(uint4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// the longest head dim of the tiles
constexpr int kD = 128;

// One 1 KiB global -> LDS copy per wave: lane l's 16 bytes land at lds_base + 16 l.
__device__ __forceinline__ void dma16(uint32_t lds_base, const void* gptr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds_base), "v"(gptr) : "memory");
}
// Same, addressed as a wave-uniform base (scalar registers) plus a 32-bit lane offset.
__device__ __forceinline__ void dma16s(uint32_t lds_base, const void* sbase, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(lds_base), "v"(voff), "s"(sbase) : "memory");
}

// a row of zeros to copy for keys past the sequence
static __device__ const uint4 kZeroRow[kD * 2 / 16] = {};

// 4 16-bit elements per lane of a transposing LDS read (V read as it is stored)
__device__ __forceinline__ i16x4_t lds_tr8(const char* base, uint32_t off) {
  typedef __attribute__((address_space(3))) i16x4_t* lptr;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(base + off));
}
// 16-byte chunk c of key row r of a V tile read that way is stored at chunk c ^ v_swz(r)
template <int D>
__device__ __forceinline__ int v_swz(int r) {
  return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}
// 16-byte LDS operand at byte offset off of base
__device__ __forceinline__ uint4 lds16(const char* base, uint32_t off) {
  return *reinterpret_cast<const uint4*>(base + off);
}

}  // namespace fs
