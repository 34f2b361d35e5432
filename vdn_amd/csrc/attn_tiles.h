// K/V tiles in LDS and 16-bit MFMA element types, shared by the attention kernels.
#pragma once

#include "common.h"

namespace vdn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef __attribute__((address_space(3))) void lds_void_t;
typedef const __attribute__((address_space(1))) void global_void_t;
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;

// Tile rows go global -> LDS through a buffer resource (buffer_load_dwordx4 ... lds): lane l's
// 16 bytes at voffset + soffset land at lds_wave_base + 16 l. Unlike the flat/global form,
// the compiler counts these on vmcnt only, so the fragment reads of the current tile keep
// exact lgkmcnt waits instead of waiting for every outstanding LDS read before each MFMA.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
}

__device__ __forceinline__ void load_to_lds16(__amdgpu_buffer_rsrc_t r, uint32_t voffset,
                                              uint32_t soffset, void* lds_wave_base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)lds_wave_base, 16, voffset, soffset, 0, 0);
}

__device__ __forceinline__ bf16x4_t lds_read_tr(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      (lds_bf16x4_t*)((__attribute__((address_space(3))) char*)(p)));
}

// the transpose read's own fp16 vector type (four __fp16), reinterpreted as f16x4
typedef __fp16 fp16x4_raw __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) fp16x4_raw lds_f16x4_t;

// The 16-bit element type of a kernel instance: bf16 (the block's) or fp16 (the reference's
// other varlen dtype). Both share the storage layout, the LDS swizzles and the transpose
// reads; they differ in the MFMA, the conversions of P and the output's rounding.
template <bool kF16>
struct Elem;

template <>
struct Elem<false> {
  typedef __bf16 type;
  typedef bf16x8 x8;
  typedef bf16x4_t x4;
  static __device__ __forceinline__ x4 read_tr(const uint16_t* p) { return lds_read_tr(p); }
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint16_t h) { return bf16_bits_to_f32(h); }
  static __device__ __forceinline__ float round(float f) { return round_bf16(f); }
  static __device__ __forceinline__ uint16_t bits(float f) { return f32_to_bf16_bits(f); }
};

template <>
struct Elem<true> {
  typedef _Float16 type;
  typedef f16x8 x8;
  typedef f16x4 x4;
  static __device__ __forceinline__ x4 read_tr(const uint16_t* p) {
    return __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
        (lds_f16x4_t*)((__attribute__((address_space(3))) char*)(p))));
  }
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint16_t h) { return f16_bits_to_f32(h); }
  static __device__ __forceinline__ float round(float f) { return round_f16(f); }
  static __device__ __forceinline__ uint16_t bits(float f) { return f32_to_f16_bits(f); }
};

// 16-byte chunk c of tile row r is stored at c ^ swz(r). K rows are read 16 rows per LDS cycle
// (one chunk each), V rows by the transpose reads 4 rows x 4 chunks per 32 lanes; a 256-byte
// bank window holds 256 / (2 D) rows, and the XOR spreads each read set over all of its 16
// chunk positions (D = 64: two rows per window).
template <int D>
__device__ __forceinline__ int swz_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
template <int D>
__device__ __forceinline__ int swz_v(int row) { return D == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); }

}  // namespace vdn
