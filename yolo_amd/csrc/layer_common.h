// Helpers shared by the attention-side layer kernels (linear.hip, qk_norm_rope.hip, cross_attention.hip): the two element types
// of the library as 16-byte pieces, and conversions.  Storage type T is float or bf16_t (raw bits); arithmetic is float.
#pragma once
#include "common.h"

namespace yolo {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A 16-byte piece of a row: 8 bf16 or 4 float.
template <bool BF16> struct Elem;
template <> struct Elem<true> { typedef __bf16 type; static constexpr int kPiece = 8; };
template <> struct Elem<false> { typedef float type; static constexpr int kPiece = 4; };

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __builtin_bit_cast(float, u & 0xffff0000u); }
// two floats -> two bf16 in one register, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    bf16x2 v;
    v[0] = (__bf16)a;
    v[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __bf16* p) { return (float)*p; }
// a parameter vector (bias, norm weight) is float or bf16 whatever the activations are
__device__ __forceinline__ float load_param(const void* p, int bf16, long long i) {
    return bf16 ? (float)((const __bf16*)p)[i] : ((const float*)p)[i];
}

// Consecutive workgroup ids go to the 8 XCDs in turn, and each XCD has an L2 of its own: give every XCD one contiguous run
// of the `total` tiles, so that neighbours, which read the same operand rows, share an L2.  A bijection for any total.
__device__ __forceinline__ unsigned xcd_chunk(unsigned id, unsigned total) {
    const unsigned q = total >> 3, r = total & 7, x = id & 7, l = id >> 3;
    return x * q + (x < r ? x : r) + l;
}

// LDS-DMA: 16 bytes per lane from global memory straight to LDS (lane i lands at base + 16 i); wait with s_waitcnt vmcnt.
__device__ __forceinline__ void dma16(const void* g, void* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// The runtime counts the threads of a launch in 32 bits.
static inline bool launchable(unsigned long long blocks, unsigned threads) { return blocks <= 0xffffffffull / threads; }

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace yolo
