// What the matrix-product kernels share: 16-byte operand fragments of the 32x32 MFMA instructions for the three element
// types, their reads from LDS, and 16-byte copies from global memory straight into LDS.
//
// A fragment is 16 bytes of one row (of A) or column (of B) per lane: lane l holds row l % 32 and, of a run of
// kFragK values of the contraction index, the half l / 32.  For 16-bit types (kFragK = 16) that is one
// v_mfma_f32_32x32x16; for fp32 (kFragK = 8) it is four v_mfma_f32_32x32x2, the j-th of which contracts the indices
// (j, 4 + j) -- any order does, as A and B agree.  The 32x32 result has its column in lane % 32 and in register r the
// row 8 (r / 4) + 4 (lane / 32) + r % 4 (result_row).
#pragma once
#include "elem.h"

namespace ps {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));

template <typename T> struct FragOf;
template <> struct FragOf<bf16> { typedef bf16x8 type; };
template <> struct FragOf<f16> { typedef f16x8 type; };
template <> struct FragOf<float> { typedef floatx4 type; };
template <typename T> using Frag = typename FragOf<T>::type;

template <typename T> constexpr int kVec = 16 / sizeof(T);     // elements of a 16-byte chunk
template <typename T> constexpr int kFragK = 2 * kVec<T>;      // contraction indices a pair of fragments covers

__device__ __forceinline__ int result_row(int r, int hi) { return 8 * (r >> 2) + 4 * hi + (r & 3); }

__device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma(f16x8 a, f16x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma(floatx4 a, floatx4 b, floatx16 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ floatx16 zero16() {
  floatx16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// Copies from global memory into LDS, 16 or 4 bytes a lane, to lds + 16 (4) lane; lds is the wave's own (uniform).
// copy_to_lds is issued past the compiler: it would have every LDS read it cannot tell apart from a copy's target wait for all
// copies in flight, which is the next tile's.  So a wave waits for its own with wait_for_copies, in front of the
// barrier behind which the tile is read.  (The instruction has no result registers, and its address is read at issue.
// M0 is a reserved register that nothing else in a kernel with these copies uses.)  For the tiled product that is 255
// instead of 307 us (16384-long contraction of 4096 x 1024, bf16).  The attention, several blocks a CU and softmax
// between its products, gains nothing from it (2 x 8 heads of 64 x 64 tokens of 64 in bf16: forward 178 against 176 us, dq 257
// against 254, dk and dv 199 against 201) and takes copy_known.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}
__device__ __forceinline__ void copy_to_lds(const void* g, const void* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_address(lds)), "v"(g) : "memory");
}
// the same as the compiler knows them (it waits by itself)
__device__ __forceinline__ void copy_known(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
__device__ __forceinline__ void copy_word_known(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
}
__device__ __forceinline__ void wait_for_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- LDS tiles ------------------------------------------------------------------------------------------------
// Along: [rows][128 bytes of the contraction index].  The 16-byte chunk c of row r lies at c ^ ((r >> 1) & 7), so that
// the 16 rows a quarter of the wave reads at one c cover all banks.
__device__ __forceinline__ int along_offset(int row, int chunk) { return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4); }

template <typename T>
__device__ __forceinline__ Frag<T> along_fragment(const char* tile, int row, int chunk) {
  return *reinterpret_cast<const Frag<T>*>(tile + along_offset(row, chunk));
}

// Across: [contraction index][ROWS elements].  16-bit types: the transposing LDS read hands each lane of 16 the four
// values of one column of a 4 x 16 block; the four contraction rows of a block lie in different 64-byte parts of
// the banks (chunk ^ 4 (k & 3); rows of 64 elements are half the banks long: chunk ^ 4 ((k >> 1) & 1)).  fp32: four
// 4-byte reads; the two halves of the wave read contraction indices 4 apart, which lie in different halves of the banks
// (chunk ^ 8 ((k >> 2) & 1)).
template <typename T, int ROWS>
__device__ __forceinline__ int across_swizzle(int k) {
  return sizeof(T) == 4 ? ((k >> 2) & 1) << 3 : ROWS == 64 ? ((k >> 1) & 1) << 2 : (k & 3) << 2;
}

// rows `row0` .. + 31, contraction indices k0 + half * kVec .. ; k0 is a multiple of 4
template <typename T, int ROWS>
__device__ __forceinline__ Frag<T> across_fragment(const char* tile, int row0, int k0, int k1, int lane) {
  // k0, k1: the first index of the fragment's first and second four (16-bit), or of its only four (fp32: k0)
  if constexpr (sizeof(T) == 2) {
    const int i = lane & 15, col = row0 + (lane & 16) + (i & 3) * 4, kr = i >> 2;
    const int within = ((((col >> 3) ^ across_swizzle<T, ROWS>(kr)) << 4) | ((col & 4) << 1));   // k0, k1: multiples of 4
    typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
    const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(tile + (k0 + kr) * (ROWS * 2) + within));
    const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(tile + (k1 + kr) * (ROWS * 2) + within));
    const shortx8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(Frag<T>, v);
  } else {
    const int col = row0 + (lane & 31);
    const int within = (((col >> 2) ^ across_swizzle<T, ROWS>(k0)) << 4) | ((col & 3) << 2);
    Frag<T> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(tile + (k0 + j) * (ROWS * 4) + within);
    return v;
  }
}

}  // namespace ps
