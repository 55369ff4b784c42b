// Building blocks of the 16-bit attention kernels on 16x16x32 MFMA: element
// types, LDS read offsets of a key block, S^T = K . Q^T and O += P . V.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "attention_split.hpp"

namespace cbk {
namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <bool F16> struct Ops;
template <> struct Ops<false> {  // bf16
  typedef s16x8 A8;
  typedef s16x4 A4;
  static __device__ __forceinline__ f32x4 mma32(const A8& a, const A8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // two floats -> two bf16 (round to nearest even) packed low/high
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, b2));
  }
  static __device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
};
template <> struct Ops<true> {  // f16
  typedef h16x8 A8;
  typedef h16x4 A4;
  static __device__ __forceinline__ f32x4 mma32(const A8& a, const A8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return __builtin_bit_cast(uint32_t, h);
  }
  static __device__ __forceinline__ float lo(uint32_t u) {
    return __half2float(__builtin_bit_cast(__half, uint16_t(u & 0xffffu)));
  }
  static __device__ __forceinline__ float hi(uint32_t u) {
    return __half2float(__builtin_bit_cast(__half, uint16_t(u >> 16)));
  }
};

// bf16 / f16 1.0 in both halves of a word: the B operand of the "ones"
// column whose MFMA accumulates each row's sum of (rounded) probabilities
template <bool F16> constexpr uint32_t kOnesPair = F16 ? 0x3c003c00u : 0x3f803f80u;

// A lane's LDS read offsets within a K or V block, bytes, the same in every
// buffer: the K fragment of dim step st and the V transposing read of column
// tile c, both for the first 16-key half (the second half is 16 rows
// further: the swizzle of row 16 + r equals that of row r).
template <int D>
struct BlockOffsets {
  uint32_t k[D / 32];
  uint32_t v[D / 16];
  __device__ __forceinline__ explicit BlockOffsets(uint32_t lane) {
    const uint32_t row = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int st = 0; st < D / 32; ++st) k[st] = (row * D + ((4 * st + grp) ^ lds_swizzle<D>(row)) * 8) * 2;
    // lane (row, grp) addresses key 4 grp + row / 4, dims 16c + 4 (row % 4) .. + 3
    // of the row-major V block
    const uint32_t vkey = 4 * grp + (row >> 2);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const uint32_t dim = 16 * c + 4 * (row & 3);
      v[c] = (vkey * D + ((dim / 8) ^ lds_swizzle<D>(vkey)) * 8 + (dim & 4)) * 2;
    }
  }
};

// S^T = K . Q^T of one block (K buffer ks) for every row tile; each K
// fragment is read from LDS once.
template <bool F16, int D, int RT>
__device__ __forceinline__ void qk_block(const uint16_t* ks, const BlockOffsets<D>& off,
                                         const typename Ops<F16>::A8 (&qf)[RT][D / 32], f32x4 (&s)[RT][2]) {
  using O = Ops<F16>;
  constexpr uint32_t kHalf = 16 * D * 2;  // bytes from a 16-key half to the next
#pragma unroll
  for (int t = 0; t < RT; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int st = 0; st < D / 32; ++st) {
    const char* kp = reinterpret_cast<const char*>(ks) + off.k[st];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const typename O::A8 kf = *reinterpret_cast<const typename O::A8*>(kp + h * kHalf);
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t][h] = O::mma32(kf, qf[t][st], s[t][h]);
    }
  }
}

// O += P . V and the row sums l += P . 1, one 16x16x32 MFMA per 16-dim column
// tile for the block's 32 keys (two 16x16x16 MFMAs cost as much each). The
// contraction runs in this lane layout's key order: k-slot 8 grp + e holds
// key 4 grp + e for e < 4 and 16 + 4 grp + e - 4 after, in P (the S^T
// registers of the two 16-key halves, concatenated) and in V (two
// transposing reads, one per half, concatenated).
template <bool F16, int D, int RT>
__device__ __forceinline__ void pv_block(const uint16_t* vs, const BlockOffsets<D>& off,
                                         const typename Ops<F16>::A8 (&pa)[RT], f32x4 (&o)[RT][D / 16],
                                         f32x4 (&ol)[RT]) {
  using O = Ops<F16>;
  constexpr uint32_t kHalf = 16 * D * 2;
  typedef short s16x4v __attribute__((ext_vector_type(4)));
  const typename O::A8 ones = __builtin_bit_cast(
      typename O::A8, u32x4{kOnesPair<F16>, kOnesPair<F16>, kOnesPair<F16>, kOnesPair<F16>});
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    // lane (row, grp) addresses key 16h + 4 grp + row / 4, dims 16c + 4 (row % 4) .. + 3 of
    // the row-major V block; ds_read_tr16_b64 hands lane j of each 16-lane group element i of
    // its group's lane 4i + j / 4, i.e. V[16h + 4 grp + i][16c + j]
    const char* vp = reinterpret_cast<const char*>(vs) + off.v[c];
    s16x4v w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4v*)((__attribute__((address_space(3))) const void*)(vp + h * kHalf)));
    const typename O::A8 vb =
        __builtin_bit_cast(typename O::A8, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
    for (int t = 0; t < RT; ++t) o[t][c] = O::mma32(pa[t], vb, o[t][c]);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) ol[t] = O::mma32(pa[t], ones, ol[t]);
}

}  // namespace
}  // namespace cbk
