// MXFP4: blocks of 32 elements in e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, 4 bits) with one power
// of two each, kept as its exponent + 127 in a byte (255: the block has no value, all NaN).
//
// Scale of a block whose largest magnitude is amax (fp32 bits m, biased exponent E = m >> 23):
//   nearest:    2^k, k = floor(log2 amax) - 2 and at least -127, so that amax 2^-k lies in [4, 8); what passes 6
//               is held as 6. The byte is max(E - 2, 0).
//   stochastic: one power more where amax 2^-k would pass 6, so that nothing is cut off and the mean of
//               a rounded element is the element.
// A block with an infinity or a NaN gets 255.
//
// Two arrangements:
//   dense    a tensor [..., C], C a multiple of 32: its bytes in order, the first of two elements in the low
//            half, and its scale bytes in order.
//   operand  a matrix [rows][cols] as the product reads it, whose contraction runs over cols: rows of
//            ceil(cols / 256) * 128 B, zeros behind cols; scales [ceil(cols / 512)][rows][16], block
//            8 s + 2 q + t of a row's 16 at byte 4 q + 2 s + t. Lane (row, q) of a matrix instruction then
//            has the scales of its four 32-element pieces of 512 columns in one word, and takes pieces
//            2 q, 2 q + 1 of each 256 (the order of a contraction is free as long as both operands keep it).
#pragma once
#include "dpa_common.hpp"

namespace dpa {
namespace mx {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;
constexpr int kStep = 256;   // columns of an operand's padding and of a step of the product
constexpr int kGroup = 512;  // columns of a group of scales

__host__ __device__ inline int64_t pitch_of(int64_t cols) { return (cols + kStep - 1) / kStep * (kStep / 2); }
__host__ __device__ inline int64_t groups_of(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

// place of block b of a row within the 16 B of its group
__host__ __device__ inline int scale_at(int b) { return 4 * ((b >> 1) & 3) + 2 * ((b >> 3) & 1) + (b & 1); }

// scale byte from the largest magnitude's bits
template <bool SR>
__device__ __forceinline__ uint32_t scale_byte(uint32_t m) {
  const int e = (int)(m >> 23);
  int k = e - 2;
  if (SR && (m & 0x7fffffu) > 0x400000u) ++k;
  if (e < 2) k = 0;
  return e == 255 ? 255u : (uint32_t)(k < 0 ? 0 : k);
}
// 2^-(byte - 127): a normal number for every byte of a finite block (at most 253)
__device__ __forceinline__ float inverse_of(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }
// 2^(byte - 127); NaN for 255
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// Eight numbers, scaled already, to eight codes: to nearest even, beyond 6 to 6 (v_cvt_scalef32_pk_fp4_f32
// at scale 1).
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
  return r;
}
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, a, b, 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, c, d, 1.0f, 1);
  return r;
}

// One number of magnitude up to 6 to its code, up where its place between two codes, in units of 2^-16 and
// rounded down, plus the 16 random bits reaches 2^16. From 1 on the place is the 22 bits behind a code's
// mantissa bit, below it the fraction of v / 0.5.
__device__ __forceinline__ uint32_t encode_sr(float v, uint32_t bits16) {
  const uint32_t u = __float_as_uint(v), a = u & 0x7fffffffu;
  const uint32_t big = ((a + (bits16 << 6)) >> 22) - 252u;
  const uint32_t small = ((uint32_t)(__uint_as_float(a) * 131072.0f) + bits16) >> 16;
  return (a >= 0x3f800000u ? big : small) | ((u >> 28) & 8u);
}

// The random bits of elements 4 i .. 4 i + 3: splitmix64(seed + i * golden ratio), 16 bits each. Elements are
// numbered in rows of whole blocks: row * (cols rounded up to 32) + col.
__device__ __forceinline__ uint64_t bits_of(uint64_t seed, uint64_t i) {
  uint64_t z = seed + i * kDropGolden;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

// D(16 x 16) += A(16 x 128) B(128 x 16) over blocks of 32: lane l supplies 32 elements of row (column of B)
// l & 15 with byte SA (SB) of its scale word, and receives D[4 (l >> 4) + t][l & 15], t = 0 .. 3.
template <int SA, int SB>
__device__ __forceinline__ v4f mfma(u32x4 a, u32x4 b, v4f c, uint32_t sa, uint32_t sb) {
  const v8i x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const v8i y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, SA, (int)sa, SB, (int)sb);
}

// elements as fp32
template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == DPA_DTYPE_F32) return static_cast<const float*>(p)[i];
  if constexpr (DT == DPA_DTYPE_BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
  if constexpr (DT == DPA_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
}
template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (DT == DPA_DTYPE_F32) static_cast<float*>(p)[i] = v;
  if constexpr (DT == DPA_DTYPE_BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)pack_bf16x2(v, v);
  if constexpr (DT == DPA_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
}

inline bool dtype_ok(int dt) { return dt == DPA_DTYPE_BF16 || dt == DPA_DTYPE_F16 || dt == DPA_DTYPE_F32; }
inline int size_of(int dt) { return dt == DPA_DTYPE_F32 ? 4 : 2; }

}  // namespace mx
}  // namespace dpa
