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
//   operand  a matrix [rows][cols] as the product reads it, whose contraction runs over cols: panels of 128
//            columns, 2 ceil(cols / 256) of them, zeros behind cols, 64 B of a row after the other (what the product
//            takes at a time is then whole lines: 64 B of rows further apart cost its loads 1.7 times the time);
//            behind them scales [ceil(cols / 512)][rows][16], block 4 t + q of a row's 16 at byte 4 q + t. Lane (row, q) of a matrix instruction over columns
//            128 t .. 128 t + 127 then has the scales of its four blocks of 512 columns in one word.
#pragma once
#include "dpa_common.hpp"

namespace dpa {
namespace mx {

constexpr int kBlock = 32;
constexpr int kStep = 256;   // columns of an operand's padding and of a step of the product
constexpr int kGroup = 512;  // columns of a group of scales

__host__ __device__ inline int64_t pitch_of(int64_t cols) { return (cols + kStep - 1) / kStep * (kStep / 2); }
__host__ __device__ inline int64_t groups_of(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

// (Rows come to the product 16 at a time, scales of up to 256: the buffer holds as many behind the last,
// which hold anything.)
__host__ __device__ inline int64_t padded_rows(int64_t rows) { return (rows + 15) & ~15ll; }
__host__ __device__ inline int64_t panel_of(int64_t rows) { return padded_rows(rows) * 64; }
inline int64_t operand_data_bytes(int64_t rows, int64_t cols) { return padded_rows(rows) * pitch_of(cols); }
inline int64_t operand_bytes(int64_t rows, int64_t cols) {
  return operand_data_bytes(rows, cols) + (groups_of(cols) * rows + 256) * 16;
}

// Sizes of a matrix that the kernels take: 32-bit numbers of 8-element groups and workgroups, and of scales
inline bool matrix_ok(int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0 || rows >= (1 << 26) || cols >= (1 << 26)) return false;
  return padded_rows(rows) * (groups_of(cols) * 64) < (1ll << 31) && padded_rows(cols) * (groups_of(rows) * 64) < (1ll << 31);
}

// place of block b of a row within the 16 B of its group
__host__ __device__ inline int scale_at(int b) { return 4 * (b & 3) + (b >> 2); }

// scale byte from the largest magnitude's bits
template <bool SR>
__device__ __forceinline__ uint32_t scale_byte(uint32_t m) {
  const int e = (int)(m >> 23);
  int k = e - 2;
  if (SR && (m & 0x7fffffu) > 0x400000u && e >= 2) ++k;
  return e == 255 ? 255u : (uint32_t)(k < 0 ? 0 : k);
}

// The conversions v_cvt_scalef32_* take a scale by its exponent bits: every byte below 255 stands as
// byte << 23, 0 for 2^-127 too, which the tests check over all bytes. A block of byte 255 gets codes of no
// meaning.
__device__ __forceinline__ float scale_bits(uint32_t byte) { return __uint_as_float(byte << 23); }
// for the way back: NaN for 255
__device__ __forceinline__ float scale_back(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23); }

typedef __bf16 pk_bf16 __attribute__((ext_vector_type(2)));

// Byte I of r: the codes of two numbers over the scale, to nearest even, beyond 6 to 6. w: a pair of a
// 16-bit type.
template <int DT, int I>
__device__ __forceinline__ uint32_t encode_pair(uint32_t r, uint32_t w, float scale) {
  if constexpr (DT == DPA_DTYPE_BF16)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(pk_bf16, w), scale, I);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w), scale, I);
}
template <int I>
__device__ __forceinline__ uint32_t encode_pair(uint32_t r, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, a, b, scale, I);
}

// The lowest 4 bits: the code of v over the scale, magnitude rounded up where its place between two codes, in
// units of 2^-16 and rounded down, plus the 16 random bits reaches 2^16 (bits: those 16 in the upper half,
// zeros below: the instruction adds them to what it cuts off). What lies above the 4 bits is of no meaning: the
// instruction's second number, which would share the bits, and three bytes that it leaves.
__device__ __forceinline__ uint32_t encode_sr(float v, uint32_t bits, float scale) {
  return __builtin_amdgcn_cvt_scalef32_sr_pk_fp4_f32(0u, v2f{v, __builtin_nondeterministic_value(v)}, bits, scale, 0);
}
// a byte of two codes, the lower bits first
__device__ __forceinline__ uint32_t two_codes(uint32_t a, uint32_t b) { return (a & 0xfu) | (b << 4); }
// the lowest bytes of a, b, c and d
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b) { return perm_b32(b, a, 0x0c0c0400u); }
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return perm_b32(perm_b32(d, c, 0x0c0c0400u), perm_b32(b, a, 0x0c0c0400u), 0x05040100u);
}

// The random bits of elements 4 i .. 4 i + 3: splitmix64(seed + i * golden ratio), 16 bits each. Elements are
// numbered in rows of whole blocks: row * (cols rounded up to 32) + col.
__device__ __forceinline__ uint64_t mix(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
__device__ __forceinline__ uint64_t bits_of(uint64_t seed, uint64_t i) { return mix(seed + i * kDropGolden); }

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
