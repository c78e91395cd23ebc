// Tensors to MXFP4 and back (format: mxfp4.hpp). All of it is bound by the bytes it moves.
#include "mxfp4.hpp"

namespace dpa {
namespace mx {

// ---------------------------------------------------------------------------------------
// Blocks along the rows: four lanes to a block, 8 elements a lane (16 B of a 16-bit type), the largest
// magnitude exchanged within the quad. Dense tensors are one long row; of an operand a wave takes 512 columns of a
// row, and what lies behind cols comes as zeros. 64 Mi elements of fp32 (302 MB moved) 59 us, 5.1 TB/s, which is
// a copy's rate here; an operand of 8192 x 4096 of bf16 (85 MB) 15 us, partly out of the caches.
// ---------------------------------------------------------------------------------------
struct RowArgs {
  const void* x;
  uint8_t *data, *scales;
  const uint64_t* seed;  // null: to nearest
  int64_t groups;      // of 8 elements, of a dense tensor
  int64_t rows, cols, ld;
  FastDiv per_rows;    // workgroups (of 512 columns) to four rows
};

// Eight neighbours of a row as they lie in memory
template <int DT>
struct Eight {
  uint4 w;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
    return i & 1 ? Elem<DT>::hi(u) : Elem<DT>::lo(u);
  }
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
  }
  __device__ __forceinline__ void load_some(const void* p, int64_t at, int64_t left) {
    const uint16_t* s = static_cast<const uint16_t*>(p) + at;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = i < left ? s[i] : 0u;
    w = uint4{u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16};
  }
  // bits of the largest magnitude, as fp32's
  __device__ __forceinline__ uint32_t amax() const {
    const us2 a = absmax8(us2{0, 0}, w);
    const uint32_t m = a.x > a.y ? a.x : a.y;
    return DT == DPA_DTYPE_BF16 ? m << 16 : __float_as_uint(Elem<DT>::lo(m));
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t r = encode_pair<DT, 0>(0u, w.x, scale);
    r = encode_pair<DT, 1>(r, w.y, scale);
    r = encode_pair<DT, 2>(r, w.z, scale);
    return encode_pair<DT, 3>(r, w.w, scale);
  }
};
template <>
struct Eight<DPA_DTYPE_F32> {
  float v[8];
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void load_some(const void* p, int64_t at, int64_t left) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? static_cast<const float*>(p)[at + i] : 0.f;
  }
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t r = encode_pair<0>(0u, v[0], v[1], scale);
    r = encode_pair<1>(r, v[2], v[3], scale);
    r = encode_pair<2>(r, v[4], v[5], scale);
    return encode_pair<3>(r, v[6], v[7], scale);
  }
};

__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, false));  // lane ^ 1
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, false));  // lane ^ 2
}

// The random bits of four elements as the conversion takes them
__device__ __forceinline__ void bits4(uint32_t (&b)[4], uint64_t z) {
  const uint32_t lo = (uint32_t)z, hi = (uint32_t)(z >> 32);
  b[0] = lo << 16, b[1] = lo & 0xffff0000u, b[2] = hi << 16, b[3] = hi & 0xffff0000u;
}

// kOperand: an operand's rows, else dense. kWide: rows of whole aligned 8-element groups.
template <int DT, bool kOperand, bool kWide, bool SR>
__global__ __launch_bounds__(256) void mxfp4_rows_kernel(const RowArgs p) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row = 0, in_row = g;
  if constexpr (kOperand) {  // a wave takes 512 columns, a workgroup four rows of them: whole lines of the panels
    const uint32_t four = fdiv(blockIdx.x, p.per_rows);
    row = 4 * (int64_t)four + (threadIdx.x >> 6);
    in_row = (int64_t)(blockIdx.x - four * p.per_rows.d) * 64 + (threadIdx.x & 63);
    if (row >= p.rows || in_row * 4 >= pitch_of(p.cols)) return;
  } else if (g >= p.groups) {
    return;  // (whole blocks: a quad ends together)
  }
  const int64_t c0 = in_row * 8, at = row * p.ld + c0;
  Eight<DT> v;
  if (!kOperand || (kWide && c0 + 8 <= p.cols))
    v.load(p.x, at);
  else
    v.load_some(p.x, at, p.cols - c0);
  const uint32_t byte = scale_byte<SR>(quad_max(v.amax()));
  const float scale = scale_bits(byte);
  uint32_t r;
  if constexpr (SR) {
    const uint64_t i4 = (uint64_t)row * (uint64_t)((p.cols + kBlock - 1) / kBlock * (kBlock / 4)) + (uint64_t)in_row * 2;
    uint32_t a[4], b[4];
    bits4(a, bits_of(*p.seed, i4));
    bits4(b, bits_of(*p.seed, i4 + 1));
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = two_codes(encode_sr(v.get(2 * i), a[2 * i], scale), encode_sr(v.get(2 * i + 1), a[2 * i + 1], scale));
      c[2 + i] = two_codes(encode_sr(v.get(4 + 2 * i), b[2 * i], scale), encode_sr(v.get(5 + 2 * i), b[2 * i + 1], scale));
    }
    r = low_bytes(c[0], c[1], c[2], c[3]);
  } else {
    r = v.codes(scale);
  }
  if constexpr (kOperand)
    *reinterpret_cast<uint32_t*>(p.data + (in_row >> 4) * panel_of(p.rows) + row * 64 + (in_row & 15) * 4) = r;
  else
    reinterpret_cast<uint32_t*>(p.data)[g] = r;
  if ((threadIdx.x & 3) == 0) {
    if constexpr (kOperand) {
      const int b = (int)(in_row >> 2);
      p.scales[((int64_t)(b >> 4) * p.rows + row) * 16 + scale_at(b & 15)] = (uint8_t)byte;
    } else {
      p.scales[g >> 2] = (uint8_t)byte;
    }
  }
}

// ---------------------------------------------------------------------------------------
// Both operands of a matrix from one read of it: its rows, and its columns (blocks down the columns, the
// matrix transposed). Eight waves take 64 rows of 256 columns; a thread holds 4 columns of 8 rows: a row's block is
// the 8 lanes beside each other, a column's the 4 waves below each other, which trade their largest magnitudes
// through LDS. The columns' codes turn in LDS and leave as 32 B of a column; the tiles below each other, which fill
// a line of 128 B, go to one XCD, whose L2 joins them. (Two or four tiles to a workgroup, the next one's loads ahead, is slower,
// from cold caches: 8192 x 4096 of bf16 37.7 and 36.2 us against 34.2, 768 x 256 of fp32 10.8 and 16.8 against 7.6.)
// Within a step 8192 x 4096 of bf16 takes 28 us, stochastically 36, 104 MB at 3.7 and 2.9 TB/s: between the bytes and
// the conversions (vector instructions hold a SIMD for 10 and 24 us of these, by the counters), a workgroup's loads,
// conversions and stores following each other; three workgroups to a CU overlap
// theirs (two, when the sums below cost registers in every variant: 27.2 us for 32768 x 768, with three 25.3).
// ---------------------------------------------------------------------------------------
struct BothArgs {
  const void* x;
  uint8_t *row_data, *row_scales, *col_data, *col_scales;
  const uint64_t* seed;
  int64_t rows, cols, ld;
  int col_tiles;
  uint32_t lines;  // of 256 rows x 256 columns
  float* sums;     // [ceil(rows / 64)][cols] down the columns, or null
};

// Four neighbours of a row
template <int DT>
struct Quad {
  uint2 w;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? w.x : w.y;
    return i & 1 ? Elem<DT>::hi(u) : Elem<DT>::lo(u);
  }
};
template <>
struct Quad<DPA_DTYPE_F32> {
  float4 w;
  __device__ __forceinline__ float get(int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
};

// Columns c0 .. c0 + 3 of a row, zeros outside of the matrix: from inside it all the same, so that loads go out
// together, without branches.
template <int DT, bool kWide>
__device__ __forceinline__ Quad<DT> quad_at(const BothArgs& p, int64_t row, int64_t c0) {
  Quad<DT> q;
  const int64_t at = min(row, p.rows - 1) * p.ld;
  const bool in = row < p.rows;
  if constexpr (kWide) {  // (cols is a multiple of 4)
    const bool on = in && c0 < p.cols;
    q.w = *reinterpret_cast<const decltype(q.w)*>(static_cast<const uint8_t*>(p.x) + (at + (c0 < p.cols ? c0 : 0)) * Elem<DT>::size);
    if (!on) q.w = decltype(q.w){};
    return q;
  }
  if constexpr (DT == DPA_DTYPE_F32) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = static_cast<const float*>(p.x)[at + min(c0 + i, p.cols - 1)];
      if (!in || c0 + i >= p.cols) v[i] = 0.f;
    }
    q.w = float4{v[0], v[1], v[2], v[3]};
  } else {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = static_cast<const uint16_t*>(p.x)[at + min(c0 + i, p.cols - 1)];
      if (!in || c0 + i >= p.cols) v[i] = 0u;
    }
    q.w = uint2{v[0] | v[1] << 16, v[2] | v[3] << 16};
  }
  return q;
}

// Magnitudes of four columns: a word each in fp32, a half each (two columns to a word) of 16-bit types
template <int DT>
struct ColMax {
  us2 a = {0, 0}, b = {0, 0};
  __device__ __forceinline__ void take(const Quad<DT>& q) {
    a = __builtin_elementwise_max(a, __builtin_bit_cast(us2, q.w.x & 0x7fff7fffu));
    b = __builtin_elementwise_max(b, __builtin_bit_cast(us2, q.w.y & 0x7fff7fffu));
  }
  static constexpr int kWords = 2;
  __device__ __forceinline__ void put(uint32_t* lds) const {
    *reinterpret_cast<uint2*>(lds) = uint2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
  }
  __device__ __forceinline__ void join(const uint32_t* lds) {
    const uint2 v = *reinterpret_cast<const uint2*>(lds);
    a = __builtin_elementwise_max(a, __builtin_bit_cast(us2, v.x));
    b = __builtin_elementwise_max(b, __builtin_bit_cast(us2, v.y));
  }
  __device__ __forceinline__ uint32_t get(int j) const {
    const uint32_t m = j == 0 ? a.x : j == 1 ? a.y : j == 2 ? b.x : b.y;
    return DT == DPA_DTYPE_BF16 ? m << 16 : __float_as_uint(Elem<DT>::lo(m));
  }
};
template <>
struct ColMax<DPA_DTYPE_F32> {
  uint32_t m[4] = {0, 0, 0, 0};
  __device__ __forceinline__ void take(const Quad<DPA_DTYPE_F32>& q) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = max(m[j], __float_as_uint(q.get(j)) & 0x7fffffffu);
  }
  static constexpr int kWords = 4;
  __device__ __forceinline__ void put(uint32_t* lds) const {
    *reinterpret_cast<uint4*>(lds) = uint4{m[0], m[1], m[2], m[3]};
  }
  __device__ __forceinline__ void join(const uint32_t* lds) {
    const uint4 v = *reinterpret_cast<const uint4*>(lds);
    m[0] = max(m[0], v.x), m[1] = max(m[1], v.y), m[2] = max(m[2], v.z), m[3] = max(m[3], v.w);
  }
  __device__ __forceinline__ uint32_t get(int j) const { return m[j]; }
};

// largest magnitude of a row's four, as fp32's bits
template <int DT>
__device__ __forceinline__ uint32_t row_max(const Quad<DT>& q) {
  if constexpr (DT == DPA_DTYPE_F32) {
    return max(max(__float_as_uint(q.w.x) & 0x7fffffffu, __float_as_uint(q.w.y) & 0x7fffffffu),
               max(__float_as_uint(q.w.z) & 0x7fffffffu, __float_as_uint(q.w.w) & 0x7fffffffu));
  } else {
    const us2 a = __builtin_elementwise_max(__builtin_bit_cast(us2, q.w.x & 0x7fff7fffu),
                                            __builtin_bit_cast(us2, q.w.y & 0x7fff7fffu));
    const uint32_t m = a.x > a.y ? a.x : a.y;
    return DT == DPA_DTYPE_BF16 ? m << 16 : __float_as_uint(Elem<DT>::lo(m));
  }
}

// Rows i and i + 1 of column j as a pair
template <int DT>
__device__ __forceinline__ uint32_t down_pair(const Quad<DT>& a, const Quad<DT>& b, int j) {
  return perm_b32(j < 2 ? b.w.x : b.w.y, j < 2 ? a.w.x : a.w.y, j & 1 ? 0x07060302u : 0x05040100u);
}

template <int DT, bool kWide, bool SR, bool kSum>
__global__ __launch_bounds__(512) void mxfp4_both_kernel(const BothArgs p) {
  constexpr int kPitch = 36;  // bytes of a column in LDS (lanes then lie in different banks)
  constexpr int kW = ColMax<DT>::kWords;
  __shared__ __attribute__((aligned(16))) uint8_t out[256 * kPitch];
  __shared__ __attribute__((aligned(16))) uint32_t tops[8][64 * kW];
  __shared__ __attribute__((aligned(8))) uint8_t bytes[2][256];
  __shared__ __attribute__((aligned(16))) float sums[kSum ? 8 : 1][256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = wave >> 2, sub = wave & 3;
  // workgroups i, i + 8, i + 16, i + 24 of 32 (on one XCD): the tiles below each other of a line
  const uint32_t line = (blockIdx.x >> 5) * 8 + (blockIdx.x & 7);
  if (line >= p.lines) return;
  const int64_t tl = line / (uint32_t)p.col_tiles, tc = line - tl * p.col_tiles, tr = 4 * tl + ((blockIdx.x >> 3) & 3);
  const int64_t c0 = tc * 256 + 4 * lane;
  const int64_t r0 = tr * 64 + 8 * wave;
  Quad<DT> x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = quad_at<DT, kWide>(p, r0 + i, c0);
  if constexpr (kSum) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += x[i].get(j);
    *reinterpret_cast<float4*>(&sums[wave][4 * lane]) = float4{s[0], s[1], s[2], s[3]};
  }
  uint32_t rnd[SR ? 8 : 1][4];
  if constexpr (SR) {
    const uint64_t z_row = (uint64_t)((p.cols + kBlock - 1) / kBlock) * (kBlock / 4) * kDropGolden;
    const uint64_t z = *p.seed + (uint64_t)r0 * z_row + (uint64_t)(c0 / 4) * kDropGolden;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits4(rnd[i], mix(z + (uint64_t)i * z_row));
  }
  ColMax<DT> top;
#pragma unroll
  for (int i = 0; i < 8; ++i) top.take(x[i]);
  top.put(&tops[wave][lane * kW]);
  // rows
  if (p.row_data) {
    uint32_t mine = 0;  // lane 8 b + i: the scale of row i, block b
    uint8_t* rows_at = p.row_data + (c0 >> 7) * panel_of(p.rows) + r0 * 64 + (c0 & 127) / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = quad_max(row_max<DT>(x[i]));
      m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, false));  // 7 - lane of 8
      const uint32_t byte = scale_byte<SR>(m);
      const float scale = scale_bits(byte);
      mine = (lane & 7) == i ? byte : mine;
      uint32_t r;
      if constexpr (SR) {
        r = low_bytes(two_codes(encode_sr(x[i].get(0), rnd[i][0], scale), encode_sr(x[i].get(1), rnd[i][1], scale)),
                      two_codes(encode_sr(x[i].get(2), rnd[i][2], scale), encode_sr(x[i].get(3), rnd[i][3], scale)));
      } else if constexpr (DT == DPA_DTYPE_F32) {
        r = encode_pair<1>(encode_pair<0>(0u, x[i].w.x, x[i].w.y, scale), x[i].w.z, x[i].w.w, scale);
      } else {
        r = encode_pair<DT, 1>(encode_pair<DT, 0>(0u, x[i].w.x, scale), x[i].w.y, scale);
      }
      if (r0 + i < p.rows) *reinterpret_cast<uint16_t*>(rows_at + 64 * i) = (uint16_t)r;
    }
    const int64_t row = r0 + (lane & 7);
    const int b = (int)(tc * 8) + (lane >> 3);
    if (row < p.rows) p.row_scales[((int64_t)(b >> 4) * p.rows + row) * 16 + scale_at(b & 15)] = (uint8_t)mine;
  }
  wait_lgkmcnt0();
  lds_barrier();
  if constexpr (kSum) {
    if (threadIdx.x < 256 && tc * 256 + threadIdx.x < p.cols && tr * 64 < p.rows) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
      p.sums[tr * p.cols + tc * 256 + threadIdx.x] = s;
    }
  }
  // columns: word `sub` of block `half`
#pragma unroll
  for (int w = 0; w < 4; ++w) top.join(&tops[4 * half + w][lane * kW]);
  uint32_t some = 0;
  float scale[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t byte = scale_byte<SR>(top.get(j));
    some |= byte << (8 * j);
    scale[j] = scale_bits(byte);
  }
  if (sub == 0) *reinterpret_cast<uint32_t*>(&bytes[half][4 * lane]) = some;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t r;
    if constexpr (SR) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c[i] = two_codes(encode_sr(x[2 * i].get(j), rnd[2 * i][j], scale[j]),
                         encode_sr(x[2 * i + 1].get(j), rnd[2 * i + 1][j], scale[j]));
      r = low_bytes(c[0], c[1], c[2], c[3]);
    } else if constexpr (DT == DPA_DTYPE_F32) {
      r = encode_pair<0>(0u, x[0].get(j), x[1].get(j), scale[j]);
      r = encode_pair<1>(r, x[2].get(j), x[3].get(j), scale[j]);
      r = encode_pair<2>(r, x[4].get(j), x[5].get(j), scale[j]);
      r = encode_pair<3>(r, x[6].get(j), x[7].get(j), scale[j]);
    } else {
      r = encode_pair<DT, 0>(0u, down_pair<DT>(x[0], x[1], j), scale[j]);
      r = encode_pair<DT, 1>(r, down_pair<DT>(x[2], x[3], j), scale[j]);
      r = encode_pair<DT, 2>(r, down_pair<DT>(x[4], x[5], j), scale[j]);
      r = encode_pair<DT, 3>(r, down_pair<DT>(x[6], x[7], j), scale[j]);
    }
    *reinterpret_cast<uint32_t*>(out + (j * 64 + lane) * kPitch + half * 16 + 4 * sub) = r;
  }
  __syncthreads();
  {
    const int at = threadIdx.x >> 1, chunk = threadIdx.x & 1;
    const int64_t col = tc * 256 + 4 * (at & 63) + (at >> 6);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(out + at * kPitch + chunk * 16);
    if (col < p.cols)
      *reinterpret_cast<uint4*>(p.col_data + (tr >> 1) * panel_of(p.cols) + col * 64 + (tr & 1) * 32 + chunk * 16) =
          uint4{w[0], w[1], w[2], w[3]};
  }
  const int64_t col = tc * 256 + (threadIdx.x >> 1), block = tr * 2 + (threadIdx.x & 1);
  if (col < p.cols)
    p.col_scales[((block >> 4) * p.cols + col) * 16 + scale_at((int)(block & 15))] = bytes[threadIdx.x & 1][threadIdx.x >> 1];
}

// ---------------------------------------------------------------------------------------
// Back: 8 elements a lane, exact in fp32, rounded once. 64 Mi elements to bf16 (170 MB) 25 us, 6.8 TB/s with the codes
// in the caches.
// ---------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void mxfp4_values_kernel(const uint32_t* data, const uint8_t* scales, void* y,
                                                           int64_t groups) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g >= groups) return;
  const uint32_t w = data[g];
  const float s = scale_back(scales[g >> 2]);
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1),
            c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
  if constexpr (DT == DPA_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(y) + 2 * g;
    o[0] = float4{a.x, a.y, b.x, b.y};
    o[1] = float4{c.x, c.y, d.x, d.y};
  } else {
    reinterpret_cast<uint4*>(y)[g] =
        uint4{Elem<DT>::pack(a.x, a.y), Elem<DT>::pack(b.x, b.y), Elem<DT>::pack(c.x, c.y), Elem<DT>::pack(d.x, d.y)};
  }
}

// ---------------------------------------------------------------------------------------
// Column sums in fp32, in a fixed order: a workgroup takes 64 columns of `span` rows, its four waves every fourth
// row; then the pieces
// ---------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void column_sum_kernel(const void* x, float* part, int64_t rows, int64_t cols,
                                                         int64_t ld, int span) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  const int64_t r0 = (int64_t)blockIdx.y * span, r1 = min(rows, r0 + span);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < cols)
    for (int64_t r = r0 + wave; r < r1; r += 16)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + 4 * i < r1) s[i] += load1<DT>(x, (r + 4 * i) * ld + c);
  sums[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (wave == 0 && c < cols)
    part[blockIdx.y * cols + c] = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
}

template <int DT, bool SR>
static int run_rows(const RowArgs& p, bool operand, bool wide, hipStream_t s) {
  const unsigned grid = (unsigned)(operand ? ceil_div(p.rows, 4) * groups_of(p.cols) : ceil_div(p.groups, 256));
  if (!operand)
    mxfp4_rows_kernel<DT, false, true, SR><<<grid, 256, 0, s>>>(p);
  else if (wide)
    mxfp4_rows_kernel<DT, true, true, SR><<<grid, 256, 0, s>>>(p);
  else
    mxfp4_rows_kernel<DT, true, false, SR><<<grid, 256, 0, s>>>(p);
  return launch_status();
}

template <int DT, bool kWide, bool SR>
static int run_both(const BothArgs& p, hipStream_t s) {
  const unsigned grid = (unsigned)(ceil_div(p.lines, 8) * 32);
  if (p.sums)
    mxfp4_both_kernel<DT, kWide, SR, true><<<grid, 512, 0, s>>>(p);
  else
    mxfp4_both_kernel<DT, kWide, SR, false><<<grid, 512, 0, s>>>(p);
  return launch_status();
}

template <int DT, bool SR>
static int run_both(const BothArgs& p, bool wide, hipStream_t s) {
  return wide ? run_both<DT, true, SR>(p, s) : run_both<DT, false, SR>(p, s);
}

template <int DT>
static int run_operands(const RowArgs& r, const BothArgs& b, bool wide, hipStream_t s) {
  if (b.col_data) return b.seed ? run_both<DT, true>(b, wide, s) : run_both<DT, false>(b, wide, s);
  return r.seed ? run_rows<DT, true>(r, true, wide, s) : run_rows<DT, false>(r, true, wide, s);
}

// rows of x to a workgroup of column_sum_kernel
static int sum_span(int64_t rows, int64_t cols) {
  int64_t pieces = 4 * num_cus() / ceil_div(cols, 64);
  if (pieces > rows / 32) pieces = rows / 32;
  if (pieces < 1) pieces = 1;
  return (int)ceil_div(rows, pieces);
}

template <int DT>
static void run_sum(const void* x, float* part, int64_t rows, int64_t cols, int64_t ld, int span, hipStream_t s) {
  column_sum_kernel<DT><<<dim3((unsigned)ceil_div(cols, 64), (unsigned)ceil_div(rows, span)), 256, 0, s>>>(x, part, rows, cols, ld, span);
}

}  // namespace mx
}  // namespace dpa

using namespace dpa;
using namespace dpa::mx;

extern "C" int dpa_mxfp4_quantize(const void* x, int dtype, int64_t n, void* data, void* scales, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  if (n < 0 || n % kBlock || ceil_div(n / 8, 256) > kMaxGroups256) return DPA_ERR_SIZE;
  if (n == 0) return DPA_OK;
  if (!x || !data || !scales) return DPA_ERR_NULL;
  if (!aligned(x, 16) || !aligned(data, 4)) return DPA_ERR_ALIGN;
  RowArgs p{};
  p.x = x, p.data = (uint8_t*)data, p.scales = (uint8_t*)scales, p.groups = n / 8;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPA_DTYPE_BF16) return run_rows<DPA_DTYPE_BF16, false>(p, false, true, s);
  if (dtype == DPA_DTYPE_F16) return run_rows<DPA_DTYPE_F16, false>(p, false, true, s);
  return run_rows<DPA_DTYPE_F32, false>(p, false, true, s);
}

extern "C" int dpa_mxfp4_dequantize(const void* data, const void* scales, void* y, int dtype, int64_t n, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  if (n < 0 || n % kBlock || ceil_div(n / 8, 256) > kMaxGroups256) return DPA_ERR_SIZE;
  if (n == 0) return DPA_OK;
  if (!y || !data || !scales) return DPA_ERR_NULL;
  if (!aligned(y, 16) || !aligned(data, 4)) return DPA_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  const unsigned grid = (unsigned)ceil_div(n / 8, 256);
  const uint32_t* d = (const uint32_t*)data;
  const uint8_t* e = (const uint8_t*)scales;
  if (dtype == DPA_DTYPE_BF16)
    mxfp4_values_kernel<DPA_DTYPE_BF16><<<grid, 256, 0, s>>>(d, e, y, n / 8);
  else if (dtype == DPA_DTYPE_F16)
    mxfp4_values_kernel<DPA_DTYPE_F16><<<grid, 256, 0, s>>>(d, e, y, n / 8);
  else
    mxfp4_values_kernel<DPA_DTYPE_F32><<<grid, 256, 0, s>>>(d, e, y, n / 8);
  return launch_status();
}

extern "C" int64_t dpa_mxfp4_operand_bytes(int64_t rows, int64_t cols) {
  return matrix_ok(rows, cols) ? operand_bytes(rows, cols) : 0;
}

extern "C" int dpa_mxfp4_operands(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                  void* by_rows, void* by_cols, float* sums, const void* seed, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  if (!matrix_ok(rows, cols) || (row_stride < cols && rows > 1)) return DPA_ERR_SIZE;
  if ((!by_rows && !by_cols) || (sums && !by_cols)) return DPA_ERR_NULL;
  if (rows == 0) return DPA_OK;
  if (!x) return DPA_ERR_NULL;
  if (!aligned(x, size_of(dtype)) || !aligned(by_rows, 16) || !aligned(by_cols, 16) || !aligned(sums, 4) || !aligned(seed, 8))
    return DPA_ERR_ALIGN;
  RowArgs r{};
  r.x = x, r.data = (uint8_t*)by_rows, r.scales = r.data + operand_data_bytes(rows, cols), r.seed = (const uint64_t*)seed;
  r.rows = rows, r.cols = cols, r.ld = row_stride;
  r.per_rows = make_fastdiv((uint32_t)groups_of(cols));
  BothArgs b{};
  b.x = x, b.row_data = r.data, b.row_scales = r.scales, b.seed = r.seed;
  b.col_data = (uint8_t*)by_cols, b.col_scales = b.col_data + operand_data_bytes(cols, rows);
  b.rows = rows, b.cols = cols, b.ld = row_stride, b.sums = sums;
  b.col_tiles = (int)ceil_div(cols, 256);
  b.lines = (uint32_t)(ceil_div(rows, 256) * b.col_tiles);
  // whole aligned vectors: 16 B of 8 elements (8 B of 4) of a 16-bit type, 16 B of 4 of fp32
  const int vec = by_cols || dtype == DPA_DTYPE_F32 ? 4 : 8;
  const bool wide = row_stride % vec == 0 && (!by_cols || cols % 4 == 0) && aligned(x, vec * size_of(dtype));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPA_DTYPE_BF16) return run_operands<DPA_DTYPE_BF16>(r, b, wide, s);
  if (dtype == DPA_DTYPE_F16) return run_operands<DPA_DTYPE_F16>(r, b, wide, s);
  return run_operands<DPA_DTYPE_F32>(r, b, wide, s);
}

extern "C" int64_t dpa_column_sum_workspace_bytes(int64_t rows, int64_t cols) {
  return rows > 0 && cols > 0 ? ceil_div(rows, sum_span(rows, cols)) * cols * 4 : 0;
}

extern "C" int dpa_column_sum(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void* y,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  if (rows <= 0 || cols <= 0 || rows >= (1 << 30) || cols > 64 * kMaxGroups256 || (row_stride < cols && rows > 1))
    return DPA_ERR_SIZE;
  if (!x || !y) return DPA_ERR_NULL;
  if (!workspace || workspace_bytes < dpa_column_sum_workspace_bytes(rows, cols)) return DPA_ERR_WORKSPACE;
  if (!aligned(x, size_of(dtype)) || !aligned(y, 4) || !aligned(workspace, 4)) return DPA_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  const int span = sum_span(rows, cols);
  const int64_t pieces = ceil_div(rows, span);
  float* part = pieces > 1 ? (float*)workspace : (float*)y;
  if (dtype == DPA_DTYPE_BF16)
    run_sum<DPA_DTYPE_BF16>(x, part, rows, cols, row_stride, span, s);
  else if (dtype == DPA_DTYPE_F16)
    run_sum<DPA_DTYPE_F16>(x, part, rows, cols, row_stride, span, s);
  else
    run_sum<DPA_DTYPE_F32>(x, part, rows, cols, row_stride, span, s);
  const int st = launch_status();
  if (st != DPA_OK || pieces <= 1) return st;
  run_sum<DPA_DTYPE_F32>(part, (float*)y, pieces, cols, cols, (int)pieces, s);
  return launch_status();
}
