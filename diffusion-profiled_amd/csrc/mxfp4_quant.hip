// Tensors to MXFP4 and back (format: mxfp4.hpp). All of it is bound by the bytes it moves.
#include "mxfp4.hpp"

namespace dpa {
namespace mx {

// ---------------------------------------------------------------------------------------
// Blocks along the rows: four lanes to a block, 8 elements a lane (16 B of a 16-bit type), the largest
// magnitude exchanged within the quad. Dense tensors are one long row; of an operand, a lane's row is
// g / per_row, and what lies behind cols comes as zeros.
// ---------------------------------------------------------------------------------------
struct RowArgs {
  const void* x;
  uint8_t *data, *scales;
  const uint64_t* seed;  // null: to nearest
  int64_t groups;        // of 8 elements
  int64_t rows, cols, ld;
  FastDiv per_row;       // groups to a padded row
};

template <int DT>
__device__ __forceinline__ void load8(float (&v)[8], const void* p, int64_t at) {
  if constexpr (DT == DPA_DTYPE_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = Elem<DT>::lo(w[i]), v[2 * i + 1] = Elem<DT>::hi(w[i]);
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, false));  // lane ^ 1
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, false));  // lane ^ 2
}

// 8 elements of a block, its largest magnitude m -> their codes; idx4: the number of the first, over 4
template <bool SR>
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], uint32_t byte, uint64_t seed, uint64_t idx4) {
  const float inv = inverse_of(byte);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = v[i] * inv;
  if constexpr (!SR) return encode8(s);
  uint32_t r = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint64_t z = bits_of(seed, idx4 + j);
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= encode_sr(s[4 * j + i], (uint32_t)(z >> (16 * i)) & 0xffffu) << (4 * (4 * j + i));
  }
  return r;
}

// kOperand: an operand's rows, else dense. kWide: rows of whole aligned 8-element groups.
template <int DT, bool kOperand, bool kWide, bool SR>
__global__ __launch_bounds__(256) void mxfp4_rows_kernel(const RowArgs p) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g >= p.groups) return;  // (whole blocks: a quad ends together)
  int64_t row = 0, in_row = g;
  if constexpr (kOperand) row = fdiv((uint32_t)g, p.per_row), in_row = g - row * p.per_row.d;
  const int64_t c0 = in_row * 8, at = row * p.ld + c0;
  float v[8];
  if constexpr (!kOperand) {
    load8<DT>(v, p.x, at);
  } else {
    if (kWide && c0 + 8 <= p.cols) {
      load8<DT>(v, p.x, at);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c0 + i < p.cols ? load1<DT>(p.x, at + i) : 0.f;
    }
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  const uint32_t byte = scale_byte<SR>(quad_max(m));
  const uint64_t pitch4 = kOperand ? (uint64_t)((p.cols + kBlock - 1) / kBlock) * (kBlock / 4) : 0;
  const uint32_t r = codes8<SR>(v, byte, SR ? *p.seed : 0, row * pitch4 + (uint64_t)in_row * 2);
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
// matrix transposed). A thread holds 4 columns of 32 rows in registers: a column's block is its own, a
// row's block the 8 lanes beside it. W waves below each other; their codes of a column meet in LDS,
// so that they leave in pieces of 16 W B.
// ---------------------------------------------------------------------------------------
struct BothArgs {
  const void* x;
  uint8_t *row_data, *row_scales, *col_data, *col_scales;
  const uint64_t* seed;
  int64_t rows, cols, ld;
  int col_tiles;
};

template <int DT>
struct Quad;  // 4 neighbours of a row
template <>
struct Quad<DPA_DTYPE_F32> {
  float4 w;
  __device__ __forceinline__ float get(int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
};
template <int DT>
struct Quad {
  uint2 w;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? w.x : w.y;
    return i & 1 ? Elem<DT>::hi(u) : Elem<DT>::lo(u);
  }
};

template <int DT>
__device__ __forceinline__ Quad<DT> quad_at(const void* x, int64_t at, int64_t left, bool wide) {
  Quad<DT> q;
  if (wide && left >= 4) {
    q.w = *reinterpret_cast<const decltype(q.w)*>(static_cast<const uint8_t*>(x) + at * Elem<DT>::size);
    return q;
  }
  if constexpr (DT == DPA_DTYPE_F32) {
    const float* s = static_cast<const float*>(x) + at;
    q.w = float4{left > 0 ? s[0] : 0.f, left > 1 ? s[1] : 0.f, left > 2 ? s[2] : 0.f, left > 3 ? s[3] : 0.f};
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(x) + at;
    const uint32_t a = left > 0 ? s[0] : 0, b = left > 1 ? s[1] : 0, c = left > 2 ? s[2] : 0, d = left > 3 ? s[3] : 0;
    q.w = uint2{a | b << 16, c | d << 16};
  }
  return q;
}

template <int DT, int W, bool kRows, bool SR>
__global__ __launch_bounds__(64 * W) void mxfp4_both_kernel(const BothArgs p, bool wide) {
  constexpr int kPitch = 16 * W + 16;  // (lanes then lie in 16 different places of the banks)
  __shared__ __attribute__((aligned(16))) uint8_t lds[256 * kPitch];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tr = blockIdx.x / (uint32_t)p.col_tiles, tc = blockIdx.x - tr * p.col_tiles;
  const int64_t block = tr * W + wave, r0 = block * 32, c0 = tc * 256 + 4 * lane, left = p.cols - c0;
  Quad<DT> x[32];
#pragma unroll
  for (int i = 0; i < 32; ++i)
    x[i] = quad_at<DT>(p.x, (r0 + i) * p.ld + c0, r0 + i < p.rows ? left : 0, wide);
  const uint64_t seed = SR ? *p.seed : 0;
  const uint64_t pitch4 = (uint64_t)((p.cols + kBlock - 1) / kBlock) * (kBlock / 4);
  auto bits = [&](int i) { return bits_of(seed, (uint64_t)(r0 + i) * pitch4 + (uint64_t)c0 / 4); };

  if constexpr (kRows) {
    const int64_t pitch = pitch_of(p.cols);
    const int b = (int)(c0 >> 5);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float v[4];
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x[i].get(j), m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
      m = quad_max(m);
      m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, false));  // 7 - lane of 8
      const uint32_t byte = scale_byte<SR>(m);
      const float inv = inverse_of(byte);
      uint32_t r;
      if constexpr (SR) {
        const uint64_t z = bits(i);
        r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) r |= encode_sr(v[j] * inv, (uint32_t)(z >> (16 * j)) & 0xffffu) << (4 * j);
      } else {
        r = encode4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      }
      if (r0 + i < p.rows) {
        *reinterpret_cast<uint16_t*>(p.row_data + (r0 + i) * pitch + c0 / 2) = (uint16_t)r;
        if ((lane & 7) == 0)
          p.row_scales[((int64_t)(b >> 4) * p.rows + r0 + i) * 16 + scale_at(b & 15)] = (uint8_t)byte;
      }
    }
  }

  uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 32; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = max(m[j], __float_as_uint(x[i].get(j)) & 0x7fffffffu);
  uint32_t byte[4];
  float inv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    byte[j] = scale_byte<SR>(m[j]), inv[j] = inverse_of(byte[j]);
    if (j < left)
      p.col_scales[((block >> 4) * p.cols + c0 + j) * 16 + scale_at((int)(block & 15))] = (uint8_t)byte[j];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {  // 8 rows: a word of each column
    uint32_t r[4] = {0, 0, 0, 0};
    if constexpr (SR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t z = bits(8 * q + i);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          r[j] |= encode_sr(x[8 * q + i].get(j) * inv[j], (uint32_t)(z >> (16 * j)) & 0xffffu) << (4 * i);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[8 * q + i].get(j) * inv[j];
        r[j] = encode8(v);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint32_t*>(lds + (j * 64 + lane) * kPitch + wave * 16 + 4 * q) = r[j];
  }
  __syncthreads();
  const int64_t pitch = pitch_of(p.rows);
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int id = it * 64 * W + threadIdx.x, line = id / W, chunk = id % W;
    const int64_t col = tc * 256 + 4 * (line & 63) + (line >> 6);
    if (col < p.cols)
      *reinterpret_cast<uint4*>(p.col_data + col * pitch + tr * (16 * W) + chunk * 16) =
          *reinterpret_cast<const uint4*>(lds + line * kPitch + chunk * 16);
  }
}

// ---------------------------------------------------------------------------------------
// Back: 8 elements a lane, exact in fp32, rounded once
// ---------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void mxfp4_values_kernel(const uint32_t* data, const uint8_t* scales, void* y,
                                                           int64_t groups) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g >= groups) return;
  const uint32_t w = data[g];
  const float s = scale_of(scales[g >> 2]);
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
            c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  if constexpr (DT == DPA_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(y) + 2 * g;
    o[0] = float4{a.x * s, a.y * s, b.x * s, b.y * s};
    o[1] = float4{c.x * s, c.y * s, d.x * s, d.y * s};
  } else {
    reinterpret_cast<uint4*>(y)[g] = uint4{Elem<DT>::pack(a.x * s, a.y * s), Elem<DT>::pack(b.x * s, b.y * s),
                                           Elem<DT>::pack(c.x * s, c.y * s), Elem<DT>::pack(d.x * s, d.y * s)};
  }
}

// ---------------------------------------------------------------------------------------
// Column sums in fp32, in a fixed order: a workgroup's 256 columns of kSumRows rows, then the pieces
// ---------------------------------------------------------------------------------------
constexpr int kSumRows = 128;

template <int DT>
__global__ __launch_bounds__(256) void column_sum_kernel(const void* x, float* part, int64_t rows, int64_t cols, int64_t ld) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const int64_t r0 = (int64_t)blockIdx.y * kSumRows, r1 = min(rows, r0 + kSumRows);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t r = r0; r < r1; r += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r + i < r1) s[i] += load1<DT>(x, (r + i) * ld + c);
  part[blockIdx.y * cols + c] = (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(256) void column_join_kernel(const float* part, float* y, int64_t pieces, int64_t cols) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t r = 0; r < pieces; r += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r + i < pieces) s[i] += part[(r + i) * cols + c];
  y[c] = (s[0] + s[1]) + (s[2] + s[3]);
}

template <int DT, bool SR>
static int run_rows(const RowArgs& p, bool operand, bool wide, hipStream_t s) {
  const unsigned grid = (unsigned)ceil_div(p.groups, 256);
  if (!operand)
    mxfp4_rows_kernel<DT, false, true, SR><<<grid, 256, 0, s>>>(p);
  else if (wide)
    mxfp4_rows_kernel<DT, true, true, SR><<<grid, 256, 0, s>>>(p);
  else
    mxfp4_rows_kernel<DT, true, false, SR><<<grid, 256, 0, s>>>(p);
  return launch_status();
}

template <int DT, int W>
static int run_both(const BothArgs& p, bool wide, hipStream_t s) {
  const int64_t row_tiles = ceil_div(p.rows, 256) * (8 / W);
  const unsigned grid = (unsigned)(row_tiles * p.col_tiles);
  if (p.row_data && p.seed)
    mxfp4_both_kernel<DT, W, true, true><<<grid, 64 * W, 0, s>>>(p, wide);
  else if (p.row_data)
    mxfp4_both_kernel<DT, W, true, false><<<grid, 64 * W, 0, s>>>(p, wide);
  else if (p.seed)
    mxfp4_both_kernel<DT, W, false, true><<<grid, 64 * W, 0, s>>>(p, wide);
  else
    mxfp4_both_kernel<DT, W, false, false><<<grid, 64 * W, 0, s>>>(p, wide);
  return launch_status();
}

template <int DT>
static int run_operands(const RowArgs& r, const BothArgs& b, bool wide, hipStream_t s) {
  if (!b.col_data) return r.seed ? run_rows<DT, true>(r, true, wide, s) : run_rows<DT, false>(r, true, wide, s);
  // Waves below each other: fewer where the workgroups would leave CUs idle
  const int64_t tiles = ceil_div(b.rows, 256) * b.col_tiles;
  if (tiles >= 2 * num_cus()) return run_both<DT, 8>(b, wide, s);
  return run_both<DT, 2>(b, wide, s);
}

// Sizes of a matrix that the kernels take: 32-bit numbers of 8-element groups and workgroups
static int check_matrix(int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0) return DPA_ERR_SIZE;
  if (rows >= (1ll << 30) || cols >= (1ll << 30)) return DPA_ERR_SIZE;
  if (rows * (pitch_of(cols) / 4) >= (1ll << 31) || cols * (pitch_of(rows) / 4) >= (1ll << 31)) return DPA_ERR_SIZE;
  return DPA_OK;
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

extern "C" int64_t dpa_mxfp4_operand_data_bytes(int64_t rows, int64_t cols) {
  return check_matrix(rows, cols) == DPA_OK ? rows * pitch_of(cols) : 0;
}

extern "C" int64_t dpa_mxfp4_operand_scale_bytes(int64_t rows, int64_t cols) {
  return check_matrix(rows, cols) == DPA_OK ? groups_of(cols) * rows * 16 : 0;
}

extern "C" int dpa_mxfp4_operands(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                  void* row_data, void* row_scales, void* col_data, void* col_scales,
                                  const void* seed, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  const int st = check_matrix(rows, cols);
  if (st != DPA_OK) return st;
  if (row_stride < cols && rows > 1) return DPA_ERR_SIZE;
  if ((!row_data) != (!row_scales) || (!col_data) != (!col_scales) || (!row_data && !col_data)) return DPA_ERR_NULL;
  if (rows == 0) return DPA_OK;
  if (!x) return DPA_ERR_NULL;
  if (!aligned(x, size_of(dtype)) || !aligned(row_data, 16) || !aligned(row_scales, 16) || !aligned(col_data, 16) ||
      !aligned(col_scales, 16) || !aligned(seed, 8))
    return DPA_ERR_ALIGN;
  RowArgs r{};
  r.x = x, r.data = (uint8_t*)row_data, r.scales = (uint8_t*)row_scales, r.seed = (const uint64_t*)seed;
  r.rows = rows, r.cols = cols, r.ld = row_stride;
  r.groups = rows * (pitch_of(cols) / 4);
  r.per_row = make_fastdiv((uint32_t)(pitch_of(cols) / 4));
  BothArgs b{};
  b.x = x, b.row_data = r.data, b.row_scales = r.scales, b.seed = r.seed;
  b.col_data = (uint8_t*)col_data, b.col_scales = (uint8_t*)col_scales;
  b.rows = rows, b.cols = cols, b.ld = row_stride;
  b.col_tiles = (int)ceil_div(cols, 256);
  // whole aligned vectors: 16 B of 8 elements (8 B of 4) of a 16-bit type, 16 B of 4 of fp32
  const int vec = col_data || dtype == DPA_DTYPE_F32 ? 4 : 8;
  const bool wide = row_stride % vec == 0 && aligned(x, vec * size_of(dtype));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPA_DTYPE_BF16) return run_operands<DPA_DTYPE_BF16>(r, b, wide, s);
  if (dtype == DPA_DTYPE_F16) return run_operands<DPA_DTYPE_F16>(r, b, wide, s);
  return run_operands<DPA_DTYPE_F32>(r, b, wide, s);
}

extern "C" int64_t dpa_column_sum_workspace_bytes(int64_t rows, int64_t cols) {
  return rows > 0 && cols > 0 ? ceil_div(rows, kSumRows) * cols * 4 : 0;
}

extern "C" int dpa_column_sum(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void* y,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  if (rows <= 0 || cols <= 0 || cols >= (1ll << 30) || ceil_div(rows, kSumRows) > 65535 || (row_stride < cols && rows > 1))
    return DPA_ERR_SIZE;
  if (!x || !y) return DPA_ERR_NULL;
  if (!workspace || workspace_bytes < dpa_column_sum_workspace_bytes(rows, cols)) return DPA_ERR_WORKSPACE;
  if (!aligned(x, size_of(dtype)) || !aligned(y, 4) || !aligned(workspace, 4)) return DPA_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  const unsigned cb = (unsigned)ceil_div(cols, 256), rb = (unsigned)ceil_div(rows, kSumRows);
  float* part = (float*)workspace;
  if (dtype == DPA_DTYPE_BF16)
    column_sum_kernel<DPA_DTYPE_BF16><<<dim3(cb, rb), 256, 0, s>>>(x, part, rows, cols, row_stride);
  else if (dtype == DPA_DTYPE_F16)
    column_sum_kernel<DPA_DTYPE_F16><<<dim3(cb, rb), 256, 0, s>>>(x, part, rows, cols, row_stride);
  else
    column_sum_kernel<DPA_DTYPE_F32><<<dim3(cb, rb), 256, 0, s>>>(x, part, rows, cols, row_stride);
  const int st = launch_status();
  if (st != DPA_OK) return st;
  column_join_kernel<<<cb, 256, 0, s>>>(part, (float*)y, rb, cols);
  return launch_status();
}
