// Dropout by the counter hash that the GroupNorm+SiLU kernels use, as an operator of its own:
// y = r + keep x / (1 - p) (r optional); the backward is the same call on dy without r. The mask
// is recomputed from (seed, element index), never stored.
//
// Bound by HBM: x (and r) read once, y written once. The hash costs two 64-bit multiplies for
// four elements, about a third of the vector time that the 4 B per element of the smallest form
// (bf16, no residual) leave at full bandwidth. 16.8 M fp32 elements with the residual and their backward
// without: 63.9 us for 335 MB, 5.2 TB/s; 3.9 M bf16 elements 4.9 us.
#include "dpa_common.hpp"

namespace dpa {
namespace drop {

struct Args {
  const void *x, *r;
  void* y;
  const uint64_t* seed;
  int64_t n;
  uint32_t keep2;  // the threshold in both halves
  float scale;
};

// 8 elements per step; word i of m covers elements 2 i, 2 i + 1. A dropped element is cleared
// before the product, so that an infinity or NaN there gives 0.
template <int DT>
__device__ __forceinline__ void step8(const Args& p, int64_t i, uint4 mk) {
  const uint32_t m[4] = {mk.x, mk.y, mk.z, mk.w};
  if constexpr (DT == DPA_DTYPE_F32) {
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const float*>(p.x) + i);
    uint4 v[2] = {x[0], x[1]};
    float4 r[2] = {};
    if (p.r) {
      const float4* rp = reinterpret_cast<const float4*>(static_cast<const float*>(p.r) + i);
      r[0] = rp[0], r[1] = rp[1];
    }
    float4* y = reinterpret_cast<float4*>(static_cast<float*>(p.y) + i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t a = m[2 * j], b = m[2 * j + 1];
      float4 o;
      o.x = __uint_as_float(v[j].x & (uint32_t)((int)(a << 16) >> 16)) * p.scale;
      o.y = __uint_as_float(v[j].y & (uint32_t)((int)a >> 16)) * p.scale;
      o.z = __uint_as_float(v[j].z & (uint32_t)((int)(b << 16) >> 16)) * p.scale;
      o.w = __uint_as_float(v[j].w & (uint32_t)((int)b >> 16)) * p.scale;
      if (p.r) o.x += r[j].x, o.y += r[j].y, o.z += r[j].z, o.w += r[j].w;
      y[j] = o;
    }
  } else {
    typedef Elem<DT> E;
    const uint4 xv = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + i);
    uint4 rv = {};
    if (p.r) rv = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.r) + i);
    const uint32_t x[4] = {xv.x & m[0], xv.y & m[1], xv.z & m[2], xv.w & m[3]};
    const uint32_t r[4] = {rv.x, rv.y, rv.z, rv.w};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = E::lo(x[j]) * p.scale, b = E::hi(x[j]) * p.scale;
      if (p.r) a += E::lo(r[j]), b += E::hi(r[j]);
      o[j] = E::pack(a, b);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + i) = uint4{o[0], o[1], o[2], o[3]};
  }
}

// one element of group i0 .. i0 + 7 (the tail, and tensors that are not aligned to 16 B)
template <int DT>
__device__ __forceinline__ void step1(const Args& p, int64_t i, uint32_t kept) {
  if constexpr (DT == DPA_DTYPE_F32) {
    float o = kept ? static_cast<const float*>(p.x)[i] * p.scale : 0.f;
    if (p.r) o += static_cast<const float*>(p.r)[i];
    static_cast<float*>(p.y)[i] = o;
  } else {
    typedef Elem<DT> E;
    float o = kept ? E::lo(static_cast<const uint16_t*>(p.x)[i]) * p.scale : 0.f;
    if (p.r) o += E::lo(static_cast<const uint16_t*>(p.r)[i]);
    static_cast<uint16_t*>(p.y)[i] = (uint16_t)E::pack(o, 0.f);
  }
}

template <int DT, bool kVec>
__global__ __launch_bounds__(256) void dropout_kernel(const Args p) {
  const uint64_t seed = *p.seed;
  const int64_t step = (int64_t)gridDim.x * 256 * 8;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < p.n; i += step) {
    const uint4 mk = drop_mask8(drop_z(seed, i), p.keep2);
    if (kVec && i + 8 <= p.n) {
      step8<DT>(p, i, mk);
    } else {
      const uint32_t m[4] = {mk.x, mk.y, mk.z, mk.w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < p.n) step1<DT>(p, i + j, m[j / 2] & (j % 2 ? 0xffff0000u : 0xffffu));
    }
  }
}

template <int DT>
static void launch(const Args& p, hipStream_t s) {
  const bool vec = aligned(p.x, 16) && aligned(p.y, 16) && (!p.r || aligned(p.r, 16));
  int64_t grid = ceil_div(p.n, 2048);
  if (grid > 1 << 20) grid = 1 << 20;
  if (vec)
    dropout_kernel<DT, true><<<(unsigned)grid, 256, 0, s>>>(p);
  else
    dropout_kernel<DT, false><<<(unsigned)grid, 256, 0, s>>>(p);
}

}  // namespace drop
}  // namespace dpa

using namespace dpa;

extern "C" int dpa_dropout(const void* x, const void* residual, void* y, int dtype, int64_t n,
                           const void* seed, float p, void* stream) {
  if (n < 0) return DPA_ERR_SIZE;
  if (!drop_p_ok(p)) return DPA_ERR_SIZE;
  if (dtype != DPA_DTYPE_BF16 && dtype != DPA_DTYPE_F32 && dtype != DPA_DTYPE_F16) return DPA_ERR_SHAPE;
  if (n == 0) return DPA_OK;
  if (!x || !y || !seed) return DPA_ERR_NULL;
  const uintptr_t a = dtype == DPA_DTYPE_F32 ? 4 : 2;
  if (!aligned(x, a) || !aligned(y, a) || !aligned(residual, a) || !aligned(seed, 8)) return DPA_ERR_ALIGN;
  drop::Args q{};
  q.x = x, q.r = residual, q.y = y, q.seed = (const uint64_t*)seed, q.n = n;
  q.keep2 = drop_threshold(p) * 0x00010001u;
  q.scale = drop_scale_of(p);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPA_DTYPE_BF16) drop::launch<DPA_DTYPE_BF16>(q, s);
  else if (dtype == DPA_DTYPE_F16) drop::launch<DPA_DTYPE_F16>(q, s);
  else drop::launch<DPA_DTYPE_F32>(q, s);
  return launch_status();
}
