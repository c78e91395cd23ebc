// The forward's split keys: how much workspace they take, and the kernels that join them.
#pragma once
#include "xattn.hpp"

namespace dpa {
namespace xattn {

// Joins the splits of a row: O = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s. Up to kJoinSplits: a
// thread per 4 dims of a row, all its loads at once. More: a wave per row, two dims per lane; its
// splits' (max, sum) come in one load, so that the sums over the splits, whose loads wait for nothing
// else, are the only loop: 4.0 us for 256 rows of 11 splits of 128 dims. (32768 rows of 2 splits: 18 us by
// waves.)
constexpr int kJoinSplits = 8;

template <class T>
__global__ __launch_bounds__(256) void xattn_join_few_kernel(const Args p) {
  const int nd = p.D / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)p.B * p.KVH * p.rows;
  if (i >= rows * nd) return;
  const int64_t at = i / nd;
  const int d0 = (int)(i - at * nd) * 4;
  float2 ml[kJoinSplits];
  float4 v[kJoinSplits];
#pragma unroll
  for (int s = 0; s < kJoinSplits; ++s)
    if (s < p.splits) {
      ml[s] = p.stat[s * rows + at];
      v[s] = *reinterpret_cast<const float4*>(p.part + (s * rows + at) * p.D + d0);
    }
  float m = -__builtin_inff();
#pragma unroll
  for (int s = 0; s < kJoinSplits; ++s)
    if (s < p.splits) m = fmaxf(m, ml[s].x);
  const float ms = m == -__builtin_inff() ? 0.f : m;
  float l = 0.f;
  float4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kJoinSplits; ++s)
    if (s < p.splits) {
      const float f = __builtin_amdgcn_exp2f(ml[s].x - ms);
      l += f * ml[s].y;
      o.x += f * v[s].x, o.y += f * v[s].y, o.z += f * v[s].z, o.w += f * v[s].w;
    }
  const int bkv = (int)(at / p.rows), row = (int)(at - (int64_t)bkv * p.rows);
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;
  const uint32_t head = fdiv(row, p.by_lq), tok = row - head * p.Lq;
  if (d0 == 0)
    p.lse[((int64_t)b * p.H + g * p.G + head) * p.Lq + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  const float il = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(p.out + (((int64_t)b * p.Lq + tok) * p.H + g * p.G + head) * p.D + d0) =
      uint2{T::pack(o.x * il, o.y * il), T::pack(o.z * il, o.w * il)};
}

template <class T>
__global__ __launch_bounds__(256) void xattn_join_kernel(const Args p) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)p.B * p.KVH * p.rows;
  const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at >= rows) return;
  const int d0 = 2 * lane;
  const bool on = d0 < p.D;
  float m = -__builtin_inff(), l = 0.f, a = 0.f, c = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 64) {
    const int n = min(64, p.splits - s0);
    float2 ml = {-__builtin_inff(), 0.f};
    if (lane < n) ml = p.stat[(s0 + lane) * rows + at];
    float top = ml.x;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top), ms = mn == -__builtin_inff() ? 0.f : mn;
    const float keep = __builtin_amdgcn_exp2f(m - ms), f = __builtin_amdgcn_exp2f(ml.x - ms);
    float sum = f * ml.y;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
    l = l * keep + sum, a *= keep, c *= keep, m = mn;
    const float* src = p.part + ((int64_t)s0 * rows + at) * p.D + (on ? d0 : 0);
    const int64_t pitch = rows * p.D;
    for (int s = 0; s < n; s += 8) {  // (past the last one: that one again, with no weight)
      float2 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float2*>(src + min(s + i, n - 1) * pitch);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float fs = s + i < n ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s + i)) : 0.f;
        a = __builtin_fmaf(fs, v[i].x, a), c = __builtin_fmaf(fs, v[i].y, c);
      }
    }
  }
  const int bkv = (int)(at / p.rows), row = (int)(at - (int64_t)bkv * p.rows);
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;
  const uint32_t head = fdiv(row, p.by_lq), tok = row - head * p.Lq;
  if (lane == 0)
    p.lse[((int64_t)b * p.H + g * p.G + head) * p.Lq + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  const float il = l == 0.f ? 0.f : 1.f / l;
  if (on)
    *reinterpret_cast<uint32_t*>(p.out + (((int64_t)b * p.Lq + tok) * p.H + g * p.G + head) * p.D + d0) =
        T::pack(a * il, c * il);
}

// ---- host ------------------------------------------------------------------------------
inline int64_t fwd_workspace(const Args& p) {
  if (p.splits <= 1) return 0;
  return align256(part_rows_bytes(p)) + (int64_t)p.splits * p.B * p.KVH * p.rows * 8;
}

template <class T>
int join_splits(const Args& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.B * p.KVH * p.rows;
  if (p.splits <= kJoinSplits)
    xattn_join_few_kernel<T><<<(unsigned)ceil_div(rows * (p.D / 4), 256), 256, 0, s>>>(p);
  else
    xattn_join_kernel<T><<<(unsigned)ceil_div(rows, 4), 256, 0, s>>>(p);
  return launch_status();
}

}  // namespace xattn
}  // namespace dpa
