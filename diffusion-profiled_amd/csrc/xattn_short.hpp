// The forward of cross attention over up to 128 keys, for keys and values of any kind that a workgroup can bring to
// LDS as rows of 16-bit elements.
#pragma once
#include "xattn.hpp"

namespace dpa {
namespace xattn {

// The bias of NB x 32 keys (0: visible, -inf: not) from visible(key); behind a barrier, which blocks of 32 keys have a
// visible one.
template <int NB, class Visible>
__device__ __forceinline__ void put_bias(float* bias, int tid, Visible visible) {
  if (tid < NB * 32) bias[tid] = visible(tid) ? 0.f : -__builtin_inff();
}
template <int NB>
__device__ __forceinline__ uint32_t active_blocks(const float* bias, int lane) {
  uint32_t act = 0;
#pragma unroll
  for (int i = 0; i < NB; ++i) act |= (__ballot(bias[32 * i + (lane & 31)] == 0.f) ? 1u : 0u) << i;
  return act;
}

// ---------------------------------------------------------------------------------------
// Forward: four waves, each with its own 32 rows of every tile of 128; the next tile's queries load
// while this one's are at work. Layouts and products as in xattn_fwd.hip.
// bring(b, g, keys, values, bias, tid, wave, lane) brings a head's keys, values and bias to LDS and returns
// active_blocks, behind a barrier.
// Bound by HBM, less what a workgroup of few tiles leaves bare at its ends: 128 x 256 queries of 4 heads of
// 64 dims over up to 77 keys 12.4 us (3.3 TB/s), 128 x 1024 of 32 dims 19.5 (3.7).
// ---------------------------------------------------------------------------------------
constexpr int short_waves(int DP) { return DP == 128 ? 2 : DP == 64 ? 3 : 4; }

template <class T, int DP, int NB, class Bring>
__device__ __forceinline__ void short_forward(const Args& p, Bring bring) {
  constexpr int KS = DP / 16, NDB = DP / 32;
  constexpr uint32_t kBlock = 32 * DP * 2, kV = NB * kBlock, kBias = 2 * kV;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBias + NB * 128];
  const uint32_t l0 = LDS_ADDR(lds);
  float* bias = reinterpret_cast<float*>(lds + kBias);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t id = work_item(p);
  if (id >= p.total) return;
  const int split = id % (uint32_t)p.splits;
  const int bkv = id / (uint32_t)p.splits;
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;
  const int t_lo = split * p.per_split, t_hi = min(p.tiles, t_lo + p.per_split);

  const uint16_t* qb = p.q + b * p.qs.b + (int64_t)g * p.G * p.qs.h;
  auto load = [&](int t, uint4(&f)[KS]) __attribute__((always_inline)) {
    const int row = t * 128 + wave * 32 + col;
    const bool on = t < t_hi && row < p.rows;
    const uint32_t hg = fdiv(on ? row : 0, p.by_lq), tok = (on ? row : 0) - hg * p.Lq;
    load_row<KS>(f, qb + (int64_t)tok * p.qs.l + hg * p.qs.h, on, h, p.D);
  };
  uint4 qf[KS];
  load(t_lo, qf);
  const uint32_t act = bring(b, g, l0, l0 + kV, bias, tid, wave, lane);
  const RowAt<DP> row_at(lane, l0);
  const TrAt<DP, NDB> tr_at(lane, l0);
  const uint32_t bias_at = opaque(l0 + kBias + 16 * h);

  for (int t = t_lo; t < t_hi; ++t) {
    v16f s[NB];
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if ((act >> i) & 1) {
        s[i] = start_at(bias_at + 128 * i);
#pragma unroll
        for (int k = 0; k < KS; ++k) s[i] = T::mfma(row_at.get(k, kBlock * i), qf[k], s[i]);
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, s[i][r]);
      }
    load(t + 1, qf);
    m = max_halves(m) * p.c2;
    const float ms = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f;
    v16f o[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d) o[d] = zero16();
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if ((act >> i) & 1) {
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          uint32_t pk[4];
#pragma unroll
          for (int r = 0; r < 8; r += 2) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][8 * s2 + r], p.c2, -ms));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][8 * s2 + r + 1], p.c2, -ms));
            l += e0 + e1;
            pk[r / 2] = T::pack(e0, e1);
          }
          const uint4 pf = {pk[0], pk[1], pk[2], pk[3]};
#pragma unroll
          for (int d = 0; d < NDB; ++d)
            o[d] = T::mfma(tr_at.get(d, kV + kBlock * i + kBlock / 2 * s2), pf, o[d]);
        }
      }
    l = sum_halves(l);
    const int row = t * 128 + wave * 32 + col;
    const bool on = row < p.rows;
    const uint32_t hg = fdiv(on ? row : 0, p.by_lq), tok = (on ? row : 0) - hg * p.Lq;
    const int head = g * p.G + hg;
    if (on && h == 0) p.lse[((int64_t)b * p.H + head) * p.Lq + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    store_row<T>(p.out + (((int64_t)b * p.Lq + tok) * p.H + head) * p.D, on, o, l == 0.f ? 0.f : 1.f / l, h, p.D);
  }
}

}  // namespace xattn
}  // namespace dpa
