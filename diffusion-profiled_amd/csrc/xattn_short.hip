// Cross attention over up to 128 keys (a prompt's 77 tokens): a workgroup keeps a key/value head's
// keys in LDS and walks over its query rows, so that a row's scores are all in registers at once.
// The forward needs no running maximum; the backward forms D = rowsum(P dP) from its own fp32 P and
// dP (it reads no output of the forward but lse) and all three gradients in one pass over q and dO.
#include <type_traits>

#include "xattn.hpp"

namespace dpa {
namespace xattn {

// Brings the head's keys and values to kl and vl (rows of NB x 32 keys) and its bias (0: visible,
// -inf: not) and gives which blocks of 32 keys have a visible one. Ends with a barrier.
template <int DP, int NB>
__device__ __forceinline__ uint32_t resident_keys(const Args& p, int b, int g, uint32_t kl, uint32_t vl,
                                                  float* bias, int tid, int wave, int lane) {
  constexpr int NG = DP / 8;
  const int klen = keys_of(p, b);
  const uint8_t* mb = p.kmask ? p.kmask + b * p.mask_b : nullptr;
  auto visible = [&](int key) __attribute__((always_inline)) { return key < klen && (!mb || mb[key] != 0); };
  const uint16_t* kb = p.k + b * p.ks.b + g * p.ks.h;
  const uint16_t* vb = p.v + b * p.vs.b + g * p.vs.h;
  for (int c0 = wave * 64; c0 < NB * 32 * NG; c0 += 256) {
    const bool vis = visible((c0 + lane) / NG);
    dma_rows<DP>(kl, c0, lane, p.D, [&](int row) __attribute__((always_inline)) {
      return vis ? kb + row * p.ks.l : static_cast<const uint16_t*>(nullptr);
    });
    dma_rows<DP>(vl, c0, lane, p.D, [&](int row) __attribute__((always_inline)) {
      return vis ? vb + row * p.vs.l : static_cast<const uint16_t*>(nullptr);
    });
  }
  if (tid < NB * 32) bias[tid] = visible(tid) ? 0.f : -__builtin_inff();
  wait_vmcnt<0>();
  wait_lgkmcnt0();
  lds_barrier();
  uint32_t act = 0;
#pragma unroll
  for (int i = 0; i < NB; ++i) act |= (__ballot(bias[32 * i + (lane & 31)] == 0.f) ? 1u : 0u) << i;
  return act;
}

// |x|^2 of 8 elements added to n
template <class T>
__device__ __forceinline__ float length2(uint4 x, float n) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    n = __builtin_fmaf(T::lo(w[i]), T::lo(w[i]), n);
    n = __builtin_fmaf(T::hi(w[i]), T::hi(w[i]), n);
  }
  return n;
}
// (a row that is not finite takes no part in a maximum: its dS is not finite either)
__device__ __forceinline__ float finite(float n) { return n < __builtin_inff() ? n : 0.f; }

// ---------------------------------------------------------------------------------------
// Forward: four waves, each with its own 32 rows of every tile of 128; the next tile's queries load
// while this one's are at work. Layouts and products as in xattn_fwd.hip.
// Bound by HBM, less what a workgroup of few tiles leaves bare at its ends: 128 x 256 queries of 4 heads of
// 64 dims over up to 77 keys 12.4 us (3.3 TB/s), 128 x 1024 of 32 dims 19.5 (3.7).
// ---------------------------------------------------------------------------------------
template <class T, int DP, int NB>
__global__ __launch_bounds__(256, DP == 128 ? 2 : DP == 64 ? 3 : 4) void xattn_short_fwd_kernel(const Args p) {
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
  const uint32_t act = resident_keys<DP, NB>(p, b, g, l0, l0 + kV, bias, tid, wave, lane);
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

// ---------------------------------------------------------------------------------------
// Backward. Per tile of 128 rows, each wave forms S^T and dP^T of its 32 rows over all keys, D from
// them, and per block of 32 keys P, dS and its part of dQ^T += K^T dS^T, all with a row in each lane
// column. dK and dV sum over rows, which those layouts hold across lanes: the block's P and dS go
// through LDS as rows of 32 keys, and each wave forms one 32 x 32 tile (or two) of dK^T = Q^T dS or
// dV^T = dO^T P of the block over the tile's 128 rows, both operands by transpose reads. Without
// kKeys only dQ is formed (the same bits).
// The scores of all keys in registers leave two waves a SIMD (one of 128 dims), which bounds it, by LDS and
// vector work in turn: the above shapes 22.1 us (3.5 TB/s) and 37.8 (2.8). Rows of P and dS laid 8 B askew
// against their writes' conflicts: no more than 1 %.
// ---------------------------------------------------------------------------------------
template <class T, int DP, int NB, bool kKeys>
__global__ __launch_bounds__(256, DP == 128 ? 1 : 2) void xattn_short_bwd_kernel(const Args p) {
  constexpr int KS = DP / 16, NDB = DP / 32;
  constexpr int NT = DP == 128 ? 2 : 1;  // tiles of a wave per block
  constexpr float kUnshift = 1.f / (1 << T::kShift);
  // LDS: keys, values, their bias; dS and P of a block (rows of 32 keys); Q and dO of the tile
  constexpr uint32_t kBlock = 32 * DP * 2, kV = NB * kBlock, kBias = 2 * kV, kPS = kBias + 1024;
  constexpr uint32_t kQG = kPS + 2 * 128 * 64, kTile = 128 * DP * 2;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kKeys ? kQG + 2 * kTile : kPS];
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
  const uint16_t* gb = p.dout + b * p.gs.b + (int64_t)g * p.G * p.gs.h;
  const float* lb = p.lse + ((int64_t)b * p.H + g * p.G) * p.Lq;  // (the rows of g in order)
  uint4 qf[KS], gf[KS];
  float lse = -__builtin_inff();
  auto load = [&](int t) __attribute__((always_inline)) {
    const int row = t * 128 + wave * 32 + col;
    const bool on = t < t_hi && row < p.rows;
    const uint32_t hg = fdiv(on ? row : 0, p.by_lq), tok = (on ? row : 0) - hg * p.Lq;
    load_row<KS>(qf, qb + (int64_t)tok * p.qs.l + hg * p.qs.h, on, h, p.D);
    load_row<KS>(gf, gb + (int64_t)tok * p.gs.l + hg * p.gs.h, on, h, p.D);
    lse = -__builtin_inff();
    if (on) lse = lb[row];
  };
  load(t_lo);
  const uint32_t act = resident_keys<DP, NB>(p, b, g, l0, l0 + kV, bias, tid, wave, lane);
  const RowAt<DP> row_at(lane, l0);
  const TrAt<DP, NDB> tr_at(lane, l0);
  const uint32_t bias_at = opaque(l0 + kBias + 16 * h);

  // this wave's tiles: of dK (mat 0) or dV, dims 32 (db0 + 2 j); with one block of dims, rows
  // 64 part .. 64 part + 63 of each tile
  const int mat = wave & 1, db0 = DP == 32 ? 0 : wave >> 1, part = DP == 32 ? wave >> 1 : 0;
  constexpr int kSteps = DP == 32 ? 4 : 8;
  v16f acc[NB][NT];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = zero16();

  const int mine = wave * 32 + col;  // row of the tile
  const uint32_t my_rows = kQG + wave * kBlock;
  uint32_t ps_at[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) ps_at[x] = opaque(l0 + kPS + wave * 2048 + col * 64 + ((x ^ swz<32>(col)) << 4) + 8 * h);
  const TrAt<32, 1> ps_tr(lane, l0 + kPS + mat * 8192 + part * 4096);
  const TrAt<DP, NT> qg_tr(lane, l0 + kQG + mat * kTile + part * 2 * kBlock, db0, 2);

  // dS's scale 2^-down with T::kScaled (the workgroup's, as its sums over rows are): |dP - D| <=
  // 2 max |v| max |dO|, lengths of the rows of the tiles so far, so that 2^(kShift - down) dS is at most
  // 2^15. It moves one way only. The waves leave their parts of the maxima in LDS. (fp16, one
  // barrier a tile more: 128 x 256 queries of 64 dims over 77 keys 24.2 -> 25.6 us, 512 x 1 80 -> 88.)
  int down = 0;
  float* most = bias + 128;  // [2: tile t & 1][4 waves] of |dO|^2, then [4] of |v|^2
  if constexpr (T::kScaled) {
    float n = 0.f;  // (of 8 dims: a row's is at most DP / 8 times the largest)
#pragma unroll
    for (uint32_t at = 0; at < kV; at += 4096)
      if (at + tid * 16 < kV) n = fmaxf(n, finite(length2<T>(__builtin_bit_cast(uint4, lds_ld16(l0 + kV + at + tid * 16)), 0.f)));
    n = wave_max(n) * (DP / 8);
    if (lane == 0) most[8 + wave] = n;
  }
  // one tile over the first N blocks of keys
  auto tile = [&](int t, auto blocks) __attribute__((always_inline)) {
    constexpr int N = decltype(blocks)::value;
    v16f dq[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d) dq[d] = zero16();
    if constexpr (N == 0) {
      load(t + 1);
    } else {
#pragma unroll
      for (int k = 0; kKeys && k < KS; ++k) {  // (every wave is past its reads of the last tile)
        lds_st16(row_at.a[k] + my_rows, qf[k]);
        lds_st16(row_at.a[k] + my_rows + kTile, gf[k]);
      }
      const float nlse2 = lse == -__builtin_inff() ? -__builtin_inff() : (float)T::kShift - lse * kLog2e;
      if constexpr (T::kScaled) {  // (before the scores: they fill the registers)
        float n = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) n = length2<T>(gf[k], n);
        n = wave_max(finite(sum_halves(n)));
        if (lane == 0) most[4 * (t & 1) + wave] = n;
        wait_lgkmcnt0();
        lds_barrier();
        const float* g = most + 4 * (t & 1);
        const float n2 = fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3])) *
                         fmaxf(fmaxf(most[8], most[9]), fmaxf(most[10], most[11]));
        // (n2 < 2^frexp, so max |v| max |dO| < 2^half of it, rounded up; 0 gives 2^0)
        const int ex = __builtin_amdgcn_readfirstlane((__builtin_amdgcn_frexp_expf(n2) + 1) >> 1);
        if (t == t_lo) {
          down = ex;
        } else if (ex > down) {
          if (mat == 0) {
            const float f = ldexpf(1.f, down - ex);
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] *= f;
          }
          down = ex;
        }
      }
      const float up = T::kScaled ? ldexpf(1.f, -down) : 1.f;
      v16f s[N], dp[N];  // (s: then P)
      float nd = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[i] = start_at(bias_at + 128 * i);
        dp[i] = zero16();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          s[i] = T::mfma(row_at.get(k, kBlock * i), qf[k], s[i]);
          dp[i] = T::mfma(row_at.get(k, kV + kBlock * i), gf[k], dp[i]);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], p.c2, nlse2));
          nd = __builtin_fmaf(-s[i][r], dp[i][r], nd);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (DP == 32) load(t + 1);
      nd = sum_halves(nd) * (T::kScaled ? kUnshift * up : kUnshift);
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          uint32_t pw[4], sw[4];
#pragma unroll
          for (int r = 0; r < 8; r += 2) {
            const float p0 = s[i][8 * s2 + r], p1 = s[i][8 * s2 + r + 1];
            pw[r / 2] = T::pack(p0, p1);
            const float d0 = dp[i][8 * s2 + r], d1 = dp[i][8 * s2 + r + 1];
            if constexpr (T::kScaled)
              sw[r / 2] = T::pack(p0 * __builtin_fmaf(d0, up, nd), p1 * __builtin_fmaf(d1, up, nd));
            else
              sw[r / 2] = T::pack(p0 * (d0 + nd), p1 * (d1 + nd));
          }
#pragma unroll
          for (int x = 0; kKeys && x < 2; ++x) {
            const uint32_t at = ps_at[2 * s2 + x];
            lds_st8(at, sw[2 * x], sw[2 * x + 1]);
            lds_st8(at + 8192, pw[2 * x], pw[2 * x + 1]);
          }
          const uint4 sf = {sw[0], sw[1], sw[2], sw[3]};
#pragma unroll
          for (int d = 0; d < NDB; ++d) dq[d] = T::mfma(tr_at.get(d, kBlock * i + kBlock / 2 * s2), sf, dq[d]);
        }
        if constexpr (kKeys) {
          wait_lgkmcnt0();
          lds_barrier();  // the block's P and dS (and the tile's Q and dO) are there
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const uint4 x = ps_tr.get(0, 1024 * k);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = T::mfma(qg_tr.get(j, kBlock / 2 * k), x, acc[i][j]);
          }
          wait_lgkmcnt0();
          lds_barrier();  // and read
        }
        if (DP != 32 && i == 0) load(t + 1);  // (no sooner: the registers that they need are the scores')
      }
    }
    const int row = t * 128 + mine;
    const bool on = row < p.rows;
    const uint32_t hg = fdiv(on ? row : 0, p.by_lq), tok = (on ? row : 0) - hg * p.Lq;
    store_row<T>(p.dq + (((int64_t)b * p.Lq + tok) * p.H + g * p.G + hg) * p.D, on, dq,
                 T::kScaled ? p.scale * ldexpf(kUnshift, down) : p.scale * kUnshift, h, p.D);
  };
  // (a loop for each number of blocks up to the last with a visible key)
  auto walk = [&](auto blocks) __attribute__((always_inline)) {
    for (int t = t_lo; t < t_hi; ++t) tile(t, blocks);
  };
  if (act >= 1u << (NB - 1)) walk(std::integral_constant<int, NB>());
  else if (NB == 4 && act >= 4) walk(std::integral_constant<int, 3>());
  else if (act >= 2) walk(std::integral_constant<int, 2>());
  else if (act) walk(std::integral_constant<int, 1>());
  else walk(std::integral_constant<int, 0>());

  if constexpr (!kKeys) return;
  const int64_t n = (int64_t)p.B * p.KVH * p.Lk;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    if constexpr (DP == 32) {  // the two halves of the rows
      float* x = reinterpret_cast<float*>(lds + kQG) + mat * 1024 + lane;
      static_assert(2 * kTile >= 2 * 1024 * 4, "the tiles fit");
      __syncthreads();
      if (part)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[64 * r] = acc[i][0][r];
      __syncthreads();
      if (part) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][0][r] += x[64 * r];
    }
    const int key = 32 * i + col;
    const bool on = key < p.Lk;
    const bool vis = bias[key] == 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int dim = 32 * (db0 + 2 * j);
      v16f a[1] = {vis ? acc[i][j] : zero16()};
      if (T::kScaled && mat == 0)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[0][r] *= ldexpf(kUnshift, down);
      if (p.splits > 1) {
        const int64_t at = (split * 2 + mat) * n + (int64_t)bkv * p.Lk + key;
        if (on) store_part(p.part + at * p.D + dim, a, h, p.D - dim);
      } else {
        uint16_t* dst = mat == 0 ? p.dk + b * p.dks.b + key * p.dks.l + g * p.dks.h
                                 : p.dv + b * p.dvs.b + key * p.dvs.l + g * p.dvs.h;
        const float f = mat == 0 ? T::kScaled ? p.scale : p.scale * kUnshift : kUnshift;
        store_row<T>(dst + dim, on, a, f, h, p.D - dim);
      }
    }
  }
}

// Up to 96 keys are three blocks of 32 in registers and LDS, more are four. (77 keys as four: 128 x 256
// queries of 64 dims forward 14.5 us for 13.0, backward 30.6 for 23.9; 128 x 1024 of 32 dims 21.1 for 20.8
// and 40.8 for 39.7.)
template <class T, int DP>
static int launch_short_fwd(const Args& p, hipStream_t s) {
  if (p.Lk <= 96) xattn_short_fwd_kernel<T, DP, 3><<<p.grid, 256, 0, s>>>(p);
  else xattn_short_fwd_kernel<T, DP, 4><<<p.grid, 256, 0, s>>>(p);
  return launch_status();
}

template <class T>
static int run_short_fwd(const Args& p, hipStream_t s) {
  switch (dim_pad(p.D)) {
    case 32: return launch_short_fwd<T, 32>(p, s);
    case 64: return launch_short_fwd<T, 64>(p, s);
    default: return launch_short_fwd<T, 128>(p, s);
  }
}

int short_fwd(const Args& p, int dtype, hipStream_t s) {
  return dtype == DPA_DTYPE_BF16 ? run_short_fwd<Bf16>(p, s) : run_short_fwd<F16>(p, s);
}

template <class T, int DP, int NB>
static int launch_short_bwd(const Args& p, hipStream_t s) {
  if (p.dk) xattn_short_bwd_kernel<T, DP, NB, true><<<p.grid, 256, 0, s>>>(p);
  else xattn_short_bwd_kernel<T, DP, NB, false><<<p.grid, 256, 0, s>>>(p);
  return launch_status();
}

template <class T>
static int run_short_bwd(const Args& p, hipStream_t s) {
  switch (dim_pad(p.D)) {
    case 32: return p.Lk <= 96 ? launch_short_bwd<T, 32, 3>(p, s) : launch_short_bwd<T, 32, 4>(p, s);
    case 64: return p.Lk <= 96 ? launch_short_bwd<T, 64, 3>(p, s) : launch_short_bwd<T, 64, 4>(p, s);
    default: return p.Lk <= 96 ? launch_short_bwd<T, 128, 3>(p, s) : launch_short_bwd<T, 128, 4>(p, s);
  }
}

int short_bwd(const Args& p, int dtype, hipStream_t s) {
  return dtype == DPA_DTYPE_BF16 ? run_short_bwd<Bf16>(p, s) : run_short_bwd<F16>(p, s);
}

}  // namespace xattn
}  // namespace dpa
