// Cross attention, backward. With P recomputed from the saved lse and D = rowsum(dO O):
//   dP = dO V^T, dS = P (dP - D), dQ = c dS K, dK = c dS^T Q, dV = P^T dO.
// Two kernels, each recomputing S and dP, so that every gradient has one writer and a fixed order
// of sums: one of query rows (dQ, and D for the other), one of keys (dK, dV, summed over the query
// heads that share them).
#include <type_traits>

#include "xattn.hpp"

namespace dpa {
namespace xattn {

// ---------------------------------------------------------------------------------------
// dQ: the forward's tiles and layouts (S^T = K Q^T, dP^T = V dO^T: a query per lane column), then
// dQ^T += K^T dS^T from transpose reads of the key rows. The product for dP^T starts from -D, as the
// one for S^T from the keys' bias, so that dS = P (dP - D) is one multiplication.
// Bound as the forward is, with three products to an exponential: bf16, 8 x 4096 queries of 8 heads of 64
// dims over 1024 keys 132 us, 780 TFLOP/s, MFMA 50 % busy.
// ---------------------------------------------------------------------------------------

// What the kernels of dQ keep of a lane's query row: q and dO as B operands, kShift - lse in base 2
// and -D, which they leave for the kernel of dK and dV (leave: this wave does). D is formed from O as it was
// rounded, half a step off per dim: the fp32 P and dP that it could be summed from pass only later, tile by
// tile, and one more pass over the keys to get it would cost as much as dQ's.
template <class T, int KS>
struct QueryRow {
  uint4 qf[KS], gf[KS];
  float nlse2, nd;
  int64_t orow;
  __device__ __forceinline__ QueryRow(const Args& p, int b, int g, int bkv, int row, bool leave, int h) {
    const bool on = row < p.rows;
    const uint32_t hg = fdiv(on ? row : 0, p.by_lq), tok = (on ? row : 0) - hg * p.Lq;
    const int head = g * p.G + hg;
    orow = ((int64_t)b * p.Lq + tok) * p.H + head;
    uint4 of[KS];
    load_row<KS>(qf, p.q + b * p.qs.b + (int64_t)tok * p.qs.l + head * p.qs.h, on, h, p.D);
    load_row<KS>(gf, p.dout + b * p.gs.b + (int64_t)tok * p.gs.l + head * p.gs.h, on, h, p.D);
    load_row<KS>(of, p.out + orow * p.D, on, h, p.D);
    nlse2 = -__builtin_inff(), nd = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t gw[4] = {gf[ks].x, gf[ks].y, gf[ks].z, gf[ks].w};
      const uint32_t ow[4] = {of[ks].x, of[ks].y, of[ks].z, of[ks].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        nd = __builtin_fmaf(-T::lo(gw[i]), T::lo(ow[i]), nd);
        nd = __builtin_fmaf(-T::hi(gw[i]), T::hi(ow[i]), nd);
      }
    }
    if (on) {
      const float e = p.lse[((int64_t)b * p.H + head) * p.Lq + tok];
      nlse2 = e == -__builtin_inff() ? -__builtin_inff() : (float)T::kShift - e * kLog2e;
    }
    nd = sum_halves(nd);
    if (on && leave && h == 0) {
      const int64_t all = (int64_t)p.B * p.KVH * p.rows, at = (int64_t)bkv * p.rows + row;
      p.row_stat[at] = nlse2;
      p.row_stat[all + at] = nd;
    }
  }
};

template <int NDB>
__device__ __forceinline__ void times(v16f (&x)[NDB], float f) {
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[d][r] *= f;
}

// Moves dS's scale, dq's with it, for these values of dP - D. The scale is part of P's exponent, in nlse2.
template <int NDB>
__device__ __forceinline__ void follow(DsScale& ds, const v16f& dp, v16f (&dq)[NDB], float& nlse2) {
  const float top = DsScale::largest(dp);
  if (!__any(ds.passes(top))) return;
  const int by = ds.move(max_halves(top));
  times(dq, ldexpf(1.f, by));
  nlse2 += (float)by;
}

// Four waves of 32 query rows each share tiles of 64 keys.
template <class T, int DP>
__global__ __launch_bounds__(256, DP == 128 ? 2 : DP == 64 ? 3 : 4) void xattn_dq_kernel(const Args p) {
  constexpr int KT = 64;
  constexpr int KS = DP / 16, NDB = DP / 32;
  constexpr float kUnshift = 1.f / (1 << T::kShift);
  constexpr uint32_t kBytes = KT * DP * 2, kBias = 4 * kBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBias + 2 * KT * 4];
  __shared__ uint32_t seen[kMaxRange / 32];
  const uint32_t l0 = LDS_ADDR(lds);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t id = work_item(p);
  if (id >= p.total) return;
  const int split = id % (uint32_t)p.splits;
  const uint32_t bt = id / (uint32_t)p.splits;
  const int tile = bt % (uint32_t)p.tiles;
  const int bkv = bt / (uint32_t)p.tiles;
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;

  const int klen = __builtin_amdgcn_readfirstlane(keys_of(p, b));
  const int nt = (klen + KT - 1) / KT;
  const int t_lo = split * p.per_split;
  int t_hi = split + 1 == p.splits ? nt : min(nt, (split + 1) * p.per_split);
  const KeyBits bits(p, b, klen, split * p.per_split * KT, t_hi * KT, seen, tid);
  t_hi = bits.tiles_to<KT>(t_hi);
  const KeyTiles<DP> keys(p, b, g, klen, l0, wave, lane);
  auto fetch = [&](int t, int buf, uint64_t word) __attribute__((always_inline)) {
    keys.fetch(t, buf, word);
    if (wave == 0)
      *reinterpret_cast<float*>(lds + kBias + buf * KT * 4 + lane * 4) = (word >> lane) & 1 ? 0.f : -__builtin_inff();
  };
  uint64_t word = 0;
  if (t_lo < t_hi) {
    word = bits.template word<KT>(t_lo);
    fetch(t_lo, 0, word);
  }

  const int row = tile * 128 + wave * 32 + col;
  const QueryRow<T, KS> q(p, b, g, bkv, row, split == 0, h);
  const RowAt<DP> row_at(lane, l0);
  const TrAt<DP, NDB> tr_at(lane, l0);
  const uint32_t bias_at = opaque(l0 + kBias + 16 * h);
  wait_vmcnt<0>();

  v16f dq[NDB], nd16;
#pragma unroll
  for (int i = 0; i < NDB; ++i) dq[i] = zero16();
#pragma unroll
  for (int r = 0; r < 16; ++r) nd16[r] = q.nd;
  DsScale ds;
  float nlse2 = T::kScaled ? q.nlse2 + DsScale::kFirst : q.nlse2;

  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    uint64_t word_next = 0;
    wait_vmcnt<0>();
    keys.ready(t, buf, word);
    wait_lgkmcnt0();
    lds_barrier();
    if (t + 1 < t_hi) {
      word_next = bits.template word<KT>(t + 1);
      fetch(t + 1, buf ^ 1, word_next);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!(uint32_t)(word >> (32 * i))) continue;
      constexpr uint32_t at = buf * 2 * kBytes;
      v16f s = start_at(bias_at + buf * KT * 4 + 128 * i), dp = nd16;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        s = T::mfma(row_at.get(k, at + kBytes / 2 * i), q.qf[k], s);
        dp = T::mfma(row_at.get(k, at + kBytes + kBytes / 2 * i), q.gf[k], dp);
      }
      if constexpr (T::kScaled) follow(ds, dp, dq, nlse2);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        uint32_t sw[4];
#pragma unroll
        for (int r = 8 * s2; r < 8 * s2 + 8; r += 2) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c2, nlse2));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], p.c2, nlse2));
          sw[(r & 7) / 2] = T::pack(p0 * dp[r], p1 * dp[r + 1]);
        }
        const uint4 sf = {sw[0], sw[1], sw[2], sw[3]};
#pragma unroll
        for (int d = 0; d < NDB; ++d) dq[d] = T::mfma(tr_at.get(d, at + kBytes / 2 * i + kBytes / 4 * s2), sf, dq[d]);
      }
    }
    word = word_next;
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = t_lo; t < t_hi; t += 2) {
    step(t, std::integral_constant<int, 0>());
    if (t + 1 < t_hi) step(t + 1, std::integral_constant<int, 1>());
  }

  const bool has_row = row < p.rows;
  if constexpr (T::kScaled) times(dq, kUnshift / ds.up);
  if (p.splits > 1) {
    if (has_row) store_part(p.part + (((int64_t)split * p.B * p.KVH + bkv) * p.rows + row) * p.D, dq, h, p.D);
    return;
  }
  store_row<T>(p.dq + q.orow * p.D, has_row, dq, T::kScaled ? p.scale : p.scale * kUnshift, h, p.D);
}

// Up to 32 rows: the four waves share them and take every fourth tile of 32 keys each.
template <class T, int DP>
__global__ __launch_bounds__(256, 1) void xattn_dq_few_kernel(const Args p) {
  constexpr int KT = 32;
  constexpr int NG = DP / 8, KS = DP / 16, NDB = DP / 32;
  constexpr float kUnshift = 1.f / (1 << T::kShift);
  constexpr int kXfer = KT * NG / 64;
  __shared__ __attribute__((aligned(1024))) uint16_t kv[4][2][2][KT * DP];
  __shared__ __attribute__((aligned(16))) float bias[4][2][KT];
  __shared__ uint32_t seen[kMaxRange / 32];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t id = work_item(p);
  if (id >= p.total) return;
  const int split = id % (uint32_t)p.splits;
  const int bkv = id / (uint32_t)p.splits;
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;

  const int klen = keys_of(p, b);
  const int nt = (klen + KT - 1) / KT;
  const int t_lo = split * p.per_split + wave;
  int t_hi = split + 1 == p.splits ? nt : min(nt, (split + 1) * p.per_split);
  const uint16_t* kb = p.k + b * p.ks.b + g * p.ks.h;
  const uint16_t* vb = p.v + b * p.vs.b + g * p.vs.h;
  const KeyBits bits(p, b, klen, split * p.per_split * KT, t_hi * KT, seen, tid);
  t_hi = bits.tiles_to<KT>(t_hi);
  auto fetch = [&](int t, int buf, uint32_t word) __attribute__((always_inline)) {
    fetch_keys<DP, kXfer, 64>(p, kb, vb, (int64_t)t * KT, word, kv[wave][buf][0], kv[wave][buf][1], 0, lane);
    if (h == 0) bias[wave][buf][col] = (word >> col) & 1 ? 0.f : -__builtin_inff();
  };
  uint32_t word = 0;
  if (t_lo < t_hi) {
    word = (uint32_t)bits.template word<KT>(t_lo);
    fetch(t_lo, 0, word);
  }
  const int row = col;
  const QueryRow<T, KS> q(p, b, g, bkv, row, split == 0 && wave == 0, h);
  wait_vmcnt<0>();

  v16f dq[NDB], nd16;
#pragma unroll
  for (int i = 0; i < NDB; ++i) dq[i] = zero16();
#pragma unroll
  for (int r = 0; r < 16; ++r) nd16[r] = q.nd;
  DsScale ds;
  float nlse2 = T::kScaled ? q.nlse2 + DsScale::kFirst : q.nlse2;

  for (int t = t_lo, buf = 0; t < t_hi; t += 4, buf ^= 1) {
    uint32_t word_next = 0;
    wait_lgkmcnt0();
    asm volatile("" ::: "memory");
    if (t + 4 < t_hi) {
      word_next = (uint32_t)bits.template word<KT>(t + 4);
      fetch(t + 4, buf ^ 1, word_next);
      wait_vmcnt<2 * kXfer>();
    } else {
      wait_vmcnt<0>();
    }
    asm volatile("" ::: "memory");
    if (word) {
      const uint16_t *kr = kv[wave][buf][0], *vr = kv[wave][buf][1];
      v16f s = start_from(bias[wave][buf], h), dp = nd16;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        s = T::mfma(frag_row<DP>(kr, col, 2 * k + h), q.qf[k], s);
        dp = T::mfma(frag_row<DP>(vr, col, 2 * k + h), q.gf[k], dp);
      }
      if constexpr (T::kScaled) follow(ds, dp, dq, nlse2);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        uint32_t sw[4];
#pragma unroll
        for (int r = 8 * s2; r < 8 * s2 + 8; r += 2) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c2, nlse2));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], p.c2, nlse2));
          sw[(r & 7) / 2] = T::pack(p0 * dp[r], p1 * dp[r + 1]);
        }
        const uint4 sf = {sw[0], sw[1], sw[2], sw[3]};
#pragma unroll
        for (int d = 0; d < NDB; ++d) dq[d] = T::mfma(frag_tr<DP>(kr, 16 * s2, d, lane), sf, dq[d]);
      }
    }
    word = word_next;
    __builtin_amdgcn_sched_barrier(0);
  }

  const float unscale = T::kScaled ? p.scale : p.scale * kUnshift;
  if constexpr (T::kScaled) times(dq, kUnshift / ds.up);  // (each wave has its own)
  __syncthreads();
  float* ox = reinterpret_cast<float*>(&kv[0][0][0][0]);  // [4][DP][32]
  static_assert(sizeof(kv) >= 4 * DP * 32 * 4, "the waves' dQ fit the buffers");
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      ox[(wave * DP + 32 * d + 8 * (r / 4) + 4 * h + r % 4) * 32 + col] = dq[d][r];
  __syncthreads();
  constexpr int ND = DP / 8;
  const int q8 = tid >> 5;
  if (row >= p.rows) return;
#pragma unroll
  for (int i = 0; i < ND; i += 4) {
    float a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) a[j] += ox[(w * DP + q8 * ND + i + j) * 32 + col];
    }
    const int dim = q8 * ND + i;
    if (dim >= p.D) continue;
    if (p.splits > 1)
      *reinterpret_cast<float4*>(p.part + (((int64_t)split * p.B * p.KVH + bkv) * p.rows + row) * p.D + dim) =
          float4{a[0], a[1], a[2], a[3]};
    else
      *reinterpret_cast<uint2*>(p.dq + q.orow * p.D + dim) =
          uint2{T::pack(a[0] * unscale, a[1] * unscale), T::pack(a[2] * unscale, a[3] * unscale)};
  }
}

// ---------------------------------------------------------------------------------------
// dK, dV: a workgroup's waves take 32 keys each (their K and V rows as B operands and the two
// accumulators in registers); tiles of 64 query rows, with their dO, lse and D, pass through LDS.
// S = Q K^T and dP = dO V^T put a key in each lane column, so P and dS are the B operands of
// dV^T += dO^T P and dK^T += Q^T dS, whose A operands are transpose reads of the same rows.
// KB = 4: four blocks of keys. KB = 2: two, each of two waves with 32 rows of every tile, which join
// in LDS at the end: twice the workgroups, for when there are few, and registers for two of 128 dims
// to a CU.
// Keys are resident and rows pass because dK and dV are the two sums: four products to an exponential and
// nothing but their operands through LDS. bf16, 8 x 4096 queries of 8 heads of 64 dims over 1024 keys 194
// us (KB = 2), 707 TFLOP/s, MFMA 39 % busy. At 128 dims a block's operands pass through LDS (32 KB a wave) in
// as many cycles as its products take.
// ---------------------------------------------------------------------------------------
static __device__ float g_pad_stat[2] = {-__builtin_inff(), 0.f};

template <class T, int DP, int KB>
__global__ __launch_bounds__(256, DP == 128 ? 2 : DP == 64 ? 3 : 4) void xattn_dkdv_kernel(const Args p) {
  constexpr int NG = DP / 8, KS = DP / 16, NDB = DP / 32;
  constexpr float kUnshift = 1.f / (1 << T::kShift);
  constexpr int kXfer = kQT * NG / 256;
  constexpr uint32_t kBytes = kQT * DP * 2, kStat = 4 * kBytes;  // [2][Q, dO], [2][-lse, -D]
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kStat + 4 * kQT * 4];
  const uint32_t l0 = LDS_ADDR(lds);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t id = work_item(p);
  if (id >= p.total) return;
  const int split = id % (uint32_t)p.splits;
  const uint32_t bt = id / (uint32_t)p.splits;
  const int tile = bt % (uint32_t)p.tiles;
  const int bkv = bt / (uint32_t)p.tiles;
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;

  const int klen = keys_of(p, b);
  const int key = tile * 32 * KB + wave % KB * 32 + col;
  const bool vis = key < klen && (!p.kmask || p.kmask[b * p.mask_b + key] != 0);
  const bool any_vis = __any(vis);  // (wave-uniform)
  uint4 kf[KS], vf[KS];
  load_row<KS>(kf, p.k + b * p.ks.b + key * p.ks.l + g * p.ks.h, vis, h, p.D);
  load_row<KS>(vf, p.v + b * p.vs.b + key * p.vs.l + g * p.vs.h, vis, h, p.D);
  const bool wg_vis = __syncthreads_or(vis);
  const int nt = wg_vis ? (p.rows + kQT - 1) / kQT : 0;
  const int t_lo = split * p.per_split;
  const int t_hi = split + 1 == p.splits ? nt : min(nt, (split + 1) * p.per_split);

  const uint16_t* qb = p.q + b * p.qs.b + (int64_t)g * p.G * p.qs.h;
  const uint16_t* gb = p.dout + b * p.gs.b + (int64_t)g * p.G * p.gs.h;
  const float* sb = p.row_stat + (int64_t)bkv * p.rows;
  const int64_t all_rows = (int64_t)p.B * p.KVH * p.rows;
  // tiles of 64 rows of one head go by constant lane offsets, the others by an address per row
  const bool fast = p.D == DP && p.qs.l >= 0 && p.gs.l >= 0 && p.qs.l < (1 << 24) && p.gs.l < (1 << 24);
  constexpr int kRows = 256 / NG;  // from one transfer to the next (a multiple of the period of swz)
  const int c = wave * 64 + lane, row0 = c / NG, g8 = ((c % NG) ^ swz<DP>(row0)) << 3;
  const uint32_t qo = (uint32_t)(row0 * (int)p.qs.l + g8) * 2, go = (uint32_t)(row0 * (int)p.gs.l + g8) * 2;
  auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
    const int r0 = t * kQT;
    const uint32_t hg = fdiv(r0, p.by_lq), at = l0 + buf * 2 * kBytes;
    const int tok = r0 - hg * p.Lq;
    if (fast && tok + kQT <= p.Lq) {
      const uint16_t* qt = qb + (int64_t)tok * p.qs.l + hg * p.qs.h;
      const uint16_t* gt = gb + (int64_t)tok * p.gs.l + hg * p.gs.h;
#pragma unroll
      for (int r = 0; r < kXfer; ++r) {
        dma16_lds_from(qt + r * kRows * p.qs.l, qo, at + wave * 1024 + 4096 * r);
        dma16_lds_from(gt + r * kRows * p.gs.l, go, at + kBytes + wave * 1024 + 4096 * r);
      }
    } else {
#pragma unroll
      for (int r = 0; r < kXfer; ++r) {
        const int c0 = wave * 64 + 256 * r;
        const int row = r0 + (c0 + lane) / NG;
        const bool on = row < p.rows;
        const uint32_t hr = fdiv(on ? row : 0, p.by_lq), tr = (on ? row : 0) - hr * p.Lq;
        const uint16_t* qr = qb + (int64_t)tr * p.qs.l + hr * p.qs.h;
        const uint16_t* gr = gb + (int64_t)tr * p.gs.l + hr * p.gs.h;
        dma_rows<DP>(at, c0, lane, p.D,
                     [&](int) __attribute__((always_inline)) { return on ? qr : static_cast<const uint16_t*>(nullptr); });
        dma_rows<DP>(at + kBytes, c0, lane, p.D,
                     [&](int) __attribute__((always_inline)) { return on ? gr : static_cast<const uint16_t*>(nullptr); });
      }
    }
    if (wave < 2) {  // -lse (wave 0) and -D (wave 1)
      const int row = r0 + lane;
      const float* a = row < p.rows ? sb + wave * all_rows + row : g_pad_stat + wave;
      dma4_lds(a, l0 + kStat + (buf * 2 + wave) * kQT * 4);
    }
  };
  wait_vmcnt<0>();  // (no wait on keys and values inside the loop)
  if (t_lo < t_hi) fetch(t_lo, 0);

  const int r_lo = KB == 4 ? 0 : wave / KB;  // this wave's block of 32 rows, the first of its blocks
  const RowAt<DP> row_at(lane, l0 + r_lo * kBytes / 2);
  const TrAt<DP, NDB> tr_at(lane, l0 + r_lo * kBytes / 2);
  const uint32_t stat_at = opaque(l0 + kStat + r_lo * 128 + 16 * h);
  v16f dk[NDB], dv[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) dk[i] = dv[i] = zero16();
  DsScale ds;  // (of the wave's keys)
  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    wait_vmcnt<0>();
    lds_barrier();
    if (t + 1 < t_hi) fetch(t + 1, buf ^ 1);
    if (any_vis) {
#pragma unroll
      for (int i = 0; i < KB / 2; ++i) {
        constexpr uint32_t at0 = buf * 2 * kBytes, st0 = buf * 2 * kQT * 4;
        const uint32_t at = at0 + kBytes / 2 * i, st = st0 + 128 * i;
        v16f s = zero16(), dp = start_at(stat_at + st + kQT * 4);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          s = T::mfma(row_at.get(k, at), kf[k], s);
          dp = T::mfma(row_at.get(k, at + kBytes), vf[k], dp);
        }
        if constexpr (T::kScaled) {
          const float top = DsScale::largest(dp);
          if (__any(ds.passes(top))) times(dk, ldexpf(1.f, ds.move_wave(top)));
        }
        const v16f e = start_at(stat_at + st);
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          uint32_t pw[4], sw[4];
#pragma unroll
          for (int r = 8 * s2; r < 8 * s2 + 8; r += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c2, e[r]));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], p.c2, e[r + 1]));
            pw[(r & 7) / 2] = T::pack(p0, p1);
            if constexpr (T::kScaled)
              sw[(r & 7) / 2] = T::pack(p0 * (dp[r] * ds.up), p1 * (dp[r + 1] * ds.up));
            else
              sw[(r & 7) / 2] = T::pack(p0 * dp[r], p1 * dp[r + 1]);
          }
          const uint4 pf = {pw[0], pw[1], pw[2], pw[3]}, sf = {sw[0], sw[1], sw[2], sw[3]};
#pragma unroll
          for (int d = 0; d < NDB; ++d) {
            dv[d] = T::mfma(tr_at.get(d, at + kBytes + kBytes / 4 * s2), pf, dv[d]);
            dk[d] = T::mfma(tr_at.get(d, at + kBytes / 4 * s2), sf, dk[d]);
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = t_lo; t < t_hi; t += 2) {
    step(t, std::integral_constant<int, 0>());
    if (t + 1 < t_hi) step(t + 1, std::integral_constant<int, 1>());
  }

  if constexpr (T::kScaled) times(dk, kUnshift / ds.up);
  if constexpr (KB == 2) {
    __syncthreads();
    float* x = reinterpret_cast<float*>(lds) + wave % KB * (2 * NDB * 1024) + lane;
    static_assert(KB * 2 * NDB * 1024 * 4 <= 4 * kBytes, "two waves' sums fit the buffers");
    if (wave >= KB) {
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[(d * 32 + r) * 64] = dk[d][r];
          x[(d * 32 + 16 + r) * 64] = dv[d][r];
        }
    }
    __syncthreads();
    if (wave >= KB) return;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dk[d][r] += x[(d * 32 + r) * 64];
        dv[d][r] += x[(d * 32 + 16 + r) * 64];
      }
  }
  const bool on = key < p.Lk;
  if (!vis) {  // (in the products an invisible key's column holds what a key of zeros would get)
#pragma unroll
    for (int i = 0; i < NDB; ++i) dk[i] = dv[i] = zero16();
  }
  if (p.splits > 1) {
    const int64_t n = (int64_t)p.B * p.KVH * p.Lk, at = (int64_t)bkv * p.Lk + key;
    if (on) {
      store_part(p.part + (split * 2 * n + at) * p.D, dk, h, p.D);
      store_part(p.part + ((split * 2 + 1) * n + at) * p.D, dv, h, p.D);
    }
    return;
  }
  store_row<T>(p.dk + b * p.dks.b + key * p.dks.l + g * p.dks.h, on, dk, T::kScaled ? p.scale : p.scale * kUnshift, h,
               p.D);
  store_row<T>(p.dv + b * p.dvs.b + key * p.dvs.l + g * p.dvs.h, on, dv, kUnshift, h, p.D);
}

// Sums of the splits, in order: of dQ (kDq), or of dK and dV. Thread: 8 dims of a row.
template <class T, bool kDq>
__global__ __launch_bounds__(256) void xattn_sum_kernel(const Args p) {
  const int nd = p.D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = kDq ? p.rows : p.Lk;
  const int64_t n = (int64_t)p.B * p.KVH * per, all = kDq ? n : 2 * n;
  if (i >= all * nd) return;
  const int64_t at = i / nd;
  const int d0 = (int)(i - at * nd) * 8;
  float o[8] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float* src = p.part + (s * all + at) * p.D + d0;
    const float4 a = *reinterpret_cast<const float4*>(src), c = *reinterpret_cast<const float4*>(src + 4);
    o[0] += a.x, o[1] += a.y, o[2] += a.z, o[3] += a.w;
    o[4] += c.x, o[5] += c.y, o[6] += c.z, o[7] += c.w;
  }
  const bool is_v = !kDq && at >= n;
  const int64_t r = is_v ? at - n : at;
  const int bkv = (int)(r / per), x = (int)(r - (int64_t)bkv * per);
  const int b = bkv / p.KVH, g = bkv - b * p.KVH;
  uint16_t* dst;
  if (kDq) {
    const uint32_t hg = fdiv(x, p.by_lq), tok = x - hg * p.Lq;
    dst = p.dq + (((int64_t)b * p.Lq + tok) * p.H + g * p.G + hg) * p.D;
  } else if (is_v) {
    dst = p.dv + b * p.dvs.b + x * p.dvs.l + g * p.dvs.h;
  } else {
    dst = p.dk + b * p.dks.b + x * p.dks.l + g * p.dks.h;
  }
  constexpr float kUnshift = 1.f / (1 << T::kShift);
  const float f = is_v ? kUnshift : T::kScaled ? p.scale : p.scale * kUnshift;
  *reinterpret_cast<uint4*>(dst + d0) = uint4{T::pack(o[0] * f, o[1] * f), T::pack(o[2] * f, o[3] * f),
                                              T::pack(o[4] * f, o[5] * f), T::pack(o[6] * f, o[7] * f)};
}

}  // namespace xattn
}  // namespace dpa

using namespace dpa;
using namespace dpa::xattn;

// lse and D of every row, then room for one kernel's partial sums at a time
static int64_t stat_bytes(const Args& p) { return align256((int64_t)p.B * p.KVH * p.rows * 8); }

static int64_t bwd_workspace(const Args& rows, const Args& keys) {
  const int64_t a = part_rows_bytes(rows), b = part_keys_bytes(keys);
  return stat_bytes(rows) + (a > b ? a : b);
}

// Never 0: a caller without one is told so at every size.
static int64_t short_workspace(const Args& k) { return align256(part_keys_bytes(k) + 1); }

extern "C" int64_t dpa_cross_attention_bwd_workspace_bytes(const DpaCrossAttention* a) {
  if (!a || check_shape(*a) != DPA_OK) return 0;
  Args r = make_args(*a), k = r;
  if (short_keys_bwd(k)) {
    plan_short(k, true);
    return short_workspace(k);
  }
  plan_rows(r, few_rows_dq(r));
  plan_keys(k);
  return bwd_workspace(r, k);
}

template <class T>
static int sum_keys(const Args& k, hipStream_t s) {
  if (k.splits <= 1 || k.Lk == 0) return DPA_OK;
  const int64_t n = (int64_t)k.B * k.KVH * k.Lk * 2 * (k.D / 8);
  xattn_sum_kernel<T, false><<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(k);
  return launch_status();
}

template <class T, int DP>
static int launch_bwd(const Args& r, const Args& k, hipStream_t s) {
  if (r.total > 0) {
    if (few_rows_dq(r))
      xattn_dq_few_kernel<T, DP><<<r.grid, 256, 0, s>>>(r);
    else
      xattn_dq_kernel<T, DP><<<r.grid, 256, 0, s>>>(r);
    int st = launch_status();
    if (st != DPA_OK) return st;
    if (r.splits > 1) {
      const int64_t n = (int64_t)r.B * r.KVH * r.rows * (r.D / 8);
      xattn_sum_kernel<T, true><<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(r);
      st = launch_status();
      if (st != DPA_OK) return st;
    }
  }
  if (k.total > 0) {
    if (few_keys(k))
      xattn_dkdv_kernel<T, DP, 2><<<k.grid, 256, 0, s>>>(k);
    else if constexpr (DP != 128)  // (few_keys holds for 128)
      xattn_dkdv_kernel<T, DP, 4><<<k.grid, 256, 0, s>>>(k);
    const int st = launch_status();
    return st != DPA_OK ? st : sum_keys<T>(k, s);
  }
  return DPA_OK;
}

template <class T>
static int run_bwd(const Args& r, const Args& k, hipStream_t s) {
  switch (dim_pad(r.D)) {
    case 32: return launch_bwd<T, 32>(r, k, s);
    case 64: return launch_bwd<T, 64>(r, k, s);
    default: return launch_bwd<T, 128>(r, k, s);
  }
}

extern "C" int dpa_cross_attention_bwd(const DpaCrossAttention* a, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  if (!a) return DPA_ERR_NULL;
  const int st = check_shape(*a);
  if (st != DPA_OK) return st;
  if (a->batch == 0) return DPA_OK;
  if (a->q_len > 0 && (!a->q || !a->out || !a->lse || !a->dout || !a->dq)) return DPA_ERR_NULL;
  if (a->kv_len > 0 && (!a->k || !a->v)) return DPA_ERR_NULL;
  if (!a->dk != !a->dv) return DPA_ERR_NULL;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) ||
      !aligned(a->dout, 16) || !aligned(a->dq, 16) || !aligned(a->dk, 16) || !aligned(a->dv, 16) ||
      !aligned(a->lse, 4) || !aligned(a->key_lengths, 4) || !strides_ok(a->q_stride) ||
      !strides_ok(a->k_stride) || !strides_ok(a->v_stride) || !strides_ok(a->dout_stride) ||
      !strides_ok(a->dk_stride) || !strides_ok(a->dv_stride))
    return DPA_ERR_ALIGN;
  Args r = make_args(*a), k = r;
  hipStream_t s = (hipStream_t)stream;
  if (short_keys_bwd(k)) {
    plan_short(k, true);
    if (!grid_ok(k)) return DPA_ERR_SIZE;
    if (!workspace || workspace_bytes < short_workspace(k)) return DPA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
    k.part = (float*)workspace;
    const int status = short_bwd(k, a->dtype, s);
    if (status != DPA_OK || !a->dk) return status;
    return a->dtype == DPA_DTYPE_BF16 ? sum_keys<Bf16>(k, s) : sum_keys<F16>(k, s);
  }
  plan_rows(r, few_rows_dq(r));
  plan_keys(k);
  if (!grid_ok(r) || (a->dk && !grid_ok(k))) return DPA_ERR_SIZE;
  const int64_t need = bwd_workspace(r, k);
  if (need) {
    if (!workspace || workspace_bytes < need) return DPA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
    r.row_stat = k.row_stat = (float*)workspace;
    r.part = k.part = (float*)((uint8_t*)workspace + stat_bytes(r));
  }
  if (a->q_len == 0) r.total = 0;
  if (!a->dk) k.total = 0;
  return a->dtype == DPA_DTYPE_BF16 ? run_bwd<Bf16>(r, k, s) : run_bwd<F16>(r, k, s);
}
