// Cross attention, forward, over keys and values held in MXFP4 (format: mxfp4.hpp, dense): the forms of
// xattn_fwd.hip, with values of the operands' type made from the 4-bit ones on the way to the products.
// The products stay those of bf16 or fp16: queries and probabilities in 4 bits would lose what the cache
// keeps. A value of the cache is exact in bf16; in fp16 it is one that fp16 holds if it was quantised from fp16.
// Scores, maxima and sums are fp32; a probability is rounded to the queries' type for the product with the values, as in
// the 16-bit forms (the sum l takes it before): the product has no operand of fp32, and the sum of two 16-bit ones would be
// twice the products. Against 64 bits outputs are then 2.1e-3 off in bf16 and 2.9e-4 in fp16 (relative norms), with
// probabilities in fp32 1.7e-3 and 2.1e-4, which the output's own rounding makes.
#include <algorithm>
#include <type_traits>

#include "mxfp4.hpp"
#include "xattn_join.hpp"
#include "xattn_short.hpp"

namespace dpa {
namespace xattn {

struct MxArgs : Args {
  const uint8_t *kd, *kx, *vd, *vx;  // elements and scales of keys and of values
  Stride kds, kxs, vds, vxs;         // in bytes
};

// Two elements (byte i of w) in the operands' type
template <class T, int I>
__device__ __forceinline__ uint32_t pair_of(uint32_t w, float scale) {
  if constexpr (std::is_same_v<T, Bf16>)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, I));
}
template <class T>
__device__ __forceinline__ uint4 eight_of(uint32_t w, float scale) {
  return uint4{pair_of<T, 0>(w, scale), pair_of<T, 1>(w, scale), pair_of<T, 2>(w, scale), pair_of<T, 3>(w, scale)};
}

struct RawBlock {
  uint4 w;
  uint32_t byte;
};
// block of a row, or zeros
__device__ __forceinline__ RawBlock raw_block(const uint8_t* data, const uint8_t* scales, bool on) {
  RawBlock r{uint4{0u, 0u, 0u, 0u}, 127u};
  if (on) {
    r.w = *reinterpret_cast<const uint4*>(data);
    r.byte = *scales;
  }
  return r;
}

// A block's 32 values as granules 4 blk .. 4 blk + 3 of row `row` of the array at `at`
template <class T, int DP>
__device__ __forceinline__ void put_block(uint32_t at, int row, int blk, const RawBlock& raw) {
  const float s = mx::scale_back(raw.byte);
  const uint32_t w[4] = {raw.w.x, raw.w.y, raw.w.z, raw.w.w};
#pragma unroll
  for (int g = 0; g < 4; ++g)
    lds_st16(at + row * DP * 2 + (((4 * blk + g) ^ swz<DP>(row)) << 4), eight_of<T>(w[g], s));
}

// ---------------------------------------------------------------------------------------
// Four waves of 32 query rows share tiles of 64 keys; a tile's blocks go through registers, one tile ahead. Bound as the
// 16-bit form is, by the products and the softmax, and by the conversions, which cost more than the shorter loads save: 8 x 1024 queries
// of 8 heads of 128 over 4096 keys 149 us, there 143; 4 x 4096 of 8 heads of 64, two to a key head, over 1031 keys in fp16 52.3,
// there 47.2. (Of 64 dims four workgroups share a CU, with 128 registers a lane, of which four addresses of
// put_block lie in scratch: every second step loads them again, one after the other.)
// ---------------------------------------------------------------------------------------
constexpr float kSlack = 8.f;

template <class T, int DP>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 4) void xattn_mxfp4_fwd_kernel(const MxArgs p) {
  constexpr int KT = 64;
  constexpr int KS = DP / 16, NDB = DP / 32, NB = DP / 32;
  constexpr int kItems = 2 * KT * NB / 256 > 0 ? 2 * KT * NB / 256 : 1;  // blocks to a thread
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

  const int row = tile * 128 + wave * 32 + col;
  const bool has_row = row < p.rows;
  const uint32_t head = fdiv(has_row ? row : 0, p.by_lq), tok = (has_row ? row : 0) - head * p.Lq;

  // this thread's blocks: of keys first, then of values
  const uint8_t *src[kItems], *sscale[kItems];
  int64_t pitch[kItems], spitch[kItems];
  int key_of[kItems], blk_of[kItems];
  bool value_of[kItems], on[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int at = tid + 256 * i, in = at % (KT * NB);
    value_of[i] = at >= KT * NB;
    key_of[i] = in / NB, blk_of[i] = in % NB;
    on[i] = at < 2 * KT * NB && blk_of[i] * 32 < p.D;
    const Stride &ds = value_of[i] ? p.vds : p.kds, &xs = value_of[i] ? p.vxs : p.kxs;
    src[i] = (value_of[i] ? p.vd : p.kd) + b * ds.b + g * ds.h + blk_of[i] * 16;
    sscale[i] = (value_of[i] ? p.vx : p.kx) + b * xs.b + g * xs.h + blk_of[i];
    pitch[i] = ds.l, spitch[i] = xs.l;
  }
  RawBlock raw[kItems];
  auto load = [&](int t, uint64_t word) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int64_t key = (int64_t)t * KT + key_of[i];
      raw[i] = raw_block(src[i] + key * pitch[i], sscale[i] + key * spitch[i], on[i] && (word >> key_of[i]) & 1);
    }
  };
  auto put = [&](int buf, uint64_t word) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (tid + 256 * i < 2 * KT * NB)
        put_block<T, DP>(l0 + buf * 2 * kBytes + (value_of[i] ? kBytes : 0), key_of[i], blk_of[i], raw[i]);
    if (wave == 0)
      *reinterpret_cast<float*>(lds + kBias + buf * KT * 4 + lane * 4) = (word >> lane) & 1 ? 0.f : -__builtin_inff();
  };

  uint64_t word = 0, next = 0;
  if (t_lo < t_hi) {
    word = bits.template word<KT>(t_lo);
    load(t_lo, word);
  }
  uint4 qf[KS];
  load_row<KS>(qf, p.q + b * p.qs.b + (int64_t)tok * p.qs.l + (g * p.G + head) * p.qs.h, has_row, h, p.D);
  if (t_lo < t_hi) {
    put(0, word);
    if (t_lo + 1 < t_hi) {
      next = bits.template word<KT>(t_lo + 1);
      load(t_lo + 1, next);
    }
  }
  const RowAt<DP> row_at(lane, l0);
  const TrAt<DP, NDB> tr_at(lane, l0 + kBytes);
  const uint32_t bias_at = opaque(l0 + kBias + 16 * h);

  v16f o[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) o[i] = zero16();
  float m = -__builtin_inff();  // what O and l stand at, in units of c2 S
  float l = 0.f;                // this lane's half of the running sum

  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    wait_lgkmcnt0();
    lds_barrier();  // tile t is there, and every wave is past its reads of the other buffer
    const uint64_t after = next;
    if (t + 1 < t_hi) {
      put(buf ^ 1, next);
      if (t + 2 < t_hi) {
        next = bits.template word<KT>(t + 2);
        load(t + 2, next);
      }
    }
    if (word) {
      v16f s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = start_at(bias_at + buf * KT * 4 + 128 * i);
#pragma unroll
        for (int k = 0; k < KS; ++k)
          s[i] = T::mfma(row_at.get(k, buf * 2 * kBytes + kBytes / 2 * i), qf[k], s[i]);
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[i][r]);
      top = max_halves(top) * p.c2;
      if (__any(top > m + kSlack)) {
        const float mn = fmaxf(top, m);
        const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= f;
      }
      const float ms = m == -__builtin_inff() ? 0.f : m;  // nothing visible yet: P = 0
#pragma unroll
      for (int i = 0; i < 2; ++i)
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
            o[d] = T::mfma(tr_at.get(d, buf * 2 * kBytes + kBytes / 2 * i + kBytes / 4 * s2), pf, o[d]);
        }
    }
    word = after;
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = t_lo; t < t_hi; t += 2) {
    step(t, std::integral_constant<int, 0>());
    if (t + 1 < t_hi) step(t + 1, std::integral_constant<int, 1>());
  }
  l = sum_halves(l);

  if (p.splits > 1) {
    if (!has_row) return;
    const int64_t at = ((int64_t)split * p.B * p.KVH + bkv) * p.rows + row;
    if (h == 0) p.stat[at] = float2{m, l};
    store_part(p.part + at * p.D, o, h, p.D);
    return;
  }
  if (has_row && h == 0)
    p.lse[((int64_t)b * p.H + g * p.G + head) * p.Lq + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  store_row<T>(p.out + (((int64_t)b * p.Lq + tok) * p.H + g * p.G + head) * p.D, has_row, o,
               l == 0.f ? 0.f : 1.f / l, h, p.D);
}

// ---------------------------------------------------------------------------------------
// Few rows: four waves share 32 rows and take every fourth tile of 32 keys each, and join their softmaxes
// in LDS. A lane's key goes straight to its A operand: dims [h DP / 2, (h + 1) DP / 2) of key l & 31, eight of
// them to a product, and the queries likewise. Values pass through LDS, whose transpose reads turn them. 16 x 8
// queries of 16 heads, four to a key head of 128, over 4096 keys 29.8 us with the join, in 16 bits 35.4.
// ---------------------------------------------------------------------------------------
template <class T, int DP>
__global__ __launch_bounds__(256, 2) void xattn_mxfp4_few_kernel(const MxArgs p) {
  constexpr int KT = 32;
  constexpr int KS = DP / 16, NDB = DP / 32, NB = DP / 32;
  constexpr int kWords = DP / 16;                       // of 8 elements, of a lane's key
  constexpr int kScales = NB > 1 ? NB / 2 : 1;          // of a lane's key
  constexpr int kItems = NB > 1 ? NB / 2 : 1;           // blocks of values to a lane
  constexpr uint32_t kBytes = KT * DP * 2, kBias = 4 * kBytes;  // [4 waves]
  constexpr uint32_t kJoin = 4 * DP * 32 * 4;           // the waves' O at the end
  constexpr uint32_t kLds = kBias + 4 * KT * 4 > kJoin ? kBias + 4 * KT * 4 : kJoin;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
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
  const int t_lo = split * p.per_split + wave;
  int t_hi = split + 1 == p.splits ? nt : min(nt, (split + 1) * p.per_split);
  const KeyBits bits(p, b, klen, split * p.per_split * KT, t_hi * KT, seen, tid);
  t_hi = bits.tiles_to<KT>(t_hi);

  const int row = tile * 32 + col;
  const bool has_row = row < p.rows;
  const uint32_t head = fdiv(has_row ? row : 0, p.by_lq), tok = (has_row ? row : 0) - head * p.Lq;

  const uint8_t* kd = p.kd + b * p.kds.b + g * p.kds.h + h * (DP / 4);
  const uint8_t* kx = p.kx + b * p.kxs.b + g * p.kxs.h + h * (DP / 64);
  const uint8_t* vd = p.vd + b * p.vds.b + g * p.vds.h;
  const uint8_t* vx = p.vx + b * p.vxs.b + g * p.vxs.h;
  uint32_t kw[kWords], ksc[kScales];
  RawBlock vraw[kItems];
  auto load = [&](int t, uint32_t word) __attribute__((always_inline)) {
    const int64_t key = (int64_t)t * KT + col;
    const bool see = (word >> col) & 1;
#pragma unroll
    for (int i = 0; i < kWords; ++i) kw[i] = 0;
#pragma unroll
    for (int i = 0; i < kScales; ++i) ksc[i] = 127;
    if constexpr (NB == 1) {
      if (see) {
        const uint2 w = *reinterpret_cast<const uint2*>(kd + key * p.kds.l);
        kw[0] = w.x, kw[1] = w.y;
        ksc[0] = kx[key * p.kxs.l];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kScales; ++i)
        if (see && h * (DP / 2) + 32 * i < p.D) {
          const uint4 w = *reinterpret_cast<const uint4*>(kd + key * p.kds.l + 16 * i);
          kw[4 * i] = w.x, kw[4 * i + 1] = w.y, kw[4 * i + 2] = w.z, kw[4 * i + 3] = w.w;
          ksc[i] = kx[key * p.kxs.l + i];
        }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int at = lane + 64 * i, vkey = (at / NB) & 31, blk = at % NB;
      const int64_t vk = (int64_t)t * KT + vkey;
      vraw[i] = raw_block(vd + vk * p.vds.l + 16 * blk, vx + vk * p.vxs.l + blk,
                          (word >> vkey) & 1 && at < KT * NB && blk * 32 < p.D);
    }
  };
  uint32_t word = 0;
  if (t_lo < t_hi) {
    word = (uint32_t)bits.template word<KT>(t_lo);
    load(t_lo, word);
  }
  uint4 qf[KS];
  {
    const uint16_t* q = p.q + b * p.qs.b + (int64_t)tok * p.qs.l + (g * p.G + head) * p.qs.h;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int dim = h * (DP / 2) + 8 * k;
      qf[k] = *static_cast<const uint4*>(has_row && dim < p.D ? static_cast<const void*>(q + dim) : g_zero16);
    }
  }
  const uint32_t v0 = l0 + wave * kBytes;
  const TrAt<DP, NDB> tr_at(lane, v0);
  const uint32_t bias_at = opaque(l0 + kBias + wave * 128 + 16 * h);

  v16f o[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) o[i] = zero16();
  float m = -__builtin_inff(), l = 0.f;

  for (int t = t_lo; t < t_hi; t += 4) {
    // this tile to its places, then the next one's loads
    u32x4 kf[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k)
      kf[k] = __builtin_bit_cast(u32x4, eight_of<T>(kw[k], mx::scale_back(ksc[NB > 1 ? k / 4 : 0])));
    asm volatile("" ::: "memory");  // (behind the reads of the tile before)
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int at = lane + 64 * i;
      if (at < KT * NB) put_block<T, DP>(v0, at / NB, at % NB, vraw[i]);
    }
    if (h == 0)
      *reinterpret_cast<float*>(lds + kBias + wave * 128 + col * 4) = (word >> col) & 1 ? 0.f : -__builtin_inff();
    asm volatile("" ::: "memory");
    const uint32_t here = word;
    if (t + 4 < t_hi) {
      word = (uint32_t)bits.template word<KT>(t + 4);
      load(t + 4, word);
    }
    wait_lgkmcnt0();
    asm volatile("" ::: "memory");
    if (here) {
      v16f s = start_at(bias_at);
#pragma unroll
      for (int k = 0; k < KS; ++k) s = T::mfma(kf[k], qf[k], s);
      float top = -__builtin_inff();
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
      top = max_halves(top) * p.c2;
      if (__any(top > m + kSlack)) {
        const float mn = fmaxf(top, m);
        const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= f;
      }
      const float ms = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        uint32_t pk[4];
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * s2 + r], p.c2, -ms));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * s2 + r + 1], p.c2, -ms));
          l += e0 + e1;
          pk[r / 2] = T::pack(e0, e1);
        }
        const uint4 pf = {pk[0], pk[1], pk[2], pk[3]};
#pragma unroll
        for (int d = 0; d < NDB; ++d) o[d] = T::mfma(tr_at.get(d, kBytes / 2 * s2), pf, o[d]);
      }
    }
  }
  l = sum_halves(l);

  // wave w leaves its (m, l) and O, then adds up a quarter of the dims
  __syncthreads();  // (every wave is past its values)
  float* ox = reinterpret_cast<float*>(lds);  // [4][DP][32]
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      ox[(wave * DP + 32 * d + 8 * (r / 4) + 4 * h + r % 4) * 32 + col] = o[d][r];
  __shared__ float ml[2][4][32];
  if (h == 0) {
    ml[0][wave][col] = m;
    ml[1][wave][col] = l;
  }
  __syncthreads();
  m = fmaxf(fmaxf(ml[0][0][col], ml[0][1][col]), fmaxf(ml[0][2][col], ml[0][3][col]));
  const float ms = m == -__builtin_inff() ? 0.f : m;
  float f[4];
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = __builtin_amdgcn_exp2f(ml[0][w][col] - ms);
    l += f[w] * ml[1][w][col];
  }
  // 8 threads per row: dims [q8 DP / 8, (q8 + 1) DP / 8) of row tid & 31
  const int q8 = tid >> 5;
  constexpr int ND = DP / 8;
  float acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) acc[i] += f[w] * ox[(w * DP + q8 * ND + i) * 32 + col];
  }
  if (!has_row) return;
  if (p.splits > 1) {
    const int64_t at = ((int64_t)split * p.B * p.KVH + bkv) * p.rows + row;
    if (q8 == 0) p.stat[at] = float2{m, l};
#pragma unroll
    for (int i = 0; i < ND; i += 4)
      if (q8 * ND + i < p.D)
        *reinterpret_cast<float4*>(p.part + at * p.D + q8 * ND + i) =
            float4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
    return;
  }
  const int64_t orow = ((int64_t)b * p.Lq + tok) * p.H + g * p.G + head;
  if (q8 == 0)
    p.lse[((int64_t)b * p.H + g * p.G + head) * p.Lq + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  const float il = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < ND; i += 4)
    if (q8 * ND + i < p.D)
      *reinterpret_cast<uint2*>(p.out + orow * p.D + q8 * ND + i) =
          uint2{T::pack(acc[i] * il, acc[i + 1] * il), T::pack(acc[i + 2] * il, acc[i + 3] * il)};
}

// ---------------------------------------------------------------------------------------
// Up to 16 rows of a key head (single tokens, their heads sharing keys): as above, on v_mfma_f32_16x16x32, whose
// columns are the rows, a tile of 32 keys to a wave, two on their way. Bound by a wave's chain of a tile, 1.5 us from its
// loads to its second product, of which a wave has eight in a row over 8192 keys of 64 heads: three or four tiles on
// their way did not shorten it (20.3 us there, 23 and 24), nor did keys that went into the product in 4 bits, against
// queries split into sums of e4m3 (half the conversions, 20.4).
//   S^T (16 keys x 16 rows) = K Q^T: lane (key l & 15, q = l >> 4) takes dims [q D / 4, (q + 1) D / 4) of its key, 8 to
//   a product. It receives the scores of row l & 15 at keys 4 q + t of each 16, which packed are the B operand of
//   O^T += V^T P^T if the sum over 32 keys runs over {4 q + t, 16 + 4 q + t} in lane q: so the values' transpose
//   reads fetch rows 4 q .. and 16 + 4 q ...
// ---------------------------------------------------------------------------------------
typedef float v4f __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ v4f mfma16(uint4 a, uint4 b, v4f c) {
  if constexpr (std::is_same_v<T, Bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// maximum and sum over the four lanes of a row
__device__ __forceinline__ float max_quarters(float x) {
  x = max_halves(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_quarters(float x) {
  x = sum_halves(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void xattn_mxfp4_token_kernel(const MxArgs p) {
  constexpr int KT = 32;
  constexpr int DP = D == 96 ? 128 : D;   // of the values' rows in LDS
  constexpr int NB = D / 32;              // blocks to a row, words of 8 dims to a lane's quarter of it
  constexpr int ND = D / 16;              // tiles of dims of O
  constexpr int kItems = NB > 1 ? (NB + 1) / 2 : 1;  // blocks of values to a lane
  constexpr uint32_t kBytes = KT * DP * 2, kJoin = 4 * D * 16 * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kBytes > kJoin ? 4 * kBytes : kJoin];
  __shared__ uint32_t seen[kMaxRange / 32];
  const uint32_t l0 = LDS_ADDR(lds);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, q = lane >> 4;
  const uint32_t id = work_item(p);
  if (id >= p.total) return;
  // the heads of a batch's keys beside each other: their pieces of a token share cache lines
  const uint32_t bs = id / (uint32_t)p.KVH;
  const int g = id - bs * p.KVH, b = bs / (uint32_t)p.splits, bkv = b * p.KVH + g;
  // (a batch's first split is another one each time: with a multiple of 8 of them the first ones, which have keys when
  // others have none, would all go to one XCD. Lengths of 1024 in 8191, 16 batches of 4 heads: 19.4 us against 20.7)
  const int turned = bs - b * p.splits + (uint32_t)b % (uint32_t)p.splits;
  const int split = turned < p.splits ? turned : turned - p.splits;

  const int klen = __builtin_amdgcn_readfirstlane(keys_of(p, b));
  const int nt = (klen + KT - 1) / KT;
  const int t_lo = split * p.per_split + wave;
  int t_hi = split + 1 == p.splits ? nt : min(nt, (split + 1) * p.per_split);
  const KeyBits bits(p, b, klen, split * p.per_split * KT, t_hi * KT, seen, tid);
  t_hi = bits.tiles_to<KT>(t_hi);

  const bool has_row = col < p.rows;
  const uint32_t head = fdiv(has_row ? col : 0, p.by_lq), tok = (has_row ? col : 0) - head * p.Lq;

  const uint8_t* kd = p.kd + b * p.kds.b + g * p.kds.h + q * (D / 8);
  const uint8_t* kx = p.kx + b * p.kxs.b + g * p.kxs.h + q * NB / 4;
  const uint8_t* vd = p.vd + b * p.vds.b + g * p.vds.h;
  const uint8_t* vx = p.vx + b * p.vxs.b + g * p.vxs.h;
  struct Raw {
    uint32_t k[2][NB], kb[2][2];
    RawBlock v[kItems];
    uint32_t word;
  };
  // A tile's loads go out together, without branches: rows behind the length are its last row, and what is not
  // visible is cleared before its use.
  auto load = [&](Raw& raw, int t) __attribute__((always_inline)) {
    raw.word = (uint32_t)bits.template word<KT>(t);
    const int last = klen - 1 - t * KT;
    const uint8_t *kt = kd + (int64_t)t * KT * p.kds.l, *kxt = kx + (int64_t)t * KT * p.kxs.l;
    const uint8_t *vt = vd + (int64_t)t * KT * p.vds.l, *vxt = vx + (int64_t)t * KT * p.vxs.l;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t row = min(16 * h + col, last);
      const uint8_t *s = kt + (uint64_t)row * (uint32_t)p.kds.l, *x = kxt + (uint64_t)row * (uint32_t)p.kxs.l;
      if constexpr (NB == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(s);
        raw.k[h][0] = w.x, raw.k[h][1] = w.y, raw.k[h][2] = w.z, raw.k[h][3] = w.w;
      } else if constexpr (NB == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(s);
        raw.k[h][0] = w.x, raw.k[h][1] = w.y;
      } else {
#pragma unroll
        for (int i = 0; i < NB; ++i) raw.k[h][i] = reinterpret_cast<const uint32_t*>(s)[i];
      }
      raw.kb[h][0] = raw.kb[h][1] = x[0];
      if constexpr (NB == 3) raw.kb[h][1] = x[q == 1 || q == 2 ? 1 : 0];
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int at = min(lane + 64 * i, KT * NB - 1), blk = at % NB;  // (lanes behind the last block: that one)
      const uint32_t row = min(at / NB, last);
      raw.v[i].w = *reinterpret_cast<const uint4*>(vt + (uint64_t)row * (uint32_t)p.vds.l + 16 * blk);
      raw.v[i].byte = vxt[(uint64_t)row * (uint32_t)p.vxs.l + blk];
    }
  };
  auto clear_hidden = [&](Raw& raw) __attribute__((always_inline)) {
    if (raw.word == ~0u) return;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (!((raw.word >> (16 * h + col)) & 1)) {
#pragma unroll
        for (int i = 0; i < NB; ++i) raw.k[h][i] = 0;
        raw.kb[h][0] = raw.kb[h][1] = 127;
      }
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (!((raw.word >> (((lane + 64 * i) / NB) & 31)) & 1)) raw.v[i] = RawBlock{uint4{0u, 0u, 0u, 0u}, 127u};
  };
  Raw r0, r1;
  if (t_lo < t_hi) load(r0, t_lo);
  uint4 qf[NB];
  {
    const uint16_t* s = p.q + b * p.qs.b + (int64_t)tok * p.qs.l + (g * p.G + head) * p.qs.h + q * (D / 4);
#pragma unroll
    for (int i = 0; i < NB; ++i)
      qf[i] = *static_cast<const uint4*>(has_row ? static_cast<const void*>(s + 8 * i) : g_zero16);
  }
  if (t_lo + 4 < t_hi) load(r1, t_lo + 4);
  const uint32_t v0 = l0 + wave * kBytes;
  // transpose reads: lane k of a quarter addresses 4 dims of row 4 q + (k >> 2) (and of the row 16 further)
  uint32_t tr[ND][2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = 4 * q + (col >> 2) + 16 * x, gr = 2 * d + ((col & 3) >> 1);
      tr[d][x] = v0 + row * DP * 2 + ((gr ^ swz<DP>(row)) << 4) + 8 * (col & 1);
    }

  v4f o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f;

  auto tile = [&](Raw& raw, int t) __attribute__((always_inline)) {
    // the tile out of its registers, then the loads of the one after the next into them
    clear_hidden(raw);
    uint4 kf[2][NB];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        // word i of quarter q lies in block (q NB + i) / 4, the first of the quarter's or the one behind it
        const bool second = NB == 3 && (3 * q + i) / 4 != 3 * q / 4;
        kf[h][i] = eight_of<T>(raw.k[h][i], mx::scale_back(second ? raw.kb[h][1] : raw.kb[h][0]));
      }
    asm volatile("" ::: "memory");  // (behind the reads of the tile before)
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int at = lane + 64 * i;
      if (at < KT * NB) put_block<T, DP>(v0, at / NB, at % NB, raw.v[i]);
    }
    asm volatile("" ::: "memory");
    const uint32_t word = raw.word;
    if (t + 8 < t_hi) load(raw, t + 8);
    if (word == 0) return;
    v4f s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[h][i] = (word >> (16 * h + 4 * q + i)) & 1 ? 0.f : -__builtin_inff();
#pragma unroll
      for (int i = 0; i < NB; ++i) s[h] = mfma16<T>(kf[h][i], qf[i], s[h]);
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = max_quarters(top) * p.c2;
    if (__any(top > m + kSlack)) {
      const float mn = fmaxf(top, m);
      const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= f;
    }
    const float ms = m == -__builtin_inff() ? 0.f : m;
    uint32_t pk[4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i], p.c2, -ms));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i + 1], p.c2, -ms));
        l += e0 + e1;
        pk[2 * h + i / 2] = T::pack(e0, e1);
      }
    const uint4 pf = {pk[0], pk[1], pk[2], pk[3]};
    wait_lgkmcnt0();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      typedef v4s __attribute__((address_space(3))) * LP;
      const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(tr[d][0])));
      const uint2 c = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(tr[d][1])));
      o[d] = mfma16<T>(uint4{a.x, a.y, c.x, c.y}, pf, o[d]);
    }
  };
  for (int t = t_lo; t < t_hi; t += 8) {
    tile(r0, t);
    if (t + 4 < t_hi) tile(r1, t + 4);
  }
  l = sum_quarters(l);

  // wave w leaves its (m, l) and O; a thread adds up D / 16 dims of a row
  __syncthreads();
  float* ox = reinterpret_cast<float*>(lds);  // [4][D][16]
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) ox[(wave * D + 16 * d + 4 * q + i) * 16 + col] = o[d][i];
  __shared__ float ml[2][4][16];
  if (q == 0) {
    ml[0][wave][col] = m;
    ml[1][wave][col] = l;
  }
  __syncthreads();
  m = fmaxf(fmaxf(ml[0][0][col], ml[0][1][col]), fmaxf(ml[0][2][col], ml[0][3][col]));
  const float ms = m == -__builtin_inff() ? 0.f : m;
  float f[4];
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = __builtin_amdgcn_exp2f(ml[0][w][col] - ms);
    l += f[w] * ml[1][w][col];
  }
  if (!has_row) return;
  const int part = tid >> 4;  // dims [part ND, (part + 1) ND)
  float acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) acc[i] += f[w] * ox[(w * D + part * ND + i) * 16 + col];
  }
  if (p.splits > 1) {
    const int64_t at = ((int64_t)split * p.B * p.KVH + bkv) * p.rows + col;
    if (part == 0) p.stat[at] = float2{m, l};
#pragma unroll
    for (int i = 0; i < ND; i += 2)
      *reinterpret_cast<float2*>(p.part + at * D + part * ND + i) = float2{acc[i], acc[i + 1]};
    return;
  }
  const int64_t orow = ((int64_t)b * p.Lq + tok) * p.H + g * p.G + head;
  if (part == 0)
    p.lse[((int64_t)b * p.H + g * p.G + head) * p.Lq + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  const float il = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < ND; i += 2)
    *reinterpret_cast<uint32_t*>(p.out + orow * D + part * ND + i) = T::pack(acc[i] * il, acc[i + 1] * il);
}

// ---------------------------------------------------------------------------------------
// Up to 128 keys: xattn_short.hpp over the values that a workgroup makes of them once. 128 x 1024 queries of 4 heads of
// 64 dims over 77 keys 28.7 us, by tiles of keys 40, in 16 bits 30.3: bound by the queries and the output.
// ---------------------------------------------------------------------------------------
template <class T, int DP, int NB>
__global__ __launch_bounds__(256, short_waves(DP)) void xattn_mxfp4_short_kernel(const MxArgs p) {
  short_forward<T, DP, NB>(p, [&](int b, int g, uint32_t kl, uint32_t vl, float* bias, int tid, int wave, int lane)
                               __attribute__((always_inline)) {
    constexpr int kRow = DP / 32;  // blocks to a row
    const int klen = keys_of(p, b);
    const uint8_t* mb = p.kmask ? p.kmask + b * p.mask_b : nullptr;
    auto visible = [&](int key) __attribute__((always_inline)) { return key < klen && (!mb || mb[key] != 0); };
    const uint8_t *kd = p.kd + b * p.kds.b + g * p.kds.h, *kx = p.kx + b * p.kxs.b + g * p.kxs.h;
    const uint8_t *vd = p.vd + b * p.vds.b + g * p.vds.h, *vx = p.vx + b * p.vxs.b + g * p.vxs.h;
    constexpr int kAll = 2 * NB * 32 * kRow;
    RawBlock raw[(kAll + 255) / 256];
#pragma unroll
    for (int i = 0; i < (kAll + 255) / 256; ++i) {
      const int at = tid + 256 * i, in = at % (kAll / 2), key = in / kRow, blk = in % kRow;
      const bool value = at >= kAll / 2, on = at < kAll && blk * 32 < p.D && visible(key);
      raw[i] = raw_block((value ? vd + key * p.vds.l : kd + key * p.kds.l) + 16 * blk,
                         (value ? vx + key * p.vxs.l : kx + key * p.kxs.l) + blk, on);
    }
#pragma unroll
    for (int i = 0; i < (kAll + 255) / 256; ++i) {
      const int at = tid + 256 * i, in = at % (kAll / 2);
      if (at < kAll) put_block<T, DP>(at >= kAll / 2 ? vl : kl, in / kRow, in % kRow, raw[i]);
    }
    put_bias<NB>(bias, tid, visible);
    wait_lgkmcnt0();
    lds_barrier();
    return active_blocks<NB>(bias, lane);
  });
}

// ---- host ------------------------------------------------------------------------------
static DpaCrossAttention shape_of(const DpaCrossAttentionMxfp4& a) {
  DpaCrossAttention c{};
  c.q = a.q, c.out = a.out, c.lse = a.lse, c.key_lengths = a.key_lengths, c.key_mask = a.key_mask;
  c.mask_stride = a.mask_stride;
  for (int i = 0; i < 3; ++i) c.q_stride[i] = a.q_stride[i];
  c.dtype = a.dtype, c.batch = a.batch, c.q_len = a.q_len, c.kv_len = a.kv_len;
  c.heads = a.heads, c.kv_heads = a.kv_heads, c.head_dim = a.head_dim, c.scale = a.scale;
  return c;
}

static int check_mx(const DpaCrossAttentionMxfp4& a) {
  const int st = check_shape(shape_of(a));
  if (st != DPA_OK) return st;
  if (a.head_dim % 32) return DPA_ERR_SHAPE;
  // (a row's place in a tile is its number times 32 bits)
  for (const int64_t tokens : {a.k_data_stride[1], a.k_scale_stride[1], a.v_data_stride[1], a.v_scale_stride[1]})
    if (tokens < 0 || tokens >= 1ll << 32) return DPA_ERR_SIZE;
  return DPA_OK;
}

static bool strides16(const int64_t* s) { return s[0] % 16 == 0 && s[1] % 16 == 0 && s[2] % 16 == 0; }

// Up to 16 rows of a key head have a form of their own
static bool token_rows(const Args& p) { return p.rows <= 16; }

static void plan_mx(Args& p) {
  if (!token_rows(p)) {
    if (short_keys_fwd(p))
      plan_short(p, false);
    else
      plan_rows(p, few_rows_fwd(p));
    return;
  }
  p.tiles = 1;
  const int64_t groups = (int64_t)p.B * p.KVH;
  // two workgroups to a CU; what fills the CUs without is not split, and no row into more than 64 parts, which the
  // join would wait for (16 queries over up to 8191 keys of 4 heads of 128, 48 MB of cache: 20.3 us, with three to a
  // CU 22.7, with four 22.0; lengths of 1024 in 8191 19.4, 15.5 and 16.4)
  const int64_t want = groups >= 2 * num_cus() ? groups : std::min<int64_t>(2 * num_cus(), 64 * groups);
  choose_splits(p, groups, ceil_div(p.Lk, 32), want, 8, kMaxRange / 32, 4);
  // A head's piece of a token is 16 to 64 B and its scales 1 to 4, so that cache lines hold those of several: the
  // heads of a split go to one XCD; splits are dealt out in turn, since lengths differ.
  p.total = (uint32_t)(groups * p.splits);
  p.unit = (uint32_t)p.KVH;
  p.by_unit = make_fastdiv(p.unit);
  p.grid = (uint32_t)(ceil_div(groups * p.splits, 8 * (int64_t)p.KVH) * 8 * p.KVH);
}

// Whether the keys of a row are split (the short form's splits are of the rows)
static bool has_parts(const Args& p) { return p.splits > 1 && (token_rows(p) || !short_keys_fwd(p)); }

template <class T, int DP>
static void launch_mx(const MxArgs& p, hipStream_t s) {
  if (short_keys_fwd(p)) {
    if (p.Lk <= 96)
      xattn_mxfp4_short_kernel<T, DP, 3><<<p.grid, 256, 0, s>>>(p);
    else
      xattn_mxfp4_short_kernel<T, DP, 4><<<p.grid, 256, 0, s>>>(p);
  } else if (few_rows_fwd(p))
    xattn_mxfp4_few_kernel<T, DP><<<p.grid, 256, 0, s>>>(p);
  else
    xattn_mxfp4_fwd_kernel<T, DP><<<p.grid, 256, 0, s>>>(p);
}

template <class T>
static int run_mx(const MxArgs& p, hipStream_t s) {
  if (token_rows(p)) {
    switch (p.D) {
      case 32: xattn_mxfp4_token_kernel<T, 32><<<p.grid, 256, 0, s>>>(p); break;
      case 64: xattn_mxfp4_token_kernel<T, 64><<<p.grid, 256, 0, s>>>(p); break;
      case 96: xattn_mxfp4_token_kernel<T, 96><<<p.grid, 256, 0, s>>>(p); break;
      default: xattn_mxfp4_token_kernel<T, 128><<<p.grid, 256, 0, s>>>(p); break;
    }
  } else {
    switch (dim_pad(p.D)) {
      case 32: launch_mx<T, 32>(p, s); break;
      case 64: launch_mx<T, 64>(p, s); break;
      default: launch_mx<T, 128>(p, s); break;
    }
  }
  const int st = launch_status();
  return st != DPA_OK || !has_parts(p) ? st : join_splits<T>(p, s);
}

}  // namespace xattn
}  // namespace dpa

using namespace dpa;
using namespace dpa::xattn;

extern "C" int64_t dpa_cross_attention_mxfp4_workspace_bytes(const DpaCrossAttentionMxfp4* a) {
  if (!a || check_mx(*a) != DPA_OK) return 0;
  Args p = make_args(shape_of(*a));
  plan_mx(p);
  return has_parts(p) ? fwd_workspace(p) : 0;
}

extern "C" int dpa_cross_attention_mxfp4(const DpaCrossAttentionMxfp4* a, void* workspace, int64_t workspace_bytes,
                                         void* stream) {
  if (!a) return DPA_ERR_NULL;
  const int st = check_mx(*a);
  if (st != DPA_OK) return st;
  if (a->batch == 0 || a->q_len == 0) return DPA_OK;
  if (!a->q || !a->out || !a->lse || (a->kv_len > 0 && (!a->k_data || !a->k_scales || !a->v_data || !a->v_scales)))
    return DPA_ERR_NULL;
  if (!aligned(a->q, 16) || !aligned(a->k_data, 16) || !aligned(a->v_data, 16) || !aligned(a->out, 16) ||
      !aligned(a->lse, 4) || !aligned(a->key_lengths, 4) || !strides_ok(a->q_stride) ||
      !strides16(a->k_data_stride) || !strides16(a->v_data_stride))
    return DPA_ERR_ALIGN;
  MxArgs p{};
  static_cast<Args&>(p) = make_args(shape_of(*a));
  p.kd = (const uint8_t*)a->k_data, p.kx = (const uint8_t*)a->k_scales;
  p.vd = (const uint8_t*)a->v_data, p.vx = (const uint8_t*)a->v_scales;
  p.kds = stride_of(a->k_data_stride), p.kxs = stride_of(a->k_scale_stride);
  p.vds = stride_of(a->v_data_stride), p.vxs = stride_of(a->v_scale_stride);
  hipStream_t s = (hipStream_t)stream;
  plan_mx(p);
  if (!grid_ok(p)) return DPA_ERR_SIZE;
  const int64_t need = has_parts(p) ? fwd_workspace(p) : 0;
  if (need) {
    if (!workspace || workspace_bytes < need) return DPA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
    p.part = (float*)workspace;
    p.stat = (float2*)((uint8_t*)workspace + align256(part_rows_bytes(p)));
  }
  return a->dtype == DPA_DTYPE_BF16 ? run_mx<Bf16>(p, s) : run_mx<F16>(p, s);
}
