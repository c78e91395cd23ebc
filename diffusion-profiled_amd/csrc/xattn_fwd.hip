// Cross attention, forward: one pass over the keys with the running maximum and sum of each
// row's softmax.
#include <type_traits>

#include "xattn_join.hpp"

namespace dpa {
namespace xattn {

// ---------------------------------------------------------------------------------------
// Four waves of 32 query rows each share tiles of 64 keys, double-buffered by DMA.
//
// Per tile a wave forms S^T = K Q^T (A: key rows from LDS, B: its queries, in registers), so lane
// l holds scores of query l & 31 at keys 8 i + 4 (l >> 5) + j; then the row's running maximum and
// sum, P = 2^(c2 S - m) rounded to the operands' type for the product (its sum is of the fp32
// values), and O^T += V^T P^T with P^T straight from those registers. A product over a tile starts
// from 0 for the visible keys and -inf for the others, which costs no instruction per score.
//
// The maximum that O and its sum stand at moves up only when a score passes it by 2^8: P then
// stays below 2^8, which fp32 and both operand types have room for, and nearly every tile goes
// without the products that move it.
//
// Bound by the products and the exponentials (a quarter-rate unit, one per score), which follow each
// other within a wave and overlap between the waves of a SIMD: hence four waves of 64 dims to a SIMD (two of 128).
// bf16, 8 x 4096 queries of 8 heads of 64 dims over 1024 keys: 108 us, 635 TFLOP/s, MFMA 34 % busy;
// fp16, 16 x 1024 of 8 heads of 128 dims over 512 keys of 2: 61 us from cold operands, 49 from cached
// ones (700 TFLOP/s). A third buffer of keys brought nothing (94 -> 98 us).
// ---------------------------------------------------------------------------------------
constexpr float kSlack = 8.f;

template <class T, int DP>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 4) void xattn_fwd_kernel(const Args p) {
  constexpr int KT = 64;
  constexpr int KS = DP / 16, NDB = DP / 32;
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

  const int row = tile * 128 + wave * 32 + col;
  const bool has_row = row < p.rows;
  const uint32_t head = fdiv(has_row ? row : 0, p.by_lq), tok = (has_row ? row : 0) - head * p.Lq;
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
  uint4 qf[KS];
  load_row<KS>(qf, p.q + b * p.qs.b + (int64_t)tok * p.qs.l + (g * p.G + head) * p.qs.h, has_row, h, p.D);
  const RowAt<DP> row_at(lane, l0);
  const TrAt<DP, NDB> tr_at(lane, l0 + kBytes);
  const uint32_t bias_at = opaque(l0 + kBias + 16 * h);
  wait_vmcnt<0>();  // (no wait on the queries inside the loop: it would take in the tile in flight)

  v16f o[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) o[i] = zero16();
  float m = -__builtin_inff();  // what O and l stand at, in units of c2 S
  float l = 0.f;                // this lane's half of the running sum

  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    uint64_t word_next = 0;
    wait_vmcnt<0>();
    keys.ready(t, buf, word);
    wait_lgkmcnt0();
    lds_barrier();  // tile t is there, and every wave is past its reads of the other buffer
    if (t + 1 < t_hi) {
      word_next = bits.template word<KT>(t + 1);
      fetch(t + 1, buf ^ 1, word_next);
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
    word = word_next;
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
// Few workgroups: the four waves share 32 rows and take every fourth tile of 32 keys each, and join
// their softmaxes in LDS at the end. Products as above. This form reads the keys and values once
// and does little with them, so it is made for bytes in flight: keys go straight to registers as A
// operands, values to LDS, each one tile ahead, and two workgroups of 128 dims fit a CU.
// fp16, 16 x 1 queries of 16 heads over 4 of up to 4097 keys of 128 dims: 20 us for 90 MB (72 of them from HBM).
// Few keys as well: three dependent trips to memory (lengths, operands, store), 5.5 us for 4 x 1
// queries over 77 keys.
// ---------------------------------------------------------------------------------------
template <class T, int DP>
__global__ __launch_bounds__(256, 2) void xattn_few_kernel(const Args p) {
  constexpr int KT = 32;
  constexpr int NG = DP / 8, KS = DP / 16, NDB = DP / 32;
  constexpr int kXfer = KT * NG / 64;
  constexpr uint32_t kBytes = KT * DP * 2, kBias = 8 * kBytes;  // [4 waves][2]
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBias + 4 * 2 * KT * 4];
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
  const uint16_t* kb = p.k + b * p.ks.b + g * p.ks.h;
  const uint16_t* vb = p.v + b * p.vs.b + g * p.vs.h;
  const KeyBits bits(p, b, klen, split * p.per_split * KT, t_hi * KT, seen, tid);
  t_hi = bits.tiles_to<KT>(t_hi);

  const int row = tile * 32 + col;
  const bool has_row = row < p.rows;
  const uint32_t head = fdiv(has_row ? row : 0, p.by_lq), tok = (has_row ? row : 0) - head * p.Lq;
  uint4 kf[2][KS];
  auto fetch = [&](int t, uint4(&k)[KS], int buf, uint32_t word) __attribute__((always_inline)) {
    const uint16_t* vt = vb + (int64_t)t * KT * p.vs.l;
    const uint32_t at = __builtin_amdgcn_readfirstlane(l0 + (wave * 2 + buf) * kBytes);
#pragma unroll
    for (int r = 0; r < kXfer; ++r)
      dma_rows<DP>(at, 64 * r, lane, p.D, [&](int row) __attribute__((always_inline)) {
        return (word >> row) & 1 ? vt + row * p.vs.l : static_cast<const uint16_t*>(nullptr);
      });
    load_row<KS>(k, kb + ((int64_t)t * KT + col) * p.ks.l, (word >> col) & 1, h, p.D);
    if (h == 0)
      *reinterpret_cast<float*>(lds + kBias + (wave * 2 + buf) * 128 + col * 4) = (word >> col) & 1 ? 0.f : -__builtin_inff();
  };
  uint32_t word = 0;
  if (t_lo < t_hi) {
    word = (uint32_t)bits.template word<KT>(t_lo);
    fetch(t_lo, kf[0], 0, word);
  }
  uint4 qf[KS];
  load_row<KS>(qf, p.q + b * p.qs.b + (int64_t)tok * p.qs.l + (g * p.G + head) * p.qs.h, has_row, h, p.D);
  const TrAt<DP, NDB> tr_at(lane, l0 + wave * 2 * kBytes);
  const uint32_t bias_at = opaque(l0 + kBias + wave * 256 + 16 * h);

  v16f o[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) o[i] = zero16();
  float m = -__builtin_inff(), l = 0.f;

  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    uint32_t word_next = 0;
    wait_vmcnt<0>();
    wait_lgkmcnt0();  // the tile is there, and the reads of the other buffer are done
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (t + 4 < t_hi) {
      word_next = (uint32_t)bits.template word<KT>(t + 4);
      fetch(t + 4, kf[buf ^ 1], buf ^ 1, word_next);
    }
    asm volatile("" ::: "memory");
    if (word) {
      v16f s = start_at(bias_at + buf * 128);
#pragma unroll
      for (int k = 0; k < KS; ++k) s = T::mfma(kf[buf][k], qf[k], s);
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
        for (int d = 0; d < NDB; ++d) o[d] = T::mfma(tr_at.get(d, buf * kBytes + kBytes / 2 * s2), pf, o[d]);
      }
    }
    word = word_next;
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = t_lo; t < t_hi; t += 8) {
    step(t, std::integral_constant<int, 0>());
    if (t + 4 < t_hi) step(t + 4, std::integral_constant<int, 1>());
  }
  l = sum_halves(l);

  // wave w leaves its (m, l) and O, then adds up a quarter of the dims
  __syncthreads();  // (every wave is past its buffers)
  float* ox = reinterpret_cast<float*>(lds);  // [4][DP][32]
  static_assert(8 * kBytes >= 4 * DP * 32 * 4, "the waves' O fit the buffers");
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

}  // namespace xattn
}  // namespace dpa

using namespace dpa;
using namespace dpa::xattn;

extern "C" int64_t dpa_cross_attention_fwd_workspace_bytes(const DpaCrossAttention* a) {
  if (!a || check_shape(*a) != DPA_OK) return 0;
  Args p = make_args(*a);
  if (short_keys_fwd(p)) return 0;
  plan_rows(p, few_rows_fwd(p));
  return fwd_workspace(p);
}

template <class T, int DP>
static void launch_fwd(const Args& p, hipStream_t s) {
  if (few_rows_fwd(p))
    xattn_few_kernel<T, DP><<<p.grid, 256, 0, s>>>(p);
  else
    xattn_fwd_kernel<T, DP><<<p.grid, 256, 0, s>>>(p);
}

template <class T>
static int run_fwd(const Args& p, hipStream_t s) {
  switch (dim_pad(p.D)) {
    case 32: launch_fwd<T, 32>(p, s); break;
    case 64: launch_fwd<T, 64>(p, s); break;
    default: launch_fwd<T, 128>(p, s); break;
  }
  const int st = launch_status();
  return st != DPA_OK || p.splits <= 1 ? st : join_splits<T>(p, s);
}

extern "C" int dpa_cross_attention_fwd(const DpaCrossAttention* a, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  if (!a) return DPA_ERR_NULL;
  const int st = check_shape(*a);
  if (st != DPA_OK) return st;
  if (a->batch == 0 || a->q_len == 0) return DPA_OK;
  if (!a->q || !a->out || !a->lse || (a->kv_len > 0 && (!a->k || !a->v))) return DPA_ERR_NULL;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) ||
      !aligned(a->lse, 4) || !aligned(a->key_lengths, 4) || !strides_ok(a->q_stride) ||
      !strides_ok(a->k_stride) || !strides_ok(a->v_stride))
    return DPA_ERR_ALIGN;
  Args p = make_args(*a);
  hipStream_t s = (hipStream_t)stream;
  if (short_keys_fwd(p)) {
    plan_short(p, false);
    if (!grid_ok(p)) return DPA_ERR_SIZE;
    return short_fwd(p, a->dtype, s);
  }
  plan_rows(p, few_rows_fwd(p));
  if (!grid_ok(p)) return DPA_ERR_SIZE;
  const int64_t need = fwd_workspace(p);
  if (need) {
    if (!workspace || workspace_bytes < need) return DPA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
    p.part = (float*)workspace;
    p.stat = (float2*)((uint8_t*)workspace + align256(part_rows_bytes(p)));
  }
  return a->dtype == DPA_DTYPE_BF16 ? run_fwd<Bf16>(p, s) : run_fwd<F16>(p, s);
}
