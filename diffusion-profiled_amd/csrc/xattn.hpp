// Cross attention of B images' query tokens to an encoder's states of another length: what the
// forward and the backward kernels share. Per (batch, key/value head g), with the G = H / KVH
// query heads that read g taken together as rows = G Lq query rows (row r: head g G + r / Lq,
// token r % Lq):
//   S = c Q K^T over the visible keys, P = softmax(S), O = P V, lse = log sum exp S.
// A key is visible below its batch's length and where its mask byte is not 0. Rows of keys and
// values that are not visible change nothing (they may hold NaN): zeros take their place in LDS,
// and their scores are -inf. Those from the length on are not read; those that the mask hides below it
// may be, where a tile goes as a whole, and are cleared in LDS. A row without a visible key gives O = 0 and lse = -inf.
//
// Products run on v_mfma_f32_32x32x16 (bf16 or fp16 operands, fp32 sums): against the 16x16x32
// form it needs half the LDS reads per product, and one query per lane column, so a row's
// softmax needs one exchange (with lane ^ 32). Head dims are multiples of 8 up to 128, padded
// with zeros to DP = 32, 64 or 128 in LDS and registers only.
#pragma once
#include "dpa_common.hpp"

namespace dpa {
namespace xattn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Stride {
  int64_t b, l, h;  // elements between batches, tokens, heads
};

struct Args {
  const uint16_t *q, *k, *v, *dout;
  uint16_t *out, *dq, *dk, *dv;  // out and dq dense [B][Lq][H][D]
  float* lse;                    // [B][H][Lq], natural logarithm
  const int32_t* klen;           // [B] or null
  const uint8_t* kmask;          // [B][Lk] or null
  Stride qs, ks, vs, gs, dks, dvs;
  int64_t mask_b;
  float* part;   // fp32 partial sums of a split axis
  float2* stat;  // forward: their (max, sum)
  float* row_stat;  // backward: kShift - lse in base 2 of every query row, then their -rowsum(dO O)
  int B, Lq, Lk, H, KVH, G, D, rows, tiles;
  int splits, per_split;  // workgroups that share one tile's loop, and its steps each
  uint32_t total;         // workgroups with work
  uint32_t grid;          // workgroups launched
  uint32_t unit;          // neighbours among them that one XCD takes
  float c2, scale;        // scale log2(e), scale
  FastDiv by_lq, by_unit;
};

// kShift: the backward forms 2^kShift P and takes the factor out of its fp32 sums at the end. In
// bf16, whose exponents have the room, that keeps probabilities down to 2^-150, where v_exp_f32
// alone gives 0 below 2^-126; it costs nothing. fp16 has room for 2^14 P, at most 1, which keeps all
// bits of probabilities down to 2^-28.
// kScaled: dS is scaled by a power of 2 that follows its size (in fp16: P (dP - D) over 4096 keys with
// gradients of 1e-5 is mostly below its subnormals, and beyond 65504 with a large loss scale).
struct Bf16 : Elem<DPA_DTYPE_BF16> {
  static constexpr int kShift = 24;
  static constexpr bool kScaled = false;
  template <class A>
  static __device__ __forceinline__ v16f mfma(A a, uint4 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

struct F16 : Elem<DPA_DTYPE_F16> {
  static constexpr int kShift = 14;
  static constexpr bool kScaled = true;
  template <class A>
  static __device__ __forceinline__ v16f mfma(A a, uint4 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// Fragments of v_mfma_f32_32x32x16: lane l supplies row (column of B) l & 31 and 8 k-elements of
// slice h = l >> 5; it receives D[8 (r / 4) + 4 h + r % 4][l & 31] in register r of 16. Two
// products chain without moving data: registers 8 s .. 8 s + 7 of a result, packed, are the B
// operand of a product over its rows 16 s + {4 h + j, 8 + 4 h + j}, whose A operand comes from
// transpose reads of those rows.
__device__ __forceinline__ v16f zero16() {
  return v16f{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

__device__ __forceinline__ uint4 ld16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }

// A rows array in LDS: rows of DP elements, the 16-B granule g of row r at g ^ swz(r). 16 rows
// read at one granule, and the 4 rows x 2 granules of a transpose read, then lie in 64 different
// banks each.
template <int DP>
__device__ __forceinline__ int swz(int r) {
  if (DP == 32) return (r >> 2) & 3;
  if (DP == 64) return (r & 6) | ((r >> 3) & 1);
  return ((r & 7) << 1) | ((r >> 3) & 1);
}

// 8 elements of row r at granule g
template <int DP>
__device__ __forceinline__ uint4 frag_row(const uint16_t* x, int r, int g) {
  return ld16(x + r * DP + ((g ^ swz<DP>(r)) << 3));
}

// Operand of the transpose of the array: dims 32 db + (lane & 31), k over its rows r0 + 4 h +
// {0..3, 8..11} (r0 a multiple of 16). The transpose read gives lane j of a group of 16 column j
// of 4 rows, the group's lanes addressing 4 elements of a row each.
template <int DP>
__device__ __forceinline__ uint4 frag_tr(const uint16_t* x, int r0, int db, int lane) {
  const int k = lane & 15, rr = k >> 2;
  const int g = 4 * db + 2 * ((lane >> 4) & 1) + ((k & 3) >> 1), half = 4 * (k & 1);
  const int r1 = r0 + 4 * (lane >> 5) + rr, r2 = r1 + 8;
  typedef v4s __attribute__((address_space(3))) * LP;
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(x + r1 * DP + ((g ^ swz<DP>(r1)) << 3) + half));
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(x + r2 * DP + ((g ^ swz<DP>(r2)) << 3) + half));
  const uint2 lo = __builtin_bit_cast(uint2, a), hi = __builtin_bit_cast(uint2, b);
  return uint4{lo.x, lo.y, hi.x, hi.y};
}

// The same reads with what depends on the lane in registers, made once: byte addresses in an array
// that starts at `base` (a multiple of 1024), to which a read adds constants (another array, its
// rows in steps of 16 or 32), which become the instruction's immediate offset. (opaque: else the
// compiler keeps a register for every sum.)
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
  asm("" : "+v"(x));
  return x;
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// (a vector: as a struct the load falls apart)
__device__ __forceinline__ u32x4 lds_ld16(uint32_t a) {
  return *(const __attribute__((address_space(3))) u32x4*)(a);
}
__device__ __forceinline__ void lds_st16(uint32_t a, uint4 v) {
  *(__attribute__((address_space(3))) u32x4*)(a) = __builtin_bit_cast(u32x4, v);
}
__device__ __forceinline__ void lds_st8(uint32_t a, uint32_t x, uint32_t y) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  *(__attribute__((address_space(3))) u32x2*)(a) = u32x2{x, y};
}

// frag_row of row l & 31, granules 2 k + (l >> 5)
template <int DP>
struct RowAt {
  uint32_t a[DP / 16];
  __device__ __forceinline__ RowAt(int lane, uint32_t base) {
    const int r = lane & 31;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      a[k] = opaque(base + r * DP * 2 + (((2 * k + (lane >> 5)) ^ swz<DP>(r)) << 4));
  }
  __device__ __forceinline__ u32x4 get(int k, uint32_t at) const { return lds_ld16(a[k] + at); }
};

// frag_tr of rows 0 .. 15, dims 32 (db0 + d) ..
template <int DP, int ND>
struct TrAt {
  uint32_t a[ND][2];
  __device__ __forceinline__ TrAt(int lane, uint32_t base, int db0 = 0, int step = 1) {
    const int k = lane & 15, r = 4 * (lane >> 5) + (k >> 2);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int g = 4 * (db0 + step * d) + 2 * ((lane >> 4) & 1) + ((k & 3) >> 1), rr = r + 8 * x;
        a[d][x] = opaque(base + rr * DP * 2 + ((g ^ swz<DP>(rr)) << 4) + 8 * (k & 1));
      }
  }
  __device__ __forceinline__ uint4 get(int d, uint32_t at) const {
    typedef v4s __attribute__((address_space(3))) * LP;
    const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(a[d][0] + at));
    const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(a[d][1] + at));
    const uint2 lo = __builtin_bit_cast(uint2, x), hi = __builtin_bit_cast(uint2, y);
    return uint4{lo.x, lo.y, hi.x, hi.y};
  }
};

// start_from of 32 floats at byte address at (with the lane's 16 h in it)
__device__ __forceinline__ v16f start_at(uint32_t at) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  v16f s;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const f32x4 v = *(const __attribute__((address_space(3))) f32x4*)(at + 32 * x);
    s[4 * x] = v.x, s[4 * x + 1] = v.y, s[4 * x + 2] = v.z, s[4 * x + 3] = v.w;
  }
  return s;
}

static __device__ __attribute__((aligned(64))) uint32_t g_zero16[4];

// 64 transfers of 16 B of a wave: chunks c0 .. c0 + 63 (c0 wave-uniform) of the rows array at lds,
// from the row pointers that src(row) gives (null: zeros).
template <int DP, class Src>
__device__ __forceinline__ void dma_rows(uint32_t lds, int c0, int lane, int D, Src src) {
  constexpr int NG = DP / 8;
  const int c = c0 + lane, row = c / NG;
  const int g = (c % NG) ^ swz<DP>(row);
  const uint16_t* s = src(row);
  const void* a = (s && 8 * g < D) ? static_cast<const void*>(s + 8 * g) : g_zero16;
  dma16_lds(a, lds + (uint32_t)c0 * 16);
}

// 16 B per lane from base (wave-uniform) + off bytes
__device__ __forceinline__ void dma16_lds_from(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0");
}

// 4 B per lane to lds + 4 * lane (lds wave-uniform).
__device__ __forceinline__ void dma4_lds(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "m0");
}

// Which keys of a workgroup's range [k0, k1) are visible, in words of 32 or 64 keys. Mask bytes are
// packed into LDS first: loaded in the loop over the keys, their waits would take in the tiles in
// flight. The host splits the keys so that a range has at most kMaxRange.
constexpr int kMaxRange = 16384;

struct KeyBits {
  const uint32_t* seen;  // LDS, null without a mask
  int klen, k0;
  int last;  // keys from here on are invisible (a multiple of 64, or the range's end)
  __device__ __forceinline__ KeyBits(const Args& p, int b, int klen_, int k0_, int k1,
                                     uint32_t* lds, int tid)
      : seen(p.kmask ? lds : nullptr), klen(klen_), k0(k0_), last(k1) {
    if (!seen) return;
    const uint8_t* mb = p.kmask + b * p.mask_b;
    const int lane = tid & 63;
    k1 = min((k1 + 63) & ~63, k0 + kMaxRange);
    for (int k = k0 + (tid & ~63); k < k1; k += blockDim.x) {
      const int key = k + lane;
      const uint64_t w = __ballot(key < klen && mb[key < klen ? key : 0] != 0);
      if (lane < 2) lds[(k - k0) / 32 + lane] = (uint32_t)(w >> (32 * lane));
    }
    __syncthreads();
    last = k0;
    for (int k = k0; k < k1; k += 64 * 64) {  // (a lane per 64 keys)
      const int at = k + 64 * lane;
      const uint64_t any = __ballot(at < k1 && (lds[(at - k0) / 32] | lds[(at - k0) / 32 + 1]) != 0);
      if (any) last = k + 64 * (64 - __builtin_clzll(any));
    }
    last = __builtin_amdgcn_readfirstlane(last);
  }
  // tiles [.., t_hi) without the invisible ones at their end
  template <int KT>
  __device__ __forceinline__ int tiles_to(int t_hi) const {
    return seen ? min(t_hi, (last + KT - 1) / KT) : t_hi;
  }
  // keys KT t .. KT t + KT - 1 (inside the range)
  template <int KT>
  __device__ __forceinline__ uint64_t word(int t) const {
    if (seen) {
      const uint32_t* s = seen + (t * KT - k0) / 32;
      const uint32_t lo = __builtin_amdgcn_readfirstlane(s[0]);
      return KT == 64 ? lo | (uint64_t)__builtin_amdgcn_readfirstlane(s[1]) << 32 : lo;
    }
    const int n = klen - t * KT;
    const uint64_t all = KT == 64 ? ~0ull : 0xffffffffull;
    return n >= KT ? all : n <= 0 ? 0 : (1ull << n) - 1;
  }
};

// Keys of batch b below its length
__device__ __forceinline__ int keys_of(const Args& p, int b) {
  if (!p.klen) return p.Lk;
  const int n = p.klen[b];
  return n < 0 ? 0 : n < p.Lk ? n : p.Lk;
}

// Tiles of 64 keys and values that a workgroup of four waves brings to LDS (rows arrays of 64 x DP:
// keys at l0 + buf * 2 kBytes, values kBytes behind). Tiles whose 64 keys are all below the length
// go by one instruction per transfer, its lane part a constant offset; then their rows that the mask
// hides are cleared in LDS (ready(), once the tile has landed). The others, heads that are not DP
// wide and rows that are far apart choose an address per row.
template <int DP>
struct KeyTiles {
  static constexpr int NG = DP / 8, kXfer = 64 * NG / 256, kRows = 256 / NG;
  static constexpr uint32_t kBytes = 64 * DP * 2;
  const uint16_t *kb, *vb;  // key 0 of the head
  int64_t kl, vl;
  uint32_t ko, vo, l0;  // (transfers of a tile are kRows rows apart, a multiple of the period of swz)
  int lane, wave, klen, D;
  bool fast;

  __device__ __forceinline__ KeyTiles(const Args& p, int b, int g, int klen_, uint32_t lds, int wave_, int lane_)
      : kb(p.k + b * p.ks.b + g * p.ks.h), vb(p.v + b * p.vs.b + g * p.vs.h), kl(p.ks.l), vl(p.vs.l),
        l0(lds), lane(lane_), wave(wave_), klen(klen_), D(p.D) {
    fast = D == DP && kl >= 0 && vl >= 0 && kl < (1 << 24) && vl < (1 << 24);
    const int c = wave * 64 + lane, row = c / NG, g8 = ((c % NG) ^ swz<DP>(row)) << 3;
    ko = (uint32_t)(row * (int)kl + g8) * 2;
    vo = (uint32_t)(row * (int)vl + g8) * 2;
  }
  __device__ __forceinline__ bool whole(int t) const { return fast && t * 64 + 64 <= klen; }

  __device__ __forceinline__ void fetch(int t, int buf, uint64_t word) const {
    const uint16_t *kt = kb + (int64_t)t * 64 * kl, *vt = vb + (int64_t)t * 64 * vl;
    const uint32_t at = l0 + buf * 2 * kBytes + wave * 1024;
    if (whole(t)) {
#pragma unroll
      for (int r = 0; r < kXfer; ++r) {
        dma16_lds_from(kt + r * kRows * kl, ko, at + 4096 * r);
        dma16_lds_from(vt + r * kRows * vl, vo, at + kBytes + 4096 * r);
      }
    } else {
#pragma unroll
      for (int r = 0; r < kXfer; ++r) {
        const int c0 = wave * 64 + 256 * r;
        dma_rows<DP>(l0 + buf * 2 * kBytes, c0, lane, D, [&](int row) __attribute__((always_inline)) {
          return (word >> row) & 1 ? kt + row * kl : static_cast<const uint16_t*>(nullptr);
        });
        dma_rows<DP>(l0 + buf * 2 * kBytes + kBytes, c0, lane, D, [&](int row) __attribute__((always_inline)) {
          return (word >> row) & 1 ? vt + row * vl : static_cast<const uint16_t*>(nullptr);
        });
      }
    }
  }
  // (before the barrier behind which tile t is read)
  __device__ __forceinline__ void ready(int t, int buf, uint64_t word) const {
    if (word == ~0ull || !whole(t)) return;
    const uint32_t at = l0 + buf * 2 * kBytes + wave * 1024 + lane * 16;
#pragma unroll
    for (int r = 0; r < kXfer; ++r) {
      const int row = (wave * 64 + 256 * r + lane) / NG;
      if (!((word >> row) & 1)) {
        lds_st16(at + 4096 * r, uint4{0u, 0u, 0u, 0u});
        lds_st16(at + kBytes + 4096 * r, uint4{0u, 0u, 0u, 0u});
      }
    }
  }
};

// A wave's kXfer transfers each of the tiles of keys and values from key k0 on into kl and vl,
// chunks c0, c0 + kStep, ...; keys whose bit in word is 0 come as zeros.
template <int DP, int kXfer, int kStep>
__device__ __forceinline__ void fetch_keys(const Args& p, const uint16_t* kb, const uint16_t* vb, int64_t k0,
                                           uint64_t word, const uint16_t* kl, const uint16_t* vl, int c0,
                                           int lane) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint16_t* base = x == 0 ? kb + k0 * p.ks.l : vb + k0 * p.vs.l;
    const int64_t pitch = x == 0 ? p.ks.l : p.vs.l;
    const uint32_t lds = LDS_ADDR(x == 0 ? kl : vl);
#pragma unroll
    for (int r = 0; r < kXfer; ++r)
      dma_rows<DP>(lds, c0 + kStep * r, lane, p.D, [&](int row) __attribute__((always_inline)) {
        return (word >> row) & 1 ? base + row * pitch : static_cast<const uint16_t*>(nullptr);
      });
  }
}

// The B operands of a row of queries (or of their gradient). Lanes without one load zeros: a branch
// around each load would keep the loads from going out together.
template <int KS>
__device__ __forceinline__ void load_row(uint4 (&f)[KS], const uint16_t* src, bool on, int h, int D) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int dim = 16 * ks + 8 * h;
    f[ks] = *static_cast<const uint4*>(on && dim < D ? static_cast<const void*>(src + dim) : g_zero16);
  }
}

// Workgroup i of the launch goes to XCD i % 8. Units of neighbours in the order of work (the row
// tiles and splits of one key/value head) go to one XCD, whose L2 then holds their keys; the units
// are dealt out to the XCDs in turn, so that ragged lengths even out.
__device__ __forceinline__ uint32_t work_item(const Args& p) {
  const uint32_t j = blockIdx.x >> 3, u = fdiv(j, p.by_unit);
  return (u * 8 + (blockIdx.x & 7)) * p.unit + (j - u * p.unit);
}

// A value's maximum or sum over lanes l and l ^ 32
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the maximum over a wave, of nothing negative: halves, rows of 16 lanes, then within a row
__device__ __forceinline__ float wave_max(float x) {
  x = max_halves(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false)));  // row_ror:8
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xf, 0xf, false)));
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x122, 0xf, 0xf, false)));
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x121, 0xf, 0xf, false)));
}

// The power of 2, `up`, at which a lane's column of 2^kShift dS stands (fp16): moved down only when a
// |dP - D| passes what the type holds, and then so far that values 2^4 larger fit too, so that nearly every
// tile goes without moving the sums. In the kernel of dK and dV a wave's columns share it, in a scalar
// register: at 128 dims it has no vector register left (175 us with one, 171 without, at 16 x 1024 below). Numbers
// down to 2^-25 of the largest that fits stay normal, so smaller columns lose nothing.
// Half a vector instruction per score, in dK one more. The fp16 backward without and with it: 16 x 1024 queries of
// 8 heads over 512 keys of 2, 128 dims, 168, 171 us; 16 x 1 of 16 heads over 4097 keys of 4 133, 142; 8 x 4096 of 64
// dims over 1024 keys 293, 298; 128 x 1024 of 32 dims over 200 keys 98, 106.
struct DsScale {
  static constexpr int kFirst = 46;  // (nothing passes before it is 2^-45)
  float up = __uint_as_float((127u + kFirst) << 23);
  // the largest of these 16 of the column's values (lane ^ 32 has as many more of them)
  static __device__ __forceinline__ float largest(const v16f& dp) {
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r & 1] = fmaxf(t[r & 1], fabsf(dp[r]));
    return fmaxf(t[0], t[1]);
  }
  // 2^kShift dS up stays below 2^15 (P is at most 1, but for its rounding)
  __device__ __forceinline__ bool passes(float top) const { return top * up > 2.f; }
  // the binary exponent by which it moves for the column's `top`, 0 if that does not pass
  __device__ __forceinline__ int move(float top) {
    if (!passes(top)) return 0;
    const int was = __builtin_amdgcn_frexp_expf(up) - 1;
    const int k = min(was, -3 - __builtin_amdgcn_frexp_expf(top));  // (top < 2^its exponent)
    up = ldexpf(1.f, k);
    return k - was;
  }
  // the same for all of the wave's columns, from its lanes' largest
  __device__ __forceinline__ int move_wave(float top) {
    const int by = move(wave_max(top));
    up = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(up)));
    return __builtin_amdgcn_readfirstlane(by);
  }
};

// f x as row l & 31 of a dense array's rows at dst (dims in the registers of the accumulators, on:
// whether the lane's row exists). Lanes l and l ^ 32 hold 4 dims of every 8; they trade halves of
// neighbouring eights, so that each stores 16 B.
template <class T, int NDB>
__device__ __forceinline__ void store_row(uint16_t* dst, bool on, const v16f (&x)[NDB], float f, int h, int D) {
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 8) {
      const auto a = __builtin_amdgcn_permlane32_swap(T::pack(x[d][r] * f, x[d][r + 1] * f),
                                                      T::pack(x[d][r + 4] * f, x[d][r + 5] * f), false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(T::pack(x[d][r + 2] * f, x[d][r + 3] * f),
                                                      T::pack(x[d][r + 6] * f, x[d][r + 7] * f), false, false);
      const int dim = 32 * d + 2 * r + 8 * h;
      if (on && dim < D) *reinterpret_cast<uint4*>(dst + dim) = uint4{a[0], b[0], a[1], b[1]};
    }
}
// the same rows in fp32
template <int NDB>
__device__ __forceinline__ void store_part(float* dst, const v16f (&x)[NDB], int h, int D) {
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int dim = 32 * d + 2 * r + 4 * h;
      if (dim < D)
        *reinterpret_cast<float4*>(dst + dim) = float4{x[d][r], x[d][r + 1], x[d][r + 2], x[d][r + 3]};
    }
}

// The accumulator of a product whose 32 rows start from b[0 .. 31] (LDS, 16-B aligned)
__device__ __forceinline__ v16f start_from(const float* b, int h) {
  v16f s;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float4 v = *reinterpret_cast<const float4*>(b + 8 * x + 4 * h);
    s[4 * x] = v.x, s[4 * x + 1] = v.y, s[4 * x + 2] = v.z, s[4 * x + 3] = v.w;
  }
  return s;
}

// ---- host ------------------------------------------------------------------------------
// Shapes and sizes of a call (its pointers apart). Everything that the kernels index in 32 bits
// (rows, keys, workgroups) is bounded here; element offsets are 64-bit.
inline int check_shape(const DpaCrossAttention& a) {
  if (a.dtype != DPA_DTYPE_BF16 && a.dtype != DPA_DTYPE_F16) return DPA_ERR_SHAPE;
  if (a.batch < 0 || a.q_len < 0 || a.kv_len < 0 || a.heads <= 0 || a.kv_heads <= 0) return DPA_ERR_SIZE;
  if (a.heads % a.kv_heads || a.head_dim <= 0 || a.head_dim > 128 || a.head_dim % 8) return DPA_ERR_SHAPE;
  if (!(a.scale > 0.f) || !(a.scale * kLog2e <= 3.4e38f)) return DPA_ERR_SIZE;
  const int64_t most = 1ll << 30;
  const int64_t rows = (int64_t)a.heads / a.kv_heads * a.q_len;
  if (rows >= most || a.kv_len >= most || (int64_t)a.batch * a.kv_heads >= most) return DPA_ERR_SIZE;
  const int64_t bkv = (int64_t)a.batch * a.kv_heads;
  if (bkv * (rows / 32 + 1) >= most || bkv * (a.kv_len / 128 + 1) >= most ||
      bkv * rows >= most * 8 || bkv * a.kv_len >= most * 8)
    return DPA_ERR_SIZE;
  return DPA_OK;
}

inline bool strides_ok(const int64_t* s) { return s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0; }
inline Stride stride_of(const int64_t* s) { return Stride{s[0], s[1], s[2]}; }

inline Args make_args(const DpaCrossAttention& a) {
  Args p{};
  p.q = (const uint16_t*)a.q, p.k = (const uint16_t*)a.k, p.v = (const uint16_t*)a.v;
  p.dout = (const uint16_t*)a.dout;
  p.out = (uint16_t*)a.out, p.dq = (uint16_t*)a.dq, p.dk = (uint16_t*)a.dk, p.dv = (uint16_t*)a.dv;
  p.lse = a.lse;
  p.klen = a.key_lengths;
  p.kmask = a.key_mask;
  p.mask_b = a.mask_stride;
  p.qs = stride_of(a.q_stride), p.ks = stride_of(a.k_stride), p.vs = stride_of(a.v_stride);
  p.gs = stride_of(a.dout_stride), p.dks = stride_of(a.dk_stride), p.dvs = stride_of(a.dv_stride);
  p.B = a.batch, p.Lq = a.q_len, p.Lk = a.kv_len, p.H = a.heads, p.KVH = a.kv_heads;
  p.G = a.heads / a.kv_heads, p.D = a.head_dim, p.rows = p.G * p.Lq;
  p.c2 = a.scale * kLog2e;
  p.scale = a.scale;
  p.by_lq = make_fastdiv(p.Lq > 0 ? p.Lq : 1);
  return p;
}

// Splits the `steps` of a loop over `groups` workgroups' worth of launches so that about `want`
// workgroups run, each of at least `least` and at most `most` steps (a multiple of `unit`).
inline void choose_splits(Args& p, int64_t groups, int64_t steps, int64_t want, int64_t least,
                          int64_t most, int64_t unit) {
  int64_t n = groups > 0 ? want / groups : 1;
  if (n > steps / least) n = steps / least;
  if (n < 1) n = 1;
  int64_t per = ceil_div(ceil_div(steps > 0 ? steps : 1, n), unit) * unit;
  if (per > most) per = most;
  p.per_split = (int)per;
  p.splits = (int)ceil_div(steps > 0 ? steps : 1, per);
}

// Sets p.unit for `total` workgroups, `per_head` of them to a key/value head, and p.grid. A
// unit is a head's work, or a batch's where a head's rows are no whole cache lines (two XCDs would
// fetch each line); with few units, an eighth of all.
inline void set_grid(Args& p, int64_t total, int64_t per_head) {
  int64_t unit = per_head * (p.D % 64 ? p.KVH : 1);
  const int64_t n = unit ? total / unit : 0;
  if (n % 8 && n < 32) unit = ceil_div(total, 8);
  if (unit < 1) unit = 1;
  p.total = (uint32_t)total;
  p.unit = (uint32_t)unit;
  p.by_unit = make_fastdiv(p.unit);
  p.grid = (uint32_t)(ceil_div(total, 8 * unit) * 8 * unit);
}

// Every kernel's workgroups have 256 threads. (The launches behind a split have fewer: it is made where few
// workgroups run.)
inline bool grid_ok(const Args& p) { return p.grid <= kMaxGroups256; }

inline int dim_pad(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// The forward's and dQ's forms: four waves of 32 rows that share tiles of keys, or four waves that
// share 32 rows and take every fourth tile each. The second reads the keys four times as often. It is
// taken for up to 32 rows of a head, and by the forward where it comes to less than two workgroups a
// CU: the first would leave CUs idle. (84 x 38 queries of 4 heads, 80 dims, over 412 keys of one: 13.4
// against 17.4 us; 15 x 1869 of 2 heads over 522 keys, which has more: 30 against 21 us. dQ, whose
// buffers leave a CU one workgroup of 128 dims, gains nothing: 26 against 19 us in the first case.)
inline bool few_rows_dq(const Args& p) { return p.rows <= 32; }
inline bool few_rows_fwd(const Args& p) {
  return p.rows <= 32 || (int64_t)p.B * p.KVH * ceil_div(p.rows, 32) < 2 * num_cus();
}

// Forms that keep a head's keys in LDS (xattn_short.hip), for up to 128 keys: what a CU's LDS holds of 128
// dims beside the backward's rows of P and dS, and the registers of scores. The forward's is for more
// than 32 rows, of which each of its waves takes 32; up to there the waves that split the keys are no
// slower. The backward's takes any number: one launch for two.
// (us, these forms against the others, replayed without the host. 128 x 256 queries of 4 heads of 64 dims
// over 77 keys: forward 12.9, 14.4, backward 24, 40; 128 x 1024 of 32 dims 20, 26 and 39, 65; 64 x 512 of
// 128 dims over 120 keys 20, 25 and 56, 84; 128 x 1024 of 64 dims over 128 keys 45, 50 and 107, 131; 128 x 64
// over 77 keys 7.7, 9.4 and 15, 23; 128 x 16 6.3, 5.9 and 14, 21; 512 x 1 of 8 heads 24.7, 23.5 and 82, 83.)
inline bool short_keys_fwd(const Args& p) { return p.rows > 32 && p.Lk <= 128; }
inline bool short_keys_bwd(const Args& p) { return p.rows > 0 && p.Lk <= 128; }

// Rows are split so that the workgroups that fit the chip at once share them; the backward's splits
// write fp32 sums of dK and dV each, so it leaves at least two tiles of rows to one.
inline void plan_short(Args& p, bool backward) {
  const int dp = dim_pad(p.D);
  const int per_cu = backward ? (dp == 128 || (dp == 64 && p.Lk > 96) ? 1 : 2) : dp == 128 ? 2 : 4;
  p.tiles = (int)ceil_div(p.rows, 128);
  const int64_t groups = (int64_t)p.B * p.KVH;
  choose_splits(p, groups, p.tiles, per_cu * num_cus(), backward ? 2 : 1, 1ll << 30, 1);
  set_grid(p, groups * p.splits, p.splits);
}

int short_fwd(const Args& p, int dtype, hipStream_t s);
int short_bwd(const Args& p, int dtype, hipStream_t s);

inline void plan_rows(Args& p, bool few) {
  p.tiles = (int)ceil_div(p.rows > 0 ? p.rows : 1, few ? 32 : 128);
  const int64_t groups = (int64_t)p.B * p.KVH * p.tiles, kt = few ? 32 : 64;
  choose_splits(p, groups, ceil_div(p.Lk, kt), (few ? 4 : 2) * num_cus(), 8, kMaxRange / kt, few ? 4 : 1);
  set_grid(p, groups * p.splits, (int64_t)p.tiles * p.splits);
}

constexpr int kQT = 64;  // rows of a tile of the kernel of dK and dV

// Its workgroups take 128 keys, or 64 where that leaves few of them, less than four to a CU, and always of
// more than 64 dims, whose sums leave a wave of the 128-key form a SIMD to itself. (8 x 4096 queries of 64
// dims over 700 of 1031 keys 251 -> 197 us with 64. The backward of 128 dims with 128 and 64: 8 x 4096 of 8
// heads over 1024 keys 549, 495; 16 x 1024 over 512 172, 159; 64 x 256 over 200 130, 121.)
inline bool few_keys(const Args& p) {
  return dim_pad(p.D) == 128 || (int64_t)p.B * p.KVH * ceil_div(p.Lk, 128) < 4 * num_cus();
}

inline void plan_keys(Args& p) {
  p.tiles = (int)ceil_div(p.Lk, few_keys(p) ? 64 : 128);
  const int64_t groups = (int64_t)p.B * p.KVH * p.tiles;
  choose_splits(p, groups, ceil_div(p.rows, kQT), 2 * num_cus(), 4, 1ll << 30, 1);
  set_grid(p, groups * p.splits, (int64_t)p.tiles * p.splits);
}

inline int64_t part_rows_bytes(const Args& p) {
  return p.splits > 1 ? (int64_t)p.splits * p.B * p.KVH * p.rows * p.D * 4 : 0;
}
inline int64_t part_keys_bytes(const Args& p) {
  return p.splits > 1 ? (int64_t)p.splits * 2 * p.B * p.KVH * p.Lk * p.D * 4 : 0;
}
inline int64_t align256(int64_t n) { return (n + 255) & ~255ll; }

}  // namespace xattn
}  // namespace dpa
