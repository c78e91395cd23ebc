// y[M][N] = a[M][K] b[N][K]^T (+ bias) over MXFP4 operands (format: mxfp4.hpp), sums in fp32.
#include <algorithm>
#include <type_traits>

#include "mxfp4.hpp"

namespace dpa {
namespace mx {

struct GemmArgs {
  const uint8_t *a, *as, *b, *bs;  // rows of M and of N
  const float* bias;
  void* y;
  float* part;  // [splits][M][N] where the contraction is split
  int64_t panel_a, panel_b;  // bytes
  const void* x;  // a before its rounding, where the kernel does that, rows ld elements apart
  int64_t ld;
  int M, N, K;
  int steps, per_split, splits;  // of 256 columns; per_split is even
  int tiles_m, tiles_n;
  int form;  // of the tiles
};

// ---------------------------------------------------------------------------------------
// Tiles of WM x WN waves of 16 FM x 16 FN each, a panel of 128 columns (64 B of a row) at a time through a ring of NH buffers
// in LDS by DMA, and their scales by the same way. Workgroups stay and take tile after tile, the next one's first
// transfers out before this one's stores. b's rows are the A operand (rows of D), in the order that gives a lane 8
// columns of y in a row and four lanes 64 B: row r of fragment i is row 32 (i / 2) + 8 (r / 4) + 4 (i % 2) + r % 4 of
// the wave's. The 16-B piece c of a row lies at c ^ turned(its r / 4): the 16 lanes that LDS serves together (rows
// 0-3 and 12-15 at one piece, 4-11 at the one beside it) then lie in 16 different places of the banks.
// Measured: 4096 x 8192 of 8192 122 to 125 us, 4.4 PFLOP/s, the matrix instructions busy 54 % of the time at 1.96 GHz. The same
// without transfers 109, without reads of LDS 111, without both 100, without the meetings too 93: the products alone,
// whose power holds the clock below its 2.4 GHz (a loop of nothing else on random operands: 6.9 PFLOP/s).
// (Four waves of 128 x 128 for 256 x 256: less read of LDS, but nothing to run while a wave waits, 161 us.)
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ int turned(int x) { return ((x ^ (x >> 1)) & 1) << 1 | x >> 1; }  // 0 2 3 1
__device__ __forceinline__ int place_b(int row) { return turned((row >> 3) & 3); }
__device__ __forceinline__ int place_a(int row) { return turned((row >> 2) & 3); }

// (else the compiler keeps a register for every sum with an address)
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
  asm("" : "+v"(x));
  return x;
}

__device__ __forceinline__ u32x4 lds16(uint32_t a) { return *(const __attribute__((address_space(3))) u32x4*)(a); }

__device__ __forceinline__ void dma16_from(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0");
}

// acc += the product, in its own registers (AT: the byte of both scale words). As instructions of their own, in
// their place: the compiler moves products of its own freely between the halves of a step, until all their fragments
// live at once, and gives results other registers than the sums had (207 registers spilled of the 128 x 64
// wave, 0.7 PFLOP/s). It does not know these for matrix instructions, so the waits are here: s_nop before a product
// whose scales or sums a vector instruction may just have written, and results_ready before the sums are read.
template <int AT>
__device__ __forceinline__ void mfma_in_place(v4f& acc, u32x4 a, u32x4 b, uint32_t sa, uint32_t sb) {
#define DPA_MFMA(SEL) \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL " cbsz:4 blgp:4" : "+v"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb))
  if constexpr (AT == 0) DPA_MFMA("op_sel_hi:[0,0,0]");
  if constexpr (AT == 1) DPA_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (AT == 2) DPA_MFMA("op_sel_hi:[1,1,0]");
  if constexpr (AT == 3) DPA_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef DPA_MFMA
}
// 16 passes and more after the last product
__device__ __forceinline__ void results_ready() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

constexpr int kBufferFlags = 0x00020000;     // of a buffer of bytes
constexpr uint32_t kNowhere = 0x80000000u;   // behind the end of every buffer here (check_gemm)

// (DT: of y, or fp32 for the sums of a split, which y then is. vec: N in whole vectors, y aligned to them)
template <int WM, int WN, int FM, int FN, int NH, int DT, bool vec>
__global__ __launch_bounds__(64 * WM * WN) void mxfp4_gemm_kernel(const GemmArgs p) {
  constexpr int kWaves = WM * WN, BM = 16 * FM * WM, BN = 16 * FN * WN;
  // NH buffers of b's rows, NH of a's (a read's place in them is an immediate offset), and scales, 16 B a row and
  // 512 columns, a group more than the ring holds
  constexpr uint32_t kBytesB = BN * 64, kBytesA = BM * 64, kA = NH * kBytesB, kS = kA + NH * kBytesA;
  constexpr uint32_t kBytesS = (BM + BN) * 16;
  constexpr int kSlots = NH / 4 + 1;
  constexpr int kXferB = BN / 16 / kWaves, kXferA = BM / 16 / kWaves, kXfer = kXferB + kXferA;
  static_assert(BN % (16 * kWaves) == 0 && BM % (16 * kWaves) == 0, "transfers of 16 rows");
  static_assert(FN % 2 == 0 && kWaves % 2 == 0 && NH % 4 == 0, "pairs of fragments; a row's place among 32; groups");
  constexpr int kPieces = (BM + BN) / 64;
  static_assert(kPieces <= kWaves, "at most a transfer of scales to a wave");
  // 8 rows of a wave's columns in turn, granule g of 4 columns of row r at g ^ r
  constexpr int kCols = 16 * FN;
  static_assert(kCols <= 64, "a row to a wave");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kS + kSlots * kBytesS + (vec ? 0 : kWaves * 8 * kCols * 4)];
  const uint32_t l0 = LDS_ADDR(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM, r = lane & 15, q = lane >> 4;
  float* turn = reinterpret_cast<float*>(lds + kS + kSlots * kBytesS) + wave * 8 * kCols;
  const uint32_t tiles = p.tiles_m * p.tiles_n, total = tiles * p.splits;
  struct Tile {
    int m0, n0, split, lo, hi;  // its 128 columns lo .. hi - 1
  };
  // Workgroup i goes to XCD i % 8, whose L2 holds the rows that its tiles share: an XCD takes an eighth of the
  // tiles in their order, kBand tiles of rows beside each other.
  constexpr uint32_t kBand = 8;
  const uint32_t share = (total + 7) / 8;
  auto place = [&](uint32_t id) { return (id & 7) * share + (id >> 3); };
  auto tile_of = [&](uint32_t id) __attribute__((always_inline)) {
    Tile c;
    id = place(id);
    c.split = id / tiles;
    id -= c.split * tiles;
    const uint32_t band = id / (kBand * p.tiles_n), rows = min(kBand, p.tiles_m - band * kBand);
    id -= band * kBand * p.tiles_n;
    const uint32_t tn = id / rows;
    c.m0 = (band * kBand + id - tn * rows) * BM, c.n0 = tn * BN;
    c.lo = 2 * c.split * p.per_split, c.hi = min(2 * p.steps, c.lo + 2 * p.per_split);
    return c;
  };
  auto there = [&](uint32_t id) { return (id >> 3) < share && place(id) < total; };
  if (!there(blockIdx.x)) return;
  Tile c = tile_of(blockIdx.x);

  // A transfer is 16 rows of a wave; its first row is the same for all lanes. Before the first of a group's go the
  // group's scales, 64 rows to a wave (waves beyond those repeat them).
  const int lr = lane >> 2;
  const uint32_t off_b = opaque(lr * 64 + (((lane & 3) ^ place_b(16 * wave + lr)) << 4));
  const uint32_t off_a = opaque(lr * 64 + (((lane & 3) ^ place_a(lr)) << 4));
  const int last_a = (int)padded_rows(p.M) - 16, last_b = (int)padded_rows(p.N) - 16;
  const int part = wave % kPieces;
  auto fetch_scales = [&](int group, int slot) __attribute__((always_inline)) {
    const uint8_t* from = part < BN / 64 ? p.bs + ((int64_t)group * p.N + c.n0 + 64 * part) * 16
                                         : p.as + ((int64_t)group * p.M + c.m0 + 64 * (part - BN / 64)) * 16;
    dma16_from(from, (uint32_t)lane * 16, l0 + kS + slot * kBytesS + part * 1024);
  };
  const uint8_t* from[kXfer];  // where each transfer goes on
  auto fetch1 = [&](int i, int buf) __attribute__((always_inline)) {
    const uint32_t at = l0 + wave * 1024;
    if (i < kXferB) {
      dma16_from(from[i], off_b, at + buf * kBytesB + i * kWaves * 1024);
      from[i] += p.panel_b;
    } else {
      dma16_from(from[i], off_a, at + kA + buf * kBytesA + (i - kXferB) * kWaves * 1024);
      from[i] += p.panel_a;
    }
  };
  // the first NH of a tile, or as many as there are
  auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kXfer; ++i)
      from[i] = i < kXferB ? p.b + c.lo * p.panel_b + min(c.n0 + 16 * (i * kWaves + wave), last_b) * 64ll
                           : p.a + c.lo * p.panel_a + min(c.m0 + 16 * ((i - kXferB) * kWaves + wave), last_a) * 64ll;
#pragma unroll
    for (int k = 0; k < NH; ++k)
      if (c.lo + k < c.hi) {
        if (k % 4 == 0) fetch_scales((c.lo + k) >> 2, k / 4);
#pragma unroll
        for (int i = 0; i < kXfer; ++i) fetch1(i, k);
      }
  };

  const int rb = 16 * FN * wn + 8 * (r >> 2) + (r & 3), ra = 16 * FM * wm + r;
  const uint32_t read_b = opaque(l0 + rb * 64 + ((q ^ place_b(rb)) << 4));
  const uint32_t read_a = opaque(l0 + kA + ra * 64 + ((q ^ place_a(ra)) << 4));
  const uint32_t read_s = opaque(l0 + kS + rb * 16 + 4 * q), read_sa = opaque(l0 + kS + BN * 16 + ra * 16 + 4 * q);
  auto lds4 = [](uint32_t a) { return *(const __attribute__((address_space(3))) uint32_t*)(a); };

  v4f acc[FN][FM];
  u32x4 fa[FM], fb[2][FN];
  uint32_t sa[FM], sb[FN], sa_next[FM], sb_next[FN];
  auto read_b4 = [&](int i, int buf) __attribute__((always_inline)) {
    return lds16(read_b + buf * kBytesB + 2048 * (i / 2) + 256 * (i % 2));
  };
  auto read_a4 = [&](int j, int buf) __attribute__((always_inline)) { return lds16(read_a + buf * kBytesA + 1024 * j); };
  auto read_scales = [&](int j, uint32_t slot) __attribute__((always_inline)) {  // of FM parts
    sa_next[j] = lds4(read_sa + slot + 256 * j);
#pragma unroll
    for (int i = j; i < FN; i += FM) sb_next[i] = lds4(read_s + slot + 512 * (i / 2) + 64 * (i % 2));
  };
  constexpr int kStores = FN / 2 * FM * Elem<DT>::size / 2;
  constexpr auto at_most = [](int n) { return n < 64 ? n : 63; };
  // Whether stores of the tile before went out behind this one's first transfers
  bool behind = false;
  uint32_t slot = 0;  // of the next group's scales
  // The products of panel h, in buffer k = (h - lo) % NH, whose fragments are there. After the first of them the wave
  // meets the others: h + 1 is there then, and every wave has read h, whose buffer takes h + NH. Fragments of
  // h + 1, transfers and scales go out between the other products (all at once they hold both waves of a SIMD up).
  // steady: NH more come after the four of this call's, and no stores are on their way.
  auto panel = [&](int h, auto number, auto steady) __attribute__((always_inline)) {
    constexpr int k = decltype(number)::value, next = (k + 1) % NH, t = k & 1;
    constexpr int kMeet = FM / 4;
    if constexpr (k % 4 == 0) {
#pragma unroll
      for (int i = 0; i < FN; ++i) sb[i] = sb_next[i];
#pragma unroll
      for (int j = 0; j < FM; ++j) sa[j] = sa_next[j];
      slot = slot + 1 == kSlots ? 0 : slot + 1;
      // Scales, and the sums of a tile's first panel, are vector instructions' results (the sums zeros, which the
      // compiler would otherwise write anew in front of the products): all of them in front of this wait
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        asm volatile("" : "+v"(sb[i]));
#pragma unroll
        for (int j = 0; j < FM; ++j) asm volatile("" : "+v"(acc[i][j]));
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) asm volatile("" : "+v"(sa[j]));
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_nop 3");
    }
    const bool more = decltype(steady)::value || h + NH < c.hi;
    // transfers behind those of h + 1
    constexpr int kGroups = [](int k) {
      int n = 0;
      for (int i = 1; i <= NH - 2; ++i) n += (k + NH - i) % 4 == 0;
      return n;
    }(k);
    constexpr int kBehind = (NH - 2) * kXfer + kGroups;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
#pragma unroll
      for (int i = 0; i < FN; ++i) mfma_in_place<k % 4>(acc[i][j], fb[t][i], fa[j], sb[i], sa[j]);
      if (j < kMeet) continue;
      if (j == kMeet) {
        __builtin_amdgcn_sched_barrier(0);
        wait_lgkmcnt0();
        if (decltype(steady)::value) {
          wait_vmcnt<kBehind>();
        } else if (h + NH <= c.hi) {
          if (k < NH - 1 && behind && h == c.lo + k)
            wait_vmcnt<at_most(kBehind + kStores)>();
          else
            wait_vmcnt<kBehind>();
        } else if (behind && c.hi - c.lo <= NH) {
          wait_vmcnt<at_most(kStores)>();
        } else {
          wait_vmcnt<0>();
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < FN; ++i) fb[1 - t][i] = read_b4(i, next);
#pragma unroll
        for (int i = 0; i < kMeet; ++i) fa[i] = read_a4(i, next);
      }
      fa[j] = read_a4(j, next);
      if constexpr (k % 4 == 3) {
        read_scales(j, slot * kBytesS);
        if (j == kMeet)
#pragma unroll
          for (int i = 0; i < kMeet; ++i) read_scales(i, slot * kBytesS);
      }
      if (more) {
        if (k % 4 == 0 && j == kMeet) fetch_scales((h + NH) >> 2, slot + NH / 4 - 1 < kSlots ? slot + NH / 4 - 1 : slot + NH / 4 - 1 - kSlots);
#pragma unroll
        for (int i = j - kMeet; i < kXfer; i += FM - kMeet) fetch1(i, k);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Sums and bias to y (16 rows of it, or 8, to a buffer whose end is theirs: what lies behind y's last row or column
  // is not stored, without a branch)
  float bias[FN / 2][8];
  const __amdgpu_buffer_rsrc_t biases = __builtin_amdgcn_make_buffer_rsrc((void*)p.bias, 0, p.N * 4, kBufferFlags);
  auto load_bias = [&](const Tile& c) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < FN / 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) bias[u][i] = 0.f;
    if (!p.bias || p.splits > 1) return;
#pragma unroll
    for (int u = 0; u < FN / 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        bias[u][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(biases, (c.n0 + 16 * FN * wn + 32 * u + 8 * q + i) * 4, 0, 0));
#pragma unroll
    for (int u = 0; u < FN / 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(bias[u][i]));  // there before the transfers behind them
  };
  auto save = [&](const Tile& c) __attribute__((always_inline)) {
    constexpr int kSize = Elem<DT>::size;
    uint8_t* y = static_cast<uint8_t*>(p.y) + (int64_t)c.split * p.M * p.N * kSize;
    const int n = c.n0 + 16 * FN * wn, m = c.m0 + 16 * FM * wm;
    auto rows_at = [&](int row, int rows) __attribute__((always_inline)) {
      const uint64_t from = (uint64_t)(y + (int64_t)min(row, p.M) * p.N * kSize);
      const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(from >> 32)) << 32 |
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)from);
      return __builtin_amdgcn_make_buffer_rsrc(
          (void*)base, 0, __builtin_amdgcn_readfirstlane(max(0, min(rows, p.M - row)) * p.N * kSize), kBufferFlags);
    };
    if constexpr (vec) {
      uint32_t off[FN / 2][kSize / 2];
#pragma unroll
      for (int u = 0; u < FN / 2; ++u)
#pragma unroll
        for (int k = 0; k < kSize / 2; ++k) {
          const int col = n + 32 * u + 8 * q + 4 * k;
          off[u][k] = col < p.N ? (uint32_t)(r * p.N + col) * kSize : kNowhere;
        }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const __amdgpu_buffer_rsrc_t rows = rows_at(m + 16 * j, 16);
#pragma unroll
        for (int u = 0; u < FN / 2; ++u) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = acc[2 * u + i / 4][j][i % 4] + bias[u][i];
          if constexpr (DT == DPA_DTYPE_F32) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]),
                                                           __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3])},
                                                     rows, off[u][k], 0, 0);
          } else {
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{Elem<DT>::pack(v[0], v[1]), Elem<DT>::pack(v[2], v[3]),
                                                         Elem<DT>::pack(v[4], v[5]), Elem<DT>::pack(v[6], v[7])},
                                                   rows, off[u][0], 0, 0);
          }
        }
      }
      return;
    }
    // Rows that no vector fits: 8 of them turn in LDS, so that neighbouring lanes store neighbours (each lane its
    // 8 one by one: 3850 x 1023 of 513 in fp32 22.5 us, against 16.3)
    const int col = lane % kCols, at = n + col;
    const uint32_t off = at < p.N ? (uint32_t)(lane / kCols * p.N + at) * kSize : kNowhere;
#pragma unroll
    for (int j = 0; j < 2 * FM; ++j) {
      if ((r >> 3) == (j & 1)) {
#pragma unroll
        for (int i = 0; i < kCols / 16; ++i) {
          v4f v = acc[i][j / 2];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += bias[i / 2][4 * (i % 2) + e];
          *reinterpret_cast<float4*>(turn + (r & 7) * kCols + (((8 * (i / 2) + 2 * q + i % 2) ^ (r & 7)) << 2)) =
              float4{v[0], v[1], v[2], v[3]};
        }
      }
      asm volatile("" ::: "memory");
      const __amdgpu_buffer_rsrc_t rows = rows_at(m + 8 * j, 8);
#pragma unroll
      for (int i = 0; i < 8 * kCols / 64; ++i) {
        const int row = i * (64 / kCols) + lane / kCols;
        const float v = turn[row * kCols + (((col >> 2) ^ row) << 2) + (col & 3)];
        const uint32_t from = off == kNowhere ? off : off + (uint32_t)(i * (64 / kCols) * p.N) * kSize;
        if constexpr (DT == DPA_DTYPE_F32)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rows, from, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b16((uint16_t)Elem<DT>::pack(v, v), rows, from, 0, 0);
      }
      asm volatile("" ::: "memory");
    }
  };
  constexpr int kAhead = (NH - 1) * kXfer + NH / 4 - 1;  // transfers behind a tile's first
  static_assert(kAhead < 64, "vmcnt");
  begin();
  for (uint32_t id = blockIdx.x;;) {
    if (c.lo + NH <= c.hi) {
      if (behind)
        wait_vmcnt<at_most(kAhead + kStores)>();
      else
        wait_vmcnt<kAhead>();
    } else if (behind) {
      wait_vmcnt<at_most(kStores)>();
    } else {
      wait_vmcnt<0>();
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    slot = 0;
#pragma unroll
    for (int j = 0; j < FM; ++j) read_scales(j, 0);
#pragma unroll
    for (int i = 0; i < FN; ++i) fb[0][i] = read_b4(i, 0);
#pragma unroll
    for (int j = 0; j < FM; ++j) fa[j] = read_a4(j, 0);
    int h = c.lo;
    auto four = [&](auto first, auto steady) __attribute__((always_inline)) {  // or two, where the columns end
      constexpr int f = decltype(first)::value;
      panel(h, std::integral_constant<int, f>(), steady);
      panel(h + 1, std::integral_constant<int, f + 1>(), steady);
      if (decltype(steady)::value || h + 2 < c.hi) {
        panel(h + 2, std::integral_constant<int, f + 2>(), steady);
        panel(h + 3, std::integral_constant<int, f + 3>(), steady);
      }
      h += 4;
    };
    typedef std::integral_constant<int, 0> First;
    typedef std::integral_constant<int, 4> Fifth;
    if constexpr (NH == 4) {
      if (behind) four(First(), std::false_type());
      while (h + 4 + NH <= c.hi) four(First(), std::true_type());
      while (h < c.hi) four(First(), std::false_type());
    } else {
      static_assert(NH == 8, "");
      if (behind) {
        four(First(), std::false_type());
        if (h < c.hi) four(Fifth(), std::false_type());
      }
      while (h + 8 + NH <= c.hi) four(First(), std::true_type()), four(Fifth(), std::true_type());
      while (h < c.hi) {
        four(First(), std::false_type());
        if (h < c.hi) four(Fifth(), std::false_type());
      }
    }
    results_ready();
    const Tile done = c;
    id += gridDim.x;
    const bool more = there(id);
    load_bias(done);
    if (more) {  // the next tile's first steps, before this one's stores
      wait_lgkmcnt0();
      lds_barrier();  // every wave is past its reads
      c = tile_of(id);
      begin();
      __builtin_amdgcn_sched_barrier(0);
      behind = vec;
    }
    save(done);
    if (!more) break;
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ---------------------------------------------------------------------------------------
// Up to 16 MT rows of an operand a: bound by the bytes of b, which go straight to registers. A workgroup takes 16
// rows of b; its eight waves take every eighth group of 512 columns, the next group's loads out before this one's
// products, and join their sums in LDS. 16 rows of 8192 into 8192 (36 MB) 7.7 us, 4.7 TB/s, and 2.5 for the rounding of x.
// ---------------------------------------------------------------------------------------
template <int MT, int DT>
__global__ __launch_bounds__(512, MT > 2 ? 2 : 4) void mxfp4_few_kernel(const GemmArgs p) {
  __shared__ float sums[8][MT][4][65];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x / (uint32_t)p.tiles_n, tn = blockIdx.x - split * p.tiles_n;
  const int n0 = tn * 16;
  const int s_lo = split * p.per_split, s_hi = min(p.steps, s_lo + p.per_split);
  const int nb = min(n0 + r, p.N - 1);
  const uint8_t* b = p.b + nb * 64ll + 16 * q;
  const uint8_t* bs = p.bs + nb * 16 + 4 * q;
  const uint8_t *a[MT], *as[MT];
  v4f acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = min(16 * j + r, p.M - 1);
    a[j] = p.a + m * 64ll + 16 * q;
    as[j] = p.as + m * 16 + 4 * q;
    acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  struct Group {
    uint32_t sb, sa[MT];
    u32x4 b[4], a[MT][4];
  };
  auto load = [&](Group& g, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t panel = 2 * s + (t < 2 || s + 1 < p.steps ? t : t - 2);
      g.b[t] = *reinterpret_cast<const u32x4*>(b + panel * p.panel_b);
#pragma unroll
      for (int j = 0; j < MT; ++j) g.a[j][t] = *reinterpret_cast<const u32x4*>(a[j] + panel * p.panel_a);
    }
    g.sb = *reinterpret_cast<const uint32_t*>(bs + (int64_t)(s >> 1) * p.N * 16);
#pragma unroll
    for (int j = 0; j < MT; ++j) g.sa[j] = *reinterpret_cast<const uint32_t*>(as[j] + (int64_t)(s >> 1) * p.M * 16);
  };
  auto multiply = [&](const Group& g, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      acc[j] = mfma<0, 0>(g.b[0], g.a[j][0], acc[j], g.sb, g.sa[j]);
      acc[j] = mfma<1, 1>(g.b[1], g.a[j][1], acc[j], g.sb, g.sa[j]);
    }
    if (s + 1 < p.steps)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        acc[j] = mfma<2, 2>(g.b[2], g.a[j][2], acc[j], g.sb, g.sa[j]);
        acc[j] = mfma<3, 3>(g.b[3], g.a[j][3], acc[j], g.sb, g.sa[j]);
      }
  };
  Group g0, g1;
  int s = s_lo + 2 * wave;
  if (s < s_hi) load(g0, s);
  for (; s < s_hi; s += 32) {
    if (s + 16 < s_hi) load(g1, s + 16);
    multiply(g0, s);
    if (s + 16 >= s_hi) break;
    if (s + 32 < s_hi) load(g0, s + 32);
    multiply(g1, s + 16);
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int t = 0; t < 4; ++t) sums[wave][j][t][lane] = acc[j][t];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * MT; e += 512) {
    const int j = e >> 8, m = 16 * j + ((e >> 4) & 15), c = e & 15, n = n0 + c;
    if (m >= p.M || n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sums[w][j][c & 3][(c >> 2) * 16 + (m & 15)];
    if (p.splits > 1)
      p.part[((int64_t)split * p.M + m) * p.N + n] = v;
    else
      store1<DT>(p.y, (int64_t)m * p.N + n, v + (p.bias ? p.bias[n] : 0.f));
  }
}

// ---------------------------------------------------------------------------------------
// Up to 16 rows of x itself. A lane of the matrix instruction takes 32 neighbours of a row, which are a block:
// it finds their scale and rounds them in its own registers, with nothing to exchange. Eight waves take every
// eighth group of 512 columns of 16 NT rows of b; the rounding of x, repeated by every workgroup, hides
// behind the loads of b. One row of 512 into 2048 3.5 us, of which a launch of nothing takes two.
// ---------------------------------------------------------------------------------------
template <int DT>
struct XBlock {  // 32 neighbours as they lie in memory
  uint4 w[4 * Elem<DT>::size / 2];
};

template <int DT>
__device__ __forceinline__ XBlock<DT> load_block(const uint8_t* x, int left) {
  constexpr int kPer = 16 / Elem<DT>::size;  // elements of 16 B
  XBlock<DT> b;
#pragma unroll
  for (int i = 0; i < 32 / kPer; ++i)
    b.w[i] = kPer * i < left ? *reinterpret_cast<const uint4*>(x + 16 * i) : uint4{0u, 0u, 0u, 0u};
  return b;
}

template <int DT>
__device__ __forceinline__ u32x4 round_block(const XBlock<DT>& b, uint32_t& byte) {
  uint32_t r[4];
  if constexpr (DT == DPA_DTYPE_F32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m = max(max(max(m, b.w[i].x & 0x7fffffffu), b.w[i].y & 0x7fffffffu), max(b.w[i].z & 0x7fffffffu, b.w[i].w & 0x7fffffffu));
    byte = scale_byte<false>(m);
    const float s = scale_bits(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = b.w[2 * i], v = b.w[2 * i + 1];
      r[i] = encode_pair<0>(0u, __uint_as_float(u.x), __uint_as_float(u.y), s);
      r[i] = encode_pair<1>(r[i], __uint_as_float(u.z), __uint_as_float(u.w), s);
      r[i] = encode_pair<2>(r[i], __uint_as_float(v.x), __uint_as_float(v.y), s);
      r[i] = encode_pair<3>(r[i], __uint_as_float(v.z), __uint_as_float(v.w), s);
    }
  } else {
    us2 a = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) a = absmax8(a, b.w[i]);
    const uint32_t m = a.x > a.y ? a.x : a.y;
    byte = scale_byte<false>(DT == DPA_DTYPE_BF16 ? m << 16 : __float_as_uint(Elem<DT>::lo(m)));
    const float s = scale_bits(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = encode_pair<DT, 0>(0u, b.w[i].x, s);
      r[i] = encode_pair<DT, 1>(r[i], b.w[i].y, s);
      r[i] = encode_pair<DT, 2>(r[i], b.w[i].z, s);
      r[i] = encode_pair<DT, 3>(r[i], b.w[i].w, s);
    }
  }
  return u32x4{r[0], r[1], r[2], r[3]};
}

template <int NT, int DX, int DT>
__global__ __launch_bounds__(512, 2) void mxfp4_token_kernel(const GemmArgs p) {
  __shared__ float sums[8][NT][4][65];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x / (uint32_t)p.tiles_n, tn = blockIdx.x - split * p.tiles_n;
  const int n0 = tn * 16 * NT;
  const int s_lo = split * p.per_split, s_hi = min(p.steps, s_lo + p.per_split);
  const uint8_t *b[NT], *bs[NT];
  v4f acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int row = min(n0 + 16 * i + r, p.N - 1);
    b[i] = p.b + row * 64ll + 16 * q;
    bs[i] = p.bs + row * 16 + 4 * q;
    acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  const uint8_t* x = static_cast<const uint8_t*>(p.x) + min(r, p.M - 1) * p.ld * Elem<DX>::size;
  uint32_t sb[NT], sb_next[NT];
  u32x4 fb[NT][4], fb_next[NT][4];
  auto fetch = [&](int s, uint32_t(&sc)[NT], u32x4(&f)[NT][4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        f[i][t] = *reinterpret_cast<const u32x4*>(b[i] + (2 * s + (t < 2 || s + 1 < p.steps ? t : t - 2)) * p.panel_b);
      sc[i] = *reinterpret_cast<const uint32_t*>(bs[i] + (int64_t)(s >> 1) * p.N * 16);
    }
  };
  int s = s_lo + 2 * wave;
  if (s < s_hi) fetch(s, sb, fb);
  for (; s < s_hi; s += 16) {
    XBlock<DX> xb[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int col = s * 256 + 128 * t + 32 * q;
      xb[t] = load_block<DX>(x + (int64_t)col * Elem<DX>::size, p.K - col);
    }
    if (s + 16 < s_hi) fetch(s + 16, sb_next, fb_next);
    uint32_t byte;
    u32x4 fa = round_block<DX>(xb[0], byte);
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = mfma<0, 0>(fb[i][0], fa, acc[i], sb[i], byte);
    fa = round_block<DX>(xb[1], byte);
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = mfma<1, 0>(fb[i][1], fa, acc[i], sb[i], byte);
    if (s + 1 < p.steps) {
      fa = round_block<DX>(xb[2], byte);
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i] = mfma<2, 0>(fb[i][2], fa, acc[i], sb[i], byte);
      fa = round_block<DX>(xb[3], byte);
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i] = mfma<3, 0>(fb[i][3], fa, acc[i], sb[i], byte);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      sb[i] = sb_next[i];
#pragma unroll
      for (int t = 0; t < 4; ++t) fb[i][t] = fb_next[i][t];
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int t = 0; t < 4; ++t) sums[wave][i][t][lane] = acc[i][t];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * NT; e += 512) {
    const int i = e >> 8, m = (e >> 4) & 15, c = e & 15, n = n0 + 16 * i + c;
    if (m >= p.M || n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sums[w][i][c & 3][(c >> 2) * 16 + m];
    if (p.splits > 1)
      p.part[((int64_t)split * p.M + m) * p.N + n] = v;
    else
      store1<DT>(p.y, (int64_t)m * p.N + n, v + (p.bias ? p.bias[n] : 0.f));
  }
}

// The splits' sums, in order, eight loads out at a time; kPer neighbours to a thread
template <int DT, int kPer>
__global__ __launch_bounds__(256) void mxfp4_join_kernel(const GemmArgs p) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * kPer, n = (int64_t)p.M * p.N;
  if (i >= n) return;
  typedef float vec __attribute__((ext_vector_type(kPer)));
  vec v = 0.f;
  for (int s = 0; s < p.splits; s += 8) {  // (past the last one: that one again, not added)
    vec x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const vec*>(p.part + min(s + k, p.splits - 1) * n + i);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s + k < p.splits) v += x[k];
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    float y = v[k];
    if (p.bias) y += p.bias[(i + k) % p.N];
    store1<DT>(p.y, i + k, y);
  }
}

// ---- host ------------------------------------------------------------------------------
constexpr int kFewRows = 64;

// Scales are addressed by 32-bit offsets of 16 B a row, tiles' rows by offsets of 256 rows
static int check_gemm(int64_t M, int64_t N, int64_t K) {
  // (16 rows of N columns are within the 2^31 bytes of a buffer)
  if (M < 0 || N < 0 || K <= 0 || M >= 1 << 26 || N >= 1 << 25 || K > 1 << 24) return DPA_ERR_SIZE;
  if (M * N >= 1ll << 36 || ceil_div(M, 128) * ceil_div(N, 16) >= kMaxGroups256 / 2) return DPA_ERR_SIZE;
  return DPA_OK;
}

// The forms of the product: 256 x 256 tiles by 8 waves, one workgroup to a CU; 128 x 128 by 4, two to a CU; 64 x 64
// by 4 with eight panels on their way, two to a CU, for little work, whose time is that of the loads' way. And how
// often the contraction is split. All by what they cost, in us: a round of workgroups tile_us and step_us for each
// step of 256 columns (step_few_us where a CU has one workgroup), a split's sums their bytes twice and a launch.
// Measured (us, 256 / 128 / 64; one after the other without a pause): 4096 x 8192 of 8192 138, 162, 229; 8192 x 4096
// of 4096 69, 79, 126; 32768 x 768 of 256 17.7, 14.9, 22.3; 2048 x 2048 of 2048 19.4, 10.1, 12.4; 512 x 4096 of 4096
// 27.4, 12.8, 10.0; 1024 x 1024 of 1024 12.9, 6.8, 5.6; 3840 x 1024 of 512 11.5, 6.8, 7.4.
struct Form {
  int side, per_cu;
  double tile_us, step_us, step_few_us;
};
constexpr Form kForms[3] = {{256, 1, 8.5, 1.65, 1.3}, {128, 2, 3.0, 1.15, 0.7}, {64, 2, 2.2, 0.43, 0.4}};
constexpr int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64};

static void plan_tiles(GemmArgs& p) {
  double best = 0.0;
  for (int f = 0; f < 3; ++f) {
    const Form& form = kForms[f];
    const int tm = (int)ceil_div(p.M, form.side), tn = (int)ceil_div(p.N, form.side);
    const int64_t tiles = (int64_t)tm * tn, cus = num_cus(), slots = cus * form.per_cu;
    for (const int n : kSplits) {
      if (n > 1 && (n * 4 > p.steps || n * tiles > slots)) break;
      const int per = (p.steps + 2 * n - 1) / (2 * n) * 2, splits = (p.steps + per - 1) / per;
      const int64_t rounds = (tiles * splits + slots - 1) / slots;
      double us = (double)rounds * (form.tile_us + std::min(per, p.steps) * (tiles * splits > cus ? form.step_us : form.step_few_us));
      if (splits > 1) us += 2.5 + (double)splits * p.M * p.N * 4 * 2 * 2e-7;
      if (best == 0.0 || us < best) {
        best = us;
        p.form = f, p.tiles_m = tm, p.tiles_n = tn, p.per_split = per, p.splits = splits;
      }
    }
  }
}

// The operand a laid out, or x itself (`token`)
static GemmArgs plan(int64_t M, int64_t N, int64_t K, bool token) {
  GemmArgs p{};
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  p.panel_a = panel_of(M), p.panel_b = panel_of(N);
  p.steps = (int)(pitch_of(K) / 128);
  if (!token && M > kFewRows) {
    plan_tiles(p);
    return p;
  }
  p.tiles_m = 1;
  p.tiles_n = (int)ceil_div(N, token && N >= 32 * num_cus() ? 32 : 16);
  int64_t n = p.tiles_n > 0 ? num_cus() / p.tiles_n : 1;
  if (n > p.steps / 32) n = p.steps / 32;
  if (n < 1) n = 1;
  p.per_split = (int)(ceil_div(ceil_div(p.steps, n), 2) * 2);
  p.splits = (int)ceil_div(p.steps, p.per_split);
  return p;
}

static int64_t part_bytes(const GemmArgs& p) { return p.splits > 1 ? (int64_t)p.splits * p.M * p.N * 4 : 0; }

static int64_t align256(int64_t n) { return (n + 255) & ~255ll; }

template <int DT>
static int join(const GemmArgs& p, hipStream_t s) {
  const int st = launch_status();
  if (st != DPA_OK || p.splits == 1) return st;
  const int64_t n = (int64_t)p.M * p.N;
  if (n % 4 == 0)
    mxfp4_join_kernel<DT, 4><<<(unsigned)ceil_div(n, 1024), 256, 0, s>>>(p);
  else
    mxfp4_join_kernel<DT, 1><<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(p);
  return launch_status();
}

// Whether 16 B of y at a time fit its rows
static bool whole_vectors(int64_t N, int dtype) { return N % (16 / size_of(dtype)) == 0; }

// The form for a y that vectors fit or not, and its workgroups
static unsigned settle(GemmArgs& p, bool vec) {
  // (The largest tiles leave no registers to turn rows. plan_tiles does not know y: such a product is costed as one of 256 x 256
  // tiles, keeps its splits, of which large ones have none, and runs as 128 x 128. Other choices were not measured.)
  if (!vec && p.form == 0) {
    p.form = 1;
    p.tiles_m = (int)ceil_div(p.M, kForms[1].side), p.tiles_n = (int)ceil_div(p.N, kForms[1].side);
  }
  const int64_t items = ceil_div((int64_t)p.tiles_m * p.tiles_n * p.splits, 8) * 8;
  return (unsigned)std::min<int64_t>(items, kForms[p.form].per_cu * num_cus() / 8 * 8);
}

template <int DT>
static int run_tiles(GemmArgs p, hipStream_t s) {
  const bool vec = whole_vectors(p.N, DT) && aligned(p.y, 16);
  const unsigned grid = settle(p, vec);
  if (p.form == 0)
    mxfp4_gemm_kernel<2, 4, 8, 4, 4, DT, true><<<grid, 512, 0, s>>>(p);
  else if (p.form == 1)
    vec ? mxfp4_gemm_kernel<2, 2, 4, 4, 4, DT, true><<<grid, 256, 0, s>>>(p) : mxfp4_gemm_kernel<2, 2, 4, 4, 4, DT, false><<<grid, 256, 0, s>>>(p);
  else
    vec ? mxfp4_gemm_kernel<2, 2, 2, 2, 8, DT, true><<<grid, 256, 0, s>>>(p) : mxfp4_gemm_kernel<2, 2, 2, 2, 8, DT, false><<<grid, 256, 0, s>>>(p);
  return launch_status();
}

template <int DT>
static int run_gemm(const GemmArgs& p, hipStream_t s) {
  if (p.M <= kFewRows) {
    const unsigned grid = (unsigned)(p.tiles_n * p.splits);
    if (p.M <= 16)
      mxfp4_few_kernel<1, DT><<<grid, 512, 0, s>>>(p);
    else if (p.M <= 32)
      mxfp4_few_kernel<2, DT><<<grid, 512, 0, s>>>(p);
    else
      mxfp4_few_kernel<4, DT><<<grid, 512, 0, s>>>(p);
  } else {
    GemmArgs g = p;
    if (p.splits > 1) g.y = p.part;
    const int st = p.splits > 1 ? run_tiles<DPA_DTYPE_F32>(g, s) : run_tiles<DT>(g, s);
    if (st != DPA_OK) return st;
  }
  return join<DT>(p, s);
}

template <int DX, int DT>
static int run_token(const GemmArgs& p, hipStream_t s) {
  const unsigned grid = (unsigned)(p.tiles_n * p.splits);
  if (p.N >= 32 * num_cus())
    mxfp4_token_kernel<2, DX, DT><<<grid, 512, 0, s>>>(p);
  else
    mxfp4_token_kernel<1, DX, DT><<<grid, 512, 0, s>>>(p);
  return join<DT>(p, s);
}

template <int DX>
static int run_token(const GemmArgs& p, int dtype, hipStream_t s) {
  if (dtype == DPA_DTYPE_BF16) return run_token<DX, DPA_DTYPE_BF16>(p, s);
  if (dtype == DPA_DTYPE_F16) return run_token<DX, DPA_DTYPE_F16>(p, s);
  return run_token<DX, DPA_DTYPE_F32>(p, s);
}

static int run(const GemmArgs& p, int dtype, hipStream_t s) {
  if (dtype == DPA_DTYPE_BF16) return run_gemm<DPA_DTYPE_BF16>(p, s);
  if (dtype == DPA_DTYPE_F16) return run_gemm<DPA_DTYPE_F16>(p, s);
  return run_gemm<DPA_DTYPE_F32>(p, s);
}

// Whether the rows of x are read by 16-B vectors within the product's launch
static bool takes_token(const void* x, int dtype, int64_t ld, int64_t M, int64_t K) {
  const int per = 16 / size_of(dtype);
  // (every workgroup reads and rounds all of x: 16 x 8192 into 8192 columns 17.3 us, laid out first 11.5 + 3.2)
  return M <= 16 && M * K * size_of(dtype) <= 65536 && K % per == 0 && (M == 1 || ld % per == 0) && aligned(x, 16);
}

}  // namespace mx
}  // namespace dpa

using namespace dpa;
using namespace dpa::mx;

extern "C" int dpa_mxfp4_gemm_plan(int64_t M, int64_t N, int64_t K, int dtype, DpaMxfp4GemmPlan* out) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  const int st = check_gemm(M, N, K);
  if (st != DPA_OK || !out) return st;
  *out = DpaMxfp4GemmPlan{};
  if (M == 0 || N == 0) return DPA_OK;
  GemmArgs p = plan(M, N, K, false);
  out->splits = p.splits;
  if (M <= kFewRows) {
    out->workgroups = p.tiles_n * p.splits;
    out->tiles = out->workgroups;
    return DPA_OK;
  }
  out->vectors = whole_vectors(N, p.splits > 1 ? DPA_DTYPE_F32 : dtype);
  out->workgroups = (int32_t)settle(p, out->vectors != 0);
  out->side = kForms[p.form].side;
  out->tiles = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  return DPA_OK;
}

extern "C" int64_t dpa_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  return check_gemm(M, N, K) == DPA_OK ? part_bytes(plan(M, N, K, false)) : 0;
}

extern "C" int dpa_mxfp4_gemm(const void* a, const void* b, const float* bias, void* y, int dtype, int64_t M, int64_t N,
                              int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  const int st = check_gemm(M, N, K);
  if (st != DPA_OK) return st;
  if (M == 0 || N == 0) return DPA_OK;
  if (!a || !b || !y) return DPA_ERR_NULL;
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(bias, 4) || !aligned(y, size_of(dtype))) return DPA_ERR_ALIGN;
  GemmArgs p = plan(M, N, K, false);
  p.a = (const uint8_t*)a, p.as = p.a + operand_data_bytes(M, K);
  p.b = (const uint8_t*)b, p.bs = p.b + operand_data_bytes(N, K);
  p.bias = bias, p.y = y;
  if (p.splits > 1) {
    if (!workspace || workspace_bytes < part_bytes(p)) return DPA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
    p.part = (float*)workspace;
  }
  return run(p, dtype, (hipStream_t)stream);
}

extern "C" int64_t dpa_mxfp4_linear_workspace_bytes(const void* x, int x_dtype, int64_t row_stride, int64_t M, int64_t N,
                                                    int64_t K) {
  if (!dtype_ok(x_dtype) || check_gemm(M, N, K) != DPA_OK || M == 0) return 0;
  if (takes_token(x, x_dtype, row_stride, M, K)) return part_bytes(plan(M, N, K, true));
  return align256(operand_bytes(M, K)) + part_bytes(plan(M, N, K, false));
}

extern "C" int dpa_mxfp4_linear(const void* x, int x_dtype, int64_t row_stride, const void* weight, const float* bias,
                                void* y, int dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(x_dtype) || !dtype_ok(dtype)) return DPA_ERR_SHAPE;
  const int st = check_gemm(M, N, K);
  if (st != DPA_OK) return st;
  if (!matrix_ok(M, K) || (row_stride < K && M > 1)) return DPA_ERR_SIZE;
  if (M == 0 || N == 0) return DPA_OK;
  if (!x || !weight || !y) return DPA_ERR_NULL;
  if (!aligned(x, size_of(x_dtype)) || !aligned(weight, 16) || !aligned(bias, 4) || !aligned(y, size_of(dtype)))
    return DPA_ERR_ALIGN;
  const int64_t need = dpa_mxfp4_linear_workspace_bytes(x, x_dtype, row_stride, M, N, K);
  if (need && (!workspace || workspace_bytes < need)) return DPA_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
  uint8_t* ws = (uint8_t*)workspace;
  hipStream_t s = (hipStream_t)stream;
  const bool token = takes_token(x, x_dtype, row_stride, M, K);
  GemmArgs p = plan(M, N, K, token);
  p.b = (const uint8_t*)weight, p.bs = p.b + operand_data_bytes(N, K);
  p.bias = bias, p.y = y;
  if (token) {
    p.x = x, p.ld = row_stride, p.part = (float*)ws;
    if (x_dtype == DPA_DTYPE_BF16) return run_token<DPA_DTYPE_BF16>(p, dtype, s);
    if (x_dtype == DPA_DTYPE_F16) return run_token<DPA_DTYPE_F16>(p, dtype, s);
    return run_token<DPA_DTYPE_F32>(p, dtype, s);
  }
  const int quantized = dpa_mxfp4_operands(x, x_dtype, M, K, row_stride, ws, nullptr, nullptr, nullptr, stream);
  if (quantized != DPA_OK) return quantized;
  p.a = ws, p.as = p.a + operand_data_bytes(M, K);
  p.part = (float*)(ws + align256(operand_bytes(M, K)));
  return run(p, dtype, s);
}
