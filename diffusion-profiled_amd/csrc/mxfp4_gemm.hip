// y[M][N] = a[M][K] b[N][K]^T (+ bias) over MXFP4 operands (format: mxfp4.hpp), sums in fp32.
#include <type_traits>

#include "mxfp4.hpp"

namespace dpa {
namespace mx {

struct GemmArgs {
  const uint8_t *a, *as, *b, *bs;  // rows of M and of N
  const float* bias;
  void* y;
  float* part;  // [splits][M][N] where the contraction is split
  int64_t pitch;
  const void* x;  // a before its rounding, where the kernel does that, rows ld elements apart
  int64_t ld;
  int M, N, K;
  int steps, per_split, splits;  // of 256 columns; per_split is even
  int tiles_m, tiles_n;
};

// v[0 .. 15] to columns n0 .. n0 + 15 of a row
template <int DT>
__device__ __forceinline__ void store16(void* y, int64_t row, int n0, int N, bool vec, const float (&v)[16]) {
  const int64_t at = row * N + n0;
  if (vec && n0 + 16 <= N) {
    if constexpr (DT == DPA_DTYPE_F32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(y) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = float4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    } else {
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + at);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        o[i] = uint4{Elem<DT>::pack(v[8 * i], v[8 * i + 1]), Elem<DT>::pack(v[8 * i + 2], v[8 * i + 3]),
                     Elem<DT>::pack(v[8 * i + 4], v[8 * i + 5]), Elem<DT>::pack(v[8 * i + 6], v[8 * i + 7])};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (n0 + i < N) store1<DT>(y, at + i, v[i]);
}

// ---------------------------------------------------------------------------------------
// Tiles of BM x BN, WM x WN waves of 64 x 64 each, steps of 256 columns (128 B of a row) through LDS by
// DMA, double-buffered. b's rows are the A operand (rows of D), in the order that gives a lane 16 columns of y in
// a row: row r of fragment i is row 16 (r / 4) + 4 i + r % 4 of the wave's 64. The 16-B piece c of a
// row lies at c ^ swz(row): the 16 lanes that LDS serves together (rows 0-3 and 12-15 at one piece,
// 4-11 at the piece two further) then lie in 16 different places of the banks.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ int swz_b(int r) { return ((r >> 1) & 1) | ((r >> 4) & 2) | (((r >> 2) ^ (r >> 3)) & 4); }
__device__ __forceinline__ int swz_a(int r) { return ((r >> 1) & 1) | ((r >> 2) & 2) | ((r ^ (r >> 1)) & 4); }

__device__ __forceinline__ u32x4 lds16(uint32_t a) { return *(const __attribute__((address_space(3))) u32x4*)(a); }

__device__ __forceinline__ void dma16_from(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0");
}

template <int WM, int WN, int DT>
__global__ __launch_bounds__(64 * WM * WN) void mxfp4_gemm_kernel(const GemmArgs p, bool vec) {
  constexpr int kWaves = WM * WN, BM = 64 * WM, BN = 64 * WN;
  constexpr uint32_t kB = BN * 128, kBuf = (BM + BN) * 128;
  constexpr int kXferB = BN / 8 / kWaves, kXferA = BM / 8 / kWaves;
  static_assert(BN % (8 * kWaves) == 0 && BM % (8 * kWaves) == 0, "transfers of 8 rows");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kBuf];
  const uint32_t l0 = LDS_ADDR(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM, r = lane & 15, q = lane >> 4;
  uint32_t id = blockIdx.x;
  const int split = id / (uint32_t)(p.tiles_m * p.tiles_n);
  id -= split * (uint32_t)(p.tiles_m * p.tiles_n);
  const int tn = id / (uint32_t)p.tiles_m, tm = id - tn * p.tiles_m;
  const int m0 = tm * BM, n0 = tn * BN;
  const int s_lo = split * p.per_split, s_hi = min(p.steps, s_lo + p.per_split);

  const uint8_t *ab = p.a + m0 * p.pitch, *bb = p.b + n0 * p.pitch;
  uint32_t off_a[kXferA], off_b[kXferB];
#pragma unroll
  for (int i = 0; i < kXferB; ++i) {
    const int row = 8 * (i * kWaves + wave) + (lane >> 3);
    off_b[i] = (uint32_t)(min(row, p.N - 1 - n0) * p.pitch) + (((lane & 7) ^ swz_b(row)) << 4);
  }
#pragma unroll
  for (int i = 0; i < kXferA; ++i) {
    const int row = 8 * (i * kWaves + wave) + (lane >> 3);
    off_a[i] = (uint32_t)(min(row, p.M - 1 - m0) * p.pitch) + (((lane & 7) ^ swz_a(row)) << 4);
  }
  auto fetch = [&](int step, int buf) __attribute__((always_inline)) {
    const uint32_t at = l0 + buf * kBuf + wave * 1024;
#pragma unroll
    for (int i = 0; i < kXferB; ++i) dma16_from(bb + step * 128ll, off_b[i], at + i * kWaves * 1024);
#pragma unroll
    for (int i = 0; i < kXferA; ++i) dma16_from(ab + step * 128ll, off_a[i], at + kB + i * kWaves * 1024);
  };
  // scales of this lane's rows, by fragment
  uint32_t at_a[4], at_b[4], sa[4], sb[4], sa_next[4], sb_next[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    at_b[i] = min(n0 + 64 * wn + 16 * (r >> 2) + 4 * i + (r & 3), p.N - 1) * 16 + 4 * q;
    at_a[i] = min(m0 + 64 * wm + 16 * i + r, p.M - 1) * 16 + 4 * q;
  }
  auto fetch_scales = [&](int group) __attribute__((always_inline)) {
    const uint8_t *ga = p.as + (int64_t)group * p.M * 16, *gb = p.bs + (int64_t)group * p.N * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sa_next[i] = *reinterpret_cast<const uint32_t*>(ga + at_a[i]);
      sb_next[i] = *reinterpret_cast<const uint32_t*>(gb + at_b[i]);
    }
  };

  const int rb = 64 * wn + 16 * (r >> 2) + (r & 3), ra = 64 * wm + r;
  uint32_t read_b[2], read_a[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    read_b[t] = l0 + rb * 128 + (((2 * q + t) ^ swz_b(rb)) << 4);
    read_a[t] = l0 + kB + ra * 128 + (((2 * q + t) ^ swz_a(ra)) << 4);
  }

  v4f acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  auto half = [&](auto buffer, auto piece) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value, t = decltype(piece)::value;
    u32x4 fb[4], fa[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) fb[i] = lds16(read_b[t] + buf * kBuf + 512 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) fa[j] = lds16(read_a[t] + buf * kBuf + 2048 * j);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i][j] = mfma<2 * buf + t, 2 * buf + t>(fb[i], fa[j], acc[i][j], sb[i], sa[j]);
  };
  auto step = [&](int s, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    wait_vmcnt<0>();
    lds_barrier();  // step s is there, and every wave is past its reads of the other buffer
    if constexpr (buf == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = sa_next[i], sb[i] = sb_next[i];
    }
    if (s + 1 < s_hi) {
      if constexpr (buf == 1) fetch_scales((s + 1) >> 1);
      fetch(s + 1, buf ^ 1);
    }
    half(buffer, std::integral_constant<int, 0>());
    half(buffer, std::integral_constant<int, 1>());
  };
  fetch_scales(s_lo >> 1);
  fetch(s_lo, 0);
  for (int s = s_lo; s < s_hi; s += 2) {
    step(s, std::integral_constant<int, 0>());
    if (s + 1 < s_hi) step(s + 1, std::integral_constant<int, 1>());
  }

  const int n = n0 + 64 * wn + 16 * q;
  float bias[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) bias[i] = p.bias && p.splits == 1 && n + i < p.N ? p.bias[n + i] : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 64 * wm + 16 * j + r;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = acc[i / 4][j][i % 4] + bias[i];
    if (m >= p.M) continue;
    if (p.splits > 1)
      store16<DPA_DTYPE_F32>(p.part, (int64_t)split * p.M + m, n, p.N, vec, v);
    else
      store16<DT>(p.y, m, n, p.N, vec, v);
  }
}

// ---------------------------------------------------------------------------------------
// Up to 16 MT rows of an operand a: bound by the bytes of b, which go straight to registers. A workgroup takes 16
// rows of b; its four waves take every fourth group of 512 columns and join their sums in LDS.
// ---------------------------------------------------------------------------------------
template <int MT, int DT>
__global__ __launch_bounds__(256) void mxfp4_few_kernel(const GemmArgs p) {
  __shared__ float sums[4][MT][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x / (uint32_t)p.tiles_n, tn = blockIdx.x - split * p.tiles_n;
  const int n0 = tn * 16;
  const int s_lo = split * p.per_split, s_hi = min(p.steps, s_lo + p.per_split);
  const int nb = min(n0 + r, p.N - 1);
  const uint8_t* b = p.b + nb * p.pitch + 32 * q;
  const uint8_t* bs = p.bs + nb * 16 + 4 * q;
  const uint8_t *a[MT], *as[MT];
  v4f acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = min(16 * j + r, p.M - 1);
    a[j] = p.a + m * p.pitch + 32 * q;
    as[j] = p.as + m * 16 + 4 * q;
    acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  for (int s = s_lo + 2 * wave; s < s_hi; s += 8) {
    const int64_t g = s >> 1;
    const uint32_t sb = *reinterpret_cast<const uint32_t*>(bs + g * p.N * 16);
    uint32_t sa[MT];
    u32x4 fb[4], fa[MT][4];
    const bool both = s + 1 < p.steps;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t at = (t < 2 || both ? s + t / 2 : s) * 128ll + 16 * (t & 1);
      fb[t] = *reinterpret_cast<const u32x4*>(b + at);
#pragma unroll
      for (int j = 0; j < MT; ++j) fa[j][t] = *reinterpret_cast<const u32x4*>(a[j] + at);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) sa[j] = *reinterpret_cast<const uint32_t*>(as[j] + g * p.M * 16);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      acc[j] = mfma<0, 0>(fb[0], fa[j][0], acc[j], sb, sa[j]);
      acc[j] = mfma<1, 1>(fb[1], fa[j][1], acc[j], sb, sa[j]);
    }
    if (both)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        acc[j] = mfma<2, 2>(fb[2], fa[j][2], acc[j], sb, sa[j]);
        acc[j] = mfma<3, 3>(fb[3], fa[j][3], acc[j], sb, sa[j]);
      }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int t = 0; t < 4; ++t) sums[wave][j][t][lane] = acc[j][t];
  __syncthreads();
  // wave t: element t of each lane's four
  const int t = wave, n = n0 + 4 * q + t;
  if (n >= p.N) return;
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = 16 * j + r;
    if (m >= p.M) continue;
    const float v = (sums[0][j][t][lane] + sums[1][j][t][lane]) + (sums[2][j][t][lane] + sums[3][j][t][lane]);
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
// behind the loads of b.
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
    b[i] = p.b + row * p.pitch + 32 * q;
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
        f[i][t] = *reinterpret_cast<const u32x4*>(b[i] + (t < 2 || s + 1 < p.steps ? s + t / 2 : s) * 128ll + 16 * (t & 1));
      sc[i] = *reinterpret_cast<const uint32_t*>(bs[i] + (int64_t)(s >> 1) * p.N * 16);
    }
  };
  int s = s_lo + 2 * wave;
  if (s < s_hi) fetch(s, sb, fb);
  for (; s < s_hi; s += 16) {
    XBlock<DX> xb[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int col = s * 256 + 256 * (t >> 1) + 64 * q + 32 * (t & 1);
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

// The splits' sums, in order
template <int DT>
__global__ __launch_bounds__(256) void mxfp4_join_kernel(const GemmArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.M * p.N;
  if (i >= n) return;
  float v = 0.f;
  for (int s = 0; s < p.splits; ++s) v += p.part[s * n + i];
  if (p.bias) v += p.bias[i % p.N];
  store1<DT>(p.y, i, v);
}

// ---- host ------------------------------------------------------------------------------
constexpr int kFewRows = 64;

// Scales are addressed by 32-bit offsets of 16 B a row, tiles' rows by offsets of 256 rows
static int check_gemm(int64_t M, int64_t N, int64_t K) {
  const int64_t most = 1ll << 26;
  if (M < 0 || N < 0 || K <= 0 || M >= most || N >= most || K > 1 << 24) return DPA_ERR_SIZE;
  if (M * N >= 1ll << 36 || ceil_div(M, 128) * ceil_div(N, 16) >= kMaxGroups256 / 2) return DPA_ERR_SIZE;
  return DPA_OK;
}

// The operand a laid out, or x itself (`token`)
static GemmArgs plan(int64_t M, int64_t N, int64_t K, bool token) {
  GemmArgs p{};
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  p.pitch = pitch_of(K);
  p.steps = (int)(p.pitch / 128);
  const bool few = token || M <= kFewRows;
  const int width = token && N >= 32 * num_cus() ? 32 : few ? 16 : 128;
  p.tiles_m = few ? 1 : (int)ceil_div(M, 128);
  p.tiles_n = (int)ceil_div(N, width);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, want = (token ? 1 : 2) * num_cus();
  int64_t n = tiles > 0 ? want / tiles : 1;
  const int64_t least = token ? 32 : few ? 8 : 4;
  if (n > p.steps / least) n = p.steps / least;
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
  mxfp4_join_kernel<DT><<<(unsigned)ceil_div((int64_t)p.M * p.N, 256), 256, 0, s>>>(p);
  return launch_status();
}

template <int DT>
static int run_gemm(const GemmArgs& p, hipStream_t s) {
  const int elems = p.splits > 1 || DT == DPA_DTYPE_F32 ? 4 : 8;
  const bool vec = p.N % elems == 0 && (p.splits > 1 || aligned(p.y, 16));
  if (p.M <= kFewRows) {
    const unsigned grid = (unsigned)(p.tiles_n * p.splits);
    if (p.M <= 16)
      mxfp4_few_kernel<1, DT><<<grid, 256, 0, s>>>(p);
    else if (p.M <= 32)
      mxfp4_few_kernel<2, DT><<<grid, 256, 0, s>>>(p);
    else
      mxfp4_few_kernel<4, DT><<<grid, 256, 0, s>>>(p);
  } else {
    mxfp4_gemm_kernel<2, 2, DT><<<(unsigned)(p.tiles_m * p.tiles_n * p.splits), 256, 0, s>>>(p, vec);
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
  return M <= 16 && K % per == 0 && (M == 1 || ld % per == 0) && aligned(x, 16);
}

}  // namespace mx
}  // namespace dpa

using namespace dpa;
using namespace dpa::mx;

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

extern "C" int64_t dpa_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (check_gemm(M, N, K) != DPA_OK || M == 0) return 0;
  const int64_t two = align256(operand_bytes(M, K)) + part_bytes(plan(M, N, K, false));
  const int64_t one = M <= 16 ? part_bytes(plan(M, N, K, true)) : 0;
  return one > two ? one : two;
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
  if (!workspace || workspace_bytes < dpa_mxfp4_linear_workspace_bytes(M, N, K)) return DPA_ERR_WORKSPACE;
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
  const int quantized = dpa_mxfp4_operands(x, x_dtype, M, K, row_stride, ws, nullptr, nullptr, stream);
  if (quantized != DPA_OK) return quantized;
  p.a = ws, p.as = p.a + operand_data_bytes(M, K);
  p.part = (float*)(ws + align256(operand_bytes(M, K)));
  return run(p, dtype, s);
}
