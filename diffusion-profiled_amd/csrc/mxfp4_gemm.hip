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
  int M, N;
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
// Up to 16 MT rows of a: bound by the bytes of b, which go straight to registers. A workgroup takes 16
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

static GemmArgs plan(int64_t M, int64_t N, int64_t K) {
  GemmArgs p{};
  p.M = (int)M, p.N = (int)N;
  p.pitch = pitch_of(K);
  p.steps = (int)(p.pitch / 128);
  const bool few = M <= kFewRows;
  p.tiles_m = few ? 1 : (int)ceil_div(M, 128);
  p.tiles_n = (int)ceil_div(N, few ? 16 : 128);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, want = 2 * num_cus();
  int64_t n = tiles > 0 ? want / tiles : 1;
  const int64_t least = few ? 8 : 4;
  if (n > p.steps / least) n = p.steps / least;
  if (n < 1) n = 1;
  p.per_split = (int)(ceil_div(ceil_div(p.steps, n), 2) * 2);
  p.splits = (int)ceil_div(p.steps, p.per_split);
  return p;
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
  const int st = launch_status();
  if (st != DPA_OK || p.splits == 1) return st;
  mxfp4_join_kernel<DT><<<(unsigned)ceil_div((int64_t)p.M * p.N, 256), 256, 0, s>>>(p);
  return launch_status();
}

}  // namespace mx
}  // namespace dpa

using namespace dpa;
using namespace dpa::mx;

extern "C" int64_t dpa_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (check_gemm(M, N, K) != DPA_OK) return 0;
  const GemmArgs p = plan(M, N, K);
  return p.splits > 1 ? p.splits * M * N * 4 : 0;
}

extern "C" int dpa_mxfp4_gemm(const void* a_data, const void* a_scales, const void* b_data, const void* b_scales,
                              const float* bias, void* y, int dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return DPA_ERR_SHAPE;
  const int st = check_gemm(M, N, K);
  if (st != DPA_OK) return st;
  if (M == 0 || N == 0) return DPA_OK;
  if (!a_data || !a_scales || !b_data || !b_scales || !y) return DPA_ERR_NULL;
  if (!aligned(a_data, 16) || !aligned(a_scales, 16) || !aligned(b_data, 16) || !aligned(b_scales, 16) ||
      !aligned(bias, 4) || !aligned(y, size_of(dtype)))
    return DPA_ERR_ALIGN;
  GemmArgs p = plan(M, N, K);
  p.a = (const uint8_t*)a_data, p.as = (const uint8_t*)a_scales;
  p.b = (const uint8_t*)b_data, p.bs = (const uint8_t*)b_scales;
  p.bias = bias, p.y = y;
  if (p.splits > 1) {
    if (!workspace || workspace_bytes < p.splits * M * N * 4) return DPA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
    p.part = (float*)workspace;
  }
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPA_DTYPE_BF16) return run_gemm<DPA_DTYPE_BF16>(p, s);
  if (dtype == DPA_DTYPE_F16) return run_gemm<DPA_DTYPE_F16>(p, s);
  return run_gemm<DPA_DTYPE_F32>(p, s);
}
