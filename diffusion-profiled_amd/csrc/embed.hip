// Token embedding, out[i] = keep scale / (1 - p) W[token i] (keep and p: an optional dropout by
// counter hash, element index i C + c), and the gradient of W,
//   dW[v] = scale / (1 - p) sum over i with token i = v of keep dout[i], in order of i,
// without atomics: the tokens are sorted, and every run of equal ones has one writer.
#include "dpa_common.hpp"

namespace dpa {
namespace embed {

struct Args {
  const void *tokens, *src;  // forward: W; backward: dout
  void* dst;                 // forward: out; backward: dW
  const uint64_t* seed;      // null: no dropout
  int64_t n;
  uint32_t V;
  int C;
  uint32_t pad;  // the token without a gradient (0xffffffff: none)
  uint32_t keep2;
  float scale, keep_scale;
  // backward
  uint32_t *key, *pos;  // sorted tokens (V: no gradient) and their positions
  float* part;          // sums of the pieces of long runs
};

// VEC (1 or 4) elements of type DT at p, in fp32 and back
template <int DT, int VEC>
__device__ __forceinline__ void load(const void* p, int64_t i, float (&v)[VEC]) {
  if constexpr (DT == DPA_DTYPE_F32) {
    if constexpr (VEC == 4) {
      const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
      v[0] = static_cast<const float*>(p)[i];
    }
  } else {
    typedef Elem<DT> E;
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    if constexpr (VEC == 4) {
      const uint2 a = *reinterpret_cast<const uint2*>(q);
      v[0] = E::lo(a.x), v[1] = E::hi(a.x), v[2] = E::lo(a.y), v[3] = E::hi(a.y);
    } else {
      v[0] = E::lo(*q);
    }
  }
}

template <int DT, int VEC>
__device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[VEC]) {
  if constexpr (DT == DPA_DTYPE_F32) {
    if constexpr (VEC == 4)
      *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = float4{v[0], v[1], v[2], v[3]};
    else
      static_cast<float*>(p)[i] = v[0];
  } else {
    typedef Elem<DT> E;
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    if constexpr (VEC == 4)
      *reinterpret_cast<uint2*>(q) = uint2{E::pack(v[0], v[1]), E::pack(v[2], v[3])};
    else
      *q = (uint16_t)E::pack(v[0], 0.f);
  }
}

// clears the dropped of VEC elements from index idx on (VEC = 4: idx a multiple of 4)
template <int VEC>
__device__ __forceinline__ void drop(uint64_t seed, int64_t idx, uint32_t keep, float (&v)[VEC]) {
  uint64_t z = drop_z(seed, idx);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z ^= z >> 31;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const uint32_t q = (uint32_t)(z >> (VEC == 4 ? 16 * i : 16 * (idx & 3))) & 0xffffu;
    if (q < keep) v[i] = 0.f;
  }
}

template <int TB>
__device__ __forceinline__ int64_t token_at(const void* t, int64_t i) {
  return TB == 8 ? static_cast<const int64_t*>(t)[i] : (int64_t)static_cast<const int32_t*>(t)[i];
}

// ---------------------------------------------------------------------------------------
// Forward. A wave per row: 4 channels per lane and step. A token outside the table gives a row of
// NaN (nothing is read for it).
// ---------------------------------------------------------------------------------------
template <int WT, int OT, int TB, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const Args p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= p.n) return;
  const int64_t t = token_at<TB>(p.tokens, row);
  const bool in = t >= 0 && t < (int64_t)p.V;
  const uint64_t seed = p.seed ? *p.seed : 0;
  for (int c = lane * VEC; c < p.C; c += 64 * VEC) {
    float v[VEC];
    if (in) {
      load<WT, VEC>(p.src, t * p.C + c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] *= p.scale;
      if (p.seed) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] *= p.keep_scale;
        drop<VEC>(seed, row * p.C + c, p.keep2 & 0xffffu, v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __builtin_nanf("");
    }
    store<OT, VEC>(p.dst, row * p.C + c, v);
  }
}

// ---------------------------------------------------------------------------------------
// Sorting the tokens (stable, so that a run keeps the order of positions). One workgroup sorts a
// chunk of up to 16384 in LDS, by radix 256; the runs of several chunks are then merged, 16 at a
// time, by rank. The other workgroups of the first launch clear dW meanwhile: with a large table
// that is most of the backward's bytes, and it hides the sort.
// ---------------------------------------------------------------------------------------
constexpr int kChunk = 16384, kSortThreads = 1024, kSortWaves = 16, kMerge = 16;

struct SortArgs {
  const void* tokens;
  uint32_t *key, *pos;
  int64_t n;
  uint32_t V, pad;
  int chunk, chunks, passes;
  uint4* zero;     // dW, 16-B units
  int64_t nzero;
  int tail;        // bytes past them
};

template <int TB>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const SortArgs p) {
  __shared__ uint32_t key[kChunk];
  __shared__ uint16_t idx[2][kChunk];
  __shared__ uint32_t hist[kSortWaves][256];
  __shared__ uint32_t wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  if ((int)blockIdx.x >= p.chunks) {
    const int64_t step = (int64_t)(gridDim.x - p.chunks) * kSortThreads;
    const int64_t i0 = (int64_t)(blockIdx.x - p.chunks) * kSortThreads + tid;
    for (int64_t i = i0; i < p.nzero; i += step) p.zero[i] = uint4{0u, 0u, 0u, 0u};
    if (i0 < p.tail) reinterpret_cast<uint8_t*>(p.zero + p.nzero)[i0] = 0;
    return;
  }

  const int64_t c0 = (int64_t)blockIdx.x * p.chunk;
  const int m = (int)(p.n - c0 < p.chunk ? p.n - c0 : p.chunk);
  for (int i = tid; i < m; i += kSortThreads) {
    const int64_t t = token_at<TB>(p.tokens, c0 + i);
    key[i] = t < 0 || t >= (int64_t)p.V || t == (int64_t)p.pad ? p.V : (uint32_t)t;
    idx[0][i] = (uint16_t)i;
  }
  const int per = (m + kSortWaves * 64 - 1) / (kSortWaves * 64) * 64;  // a wave's part
  const int lo = wave * per, hi = min(m, lo + per);
  for (int pass = 0; pass < p.passes; ++pass) {
    const uint16_t* a = idx[pass & 1];
    uint16_t* o = idx[(pass & 1) ^ 1];
    const int shift = 8 * pass;
    for (int i = tid; i < kSortWaves * 256; i += kSortThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    for (int i = lo + lane; i < hi; i += 64) atomicAdd(&hist[wave][(key[a[i]] >> shift) & 255], 1u);
    __syncthreads();
    // each (digit, wave)'s first place: digits in order, waves in order within a digit
    uint32_t sum = 0;
    if (tid < 256) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = hist[w][tid];
        hist[w][tid] = sum;
        sum += c;
      }
      uint32_t incl = sum;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint32_t x = __shfl_up(incl, off, 64);
        if (lane >= off) incl += x;
      }
      if (lane == 63) wsum[wave] = incl;
      sum = incl - sum;
    }
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < wave; ++w) sum += wsum[w];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) hist[w][tid] += sum;
    }
    __syncthreads();
    // 64 at a time, in order: a lane's place is its digit's next one plus the equal digits in
    // lower lanes
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const int i = i0 + lane;
      const bool on = i < hi;
      const uint32_t x = on ? a[i] : 0;
      const uint32_t d = on ? (key[x] >> shift) & 255 : 0;
      uint64_t same = __ballot(on);
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const uint64_t ones = __ballot((d >> bit) & 1);
        same &= (d >> bit) & 1 ? ones : ~ones;
      }
      const int before = __popcll(same & ((1ull << lane) - 1));
      uint32_t base = 0;
      if (on) base = hist[wave][d];
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
      if (on && before == 0) hist[wave][d] = base + (uint32_t)__popcll(same);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      if (on) o[base + before] = (uint16_t)x;
    }
    __syncthreads();
  }
  const uint16_t* a = idx[p.passes & 1];
  for (int i = tid; i < m; i += kSortThreads) {
    p.key[c0 + i] = key[a[i]];
    p.pos[c0 + i] = (uint32_t)(c0 + a[i]);
  }
}

// One round of merges: groups of kMerge sorted runs of len. An element goes to the place that the
// elements before it take: those of its own run, the not larger ones of the runs before, the
// smaller ones of the runs after.
__global__ __launch_bounds__(256) void embed_merge_kernel(const uint32_t* __restrict__ key,
                                                          const uint32_t* __restrict__ pos,
                                                          uint32_t* __restrict__ okey,
                                                          uint32_t* __restrict__ opos, int64_t n,
                                                          int64_t len) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const uint32_t k = key[i];
  const int64_t run = i / len, first = run / kMerge * kMerge;
  int64_t at = first * len + (i - run * len);
#pragma unroll 4
  for (int r = 0; r < kMerge; ++r) {
    const int64_t s = (first + r) * len;
    if (first + r == run || s >= n) continue;
    const uint32_t want = first + r < run ? k + 1 : k;  // count keys < want (k <= V < 2^31)
    int64_t lo = s, hi = s + len < n ? s + len : n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (key[mid] < want) lo = mid + 1;
      else hi = mid;
    }
    at += lo - s;
  }
  okey[at] = k;
  opos[at] = pos[i];
}

// ---------------------------------------------------------------------------------------
// Sums of the runs. A wave owns 16 sorted places and 256 channels (4 per lane) and sums each run
// that starts there, up to 64 places of it. A longer run is cut into pieces of 64 from its start,
// each owned by the wave of the piece's first place: its fp32 sums go to `part`, and a second
// launch adds them up in order. Slot of a piece that starts at place i: 2 (i / 64) + (1 if it is
// the run's first): a run with several pieces is longer than 64, so no two meet.
// ---------------------------------------------------------------------------------------
constexpr int kOwn = 16, kPiece = 64;

__device__ __forceinline__ int64_t lower_bound(const uint32_t* key, int64_t n, uint32_t want) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (key[mid] < want) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <int GT, int WT, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const Args p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i0 = ((int64_t)blockIdx.x * 4 + wave) * kOwn;
  const int c = (blockIdx.y * 64 + lane) * VEC, cl = c < p.C ? c : 0;
  if (i0 >= p.n) return;
  // lanes 0 .. 15: the places' keys, those before them and those 64 before
  const int64_t i = i0 + lane;
  const bool mine = lane < kOwn && i < p.n;
  const uint32_t k = mine ? p.key[i] : p.V;
  const bool valid = k != p.V;
  const uint32_t k1 = mine && i >= 1 ? p.key[i - 1] : p.V, k64 = mine && i >= kPiece ? p.key[i - kPiece] : p.V;
  uint64_t starts = __ballot(valid && (i == 0 || k1 != k));
  const uint64_t firsts = starts;
  const uint64_t deep = __ballot(valid && i >= kPiece && k64 == k);
  if (deep) {  // places of one long run: where its next piece starts
    const uint32_t kd = __builtin_amdgcn_readlane(k, __builtin_ctzll(deep));
    const int64_t s = lower_bound(p.key, p.n, kd);
    const int64_t next = s + (i0 - s + kPiece - 1) / kPiece * kPiece;
    if (next >= i0 && next < i0 + kOwn) starts |= deep & (1ull << (next - i0));
  }
  const uint64_t seed = p.seed ? *p.seed : 0;
  while (starts) {
    const int j0 = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int64_t s = i0 + j0;
    const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane(k, j0);
    const bool here = s + lane < p.n && p.key[s + lane] == kr;
    const uint64_t run = __ballot(here);
    const int len = run == ~0ull ? 64 : __builtin_ctzll(~run);
    const uint32_t ps = here ? p.pos[s + lane] : 0;
    const bool first = (firsts >> j0) & 1;
    const bool more = len == 64 && s + 64 < p.n && p.key[s + 64] == kr;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    // (every lane goes through the loads, lanes past the row at its start: the positions come
    // from other lanes' registers)
    int j = 0;
    for (; j + 8 <= len; j += 8) {
      float v[8][VEC];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        load<GT, VEC>(p.src, (int64_t)(uint32_t)__builtin_amdgcn_readlane(ps, j + u) * p.C + cl, v[u]);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (p.seed)
          drop<VEC>(seed, (int64_t)(uint32_t)__builtin_amdgcn_readlane(ps, j + u) * p.C + cl,
                    p.keep2 & 0xffffu, v[u]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
      }
    }
    for (; j < len; ++j) {
      const int64_t at = (int64_t)(uint32_t)__builtin_amdgcn_readlane(ps, j) * p.C + cl;
      float v[VEC];
      load<GT, VEC>(p.src, at, v);
      if (p.seed) drop<VEC>(seed, at, p.keep2 & 0xffffu, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += v[e];
    }
    if (c >= p.C) continue;
    if (!first || more) {
      store<DPA_DTYPE_F32, VEC>(p.part, (2 * (s / kPiece) + (first ? 1 : 0)) * p.C + c, acc);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] *= p.scale * p.keep_scale;
      store<WT, VEC>(p.dst, (int64_t)kr * p.C + c, acc);
    }
  }
}

// The pieces of the long run that starts among a workgroup's 64 places, if one does: each wave adds
// up a quarter of them in order, then the quarters.
template <int WT, int VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(const Args p) {
  __shared__ float red[4][64][VEC];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * kPiece + lane;
  const uint32_t k = i < p.n ? p.key[i] : p.V;
  const bool start = k != p.V && (i == 0 || p.key[i - 1] != k) && i + kPiece < p.n && p.key[i + kPiece] == k;
  const uint64_t m = __ballot(start);
  if (!m) return;  // (the same in every wave)
  const int j0 = __builtin_ctzll(m);
  const int64_t s = (int64_t)blockIdx.x * kPiece + j0;
  const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane(k, j0);
  const int64_t pieces = (lower_bound(p.key, p.n, kr + 1) - s + kPiece - 1) / kPiece;
  const int64_t per = (pieces + 3) / 4, lo = wave * per, hi = lo + per < pieces ? lo + per : pieces;
  const int c = (blockIdx.y * 64 + lane) * VEC;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  if (c < p.C) {
#pragma unroll 8
    for (int64_t q = lo; q < hi; ++q) {
      float v[VEC];
      load<DPA_DTYPE_F32, VEC>(p.part, (2 * ((s + q * kPiece) / kPiece) + (q == 0 ? 1 : 0)) * p.C + c, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) red[wave][lane][e] = acc[e];
  __syncthreads();
  if (wave != 0 || c >= p.C) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    acc[e] = (red[0][lane][e] + red[1][lane][e] + red[2][lane][e] + red[3][lane][e]) *
             (p.scale * p.keep_scale);
  store<WT, VEC>(p.dst, (int64_t)kr * p.C + c, acc);
}

// ---- host ------------------------------------------------------------------------------
static bool dtype_ok(int d) { return d == DPA_DTYPE_BF16 || d == DPA_DTYPE_F32 || d == DPA_DTYPE_F16; }
static int dtype_size(int d) { return d == DPA_DTYPE_F32 ? 4 : 2; }

static int check(int64_t n, int64_t V, int C, int token_bytes, int t1, int t2, const void* seed, float p) {
  if (token_bytes != 4 && token_bytes != 8) return DPA_ERR_SHAPE;
  if (!dtype_ok(t1) || !dtype_ok(t2)) return DPA_ERR_SHAPE;
  if (n < 0 || n >= (1ll << 31) - 64 || V <= 0 || V >= (1ll << 31) - 1 || C <= 0 || C > 1 << 20) return DPA_ERR_SIZE;
  if (seed && !drop_p_ok(p)) return DPA_ERR_SIZE;
  if (!aligned(seed, 8)) return DPA_ERR_ALIGN;
  return DPA_OK;
}

static void set_drop(Args& a, const void* seed, float p) {
  a.seed = (const uint64_t*)seed;
  a.keep2 = seed ? drop_threshold(p) * 0x00010001u : 0;
  a.keep_scale = seed ? drop_scale_of(p) : 1.f;
}

// 4 channels per lane need whole groups of 4 and rows aligned to them
static bool vec_ok(const Args& a, int t_src, int t_dst) {
  return a.C % 4 == 0 && aligned(a.src, 4 * dtype_size(t_src)) && aligned(a.dst, 4 * dtype_size(t_dst));
}

template <int WT, int OT>
static void launch_fwd(const Args& a, int token_bytes, hipStream_t s) {
  const unsigned grid = (unsigned)ceil_div(a.n, 4);
  const bool v = vec_ok(a, WT, OT);
  if (token_bytes == 8) {
    if (v) embed_fwd_kernel<WT, OT, 8, 4><<<grid, 256, 0, s>>>(a);
    else embed_fwd_kernel<WT, OT, 8, 1><<<grid, 256, 0, s>>>(a);
  } else {
    if (v) embed_fwd_kernel<WT, OT, 4, 4><<<grid, 256, 0, s>>>(a);
    else embed_fwd_kernel<WT, OT, 4, 1><<<grid, 256, 0, s>>>(a);
  }
}

template <int GT, int WT>
static int launch_sum(const Args& a, hipStream_t s) {
  const bool v = vec_ok(a, GT, WT);
  const dim3 g1((unsigned)ceil_div(a.n, 4 * kOwn), (unsigned)ceil_div(a.C, v ? 256 : 64));
  const dim3 g2((unsigned)ceil_div(a.n, kPiece), g1.y);
  if (v) embed_sum_kernel<GT, WT, 4><<<g1, 256, 0, s>>>(a);
  else embed_sum_kernel<GT, WT, 1><<<g1, 256, 0, s>>>(a);
  const int st = launch_status();
  if (st != DPA_OK || a.n <= kPiece) return st;  // no run can be long
  if (v) embed_join_kernel<WT, 4><<<g2, 256, 0, s>>>(a);
  else embed_join_kernel<WT, 1><<<g2, 256, 0, s>>>(a);
  return launch_status();
}

// f<T1, T2>(args ...) for the types d1, d2
#define EMBED_BY_TYPES(d1, d2, CALL)                                        \
  switch ((d1) * 3 + (d2)) {                                               \
    case DPA_DTYPE_BF16 * 3 + DPA_DTYPE_BF16: CALL(DPA_DTYPE_BF16, DPA_DTYPE_BF16); break; \
    case DPA_DTYPE_BF16 * 3 + DPA_DTYPE_F32: CALL(DPA_DTYPE_BF16, DPA_DTYPE_F32); break;   \
    case DPA_DTYPE_BF16 * 3 + DPA_DTYPE_F16: CALL(DPA_DTYPE_BF16, DPA_DTYPE_F16); break;   \
    case DPA_DTYPE_F32 * 3 + DPA_DTYPE_BF16: CALL(DPA_DTYPE_F32, DPA_DTYPE_BF16); break;   \
    case DPA_DTYPE_F32 * 3 + DPA_DTYPE_F32: CALL(DPA_DTYPE_F32, DPA_DTYPE_F32); break;     \
    case DPA_DTYPE_F32 * 3 + DPA_DTYPE_F16: CALL(DPA_DTYPE_F32, DPA_DTYPE_F16); break;     \
    case DPA_DTYPE_F16 * 3 + DPA_DTYPE_BF16: CALL(DPA_DTYPE_F16, DPA_DTYPE_BF16); break;   \
    case DPA_DTYPE_F16 * 3 + DPA_DTYPE_F32: CALL(DPA_DTYPE_F16, DPA_DTYPE_F32); break;     \
    default: CALL(DPA_DTYPE_F16, DPA_DTYPE_F16); break;                    \
  }

// Up to kChunk tokens in one workgroup; more in runs of half that, which sort in half the time on
// more CUs and are merged
static int chunk_of(int64_t n) { return n <= kChunk ? kChunk : kChunk / 2; }

static int64_t align256(int64_t n) { return (n + 255) & ~255ll; }

}  // namespace embed
}  // namespace dpa

using namespace dpa;
using namespace dpa::embed;

extern "C" int dpa_embedding_fwd(const void* tokens, int token_bytes, const void* weight,
                                 int weight_dtype, void* out, int out_dtype, int64_t n, int64_t V,
                                 int C, float scale, const void* drop_seed, float drop_p,
                                 void* stream) {
  const int st = check(n, V, C, token_bytes, weight_dtype, out_dtype, drop_seed, drop_p);
  if (st != DPA_OK) return st;
  if (n == 0) return DPA_OK;
  if (!tokens || !weight || !out) return DPA_ERR_NULL;
  if (!aligned(tokens, token_bytes) || !aligned(weight, dtype_size(weight_dtype)) ||
      !aligned(out, dtype_size(out_dtype)))
    return DPA_ERR_ALIGN;
  Args a{};
  a.tokens = tokens, a.src = weight, a.dst = out;
  a.n = n, a.V = (uint32_t)V, a.C = C, a.scale = scale;
  set_drop(a, drop_seed, drop_p);
  hipStream_t s = (hipStream_t)stream;
#define FWD(A, B) launch_fwd<A, B>(a, token_bytes, s)
  EMBED_BY_TYPES(weight_dtype, out_dtype, FWD)
#undef FWD
  return launch_status();
}

// two key and two position arrays, and the pieces' sums
extern "C" int64_t dpa_embedding_bwd_workspace_bytes(int64_t n, int C) {
  if (n <= 0 || C <= 0) return 0;
  return 4 * align256(4 * n) + ceil_div(n, kPiece) * 2 * C * 4;
}

extern "C" int dpa_embedding_bwd(const void* dout, int dout_dtype, const void* tokens,
                                 int token_bytes, void* dweight, int weight_dtype, int64_t n,
                                 int64_t V, int C, float scale, int64_t padding_idx,
                                 const void* drop_seed, float drop_p, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  int st = check(n, V, C, token_bytes, dout_dtype, weight_dtype, drop_seed, drop_p);
  if (st != DPA_OK) return st;
  if (!dweight || (n > 0 && (!dout || !tokens))) return DPA_ERR_NULL;
  if (!aligned(dweight, 16) || !aligned(tokens, token_bytes) || !aligned(dout, dtype_size(dout_dtype)))
    return DPA_ERR_ALIGN;
  if (n > 0 && (!workspace || workspace_bytes < dpa_embedding_bwd_workspace_bytes(n, C)))
    return DPA_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
  uint8_t* w = (uint8_t*)workspace;
  const int64_t arr = align256(4 * n);
  uint32_t* key[2] = {(uint32_t*)w, (uint32_t*)(w + arr)};
  uint32_t* pos[2] = {(uint32_t*)(w + 2 * arr), (uint32_t*)(w + 3 * arr)};
  hipStream_t s = (hipStream_t)stream;

  SortArgs q{};
  q.tokens = tokens, q.key = key[0], q.pos = pos[0], q.n = n;
  q.V = (uint32_t)V;
  q.pad = padding_idx >= 0 && padding_idx < V ? (uint32_t)padding_idx : 0xffffffffu;
  q.chunk = chunk_of(n);
  q.chunks = (int)ceil_div(n, q.chunk);
  while ((V >> (8 * q.passes)) > 0) ++q.passes;
  const int64_t bytes = V * C * dtype_size(weight_dtype);
  q.zero = (uint4*)dweight, q.nzero = bytes / 16, q.tail = (int)(bytes % 16);
  int64_t fill = ceil_div(q.nzero + 1, kSortThreads * 4);
  if (fill > 2 * num_cus()) fill = 2 * num_cus();
  const unsigned grid = (unsigned)(q.chunks + fill);
  if (token_bytes == 8) embed_sort_kernel<8><<<grid, kSortThreads, 0, s>>>(q);
  else embed_sort_kernel<4><<<grid, kSortThreads, 0, s>>>(q);
  st = launch_status();
  if (st != DPA_OK || n == 0) return st;
  int at = 0;
  for (int64_t len = q.chunk; len < n; len *= kMerge, at ^= 1) {
    embed_merge_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(key[at], pos[at], key[at ^ 1],
                                                                   pos[at ^ 1], n, len);
    st = launch_status();
    if (st != DPA_OK) return st;
  }
  Args a{};
  a.src = dout, a.dst = dweight, a.n = n, a.V = (uint32_t)V, a.C = C, a.scale = scale;
  a.key = key[at], a.pos = pos[at], a.part = (float*)(w + 4 * arr);
  set_drop(a, drop_seed, drop_p);
#define SUM(A, B) st = launch_sum<A, B>(a, s)
  EMBED_BY_TYPES(dout_dtype, weight_dtype, SUM)
#undef SUM
  return st;
}
