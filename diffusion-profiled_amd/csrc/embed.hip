// Token embedding, out[i] = keep scale / (1 - p) W[token i] (keep and p: an optional dropout by
// counter hash, element index i C + c), and the gradient of W,
//   dW[v] = scale / (1 - p) sum over i with token i = v of keep dout[i], in a fixed order,
// without atomics: the tokens are sorted (stable), and every run of equal ones has one writer.
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
  // forward: 16-B units of out's rows, as the table has them
  uint32_t units;
  FastDiv by_row;
};

// VEC (1, 4 or 8) elements of type DT at p, in fp32 and back
template <int DT, int VEC>
__device__ __forceinline__ void load(const void* p, int64_t i, float (&v)[VEC]) {
  if constexpr (DT == DPA_DTYPE_F32) {
    const float* q = static_cast<const float*>(p) + i;
    if constexpr (VEC == 1) {
      v[0] = *q;
    } else {
#pragma unroll
      for (int x = 0; x < VEC; x += 4) {
        const float4 a = *reinterpret_cast<const float4*>(q + x);
        v[x] = a.x, v[x + 1] = a.y, v[x + 2] = a.z, v[x + 3] = a.w;
      }
    }
  } else {
    typedef Elem<DT> E;
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    if constexpr (VEC == 8) {
      const uint4 a = *reinterpret_cast<const uint4*>(q);
      v[0] = E::lo(a.x), v[1] = E::hi(a.x), v[2] = E::lo(a.y), v[3] = E::hi(a.y);
      v[4] = E::lo(a.z), v[5] = E::hi(a.z), v[6] = E::lo(a.w), v[7] = E::hi(a.w);
    } else if constexpr (VEC == 4) {
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
    float* q = static_cast<float*>(p) + i;
    if constexpr (VEC == 1) {
      *q = v[0];
    } else {
#pragma unroll
      for (int x = 0; x < VEC; x += 4)
        *reinterpret_cast<float4*>(q + x) = float4{v[x], v[x + 1], v[x + 2], v[x + 3]};
    }
  } else {
    typedef Elem<DT> E;
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    if constexpr (VEC == 8)
      *reinterpret_cast<uint4*>(q) = uint4{E::pack(v[0], v[1]), E::pack(v[2], v[3]), E::pack(v[4], v[5]),
                                           E::pack(v[6], v[7])};
    else if constexpr (VEC == 4)
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
// Forward. A token outside the table gives a row of NaN (nothing is read for it). Bound by HBM: rows
// of the table read, out written.
// Where rows are whole units of 16 B of the table's type: a thread per unit, four of them apart, so
// that their tokens load together and then their rows. Else a wave per row, an element per lane.
// 130816 tokens of 768 (bf16): 54 us, 5.1 TB/s, the copy rate (one unit a thread: 66).
// ---------------------------------------------------------------------------------------
template <int WT, int OT, int VEC>
__device__ __forceinline__ void embed_store(const Args& p, uint64_t seed, bool in, int64_t at, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = in ? v[i] * p.scale : __builtin_nanf("");
  if (p.seed && in) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= p.keep_scale;
    if constexpr (VEC == 8) {
      float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
      drop<4>(seed, at, p.keep2 & 0xffffu, a);
      drop<4>(seed, at + 4, p.keep2 & 0xffffu, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
      drop<VEC>(seed, at, p.keep2 & 0xffffu, v);
    }
  }
  store<OT, VEC>(p.dst, at, v);
}

template <int WT, int OT, int TB>
__global__ __launch_bounds__(256) void embed_units_kernel(const Args p) {
  constexpr int VEC = 16 / (WT == DPA_DTYPE_F32 ? 4 : 2), U = 4;
  const uint64_t seed = p.seed ? *p.seed : 0;
  const uint32_t i0 = blockIdx.x * (256 * U) + threadIdx.x;
  int64_t t[U];
  uint32_t c[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = i0 + 256 * u, row = fdiv(i < p.units ? i : 0, p.by_row);
    c[u] = ((i < p.units ? i : 0) - row * p.by_row.d) * VEC;
    t[u] = token_at<TB>(p.tokens, row);
  }
  float v[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool in = t[u] >= 0 && t[u] < (int64_t)p.V;
    load<WT, VEC>(p.src, (in ? t[u] * p.C : 0) + c[u], v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = i0 + 256 * u;
    if (i < p.units) embed_store<WT, OT, VEC>(p, seed, t[u] >= 0 && t[u] < (int64_t)p.V, (int64_t)i * VEC, v[u]);
  }
}

template <int WT, int OT, int TB>
__global__ __launch_bounds__(256) void embed_rows_kernel(const Args p) {
  const int lane = threadIdx.x & 63;
  const uint64_t seed = p.seed ? *p.seed : 0;
  for (int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < p.n;
       row += (int64_t)gridDim.x * 4) {
    const int64_t t = token_at<TB>(p.tokens, row);
    const bool in = t >= 0 && t < (int64_t)p.V;
    for (int c = lane; c < p.C; c += 64) {
      float v[1] = {0.f};
      if (in) load<WT, 1>(p.src, t * p.C + c, v);
      embed_store<WT, OT, 1>(p, seed, in, row * p.C + c, v);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Sorting the tokens (stable, so that a run keeps the order of positions). A workgroup sorts a chunk
// of 1024 in LDS, by radix 256, which takes about 5 us however many chunks there are; the sorted runs
// are then merged 16 at a time by rank, with every 32nd key of a run in LDS to search first. The
// other workgroups of these launches clear dW meanwhile, each launch a part of it: with a large
// table that is most of the backward's bytes, and it hides most of the sort: 9856 tokens into 32768 x 512
// fp32 (67 MB) sort 8.4 us, merge 12.8; 130816 into 50001 x 768 bf16 (77 MB) sort 7.5, two merges 18.3 each.
// ---------------------------------------------------------------------------------------
constexpr int kChunk = 1024, kSortWaves = kChunk / 64, kMerge = 16, kSample = 32;
constexpr int kBatch = 16;  // rows that a wave loads together

struct Fill {  // clears 16-B units and the bytes past them
  uint4* at;
  int64_t n;
  int tail;
  __device__ __forceinline__ void run(int block, int blocks, int threads, int tid) const {
    const int64_t step = (int64_t)blocks * threads, i0 = (int64_t)block * threads + tid;
    for (int64_t i = i0; i < n; i += step) at[i] = uint4{0u, 0u, 0u, 0u};
    if (i0 < tail) reinterpret_cast<uint8_t*>(at + n)[i0] = 0;
  }
};

struct SortArgs {
  const void* tokens;
  uint32_t *key, *pos, *sample;
  int64_t n;
  uint32_t V, pad;
  int chunks, passes;
  Fill fill;
};

struct ChunkLds {
  uint32_t key[kChunk];
  uint16_t idx[2][kChunk];
  uint32_t hist[kSortWaves][256];
  uint32_t wsum[4];
};

// Sorts the chunk's m keys (key[0 .. m), by the workgroup, a thread each) by their lowest 8 `passes`
// bits: gives the places' original places. Ends with a barrier.
__device__ __forceinline__ const uint16_t* sort_chunk(ChunkLds& s, int m, int passes, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const bool on = tid < m;
  if (on) s.idx[0][tid] = (uint16_t)tid;
  for (int pass = 0; pass < passes; ++pass) {
    const uint16_t* a = s.idx[pass & 1];
    uint16_t* o = s.idx[(pass & 1) ^ 1];
    for (int i = tid; i < kSortWaves * 256; i += kChunk) (&s.hist[0][0])[i] = 0;
    __syncthreads();
    // a wave's places in order: how many lower lanes share this one's digit, and how many lanes do
    const uint32_t x = on ? a[tid] : 0;
    const uint32_t d = on ? (s.key[x] >> (8 * pass)) & 255 : 0;
    uint64_t same = __ballot(on);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const uint64_t ones = __ballot((d >> bit) & 1);
      same &= (d >> bit) & 1 ? ones : ~ones;
    }
    const int before = __popcll(same & ((1ull << lane) - 1));
    if (on && before == 0) s.hist[wave][d] = (uint32_t)__popcll(same);
    __syncthreads();
    // each (digit, wave)'s first place: digits in order, waves in order within a digit
    uint32_t sum = 0, first[kSortWaves];
    if (tid < 256) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) first[w] = s.hist[w][tid];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = first[w];
        first[w] = sum;
        sum += c;
      }
      uint32_t incl = sum;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint32_t y = __shfl_up(incl, off, 64);
        if (lane >= off) incl += y;
      }
      if (lane == 63) s.wsum[wave] = incl;
      sum = incl - sum;
    }
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < wave; ++w) sum += s.wsum[w];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) s.hist[w][tid] = first[w] + sum;
    }
    __syncthreads();
    if (on) o[s.hist[wave][d] + before] = (uint16_t)x;
    __syncthreads();
  }
  return s.idx[passes & 1];
}

// a token's key: V for those without a gradient
template <int TB>
__device__ __forceinline__ uint32_t key_of(const void* tokens, int64_t i, uint32_t V, uint32_t pad) {
  const int64_t t = token_at<TB>(tokens, i);
  return t < 0 || t >= (int64_t)V || t == (int64_t)pad ? V : (uint32_t)t;
}

template <int TB>
__global__ __launch_bounds__(kChunk) void embed_sort_kernel(const SortArgs p) {
  __shared__ ChunkLds s;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= p.chunks) {
    p.fill.run(blockIdx.x - p.chunks, gridDim.x - p.chunks, kChunk, tid);
    return;
  }
  const int64_t c0 = (int64_t)blockIdx.x * kChunk;
  const int m = (int)(p.n - c0 < kChunk ? p.n - c0 : kChunk);
  if (tid < m) s.key[tid] = key_of<TB>(p.tokens, c0 + tid, p.V, p.pad);
  const uint16_t* order = sort_chunk(s, m, p.passes, tid);
  if (tid < m) {
    const uint32_t x = order[tid], k = s.key[x];
    p.key[c0 + tid] = k;
    p.pos[c0 + tid] = (uint32_t)(c0 + x);
    if (tid % kSample == 0) p.sample[(c0 + tid) / kSample] = k;
  }
}

// ---------------------------------------------------------------------------------------
// Up to kSmall tokens: the whole gradient in one launch, for whose others a small call would wait (512
// tokens, 663 rows of 768: 12.2 us; with 1000 tokens it would be 17.9, and the three launches of the
// form for more 14.7).
// `slices` workgroups of 64 channels sort the tokens, each for itself, and sum: a wave takes 16 or
// 32 sorted places; a run that goes on in the next wave is finished, in order, by the wave in which it
// starts, from what the others leave in LDS. The other workgroups clear the rows that no token names
// (a bit per row in LDS).
// ---------------------------------------------------------------------------------------
constexpr int kSmall = 512;
constexpr int kSmallRows = 1 << 18;  // rows that the bits have room for

template <int GT, int WT, int TB>
__global__ __launch_bounds__(kChunk) void embed_small_kernel(const Args p, const void* tokens, int slices, int passes) {
  __shared__ union {
    struct {
      ChunkLds sort;
      float head[kSortWaves][64];
    };
    uint32_t named[kSmallRows / 32];
  } s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = (int)p.n;

  if ((int)blockIdx.x >= slices) {
    for (int i = tid; i < (int)(p.V + 31) / 32; i += kChunk) s.named[i] = 0;
    __syncthreads();
    if (tid < n) {
      const uint32_t k = key_of<TB>(tokens, tid, p.V, p.pad);
      if (k != p.V) atomicOr(&s.named[k / 32], 1u << (k % 32));
    }
    __syncthreads();
    const int64_t step = (int64_t)(gridDim.x - slices) * kSortWaves;
    const int bytes = p.C * Elem<WT>::size;
    for (int64_t r = (int64_t)(blockIdx.x - slices) * kSortWaves + wave; r < p.V; r += step) {
      if ((s.named[r / 32] >> (r % 32)) & 1) continue;
      uint8_t* row = static_cast<uint8_t*>(p.dst) + r * bytes;
      if (bytes % 16 == 0)
        for (int i = lane * 16; i < bytes; i += 1024) *reinterpret_cast<uint4*>(row + i) = uint4{0u, 0u, 0u, 0u};
      else
        for (int i = lane * 2; i < bytes; i += 128) *reinterpret_cast<uint16_t*>(row + i) = 0;
    }
    return;
  }

  if (tid < n) s.sort.key[tid] = key_of<TB>(tokens, tid, p.V, p.pad);
  const uint16_t* order = sort_chunk(s.sort, n, passes, tid);
  const int per = (n + kSortWaves * kBatch - 1) / (kSortWaves * kBatch) * kBatch;  // a wave's places
  static_assert(kSmall <= 2 * kSortWaves * kBatch, "16 or 32 places");
  const int place = wave * per + lane;
  const bool on = lane < per && place < n;
  const uint32_t at = on ? order[place] : 0;
  const uint32_t k = on ? s.sort.key[at] : p.V;
  const uint32_t before = on && place > 0 ? s.sort.key[order[place - 1]] : p.V;
  const int count = __popcll(__ballot(k != p.V));  // (V's are behind the others)
  const uint64_t starts = __ballot(k != p.V && (place == 0 || before != k));
  const int c = blockIdx.x * 64 + lane, cl = c < p.C ? c : 0;
  const uint64_t seed = p.seed ? *p.seed : 0;
  const float factor = p.scale * p.keep_scale;

  float acc = 0.f;
  int from = starts & 1 ? 0 : -1;  // where the run at work starts (-1: in a wave before)
  auto leave = [&](int end) __attribute__((always_inline)) {
    if (from < 0) {
      s.head[wave][lane] = acc;
    } else if (end < per && c < p.C) {
      const float v[1] = {acc * factor};
      store<WT, 1>(p.dst, (int64_t)(uint32_t)__builtin_amdgcn_readlane(k, from) * p.C + c, v);
    }
  };
  for (int j = 0; j < count; j += kBatch) {
    float v[kBatch][1];
    uint32_t pj[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      pj[u] = (uint32_t)__builtin_amdgcn_readlane(at, j + u < count ? j + u : count - 1);
      load<GT, 1>(p.src, (int64_t)pj[u] * p.C + cl, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (j + u >= count) break;
      if (j + u > 0 && ((starts >> (j + u)) & 1)) {
        leave(j + u);
        from = j + u;
        acc = 0.f;
      }
      if (p.seed) drop<1>(seed, (int64_t)pj[u] * p.C + cl, p.keep2 & 0xffffu, v[u]);
      acc += v[u][0];
    }
  }
  if (count > 0) leave(count);
  __syncthreads();
  if (count < per || from < 0) return;
  const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane(k, from);
  for (int w = wave + 1; w < kSortWaves; ++w) {
    const int lo = w * per, hi = lo + per - 1;
    if (lo >= n || s.sort.key[order[lo]] != kr) break;
    acc += s.head[w][lane];
    if (hi >= n || s.sort.key[order[hi]] != kr) break;
  }
  if (c < p.C) {
    const float v[1] = {acc * factor};
    store<WT, 1>(p.dst, (int64_t)kr * p.C + c, v);
  }
}

// One round of merges: groups of kMerge sorted runs of len (a multiple of kChunk). An element goes to
// the place that the elements before it take: those of its own run, the not larger ones of the runs
// before, the smaller ones of the runs after.
constexpr int kTable = 512;  // keys of a run in LDS

struct MergeArgs {
  const uint32_t *key, *pos, *sample;
  uint32_t *okey, *opos, *osample;
  int64_t n, len;
  int log_per, log_rows;  // keys from one table entry to the next, entries of a run
  int blocks;             // of 256 places; the others clear
  Fill fill;
};

__global__ __launch_bounds__(256) void embed_merge_kernel(const MergeArgs p) {
  __shared__ uint32_t table[kMerge * kTable];
  if ((int)blockIdx.x >= p.blocks) {
    p.fill.run(blockIdx.x - p.blocks, gridDim.x - p.blocks, 256, threadIdx.x);
    return;
  }
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t run = (int64_t)blockIdx.x * 256 / p.len, first = run / kMerge * kMerge;  // (of the workgroup)
  for (int x = threadIdx.x; x < kMerge << p.log_rows; x += 256) {
    const int64_t at = first * p.len + ((int64_t)x << p.log_per);
    table[x] = at < p.n ? p.sample[at / kSample] : 0xffffffffu;
  }
  __syncthreads();
  if (i >= p.n) return;
  const uint32_t k = p.key[i], n = (uint32_t)p.n;
  // how many table entries, then keys up to the next entry, are smaller: halving steps, the same for
  // every run, so that the runs' reads go out together
  uint32_t a[kMerge], want[kMerge];  // (k <= V < 2^31)
#pragma unroll
  for (int r = 0; r < kMerge; ++r) a[r] = r << p.log_rows, want[r] = first + r < run ? k + 1 : k;
  for (int st = 1 << p.log_rows >> 1; st > 0; st >>= 1) {
#pragma unroll
    for (int r = 0; r < kMerge; ++r) a[r] += table[a[r] + st - 1] < want[r] ? st : 0;
  }
#pragma unroll
  for (int r = 0; r < kMerge; ++r) a[r] = a[r] - (r << p.log_rows) + (table[a[r]] < want[r] ? 1 : 0);
  // (with a entries smaller, so is the run's key at (a - 1) per: the count goes on behind it)
  uint32_t at[kMerge];
#pragma unroll
  for (int r = 0; r < kMerge; ++r) {
    const int64_t s = (first + r) * p.len;
    at[r] = (uint32_t)(s < p.n ? s : p.n) + ((a[r] ? a[r] - 1 : 0) << p.log_per);
  }
  for (uint32_t st = 1u << p.log_per >> 1; st > 0; st >>= 1) {
    uint32_t x[kMerge];
#pragma unroll
    for (int r = 0; r < kMerge; ++r) x[r] = p.key[min(at[r] + st, n - 1)];
#pragma unroll
    for (int r = 0; r < kMerge; ++r) at[r] += (at[r] + st < n) & (x[r] < want[r]) ? st : 0;
  }
  int64_t place = first * p.len + (i - run * p.len);
#pragma unroll
  for (int r = 0; r < kMerge; ++r)
    if (first + r != run && a[r] > 0) place += (int64_t)at[r] + 1 - (first + r) * p.len;
  p.okey[place] = k;
  p.opos[place] = p.pos[i];
  if (place % kSample == 0) p.osample[place / kSample] = k;
}

// ---------------------------------------------------------------------------------------
// Sums of the runs. A wave owns 16 sorted places and 256 channels (4 per lane) and sums each run
// that starts there, up to 32 places of it. A longer run is cut into pieces of 32 from its start,
// each owned by the wave of the piece's first place: its fp32 sums go to `part`, and a second
// launch adds them up in order. Slot of a piece that starts at place i: 2 (i / 32) + (1 if it is
// the run's first): a run with several pieces is longer than 32, so no two meet.
// The runs that a wave sums lie side by side, so their places load together, kBatch rows at a time
// whatever runs they belong to, and a run is stored where the next one begins.
// Bound by gathered rows: 130816 of 1.5 KB 51 us, 3.3 TB/s of HBM (the bytes without the caches' share:
// 4.6), and 8.9 for the pieces; 9856 of 2 KB 10.8 and 3.9, the time of a few dependent trips.
// ---------------------------------------------------------------------------------------
constexpr int kOwn = 16, kPiece = 32;

// The first of the n sorted keys that is not smaller than want, by a wave: 64 probes a step
__device__ __forceinline__ int64_t lower_bound(const uint32_t* key, int64_t n, uint32_t want, int lane) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) >> 6, at = lo + lane * step;
    const int below = __popcll(__ballot(at < hi && key[at < hi ? at : lo] < want));
    if (below == 0) break;
    const int64_t next = lo + below * step;
    lo += (below - 1) * step + 1;
    hi = next < hi ? next : hi;
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
  // the keys of places i0 + lane, those one and 32 before, and the places' positions (V: no gradient,
  // and past the end)
  const int64_t i = i0 + lane;
  const uint32_t k = i < p.n ? p.key[i] : p.V;
  const uint32_t k1 = i >= 1 && i < p.n ? p.key[i - 1] : p.V;
  const uint32_t k64 = i >= kPiece && i < p.n ? p.key[i - kPiece] : p.V;
  const uint32_t ps = i < p.n ? p.pos[i] : 0;
  const uint64_t own = (1ull << kOwn) - 1;
  const uint64_t firsts = __ballot(k != p.V && (i == 0 || k1 != k));  // (all 64 places)
  uint64_t starts = firsts & own;
  const uint64_t deep = __ballot(k != p.V && i >= kPiece && k64 == k) & own;
  if (deep) {  // places of one long run: where its next piece starts
    const uint32_t kd = __builtin_amdgcn_readlane(k, __builtin_ctzll(deep));
    const int64_t s = lower_bound(p.key, i0, kd, lane);
    const int64_t next = s + (i0 - s + kPiece - 1) / kPiece * kPiece;
    if (next >= i0 && next < i0 + kOwn) starts |= deep & (1ull << (next - i0));
  }
  if (!starts) return;
  // the last of them ends at place `end`: 32 further on, or at the next run
  const int j_last = 63 - __builtin_clzll(starts);
  const uint32_t k_last = (uint32_t)__builtin_amdgcn_readlane(k, j_last);
  const uint64_t away = __ballot(k != k_last) & ~((2ull << j_last) - 1);
  static_assert(kOwn + kPiece < 64, "a wave's runs and what follows are in its lanes");
  int end = away ? __builtin_ctzll(away) : 64;
  const bool more = end > j_last + kPiece;  // it goes on behind its piece
  if (end > j_last + kPiece) end = j_last + kPiece;

  const uint64_t seed = p.seed ? *p.seed : 0;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  int from = __builtin_ctzll(starts);  // the run at work
  auto finish = [&]() __attribute__((always_inline)) {
    const bool first = (firsts >> from) & 1;
    if (c < p.C && ((starts >> from) & 1)) {
      if (!first || (from == j_last && more)) {
        store<DPA_DTYPE_F32, VEC>(p.part, (2 * ((i0 + from) / kPiece) + (first ? 1 : 0)) * p.C + c, acc);
      } else {
        const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane(k, from);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= p.scale * p.keep_scale;
        store<WT, VEC>(p.dst, (int64_t)kr * p.C + c, acc);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  };
  // (every lane goes through the loads, lanes past the row at its start: the positions come from
  // other lanes' registers)
  for (int j = from; j < end; j += kBatch) {
    float v[kBatch][VEC];
    uint32_t pj[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int x = j + u < end ? j + u : end - 1;
      pj[u] = (uint32_t)__builtin_amdgcn_readlane(ps, x);
      load<GT, VEC>(p.src, (int64_t)pj[u] * p.C + cl, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (j + u >= end) break;
      if (j + u > from && j + u < kOwn && ((starts >> (j + u)) & 1)) {
        finish();
        from = j + u;
      }
      if (p.seed) drop<VEC>(seed, (int64_t)pj[u] * p.C + cl, p.keep2 & 0xffffu, v[u]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
    }
  }
  finish();
}

// The pieces of the long run that starts among a workgroup's 32 places, if one does: each wave adds
// up a quarter of them in order, then the quarters.
template <int WT, int VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(const Args p) {
  __shared__ float red[4][64][VEC];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * kPiece + lane;
  const uint32_t k = lane < kPiece && i < p.n ? p.key[i] : p.V;
  const bool start = k != p.V && (i == 0 || p.key[i - 1] != k) && i + kPiece < p.n && p.key[i + kPiece] == k;
  const uint64_t m = __ballot(start);
  if (!m) return;  // (the same in every wave)
  const int j0 = __builtin_ctzll(m);
  const int64_t s = (int64_t)blockIdx.x * kPiece + j0;
  const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane(k, j0);
  const int64_t pieces = (lower_bound(p.key, p.n, kr + 1, lane) - s + kPiece - 1) / kPiece;
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
static void launch_fwd(Args& a, int token_bytes, hipStream_t s) {
  constexpr int VEC = 16 / (WT == DPA_DTYPE_F32 ? 4 : 2);
  const int64_t units = a.n * (a.C / VEC);
  if (a.C % VEC == 0 && units < 1ll << 31 && aligned(a.src, 16) &&
      aligned(a.dst, VEC * dtype_size(OT) < 16 ? VEC * dtype_size(OT) : 16)) {
    a.units = (uint32_t)units;
    a.by_row = make_fastdiv(a.C / VEC);
    const unsigned grid = (unsigned)ceil_div(units, 1024);
    if (token_bytes == 8) embed_units_kernel<WT, OT, 8><<<grid, 256, 0, s>>>(a);
    else embed_units_kernel<WT, OT, 4><<<grid, 256, 0, s>>>(a);
    return;
  }
  const int64_t groups = ceil_div(a.n, 4);
  const unsigned grid = (unsigned)(groups < 1 << 22 ? groups : 1 << 22);
  if (token_bytes == 8) embed_rows_kernel<WT, OT, 8><<<grid, 256, 0, s>>>(a);
  else embed_rows_kernel<WT, OT, 4><<<grid, 256, 0, s>>>(a);
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

template <int GT, int WT>
static int launch_small(const Args& a, const void* tokens, int token_bytes, int passes, hipStream_t s) {
  const int slices = (int)ceil_div(a.C, 64);
  int64_t fill = ceil_div(a.V, kSortWaves * 4);
  if (fill > 2 * num_cus()) fill = 2 * num_cus();
  const unsigned grid = (unsigned)(slices + fill);
  if (token_bytes == 8) embed_small_kernel<GT, WT, 8><<<grid, kChunk, 0, s>>>(a, tokens, slices, passes);
  else embed_small_kernel<GT, WT, 4><<<grid, kChunk, 0, s>>>(a, tokens, slices, passes);
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

// two arrays of keys, two of positions and two of samples, and the pieces' sums
extern "C" int64_t dpa_embedding_bwd_workspace_bytes(int64_t n, int C) {
  if (n <= 0 || C <= 0) return 0;
  return 4 * align256(4 * n) + 2 * align256(4 * ceil_div(n, kSample)) + ceil_div(n, kPiece) * 2 * C * 4;
}

extern "C" int dpa_embedding_bwd(const void* dout, int dout_dtype, const void* tokens,
                                 int token_bytes, void* dweight, int weight_dtype, int64_t n,
                                 int64_t V, int C, float scale, int64_t padding_idx,
                                 const void* drop_seed, float drop_p, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  int st = check(n, V, C, token_bytes, dout_dtype, weight_dtype, drop_seed, drop_p);
  if (st != DPA_OK) return st;
  // (a workgroup of 256 for 32 places: the join's grid)
  if (ceil_div(n, kPiece) > kMaxGroups256) return DPA_ERR_SIZE;
  if (!dweight || (n > 0 && (!dout || !tokens))) return DPA_ERR_NULL;
  if (!aligned(dweight, 16) || !aligned(tokens, token_bytes) || !aligned(dout, dtype_size(dout_dtype)))
    return DPA_ERR_ALIGN;
  if (n > 0 && (!workspace || workspace_bytes < dpa_embedding_bwd_workspace_bytes(n, C)))
    return DPA_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return DPA_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  const uint32_t pad = padding_idx >= 0 && padding_idx < V ? (uint32_t)padding_idx : 0xffffffffu;
  int passes = 0;
  while ((V >> (8 * passes)) > 0) ++passes;
  Args a{};
  a.src = dout, a.dst = dweight, a.n = n, a.V = (uint32_t)V, a.C = C, a.scale = scale, a.pad = pad;
  set_drop(a, drop_seed, drop_p);
  if (n > 0 && n <= kSmall && V <= kSmallRows) {
#define SMALL(A, B) st = launch_small<A, B>(a, tokens, token_bytes, passes, s)
    EMBED_BY_TYPES(dout_dtype, weight_dtype, SMALL)
#undef SMALL
    return st;
  }

  uint8_t* w = (uint8_t*)workspace;
  const int64_t arr = align256(4 * n), smp = align256(4 * ceil_div(n, kSample));
  uint32_t* key[2] = {(uint32_t*)w, (uint32_t*)(w + arr)};
  uint32_t* pos[2] = {(uint32_t*)(w + 2 * arr), (uint32_t*)(w + 3 * arr)};
  uint32_t* sample[2] = {(uint32_t*)(w + 4 * arr), (uint32_t*)(w + 4 * arr + smp)};

  // dW, in equal parts to the launches of the sort
  int launches = 1;
  for (int64_t len = kChunk; len < n; len *= kMerge) ++launches;
  const int64_t bytes = V * C * dtype_size(weight_dtype), units = bytes / 16, part = ceil_div(units, launches);
  auto fill = [&](int i, int threads, int* blocks) {
    const int64_t lo = i * part < units ? i * part : units, hi = lo + part < units ? lo + part : units;
    const int64_t most = 2 * num_cus() * (1024 / threads), want = ceil_div(hi - lo + 1, threads * 4);
    *blocks = (int)(want < most ? want : most);
    return Fill{(uint4*)dweight + lo, hi - lo, i + 1 == launches ? (int)(bytes % 16) : 0};
  };

  SortArgs q{};
  q.tokens = tokens, q.key = key[0], q.pos = pos[0], q.sample = sample[0], q.n = n;
  q.V = (uint32_t)V, q.pad = pad, q.passes = passes;
  q.chunks = (int)ceil_div(n, kChunk);
  int blocks;
  q.fill = fill(0, kChunk, &blocks);
  const unsigned grid = (unsigned)(q.chunks + blocks);
  if (token_bytes == 8) embed_sort_kernel<8><<<grid, kChunk, 0, s>>>(q);
  else embed_sort_kernel<4><<<grid, kChunk, 0, s>>>(q);
  st = launch_status();
  if (st != DPA_OK || n == 0) return st;
  int at = 0, round = 0;
  for (int64_t len = kChunk; len < n; len *= kMerge, at ^= 1) {
    MergeArgs m{};
    m.key = key[at], m.pos = pos[at], m.sample = sample[at];
    m.okey = key[at ^ 1], m.opos = pos[at ^ 1], m.osample = sample[at ^ 1];
    m.n = n, m.len = len;
    while ((kSample << m.log_rows) < len && (1 << m.log_rows) < kTable) ++m.log_rows;
    while (((int64_t)1 << (m.log_rows + m.log_per)) < len) ++m.log_per;
    m.blocks = (int)ceil_div(n, 256);
    m.fill = fill(++round, 256, &blocks);
    embed_merge_kernel<<<(unsigned)(m.blocks + blocks), 256, 0, s>>>(m);
    st = launch_status();
    if (st != DPA_OK) return st;
  }
  a.key = key[at], a.pos = pos[at], a.part = (float*)(w + 4 * arr + 2 * smp);
#define SUM(A, B) st = launch_sum<A, B>(a, s)
  EMBED_BY_TYPES(dout_dtype, weight_dtype, SUM)
#undef SUM
  return st;
}
