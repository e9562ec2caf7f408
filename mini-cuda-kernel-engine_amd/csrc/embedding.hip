// embedding.hip -- rows of a table by token, and the table's gradient.
//
//   out[r] = scale table[tokens[r]]
//   dtable[v] = scale sum over r with tokens[r] = v of dout[r]      (or added to dtable[v])
//
// The gradient adds each token's rows up in an order that the tokens and the extents fix: parts of
// them in the order of r, and then the parts.  The sums of few tokens are each made by the workgroup
// of the token's first position.  More tokens are sorted (stably), the sorted positions are cut into
// chunks of equal length, and a workgroup walks a chunk and stores a token's sum where the token
// changes.  A token whose positions lie in several chunks leaves a sum in the workspace for each,
// which the launch behind adds up.  So no sum depends on the order of atomics, and a token
// that is half of the batch (a frequent word, a pad token) takes as many workgroups as any other
// half.
//
//   order   up to 16384 tokens: each one's place counted.  More: runs of 1024 sorted, each in one
//           workgroup, and merged four at a time
//   sums    by chunk
//   join    of the sums of tokens that cross chunks
//
// The zeros of tokens that are not there are written by more workgroups of the first launch, which
// they hide: a table of 131072 x 4096 bf16 is 1 GB of them.
//
// All sums are fp32 and each value of dtable is rounded once.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "common.hpp"
#include "device_math.hpp"
#include "elem.hpp"

namespace mcke_amd {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxCols = int64_t{1} << 24;

// ---------------------------------------------------------------------------
// Lookup.  2^tpr_log2 lanes a row, U vectors of the table's type a lane.
// ---------------------------------------------------------------------------
template <typename T, typename O, int U, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(
    const int64_t* __restrict__ tokens, const T* __restrict__ table, O* __restrict__ out,
    int64_t rows, int64_t vocab, int cols, float scale, int tpr_log2) {
  constexpr int N = kVecElems<T>;
  const int t = threadIdx.x & ((1 << tpr_log2) - 1);
  const int64_t per_block = kThreads >> tpr_log2;
  const int64_t j0 = ((static_cast<int64_t>(blockIdx.y) * U) << tpr_log2) + t;
  for (int64_t r = blockIdx.x * per_block + (threadIdx.x >> tpr_log2); r < rows;
       r += gridDim.x * per_block) {
    const int64_t token = tokens[r];
    const bool there = token >= 0 && token < vocab;
    const T* row = table + (there ? token : 0) * cols;
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Cols<N, WHOLE> at(j0 + (static_cast<int64_t>(u) << tpr_log2), cols);
      if (at.any && there) {
        at.load(v[u], row);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[u][e] = token < 0 ? 0.0f : __builtin_nanf("");
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Cols<N, WHOLE> at(j0 + (static_cast<int64_t>(u) << tpr_log2), cols);
      if (!at.any) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] *= scale;
      at.store(out + r * cols, v[u]);
    }
  }
}

// ---------------------------------------------------------------------------
// Tokens in order: `keys` and the positions `ids` they come from.  Tokens outside 0 .. vocab - 1
// have the key `vocab`: they come behind all others and are left out.
// ---------------------------------------------------------------------------
constexpr int kRun = 1024;
constexpr int kSortWaves = kRun / kWave;

__device__ __forceinline__ int key_of(const int64_t* __restrict__ tokens, int64_t i, int vocab) {
  const int64_t token = tokens[i];
  return static_cast<int>(token >= 0 && token < vocab ? token : vocab);
}

typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Zeros in `bytes` (an even number) at p (2-byte aligned), by `blocks` workgroups.  Each has one
// piece of them: strided through by all, 1 GB took 260 us, in pieces 165.  (Over two launches 200:
// each has to drain its stores.)
struct Zeros {
  char* p;
  int64_t bytes;
  __device__ __forceinline__ void fill(int64_t block, int64_t blocks) const {
    const int64_t vecs = bytes / 16, per = (vecs + blocks - 1) / blocks;
    const int64_t end = (block + 1) * per < vecs ? (block + 1) * per : vecs;
    for (int64_t i = block * per + threadIdx.x; i < end; i += kRun)
      __builtin_nontemporal_store(u32x4_a2{0u, 0u, 0u, 0u},
                                  reinterpret_cast<u32x4_a2*>(p + 16 * i));
    if (block == 0 && static_cast<int64_t>(threadIdx.x) < bytes % 16 / 2)
      *reinterpret_cast<uint16_t*>(p + 16 * vecs + 2 * threadIdx.x) = 0;
  }
};

// Up to kCount tokens.  A token's place is how many are smaller, and how many equal ones are
// before it: a workgroup has 64 tokens, a lane each, and its waves deal out all of the keys in
// chunks of 64 (in LDS; a chunk is compared with before, behind or at the workgroup's own).
// 16384^2 comparisons are two operations each, 14 us over all CUs; sorted by one workgroup the
// same took 24, in runs of 1024 and two merges 26.  Counting takes the square of the tokens, merges a
// launch for each four times as many: gradients over 8000 x 1024 bf16 take 39 us counted and 44 merged
// at 10000 tokens, 52 and 50 at 16384 (226 and 245 over 131072 x 4096, whose zeros hide the count),
// 69 and 58 at 16385, 85 and 61 at 20000, 125 and 66 at 32768.  Workgroups from `blocks` on write
// zeros.
constexpr int kCount = 16384;

__global__ __launch_bounds__(kRun) void embed_count_kernel(const int64_t* __restrict__ tokens,
                                                          int* __restrict__ keys,
                                                          int* __restrict__ ids, int n, int vocab,
                                                          int blocks, Zeros zeros) {
  __shared__ __attribute__((aligned(16))) int all[kCount];
  __shared__ int counts[kSortWaves][kWave];
  const int block = blockIdx.x;
  if (block >= blocks) {
    zeros.fill(block - blocks, gridDim.x - blocks);
    return;
  }
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int chunks = (n + kWave - 1) / kWave;
  // (INT32_MAX is below nothing: keys go up to 2^31 - 2.)
#pragma unroll 16
  for (int i = threadIdx.x; i < chunks * kWave; i += kRun)
    all[i] = i < n ? key_of(tokens, i, vocab) : INT32_MAX;
  __syncthreads();
  const int mine = block * kWave + lane, key = all[mine];
  int count = 0;
  for (int c = wave; c < chunks; c += kSortWaves) {
    if (c == block) {
#pragma unroll 1
      for (int j = 0; j < kWave; ++j) {
        const int k = all[c * kWave + j];
        count += k < key || (k == key && j < lane) ? 1 : 0;
      }
    } else {
      const int below = c < block ? key : key - 1;
#pragma unroll 4
      for (int j = 0; j < kWave; j += 4) {
        const i32x4 k = *reinterpret_cast<const i32x4*>(all + c * kWave + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) count += k[e] <= below ? 1 : 0;
      }
    }
  }
  counts[wave][lane] = count;
  __syncthreads();
  if (wave > 0 || mine >= n) return;
  for (int w = 1; w < kSortWaves; ++w) count += counts[w][lane];
  keys[count] = key;
  ids[count] = mine;
}

// More tokens.  A run of 1024 is sorted by one workgroup, a token to a lane: least significant
// digit first, up to nine bits a pass.  A lane's rank among equal digits of its wave comes from
// ballots, and the wave's counters, one a digit, give where its waves' tokens of each digit begin.
constexpr int kMaxDigit = 9;

__device__ __forceinline__ void sort_run(const int64_t* __restrict__ tokens, int* __restrict__ keys,
                                         int* __restrict__ ids, int64_t n, int vocab,
                                         int64_t base) {
  __shared__ uint32_t skey[kRun];
  __shared__ uint16_t sid[kRun];
  __shared__ uint32_t count[kSortWaves << kMaxDigit];
  __shared__ uint32_t totals[kSortWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  uint32_t id = threadIdx.x;
  const int64_t i = base + id;
  uint32_t key = static_cast<uint32_t>(i < n ? key_of(tokens, i, vocab) : vocab);
  const int bits = 32 - __builtin_clz(static_cast<unsigned>(vocab));
  const int passes = (bits + kMaxDigit - 1) / kMaxDigit;
  const int width = (bits + passes - 1) / passes, digits = 1 << width;
  for (int shift = 0; shift < bits; shift += width) {
    for (int c = threadIdx.x; c < kSortWaves * digits; c += kRun) count[c] = 0;
    __syncthreads();
    const uint32_t d = (key >> shift) & (digits - 1);
    uint64_t same = ~uint64_t{0};
    for (int b = 0; b < width; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? set : ~set;
    }
    const uint32_t rank = __popcll(same & ((uint64_t{1} << lane) - 1));
    if (rank == 0) count[wave * digits + d] = __popcll(same);
    __syncthreads();
    // The counters' sums before each, by digit and then by wave.
    const int entries = kSortWaves * digits;
    const int per = (entries + kRun - 1) / kRun;
    const int e0 = threadIdx.x * per;
    uint32_t sum = 0;
    for (int e = e0; e < e0 + per && e < entries; ++e)
      sum += count[(e % kSortWaves) * digits + e / kSortWaves];
    uint32_t upto = sum;
#pragma unroll
    for (int s = 1; s < kWave; s *= 2) {
      const uint32_t other = __shfl_up(upto, s);
      if (lane >= s) upto += other;
    }
    if (lane == kWave - 1) totals[wave] = upto;
    __syncthreads();
    uint32_t start = upto - sum;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) start += w < wave ? totals[w] : 0;
    for (int e = e0; e < e0 + per && e < entries; ++e) {
      uint32_t& c = count[(e % kSortWaves) * digits + e / kSortWaves];
      const uint32_t have = c;
      c = start;
      start += have;
    }
    __syncthreads();
    const uint32_t to = count[wave * digits + d] + rank;
    skey[to] = key;
    sid[to] = static_cast<uint16_t>(id);
    __syncthreads();
    key = skey[threadIdx.x];
    id = sid[threadIdx.x];
    __syncthreads();
  }
  // What fills up the last run is behind all of the run's own tokens.
  if (i < n) {
    keys[i] = static_cast<int>(key);
    ids[i] = static_cast<int>(base + id);
  }
}

// Workgroups 0 .. runs - 1 sort a run each, the others write zeros.
__global__ __launch_bounds__(kRun) void embed_sort_kernel(const int64_t* __restrict__ tokens,
                                                         int* __restrict__ keys,
                                                         int* __restrict__ ids, int n, int vocab,
                                                         int runs, Zeros zeros) {
  if (static_cast<int>(blockIdx.x) < runs)
    sort_run(tokens, keys, ids, n, vocab, static_cast<int64_t>(blockIdx.x) * kRun);
  else
    zeros.fill(blockIdx.x - runs, gridDim.x - runs);
}

// Four sorted runs of `len` become one: an element's place is its own in its run plus, for each
// other run, how many there come before it (equal keys: those of earlier runs).  The searches of
// the runs go in step, in LDS: all of their keys where they are 1024 long, else every
// len / 1024-th and the last few steps in memory.  (Sixteen runs at once: 15 searches an element
// took 20 us for 16384 tokens, and 44 with all steps in memory.)
constexpr int kMergeWays = 4, kSamples = kRun;

__global__ __launch_bounds__(kThreads) void embed_merge_kernel(const int* __restrict__ keys,
                                                              const int* __restrict__ ids,
                                                              int* __restrict__ keys_out,
                                                              int* __restrict__ ids_out, int n,
                                                              int len) {
  __shared__ int samples[kMergeWays * kSamples];
  // Runs are whole workgroups long, so a workgroup's elements are one run's.
  const unsigned i0 = blockIdx.x * kThreads, run = i0 / static_cast<unsigned>(len);
  const int mine = run % kMergeWays, apart = len / kSamples;
  const int64_t first = static_cast<int64_t>(run - mine) * len;
#pragma unroll
  for (int k = 0; k < kMergeWays * kSamples / kThreads; ++k) {
    const int q = k * kThreads + threadIdx.x;
    const int64_t at = first + static_cast<int64_t>(q) * apart;
    samples[q] = at < n ? keys[at] : INT32_MAX;
  }
  const unsigned i = i0 + threadIdx.x;
  const int key = i < static_cast<unsigned>(n) ? keys[i] : 0;
  const int id = i < static_cast<unsigned>(n) ? ids[i] : 0;
  __syncthreads();
  if (i >= static_cast<unsigned>(n)) return;
  // Of run w, the samples that come before this element: up to `key` in earlier runs, below it in
  // later ones (keys are >= 0).
  int below[kMergeWays] = {};
#pragma unroll 1
  for (int s = kSamples; s > 0; s /= 2) {
#pragma unroll
    for (int w = 0; w < kMergeWays; ++w) {
      const int at = below[w] + s;
      if (at <= kSamples && samples[w * kSamples + at - 1] <= key - (w > mine)) below[w] = at;
    }
  }
  // Between the last of them and the next sample: `apart` - 1 elements.
  int64_t lo[kMergeWays];
#pragma unroll
  for (int w = 0; w < kMergeWays; ++w)
    lo[w] = below[w] > 0 ? int64_t{below[w] - 1} * apart + 1 : 0;
#pragma unroll 1
  for (int s = apart / 2; s > 0; s /= 2) {
#pragma unroll
    for (int w = 0; w < kMergeWays; ++w) {
      const int64_t at = first + static_cast<int64_t>(w) * len + lo[w] + s - 1;
      if (below[w] > 0 && w != mine && at < n && keys[at] <= key - (w > mine)) lo[w] += s;
    }
  }
  int64_t to = first + (i - static_cast<int64_t>(run) * len);
#pragma unroll
  for (int w = 0; w < kMergeWays; ++w) to += w == mine ? 0 : lo[w];
  keys_out[to] = key;
  ids_out[to] = id;
}

// ---------------------------------------------------------------------------
// Sums
// ---------------------------------------------------------------------------
template <typename T, int N, bool WHOLE>
__device__ __forceinline__ void store_sum(T* __restrict__ row, const Cols<N, WHOLE>& at,
                                          const float (&sum)[N], float scale, bool accumulate) {
  float v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = scale * sum[e];
  if (accumulate) {
    float old[N];
    at.load(old, row);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += old[e];
  }
  at.store(row, v);
}

// 2^tpr_log2 lanes walk a chunk: positions chunk * P .. of the sorted tokens.  A token that began
// before the chunk leaves its sum at partials[2 chunk], one that goes on behind it at
// partials[2 chunk + 1] (at [2 chunk] if it does both).
// WAVES: a chunk is whole waves', and what it reads of the tokens is the same for all lanes.
constexpr int kAhead = 8;       // rows whose loads are in flight

template <typename T, typename O, bool WHOLE, bool WAVES>
__global__ __launch_bounds__(kThreads) void embed_sums_kernel(
    const int* __restrict__ keys, const int* __restrict__ ids, const O* __restrict__ dout,
    T* __restrict__ dtable, float* __restrict__ partials, int64_t n, int vocab, int cols, int64_t P,
    int tiles, int tpr_log2, float scale, bool accumulate) {
  constexpr int N = kVecElems<O>;
  int group = threadIdx.x >> tpr_log2;
  if constexpr (WAVES) group = __builtin_amdgcn_readfirstlane(group);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x / tiles) * (kThreads >> tpr_log2) + group;
  const Cols<N, WHOLE> at((static_cast<int64_t>(blockIdx.x % tiles) << tpr_log2) +
                              (threadIdx.x & ((1 << tpr_log2) - 1)), cols);
  const int64_t begin = chunk * P, end = begin + P < n ? begin + P : n;
  // (All lanes of a wave take part in what its lanes tell each other.)
  if (begin >= n || (WAVES ? __ballot(at.any) == 0 : !at.any)) return;
  int key = keys[begin];
  if (key == vocab) return;
  bool head = begin > 0 && keys[begin - 1] == key;
  float sum[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = 0.0f;
  // Takes a row whose next token is `next`; true where the chunk's tokens end.
  auto take = [&](const PackT<O, N>& v, int next, bool last) {
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] += static_cast<float>(v[e]);
    const bool goes_on = next == key;
    if (goes_on && !last) return false;
    if (at.any) {
      if (head || goes_on)
        at.store(partials + (2 * chunk + (head ? 0 : 1)) * cols, sum);
      else
        store_sum<T, N, WHOLE>(dtable + static_cast<int64_t>(key) * cols, at, sum, scale,
                               accumulate);
    }
    head = false;
    key = next;
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.0f;
    return key == vocab;
  };
  if constexpr (WAVES) {
    // 64 positions at a time, one to a lane; the rows that they name are loaded ahead of the
    // additions, which wait for no other load.
    const int lane = threadIdx.x % kWave;
    for (int64_t s0 = begin; s0 < end; s0 += kWave) {
      const int m = static_cast<int>(end - s0 < kWave ? end - s0 : kWave);
      const int64_t i = s0 + (lane < m ? lane : m - 1);
      const int id = ids[i], after = i + 1 < n ? keys[i + 1] : vocab;
      auto load = [&](int k, PackT<O, N> (&v)[kAhead]) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int row = __builtin_amdgcn_readlane(id, k + u < m ? k + u : m - 1);
          if (at.any) v[u] = at.load_raw(dout + static_cast<int64_t>(row) * cols);
        }
      };
      PackT<O, N> v[kAhead] = {}, w[kAhead] = {};
      load(0, v);
      for (int k = 0; k < m; k += kAhead) {
        if (k + kAhead < m) load(k + kAhead, w);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (k + u >= m) break;
          if (take(v[u], __builtin_amdgcn_readlane(after, k + u), s0 + k + u + 1 == end)) return;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = w[u];
      }
    }
  } else {
    for (int64_t i0 = begin; i0 < end; i0 += kAhead) {
      PackT<O, N> v[kAhead];
      int next[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t i = i0 + k < end ? i0 + k : end - 1;
        next[k] = i + 1 < n ? keys[i + 1] : vocab;
        v[k] = at.load_raw(dout + static_cast<int64_t>(ids[i]) * cols);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i0 + k >= end) break;
        if (take(v[k], next[k], i0 + k + 1 == end)) return;
      }
    }
  }
}

// Tokens that begin in one chunk and end in a later one.  Each group of 2^tpr_log2 lanes looks
// at a chunk, and adds up its token's sums if that ends within kNear chunks.  Tokens that go
// further are added up by all groups, which deal out the later chunks (of G groups each every
// G-th); then the groups' sums are added up.
constexpr int kNear = 16;

template <typename T, int N, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embed_join_kernel(
    const int* __restrict__ keys, T* __restrict__ dtable, const float* __restrict__ partials,
    int64_t n, int vocab, int cols, int64_t P, int chunks, int tiles, int tpr_log2, float scale,
    bool accumulate) {
  __shared__ float fold[kThreads * N];
  __shared__ int far_key[32];                 // of each group's chunk, or -1
  const int groups = kThreads >> tpr_log2, tpr = 1 << tpr_log2;
  const int group = threadIdx.x >> tpr_log2, t = threadIdx.x & (tpr - 1);
  const int c0 = blockIdx.x / tiles * groups;
  const Cols<N, WHOLE> at((static_cast<int64_t>(blockIdx.x % tiles) << tpr_log2) + t, cols);
  // Adds up the first sums of chunks c, c + step, .. up to `last`.
  auto add = [&](float (&sum)[N], int c, int last, int step) {
    constexpr int U = WHOLE ? 8 : 4;
    for (; c <= last; c += U * step) {
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
        at.load(v[u], partials + 2 * static_cast<int64_t>(c + u * step <= last ? c + u * step : last) *
                                     cols);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * step > last) break;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[u][e];
      }
    }
  };
  float sum[N];
  const int mine = c0 + group;
  int far = -1;
  if (mine + 1 < chunks) {
    const int64_t begin = mine * P, end = begin + P;
    const int key = keys[end - 1], before = begin > 0 ? keys[begin - 1] : -1;
    int later = 0;                            // chunks that begin with the token
#pragma unroll
    for (int u = 0; u < kNear; ++u)
      later += mine + 1 + u < chunks && keys[end + u * P] == key ? 1 : 0;
    if (key != vocab && before != key && later > 0) {
      if (later == kNear) {
        far = key;
      } else if (at.any) {
        at.load(sum, partials + (2 * static_cast<int64_t>(mine) + 1) * cols);
        add(sum, mine + 1, mine + later, 1);
        store_sum<T, N, WHOLE>(dtable + static_cast<int64_t>(key) * cols, at, sum, scale,
                               accumulate);
      }
    }
  }
  if (t == 0) far_key[group] = far;
  __syncthreads();
  for (int g = 0; g < groups; ++g) {
    const int key = far_key[g], chunk = c0 + g;
    if (key < 0) continue;
    int last = chunk;
    for (int c = chunk + 1; c < chunks; c += kThreads) {
      const int q = c + static_cast<int>(threadIdx.x);
      const int have = __syncthreads_count(q < chunks && keys[q * P] == key);
      last += have;
      if (have < kThreads) break;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.0f;
    if (at.any) add(sum, chunk + 1 + group, last, groups);
#pragma unroll
    for (int e = 0; e < N; ++e) fold[e * kThreads + threadIdx.x] = sum[e];
    __syncthreads();
    if (group == 0 && at.any) {
      at.load(sum, partials + (2 * static_cast<int64_t>(chunk) + 1) * cols);
      for (int k = 0; k < groups; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += fold[e * kThreads + k * tpr + t];
      store_sum<T, N, WHOLE>(dtable + static_cast<int64_t>(key) * cols, at, sum, scale,
                             accumulate);
    }
    __syncthreads();      // fold is written again
  }
}

// Few tokens: nothing is sorted.  A workgroup has a position, and goes on where that is its token's
// first: the token's positions are listed in order, one or two waves have a tile of columns each and
// the others the same tiles of later positions.  Up to 512 tokens and 2048 workgroups: 500 tokens
// over 8000 x 512 bf16 take 8.3 us and 16.2 in order of tokens, 4096 columns of 1000 13.2 and 17.9,
// 4096 columns of fp32 (4000 workgroups) 38.6 and 34.3.  (512 times the same token: 512 columns 15.0
// and 24.6, 4096 32.7 and 29.4.)
constexpr int kOnce = 512, kOnceWaves = kOnce / kWave, kOnceAhead = 16;
constexpr int64_t kOnceMost = 2048;             // workgroups

template <typename T, typename O, bool WHOLE>
__global__ __launch_bounds__(kOnce) void embed_once_kernel(
    const int64_t* __restrict__ tokens, const O* __restrict__ dout, T* __restrict__ dtable, int n,
    int vocab, int cols, int tiles, int slots_log2, float scale, bool accumulate) {
  constexpr int N = kVecElems<O>;
  __shared__ int keys[kOnce];
  __shared__ int ids[kOnce];
  __shared__ float parts[kOnceWaves][N * kWave];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int mine = blockIdx.x / tiles;
  keys[threadIdx.x] =
      static_cast<int>(threadIdx.x) < n ? key_of(tokens, threadIdx.x, vocab) : vocab;
  __syncthreads();
  const int key = keys[mine];
  if (key == vocab) return;
  int count = 0, before = 0;               // positions of the token; of them in earlier waves'
  bool earlier = false;
#pragma unroll
  for (int w = 0; w < kOnceWaves; ++w) {
    const uint64_t set = __ballot(keys[w * kWave + lane] == key);
    const int at = mine - w * kWave;       // where this position is in the wave's
    earlier |= (at >= kWave ? set : at > 0 ? set & ((uint64_t{1} << at) - 1) : 0) != 0;
    if (w < wave) before += __popcll(set);
    if (w == wave && (set >> lane & 1))
      ids[before + __popcll(set & ((uint64_t{1} << lane) - 1))] = static_cast<int>(threadIdx.x);
    count += __popcll(set);
  }
  if (earlier) return;
  __syncthreads();
  const int slots = 1 << slots_log2, splits = kOnceWaves >> slots_log2;
  const int slot = wave % slots, split = wave / slots;
  const Cols<N, WHOLE> at(
      (static_cast<int64_t>(blockIdx.x % tiles) * slots + slot) * kWave + lane, cols);
  // Positions a wave: one load's worth at least.
  const int even = (count + splits - 1) / splits, per = even > kOnceAhead ? even : kOnceAhead;
  const int begin = split * per, end = begin + per < count ? begin + per : count;
  float sum[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = 0.0f;
  auto add = [&]<int U>(int k) {
    PackT<O, N> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = at.load_raw(dout + static_cast<int64_t>(ids[k + u < end ? k + u : end - 1]) * cols);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < end)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += static_cast<float>(v[u][e]);
  };
  if (at.any) {
    int k = begin;
    for (; k + kOnceAhead <= end; k += kOnceAhead) add.template operator()<kOnceAhead>(k);
    for (; k < end; k += 2) add.template operator()<2>(k);
  }
  if (per < count) {
#pragma unroll
    for (int e = 0; e < N; ++e) parts[wave][e * kWave + lane] = sum[e];
    __syncthreads();
    if (split == 0)
      for (int p = 1; p * per < count; ++p)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += parts[p * slots + slot][e * kWave + lane];
  }
  if (split == 0 && at.any)
    store_sum<T, N, WHOLE>(dtable + static_cast<int64_t>(key) * cols, at, sum, scale, accumulate);
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }


// Lanes that a row takes, as 2^this: as many as cover it with vectors of N, 8 to a workgroup.
int lanes_log2(int64_t cols, int n) {
  int log2 = 3;
  while (log2 < 8 && (int64_t{n} << log2) < cols) ++log2;
  return log2;
}

// Positions a chunk: up to 512 workgroups of chunks.  (By vectors of 8: of rows and cols alone, so
// that the workspace is sized without the types.)
int64_t chunk_of(int64_t rows, int64_t cols) {
  const int64_t chunks = int64_t{512} << (8 - lanes_log2(cols, 8));
  int64_t p = 4;
  while (chunks * p < rows) p *= 2;
  return p;
}

struct Workspace {
  int64_t list, partials;       // bytes of a list of tokens or positions; of the partial sums
  int lists;                    // 2, or 4 where runs are merged
  Workspace(int64_t rows, int64_t cols) {
    list = (4 * rows + 15) / 16 * 16;
    lists = rows > kCount ? 4 : 2;
    partials = 2 * ceil_div(rows, chunk_of(rows, cols)) * cols * 4;
  }
  int64_t bytes() const { return list * lists + partials; }
};

int check_extents(const std::string& who, int table_dtype, int out_dtype, const char* out_name,
                  int64_t rows, int64_t vocab, int64_t cols, float scale) {
  if (!is_dtype(table_dtype)) return invalid(who + ": unknown table_dtype " + std::to_string(table_dtype));
  if (out_dtype != MCKE_DTYPE_F32 && out_dtype != table_dtype)
    return invalid(who + ": " + out_name + " must be MCKE_DTYPE_F32 or table_dtype, got " +
                   std::to_string(out_dtype));
  if (rows < 0 || vocab < 0 || cols < 0) return invalid(who + ": negative extent");
  if (rows > INT32_MAX || vocab >= INT32_MAX || cols > kMaxCols)
    return invalid(who + ": too large: rows up to 2^31 - 1, vocab up to 2^31 - 2, cols up to 2^24");
  if (!std::isfinite(scale)) return invalid(who + ": scale must be finite");
  return ok();
}

template <typename T, typename O>
int launch_fwd(const int64_t* tokens, const void* table, void* out, int64_t rows, int64_t vocab,
               int64_t cols, float scale, hipStream_t s) {
  constexpr int N = kVecElems<T>;
  const int64_t vecs = ceil_div(cols, N);
  const int tpr_log2 = lanes_log2(cols, N);
  const int u = vecs > 256 ? 2 : 1;
  const int64_t y = ceil_div(vecs, int64_t{u} << tpr_log2);
  const int64_t groups = ceil_div(rows, kThreads >> tpr_log2);
  const int64_t most = (int64_t{1} << 22) / y;        // of 2^24 threads to the grid's 2^32
  const dim3 grid(static_cast<unsigned>(groups < most ? groups : most), static_cast<unsigned>(y));
  const bool whole = cols % N == 0;
  auto* fn = u == 2 ? (whole ? &embed_fwd_kernel<T, O, 2, true> : &embed_fwd_kernel<T, O, 2, false>)
                    : (whole ? &embed_fwd_kernel<T, O, 1, true> : &embed_fwd_kernel<T, O, 1, false>);
  fn<<<grid, kThreads, 0, s>>>(tokens, static_cast<const T*>(table), static_cast<O*>(out), rows,
                               vocab, static_cast<int>(cols), scale, tpr_log2);
  MCKE_LAUNCH_CHECK("embed_fwd_kernel");
  return ok();
}

struct BwdArgs {
  const int64_t* tokens;
  const void* dout;
  void* dtable;
  int64_t rows, vocab, cols;
  float scale;
  bool accumulate;
  char* ws;
  hipStream_t s;
};

template <typename T, typename O, bool WHOLE>
int launch_sums(const BwdArgs& a, const int* keys, const int* ids, float* partials) {
  constexpr int N = kVecElems<O>;
  const int64_t P = chunk_of(a.rows, a.cols), chunks = ceil_div(a.rows, P);
  const int tpr_log2 = lanes_log2(a.cols, N), groups = kThreads >> tpr_log2;
  const int tiles = static_cast<int>(ceil_div(a.cols, int64_t{N} << tpr_log2));
  const int vocab = static_cast<int>(a.vocab), cols = static_cast<int>(a.cols);
  const unsigned grid = static_cast<unsigned>(ceil_div(chunks, groups) * tiles);
  auto* fn = tpr_log2 >= 6 ? &embed_sums_kernel<T, O, WHOLE, true>
                           : &embed_sums_kernel<T, O, WHOLE, false>;
  fn<<<grid, kThreads, 0, a.s>>>(keys, ids, static_cast<const O*>(a.dout),
                                 static_cast<T*>(a.dtable), partials, a.rows, vocab, cols, P, tiles,
                                 tpr_log2, a.scale, a.accumulate);
  MCKE_LAUNCH_CHECK("embed_sums_kernel");
  if (chunks == 1) return ok();
  // The join has few sums to a lane: at most a wave a row, so that there are four groups or more.
  const int join_log2 = tpr_log2 < 6 ? tpr_log2 : 6;
  const int join_tiles = static_cast<int>(ceil_div(a.cols, int64_t{N} << join_log2));
  const unsigned join_grid =
      static_cast<unsigned>(ceil_div(chunks, kThreads >> join_log2) * join_tiles);
  embed_join_kernel<T, N, WHOLE><<<join_grid, kThreads, 0, a.s>>>(
      keys, static_cast<T*>(a.dtable), partials, a.rows, vocab, cols, P, static_cast<int>(chunks),
      join_tiles, join_log2, a.scale, a.accumulate);
  MCKE_LAUNCH_CHECK("embed_join_kernel");
  return ok();
}

// Workgroups a position.
template <typename O> int64_t once_tiles(int64_t cols) {
  return ceil_div(cols, 2 * kVecElems<O> * kWave);
}

template <typename T, typename O, bool WHOLE> int launch_once(const BwdArgs& a) {
  const int64_t tiles = once_tiles<O>(a.cols);
  const int slots_log2 = a.cols > kVecElems<O> * kWave ? 1 : 0;
  embed_once_kernel<T, O, WHOLE><<<static_cast<unsigned>(a.rows * tiles), kOnce, 0, a.s>>>(
      a.tokens, static_cast<const O*>(a.dout), static_cast<T*>(a.dtable), static_cast<int>(a.rows),
      static_cast<int>(a.vocab), static_cast<int>(a.cols), static_cast<int>(tiles), slots_log2,
      a.scale, a.accumulate);
  MCKE_LAUNCH_CHECK("embed_once_kernel");
  return ok();
}

template <typename T, typename O> int launch_bwd(const BwdArgs& a) {
  const Workspace w(a.rows, a.cols);
  int* keys = reinterpret_cast<int*>(a.ws);
  int* ids = reinterpret_cast<int*>(a.ws + w.list);
  // Zeros in pieces of 32 KB at least, 4096 at most (512 of them 3 us slower for 1 GB, 16384 25).
  const Zeros zeros{static_cast<char*>(a.dtable),
                    a.accumulate ? 0 : a.vocab * a.cols * static_cast<int64_t>(sizeof(T))};
  const int64_t pieces = ceil_div(zeros.bytes, 32 * 1024), fill = pieces < 4096 ? pieces : 4096;
  const bool once = a.rows <= kOnce && a.rows * once_tiles<O>(a.cols) <= kOnceMost;
  const bool count = a.rows <= kCount;
  const int64_t blocks = once ? 0 : ceil_div(a.rows, count ? kWave : kRun);
  if (blocks + fill > 0) {
    auto* fn = count ? &embed_count_kernel : &embed_sort_kernel;
    fn<<<static_cast<unsigned>(blocks + fill), kRun, 0, a.s>>>(
        a.tokens, keys, ids, static_cast<int>(a.rows), static_cast<int>(a.vocab),
        static_cast<int>(blocks), zeros);
    MCKE_LAUNCH_CHECK("embed_count_kernel or embed_sort_kernel");
  }
  if (a.rows == 0) return ok();
  if (once)
    return a.cols % kVecElems<O> == 0 ? launch_once<T, O, true>(a) : launch_once<T, O, false>(a);
  int turn = 0;
  for (int64_t len = kRun; !count && len < a.rows; len *= kMergeWays, ++turn) {
    int* to = reinterpret_cast<int*>(a.ws + (turn % 2 ? 0 : 2 * w.list));
    int* ids_to = reinterpret_cast<int*>(reinterpret_cast<char*>(to) + w.list);
    embed_merge_kernel<<<static_cast<unsigned>(ceil_div(a.rows, kThreads)), kThreads, 0, a.s>>>(
        keys, ids, to, ids_to, static_cast<int>(a.rows), static_cast<int>(len));
    MCKE_LAUNCH_CHECK("embed_merge_kernel");
    keys = to;
    ids = ids_to;
  }
  float* partials = reinterpret_cast<float*>(a.ws + w.list * w.lists);
  return a.cols % kVecElems<O> == 0 ? launch_sums<T, O, true>(a, keys, ids, partials)
                                    : launch_sums<T, O, false>(a, keys, ids, partials);
}

}  // namespace
}  // namespace mcke_amd

using namespace mcke_amd;

extern "C" {

int mcke_launch_embedding(const int64_t* tokens, const void* table, void* out, int table_dtype,
                          int out_dtype, int64_t rows, int64_t vocab, int64_t cols, float scale,
                          void* stream) {
  const std::string who = "launch_embedding";
  if (int rc = check_extents(who, table_dtype, out_dtype, "out_dtype", rows, vocab, cols, scale))
    return rc;
  if (rows == 0 || cols == 0) return ok();
  if (!tokens || !out || (vocab > 0 && !table)) return invalid(who + ": null pointer");
  const uint64_t te = dtype_bytes(table_dtype), oe = dtype_bytes(out_dtype);
  if (!aligned(tokens, 8) || !aligned(table, te) || !aligned(out, oe))
    return invalid(who + ": a pointer is not aligned to its type");
  const uint64_t n = rows, c = cols, v = vocab;
  if (overlap(out, n * c * oe, tokens, 8 * n) || overlap(out, n * c * oe, table, v * c * te))
    return invalid(who + ": output overlaps an input, which violates the __restrict__ contract");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (table_dtype == MCKE_DTYPE_F32)
    return launch_fwd<float, float>(tokens, table, out, rows, vocab, cols, scale, s);
  if (table_dtype == MCKE_DTYPE_F16)
    return out_dtype == MCKE_DTYPE_F32
               ? launch_fwd<_Float16, float>(tokens, table, out, rows, vocab, cols, scale, s)
               : launch_fwd<_Float16, _Float16>(tokens, table, out, rows, vocab, cols, scale, s);
  return out_dtype == MCKE_DTYPE_F32
             ? launch_fwd<__bf16, float>(tokens, table, out, rows, vocab, cols, scale, s)
             : launch_fwd<__bf16, __bf16>(tokens, table, out, rows, vocab, cols, scale, s);
}

size_t mcke_embedding_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t cols) {
  if (rows <= 0 || rows > INT32_MAX || vocab <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  return static_cast<size_t>(Workspace(rows, cols).bytes());
}

int mcke_launch_embedding_backward(const int64_t* tokens, const void* dout, void* dtable,
                                   int dout_dtype, int table_dtype, int64_t rows, int64_t vocab,
                                   int64_t cols, float scale, int accumulate, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const std::string who = "launch_embedding_backward";
  if (int rc = check_extents(who, table_dtype, dout_dtype, "dout_dtype", rows, vocab, cols, scale))
    return rc;
  if (vocab == 0 || cols == 0) return ok();
  if (!dtable || (rows > 0 && (!tokens || !dout))) return invalid(who + ": null pointer");
  const uint64_t te = dtype_bytes(table_dtype), oe = dtype_bytes(dout_dtype);
  if (!aligned(tokens, 8) || !aligned(dtable, te) || !aligned(dout, oe))
    return invalid(who + ": a pointer is not aligned to its type");
  const size_t need = mcke_embedding_backward_workspace_bytes(rows, vocab, cols);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return invalid(who + ": the sorted tokens need a 16-byte aligned workspace of " +
                   std::to_string(need) + " bytes, got " +
                   std::to_string(workspace ? workspace_bytes : 0));
  const uint64_t n = rows, c = cols, table = static_cast<uint64_t>(vocab) * c * te;
  if (overlap(dtable, table, tokens, 8 * n) || overlap(dtable, table, dout, n * c * oe) ||
      overlap(workspace, need, tokens, 8 * n) || overlap(workspace, need, dout, n * c * oe) ||
      overlap(workspace, need, dtable, table))
    return invalid(who + ": the output or the workspace overlaps another operand, which violates "
                         "the __restrict__ contract");
  const BwdArgs a{tokens, dout, dtable, rows, vocab, cols, scale, accumulate != 0,
                  static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
  if (table_dtype == MCKE_DTYPE_F32) return launch_bwd<float, float>(a);
  if (table_dtype == MCKE_DTYPE_F16)
    return dout_dtype == MCKE_DTYPE_F32 ? launch_bwd<_Float16, float>(a)
                                        : launch_bwd<_Float16, _Float16>(a);
  return dout_dtype == MCKE_DTYPE_F32 ? launch_bwd<__bf16, float>(a)
                                      : launch_bwd<__bf16, __bf16>(a);
}

}  // extern "C"
