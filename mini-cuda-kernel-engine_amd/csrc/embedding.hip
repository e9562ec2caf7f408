// embedding.hip -- rows of a table by token, and the table's gradient.
//
//   out[r] = scale table[tokens[r]]
//   dtable[v] = scale sum over r with tokens[r] = v of dout[r]      (or added to dtable[v])
//
// The gradient adds each token's rows up in the order of r, whatever the launch: the tokens are
// sorted (stably), the sorted positions are cut into chunks of equal length, and a workgroup
// walks a chunk and stores a token's sum where the token changes.  A token whose positions lie
// in several chunks leaves a sum in the workspace for each, which the launch behind adds up in
// order.  So no sum depends on the order of atomics, and a token that is half of the batch (a
// frequent word, a pad token) takes as many workgroups as any other half.
//
//   launch 1  sorts runs of tokens, each in one workgroup's LDS, beside workgroups that write the
//             zeros of tokens that are not there: a table of 131072 x 4096 bf16 is 1 GB of them,
//             which hides the sort
//   (merges   eight runs at a time, where there is more than one)
//   launch 2  sums by chunk      launch 3  sums of tokens that cross chunks
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

// N values at the alignment of one.
template <typename T, int N> struct Pack {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N> using PackT = typename Pack<T, N>::type;

template <typename T, int N>
__device__ __forceinline__ void load_cols(float (&v)[N], const T* __restrict__ p) {
  const PackT<T, N> w = *reinterpret_cast<const PackT<T, N>*>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = static_cast<float>(w[e]);
}

// A lane's N columns of a row: columns j N .. j N + N - 1.  In rows that are not whole vectors
// (WHOLE false) the last one is moved back to end with the row, and its first `skip` columns are
// its neighbour's too; a row shorter than a vector is one vector cut at `n`.
template <int N, bool WHOLE> struct Cols {
  int c, skip, n;
  bool any;
  __device__ __forceinline__ Cols(int64_t j, int cols) {
    const int64_t first = j * N;
    any = first < cols;
    c = static_cast<int>(first);
    skip = 0;
    n = N;
    if constexpr (!WHOLE) {
      if (first + N > cols) {
        c = cols > N ? cols - N : 0;
        skip = static_cast<int>(first) - c;
        n = cols < N ? cols : N;
      }
    }
  }
  template <typename T> __device__ __forceinline__ void load(float (&v)[N], const T* row) const {
    if (WHOLE || n == N) {
      load_cols<T, N>(v, row + c);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = e < n ? static_cast<float>(row[c + e]) : 0.0f;
    }
  }
  // Columns that are this lane's alone, so that each is written once.
  template <typename T> __device__ __forceinline__ void store(T* row, const float (&v)[N]) const {
    if (WHOLE || (skip == 0 && n == N)) {
      PackT<T, N> w;
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = static_cast<T>(v[e]);
      *reinterpret_cast<PackT<T, N>*>(row + c) = w;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e >= skip && e < n) row[c + e] = static_cast<T>(v[e]);
    }
  }
};

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
// Sorted tokens.  A run of 1024 J tokens is sorted by one workgroup: least significant digit
// first, up to nine bits a pass.  A wave holds 64 J consecutive positions, 64 to a register, so
// that "earlier" is a lower register, then a lower lane.  A lane's rank among equal digits of
// its register comes from ballots; the wave's counters, one a digit, give what came before.
// Tokens outside 0 .. vocab - 1 have the key `vocab`: they sort behind all others and are left
// out.
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kMaxDigit = 9;

template <int J>
__device__ __forceinline__ void sort_run(const int64_t* __restrict__ tokens, int* __restrict__ keys,
                                         int* __restrict__ ids, int64_t n, int vocab,
                                         int64_t base) {
  __shared__ uint32_t skey[kSortThreads * J];
  __shared__ uint16_t sid[kSortThreads * J];
  __shared__ uint32_t count[kSortWaves << kMaxDigit];
  __shared__ uint32_t totals[kSortWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int at0 = wave * (kWave * J) + lane;

  uint32_t key[J], id[J], rank[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    id[j] = at0 + j * kWave;
    const int64_t i = base + id[j];
    const int64_t token = i < n ? tokens[i] : -1;
    key[j] = static_cast<uint32_t>(token >= 0 && token < vocab ? token : vocab);
  }
  const int bits = 32 - __builtin_clz(static_cast<unsigned>(vocab));
  const int passes = (bits + kMaxDigit - 1) / kMaxDigit;
  const int width = (bits + passes - 1) / passes, digits = 1 << width;
  for (int shift = 0; shift < bits; shift += width) {
    for (int c = threadIdx.x; c < kSortWaves * digits; c += kSortThreads) count[c] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t d = (key[j] >> shift) & (digits - 1);
      uint64_t same = ~uint64_t{0};
      for (int b = 0; b < width; ++b) {
        const uint64_t set = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
      }
      const int before = __popcll(same & ((uint64_t{1} << lane) - 1));
      uint32_t old = 0;
      if (before == 0) old = atomicAdd(&count[wave * digits + d], __popcll(same));
      rank[j] = __shfl(old, __builtin_ctzll(same)) + before;
    }
    __syncthreads();
    // The counters' sums before each, by digit and then by wave.
    const int entries = kSortWaves * digits;
    const int per = (entries + kSortThreads - 1) / kSortThreads;
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
    for (int w = 0; w < wave; ++w) start += totals[w];
    for (int e = e0; e < e0 + per && e < entries; ++e) {
      uint32_t& c = count[(e % kSortWaves) * digits + e / kSortWaves];
      const uint32_t have = c;
      c = start;
      start += have;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t to = count[wave * digits + ((key[j] >> shift) & (digits - 1))] + rank[j];
      skey[to] = key[j];
      sid[to] = static_cast<uint16_t>(id[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      key[j] = skey[at0 + j * kWave];
      id[j] = sid[at0 + j * kWave];
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    // What fills up the last run is behind all of the run's own tokens.
    const int64_t i = base + at0 + j * kWave;
    if (i < n) {
      keys[i] = static_cast<int>(key[j]);
      ids[i] = static_cast<int>(base + id[j]);
    }
  }
}

typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// Workgroups 0 .. runs - 1 sort a run each, the others fill `zeros` bytes (an even number) at
// `fill` (2-byte aligned).
template <int J>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(
    const int64_t* __restrict__ tokens, int* __restrict__ keys, int* __restrict__ ids, int64_t n,
    int vocab, int runs, char* __restrict__ fill, int64_t zeros) {
  if (static_cast<int>(blockIdx.x) < runs) {
    sort_run<J>(tokens, keys, ids, n, vocab,
                static_cast<int64_t>(blockIdx.x) * (kSortThreads * J));
    return;
  }
  const int64_t step = static_cast<int64_t>(gridDim.x - runs) * kSortThreads;
  int64_t i = static_cast<int64_t>(blockIdx.x - runs) * kSortThreads + threadIdx.x;
  if (i < zeros % 16 / 2) *reinterpret_cast<uint16_t*>(fill + zeros / 16 * 16 + 2 * i) = 0;
  for (; i < zeros / 16; i += step)
    __builtin_nontemporal_store(u32x4_a2{0u, 0u, 0u, 0u},
                                reinterpret_cast<u32x4_a2*>(fill + 16 * i));
}

// Eight sorted runs of `len` become one: an element's place is its own in its run plus, for each
// other run, how many there come before it (equal keys: those of earlier runs).
constexpr int kMergeWays = 8;

__global__ __launch_bounds__(kThreads) void embed_merge_kernel(
    const int* __restrict__ keys, const int* __restrict__ ids, int* __restrict__ keys_out,
    int* __restrict__ ids_out, int64_t n, int64_t len) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const int key = keys[i];
  const int64_t run = i / len, first = run / kMergeWays * kMergeWays;
  int64_t to = first * len + (i - run * len);
  for (int64_t other = first; other < first + kMergeWays && other * len < n; ++other) {
    if (other == run) continue;
    const int upto = other < run ? key : key - 1;    // keys are >= 0
    const int64_t begin = other * len, end = begin + len < n ? begin + len : n;
    int64_t lo = begin, hi = end;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (keys[mid] <= upto) lo = mid + 1;
      else hi = mid;
    }
    to += lo - begin;
  }
  keys_out[to] = key;
  ids_out[to] = ids[i];
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

// Workgroup (chunk, columns): positions chunk * P .. of the sorted tokens.  A token that began
// before the chunk leaves its sum at partials[2 chunk], one that goes on behind it at
// partials[2 chunk + 1] (at [2 chunk] if it does both).
constexpr int kAhead = 8;       // rows whose loads are in flight

template <typename T, typename O, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embed_sums_kernel(
    const int* __restrict__ keys, const int* __restrict__ ids, const O* __restrict__ dout,
    T* __restrict__ dtable, float* __restrict__ partials, int64_t n, int vocab, int cols, int64_t P,
    int tiles, float scale, bool accumulate) {
  constexpr int N = kVecElems<O>;
  const int64_t chunk = blockIdx.x / tiles;
  const Cols<N, WHOLE> at(static_cast<int64_t>(blockIdx.x % tiles) * kThreads + threadIdx.x, cols);
  if (!at.any) return;
  const int64_t begin = chunk * P, end = begin + P < n ? begin + P : n;
  int key = keys[begin];
  if (key == vocab) return;
  bool head = begin > 0 && keys[begin - 1] == key;
  float sum[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = 0.0f;
  for (int64_t i0 = begin; i0 < end; i0 += kAhead) {
    float v[kAhead][N];
    int next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k < end ? i0 + k : end - 1;
      next[k] = i + 1 < n ? keys[i + 1] : vocab;
      at.load(v[k], dout + static_cast<int64_t>(ids[i]) * cols);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= end) break;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += v[k][e];
      const bool last = i0 + k + 1 == end, goes_on = next[k] == key;
      if (goes_on && !last) continue;
      if (head || goes_on)
        at.store(partials + (2 * chunk + (head ? 0 : 1)) * cols, sum);
      else
        store_sum<T, N, WHOLE>(dtable + static_cast<int64_t>(key) * cols, at, sum, scale,
                               accumulate);
      head = false;
      key = next[k];
      if (key == vocab) return;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = 0.0f;
    }
  }
}

// A token that begins in this chunk and ends in a later one.
template <typename T, int N, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embed_join_kernel(
    const int* __restrict__ keys, T* __restrict__ dtable, const float* __restrict__ partials,
    int64_t n, int vocab, int cols, int64_t P, int tiles, float scale, bool accumulate) {
  const int64_t chunk = blockIdx.x / tiles, begin = chunk * P, end = begin + P;
  if (end >= n) return;
  const int key = keys[end - 1];
  if (key == vocab || keys[end] != key || (begin > 0 && keys[begin - 1] == key)) return;
  const Cols<N, WHOLE> at(static_cast<int64_t>(blockIdx.x % tiles) * kThreads + threadIdx.x, cols);
  if (!at.any) return;
  int64_t lo = end, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (keys[mid] <= key) lo = mid + 1;
    else hi = mid;
  }
  const int64_t last = (lo - 1) / P;
  float sum[N];
  at.load(sum, partials + (2 * chunk + 1) * cols);
  constexpr int U = 8;
  for (int64_t c0 = chunk + 1; c0 <= last; c0 += U) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
      at.load(v[u], partials + 2 * (c0 + u <= last ? c0 + u : last) * cols);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u > last) break;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += v[u][e];
    }
  }
  store_sum<T, N, WHOLE>(dtable + static_cast<int64_t>(key) * cols, at, sum, scale, accumulate);
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }

// Tokens a run: as few registers a lane as hold them in one run, else the most.
int run_registers(int64_t rows) { return rows <= kSortThreads ? 1 : rows <= 4 * kSortThreads ? 4 : 16; }
int64_t runs_of(int64_t rows) { return ceil_div(rows, kSortThreads * run_registers(rows)); }

// Positions a chunk: up to 512 chunks, so that the join of a token that is all of the batch adds
// up no more than that.
int64_t chunk_of(int64_t rows) {
  int64_t p = 4;
  while (512 * p < rows) p *= 2;
  return p;
}

struct Workspace {
  int64_t list, partials;       // bytes of a list of tokens or positions; of the partial sums
  int lists;                    // 2, or 4 where runs are merged
  Workspace(int64_t rows, int64_t cols) {
    list = (4 * rows + 15) / 16 * 16;
    lists = runs_of(rows) > 1 ? 4 : 2;
    partials = 2 * ceil_div(rows, chunk_of(rows)) * cols * 4;
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
  int tpr_log2 = 3;
  while (tpr_log2 < 8 && (int64_t{1} << tpr_log2) < vecs) ++tpr_log2;
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

template <int J> int launch_sort(const BwdArgs& a, int* keys, int* ids, int64_t zeros) {
  const int runs = a.rows > 0 ? static_cast<int>(runs_of(a.rows)) : 0;
  const int64_t fills = ceil_div(zeros, 16 * kSortThreads);
  const unsigned grid = static_cast<unsigned>(runs + (fills < 1024 ? fills : 1024));
  if (grid == 0) return ok();
  embed_sort_kernel<J><<<grid, kSortThreads, 0, a.s>>>(a.tokens, keys, ids, a.rows,
                                                       static_cast<int>(a.vocab), runs,
                                                       static_cast<char*>(a.dtable), zeros);
  MCKE_LAUNCH_CHECK("embed_sort_kernel");
  return ok();
}

template <typename T, typename O, bool WHOLE>
int launch_sums(const BwdArgs& a, const int* keys, const int* ids, float* partials) {
  constexpr int N = kVecElems<O>;
  const int64_t P = chunk_of(a.rows), chunks = ceil_div(a.rows, P);
  const int tiles = static_cast<int>(ceil_div(a.cols, int64_t{N} * kThreads));
  const int vocab = static_cast<int>(a.vocab), cols = static_cast<int>(a.cols);
  embed_sums_kernel<T, O, WHOLE><<<static_cast<unsigned>(chunks * tiles), kThreads, 0, a.s>>>(
      keys, ids, static_cast<const O*>(a.dout), static_cast<T*>(a.dtable), partials, a.rows, vocab,
      cols, P, tiles, a.scale, a.accumulate);
  MCKE_LAUNCH_CHECK("embed_sums_kernel");
  if (chunks == 1) return ok();
  embed_join_kernel<T, N, WHOLE>
      <<<static_cast<unsigned>((chunks - 1) * tiles), kThreads, 0, a.s>>>(
          keys, static_cast<T*>(a.dtable), partials, a.rows, vocab, cols, P, tiles, a.scale,
          a.accumulate);
  MCKE_LAUNCH_CHECK("embed_join_kernel");
  return ok();
}

template <typename T, typename O> int launch_bwd(const BwdArgs& a) {
  const Workspace w(a.rows, a.cols);
  int* keys = reinterpret_cast<int*>(a.ws);
  int* ids = reinterpret_cast<int*>(a.ws + w.list);
  const int64_t zeros =
      a.accumulate ? 0 : a.vocab * a.cols * static_cast<int64_t>(sizeof(T));
  const int J = run_registers(a.rows);
  if (int rc = J == 1   ? launch_sort<1>(a, keys, ids, zeros)
               : J == 4 ? launch_sort<4>(a, keys, ids, zeros)
                        : launch_sort<16>(a, keys, ids, zeros))
    return rc;
  if (a.rows == 0) return ok();
  for (int64_t len = int64_t{kSortThreads} * J, turn = 0; len < a.rows; len *= kMergeWays, ++turn) {
    int* to = reinterpret_cast<int*>(a.ws + (turn % 2 ? 0 : 2 * w.list));
    int* ids_to = reinterpret_cast<int*>(reinterpret_cast<char*>(to) + w.list);
    embed_merge_kernel<<<static_cast<unsigned>(ceil_div(a.rows, kThreads)), kThreads, 0, a.s>>>(
        keys, ids, to, ids_to, a.rows, len);
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
