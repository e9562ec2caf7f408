// token_logprobs.hip -- log probabilities of given tokens, the entropy and the most likely
// alternatives of each row of logits, and the gradient of the first two.
//
//   z = scale x,  lse = log sum exp z,  logprob = z[token] - lse
//   entropy = -sum p log p,  p = exp(z - lse)
//   alternatives: the top_k largest logits by (value, then lowest index), and their z - lse
//
//   d logprob / d z_j = [j == token] - p_j,   d entropy / d z_j = -p_j (log p_j + entropy)
//
// One pass over a row carries, per lane, the largest logit m, d = sum 2^u and
// e = sum u 2^u with u = (x - m) scale log2 e <= 0 (the online softmax with one more sum).
// Two states join at M = max(m1, m2) with delta = (m - M) scale log2 e:
//   d -> 2^delta d,   e -> 2^delta (e + delta d)
// and then lse = scale M + ln d,  entropy = ln d - ln2 e / d, so neither needs p itself.
// A masked logit (-inf) adds nothing to either; u and delta are held above -1e4, where 2^u is
// already 0, so that 0 times -inf does not arise.  All arithmetic is fp32.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "common.hpp"
#include "device_math.hpp"
#include "elem.hpp"

namespace mcke_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxTop = 64;             // a list lies across a wave, an entry to a lane
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1.0e4f;

// ---------------------------------------------------------------------------
// The sums
// ---------------------------------------------------------------------------
struct Sums {
  float m, d, e;
};

__device__ __forceinline__ Sums no_sums() { return {-INFINITY, 0.0f, 0.0f}; }

// What a state's exponents move by when the maximum becomes `to`.
__device__ __forceinline__ float shift_of(float m, float to, float c) {
  return m == to ? 0.0f : fmaxf((m - to) * c, kFar);
}

__device__ __forceinline__ Sums moved(Sums s, float to, float c) {
  const float t = shift_of(s.m, to, c), f = __builtin_amdgcn_exp2f(t);
  return {to, f * s.d, f * (s.e + t * s.d)};
}

__device__ __forceinline__ float first_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// The states of a wave's lanes, or of the workgroup's waves, as one: each moved to the largest
// m, then added up in a fixed order.  A lane's own product and its neighbour's go into one
// multiply-add, which rounds the one and not the other: the lanes' sums differ in their last bit,
// and every lane takes the first one's.
__device__ __forceinline__ Sums wave_join(Sums s, float c) {
  s = moved(s, wave_max(s.m), c);
  return {s.m, first_lane(wave_sum(s.d)), first_lane(wave_sum(s.e))};
}
__device__ __forceinline__ Sums block_join(const Sums (&waves)[kWaves], float c) {
  float m = waves[0].m;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, waves[w].m);
  Sums s{m, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Sums q = moved(waves[w], m, c);
    s.d += q.d;
    s.e += q.e;
  }
  return s;
}

// Takes in N values whose largest is m, at one fused multiply-add an exponent: with r = from c
// rounded and lo = from c - r (exact, by another one), the exponents are v c - r - lo, and what
// all of them have in common comes out of the sums as 2^-lo:
//   sum 2^u = 2^-lo d,  sum u 2^u = 2^-lo (e - lo d)   with  d = sum 2^(v c - r), e = sum (v c - r) 2^(v c - r)
// The multiply-add rounds once, at the size of its result, so large logits lose nothing to the
// product.  lo stays below 32 as |r| is held to 2^30 with a smaller c: past that two logits that
// differ are 64 apart in the exponent either way, and the smaller one's 2^u is nothing.
// (Difference, then product: 4096 x 32768 bf16 with the top 20 55.0 us, this 52.8.)
template <int N, bool ENTROPY>
__device__ __forceinline__ void add_values(Sums& s, const float (&v)[N], float m, float c) {
  constexpr float kMost = 1073741824.0f;
  const float to = fmaxf(s.m, m);
  s = moved(s, to, c);
  const float from = to == -INFINITY ? 0.0f : to;
  const float cc = fabsf(from * c) > kMost ? kMost / fabsf(from) : c;
  const float r = from * cc, lo = __builtin_fmaf(from, cc, -r);
  float d = 0.0f, e = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float u = __builtin_fmaf(v[i], cc, -r);
    const float p = __builtin_amdgcn_exp2f(u);
    d += p;
    if constexpr (ENTROPY) e += p * fmaxf(u, kFar);
  }
  const float f = __builtin_amdgcn_exp2f(-lo);
  s.d += f * d;
  if constexpr (ENTROPY) s.e += f * (e - lo * d);
}

// ---------------------------------------------------------------------------
// The alternatives
// ---------------------------------------------------------------------------
// A value's bits in an order that whole numbers have too; -0 counts as +0.  Above 0 for every
// value.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Value and index as one number that orders by value, then by lowest index.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  return static_cast<uint64_t>(order_of(v)) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) {
  return 0xFFFFFFFFu - static_cast<uint32_t>(k);
}

// A value that at least k of the workgroup's logits reach, and few more: the k-th largest of the
// largest of each quad of lanes, up to kQuadTop, else of each lane (20 of 64 quads: some 24 of
// normally distributed logits reach it).  A value's rank is how many are larger, counted from
// LDS, and the bound is the least of those that rank below k.  (Bisecting the values' bits with
// ballots took 2770 cycles for 256 of them: each count passes through a scalar register.)
// Every lane calls it, with m its largest logit and not a NaN; `lds` holds kThreads floats, and
// `mins` kWaves.  -inf, which every logit reaches, where k of them have no logits.
constexpr int kQuadTop = 24;

template <int N>
__device__ __forceinline__ int count_larger(const float* lds, float v) {
  int n = 0;
#pragma unroll 8
  for (int i = 0; i < N; i += 4) {
    const f32x4 o = *reinterpret_cast<const f32x4*>(lds + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) n += o[e] > v;
  }
  return n;
}

// The first half, before a barrier of the workgroup.
__device__ __forceinline__ void put_largest(float m, int k, float* lds) {
  if (k > kQuadTop) {
    lds[threadIdx.x] = m;
  } else {
    m = wave_max<4>(m);
    if (threadIdx.x % 4 == 0) lds[threadIdx.x / 4] = m;
  }
}

// The second, behind it.
__device__ __forceinline__ float bound_of(float m, int k, const float* lds, float* mins) {
  const int lane = threadIdx.x % kWave;
  if (k <= kQuadTop) {                                   // every wave for itself
    const float v = lds[lane];
    return -wave_max(count_larger<kThreads / 4>(lds, v) < k ? -v : -INFINITY);
  }
  const float least = -wave_max(count_larger<kThreads>(lds, m) < k ? -m : -INFINITY);
  if (lane == 0) mins[threadIdx.x / kWave] = least;
  __syncthreads();
  float all = mins[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = fminf(all, mins[w]);
  return all;
}

// A wave's list: lane i holds the i-th best so far.  Elements come in the order of their
// indices, so one that equals the worst of a full list loses to it.  A NaN is never taken.
struct TopList {
  float v;          // lane's entry
  uint32_t i;
  int count, k;     // uniform
  float least;      // uniform: what a new element has to reach

  __device__ __forceinline__ void start(int top_k) {
    v = 0.0f;
    i = 0;
    count = 0;
    k = top_k;
    least = -INFINITY;
  }
  __device__ __forceinline__ void insert(float x, uint32_t index) {
    const int lane = threadIdx.x % kWave;
    const int at = __popcll(__ballot(lane < count && v >= x));
    const float pv = __shfl_up(v, 1, 64);
    const uint32_t pi = __shfl_up(i, 1, 64);
    if (lane > at) {
      v = pv;
      i = pi;
    } else if (lane == at) {
      v = x;
      i = index;
    }
    if (count < k) ++count;
    if (count == k) {
      // The next larger float: past +inf a NaN, which nothing reaches.
      const float worst =
          __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), k - 1));
      const int b = __builtin_bit_cast(int, worst + 0.0f);
      least = __builtin_bit_cast(float, b >= 0 ? b + 1 : b - 1);
    }
  }
  // The lanes' values x[0 ..], lane l's first one at index first + VE * l, m the lane's largest.
  template <int VE>
  __device__ __forceinline__ void offer(const float (&x)[VE], float m, uint32_t first) {
    uint64_t hot = __ballot(m >= least);
    while (hot) {
      const int l = __ffsll(static_cast<unsigned long long>(hot)) - 1;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float y =
            __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x[e]), l));
        if (y >= least) insert(y, first + static_cast<uint32_t>(VE * l + e));
      }
      hot &= hot - 1;
      hot &= __ballot(m >= least);
    }
  }
};

// The keys a workgroup has put down, in an order that does not matter to what comes of them.
constexpr int kMaxKeys = 1024;
struct KeyList {
  uint64_t keys[kMaxKeys];
  int count;               // past kMaxKeys only counted

  // Before the first key and a barrier: what rank_keys reads past the end of a short list is 0.
  __device__ __forceinline__ void clear() {
    if (threadIdx.x < kWave + 16) keys[threadIdx.x] = 0;
    if (threadIdx.x == 0) count = 0;
  }
  __device__ __forceinline__ void put(uint64_t key) {
    const int at = atomicAdd(&count, 1);
    if (at < kMaxKeys) keys[at] = key;
  }
};

// Calls out(i, key) for the top_k largest of n keys, all different, in their order, each from some
// lane, and with key 0 for what is left of top_k.
template <class F>
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int top_k, F out) {
  if (n <= kWave) {                                      // a key to a lane of the first wave
    if (threadIdx.x >= kWave) return;
    const int i = threadIdx.x;
    const uint64_t mine = keys[i];
    int rank = 0;
    for (int j = 0; j < n; j += 16) {
#pragma unroll
      for (int e = 0; e < 16; ++e) rank += keys[j + e] > mine;
    }
    if (i >= n) rank = i;
    if (rank < top_k) out(rank, mine);
    return;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = keys[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += keys[j] > mine;
    if (rank < top_k) out(rank, mine);
  }
}

// ---------------------------------------------------------------------------
// Kernels
// ---------------------------------------------------------------------------
struct RowOut {
  const int64_t* tokens;
  float *logprobs, *entropy, *lse, *top_logprobs;
  int64_t* top_ids;
};

// A row's results from its sums, its n keys and its token's logit.
__device__ __forceinline__ void write_row(const RowOut& o, int64_t r, int64_t vocab, int64_t token,
                                          float logit, Sums s, const uint64_t* keys, int n,
                                          int top_k, float scale) {
  const float ln_d = logf(s.d);
  const bool empty = s.m == -INFINITY && s.d == 0.0f;   // every logit is masked
  if (threadIdx.x == kThreads - 1) {                    // the first wave ranks meanwhile
    if (o.logprobs) {
      float lp = __builtin_nanf("");                    // no such token
      if (token < vocab) lp = empty ? -INFINITY : (logit - s.m) * scale - ln_d;
      o.logprobs[r] = lp;
    }
    if (o.entropy) o.entropy[r] = empty ? 0.0f : ln_d - kLn2 * (s.e / s.d);
    if (o.lse) o.lse[r] = empty ? -INFINITY : s.m * scale + ln_d;
  }
  if (top_k == 0) return;
  rank_keys(keys, n, top_k, [&](int i, uint64_t k) {
    const float v = empty ? -INFINITY : (key_value(k) - s.m) * scale - ln_d;
    if (o.top_logprobs) o.top_logprobs[r * top_k + i] = k ? v : __builtin_nanf("");
    if (o.top_ids) o.top_ids[r * top_k + i] = k ? static_cast<int64_t>(key_index(k)) : -1;
  });
}

__device__ __forceinline__ void write_no_row(const RowOut& o, int64_t r, int top_k) {
  if (threadIdx.x == 0) {
    if (o.logprobs) o.logprobs[r] = 0.0f;
    if (o.entropy) o.entropy[r] = 0.0f;
    if (o.lse) o.lse[r] = 0.0f;
  }
  for (int i = threadIdx.x; i < top_k; i += kThreads) {
    if (o.top_logprobs) o.top_logprobs[r * top_k + i] = 0.0f;
    if (o.top_ids) o.top_ids[r * top_k + i] = -1;
  }
}

// The row's token (0 where there are none) and its logit.
template <typename T>
__device__ __forceinline__ float token_logit(const RowOut& o, const T* row, int64_t vocab,
                                             int64_t token) {
  return o.logprobs && token >= 0 && token < vocab ? static_cast<float>(row[token]) : 0.0f;
}

// A part of a row as it lies in the workspace.
struct Part {
  float m, d, e, unused;
};

template <typename T>
__device__ __forceinline__ VecT16<T> load_logits(const T* row, int64_t j, int64_t vocab) {
  constexpr int VE = kVecElems<T>;
  if ((j + 1) * VE <= vocab) return load_vec<T>(row + j * VE);
  return load_part<T>(row + j * VE, static_cast<int>(vocab - j * VE), -INFINITY);
}

typedef uint32_t u32x4_of __attribute__((ext_vector_type(4)));

// A wave's consecutive 16-bit vectors from loads that began an element early, at 4-byte
// addresses: each dword is two halves of neighbours, the last one's second half the next lane's
// first dword, or `after` for lane 63.
template <typename T>
__device__ __forceinline__ VecT16<T> shifted(VecT16<T> w, uint32_t after) {
  constexpr int kWaveShl1 = 0x130;                        // a lane reads the one above it
  const u32x4_of d = __builtin_bit_cast(u32x4_of, w);
  const uint32_t next = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
      static_cast<int>(after), static_cast<int>(d[0]), kWaveShl1, 0xF, 0xF, false));
  const u32x4_of o = {__builtin_amdgcn_alignbit(d[1], d[0], 16),
                      __builtin_amdgcn_alignbit(d[2], d[1], 16),
                      __builtin_amdgcn_alignbit(d[3], d[2], 16),
                      __builtin_amdgcn_alignbit(next, d[3], 16)};
  return __builtin_bit_cast(VecT16<T>, o);
}

// The alternatives of vectors first .. end - 1 of a row, in any order and with any ties: a list
// per wave, elements in the order of their indices.  Returns how many keys the waves put down;
// every lane of the workgroup calls it, and a barrier follows.
template <typename T>
__device__ __noinline__ int list_keys(const T* row, int64_t first, int64_t end, int64_t vocab,
                                      int top_k, KeyList* list, int* counts) {
  constexpr int VE = kVecElems<T>;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  TopList top;
  top.start(top_k);
  for (int64_t j0 = first + wave * kWave; j0 < end; j0 += kThreads) {
    const int64_t j = j0 + lane;
    float v[VE], m = __builtin_nanf("");
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = m;              // past the end nothing is offered
    if (j < end) {
      const VecT16<T> w = load_logits<T>(row, j, vocab);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (j * VE + e < vocab) v[e] = static_cast<float>(w[e]);
#pragma unroll
      for (int e = 0; e < VE; ++e) m = fmaxf(m, v[e]);
    }
    top.offer<VE>(v, m, static_cast<uint32_t>(j0 * VE));
  }
  if (lane == 0) counts[wave] = top.count;
  if (threadIdx.x < kWave + 16) list->keys[threadIdx.x] = 0;
  __syncthreads();
  int before = 0, n = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += counts[w];
    n += counts[w];
  }
  if (lane < top.count) list->keys[before + lane] = key_of(top.v, top.i);
  return n;
}

// Logit i of a dword of T.
template <typename T> __device__ __forceinline__ float value_of(uint32_t d, int i) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, d);
  else
    return static_cast<float>(
        __builtin_bit_cast(T, static_cast<uint16_t>(i ? d >> 16 : d & 0xFFFFu)));
}

// Puts down the logits of a lane's vectors j, j + kThreads, ... that reach `least`.  Which do is a
// bit each of one number, whose few bits a loop picks out.
template <typename T, int N>
__device__ __forceinline__ void put_keys(const VecT16<T> (&w)[N], int64_t j, int64_t end,
                                         int64_t vocab, float least, KeyList& list) {
  constexpr int VE = kVecElems<T>, PER = VE / 4;         // logits of a dword
  static_assert(N * VE <= 32, "a bit each");
  uint32_t hit = 0;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int e = 0; e < VE; ++e)
      hit |= static_cast<float>(w[u][e]) >= least ? 1u << (u * VE + e) : 0u;   // never a NaN
  while (hit) {
    const int k = __ffs(hit) - 1;
    hit &= hit - 1;
    const int64_t ju = j + k / VE * kThreads, index = ju * VE + k % VE;
    if (ju >= end || index >= vocab) continue;
    uint32_t d = 0;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        d = k / PER == 4 * u + i ? __builtin_bit_cast(u32x4_of, w[u])[i] : d;
    list.put(key_of(value_of<T>(d, k % PER), static_cast<uint32_t>(index)));
  }
}

// Workgroup (row, part): vectors part * per_part on, in rounds of U vectors a lane, each
// round's loads a round ahead of its work.  With one part the row's results are written here,
// else its sums and keys go to the workspace.
//
// Alternatives cost the pass next to nothing per logit: a lane has the largest of its own logits in
// its sums, and keeps it for each quarter of its rounds.  The top_k-th largest of the lanes' is
// a bound that at least top_k logits reach and few others do; only quarters whose largest
// reaches it have any, so those are read again (from the caches) and the logits that reach the
// bound are put down and ranked.  Where more than kMaxKeys reach it (ties, masks, sorted rows)
// list_keys does it instead.
constexpr int kUnroll = 4, kQuarters = 4;
template <typename T, int U, bool ENTROPY>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ x, RowOut o,
                                                            Part* __restrict__ parts_out,
                                                            uint64_t* __restrict__ keys_out,
                                                            int64_t vocab, int64_t row_stride,
                                                            int parts, int64_t per_part,
                                                            float scale, int top_k) {
  constexpr int VE = kVecElems<T>, kRound = U * kThreads;
  __shared__ KeyList list;
  __shared__ __attribute__((aligned(16))) float largest[kThreads];
  __shared__ float mins[kWaves];
  __shared__ Sums waves[kWaves];
  __shared__ int hot[kQuarters * kThreads], hot_count, wave_counts[kWaves];
  const int64_t r = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x % parts);
  const T* row = x + r * row_stride;
  const float c = scale * kLog2e;
  const int t = threadIdx.x, lane = t % kWave, wave = t / kWave;
  const int64_t all = (vocab + VE - 1) / VE, first = part * per_part;
  const int64_t end = first + per_part < all ? first + per_part : all;
  const int n_vecs = static_cast<int>(end > first ? end - first : 0);
  const int rounds = (n_vecs + kRound - 1) / kRound;
  const int quarter = (rounds + kQuarters - 1) / kQuarters;        // rounds of one

  // 16-bit rows off 4-byte addresses: vectors at 2-byte addresses take the load units twice, so they
  // are read an element early and shifted into place, the same lanes' the same bits (bf16, data
  // past the caches: 4096 x 50257 83.5 -> 74.2 us beside 71.3 for 50256, 2048 x 131071 104 -> 89.2).
  // What lies before the row is not its own and is not read: the row's first vector is loaded from
  // its second element on, and the first one by itself.
  const bool odd = sizeof(T) == 2 && reinterpret_cast<uintptr_t>(row) / 2 % 2 == 1;
  const T* from = odd ? row - 1 : row;
  // Rounds that lie in the row, in an odd one with an element behind them.
  const int64_t whole = (vocab - (odd ? 1 : 0)) / VE - first;
  const int full = static_cast<int>(whole < n_vecs ? whole : n_vecs) / kRound;

  // Round i: vectors first + i * kRound + u * kThreads + t, and the dword behind each of the wave's
  // U runs of them, in its last U lanes.
  auto load = [&](int i, VecT16<T> (&w)[U], [[maybe_unused]] uint32_t& after) {
    const int64_t j = first + static_cast<int64_t>(i) * kRound + t;
    if (i < full) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        w[u] = load_stream<T>(from + (j + u * kThreads) * VE + (u == 0 && odd && j == 0 ? 2 : 0));
      if constexpr (sizeof(T) == 2) {
        if (odd && lane >= kWave - U) {
          const int64_t behind = j - lane + kWave + (lane - (kWave - U)) * kThreads;
          after = *reinterpret_cast<const uint32_t*>(from + behind * VE);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        w[u] = j + u * kThreads < end ? load_logits<T>(row, j + u * kThreads, vocab)
                                      : load_part<T>(row, 0, -INFINITY);
    }
  };
  // Before any load of the row: without a token it is not read.  (Behind the first ones no faster:
  // 4 x 131072 bf16 9.75 us and 9.87, with the top 20; half the rows without a token, 2048 x 131072
  // 61.8 and 60.2.)
  const int64_t token = o.tokens ? o.tokens[r] : 0;
  if (token < 0) {
    if (parts == 1) write_no_row(o, r, top_k);
    return;
  }
  VecT16<T> w[U];
  uint32_t after = 0;
  load(0, w, after);
  const float logit = token_logit<T>(o, row, vocab, token);
  Sums s = no_sums();
  float quarter_m[kQuarters];
#pragma unroll
  for (int q = 0; q < kQuarters; ++q) {
    quarter_m[q] = -INFINITY;
    const int stop = (q + 1) * quarter < rounds ? (q + 1) * quarter : rounds;
    for (int i = q * quarter; i < stop; ++i) {
      VecT16<T> n[U];
      uint32_t after_n = 0;
      // Before the next loads are out: behind them it takes 98 registers for 82.
      if constexpr (sizeof(T) == 2) {
        if (odd && i < full) {
          if (i == 0 && first + t == 0) {
            const u32x4_of d = __builtin_bit_cast(u32x4_of, w[0]);
            const uint32_t d0 = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row)) << 16;
            w[0] = __builtin_bit_cast(VecT16<T>, u32x4_of{d0, d[0], d[1], d[2]});
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            w[u] = shifted<T>(w[u], __builtin_amdgcn_readlane(after, kWave - U + u));
        }
      }
      if (i + 1 < rounds) load(i + 1, n, after_n);
      float v[U * VE];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VE; ++e) v[u * VE + e] = static_cast<float>(w[u][e]);
      float m = v[0];
#pragma unroll
      for (int e = 1; e < U * VE; ++e) m = fmaxf(m, v[e]);
      quarter_m[q] = fmaxf(quarter_m[q], m);
      add_values<U * VE, ENTROPY>(s, v, m, c);
      if (i + 1 < rounds) {
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = n[u];
        after = after_n;
      }
    }
  }

  if (t == 0) hot_count = 0;
  list.clear();
  const float mine = s.m;
  if (top_k > 0) put_largest(mine, top_k, largest);
  s = wave_join(s, c);
  if (lane == 0) waves[wave] = s;
  __syncthreads();
  s = block_join(waves, c);

  int n_keys = 0;
  if (top_k > 0) {
    const float least = bound_of(mine, top_k, largest, mins);
    if (rounds <= 1) {                                  // the lane still has its vectors
      if (mine >= least) put_keys<T, U>(w, first + t, end, vocab, least, list);
    } else {
      const int per_hot = quarter * U;                  // vectors of a lane's quarter
#pragma unroll
      for (int q = 0; q < kQuarters; ++q)
        if (quarter_m[q] >= least && q * quarter < rounds)
          hot[atomicAdd(&hot_count, 1)] = q * per_hot * kThreads + t;
      __syncthreads();
      const int items = hot_count * per_hot;
      for (int i = t; i < items; i += kThreads) {
        const int h = i / per_hot;
        const int64_t j = first + hot[h] + static_cast<int64_t>(i - h * per_hot) * kThreads;
        if (j >= end) continue;
        const VecT16<T> one[1] = {load_logits<T>(row, j, vocab)};
        put_keys<T, 1>(one, j, end, vocab, least, list);
      }
    }
    __syncthreads();
    n_keys = list.count;
    if (n_keys > kMaxKeys) {
      __syncthreads();                                  // everybody has read the count
      n_keys = list_keys<T>(row, first, end, vocab, top_k, &list, wave_counts);
      __syncthreads();
    }
  }
  if (parts == 1) {
    write_row(o, r, vocab, token, logit, s, list.keys, n_keys, top_k, scale);
    return;
  }
  if (t == kThreads - 1) parts_out[blockIdx.x] = Part{s.m, s.d, s.e, 0.0f};
  if (top_k > 0)
    rank_keys(list.keys, n_keys, top_k, [&](int i, uint64_t k) {
      keys_out[static_cast<int64_t>(blockIdx.x) * top_k + i] = k;
    });
}

// A row's parts joined, a workgroup per row.  Keys: the top_k-th largest of the lanes' largest is
// a bound again, and those that reach it are ranked.
constexpr int kMaxParts = 64, kKeysPerLane = kMaxKeys / kThreads;
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(
    const T* __restrict__ x, RowOut o, const Part* __restrict__ parts_in,
    const uint64_t* __restrict__ keys_in, int64_t vocab, int64_t row_stride, int parts,
    float scale, int top_k) {
  __shared__ KeyList list;
  __shared__ __attribute__((aligned(16))) float largest[kThreads];
  __shared__ float mins[kWaves];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t % kWave;
  const int n = parts * top_k;
  uint64_t key[kKeysPerLane];
#pragma unroll
  for (int i = 0; i < kKeysPerLane; ++i)
    key[i] = t + i * kThreads < n ? keys_in[r * n + t + i * kThreads] : 0;
  Sums s = no_sums();
  if (lane < parts) {
    const Part q = parts_in[r * parts + lane];
    s = Sums{q.m, q.d, q.e};
  }
  const int64_t token = o.tokens ? o.tokens[r] : 0;
  if (token < 0) {
    write_no_row(o, r, top_k);
    return;
  }
  const float logit = token_logit<T>(o, x + r * row_stride, vocab, token);
  if (top_k > 0) {
    list.clear();
    uint64_t most = key[0];
#pragma unroll
    for (int i = 1; i < kKeysPerLane; ++i) most = key[i] > most ? key[i] : most;
    const float m = most ? key_value(most) : -INFINITY;
    put_largest(m, top_k, largest);
    __syncthreads();
    const float least = bound_of(m, top_k, largest, mins);
#pragma unroll
    for (int i = 0; i < kKeysPerLane; ++i)
      if (key[i] && key_value(key[i]) >= least) list.put(key[i]);
    __syncthreads();
  }
  const float c = scale * kLog2e;
  write_row(o, r, vocab, token, logit, wave_join(s, c), list.keys, top_k > 0 ? list.count : 0, top_k,
            scale);
}

// dlogits = scale (g ([j == token] - p_j) - h p_j (log p_j + entropy)), g and h the gradients
// of the row's logprob and entropy: a workgroup per kBackVecs * kThreads vectors of a row, a lane's
// loads all out before the row's own values but its token are looked at.  A row without a token is
// not read (2048 x 131072 bf16: half the rows without one 169 -> 130 us, none 84.6 -> 86.5 at 1024
// rows, with the loads behind the token).
constexpr int kBackVecs = 2;
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_backward_kernel(
    const T* __restrict__ x, const int64_t* __restrict__ tokens, const float* __restrict__ lse_in,
    const float* __restrict__ entropy, const float* __restrict__ dlogprobs,
    const float* __restrict__ dentropy, T* __restrict__ dx, int64_t vocab, int64_t row_stride,
    int per_row, float scale) {
  constexpr int VE = kVecElems<T>, V = kBackVecs;
  const int64_t r = blockIdx.x / per_row;
  const int64_t at0 =
      (static_cast<int64_t>(blockIdx.x % per_row) * (V * kThreads) + threadIdx.x) * VE;
  const T* in = x + r * row_stride;
  T* out = dx + r * row_stride;
  const int64_t token = tokens ? tokens[r] : 0;
  VecT16<T> w[V];
  if (token >= 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t at = at0 + i * (kThreads * VE);
      if (at + VE <= vocab) w[i] = load_stream<T>(in + at);
      else if (at < vocab) w[i] = load_part<T>(in + at, static_cast<int>(vocab - at), 0.0f);
    }
  }
  const float lse = lse_in[r];
  // No token or no probability: no gradient.  No such token: a NaN, as forward.
  const bool none = token < 0 || lse == -INFINITY || token >= vocab;
  const float instead = token < vocab ? 0.0f : __builtin_nanf("");
  const float g = dlogprobs ? scale * dlogprobs[r] : 0.0f;
  const float h = dentropy ? scale * dentropy[r] : 0.0f;
  const float a = dentropy ? -(g + h * entropy[r]) : -g;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int64_t at = at0 + i * (kThreads * VE);
    if (at >= vocab) break;
    VecT16<T> y;
    if (none) {
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] = static_cast<T>(instead);
    } else {
      float d[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float lp = static_cast<float>(w[i][e]) * scale - lse;
        d[e] = __builtin_amdgcn_exp2f(lp * kLog2e) * (a - h * fmaxf(lp, kFar));
      }
      if (dlogprobs && token >= at && token < at + VE) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (at + e == token) d[e] += g;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] = static_cast<T>(d[e]);
    }
    if (at + VE <= vocab) store_stream<T>(out + at, y);
    else store_part<T>(out + at, y, static_cast<int>(vocab - at));
  }
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------
// How many workgroups share a row: one where that is sooner done than the second launch, else as
// many as fill the GPU, at least 2048 logits each, and no more keys than the joining workgroup
// holds.  One workgroup's time goes by the row's bytes; what sharing costs grows with the rows, whose
// workgroups fill the GPU anyway, and with alternatives, which every part ranks (above kQuadTop by a
// longer count).  Up to 32768 logits of any type a row stays whole.  One workgroup and shared, us:
//                     no alternatives              top 20                       top 64
//   16 x 32768   bf16   6.1   6.7                    8.5  10.1                   11.8  17.3
//   16 x 50264          8.0   7.3                   10.8  10.0                   15.3  17.9
//   64 x 50264          8.2   7.6                   11.1  12.9                   15.8  22.1
//   64 x 100000        12.4   9.4                   16.4  15.6                   22.1  24.7
//   128 x 65536         9.1   9.6                   12.1  15.7                   16.7  23.2
//   128 x 131072       14.6  12.1                   18.8  18.2                   24.6  26.3
//   250 x 131072       15.6  17.0                   19.9  23.1                   26.0  30.6
//   250 x 262144       27.4  27.2                   33.1  33.0                   42.9  43.4
//   64 x 32768   fp32   8.0   7.4                   10.7  12.1                   15.3  21.0
//   64 x 65536         13.0   8.3                   17.0  13.7                   22.4  22.6
//   128 x 32768         8.3   8.4                   11.2  13.7                   15.7  20.9
//   128 x 65536        13.4  10.8                   17.4  16.4                   22.9  24.5
//   250 x 65536        14.8  15.2                   18.7  21.0                   24.6  27.9
//   256 x 262144       48.2  44.0                   57.1  53.5                   72.8  66.8
//   400 x 262144       60.3  71.5                   71.1  85.4                   92.5 104.5
int64_t whole_row_bytes(int64_t rows, int top_k) {
  return 1000 * (72 + rows * rows / 160 + (top_k == 0 ? 0 : rows < 80 ? rows : 80) +
                 (top_k > kQuadTop ? 80 : 0));
}
int parts_of(int64_t rows, int64_t vocab, int top_k, int64_t elem_bytes) {
  if (rows > 256 || vocab <= 32768 || vocab * elem_bytes <= whole_row_bytes(rows, top_k)) return 1;
  int64_t p = 1024 / (rows > 0 ? rows : 1);
  const int64_t most = (vocab + 2047) / 2048;
  if (p > most) p = most;
  if (p > kMaxParts) p = kMaxParts;
  if (top_k > 0 && p > kMaxKeys / top_k) p = kMaxKeys / top_k;
  return p < 1 ? 1 : static_cast<int>(p);
}
size_t workspace_of(int64_t rows, int top_k, int parts) {
  if (parts == 1) return 0;
  return static_cast<size_t>(rows) * parts * (sizeof(Part) + sizeof(uint64_t) * top_k);
}

struct RowArgs {
  const void* logits;
  RowOut o;
  int64_t rows, vocab, row_stride;
  float scale;
  int top_k;
  void* ws;
  hipStream_t s;
};

template <typename T, int U> auto* logprobs_kernel_for(bool entropy) {
  return entropy ? &logprobs_kernel<T, U, true> : &logprobs_kernel<T, U, false>;
}

template <typename T> int logprobs(const RowArgs& a) {
  const int parts = parts_of(a.rows, a.vocab, a.top_k, sizeof(T));
  const int64_t vecs = (a.vocab + kVecElems<T> - 1) / kVecElems<T>;
  const int64_t per_part = (vecs + parts - 1) / parts;
  const T* x = static_cast<const T*>(a.logits);
  Part* sums = static_cast<Part*>(a.ws);
  uint64_t* keys = reinterpret_cast<uint64_t*>(sums + (parts > 1 ? a.rows * parts : 0));
  const unsigned grid = static_cast<unsigned>(a.rows * parts);
  // A short row takes as few vectors a lane as hold it: 4096 x 1000 bf16 10.2 us, with four 15.8.
  auto* fn = logprobs_kernel_for<T, kUnroll>(a.o.entropy);
  if (per_part <= kThreads) fn = logprobs_kernel_for<T, 1>(a.o.entropy);
  else if (per_part <= 2 * kThreads) fn = logprobs_kernel_for<T, 2>(a.o.entropy);
  fn<<<grid, kThreads, 0, a.s>>>(x, a.o, sums, keys, a.vocab, a.row_stride, parts, per_part,
                                 a.scale, a.top_k);
  MCKE_LAUNCH_CHECK("logprobs_kernel");
  if (parts > 1) {
    logprobs_join_kernel<T><<<static_cast<unsigned>(a.rows), kThreads, 0, a.s>>>(
        x, a.o, sums, keys, a.vocab, a.row_stride, parts, a.scale, a.top_k);
    MCKE_LAUNCH_CHECK("logprobs_join_kernel");
  }
  return ok();
}

int check_logits(const char* who, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                 float scale) {
  auto no = [&](const std::string& what) { return invalid(std::string(who) + ": " + what); };
  if (!is_dtype(dtype)) return no("unknown dtype " + std::to_string(dtype));
  if (rows < 0 || vocab < 0) return no("negative extent");
  if (vocab > 2147483647LL) return no("vocab exceeds INT32_MAX");
  if (row_stride < vocab) return no("row_stride is less than vocab");
  if (rows > 0 && row_stride > INT64_MAX / 16 / rows) return no("extent too large");
  if (!(scale > 0.0f) || std::isinf(scale * kLog2e))
    return no("scale must be finite and above zero");
  return ok();
}

// Bytes from the first logit to behind the last.
uint64_t logits_bytes(int dtype, int64_t rows, int64_t vocab, int64_t row_stride) {
  return dtype_bytes(dtype) * (static_cast<uint64_t>(rows - 1) * row_stride + vocab);
}

}  // namespace
}  // namespace mcke_amd

using namespace mcke_amd;

extern "C" {

size_t mcke_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top_k) {
  if (rows <= 0 || vocab <= 0 || vocab > 2147483647LL || top_k < 0 || top_k > kMaxTop) return 0;
  // The most that any type needs: where 16-bit rows are shared, those of fp32 are, by as many.
  return workspace_of(rows, top_k, parts_of(rows, vocab, top_k, 4));
}

int mcke_launch_token_logprobs(const void* logits, const int64_t* tokens, float* logprobs_out,
                               float* entropy, float* lse, float* top_logprobs, int64_t* top_ids,
                               int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                               float scale, int top_k, void* workspace, size_t workspace_bytes,
                               void* stream) {
  const char* who = "launch_token_logprobs";
  if (int rc = check_logits(who, dtype, rows, vocab, row_stride, scale)) return rc;
  if (top_k < 0 || top_k > kMaxTop || top_k > vocab)
    return invalid("launch_token_logprobs: top_k must be between 0 and 64 and at most vocab");
  if (rows == 0 || vocab == 0) return ok();
  if (!logits) return invalid("launch_token_logprobs: null pointer");
  if (logprobs_out && !tokens)
    return invalid("launch_token_logprobs: log probabilities need tokens");
  if (top_k > 0 && !top_logprobs && !top_ids)
    return invalid("launch_token_logprobs: top_k without an output for the alternatives");
  if (!logprobs_out && !entropy && !lse && top_k == 0)
    return invalid("launch_token_logprobs: no output is asked for");
  if (!aligned(logits, dtype_bytes(dtype)) || !aligned(tokens, 8) || !aligned(logprobs_out, 4) ||
      !aligned(entropy, 4) || !aligned(lse, 4) || !aligned(top_logprobs, 4) || !aligned(top_ids, 8))
    return invalid("launch_token_logprobs: a pointer is not aligned to its type");
  const int parts = parts_of(rows, vocab, top_k, static_cast<int64_t>(dtype_bytes(dtype)));
  if (rows * parts > int64_t{UINT32_MAX} / kThreads)
    return invalid("launch_token_logprobs: rows exceed the grid's 32-bit work size");
  const size_t need = workspace_of(rows, top_k, parts);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return invalid("launch_token_logprobs: these rows need a 16-byte aligned workspace of " +
                   std::to_string(need) + " bytes, got " +
                   std::to_string(workspace ? workspace_bytes : 0));
  const uint64_t in = logits_bytes(dtype, rows, vocab, row_stride), n = rows, k = top_k;
  if (top_k == 0) top_logprobs = nullptr, top_ids = nullptr;
  const void* outs[] = {logprobs_out, entropy, lse, top_logprobs, top_ids,
                        need > 0 ? workspace : nullptr};
  const uint64_t out_bytes[] = {4 * n, 4 * n, 4 * n, 4 * n * k, 8 * n * k, need};
  for (int i = 0; i < 6; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], logits, in) ||
               overlap(outs[i], out_bytes[i], tokens, 8 * n);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid("launch_token_logprobs: an output or the workspace overlaps another operand, "
                     "which violates the __restrict__ contract");
  }
  const RowArgs a{logits, RowOut{tokens, logprobs_out, entropy, lse, top_logprobs, top_ids},
                 rows, vocab, row_stride, scale, top_k, workspace,
                 static_cast<hipStream_t>(stream)};
  if (dtype == MCKE_DTYPE_F32) return logprobs<float>(a);
  if (dtype == MCKE_DTYPE_F16) return logprobs<_Float16>(a);
  return logprobs<__bf16>(a);
}

int mcke_launch_token_logprobs_backward(const void* logits, const int64_t* tokens,
                                        const float* lse, const float* entropy,
                                        const float* dlogprobs, const float* dentropy,
                                        void* dlogits, int dtype, int64_t rows, int64_t vocab,
                                        int64_t row_stride, float scale, void* stream) {
  const char* who = "launch_token_logprobs_backward";
  if (int rc = check_logits(who, dtype, rows, vocab, row_stride, scale)) return rc;
  if (rows == 0 || vocab == 0) return ok();
  if (!logits || !lse || !dlogits)
    return invalid("launch_token_logprobs_backward: null pointer");
  if (!dlogprobs && !dentropy)
    return invalid("launch_token_logprobs_backward: no gradient is given");
  if (dlogprobs && !tokens)
    return invalid("launch_token_logprobs_backward: dlogprobs need tokens");
  if (dentropy && !entropy)
    return invalid("launch_token_logprobs_backward: dentropy needs the entropies");
  const uint64_t e = dtype_bytes(dtype), n = rows;
  if (!aligned(logits, e) || !aligned(dlogits, e) || !aligned(tokens, 8) || !aligned(lse, 4) ||
      !aligned(entropy, 4) || !aligned(dlogprobs, 4) || !aligned(dentropy, 4))
    return invalid("launch_token_logprobs_backward: a pointer is not aligned to its type");
  const uint64_t bytes = logits_bytes(dtype, rows, vocab, row_stride);
  if (overlap(dlogits, bytes, logits, bytes) || overlap(dlogits, bytes, tokens, 8 * n) ||
      overlap(dlogits, bytes, lse, 4 * n) || overlap(dlogits, bytes, entropy, 4 * n) ||
      overlap(dlogits, bytes, dlogprobs, 4 * n) || overlap(dlogits, bytes, dentropy, 4 * n))
    return invalid("launch_token_logprobs_backward: dlogits overlaps an input, which violates the "
                   "__restrict__ contract");
  const int64_t per_wg = kBackVecs * kThreads * (16 / static_cast<int64_t>(e));
  const int64_t per_row = (vocab + per_wg - 1) / per_wg;
  if (rows * per_row > int64_t{UINT32_MAX} / kThreads)
    return invalid("launch_token_logprobs_backward: rows x vocab exceed the grid's 32-bit work "
                   "size");
  const unsigned grid = static_cast<unsigned>(rows * per_row);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&]<typename T>(T*) {
    logprobs_backward_kernel<T><<<grid, kThreads, 0, s>>>(
        static_cast<const T*>(logits), tokens, lse, entropy, dlogprobs, dentropy,
        static_cast<T*>(dlogits), vocab, row_stride, static_cast<int>(per_row), scale);
    MCKE_LAUNCH_CHECK("logprobs_backward_kernel");
    return ok();
  };
  if (dtype == MCKE_DTYPE_F32) return launch(static_cast<float*>(nullptr));
  if (dtype == MCKE_DTYPE_F16) return launch(static_cast<_Float16*>(nullptr));
  return launch(static_cast<__bf16*>(nullptr));
}

}  // extern "C"
