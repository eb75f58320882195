// One step of beam search, and the sentences that its steps leave behind.
//
// The step, for the K beams of a sentence with running scores r[k] and logits x[k, :]:
//
//   lse[k]   = log sum_t exp(x[k, t])
//   s[k, t]  = r[k] + (x[k, t] - lse[k])
//   the 2K best (k, t): by s, then the lowest beam, then the largest logit, then the lowest token
//   -> those that end the sentence join the pool of finished sentences, the K best others go on.
//
// One cluster of blocks per sentence reads every logit once; a warp owns a slice of one beam's row (a "unit").
// What a kernel of this size costs is not the bytes but the steps that wait for one another (a cluster barrier is some 900
// cycles, as much as the exponentials of a block's 32 KB), so there is one exchange (and before the first word of it a
// barrier that says that every block has started: arrived at before the pass over the logits, waited for behind it):
//
//   * In a block, the warps of one row form a segment.  The n-th largest of the maxima of groups of its lanes is a bound
//     that n of its elements reach, so only lanes whose own maximum reaches it look at their elements again: for n = 8
//     about nine candidates per segment are left.
//   * Those, the bounds and the slices' maxima and sums of exponentials go to the cluster's first block, which makes the
//     log-sums, scores the candidates, keeps those that reach the best segment's bound (and thins them out by a bound of
//     their own where they are many, n = 32) and ranks the rest by counting.
//   * Where that fails - fewer finite candidates than n, or hundreds of equal ones - every warp makes the sorted list of its
//     slice's n best instead and the first block merges the lists.
//
// Exponentials are float32 (off by 2^-22 at most, 5e-8 too small on average, and by the rounding of their arguments), 32 of a
// lane are summed in float32, everything from there on and the scores in float64.  Log-sums came out within 1.4e-7 of the
// exact ones (rows of 1000 to 250112 logits, of standard deviation 0.3 to 6, and peaked ones): candidates of different beams
// are told apart to that, those of one beam exactly.  (With a lane's whole sum in float32 1.6e-6 where it had 2000 terms.)
//
// Measured on B200 (device time, launches in a graph): 7.1 us for one sentence of 4 beams x 32128 bf16 logits, 11.6 us for
// 64 of them (16.4 MB), 21.1 us for 8 sentences of 16 beams x 65537 float32 logits (33.6 MB; the pass itself 5.8 us, at
// the copy rate).  Of the first, about 1400 cycles are the first reads, 2100 the exponentials (one unit of 16 a clock),
// 1000 the barrier, 8000 the short steps around it; that every block has started costs 0.1 to 0.2 us of them, the sums in
// float64 0.07.  A second exchange with a bound over the whole sentence, float64 second looks and unrolled one-shot code
// (126 KB) cost 9.0, 12.0 and 9.2 us.
//
// The reference has no beam search of its own (its heads inherit it: src/turbot5/heads/t5_heads.py:100-130).
#include "t5b_common.cuh"

#include <cooperative_groups.h>

#include <atomic>
#include <new>
#include <type_traits>

namespace cg = cooperative_groups;

namespace t5b {
namespace beam {

constexpr int WARPS = 16;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_UNITS = WARPS * MAX_CLUSTER;
constexpr int MAX_FOUND = 1024;          // candidates of a sentence, an equal share for each block of the cluster
constexpr int FEW = 128;                 // candidates that are ranked by counting
constexpr int MAX_BEAMS = 16;
constexpr int TOKEN_BITS = 27;
constexpr uint32_t TOKEN_MASK = (1u << TOKEN_BITS) - 1;

struct Params {
  const void* logits; int64_t row_stride;
  const float* scores; const float* fin_scores; const int32_t* fin_steps; const int32_t* fin_beams; const uint8_t* done;
  const int64_t* pos;
  int64_t* tokens_out; int32_t* parents_out; float* scores_out;
  float* fin_scores_out; int32_t* fin_steps_out; int32_t* fin_beams_out; uint8_t* done_out;
  int32_t* hist_tokens; int32_t* hist_parents; int64_t hist_steps;
  int32_t B, K, V, n;                    // n candidates
  int32_t S, cluster_log2;               // slices per row; blocks per sentence
  uint32_t unit_magic, slice_magic;      // ceil(2^16 / S), ceil(2^32 / S)
  int64_t eos, pad;
  double length_penalty;
  int32_t early_stopping;
};

// (score, key) orders candidates: key = lowest beam, then largest logit, then lowest token
struct Cand { double score; uint64_t key; };
__device__ __forceinline__ bool better(double sa, uint64_t ka, double sb, uint64_t kb) { return sa > sb || (sa == sb && ka > kb); }
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x == x ? x + 0.f : -INFINITY;      // NaN: never chosen; -0 is 0
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t make_key(int beam, float logit, int token) {
  return (uint64_t)(31 - beam) << 59 | (uint64_t)ordered(logit) << TOKEN_BITS | (TOKEN_MASK - (uint32_t)token);
}
__device__ __forceinline__ int key_beam(uint64_t k) { return 31 - (int)(k >> 59); }
__device__ __forceinline__ int key_token(uint64_t k) { return (int)(TOKEN_MASK - ((uint32_t)k & TOKEN_MASK)); }
__device__ __forceinline__ float key_logit(uint64_t k) { return unordered((uint32_t)(k >> TOKEN_BITS)); }

// A row's part in the scores.  A row of -inf or NaN only, or one whose running score is -inf, has nothing to choose;
// where logits are +inf, those share the whole probability.
struct Row { double run, lse, log_inf; int state; };   // state: 0 ordinary, 1 nothing to choose, 2 has +inf
__device__ __forceinline__ double score_of(const Row& r, float x) {
  if (r.state == 1 || !(x == x)) return -INFINITY;
  if (r.state == 2) return x == INFINITY ? r.run - r.log_inf : -(double)INFINITY;
  const double s = r.run + ((double)x - r.lse);
  return s == s ? s : -(double)INFINITY;
}

// ln x for 1 <= x < 2^60 to about 1e-13: x = 2^e f, f in [0.7, 1.42), ln f = 2 artanh((f - 1) / (f + 1)) by its series.
__device__ __forceinline__ double log_of(double x) {
  int64_t bits = __double_as_longlong(x);
  int e = (int)(bits >> 52) - 1023;
  double f = __longlong_as_double((bits & 0xfffffffffffffll) | 0x3ff0000000000000ll);
  if (f > 1.4142135623730951) { f *= 0.5; ++e; }
  double r = (double)__frcp_rn((float)(f + 1.0));        // 1 / (f + 1): 24 bits, doubled once
  r = r * (2.0 - (f + 1.0) * r);
  const double s = (f - 1.0) * r, q = s * s, q2 = q * q, q4 = q2 * q2;
  const double even = (1.0 + q * (1.0 / 3)) + q2 * (1.0 / 5 + q * (1.0 / 7));
  const double odd = (1.0 / 9 + q * (1.0 / 11)) + q2 * (1.0 / 13 + q * (1.0 / 15));
  return e * 0.6931471805599453 + 2.0 * s * (even + q4 * odd);
}

template <typename T> struct Pack;
template <> struct Pack<float> { static constexpr int N = 4; static constexpr uint32_t none = 0xff800000u; };
template <> struct Pack<__half> { static constexpr int N = 8; static constexpr uint32_t none = 0xfc00fc00u; };
template <> struct Pack<__nv_bfloat16> { static constexpr int N = 8; static constexpr uint32_t none = 0xff80ff80u; };

template <typename T> __device__ __forceinline__ void unpack(const uint4& u, float* f);
template <> __device__ __forceinline__ void unpack<float>(const uint4& u, float* f) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  #pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void unpack<__half>(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}

// Which of U vectors' elements are at least `least`: bits q and q + 16 (16-bit types: the two halves of word q) or bit q.
template <typename T, int U> __device__ __forceinline__ uint32_t mask_of(const uint4 (&u)[U], float least) {
  uint32_t mask = 0;
  #pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = 4 * i + j;
      if constexpr (sizeof(T) == 4) mask |= __uint_as_float(w[j]) >= least ? 1u << q : 0u;
      else if constexpr (std::is_same<T, __half>::value)
        mask |= __hge2_mask(*reinterpret_cast<const __half2*>(&w[j]), __float2half2_rn(least)) & (0x00010001u << q);
      else
        mask |= __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[j]), __float2bfloat162_rn(least)) & (0x00010001u << q);
    }
  }
  return mask;
}
// One of a vector's 2^sub equal parts, -inf in place of the others.
template <typename T> __device__ __forceinline__ uint4 part_of(const uint4& u, int sub, int part) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    if ((sub < 3 ? j >> (2 - sub) : 2 * j + (part & 1)) != part) w[j] = Pack<T>::none;
    else if (sub == 3) w[j] = part & 1 ? (w[j] & 0xffff0000u) | (Pack<T>::none & 0xffffu) : (w[j] & 0xffffu) | (Pack<T>::none & 0xffff0000u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T> struct Lowest;     // the lowest finite number: the bound of what can be chosen
template <> struct Lowest<float> { static constexpr float value = -3.402823466e38f; };
template <> struct Lowest<__half> { static constexpr float value = -65504.f; };
template <> struct Lowest<__nv_bfloat16> { static constexpr float value = -3.38953139e38f; };

// A warp's slice of one row: 16-byte vectors [v0, v1) of the row's aligned middle; the first slice also has the
// elements before it, the last one those behind it (fewer than a vector each, one per lane).
template <typename T> struct Slice {
  const T* row; const uint4* mid;
  int v0, v1, head, tail, V;             // elements [0, head) and [tail, V) outside the vectors, if this slice has them
  __device__ __forceinline__ Slice(const T* r, int V_, int part, int S, uint32_t magic) : row(r), V(V_) {
    constexpr int N = Pack<T>::N;
    const int mis = (int)(((uintptr_t)r & 15) / sizeof(T));
    const int before = min(mis ? N - mis : 0, V_);
    const int nv = (V_ - before) / N;
    mid = (const uint4*)(r + before);
    const int each = (S == 1 ? nv : (int)__umulhi((unsigned)nv, magic)) + 1;      // at least nv / S, without a division
    v0 = (int)min((int64_t)part * each, (int64_t)nv); v1 = min(v0 + each, nv);
    head = part == 0 ? before : 0;
    tail = part == S - 1 ? before + nv * N : V_;
    first = before;
  }
  int first;                             // element index of the first vector
  // f(logit, token) for every element of one lane; the same elements whichever lane of the warp asks
  template <typename F> __device__ __forceinline__ void each(int lane, F f) const {
    if (lane < head) f(to_float<T>(row[lane]), lane);
    if (tail + lane < V) f(to_float<T>(row[tail + lane]), tail + lane);
    #pragma unroll 1
    for (int v = v0 + lane; v < v1; v += 32)
      #pragma unroll 1
      for (int e = 0; e < Pack<T>::N; ++e) f(to_float<T>(row[first + v * Pack<T>::N + e]), first + v * Pack<T>::N + e);
  }
};

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ double warp_sum(double v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The two halves of a barrier of the cluster that says that every block has started.  Nothing that is written before it is
// read by another block, so it orders no memory (with a release 0.3 to 0.8 us of the step went to it: the fence waits for
// the logits' first reads).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Sum of exponentials of a slice that holds NaN (left out) or +inf (counted): rare, and kept out of the way.
template <typename T>
__device__ __noinline__ double careful_sum(const Slice<T>& sl, float most, int lane) {
  double t = 0.0;
  sl.each(lane, [&](float x, int) {
    if (x == x) t += most == INFINITY ? (x == INFINITY ? 1.0 : 0.0) : most > -INFINITY ? (double)fast_exp2((x - most) * kLog2e) : 0.0;
  });
  return warp_sum(t);
}

// Sorted list of the n best keys of a slice, lane i the i-th best (0 = none).
template <typename T>
__device__ __noinline__ uint64_t best_of_slice(const Slice<T>& sl, int beam, int n, int lane) {
  uint64_t mine = 0;
  auto insert = [&](uint64_t key) {
    // key: one candidate per lane, 0 where there is none
    const uint64_t last = __shfl_sync(0xffffffffu, mine, n - 1);
    uint32_t todo = __ballot_sync(0xffffffffu, key > last);
    while (todo) {
      const uint64_t k = __shfl_sync(0xffffffffu, key, __ffs(todo) - 1);
      todo &= todo - 1;
      const int at = __popc(__ballot_sync(0xffffffffu, mine > k));
      const uint64_t up = __shfl_up_sync(0xffffffffu, mine, 1);
      mine = lane < at ? mine : lane == at ? k : up;
      if (lane >= n) mine = 0;
    }
  };
  // vectors in turn, the next one on its way; then the elements before and behind them
  constexpr int N = Pack<T>::N;
  uint4 next = make_uint4(0, 0, 0, 0);
  if (sl.v0 + lane < sl.v1) next = __ldg(sl.mid + sl.v0 + lane);
  #pragma unroll 1
  for (int v = sl.v0 + lane; v - lane < sl.v1; v += 32) {
    const uint4 w = next;
    const bool in = v < sl.v1;
    if (v + 32 < sl.v1) next = __ldg(sl.mid + v + 32);
    float x[N];
    unpack<T>(w, x);
    #pragma unroll
    for (int e = 0; e < N; ++e) insert(in ? make_key(beam, x[e], sl.first + v * N + e) : 0);
  }
  insert(lane < sl.head ? make_key(beam, to_float<T>(sl.row[lane]), lane) : 0);
  insert(sl.tail + lane < sl.V ? make_key(beam, to_float<T>(sl.row[sl.tail + lane]), sl.tail + lane) : 0);
  return mine;
}

struct Shared {
  double usum[MAX_UNITS];
  float umax[MAX_UNITS];
  float reached[MAX_UNITS];              // what n elements of a segment reach, at its first slice (-inf elsewhere)
  alignas(16) float group[THREADS];      // maxima of groups of lanes, a segment's from its first warp's place on
  float bound[WARPS];                    // found by this warp; the smallest of a segment's holds
  Row rows[MAX_BEAMS];                   // running rows, in order
  double inv_length;
  int counts[MAX_CLUSTER];               // candidates found by each block
  int found_here, overflow, kept;
  uint32_t threshold;                    // a score that n candidates reach, ordered bits of a float
  union {
    struct {
      uint64_t found[MAX_FOUND];         // their keys
      double score[MAX_FOUND];           // scores and keys, one candidate behind the other
      uint64_t key[MAX_FOUND];
    };
    struct {
      uint64_t lists[WARPS][32];         // sorted keys of a slice
      uint64_t merged[WARPS][32];        // of a segment, at its first warp
      int segment[MAX_BEAMS + MAX_CLUSTER];
      Cand heads[WARPS];
    };
  };
  Cand best[FEW];                        // candidates that are left
  Cand chosen[2][2 * MAX_BEAMS];         // the n best in order, for each of the warps that decide
};

// The n-th largest of a segment's group maxima: a value that at least n of its elements reach (-inf where too few groups
// have a finite one).  Every thread brings its own maximum, 2^shift lanes form a group; then threads count
// for each group how many are above it, and the smallest that fewer than n exceed is the bound.
__device__ __noinline__ float segment_bound(Shared& sm, float mine, int n, int warp, int lane, int first, int warps, int shift) {
  if (shift > 0) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  if (shift > 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
  if (shift > 2) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 4));
  if (shift > 3) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 8));
  const int groups = warps * 32 >> shift, at = first * 32, here = warp - first;
  if ((lane & ((1 << shift) - 1)) == 0) sm.group[at + ((here * 32 + lane) >> shift)] = mine;
  __syncthreads();
  // four threads per group, as far as the segment has them (a group each otherwise); up to three groups that do not fill a
  // vector are not counted, which can only lower the bound
  const int share = warps > 7 ? 2 : 0, t = here * 32 + lane, g = t >> share;
  if (here << 5 < groups << share) {
    const float own = g < groups ? sm.group[at + g] : -INFINITY;
    int above = 0;
    const float4* every = (const float4*)(sm.group + at);
    auto count = [&](const float4& o) { above += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own); };
    if (share) {                         // at most 16 vectors, four a thread, read together
      float4 o[4];
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = (t & 3) + 4 * i;
        o[i] = j < groups / 4 ? every[j] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
      #pragma unroll
      for (int i = 0; i < 4; ++i) count(o[i]);
      above += __shfl_xor_sync(0xffffffffu, above, 1);
      above += __shfl_xor_sync(0xffffffffu, above, 2);
    } else {
      #pragma unroll 4
      for (int j = 0; j < groups / 4; ++j) count(every[j]);
    }
    const float least = -warp_max(above < n && g < groups ? -own : -INFINITY);
    if (lane == 0) sm.bound[warp] = least;
  }
  __syncthreads();
  float least = sm.bound[first];
  #pragma unroll
  for (int i = 1; i < 8; ++i) least = fminf(least, i << 5 < groups << share ? sm.bound[first + i] : INFINITY);
  return least;
}
// lanes per group (their logarithm) so that 33 to 64 groups come out, 17 to 32 for few candidates (8 of 32 groups leave
// 9.2 elements on average, 8 of 64 leave 8.5), 32 of a single warp
__device__ __forceinline__ int group_shift(int warps, int n) {
  const int shift = warps > 8 ? 3 : warps > 4 ? 2 : warps > 2 ? 1 : 0;
  return n <= 8 && warps > 1 ? shift + 1 : shift;
}

// What the step decides from its n best candidates, best first; a warp each, lane i has candidate i.
struct Pool { float score; int step, beam; };

// The pool: its entries and the ended candidates among the K best, larger first, earlier first among equals.
__device__ __forceinline__ void settle(const Params& p, const Cand* best, int b, int lane, const Pool& pool, int64_t pos, double inv_length) {
  const int K = p.K;
  const unsigned all = 0xffffffffu;
  const double score = lane < p.n ? best[lane].score : -INFINITY;
  const uint64_t key = lane < p.n ? best[lane].key : 0;
  const bool ends = lane < p.n && (int64_t)key_token(key) == p.eos;
  const bool joins = ends && lane < K && score > -INFINITY;
  const unsigned joining = __ballot_sync(all, joins), others = __ballot_sync(all, lane < p.n && !ends);
  const float highest = (float)__shfl_sync(all, score, __ffs(others) - 1);           // the first that goes on
  const float old = lane < K && pool.score == pool.score ? pool.score : -INFINITY;
  const float joining_score = (float)(score * inv_length);         // (0 x inf, a penalty beyond all numbers: NaN)
  const float fresh = joins && joining_score == joining_score ? joining_score : -INFINITY;
  int old_rank = lane, new_rank = 0;
  const float next = __shfl_down_sync(all, old, 1);
  if (joining || __any_sync(all, lane < K - 1 && next > old)) {
    old_rank = 0;
    #pragma unroll 1
    for (int j = 0; j < K; ++j) {
      const float o = __shfl_sync(all, old, j);
      old_rank += o > old || (o == old && j < lane);
      new_rank += o >= fresh;
    }
    #pragma unroll 1
    for (unsigned m = joining; m; m &= m - 1) {
      const int j = __ffs(m) - 1;
      const float o = __shfl_sync(all, fresh, j);
      old_rank += o > old;
      new_rank += o > fresh || (o == fresh && j < lane);
    }
  }
  if (lane < K && old_rank < K) {
    const int64_t to = (int64_t)b * K + old_rank;
    p.fin_scores_out[to] = old; p.fin_steps_out[to] = pool.step; p.fin_beams_out[to] = pool.beam;
  }
  if (joins && new_rank < K) {
    const int64_t to = (int64_t)b * K + new_rank;
    p.fin_scores_out[to] = fresh; p.fin_steps_out[to] = (int)pos; p.fin_beams_out[to] = key_beam(key);
  }
  // whoever came last in the pool (one of them is there: K entries and the joining ones fill it)
  const bool last_old = lane < K && old_rank == K - 1, last_new = joins && new_rank == K - 1;
  if (last_old || last_new) {
    const float worst = last_old ? old : fresh;
    bool full = worst > -INFINITY;
    if (!p.early_stopping) full = full && (double)worst >= (double)highest * inv_length;
    p.done_out[b] = full || highest == -INFINITY;
  }
}

// The K best that go on: one continuation of a beam stays in its place, further ones take the free places in order.
__device__ __forceinline__ void go_on(const Params& p, const Cand* best, int b, int lane, int64_t pos) {
  const int K = p.K;
  const unsigned all = 0xffffffffu, below = (1u << lane) - 1;
  const uint64_t key = lane < p.n ? best[lane].key : 0;
  const int token = key_token(key), beam = key_beam(key);
  const bool may = lane < p.n && (int64_t)token != p.eos;
  const int order = __popc(__ballot_sync(all, may) & below);
  const bool on = may && order < K;
  unsigned same = 0, used = 0;
  #pragma unroll 4
  for (int j = 0; j < K; ++j) {
    const unsigned those = __ballot_sync(all, on && beam == j);
    if (beam == j) same = those;
    used |= those ? 1u << j : 0u;
  }
  const bool further = on && (same & below) != 0;
  const unsigned again = __ballot_sync(all, further);
  unsigned open = ~used & ((1u << K) - 1);
  int place = beam;
  if (further) {
    #pragma unroll 1
    for (int skip = __popc(again & below); skip > 0; --skip) open &= open - 1;
    place = __ffs(open) - 1;
  }
  if (on && (unsigned)place < (unsigned)K) {
    const int64_t to = (int64_t)b * K + place;
    p.tokens_out[to] = token; p.parents_out[to] = beam; p.scores_out[to] = (float)best[lane].score;
    if (p.hist_tokens && pos >= 0 && pos < p.hist_steps) {
      const int64_t h = pos * p.B * K + to;
      p.hist_tokens[h] = token; p.hist_parents[h] = beam;
    }
  }
}

// SHORT: slices of at most 16 vectors, each of which 2^sub lanes share, so that a segment's bound has groups enough to be
// taken from (small vocabularies: 10 beams x 384 bf16 8.2 us, 39 by the lists without it; 5 x 1000 8.2 and 37).
template <typename T, bool SHORT>
__global__ void __launch_bounds__(THREADS, 2)
step_kernel(const __grid_constant__ Params p) {
  __shared__ Shared sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = 1 << p.cluster_log2, rank = (int)(blockIdx.x & (C - 1));
  const int b = blockIdx.x >> p.cluster_log2;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int K = p.K, n = p.n, S = p.S;
  const int64_t at = (int64_t)b * K;

  // the first logits are on their way before anything else is known
  const int unit = rank * WARPS + warp, row = (int)(unit * p.unit_magic >> 16);
  const bool owns = row < K;
  const int k = owns ? row : 0;
  const Slice<T> sl((const T*)p.logits + (at + k) * p.row_stride, p.V, owns ? unit - row * S : 0, S, p.slice_magic);
  constexpr int N = Pack<T>::N, U = SHORT ? 1 : 4;
  const int span = sl.v1 - sl.v0, sub = !SHORT ? 0 : span > 8 ? 1 : span > 4 || N == 4 ? 2 : 3, of = lane >> sub;
  uint4 u[U];
  #pragma unroll
  for (int i = 0; i < U; ++i) {
    u[i] = make_uint4(Pack<T>::none, Pack<T>::none, Pack<T>::none, Pack<T>::none);
    if (owns && sl.v0 + of + 32 * i < sl.v1) u[i] = __ldg(sl.mid + sl.v0 + of + 32 * i);
  }
  if (SHORT) u[0] = part_of<T>(u[0], sub, lane & ((1 << sub) - 1));
  const float x_head = owns && lane < sl.head ? to_float<T>(sl.row[lane]) : -INFINITY;
  const float x_tail = owns && sl.tail + lane < sl.V ? to_float<T>(sl.row[sl.tail + lane]) : -INFINITY;
  // what the last part needs
  const int64_t pos = *p.pos;
  const float run = p.scores[at + k], row_run = warp < K ? p.scores[at + warp] : -INFINITY;
  Pool pool = {0.f, 0, 0};
  if (rank == 0 && warp == 1 && lane < K) pool = Pool{p.fin_scores[at + lane], p.fin_steps[at + lane], p.fin_beams[at + lane]};

  if (p.done[b]) {                       // the whole cluster: nothing changes any more
    if (rank == 0 && tid < K) {
      p.tokens_out[at + tid] = p.pad; p.parents_out[at + tid] = tid; p.scores_out[at + tid] = p.scores[at + tid];
      p.fin_scores_out[at + tid] = p.fin_scores[at + tid];
      p.fin_steps_out[at + tid] = p.fin_steps[at + tid]; p.fin_beams_out[at + tid] = p.fin_beams[at + tid];
      if (p.hist_tokens && pos >= 0 && pos < p.hist_steps) {
        p.hist_tokens[(pos * p.B + b) * K + tid] = (int32_t)p.pad; p.hist_parents[(pos * p.B + b) * K + tid] = tid;
      }
      if (tid == 0) p.done_out[b] = 1;
    }
    return;
  }

  // ---- one pass over the logits: maximum and sum of exponentials of a slice
  Shared* lead = cluster.map_shared_rank(&sm, 0);
  const bool active = owns && run > -INFINITY;
  // a lane's maximum, its vector with the largest element and what its other vectors reach at most
  float m = -INFINITY, in_best = -INFINITY, in_others = -INFINITY;
  int best_at = 0;
  if (tid == 0) { sm.found_here = 0; sm.overflow = 0; sm.kept = 0; sm.threshold = 0; }
  cluster_arrive();
  float wm = -INFINITY;
  double total = 0.0;
  if (active) {
    m = fmaxf(fmaxf(x_head, x_tail), -INFINITY);         // (NaN only: -inf)
    const float edge = m > -INFINITY ? m : 0.f;
    double s = fast_exp2((x_head - edge) * kLog2e) + fast_exp2((x_tail - edge) * kLog2e);
    #pragma unroll 1
    for (int v = sl.v0; v < sl.v1; v += 32 * U) {
      float m_new = m;
      #pragma unroll
      for (int i = 0; i < U; ++i)
        if (v + 32 * i < sl.v1) {        // (the same for the whole warp)
          float x[N];
          unpack<T>(u[i], x);
          float most = -INFINITY;
          #pragma unroll
          for (int e = 0; e < N; e += 4) most = fmaxf(most, fmaxf(fmaxf(x[e], x[e + 1]), fmaxf(x[e + 2], x[e + 3])));
          in_others = fmaxf(in_others, fminf(in_best, most));
          if (most > in_best) { in_best = most; best_at = v + 32 * i; }
          m_new = fmaxf(m_new, most);
        }
      const float ref = m_new > -INFINITY ? m_new : 0.f;
      const double moved = fast_exp2((m - ref) * kLog2e);
      m = m_new;
      float batch = 0.f;
      const bool more = v + 32 * U < sl.v1;
      #pragma unroll
      for (int i = 0; i < U; ++i)
        if (v + 32 * i < sl.v1) {
          float x[N];
          unpack<T>(u[i], x);
          if (more) {                    // the place is free: the next batch's vector
            const int next = v + lane + 32 * (U + i);
            if (next < sl.v1) u[i] = __ldg(sl.mid + next);
            else u[i] = make_uint4(Pack<T>::none, Pack<T>::none, Pack<T>::none, Pack<T>::none);
          }
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          #pragma unroll
          for (int e = 0; e < N; ++e) part[e & 3] += fast_exp2((x[e] - ref) * kLog2e);
          batch += (part[0] + part[1]) + (part[2] + part[3]);
        }
      s = s * moved + batch;
    }
    wm = warp_max(m);
    if (__any_sync(0xffffffffu, !(s == s) || m == INFINITY)) {      // NaN or +inf among the logits
      total = careful_sum<T>(sl, wm, lane);
    } else {
      total = warp_sum(wm > -INFINITY ? s * (double)fast_exp2((m - wm) * kLog2e) : 0.0);
    }
  }
  // every block has started: from here on the first one's memory may be written, where it writes nothing itself
  cluster_wait();
  if (active && lane == 0) { lead->umax[unit] = wm; lead->usum[unit] = total; }

  // ---- the candidates of this block's segments
  const int first = active ? max(k * S - rank * WARPS, 0) : warp;                    // the segment's warps
  const int warps = active ? min((k + 1) * S - rank * WARPS, WARPS) - first : 1;
  const float reached = segment_bound(sm, m, n, warp, lane, first, warps, group_shift(warps, n));
  const float least = fmaxf(reached, Lowest<T>::value);
  const int share = MAX_FOUND >> p.cluster_log2;
  if (active) {
    if (lane == 0) lead->reached[unit] = warp == first ? reached : -INFINITY;
    const bool mine = m >= least;
    auto push = [&](float x, int token) {
      const int i = atomicAdd(&sm.found_here, 1);
      if (i < share) lead->found[rank * share + i] = make_key(k, x, token);
    };
    if (mine) {
      if (x_head >= least) push(x_head, lane);
      if (x_tail >= least) push(x_tail, sl.tail + lane);
    }
    auto push_vector = [&](const uint4& w, int v) {
      const uint4 one[1] = {w};
      #pragma unroll 1
      for (uint32_t mask = mask_of<T, 1>(one, least); mask; mask &= mask - 1) {
        const int bit = __ffs(mask) - 1, e = N == 8 ? 2 * (bit & 3) + (bit >> 4) : bit & 3;
        float x[N], found = 0.f;
        unpack<T>(w, x);
        #pragma unroll
        for (int j = 0; j < N; ++j) if (e == j) found = x[j];
        push(found, sl.first + v * N + e);
      }
    };
    // most lanes have one vector that reaches the bound: still in registers where the slice is four vectors a lane
    const bool one = mine && in_best >= least && in_others < least;
    if (__any_sync(0xffffffffu, one)) {
      uint4 w = u[0];
      if (sl.v1 - sl.v0 <= 32 * U) {
        #pragma unroll
        for (int j = 1; j < U; ++j) if (best_at == sl.v0 + 32 * j) w = u[j];
      } else if (one) {
        w = __ldg(sl.mid + best_at + lane);
      }
      if (one) push_vector(w, best_at + of);
    }
    #pragma unroll 1
    for (uint32_t todo = __ballot_sync(0xffffffffu, mine && in_others >= least); todo; todo &= todo - 1) {
      // more than can be used: the lists will do it (other warps add to the number: what one lane has read holds)
      if (__shfl_sync(0xffffffffu, *(volatile int*)&sm.found_here, 0) > share) break;
      const int who = __ffs(todo) - 1;                   // several: its vectors again, by the whole warp
      #pragma unroll 1
      for (int v = sl.v0 + who + 32 * lane; v < sl.v1; v += 32 * 32) push_vector(__ldg(sl.mid + v), v);
      __syncwarp();
    }
  }
  __syncthreads();
  if (tid == 0) lead->counts[rank] = sm.found_here;
  cluster.sync();

  // ---- the first block: log-sums, scores, the n best
  if (rank == 0) {
    if (warp < K) {
      // a lane's slices first (one, with four beams and eight blocks), then the warp's
      float mine = -INFINITY, reach = -INFINITY;
      double sum = 0.0;
      #pragma unroll 1
      for (int i = row_run > -INFINITY ? lane : S; i < S; i += 32) {
        const float um = sm.umax[warp * S + i];
        const double us = sm.usum[warp * S + i];
        reach = fmaxf(reach, sm.reached[warp * S + i]);
        if (um > mine) { sum = us + (mine > -INFINITY && um < INFINITY ? sum * (double)fast_exp2((mine - um) * kLog2e) : 0.0); mine = um; }
        else if (um == mine) sum += um > -INFINITY ? us : 0.0;
        else if (um > -INFINITY && mine < INFINITY) sum += us * (double)fast_exp2((um - mine) * kLog2e);
      }
      const float most = warp_max(mine);
      reach = warp_max(reach);
      if (mine < most) sum = mine > -INFINITY && most < INFINITY ? sum * (double)fast_exp2((mine - most) * kLog2e) : 0.0;
      sum = log_of(warp_sum(sum));
      if (lane == 0) {
        const Row r{row_run, (double)most + sum, sum, !(most > -INFINITY) ? 1 : most == INFINITY ? 2 : 0};
        sm.rows[warp] = r;
        atomicMax(&sm.threshold, ordered(__double2float_rd(score_of(r, reach))));
      }
    }
    if (warp == WARPS - 1 && lane == 1) {                // (K = 16: this warp has a row as well)
      const double steps = (double)(pos + 1);
      sm.inv_length = p.length_penalty == 1.0 ? 1.0 / steps : p.length_penalty == 0.0 ? 1.0 : pow(steps, -p.length_penalty);
    }
    int total = 0, before = 0;
    bool fits = true;
    #pragma unroll
    for (int r = 0; r < MAX_CLUSTER; ++r) {
      const int c = r < C ? sm.counts[r] : 0;            // (each block has written its own)
      fits = fits && c <= share;
      before += r < (warp & (C - 1)) ? c : 0;
      total += c;
    }
    __syncthreads();
    const double threshold = (double)unordered(sm.threshold);
    if (fits) {
      // warps take the blocks' lists in turn
      const int r = warp & (C - 1), step = WARPS * 32 >> p.cluster_log2;
      #pragma unroll 1
      for (int i = (warp >> p.cluster_log2) * 32 + lane; i < sm.counts[r]; i += step) {
        const uint64_t key = sm.found[r * share + i];
        const double score = score_of(sm.rows[key_beam(key)], key_logit(key));
        sm.score[before + i] = score; sm.key[before + i] = key;
        if (score >= threshold && score > -INFINITY) {
          const int at = atomicAdd(&sm.kept, 1);
          if (at < FEW) sm.best[at] = Cand{score, key};
        }
      }
    }
    __syncthreads();
    int count = sm.kept;
    bool done = fits && count >= n;
    if (done && count > FEW) {
      // many: the bound of a segment again, over all candidates (thread t has candidates t / 8 + 64 * (t % 8) and 512
      // further on)
      const int i0 = (tid >> 3) + 64 * (tid & 7), i1 = i0 + THREADS;
      const float f0 = i0 < total ? __double2float_rd(sm.score[i0]) : -INFINITY;
      const float f1 = i1 < total ? __double2float_rd(sm.score[i1]) : -INFINITY;
      const float least = segment_bound(sm, fmaxf(f0, f1), n, warp, lane, 0, WARPS, 3);
      if (tid == 0) sm.kept = 0;
      __syncthreads();
      if (f0 >= least && f0 > -INFINITY) { const int i = atomicAdd(&sm.kept, 1); if (i < FEW) sm.best[i] = Cand{sm.score[i0], sm.key[i0]}; }
      if (f1 >= least && f1 > -INFINITY) { const int i = atomicAdd(&sm.kept, 1); if (i < FEW) sm.best[i] = Cand{sm.score[i1], sm.key[i1]}; }
      __syncthreads();
      count = sm.kept;
      done = count >= n && count <= FEW;
    }
    if (done) {
      asm volatile("barrier.cluster.arrive.relaxed.aligned;");               // the others may go: nothing more reaches them
      if (count <= 32) {
        // two warps, each for itself: lane i counts for candidate i, then one sees to the beams and one to the pool
        if (warp > 1) return;
        const Cand mine = lane < count ? sm.best[lane] : Cand{-INFINITY, 0};
        int above = 0;
        #pragma unroll 4
        for (int j = 0; j < count; ++j) above += better(sm.best[j].score, sm.best[j].key, mine.score, mine.key);
        if (lane < count && above < n) sm.chosen[warp][above] = mine;
        __syncwarp();
      } else {
        // four threads count for each of the candidates
        const int i = tid >> 2;
        const Cand mine = i < count ? sm.best[i] : Cand{-INFINITY, 0};
        int above = 0;
        #pragma unroll 2
        for (int j = tid & 3; j < count; j += 4) above += better(sm.best[j].score, sm.best[j].key, mine.score, mine.key);
        above += __shfl_xor_sync(0xffffffffu, above, 1);
        above += __shfl_xor_sync(0xffffffffu, above, 2);
        if (i < count && (tid & 3) < 2 && above < n) sm.chosen[tid & 1][above] = mine;
        __syncthreads();
      }
      if (warp == 0) go_on(p, sm.chosen[0], b, lane, pos);
      if (warp == 1) settle(p, sm.chosen[1], b, lane, pool, pos, sm.inv_length);
      return;
    }
    if (tid < C) cluster.map_shared_rank(&sm, tid)->overflow = 1;
  }
  cluster.sync();
  if (!sm.overflow) return;

  // ---- too few or too many candidates: a sorted list per slice of every row, one per segment of those (an element's place
  // in the segment is the number of larger ones in each of its lists), and the n best of all in turn by the first block
  sm.merged[warp][lane] = 0;
  if (owns) sm.lists[warp][lane] = best_of_slice<T>(sl, k, n, lane);
  __syncthreads();
  if (owns && lane < n) {
    const uint64_t mine = sm.lists[warp][lane];
    const int from = max(k * S - rank * WARPS, 0), to = min((k + 1) * S - rank * WARPS, WARPS);
    int above = 0;
    #pragma unroll 2
    for (int w = from; w < to; ++w) {
      int more = 0;                      // sorted: a search for the first that is not larger
      #pragma unroll
      for (int half = 32; half > 0; half >>= 1)
        if (more + half <= n && sm.lists[w][more + half - 1] > mine) more += half;
      above += more;
    }
    if (mine && above < n) sm.merged[from][above] = mine;
  }
  if (tid == 0) sm.kept = 0;
  cluster.sync();
  if (rank == 0) {
    // every thread has two candidates: number tid % 32 of two of the segments (at most K + C - 1 of them)
    if (tid < C * WARPS && tid < K * S && (tid % WARPS == 0 || tid % S == 0)) sm.segment[atomicAdd(&sm.kept, 1)] = tid;
    __syncthreads();
    Cand mine[2];
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      mine[i] = Cand{-INFINITY, 0};
      const int at = (tid >> 5) + i * WARPS;
      if (at < sm.kept) {
        const int u = sm.segment[at];
        mine[i].key = cluster.map_shared_rank(&sm, u / WARPS)->merged[u % WARPS][lane];
        if (mine[i].key) mine[i].score = score_of(sm.rows[key_beam(mine[i].key)], key_logit(mine[i].key));
      }
    }
    #pragma unroll 1
    for (int i = 0; i < n; ++i) {
      Cand top = better(mine[1].score, mine[1].key, mine[0].score, mine[0].key) ? mine[1] : mine[0];
      #pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double os = __shfl_xor_sync(0xffffffffu, top.score, o);
        const uint64_t ok = __shfl_xor_sync(0xffffffffu, top.key, o);
        if (better(os, ok, top.score, top.key)) { top.score = os; top.key = ok; }
      }
      if (lane == 0) sm.heads[warp] = top;
      __syncthreads();
      top = sm.heads[0];
      #pragma unroll 5
      for (int w = 1; w < WARPS; ++w) if (better(sm.heads[w].score, sm.heads[w].key, top.score, top.key)) top = sm.heads[w];
      if (tid < 2) sm.chosen[tid][i] = top;
      #pragma unroll
      for (int j = 0; j < 2; ++j) if (mine[j].key == top.key) mine[j] = Cand{-INFINITY, 0};
      __syncthreads();
    }
    if (warp == 0) go_on(p, sm.chosen[0], b, lane, pos);
    if (warp == 1) settle(p, sm.chosen[1], b, lane, pool, pos, sm.inv_length);
  }
  cluster.sync();                        // nobody leaves while its shared memory is read
}

// ---- sentences from the history of tokens and parents -------------------------------------------------------------
//
// Bound by the length of its chains, not by bytes: 7.7 us for 64 searches x 8 sentences x 512 steps, 3.8 us for one of 32.
// Walking back from the last token is a chain of dependent reads.  A block per sentence brings a segment of tokens and
// parents into shared memory (every read in flight at once) and cuts it into pieces: every piece is walked from each of
// its K possible beams, the pieces' results are chained per returned sentence, and the pieces are walked again from the
// beam that is now known.  Three short chains instead of one of T reads from memory.
constexpr int SEGMENT = 1024;            // steps in shared memory at a time
constexpr int SEQ_THREADS = 512;
constexpr int PIECES = 32;

struct SequenceParams {
  const int32_t* tokens; const int32_t* parents; const float* scores; const float* fin_scores;
  const int32_t* fin_steps; const int32_t* fin_beams; const uint8_t* done;
  int64_t* out; float* out_scores;
  int32_t T, B, K, R, k_log2;            // 2^k_log2 >= K
  int64_t eos, pad;
  double length;
};

__global__ void __launch_bounds__(SEQ_THREADS)
sequences_kernel(const __grid_constant__ SequenceParams p) {
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ int last[MAX_BEAMS], from[MAX_BEAMS], cur[MAX_BEAMS];
  __shared__ bool ended[MAX_BEAMS], none[MAX_BEAMS];
  __shared__ int2 cut[MAX_BEAMS];                          // last step with a token of its own, and the end token's
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int K = p.K, R = p.R, T = p.T, kl = p.k_log2;
  const int seg = min(SEGMENT, T), pitch = (seg + 31) / 32 * 32 + 4;       // (no bank conflicts by step or by beam)
  int32_t* words = (int32_t*)raw;                          // [K][pitch]
  uint8_t* par = raw + (size_t)K * pitch * 4;              // [seg][2^kl]
  uint8_t* path = par + ((size_t)seg << kl);               // [R][pitch]
  uint8_t* jump = path + (size_t)R * pitch;                // [PIECES][2^kl]
  const int x_of = tid & ((1 << kl) - 1), t_of = tid >> kl, rows = SEQ_THREADS >> kl;

  // the candidates: lanes [0, K) of the first warp the pool, [K, 2K) the running beams
  float value = -INFINITY;
  int their_step = 0, their_beam = 0;
  bool finished = false;
  if (warp == 0) {
    const int64_t at = (int64_t)b * K;
    finished = p.done[b];
    if (lane < K) { value = p.fin_scores[at + lane]; their_step = p.fin_steps[at + lane]; their_beam = p.fin_beams[at + lane]; }
    else if (lane < 2 * K) value = p.scores[at + lane - K];
  }
  for (int hi = T; hi > 0; hi -= seg) {
    const int lo = max(0, hi - seg), len = hi - lo;
    // par[i]: the beam at step lo + i - 1 of each beam at step lo + i
    #pragma unroll 1
    for (int t0 = 0; t0 < len; t0 += 8 * rows) {
      int w[8], q[8];
      #pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + i * rows + t_of;
        const int64_t at = ((int64_t)(lo + t) * p.B + b) * K + x_of;
        const bool in = t < len && x_of < K;
        w[i] = in ? __ldg(p.tokens + at) : 0;
        q[i] = in ? __ldg(p.parents + at) : 0;
      }
      #pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + i * rows + t_of;
        if (t < len && x_of < K) { words[x_of * pitch + t] = w[i]; par[t << kl | x_of] = (uint8_t)min(max(q[i], 0), K - 1); }
      }
    }
    if (hi == T && warp == 0) {
      // the best of them, best first
      if (lane >= K) value = finished || lane >= 2 * K ? -INFINITY : (float)((double)value / p.length);
      if (!(value == value)) value = -INFINITY;
      int above = 0;
      #pragma unroll 4
      for (int j = 0; j < 2 * K; ++j) {
        const float o = __shfl_sync(0xffffffffu, value, j);
        above += o > value || (o == value && j < lane);
      }
      if (lane < 2 * K && above < R) {
        const bool e = lane < K;
        ended[above] = e; none[above] = value == -INFINITY;
        // an ended sentence's end token stands at its step, its beams are those up to the step before
        last[above] = e ? min(max(their_step, 0), T - 1) : T - 1;
        from[above] = e ? min(max(their_beam, 0), K - 1) : lane - K;
        cur[above] = 0;
        p.out_scores[(int64_t)b * R + above] = value;
      }
    }
    __syncthreads();
    int pl = 0;                                            // pieces of 2^pl steps, at most PIECES of them
    while (2 << 2 * pl < len) ++pl;
    const int pieces = (len + (1 << pl) - 1) >> pl;
    if (x_of < K)
      #pragma unroll 1
      for (int c = t_of; c < pieces; c += rows) {
        int x = x_of;
        const uint8_t* at = par + ((min((c + 1) << pl, len) - 1) << kl);
        #pragma unroll 4
        for (int j = min((c + 1) << pl, len) - (c << pl); j > 0; --j, at -= 1 << kl) x = at[x];
        jump[c << kl | x_of] = (uint8_t)x;
      }
    __syncthreads();
    // the beam at the last step of every piece per sentence, backwards; kept there in path
    if (tid < R) {
      const int stop = (ended[tid] ? last[tid] - 1 : last[tid]) - lo;                  // its last step, in this segment's
      int x = cur[tid], c = pieces - 1;
      if (stop >= 0 && stop < len) {                       // ... which is in here: its piece is walked step by step
        c = stop >> pl;
        x = from[tid];
        path[tid * pitch + stop] = (uint8_t)x;
        for (int j = stop; j >= c << pl; --j) x = par[j << kl | x];
        --c;
      } else if (stop < 0) {
        c = -1;
      }
      uint8_t* at = path + tid * pitch;
      #pragma unroll 1
      for (; c >= 0; --c) {
        at[min((c + 1) << pl, len) - 1] = (uint8_t)x;
        x = jump[c << kl | x];
      }
      cur[tid] = x;
    }
    __syncthreads();
    for (int r = warp; r < R; r += SEQ_THREADS / 32) {
      const int a = lane << pl, stop = (ended[r] ? last[r] - 1 : last[r]) - lo;
      int j = min(min(a + (1 << pl), len) - 1, stop);
      if (lane >= pieces || j < a) continue;
      int x = path[r * pitch + j];
      #pragma unroll 1
      for (; j > a; --j) { x = par[j << kl | x]; path[r * pitch + j - 1] = (uint8_t)x; }
    }
    __syncthreads();
    // a thread has a step of every sentence
    #pragma unroll 1
    for (int r = warp; r < R; r += SEQ_THREADS / 32) cut[r] = make_int2((none[r] ? -1 : ended[r] ? last[r] - 1 : last[r]) - lo,
                                                                        (ended[r] && !none[r] ? last[r] : -1) - lo);
    __syncthreads();
    for (int i = tid; i < len; i += SEQ_THREADS) {
      int64_t* out = p.out + (int64_t)b * R * T + lo + i;
      #pragma unroll 4
      for (int r = 0; r < R; ++r, out += T) {
        const int2 at = cut[r];
        const int beam = i <= at.x ? path[r * pitch + i] : 0;
        const int word = words[beam * pitch + i];
        *out = i <= at.x ? (int64_t)word : i == at.y ? p.eos : p.pad;
      }
    }
    __syncthreads();
  }
}

// What the current device says of a kernel, asked once.
template <typename T, bool SHORT>
struct Fit {
  int clusters[5];                       // resident clusters of 1, 2, 4, 8, 16 blocks
  static const Fit* get() {
    static std::atomic<const Fit*> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (const Fit* f = known[dev]) return f;
    Fit* f = new (std::nothrow) Fit;     // kept for the life of the process (a second thread may find the same again)
    if (!f) return nullptr;
    if (!resident_clusters((const void*)step_kernel<T, SHORT>, THREADS, 0, f->clusters)) { delete f; return nullptr; }
    known[dev] = f;
    return f;
  }
};

static int cluster_log2(int B, int K, int64_t bytes, const int (&clusters)[5]) {
  // The whole batch is resident; more blocks per sentence shorten its pass, 16 only where a slice would not fit a warp's
  // registers with 8 (a sentence of 4 x 32128 16-bit logits: 7.9 us with 8, 8.5 with 16; of 16 x 65537 float32: 26.7 and
  // 21.6) and one block per multiprocessor is enough.  A beam has two warps at least, for the number of groups that its
  // bound is taken from.
  int c = bytes > 8 * WARPS * 32 * 4 * 16 ? 4 : 3;
  while (c > (K > 8 ? 1 : 0) && (B > clusters[c] || (c == 4 && B * 16ll > 148))) --c;
  return c;
}

template <typename T, bool SHORT>
static int launch_blocks(const Params& p, cudaStream_t stream) {
  if (!Fit<T, SHORT>::get()) return T5B_ERR_LAUNCH;                      // (which allows the launch such clusters)
  const unsigned C = 1u << p.cluster_log2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.B * C); cfg.blockDim = dim3(THREADS); cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, step_kernel<T, SHORT>, p) == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}

template <typename T>
static int launch_step(Params p, cudaStream_t stream) {
  const auto* fit = Fit<T, false>::get();
  if (!fit) return T5B_ERR_LAUNCH;
  p.cluster_log2 = cluster_log2(p.B, p.K, (int64_t)p.K * p.V * sizeof(T), fit->clusters);
  p.S = (WARPS << p.cluster_log2) / p.K;
  p.unit_magic = (65536u + p.S - 1) / p.S; p.slice_magic = (uint32_t)(((1ull << 32) + p.S - 1) / p.S);
  return p.V / Pack<T>::N / p.S + 1 <= 16 ? launch_blocks<T, true>(p, stream) : launch_blocks<T, false>(p, stream);
}

}  // namespace beam
}  // namespace t5b

using namespace t5b;

extern "C" int t5b_beam_search_step(const t5b_beam_step_args* a, void* stream) {
  if (!a) return T5B_ERR_ARG;
  if (a->dtype != T5B_F32 && a->dtype != T5B_F16 && a->dtype != T5B_BF16) return T5B_ERR_DTYPE;
  if (a->B < 0 || a->num_beams < 1 || a->num_beams > beam::MAX_BEAMS || a->vocab < 2 || a->vocab > (1 << beam::TOKEN_BITS) ||
      a->B > (1 << 24)) return T5B_ERR_SHAPE;
  if (a->B == 0) return T5B_OK;
  if (!a->logits || !a->scores || !a->finished_scores || !a->finished_steps || !a->finished_beams || !a->done || !a->pos ||
      !a->tokens_out || !a->parents_out || !a->scores_out || !a->finished_scores_out || !a->finished_steps_out ||
      !a->finished_beams_out || !a->done_out) return T5B_ERR_ARG;
  if ((a->history_tokens != nullptr) != (a->history_parents != nullptr)) return T5B_ERR_ARG;
  if (!(a->length_penalty == a->length_penalty)) return T5B_ERR_ARG;
  if ((uintptr_t)a->logits % dtype_bytes(a->dtype)) return T5B_ERR_ALIGN;
  beam::Params p;
  p.logits = a->logits; p.row_stride = a->logits_stride;
  p.scores = a->scores; p.fin_scores = a->finished_scores; p.fin_steps = a->finished_steps; p.fin_beams = a->finished_beams;
  p.done = a->done; p.pos = a->pos;
  p.tokens_out = a->tokens_out; p.parents_out = a->parents_out; p.scores_out = a->scores_out;
  p.fin_scores_out = a->finished_scores_out; p.fin_steps_out = a->finished_steps_out;
  p.fin_beams_out = a->finished_beams_out; p.done_out = a->done_out;
  p.hist_tokens = a->history_tokens; p.hist_parents = a->history_parents; p.hist_steps = a->history_steps;
  p.B = a->B; p.K = a->num_beams; p.V = a->vocab; p.n = 2 * a->num_beams;
  p.eos = a->eos_token_id; p.pad = a->pad_token_id;
  p.length_penalty = a->length_penalty; p.early_stopping = a->early_stopping;
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case T5B_F32: return beam::launch_step<float>(p, st);
    case T5B_F16: return beam::launch_step<__half>(p, st);
    default: return beam::launch_step<__nv_bfloat16>(p, st);
  }
}

extern "C" int t5b_beam_search_sequences(const t5b_beam_sequences_args* a, void* stream) {
  if (!a) return T5B_ERR_ARG;
  if (a->B < 0 || a->num_beams < 1 || a->num_beams > beam::MAX_BEAMS || a->num_return < 1 || a->num_return > a->num_beams ||
      a->steps < 1) return T5B_ERR_SHAPE;
  if (a->B == 0) return T5B_OK;
  if (!a->tokens || !a->parents || !a->scores || !a->finished_scores || !a->finished_steps || !a->finished_beams || !a->done ||
      !a->sequences || !a->sequence_scores) return T5B_ERR_ARG;
  if (!(a->length_penalty == a->length_penalty)) return T5B_ERR_ARG;
  beam::SequenceParams p;
  p.tokens = a->tokens; p.parents = a->parents; p.scores = a->scores; p.fin_scores = a->finished_scores;
  p.fin_steps = a->finished_steps; p.fin_beams = a->finished_beams; p.done = a->done;
  p.out = a->sequences; p.out_scores = a->sequence_scores;
  p.T = a->steps; p.B = a->B; p.K = a->num_beams; p.R = a->num_return;
  p.eos = a->eos_token_id; p.pad = a->pad_token_id;
  p.length = pow((double)a->steps, a->length_penalty);
  for (p.k_log2 = 0; 1 << p.k_log2 < p.K;) ++p.k_log2;
  const int seg = a->steps < beam::SEGMENT ? a->steps : beam::SEGMENT, pitch = (seg + 31) / 32 * 32 + 4;
  const size_t smem = (size_t)p.K * pitch * 4 + ((size_t)(seg + beam::PIECES) << p.k_log2) + (size_t)p.R * pitch;
  if (smem > 32 * 1024) {
    constexpr int most = (beam::SEGMENT + 36) * 6 * beam::MAX_BEAMS;
    if (cudaFuncSetAttribute(beam::sequences_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return T5B_ERR_LAUNCH;
  }
  beam::sequences_kernel<<<(unsigned)p.B, beam::SEQ_THREADS, smem, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}
