// One step of beam search, and the sentences that its steps leave behind.
//
// The step, for the K beams of a sentence with running scores r[k] and logits x[k, :]:
//
//   lse[k]   = log sum_t exp(x[k, t])
//   s[k, t]  = r[k] + (x[k, t] - lse[k])
//   the 2K best (k, t): by s, then the lowest beam, then the largest logit, then the lowest token
//   -> those that end the sentence join the pool of finished sentences, the K best others go on.
//
// One cluster of blocks per sentence reads every logit once.  A warp owns a slice of one beam's row (a "unit") and
// keeps the slice's maximum and sum of exponentials; after one exchange over the cluster's shared memory every block
// knows lse[] and the maxima of all slices.  The n-th largest of those maxima (as scores) is a bound that n
// candidates reach, so only lanes whose own maximum reaches it look at their elements again: for n = 8 out of 128
// slices about nine candidates are left, and one block ranks them by counting.  Where the bound does not thin the
// candidates out (fewer finite ones than n, or hundreds of equal ones) every warp makes the sorted list of its slice's
// n best instead and one block merges the lists.  Sums of exponentials are float32 within a lane (a few dozen terms)
// and float64 from there on, as are the scores: two candidates of different beams are told apart to about 1e-8.
//
// The reference has no beam search of its own (its heads inherit it: src/turbot5/heads/t5_heads.py:100-130).
#include "t5b_common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace t5b {
namespace beam {

constexpr int WARPS = 16;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_UNITS = WARPS * MAX_CLUSTER;
constexpr int MAX_GROUPS = 128;          // maxima that the bound is taken from
constexpr int MAX_SURVIVORS = 256;
constexpr int MAX_BEAMS = 16;
constexpr int MAX_CAND = 2 * MAX_BEAMS;  // one candidate per lane in the end
constexpr int TOKEN_BITS = 27;
constexpr uint32_t TOKEN_MASK = (1u << TOKEN_BITS) - 1;

struct Params {
  const void* logits; int64_t row_stride;
  const float* scores; const float* fin_scores; const int32_t* fin_steps; const int32_t* fin_beams; const uint8_t* done;
  const int64_t* pos;
  int64_t* tokens_out; int32_t* parents_out; float* scores_out;
  float* fin_scores_out; int32_t* fin_steps_out; int32_t* fin_beams_out; uint8_t* done_out;
  int32_t* hist_tokens; int32_t* hist_parents; int64_t hist_steps;
  int32_t B, K, V, n, S;                 // n candidates; S slices per row
  int32_t groups;                        // maxima published per slice: 1 or 4
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

// A warp's slice of one row: 16-byte vectors [v0, v1) of the row's aligned middle; the first slice also has the
// elements before it, the last one those behind it (fewer than a vector each, one per lane).
template <typename T> struct Slice {
  const T* row; const uint4* mid;
  int v0, v1, head, tail, V;             // elements [0, head) and [tail, V) outside the vectors, if this slice has them
  __device__ __forceinline__ Slice(const T* r, int V_, int part, int S) : row(r), V(V_) {
    constexpr int N = Pack<T>::N;
    const int mis = (int)(((uintptr_t)r & 15) / sizeof(T));
    const int before = min(mis ? N - mis : 0, V_);
    const int nv = (V_ - before) / N;
    mid = (const uint4*)(r + before);
    v0 = (int)((int64_t)part * nv / S); v1 = (int)((int64_t)(part + 1) * nv / S);
    head = part == 0 ? before : 0;
    tail = part == S - 1 ? before + nv * N : V_;
    first = before;
  }
  int first;                             // element index of the first vector
  // f(logit, token) for every element of one lane; the same elements whichever lane of the warp asks
  template <typename F> __device__ __forceinline__ void each(int lane, F f) const {
    if (lane < head) f(to_float<T>(row[lane]), lane);
    if (tail + lane < V) f(to_float<T>(row[tail + lane]), tail + lane);
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 u = __ldg(mid + v);
      float x[Pack<T>::N];
      unpack<T>(u, x);
      #pragma unroll
      for (int e = 0; e < Pack<T>::N; ++e) f(x[e], first + v * Pack<T>::N + e);
    }
  }
};

__device__ __forceinline__ double warp_sum(double v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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
  insert(lane < sl.head ? make_key(beam, to_float<T>(sl.row[lane]), lane) : 0);
  insert(sl.tail + lane < sl.V ? make_key(beam, to_float<T>(sl.row[sl.tail + lane]), sl.tail + lane) : 0);
  for (int v = sl.v0; v < sl.v1; v += 32) {
    const bool in = v + lane < sl.v1;
    float x[Pack<T>::N];
    if (in) unpack<T>(__ldg(sl.mid + v + lane), x);
    #pragma unroll
    for (int e = 0; e < Pack<T>::N; ++e)
      insert(in ? make_key(beam, x[e], sl.first + (v + lane) * Pack<T>::N + e) : 0);
  }
  return mine;
}

struct Shared {
  double usum[MAX_UNITS];
  float umax[MAX_UNITS];
  float gmax[MAX_GROUPS];
  float gscore[MAX_GROUPS];
  Row rows[MAX_BEAMS];
  Cand found[MAX_SURVIVORS];
  Cand best[MAX_CAND];
  uint64_t lists[WARPS][32];
  Cand heads[WARPS];
  float bound;
  int count;
};

// What the step decides from its n best candidates, by one warp: lane i has candidate i (best first).
__device__ __forceinline__ void decide(const Params& p, const Cand* best, int b, int lane, double length) {
  const int K = p.K, n = p.n;
  const unsigned all = 0xffffffffu, below = (1u << lane) - 1;
  const int64_t at = (int64_t)b * K + lane;
  const bool valid = lane < n;
  const double score = valid ? best[lane].score : -INFINITY;
  const uint64_t key = valid ? best[lane].key : 0;
  const int token = valid ? key_token(key) : 0, beam = valid ? key_beam(key) : 0;
  const bool ends = valid && (int64_t)token == p.eos;
  // the pool: its entries and the ended candidates among the K best, larger first, earlier first among equals
  const bool joins = ends && lane < K && score > -INFINITY;
  float old = lane < K ? p.fin_scores[at] : -INFINITY;
  if (!(old == old)) old = -INFINITY;
  const int old_step = lane < K ? p.fin_steps[at] : 0, old_beam = lane < K ? p.fin_beams[at] : 0;
  const float fresh = joins ? (float)(score / length) : -INFINITY;
  const unsigned joining = __ballot_sync(all, joins);
  int old_rank = 0, new_rank = 0;
  for (int j = 0; j < K; ++j) {
    const float o = __shfl_sync(all, old, j);
    old_rank += o > old || (o == old && j < lane);
    new_rank += o >= fresh;
  }
  for (unsigned m = joining; m; m &= m - 1) {
    const int j = __ffs(m) - 1;
    const float o = __shfl_sync(all, fresh, j);
    old_rank += o > old;
    new_rank += o > fresh || (o == fresh && j < lane);
  }
  const int step = (int)(*p.pos);
  if (lane < K && old_rank < K) {
    const int64_t to = (int64_t)b * K + old_rank;
    p.fin_scores_out[to] = old; p.fin_steps_out[to] = old_step; p.fin_beams_out[to] = old_beam;
  }
  if (joins && new_rank < K) {
    const int64_t to = (int64_t)b * K + new_rank;
    p.fin_scores_out[to] = fresh; p.fin_steps_out[to] = step; p.fin_beams_out[to] = beam;
  }
  const unsigned worst_old = __ballot_sync(all, lane < K && old_rank == K - 1);
  const unsigned worst_new = __ballot_sync(all, joins && new_rank == K - 1);
  const float worst = worst_old ? __shfl_sync(all, old, __ffs(worst_old) - 1) : __shfl_sync(all, fresh, __ffs(worst_new) - 1);
  // the K best that go on: one continuation of a beam stays in its place, further ones take the free places in order
  const int order = __popc(__ballot_sync(all, valid && !ends) & below);
  const bool on = valid && !ends && order < K;
  const unsigned goes = __ballot_sync(all, on);
  const unsigned same = __match_any_sync(all, on ? beam : 64 + lane);
  const bool further = on && (same & below & goes) != 0;
  const unsigned again = __ballot_sync(all, further);
  const unsigned used = __reduce_or_sync(all, on ? 1u << beam : 0u);
  unsigned open = ~used & ((1u << K) - 1);
  int place = beam;
  if (further) {
    for (int skip = __popc(again & below); skip > 0; --skip) open &= open - 1;
    place = __ffs(open) - 1;
  }
  const float kept = (float)score;
  if (on && place >= 0) {
    const int64_t to = (int64_t)b * K + place;
    p.tokens_out[to] = token; p.parents_out[to] = beam; p.scores_out[to] = kept;
    if (p.hist_tokens && step >= 0 && step < p.hist_steps) {
      const int64_t h = (int64_t)step * p.B * K + to;
      p.hist_tokens[h] = token; p.hist_parents[h] = beam;
    }
  }
  const unsigned top = __reduce_max_sync(all, on ? ordered(kept) : 0u);
  const float highest = unordered(top);
  if (lane == 0) {
    bool full = worst > -INFINITY;
    if (!p.early_stopping) full = full && (double)worst >= (double)highest / length;
    p.done_out[b] = full || highest == -INFINITY;
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2)
step_kernel(const __grid_constant__ Params p) {
  __shared__ Shared sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int K = p.K, n = p.n, S = p.S, G = p.groups;
  const int64_t at = (int64_t)b * K;

  if (p.done[b]) {                       // the whole cluster: nothing changes any more
    if (rank == 0 && tid < K) {
      p.tokens_out[at + tid] = p.pad; p.parents_out[at + tid] = tid; p.scores_out[at + tid] = p.scores[at + tid];
      p.fin_scores_out[at + tid] = p.fin_scores[at + tid];
      p.fin_steps_out[at + tid] = p.fin_steps[at + tid]; p.fin_beams_out[at + tid] = p.fin_beams[at + tid];
      const int64_t step = *p.pos;
      if (p.hist_tokens && step >= 0 && step < p.hist_steps) {
        p.hist_tokens[(step * p.B + b) * K + tid] = (int32_t)p.pad; p.hist_parents[(step * p.B + b) * K + tid] = tid;
      }
      if (tid == 0) p.done_out[b] = 1;
    }
    return;
  }

  // ---- one pass over the logits: maximum and sum of exponentials of a slice
  const int unit = rank * WARPS + warp, k = unit / S;
  const bool active = k < K;
  const Slice<T> sl((const T*)p.logits + (at + (active ? k : 0)) * p.row_stride, p.V, active ? unit % S : 0, S);
  float m = -INFINITY;
  if (tid == 0) { sm.count = 0; sm.bound = -INFINITY; }
  if (active) {
    constexpr int N = Pack<T>::N, U = 4;
    float s = 0.f;
    auto add = [&](float x) {
      const float m_new = fmaxf(m, x);
      if (m_new > -INFINITY) { s = s * fast_exp2((m - m_new) * kLog2e) + fast_exp2((x - m_new) * kLog2e); m = m_new; }
      else if (!(x == x)) s = x;
    };
    if (lane < sl.head) add(to_float<T>(sl.row[lane]));
    if (sl.tail + lane < sl.V) add(to_float<T>(sl.row[sl.tail + lane]));
    for (int v = sl.v0 + lane; v < sl.v1; v += 32 * U) {
      uint4 u[U];
      #pragma unroll
      for (int i = 0; i < U; ++i)
        u[i] = v + 32 * i < sl.v1 ? __ldg(sl.mid + v + 32 * i) : make_uint4(Pack<T>::none, Pack<T>::none, Pack<T>::none, Pack<T>::none);
      float m_new = m;
      #pragma unroll
      for (int i = 0; i < U; ++i) {
        float x[N];
        unpack<T>(u[i], x);
        #pragma unroll
        for (int e = 0; e < N; ++e) m_new = fmaxf(m_new, x[e]);
      }
      const float ref = m_new > -INFINITY ? m_new : 0.f;
      s *= fast_exp2((m - ref) * kLog2e);
      m = m_new;
      #pragma unroll
      for (int i = 0; i < U; ++i) {
        float x[N];
        unpack<T>(u[i], x);
        #pragma unroll
        for (int e = 0; e < N; ++e) s += fast_exp2((x[e] - ref) * kLog2e);
      }
    }
    float gm = m;
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 1));
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 4));
    float wm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 8));
    wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 16));
    double total;
    if (__any_sync(0xffffffffu, !(s == s) || m == INFINITY)) {      // NaN or +inf among the logits
      double t = 0.0;
      sl.each(lane, [&](float x, int) {
        if (x == x) t += wm == INFINITY ? (x == INFINITY ? 1.0 : 0.0) : wm > -INFINITY ? (double)fast_exp2((x - wm) * kLog2e) : 0.0;
      });
      total = warp_sum(t);
    } else {
      total = warp_sum(wm > -INFINITY ? (double)(s * fast_exp2((m - wm) * kLog2e)) : 0.0);
    }
    if (lane < C) {
      Shared* to = cluster.map_shared_rank(&sm, lane);
      to->umax[unit] = wm; to->usum[unit] = total;
      if (G == 1) to->gmax[unit] = wm;
    }
    if (G == 4 && (lane & 7) == 0)
      for (int r = 0; r < C; ++r) cluster.map_shared_rank(&sm, r)->gmax[unit * 4 + lane / 8] = gm;
  }
  cluster.sync();

  // ---- every block: the rows' log-sums, then the bound that n candidates reach
  if (warp < K) {
    float rm = -INFINITY;
    for (int i = lane; i < S; i += 32) rm = fmaxf(rm, sm.umax[warp * S + i]);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) rm = fmaxf(rm, __shfl_xor_sync(0xffffffffu, rm, o));
    double t = 0.0;
    for (int i = lane; i < S; i += 32) {
      const float um = sm.umax[warp * S + i];
      if (um > -INFINITY) t += um == rm ? sm.usum[warp * S + i] : sm.usum[warp * S + i] * (double)fast_exp2((um - rm) * kLog2e);
    }
    if (rm == INFINITY) {                // only the slices that have it count
      t = 0.0;
      for (int i = lane; i < S; i += 32) if (sm.umax[warp * S + i] == INFINITY) t += sm.usum[warp * S + i];
    }
    t = warp_sum(t);
    if (lane == 0) {
      const float run = p.scores[at + warp];
      Row r;
      r.run = run; r.log_inf = 0.0; r.lse = 0.0;
      r.state = rm == -INFINITY || !(run > -INFINITY) ? 1 : rm == INFINITY ? 2 : 0;
      if (r.state == 0) r.lse = (double)rm + log(t);
      if (r.state == 2) r.log_inf = log(t);
      sm.rows[warp] = r;
    }
  }
  __syncthreads();
  const int groups = K * S * G;
  for (int g = tid; g < groups; g += THREADS)
    sm.gscore[g] = __double2float_rd(score_of(sm.rows[g / G / S], sm.gmax[g]));
  __syncthreads();
  for (int g = tid; g < groups; g += THREADS) {
    const float mine = sm.gscore[g];
    int above = 0;
    for (int j = 0; j < groups; ++j) {
      const float o = sm.gscore[j];
      above += o > mine || (o == mine && j < g);
    }
    if (above == n - 1) sm.bound = mine;
  }
  __syncthreads();
  const float bound = sm.bound;

  // ---- the candidates that reach the bound
  bool by_lists = !(bound > -INFINITY);
  Shared* lead = cluster.map_shared_rank(&sm, 0);
  if (!by_lists && active) {
    const Row r = sm.rows[k];
    if (score_of(r, m) >= (double)bound) {
      sl.each(lane, [&](float x, int token) {
        const double s = score_of(r, x);
        if (s >= (double)bound) {
          const int i = atomicAdd(&lead->count, 1);
          if (i < MAX_SURVIVORS) lead->found[i] = Cand{s, make_key(k, x, token)};
        }
      });
    }
  }
  cluster.sync();
  by_lists = by_lists || lead->count > MAX_SURVIVORS;

  if (by_lists) {
    if (active) sm.lists[warp][lane] = best_of_slice<T>(sl, k, n, lane);
    cluster.sync();
    if (rank == 0) {
      int next = 0;
      const bool has = tid < K * S;
      Cand mine{-INFINITY, 0};
      auto take = [&]() {
        mine.key = next < n ? cluster.map_shared_rank(&sm, tid / WARPS)->lists[tid % WARPS][next] : 0;
        mine.score = mine.key ? score_of(sm.rows[tid / S], key_logit(mine.key)) : -INFINITY;
      };
      if (has) take();
      for (int i = 0; i < n; ++i) {
        Cand top = mine;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const double os = __shfl_xor_sync(0xffffffffu, top.score, o);
          const uint64_t ok = __shfl_xor_sync(0xffffffffu, top.key, o);
          if (better(os, ok, top.score, top.key)) { top.score = os; top.key = ok; }
        }
        if (lane == 0) sm.heads[warp] = top;
        __syncthreads();
        top = sm.heads[0];
        #pragma unroll
        for (int w = 1; w < WARPS; ++w) if (better(sm.heads[w].score, sm.heads[w].key, top.score, top.key)) top = sm.heads[w];
        if (tid == 0) sm.best[i] = top;
        if (mine.key && mine.key == top.key) { ++next; take(); }
        __syncthreads();
      }
    }
  } else if (rank == 0) {
    const int found = sm.count;
    for (int i = tid; i < found; i += THREADS) {
      const Cand mine = sm.found[i];
      int above = 0;
      for (int j = 0; j < found; ++j) above += better(sm.found[j].score, sm.found[j].key, mine.score, mine.key);
      if (above < n) sm.best[above] = mine;
    }
    __syncthreads();
  }
  if (rank == 0 && warp == 0) {
    const double steps = (double)(*p.pos + 1);
    const double length = p.length_penalty == 1.0 ? steps : p.length_penalty == 0.0 ? 1.0 : pow(steps, p.length_penalty);
    decide(p, sm.best, b, lane, length);
  }
  cluster.sync();                        // nobody leaves while its shared memory is read
}

// ---- sentences from the history of tokens and parents -------------------------------------------------------------
//
// Walking back from the last token is a chain of dependent reads.  A block per sentence brings a segment of the parents
// into shared memory and cuts it into pieces: every piece is walked from each of its K possible beams at once, the
// pieces' results are chained per returned sentence, and the pieces are walked again from the beam that is now known.
constexpr int SEGMENT = 1024;            // steps in shared memory at a time
constexpr int SEQ_THREADS = 256;

struct SequenceParams {
  const int32_t* tokens; const int32_t* parents; const float* scores; const float* fin_scores;
  const int32_t* fin_steps; const int32_t* fin_beams; const uint8_t* done;
  int64_t* out; float* out_scores;
  int32_t T, B, K, R;
  int64_t eos, pad;
  double length;
};

__global__ void __launch_bounds__(SEQ_THREADS)
sequences_kernel(const __grid_constant__ SequenceParams p) {
  extern __shared__ uint8_t raw[];
  __shared__ int last[MAX_BEAMS], from[MAX_BEAMS], cur[MAX_BEAMS];
  __shared__ bool ended[MAX_BEAMS], none[MAX_BEAMS];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const int K = p.K, R = p.R, T = p.T;
  const int seg = min(SEGMENT, T);
  uint8_t* par = raw;                    // [seg][K]
  uint8_t* path = par + seg * K;         // [R][seg]
  uint8_t* jump = path + seg * R;        // [pieces][K], pieces <= 32

  if (tid < 32) {
    // candidates: lanes [0, K) the pool, [K, 2K) the running beams
    const int64_t at = (int64_t)b * K;
    float v = -INFINITY;
    if (lane < K) v = p.fin_scores[at + lane];
    else if (lane < 2 * K && !p.done[b]) v = (float)((double)p.scores[at + lane - K] / p.length);
    if (!(v == v)) v = -INFINITY;
    int above = 0;
    for (int j = 0; j < 2 * K; ++j) {
      const float o = __shfl_sync(0xffffffffu, v, j);
      above += o > v || (o == v && j < lane);
    }
    if (lane < 2 * K && above < R) {
      const bool e = lane < K;
      ended[above] = e; none[above] = v == -INFINITY;
      // an ended sentence's end token stands at its step, its beams are those up to the step before
      last[above] = e ? min(max(p.fin_steps[at + lane], 0), T - 1) : T - 1;
      from[above] = e ? min(max(p.fin_beams[at + lane], 0), K - 1) : lane - K;
      p.out_scores[(int64_t)b * R + above] = v;
    }
  }
  __syncthreads();
  if (tid < R) cur[tid] = 0;
  for (int hi = T; hi > 0; hi -= seg) {
    const int lo = max(0, hi - seg), len = hi - lo;
    // par[i]: the beam at step lo + i - 1 of each beam at step lo + i
    for (int i = tid; i < len * K; i += SEQ_THREADS) {
      const int t = lo + i / K, x = i % K;
      par[i] = (uint8_t)min(max(p.parents[((int64_t)t * p.B + b) * K + x], 0), K - 1);
    }
    __syncthreads();
    const int piece = (len + 31) / 32, pieces = (len + piece - 1) / piece;
    for (int i = tid; i < pieces * K; i += SEQ_THREADS) {
      const int c = i / K;
      int x = i % K;
      for (int j = min((c + 1) * piece, len) - 1; j >= c * piece; --j) x = par[j * K + x];
      jump[i] = (uint8_t)x;
    }
    __syncthreads();
    // entry beam of every piece per sentence (kept in path's last step of the piece), backwards
    if (tid < R) {
      const int stop = ended[tid] ? last[tid] - 1 : last[tid];
      int x = cur[tid];
      for (int c = pieces - 1; c >= 0; --c) {
        const int a = c * piece, z = min(a + piece, len) - 1;
        path[tid * seg + z] = (uint8_t)x;
        if (lo + a > stop) continue;                     // the sentence ends before this piece
        if (lo + z >= stop) {                            // ... inside it: walked step by step
          x = from[tid];
          for (int j = stop - lo; j >= a; --j) x = par[j * K + x];
        } else {
          x = jump[c * K + x];
        }
      }
      cur[tid] = x;
    }
    __syncthreads();
    for (int i = tid; i < R * pieces; i += SEQ_THREADS) {
      const int r = i / pieces, c = i % pieces, a = c * piece, z = min(a + piece, len) - 1;
      const int stop = ended[r] ? last[r] - 1 : last[r];
      int x = path[r * seg + z], j = z;
      if (lo + z >= stop) { j = min(z, stop - lo); x = from[r]; }
      for (; j >= a; --j) { path[r * seg + j] = (uint8_t)x; x = par[j * K + x]; }
    }
    __syncthreads();
    for (int i = tid; i < R * len; i += SEQ_THREADS) {
      const int r = i / len, t = lo + i % len;
      int64_t word = p.pad;
      if (!none[r]) {
        if (ended[r] && t == last[r]) word = p.eos;
        else if (t <= last[r]) word = p.tokens[((int64_t)t * p.B + b) * K + path[r * seg + t - lo]];
      }
      p.out[((int64_t)b * R + r) * T + t] = word;
    }
    __syncthreads();
  }
}

static int cluster_blocks(int B) {
  // A block per multiprocessor and a half keeps the whole batch resident; more blocks per sentence shorten its pass.
  int C = MAX_CLUSTER;
  while (C > 1 && (long long)B * C > 2 * 148) C /= 2;
  return C;
}

template <typename T>
static int launch_step(Params p, cudaStream_t stream) {
  const int C = cluster_blocks(p.B);
  p.S = C * WARPS / p.K;
  p.groups = C * WARPS <= 32 ? 4 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * C)); cfg.blockDim = dim3(THREADS); cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, step_kernel<T>, p) == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
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
  p.B = a->B; p.K = a->num_beams; p.V = a->vocab; p.n = 2 * a->num_beams; p.S = 1; p.groups = 1;
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
  const int seg = a->steps < beam::SEGMENT ? a->steps : beam::SEGMENT;
  const size_t smem = (size_t)seg * (p.K + p.R) + 32 * p.K;
  beam::sequences_kernel<<<(unsigned)p.B, beam::SEQ_THREADS, smem, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}
