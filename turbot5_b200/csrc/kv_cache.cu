// Decoder caches: keys and values into 8-bit blocks, and the reordering of beams.
//
// An 8-bit cache holds e4m3 numbers (B, H, capacity, D) and one float32 scale per 64 tokens and head, a power of two:
//
//   scale = the smallest 2^e with max |x| <= 448 * 2^e  (-100 <= e <= 120),   stored = round_e4m3(x / scale)
//
// With a power of two the division is exact, so one rounding of three mantissa bits is all that is lost, and tokens that
// join a block with a larger scale move the older ones by whole exponents: nothing is rounded twice unless it falls
// below the smallest normal number of the format.
//
// The reference keeps its cache in the model's type and reorders it with index_select per tensor
// (src/turbot5/model/attentions.py:198,229-234; src/turbot5/heads/t5_heads.py:100-130 inherits the generation loop).
#include "t5b_common.cuh"

#include <type_traits>

namespace t5b {
namespace kvcache {

constexpr int BLOCK = T5B_CACHE_BLOCK;
constexpr int LOWEST = -100, HIGHEST = 120;

// two floats -> two e4m3 numbers, nearest even, saturating (NaN stays NaN)
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// exponent of the scale for a block whose largest finite magnitude has these bits
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  // |x| = 1.f * 2^e; 448 = 1.75 * 2^8: one more where 1.f > 1.75 (below the normal numbers the clamp decides)
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, LOWEST), HIGHEST);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

struct FillParams {
  const void* src[2]; uint8_t* cache[2]; float* scale[2];
  int64_t src_b[2], src_h[2], src_m[2];       // element strides
  int64_t cache_b[2], cache_h[2], scale_b[2], scale_h[2];
  const int64_t* start_ptr; int64_t start;
  const int32_t* seqlens;
  int32_t B, H, M, cap;
  int32_t aligned[2];                         // 8 elements of a row start on 16 bytes
};

// Eight consecutive elements of a row as they stand in memory.
template <typename T> struct Piece {
  static constexpr int WORDS = 2 * sizeof(T);
  uint32_t w[WORDS];
  __device__ __forceinline__ void zero() {
    #pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p, bool aligned) {
    if (aligned) {
      #pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 u = __ldg((const uint4*)p + i);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else if constexpr (sizeof(T) == 4) {
      #pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(p[i]);
    } else {
      const uint16_t* e = (const uint16_t*)p;
      #pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    }
  }
  // Largest magnitude so far, as bits without their sign, two 16-bit numbers side by side where T is one.
  __device__ __forceinline__ uint32_t largest(uint32_t most) const {
    #pragma unroll
    for (int i = 0; i < WORDS; ++i)
      if constexpr (sizeof(T) == 4) most = max(most, w[i] & 0x7fffffffu);
      else most = __vmaxu2(most, w[i] & 0x7fff7fffu);
    return most;
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
      else if constexpr (std::is_same<T, __nv_bfloat16>::value) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      else x[i] = i & 1 ? __high2float(*reinterpret_cast<const __half2*>(&w[i / 2])) : __low2float(*reinterpret_cast<const __half2*>(&w[i / 2]));
    }
  }
};
// the larger of a word's numbers as the bits of a float
template <typename T> __device__ __forceinline__ uint32_t as_float_bits(uint32_t most) {
  if constexpr (sizeof(T) == 4) return most;
  const uint32_t m = max(most >> 16, most & 0xffffu);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}
__device__ __forceinline__ uint32_t magnitude(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;            // infinities saturate, NaN stays NaN: neither sets a scale
}
__device__ __forceinline__ uint2 pack8(const float (&x)[8], float inv) {
  float y[8];
  #pragma unroll
  for (int i = 0; i < 8; i += 2) mul2(y[i], y[i + 1], x[i], x[i + 1], inv, inv);
  return make_uint2(to_e4m3x2(y[0], y[1]) | to_e4m3x2(y[2], y[3]) << 16, to_e4m3x2(y[4], y[5]) | to_e4m3x2(y[6], y[7]) << 16);
}
__device__ __forceinline__ uint2 rescale8(uint2 v, float f) {
  const float2 a = from_e4m3x2(v.x & 0xffffu), b = from_e4m3x2(v.x >> 16), c = from_e4m3x2(v.y & 0xffffu), d = from_e4m3x2(v.y >> 16);
  const float x[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  return pack8(x, f);
}

// A team of TEAM threads fills one block of 64 tokens of one head, keys or values.  TEAM 128 for prompts: every thread
// holds its share of the block between the search for the largest and the rounding (one read of the source), as packed
// as it came: magnitudes are compared as whole numbers, two at a time, which leaves 3.5 instructions per element (12 with
// floats throughout): 11.2 us for 53 MB instead of 22.8, and 805 MB at the measured copy rate (119 us).  TEAM 32 for
// single tokens: a warp has one row to write, four heads share a block of threads.
template <typename T, int D, int TEAM>
__global__ void __launch_bounds__(128)
fill_kernel(const __grid_constant__ FillParams p) {
  constexpr int PARTS = D / 8;                                     // 8-element pieces of a row
  constexpr int PER = TEAM == 32 ? 1 : BLOCK * PARTS / TEAM;       // pieces per thread
  constexpr int TOKENS = TEAM == 32 ? 1 : TEAM / PARTS;            // tokens from one of a thread's pieces to the next
  __shared__ uint32_t largest[4];
  const int lane = threadIdx.x % TEAM;
  const int head = TEAM == 32 ? blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x;
  const int b = blockIdx.z >> 1, kv = blockIdx.z & 1;
  if (TEAM == 32 && head >= p.H) return;                           // whole warps
  const int64_t start = p.start_ptr ? *p.start_ptr : p.start;
  const int count = p.seqlens ? min(max(p.seqlens[b], 0), p.M) : p.M;
  if (start < 0 || start >= p.cap) return;
  const int64_t end = min(start + (int64_t)count, (int64_t)p.cap);
  const int64_t first = (start / BLOCK + blockIdx.y) * BLOCK;      // the block's first token
  const int64_t begin = first > start ? first : start;
  if (begin >= end) return;                                        // the same for the whole team
  // within the block, the written tokens are [lo, hi)
  const int lo = (int)(begin - first), hi = (int)min(end - first, (int64_t)BLOCK);
  const int token = (TEAM == 32 ? lo : 0) + lane / PARTS, part = lane % PARTS * 8;
  const T* src = (const T*)p.src[kv] + (int64_t)b * p.src_b[kv] + (int64_t)head * p.src_h[kv] + (first - start + token) * p.src_m[kv] + part;
  uint8_t* cache = p.cache[kv] + (int64_t)b * p.cache_b[kv] + (int64_t)head * p.cache_h[kv] + first * D;
  float* scale = p.scale[kv] + (int64_t)b * p.scale_b[kv] + (int64_t)head * p.scale_h[kv] + first / BLOCK;
  const bool kept = lo > 0;                                        // older tokens share the block
  const float was = kept ? *scale : 0.f;

  Piece<T> x[PER];
  #pragma unroll
  for (int i = 0; i < PER; ++i) {
    x[i].zero();
    const int t = token + i * TOKENS;
    if (TEAM == 32 ? lane < PARTS : t >= lo && t < hi) x[i].load(src + (int64_t)i * TOKENS * p.src_m[kv], p.aligned[kv]);
  }
  uint32_t words = 0;
  #pragma unroll
  for (int i = 0; i < PER; ++i) words = x[i].largest(words);
  uint32_t most = as_float_bits<T>(words);
  if (most >= 0x7f800000u) {                                       // infinities or NaN: without them
    most = 0;
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
      float f[8];
      x[i].floats(f);
      #pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, magnitude(f[j]));
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (TEAM > 32) {
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x / 32] = most;
    __syncthreads();
    most = max(max(largest[0], largest[1]), max(largest[2], largest[3]));
  }
  const float now = fmaxf(pow2(scale_exponent(most)), was);
  const float inv = 1.f / now;
  if (kept && now > was) {
    // the older tokens follow to the larger scale
    const float f = was * inv;
    for (int i = lane; i < lo * PARTS; i += TEAM) {
      uint2* at = (uint2*)cache + i;
      *at = rescale8(*at, f);
    }
  }
  #pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = token + i * TOKENS;
    if (TEAM == 32 ? lane < PARTS : t >= lo && t < hi) {
      float f[8];
      x[i].floats(f);
      *(uint2*)(cache + t * D + part) = pack8(f, inv);
    }
  }
  if (kept) { if (TEAM == 32) __syncwarp(); else __syncthreads(); }  // every thread has read the old scale
  if (lane == 0) *scale = now;
}

// ---- reordering of beams -------------------------------------------------------------------------------------------
//
// Bound by the bytes of the beams that change.  A thread owns offsets of all beams of a sentence: it loads what the
// changed beams are to become, then stores it, so the caches are permuted in place without a second copy and without
// ordering between threads, whatever the parents are.  Beams that stay are neither read nor written, nor is what lies
// behind the tokens in use; all layers are one launch.  Two offsets at a time with four beams keep 64 registers and 32
// warps: 96.0 us for 590 MB, 94 % of the measured copy rate (one offset at a time 114, four with two blocks per
// multiprocessor 104, four with three spill in the loop: 120).
//
// How much of a cache is in use is known on the device only, so the grid is made for its capacity and a block that finds
// nothing costs as much as one that moves 16 KB: heads share a few hundred blocks, each of which takes piece after piece,
// and short heads get blocks of 64 threads.  16 beams of 104 of 470 tokens (92 MB): 24 us, 77 with a block per piece; 3
// beams of 37 of 229 tokens in 24 layers (65 MB): 19 and 40.
constexpr int REORDER_THREADS = 2 * 148 * 256;             // (148 multiprocessors) beyond these a block takes several pieces

constexpr int in_flight(int beams) { return beams == 16 ? 1 : 2; }

struct ReorderGroup {
  void* base[T5B_REORDER_MAX_TENSORS];
  int64_t outer_b, row_b, head_b;       // byte strides of dims 0, 1, 2
  int32_t n, outer;                     // tensors; dim 0
};
struct ReorderParams {
  ReorderGroup g[2];
  const int32_t* parents; const int32_t* seqlens;
  int32_t K, H, cap, units, chunks;     // units per token; blocks per head
};

// One offset of all beams at a time, UN of them in flight: `at(i)` is the i-th offset's address in the first beam.
template <typename U, int KM, int UN, int THREADS, typename F>
__device__ __forceinline__ void move_beams(int first, int total, int64_t row_b, const int (&parent)[KM], uint32_t changed, F at) {
  U v[UN][KM];
  #pragma unroll
  for (int u = 0; u < UN; ++u) {
    const int i = first + u * THREADS;
    if (i < total) {
      const char* from = at(i);
      #pragma unroll
      for (int j = 0; j < KM; ++j)
        if (changed >> j & 1) v[u][j] = *(const U*)(from + (int64_t)parent[j] * row_b);
    }
  }
  #pragma unroll
  for (int u = 0; u < UN; ++u) {
    const int i = first + u * THREADS;
    if (i < total) {
      char* to = at(i);
      #pragma unroll
      for (int j = 0; j < KM; ++j)
        if (changed >> j & 1) *(U*)(to + (int64_t)j * row_b) = v[u][j];
    }
  }
}

// A block has UN units a thread of one head's tokens, or some times as many, or all scales of one tensor (blocks behind
// those of the caches).
template <typename U, int KM, int THREADS>
__global__ void __launch_bounds__(THREADS, (KM == 4 ? 4 : KM == 8 ? 3 : 2) * 256 / THREADS)
reorder_kernel(const __grid_constant__ ReorderParams p) {
  constexpr int UN = in_flight(KM);
  const int b = blockIdx.y, K = p.K, tid = threadIdx.x;
  int parent[KM], len = 0;
  uint32_t changed = 0;
  #pragma unroll
  for (int j = 0; j < KM; ++j) {
    parent[j] = j;
    if (j < K) {
      const int q = p.parents[(int64_t)b * K + j];
      if (p.seqlens) len = max(len, p.seqlens[(int64_t)b * K + j]);
      if (q >= 0 && q < K && q != j) { parent[j] = q; changed |= 1u << j; }
    }
  }
  if (!changed) return;
  len = p.seqlens ? min(len, p.cap) : p.cap;
  const int blocks = p.g[0].n * p.g[0].outer * p.H * p.chunks;
  if ((int)blockIdx.x < blocks) {
    const ReorderGroup& g = p.g[0];
    const int chunk = blockIdx.x % p.chunks, rest = blockIdx.x / p.chunks, h = rest % p.H, z = rest / p.H;
    char* base = (char*)g.base[z / g.outer] + (int64_t)(z % g.outer) * g.outer_b + (int64_t)b * K * g.row_b + (int64_t)h * g.head_b;
    const int total = len * p.units;
    #pragma unroll 1
    for (int i = chunk * THREADS * UN + tid; i < total; i += p.chunks * THREADS * UN)
      move_beams<U, KM, UN, THREADS>(i, total, g.row_b, parent, changed, [&](int k) { return base + (int64_t)k * sizeof(U); });
  } else {
    const ReorderGroup& g = p.g[1];
    const int z = blockIdx.x - blocks, per_head = (len + BLOCK - 1) / BLOCK, total = per_head * p.H;
    char* base = (char*)g.base[z / g.outer] + (int64_t)(z % g.outer) * g.outer_b + (int64_t)b * K * g.row_b;
    for (int i = tid; i < total; i += THREADS * UN)
      move_beams<uint32_t, KM, UN, THREADS>(i, total, g.row_b, parent, changed, [&](int k) {
        const int h = k / per_head;
        return base + (int64_t)h * g.head_b + (int64_t)(k - h * per_head) * 4;
      });
  }
}

template <typename U, int KM, int THREADS>
static int launch_reorder(ReorderParams& p, int B, cudaStream_t stream) {
  constexpr int CHUNK = THREADS * in_flight(KM);
  const int64_t units = (int64_t)p.cap * p.units;
  if constexpr (THREADS > 64)
    if (units <= CHUNK / 2) return launch_reorder<U, KM, 64>(p, B, stream);
  // as many blocks as the whole capacity needs, but not more than some rounds of them: the tokens in use are known on the
  // device only
  const int64_t heads = (int64_t)p.g[0].n * p.g[0].outer * p.H, most = REORDER_THREADS / THREADS / (heads * B);
  const int64_t chunks = (units + CHUNK - 1) / CHUNK;
  p.chunks = (int)(most < 1 ? 1 : chunks < most ? chunks : most);
  const int64_t blocks = heads * p.chunks + (int64_t)p.g[1].n * p.g[1].outer;
  if (blocks > 0x7fffffffll || units > 0x7fffffffll - (1 << 24)) return T5B_ERR_SHAPE;
  reorder_kernel<U, KM, THREADS><<<dim3((unsigned)blocks, (unsigned)B), THREADS, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}

template <typename U>
static int launch_reorder_beams(ReorderParams& p, int B, cudaStream_t stream) {
  if (p.K <= 4) return launch_reorder<U, 4, 256>(p, B, stream);
  if (p.K <= 8) return launch_reorder<U, 8, 256>(p, B, stream);
  return launch_reorder<U, 16, 256>(p, B, stream);
}

template <typename T, int D>
static int launch_fill(const FillParams& p, cudaStream_t stream) {
  if (p.M == 1) {
    fill_kernel<T, D, 32><<<dim3((p.H + 3) / 4, 1, 2 * p.B), 128, 0, stream>>>(p);
  } else {
    const int blocks = (p.M + BLOCK - 2) / BLOCK + 1;      // wherever the first token stands in its block
    fill_kernel<T, D, 128><<<dim3(p.H, blocks, 2 * p.B), 128, 0, stream>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}

template <typename T>
static int launch_fill_d(const FillParams& p, int D, cudaStream_t stream) {
  switch (D) {
    case 16: return launch_fill<T, 16>(p, stream);
    case 32: return launch_fill<T, 32>(p, stream);
    case 64: return launch_fill<T, 64>(p, stream);
    case 128: return launch_fill<T, 128>(p, stream);
  }
  return T5B_ERR_HEAD_DIM;
}

}  // namespace kvcache
}  // namespace t5b

using namespace t5b;

extern "C" int t5b_cache_quantize(const t5b_cache_quantize_args* a, void* stream) {
  if (!a) return T5B_ERR_ARG;
  if (a->dtype != T5B_F32 && a->dtype != T5B_F16 && a->dtype != T5B_BF16) return T5B_ERR_DTYPE;
  if (a->D != 16 && a->D != 32 && a->D != 64 && a->D != 128) return T5B_ERR_HEAD_DIM;
  if (a->B < 0 || a->H < 0 || a->M < 0 || a->capacity < 0 || a->capacity % T5B_CACHE_BLOCK || a->B > 32767 || a->H > 65535 ||
      a->M > 65534 * T5B_CACHE_BLOCK + 1) return T5B_ERR_SHAPE;
  if (!a->start_ptr && a->start < 0) return T5B_ERR_ARG;
  if (a->B == 0 || a->H == 0 || a->M == 0) return T5B_OK;
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale) return T5B_ERR_ARG;
  if (!a->start_ptr && a->start > (int64_t)a->capacity - a->M) return T5B_ERR_SHAPE;
  const int es = dtype_bytes(a->dtype);
  kvcache::FillParams p;
  p.src[0] = a->k; p.src[1] = a->v;
  p.cache[0] = (uint8_t*)a->k_cache; p.cache[1] = (uint8_t*)a->v_cache;
  p.scale[0] = a->k_scale; p.scale[1] = a->v_scale;
  p.src_b[0] = a->k_stride_b; p.src_h[0] = a->k_stride_h; p.src_m[0] = a->k_stride_m;
  p.src_b[1] = a->v_stride_b; p.src_h[1] = a->v_stride_h; p.src_m[1] = a->v_stride_m;
  for (int i = 0; i < 2; ++i) {
    p.cache_b[i] = a->cache_stride_b; p.cache_h[i] = a->cache_stride_h;
    p.scale_b[i] = a->scale_stride_b; p.scale_h[i] = a->scale_stride_h;
    if ((uintptr_t)p.src[i] % es) return T5B_ERR_ALIGN;
    p.aligned[i] = (uintptr_t)p.src[i] % 16 == 0 && p.src_b[i] * es % 16 == 0 && p.src_h[i] * es % 16 == 0 && p.src_m[i] * es % 16 == 0;
    if ((uintptr_t)p.cache[i] % 16 || (uintptr_t)p.scale[i] % 4) return T5B_ERR_ALIGN;
  }
  if (a->cache_stride_b % 16 || a->cache_stride_h % 16) return T5B_ERR_ALIGN;
  p.start_ptr = a->start_ptr; p.start = a->start; p.seqlens = a->seqlens;
  p.B = a->B; p.H = a->H; p.M = a->M; p.cap = a->capacity;
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case T5B_F32: return kvcache::launch_fill_d<float>(p, a->D, st);
    case T5B_F16: return kvcache::launch_fill_d<__half>(p, a->D, st);
    default: return kvcache::launch_fill_d<__nv_bfloat16>(p, a->D, st);
  }
}

extern "C" int t5b_beam_cache_reorder(const t5b_cache_reorder_args* a, void* stream) {
  if (!a) return T5B_ERR_ARG;
  if (a->B < 0 || a->num_beams < 1 || a->num_beams > 16 || a->H < 0 || a->capacity < 0 || a->outer < 0 || a->n_caches < 0 ||
      a->n_scales < 0 || a->token_bytes < 1 || a->n_caches > T5B_REORDER_MAX_TENSORS || a->n_scales > T5B_REORDER_MAX_TENSORS ||
      a->B > 65535 || (int64_t)(a->n_caches + a->n_scales) * a->outer > 65535) return T5B_ERR_SHAPE;
  if (a->B == 0 || a->H == 0 || a->capacity == 0 || a->outer == 0 || a->n_caches + a->n_scales == 0) return T5B_OK;
  if (!a->parents || a->n_caches == 0) return T5B_ERR_ARG;         // scales go with their caches: heads set the grid
  kvcache::ReorderParams p;
  kvcache::ReorderGroup& c = p.g[0];
  kvcache::ReorderGroup& s = p.g[1];
  uint64_t all = (uint64_t)(a->cache_stride_outer | a->cache_stride_row | a->cache_stride_head | a->token_bytes);
  for (int i = 0; i < a->n_caches; ++i) {
    if (!a->caches[i]) return T5B_ERR_ARG;
    c.base[i] = a->caches[i];
    all |= (uint64_t)(uintptr_t)a->caches[i];
  }
  uint64_t sall = (uint64_t)(a->scale_stride_outer | a->scale_stride_row | a->scale_stride_head);
  for (int i = 0; i < a->n_scales; ++i) {
    if (!a->scales[i]) return T5B_ERR_ARG;
    s.base[i] = a->scales[i];
    sall |= (uint64_t)(uintptr_t)a->scales[i];
  }
  if (a->n_scales && sall % 4) return T5B_ERR_ALIGN;
  const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;     // whole units on every way through the strides
  c.outer_b = a->cache_stride_outer; c.row_b = a->cache_stride_row; c.head_b = a->cache_stride_head;
  c.n = a->n_caches; c.outer = a->outer;
  s.outer_b = a->scale_stride_outer; s.row_b = a->scale_stride_row; s.head_b = a->scale_stride_head;
  s.n = a->n_scales; s.outer = a->outer;
  p.parents = a->parents; p.seqlens = a->seqlens;
  p.K = a->num_beams; p.H = a->H; p.cap = a->capacity; p.units = a->token_bytes / unit;
  cudaStream_t st = (cudaStream_t)stream;
  if (unit == 16) return kvcache::launch_reorder_beams<uint4>(p, a->B, st);
  if (unit == 4) return kvcache::launch_reorder_beams<uint32_t>(p, a->B, st);
  return kvcache::launch_reorder_beams<uint8_t>(p, a->B, st);
}
