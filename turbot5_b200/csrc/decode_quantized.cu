// Decoding against an 8-bit cache: a few query rows per (batch, head), keys and values as e4m3 numbers with one
// power-of-two scale per 64 tokens and head.
//
//   out = softmax(sm_scale * q (K * s_K)^T + table[bucket(n - position), h] (+ causal mask)) (V * s_V)
//
// Bound by the bytes of the cache, half of a 16-bit one: at 6.5 TB/s a multiprocessor has to take in 23 numbers per
// clock, each of which has to be widened and multiplied.  Doing that in float32 would take 2.5 instructions per number
// and query row; here one conversion per two numbers makes fp16 pairs and the warp-wide m16n8k16 product does the rest
// for up to eight rows at the cost of one.  (The tensor unit is idle for 95 % of the time; its larger forms would need
// the same conversion.  Widening by integer shifts instead of the conversion unit measured 4 to 9 % slower.)
//
//   * S^T = K Q^T: the keys are the rows of the product.  A lane's 16 bytes of a key are four k-steps of the A operand
//     as they stand (the order of the head dim inside a k-step is free, the queries are read in the same order).
//   * O^T = V^T P^T: the head dim is the rows.  A byte permute joins two keys' bytes to pairs along the key dim.  Which
//     key is which row of a 16-key tile is free as well: the order is such that reading values has no bank conflicts.
//   * P^T comes out of S^T's registers by one 8x8 transpose of 16-bit pairs.
//   * fp16 products of e4m3 numbers are exact in float32; a row of q is scaled by a power of two to 2^15 at most, which holds
//     bf16 exactly down to 2^-31 of the row's largest element (fp16 2^-28), and to 2^-39 of it below.  P is carried as hi + lo:
//     with up to four rows, row r has columns 2r and 2r + 1 of the product, one for each half (a lane then makes the
//     weights of one row only); with up to eight rows the product is issued twice.  An item's weights are made relative to
//     its own largest one, which is 2^14: hi + lo then hold 22 bits of every weight down to 2^-17 of that, and 2^-39 of it
//     below.  (Relative to a running maximum of 1 the weights of a long faint tail behind one leading key fell among fp16's
//     subnormal numbers: up to 2e-3 of the result at 2^-15, all of it below 2^-25.)
//
// A warp works on items of 32 or 64 keys of one block of 64 (so an item has one scale), with its own running maximum and
// sum and its own ring of stages in shared memory that asynchronous copies fill ahead (registers alone held too little in
// flight: 206 us for 1.07 GB, 166 with the ring, the floor at the measured copy rate 164).  That is at 1965 MHz, in bursts
// of some milliseconds.  A second of it draws the 1000 W that the GPU may take, and with the clock at 1450 MHz it takes 188
// us, 193 as calls one behind the other (half of the issue slots are taken).  Warps merge in shared memory, the blocks
// of a (batch, head) that share a long cache form a cluster and merge through distributed shared memory: no workspace,
// no counters, no second launch.  The bias is looked up for items within the largest distance of a query only, from a
// table of the item's distances that the warp makes for itself.
//
// Semantics: the cached step of T5Attention.forward (src/turbot5/model/attentions.py:198,229-234), the merge rule of
// src/turbot5/ops/flash_decoding.py:47-55, as in decode.cu.
#include "t5b_common.cuh"

#include <cooperative_groups.h>

#include <atomic>
#include <new>

namespace cg = cooperative_groups;

namespace t5b {
namespace decq {

constexpr int BLOCK = T5B_CACHE_BLOCK;
constexpr float LOWEST = -3.402823466e38f;   // where a running maximum starts: finite, so that differences from it are numbers
// 16-key tiles of an item, and how its stages lie in shared memory: keys, values, two scales
template <int D> struct Ring {
  static constexpr int SUB = D == 128 ? 2 : D == 64 ? 2 : 4;
  static constexpr int STAGES = D == 128 ? 2 : 3;
  static constexpr int ITEM = SUB * 16;
  static constexpr int BYTES = 2 * ITEM * D + 16;
  static constexpr int WARP_BYTES = STAGES * BYTES;
};

struct Params {
  const void* q; const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale; void* out;
  const void* table; const int32_t* seqlens_k;
  int64_t q_stride_b, q_stride_h, q_stride_m;
  int64_t k_stride_b, k_stride_h, v_stride_b, v_stride_h;
  int64_t ks_stride_b, ks_stride_h, vs_stride_b, vs_stride_h;
  int64_t o_stride_b, o_stride_h, o_stride_m;
  int64_t table_stride0;
  int32_t table_dtype, B, H, M, N, causal, q_pos_offset, row_groups, q_aligned;
  float scale_log2;
};

// four e4m3 numbers -> two fp16 pairs
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void copy_async16(uint32_t to, const void* from, bool in) {   // zeros where `in` is false
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// BYTES consecutive bytes of a row in shared memory into words
template <int BYTES> __device__ __forceinline__ void read_bytes(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES == 2) {
    w[0] = *(const uint16_t*)p;
  } else if constexpr (BYTES == 4) {
    w[0] = *(const uint32_t*)p;
  } else if constexpr (BYTES == 8) {
    const uint2 u = *(const uint2*)p;
    w[0] = u.x; w[1] = u.y;
  } else {
    #pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 u = *(const uint4*)(p + 64 * i);
      w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
    }
  }
}

// Element of the head dim that lane c holds as element e (0 .. 3) of k-step j of the first product.
template <int D> __device__ __forceinline__ int dim_of(int c, int j, int e) {
  return D == 128 ? j / 4 * 64 + 16 * c + 4 * (j & 3) + e : D / 4 * c + 4 * j + e;
}

// TILES 1: up to four rows, each with two columns of the products (hi and lo of its weights).  TILES 2: up to eight rows,
// a column each, the second product twice.
template <typename T, int D, int TILES, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, TILES == 1 && D <= 64 ? 16 / WARPS : 1)
decode_quantized_kernel(const __grid_constant__ Params p, const __grid_constant__ BucketSpec spec) {
  using R = Ring<D>;
  constexpr int THREADS = WARPS * 32;
  constexpr int ROWS = 4 * TILES;
  constexpr int KSTEPS = D / 16;         // k-steps of S^T, 16-row tiles of O^T
  constexpr int KB = D / 4, VB = D / 8;  // bytes of a key / value row that a lane holds
  constexpr int KW = KB / 4, VW = (VB + 3) / 4;
  constexpr int SUB = R::SUB, ITEM = R::ITEM, STAGES = R::STAGES;
  constexpr int COLS = TILES;            // columns of this lane that are rows of their own
  constexpr int NEAR = ITEM + ROWS;      // distances between an item's keys and the rows
  static_assert(ROWS * D * 4 <= R::WARP_BYTES, "a warp's result takes the place of its ring");
  extern __shared__ __align__(16) uint8_t rings[];
  __shared__ float near_bias[WARPS][NEAR];
  __shared__ float sm_m[WARPS][ROWS], sm_l[WARPS][ROWS];
  __shared__ float out_m[ROWS], out_l[ROWS], out_o[ROWS][D];

  cg::cluster_group cluster = cg::this_cluster();
  const int C = gridDim.x, rank = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int key_of_g = (g >> 1) + 4 * (g & 1);             // the key of row g of a tile; row g + 8: 8 more
  const int h = blockIdx.y, b = p.row_groups == 1 ? blockIdx.z : blockIdx.z / p.row_groups;
  const int m0 = (blockIdx.z - b * p.row_groups) * ROWS;
  // ---- everything that waits for nothing is requested first: the length, the queries (column n of the products is row
  // m0 + n / 2 or, with TILES 2, m0 + n), the head's bias table (lane i has bucket i) and the buckets' first distances
  const int given_len = p.seqlens_k ? p.seqlens_k[b] : p.N;
  uint2 raw[KSTEPS];                     // four elements each
  {
    const int row = m0 + (TILES == 1 ? g >> 1 : g);
    const T* qp = (const T*)p.q + (int64_t)b * p.q_stride_b + (int64_t)h * p.q_stride_h + (int64_t)(row < p.M ? row : 0) * p.q_stride_m;
    #pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      raw[j] = make_uint2(0, 0);
      if (row < p.M) {
        const T* at = qp + dim_of<D>(c, j, 0);
        if (p.q_aligned) {
          raw[j] = __ldg((const uint2*)at);
        } else {
          const uint16_t* e = (const uint16_t*)at;
          raw[j] = make_uint2(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16);
        }
      }
    }
  }
  const bool has_bias = p.table != nullptr;
  const int buckets = spec.bidirectional ? 2 * spec.n_side : spec.n_side;
  float lane_bias = 0.f;
  int lane_first = 1 << 30;
  if (has_bias && buckets <= 32) {
    if (lane < buckets) lane_bias = load_table(p.table, p.table_dtype, (int64_t)lane * p.table_stride0 + h);
    if (lane < spec.n_first) lane_first = spec.first[lane];
  }
  auto bias_of = [&](int delta) -> float {               // by whole warps
    if (buckets > 32) return kLog2e * load_table(p.table, p.table_dtype, (int64_t)bucket_of_delta(spec, delta) * p.table_stride0 + h);
    const int d = min(spec.bidirectional ? abs(delta) : max(-delta, 0), spec.max_distance);
    int n = 0;                                           // first distances that d reaches: a search over the lanes
    #pragma unroll
    for (int half = 16; half > 0; half >>= 1) n += __shfl_sync(0xffffffffu, lane_first, n + half - 1) <= d ? half : 0;
    return kLog2e * __shfl_sync(0xffffffffu, lane_bias, n + (spec.bidirectional && delta > 0 ? spec.n_side : 0));
  };
  const int kv_len = min(max(given_len, 0), p.N);
  const int qoff = p.q_pos_offset >= 0 ? p.q_pos_offset : kv_len - p.M;
  const int md = spec.max_distance;
  // keys behind the last visible one of the last row are never touched
  const int first_pos = qoff + m0, last_pos = qoff + min(m0 + ROWS, p.M) - 1;
  const int n_end = p.causal ? min(kv_len, max(last_pos + 1, 0)) : kv_len;
  const int items = (n_end + ITEM - 1) / ITEM, step = C * WARPS;

  uint8_t* ring = rings + warp * R::WARP_BYTES;
  const uint8_t* kb = p.k + (int64_t)b * p.k_stride_b + (int64_t)h * p.k_stride_h + lane * 16;
  const uint8_t* vb = p.v + (int64_t)b * p.v_stride_b + (int64_t)h * p.v_stride_h + lane * 16;
  const float* ks = p.k_scale + (int64_t)b * p.ks_stride_b + (int64_t)h * p.ks_stride_h;
  const float* vs = p.v_scale + (int64_t)b * p.vs_stride_b + (int64_t)h * p.vs_stride_h;
  // an item's rows lie one behind the other: 16 bytes a lane; zeros behind the last key
  auto request = [&](int it, int stage) {
    if (it < items) {
      const int n0 = it * ITEM;
      const int64_t from = (int64_t)n0 * D;
      const uint32_t to = smem_u32(ring + stage * R::BYTES) + lane * 16;
      const int bytes = min(n_end - n0, ITEM) * D - lane * 16;      // of this lane's first piece on
      #pragma unroll
      for (int i = 0; i < (ITEM * D + 511) / 512; ++i)
        if (ITEM * D % 512 == 0 || lane * 16 + i * 512 < ITEM * D) {
          const bool in = i * 512 < bytes;
          copy_async16(to + i * 512, kb + (in ? from + i * 512 : 0), in);
          copy_async16(to + ITEM * D + i * 512, vb + (in ? from + i * 512 : 0), in);
        }
      if (lane < 2) copy_async4(smem_u32(ring + stage * R::BYTES + 2 * ITEM * D) + 4 * lane, (lane ? vs : ks) + n0 / BLOCK);
    }
    copy_commit();
  };
  int it = rank * WARPS + warp;
  #pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) request(it + i * step, i);

  // ---- queries, scaled to fp16's upper end
  uint32_t qf[KSTEPS][2];
  float col_scale[COLS];                 // of this lane's rows: c (TILES 1) or 2c and 2c + 1
  int col_pos[COLS];
  {
    float x[KSTEPS][4], most = 0.f;
    #pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      const T* t = reinterpret_cast<const T*>(&raw[j]);
      #pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = to_float<T>(t[e]);
        most = fmaxf(most, fabsf(x[j][e]));
      }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // a power of two: the largest element becomes 2^14 .. 2^15 (or less, of rows below 2^-111)
    const float unit = __uint_as_float(max(__float_as_uint(most) & 0x7f800000u, 0x08000000u) - (14u << 23));
    const float inv = 1.f / unit;
    #pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      qf[j][0] = pack_half2(x[j][0] * inv, x[j][1] * inv);
      qf[j][1] = pack_half2(x[j][2] * inv, x[j][3] * inv);
    }
    #pragma unroll
    for (int i = 0; i < COLS; ++i) {
      const int r = TILES == 1 ? c : 2 * c + i;
      col_scale[i] = __shfl_sync(0xffffffffu, unit, (TILES == 1 ? 2 * r : r) * 4) * p.scale_log2;
      col_pos[i] = first_pos + r;
    }
  }

  float bias_before = 0.f, bias_after = 0.f;
  if (has_bias) {
    bias_before = bias_of(-md);
    bias_after = bias_of(md);
  }

  float m_run[COLS], l_run[COLS];
  #pragma unroll
  for (int i = 0; i < COLS; ++i) { m_run[i] = LOWEST; l_run[i] = 0.f; }
  float acc[TILES][KSTEPS][4];
  #pragma unroll
  for (int t = 0; t < TILES; ++t)
    #pragma unroll
    for (int i = 0; i < KSTEPS; ++i)
      #pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][i][e] = 0.f;

  int stage = 0;
  #pragma unroll 1
  for (; it < items; it += step) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    request(it + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);    // (the stage that the last turn has read)
    const uint8_t* keys = ring + stage * R::BYTES;
    const uint8_t* values = keys + ITEM * D;
    const float k_scale = *(const float*)(values + ITEM * D), v_scale = *(const float*)(values + ITEM * D + 4);
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    const int n0 = it * ITEM;
    const bool whole = n0 + ITEM <= n_end && (!p.causal || n0 + ITEM - 1 <= first_pos);
    // ---- scores of the item's keys
    float s[SUB][2 * COLS];              // this lane's two keys of each tile, this lane's rows
    #pragma unroll
    for (int t = 0; t < SUB; ++t) {
      uint32_t k0[KW], k1[KW];
      const uint8_t* at = keys + (t * 16 + key_of_g) * D + (D == 128 ? 16 : KB) * c;
      read_bytes<KB>(at, k0);
      read_bytes<KB>(at + 8 * D, k1);
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      #pragma unroll
      for (int j = 0; j < KSTEPS; ++j) {
        uint32_t a0, a1, a2, a3;
        widen(k0[j], a0, a2);
        widen(k1[j], a1, a3);
        mma_16816(d, a0, a1, a2, a3, qf[j][0], qf[j][1]);
      }
      #pragma unroll
      for (int i = 0; i < COLS; ++i) { s[t][i] = d[i]; s[t][COLS + i] = d[2 + i]; }
    }
    float f[COLS];
    #pragma unroll
    for (int i = 0; i < COLS; ++i) f[i] = col_scale[i] * k_scale;
    // ---- bias: one value beyond the largest distance on either side, a small table within it
    float far_bias = 0.f;
    bool near = false;
    if (has_bias) {
      const bool before = n0 + ITEM - 1 - first_pos <= -md, after = n0 - last_pos >= md;
      near = !before && !after;
      if (near) {
        // entry i: key n0 + i - (ROWS - 1) and the first row
        __syncwarp();
        #pragma unroll 1
        for (int i = 0; i < NEAR - 1; i += 32) {
          const float v = bias_of(n0 + i + lane - (ROWS - 1) - first_pos);
          if (i + lane < NEAR - 1) near_bias[warp][i + lane] = v;
        }
        __syncwarp();
      } else {
        far_bias = before ? bias_before : bias_after;
      }
    }
    float mx[COLS];
    #pragma unroll
    for (int i = 0; i < COLS; ++i) mx[i] = -INFINITY;
    #pragma unroll
    for (int t = 0; t < SUB; ++t)
      #pragma unroll
      for (int e = 0; e < 2 * COLS; ++e) {
        const int i = e % COLS, key = t * 16 + key_of_g + 8 * (e / COLS);
        float bias = far_bias;
        if (near) bias = near_bias[warp][key + ROWS - 1 - (col_pos[i] - first_pos)];
        s[t][e] = fmaf(s[t][e], f[i], bias);
        if (!whole && (n0 + key >= n_end || (p.causal && n0 + key > col_pos[i]))) s[t][e] = -INFINITY;
        mx[i] = fmaxf(mx[i], s[t][e]);
      }
    // ---- running maximum, weights: those of an item relative to its own largest one, 2^14, and `beta` from there to the
    // running maximum (scores beyond 2^20, whose steps are too wide for the 14, relative to 1)
    float alpha[COLS], beta[COLS], ref[COLS];
    #pragma unroll
    for (int i = 0; i < COLS; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 4));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 8));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 16));
      const float m_new = fmaxf(m_run[i], mx[i]);
      ref[i] = fmaxf(mx[i], LOWEST);
      if (fabsf(ref[i]) < 1048576.f) ref[i] -= 14.f;
      alpha[i] = fast_exp2(m_run[i] - m_new);
      beta[i] = fast_exp2(ref[i] - m_new);
      m_run[i] = m_new;
    }
    float sum[COLS];
    float part[TILES][KSTEPS][4];
    #pragma unroll
    for (int t = 0; t < TILES; ++t)
      #pragma unroll
      for (int i = 0; i < KSTEPS; ++i)
        #pragma unroll
        for (int e = 0; e < 4; ++e) part[t][i][e] = 0.f;
    #pragma unroll
    for (int t = 0; t < SUB; ++t) {
      float w[2 * COLS], hi[2 * COLS], lo[2 * COLS];
      #pragma unroll
      for (int e = 0; e < 2 * COLS; ++e) {
        w[e] = fast_exp2(s[t][e] - ref[e % COLS]);
        sum[e % COLS] = t == 0 && e < COLS ? w[e] : sum[e % COLS] + w[e];
        hi[e] = __uint_as_float(__float_as_uint(w[e]) & 0xffffe000u);
        lo[e] = w[e] - hi[e];
      }
      uint32_t b0, b1, c0 = 0, c1 = 0;
      if constexpr (TILES == 1) {        // columns 2c and 2c + 1: hi and lo
        b0 = transpose_8x8(pack_half2(hi[0], lo[0]));
        b1 = transpose_8x8(pack_half2(hi[1], lo[1]));
      } else {
        b0 = transpose_8x8(pack_half2(hi[0], hi[1]));
        b1 = transpose_8x8(pack_half2(hi[2], hi[3]));
        c0 = transpose_8x8(pack_half2(lo[0], lo[1]));
        c1 = transpose_8x8(pack_half2(lo[2], lo[3]));
      }
      uint32_t v0[VW], v1[VW], v2[VW], v3[VW];
      const uint8_t* at = values + (t * 16 + c) * D + VB * g;
      read_bytes<VB>(at, v0); read_bytes<VB>(at + 4 * D, v1); read_bytes<VB>(at + 8 * D, v2); read_bytes<VB>(at + 12 * D, v3);
      #pragma unroll
      for (int i = 0; i < KSTEPS; ++i) {
        // rows g and g + 8 of tile i: bytes 2i and 2i + 1 of this lane's piece; pairs of keys (0, 1) and (2, 3)
        const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
        uint32_t a0, a1, a2, a3;
        widen(__byte_perm(v0[i / 2], v1[i / 2], sel), a0, a1);
        widen(__byte_perm(v2[i / 2], v3[i / 2], sel), a2, a3);
        mma_16816(part[0][i], a0, a1, a2, a3, b0, b1);
        if constexpr (TILES == 2) mma_16816(part[1][i], a0, a1, a2, a3, c0, c1);
      }
    }
    #pragma unroll
    for (int i = 0; i < COLS; ++i) {
      l_run[i] = fmaf(sum[i], beta[i], l_run[i] * alpha[i]);
      beta[i] *= v_scale;
    }
    #pragma unroll
    for (int t = 0; t < TILES; ++t)
      #pragma unroll
      for (int i = 0; i < KSTEPS; ++i)
        #pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][i][e] = fmaf(part[t][i][e], beta[TILES == 1 ? 0 : e & 1], acc[t][i][e] * alpha[TILES == 1 ? 0 : e & 1]);
  }
  copy_wait<0>();
  __syncwarp();                          // the ring is free for the warp's result
  float* sm_o = (float*)ring;            // [ROWS][D]

  // ---- the warp's result: hi + lo, sums over the lanes that share a row
  #pragma unroll
  for (int i = 0; i < COLS; ++i) {
    l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 4);
    l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 8);
    l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 16);
    if (g == 0) { sm_m[warp][COLS * c + i] = m_run[i]; sm_l[warp][COLS * c + i] = l_run[i]; }
  }
  #pragma unroll
  for (int i = 0; i < KSTEPS; ++i)
    #pragma unroll
    for (int e = 0; e < 2; ++e) {        // bytes 2i and 2i + 1
      if constexpr (TILES == 1) {
        sm_o[c * D + VB * g + 2 * i + e] = acc[0][i][2 * e] + acc[0][i][2 * e + 1];
      } else {
        sm_o[2 * c * D + VB * g + 2 * i + e] = acc[0][i][2 * e] + acc[1][i][2 * e];
        sm_o[(2 * c + 1) * D + VB * g + 2 * i + e] = acc[0][i][2 * e + 1] + acc[1][i][2 * e + 1];
      }
    }
  __syncthreads();

  // ---- the block's result, then the cluster's
  for (int i = tid; i < ROWS * D; i += THREADS) {
    const int r = i / D, d = i % D;
    float mm = -INFINITY;
    #pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, sm_m[w][r]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float l = 0.f, o = 0.f;
    #pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = fast_exp2(sm_m[w][r] - ref);
      l += sm_l[w][r] * f;
      o += ((const float*)(rings + w * R::WARP_BYTES))[r * D + d] * f;
    }
    if (C == 1) {
      if (m0 + r < p.M)
        ((T*)p.out)[(int64_t)b * p.o_stride_b + (int64_t)h * p.o_stride_h + (int64_t)(m0 + r) * p.o_stride_m + d] =
            from_float<T>(l == 0.f ? 0.f : o / l);
    } else {
      out_o[r][d] = o;
      if (d == 0) { out_m[r] = mm; out_l[r] = l; }
    }
  }
  if (C == 1) return;
  cluster.sync();
  for (int i = rank * THREADS + tid; i < ROWS * D; i += C * THREADS) {
    const int r = i / D, d = i % D;
    float mm = -INFINITY;
    for (int k = 0; k < C; ++k) mm = fmaxf(mm, *cluster.map_shared_rank(&out_m[r], k));
    const float ref = mm == -INFINITY ? 0.f : mm;
    float l = 0.f, o = 0.f;
    for (int k = 0; k < C; ++k) {
      const float f = fast_exp2(*cluster.map_shared_rank(&out_m[r], k) - ref);
      l += *cluster.map_shared_rank(&out_l[r], k) * f;
      o += *cluster.map_shared_rank(&out_o[r][d], k) * f;
    }
    if (m0 + r < p.M)
      ((T*)p.out)[(int64_t)b * p.o_stride_b + (int64_t)h * p.o_stride_h + (int64_t)(m0 + r) * p.o_stride_m + d] =
          from_float<T>(l == 0.f ? 0.f : o / l);
  }
  cluster.sync();                        // nobody leaves while its shared memory is read
}

// What the current device says of a kernel, asked once: how many blocks, and clusters of 1, 2, 4, 8 and 16, are resident.
template <typename T, int D, int TILES, int WARPS>
struct Fit {
  int resident = 0, clusters[5];
  static const Fit* get() {
    static std::atomic<const Fit*> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (const Fit* f = known[dev]) return f;
    const auto kernel = decode_quantized_kernel<T, D, TILES, WARPS>;
    constexpr int smem = WARPS * Ring<D>::WARP_BYTES;
    int per_sm = 0, sms = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, WARPS * 32, smem) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return nullptr;
    Fit* f = new (std::nothrow) Fit;     // kept for the life of the process (a second thread may find the same again)
    if (!f) return nullptr;
    f->resident = per_sm * sms;
    if (!resident_clusters((const void*)kernel, WARPS * 32, smem, f->clusters)) { delete f; return nullptr; }
    known[dev] = f;
    return f;
  }
};

template <typename T, int D, int TILES, int WARPS>
static int launch(const Params& p, const BucketSpec& spec, int C, cudaStream_t stream) {
  constexpr int smem = WARPS * Ring<D>::WARP_BYTES;
  if (!Fit<T, D, TILES, WARPS>::get()) return T5B_ERR_LAUNCH;            // (which allows the launch that much shared memory)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)C, (unsigned)p.H, (unsigned)(p.B * p.row_groups));
  cfg.blockDim = dim3(WARPS * 32); cfg.stream = stream; cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, decode_quantized_kernel<T, D, TILES, WARPS>, p, spec) == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}

// Warps per head.  What a block costs beyond its keys (lengths, queries, bias, two merges) and how the last blocks fill the
// GPU decide, so the split goes by heads = B * H * groups of rows and by the items of a whole cache (us on B200):
//   * up to 212 heads, if all of their blocks are resident at a time: a block of eight warps each (192 heads x 2048 keys:
//     9.4, with four warps 10.3; 160 x 1024 of 128 columns, where one such block fits: 19.9 and 16.4), and clusters up to
//     1700 warps in all as long as a warp keeps four items and all are resident (12 x 102400: 36.1 in clusters of 16, 267
//     without; 24 x 9664 of 128 columns, 5 rows: 23.3 in clusters of 4, 29.7 of 8, which are not);
//   * short caches of many heads: two warps (768 x 512: 12.8, with four 14.3), and more heads than blocks of four warps are
//     resident, up to half as many more (512 x 4096 of 128 columns: 96.8, with four 115.7);
//   * else four warps (1536 x 2048: 66.9, with two 78.8), two blocks per head for long caches of 400 to 1200 heads, where
//     one block per head leaves the last round of blocks half empty (x 8192, two blocks and one: 448 heads 84 and 89, 640
//     115 and 136, 768 129 and 146, 1024 173 and 181, 1152 197 and 190; of 128 columns 448 heads 176 and 198, 640 217 and
//     256, 1024 352 and 357; x 4096 neither is ahead: 448 heads 47.5 and 47.2, 640 64.0 and 65.1, 1024 90.9 and 91.0).
template <typename T, int D, int TILES>
static int launch_split(const Params& p, const BucketSpec& spec, cudaStream_t stream) {
  const int64_t heads = (int64_t)p.B * p.H * p.row_groups, items = (p.N + Ring<D>::ITEM - 1) / Ring<D>::ITEM;
  if (heads <= 212 && items >= 16) {
    const auto* fit = Fit<T, D, TILES, 8>::get();
    if (!fit) return T5B_ERR_LAUNCH;
    if (heads <= fit->resident) {
      int c = 0;
      while (c < 4 && heads * (16 << c) <= 1700 && items >= 64 << c && heads <= fit->clusters[c + 1]) ++c;
      return launch<T, D, TILES, 8>(p, spec, 1 << c, stream);
    }
  }
  if (heads > 400 && heads < 1200 && items >= 256) return launch<T, D, TILES, 4>(p, spec, 2, stream);
  const auto* fit = Fit<T, D, TILES, 4>::get();
  if (!fit) return T5B_ERR_LAUNCH;
  if ((heads >= 512 && items <= 16) || (heads > fit->resident && 2 * heads <= 3 * fit->resident))
    return launch<T, D, TILES, 2>(p, spec, 1, stream);
  return launch<T, D, TILES, 4>(p, spec, 1, stream);
}

template <typename T, int D>
static int launch_rows(Params& p, const BucketSpec& spec, cudaStream_t stream) {
  p.row_groups = p.M <= 4 ? 1 : (p.M + 7) / 8;
  if ((int64_t)p.B * p.row_groups > 65535) return T5B_ERR_SHAPE;
  return p.M <= 4 ? launch_split<T, D, 1>(p, spec, stream) : launch_split<T, D, 2>(p, spec, stream);
}

template <typename T>
static int launch_type(Params& p, int D, const BucketSpec& spec, cudaStream_t stream) {
  switch (D) {
    case 16: return launch_rows<T, 16>(p, spec, stream);
    case 32: return launch_rows<T, 32>(p, spec, stream);
    case 64: return launch_rows<T, 64>(p, spec, stream);
    case 128: return launch_rows<T, 128>(p, spec, stream);
  }
  return T5B_ERR_HEAD_DIM;
}

}  // namespace decq
}  // namespace t5b

using namespace t5b;

extern "C" int t5b_decode_quantized_fwd(const t5b_decode_quantized_args* a, void* stream) {
  if (!a) return T5B_ERR_ARG;
  if (a->dtype != T5B_F16 && a->dtype != T5B_BF16) return T5B_ERR_DTYPE;
  if (a->D != 16 && a->D != 32 && a->D != 64 && a->D != 128) return T5B_ERR_HEAD_DIM;
  if (a->B < 0 || a->H < 0 || a->M < 0 || a->N < 0 || a->N > 0x7fffffff - (T5B_CACHE_BLOCK - 1) || a->H > 65535 ||
      a->M > (1 << 20)) return T5B_ERR_SHAPE;
  if (a->B == 0 || a->H == 0 || a->M == 0) return T5B_OK;
  if (a->q_pos_offset > 0x7fffffff - a->M - 2 * T5B_CACHE_BLOCK) return T5B_ERR_ARG;      // positions are 32-bit numbers
  if (!a->q || !a->out || (a->N > 0 && (!a->k || !a->v || !a->k_scale || !a->v_scale))) return T5B_ERR_ARG;
  if ((uintptr_t)a->k % 16 || (uintptr_t)a->v % 16 || (uintptr_t)a->q % 2 || (uintptr_t)a->k_scale % 4 || (uintptr_t)a->v_scale % 4)
    return T5B_ERR_ALIGN;
  if (a->k_stride_b % 16 || a->k_stride_h % 16 || a->v_stride_b % 16 || a->v_stride_h % 16) return T5B_ERR_ALIGN;
  BucketSpec spec;
  spec.n_side = 2; spec.bidirectional = 0; spec.max_distance = 1; spec.n_first = 0;
  if (a->table) {
    if (a->table_dtype != T5B_F32 && a->table_dtype != T5B_F16 && a->table_dtype != T5B_BF16) return T5B_ERR_DTYPE;
    const int st = make_bucket_spec(a->num_buckets, a->max_distance, a->causal ? 0 : 1, &spec);
    if (st != T5B_OK) return st;
    if (spec.max_distance > 2048) return T5B_ERR_UNSUPPORTED;
  }
  decq::Params p;
  p.q = a->q; p.k = (const uint8_t*)a->k; p.v = (const uint8_t*)a->v; p.k_scale = a->k_scale; p.v_scale = a->v_scale;
  p.out = a->out; p.table = a->table; p.seqlens_k = a->seqlens_k;
  p.q_stride_b = a->q_stride_b; p.q_stride_h = a->q_stride_h; p.q_stride_m = a->q_stride_m;
  p.k_stride_b = a->k_stride_b; p.k_stride_h = a->k_stride_h; p.v_stride_b = a->v_stride_b; p.v_stride_h = a->v_stride_h;
  p.ks_stride_b = a->k_scale_stride_b; p.ks_stride_h = a->k_scale_stride_h;
  p.vs_stride_b = a->v_scale_stride_b; p.vs_stride_h = a->v_scale_stride_h;
  p.o_stride_b = a->o_stride_b; p.o_stride_h = a->o_stride_h; p.o_stride_m = a->o_stride_m;
  p.table_stride0 = a->table_stride0; p.table_dtype = a->table_dtype;
  p.B = a->B; p.H = a->H; p.M = a->M; p.N = a->N; p.causal = a->causal; p.q_pos_offset = a->q_pos_offset; p.row_groups = 1;
  p.scale_log2 = a->sm_scale * kLog2e;
  p.q_aligned = (uintptr_t)a->q % 8 == 0 && a->q_stride_b % 4 == 0 && a->q_stride_h % 4 == 0 && a->q_stride_m % 4 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == T5B_F16) return decq::launch_type<__half>(p, a->D, spec, st);
  return decq::launch_type<__nv_bfloat16>(p, a->D, spec, st);
}
