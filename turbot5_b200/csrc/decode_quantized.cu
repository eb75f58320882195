// Decoding against an 8-bit cache: a few query rows per (batch, head), keys and values as e4m3 numbers with one
// power-of-two scale per 64 tokens and head.
//
//   out = softmax(sm_scale * q (K * s_K)^T + table[bucket(n - position), h] (+ causal mask)) (V * s_V)
//
// Bound by the bytes of the cache, half of a 16-bit one: at 6.5 TB/s a multiprocessor has to take in 23 numbers per
// clock, each of which has to be widened and multiplied.  Doing that in float32 would take 2.5 instructions per number
// and query row; here one conversion per two numbers makes fp16 pairs and the warp-wide m16n8k16 product does the rest
// for up to eight rows at the cost of one.
//
//   * S^T = K Q^T: the keys are the rows of the product.  A lane's 16 bytes of a key are four k-steps of the A operand
//     as they stand (the order of the head dim inside a k-step is free, the queries are read in the same order).
//   * O^T = V^T P^T: the head dim is the rows.  A byte permute joins two keys' bytes to pairs along the key dim.
//   * P^T comes out of S^T's registers by one 8x8 transpose of 16-bit pairs.
//   * fp16 products of e4m3 numbers are exact in float32; q is scaled to 1 by a power of two.  P is carried as
//     hi + lo in two columns: with up to four rows the eight columns hold each row twice, with up to eight rows the
//     product is issued twice, so P keeps 22 bits and the result is as exact as float32 weights would make it.
//
// A warp owns blocks of 64 keys (so a block has one scale), with its own running maximum and sum; warps merge in shared
// memory, the blocks of a (batch, head) that share a long cache form a cluster and merge through distributed shared
// memory: no workspace, no counters, no second launch.
//
// Semantics: the cached step of T5Attention.forward (src/turbot5/model/attentions.py:198,229-234), the merge rule of
// src/turbot5/ops/flash_decoding.py:47-55, as in decode.cu.
#include "t5b_common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace t5b {
namespace decq {

constexpr int BLOCK = T5B_CACHE_BLOCK;
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_CLUSTER = 8;

struct Params {
  const void* q; const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale; void* out;
  const void* table; const int32_t* seqlens_k;
  int64_t q_stride_b, q_stride_h, q_stride_m;
  int64_t k_stride_b, k_stride_h, v_stride_b, v_stride_h;
  int64_t ks_stride_b, ks_stride_h, vs_stride_b, vs_stride_h;
  int64_t o_stride_b, o_stride_h, o_stride_m;
  int64_t table_stride0;
  int32_t table_dtype, B, H, M, N, causal, q_pos_offset, row_groups;
  float scale_log2;
};

__device__ __forceinline__ uint32_t half2_of_e4m3x2(uint32_t two_bytes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two_bytes));
  return h;
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

// BYTES consecutive bytes of a row into words, streaming
template <int BYTES> __device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES == 2) {
    uint16_t t;
    asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(t) : "l"(p));
    w[0] = t;
  } else if constexpr (BYTES == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  } else if constexpr (BYTES == 8) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    #pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3]) : "l"(p + 64 * i));
  }
}

// Element of the head dim that lane c holds as element e (0 .. 3) of k-step j of the first product.
template <int D> __device__ __forceinline__ int dim_of(int c, int j, int e) {
  return D == 128 ? j / 4 * 64 + 16 * c + 4 * (j & 3) + e : D / 4 * c + 4 * j + e;
}

// TILES 1: up to four rows, hi and lo of P in the columns of one product.  TILES 2: up to eight rows, two products.
template <typename T, int D, int TILES>
__global__ void __launch_bounds__(THREADS)
decode_quantized_kernel(const __grid_constant__ Params p, const __grid_constant__ BucketSpec spec) {
  constexpr int ROWS = 4 * TILES;
  constexpr int KSTEPS = D / 16;         // k-steps of S^T, 16-row tiles of O^T
  constexpr int KB = D / 4, VB = D / 8;  // bytes of a key / value row that a lane holds
  constexpr int KW = KB / 4, VW = (VB + 3) / 4;
  constexpr int SUB = D == 128 ? 2 : 4;  // 16-key tiles whose loads are in flight together
  extern __shared__ float lut[];
  __shared__ float sm_m[WARPS][8], sm_l[WARPS][8];
  __shared__ float sm_o[WARPS][ROWS][D];
  __shared__ float out_m[ROWS], out_l[ROWS], out_o[ROWS][D];

  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z / p.row_groups, m0 = blockIdx.z % p.row_groups * ROWS;
  const int kv_len = p.seqlens_k ? min(max(p.seqlens_k[b], 0), p.N) : p.N;
  const int qoff = p.q_pos_offset >= 0 ? p.q_pos_offset : kv_len - p.M;
  const int md = spec.max_distance;
  const bool has_bias = p.table != nullptr;
  if (has_bias) {
    for (int i = tid; i < 2 * md + 1; i += THREADS)
      lut[i] = load_table(p.table, p.table_dtype, (int64_t)bucket_of_delta(spec, i - md) * p.table_stride0 + h) * kLog2e;
    __syncthreads();
  }

  // ---- queries: column n of the products is row m0 + n (TILES 2) or m0 + n % 4 (TILES 1), scaled to at most 1
  uint32_t qf[KSTEPS][2];
  float col_scale[2];                    // of this lane's columns 2c and 2c + 1
  int col_pos[2];
  {
    const int row = m0 + (TILES == 1 ? (g & 3) : g);
    const bool in = row < p.M;
    const T* qp = (const T*)p.q + (int64_t)b * p.q_stride_b + (int64_t)h * p.q_stride_h + (int64_t)(in ? row : 0) * p.q_stride_m;
    float x[KSTEPS][4], most = 0.f;
    #pragma unroll
    for (int j = 0; j < KSTEPS; ++j)
      #pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = in ? to_float<T>(qp[dim_of<D>(c, j, e)]) : 0.f;
        most = fmaxf(most, fabsf(x[j][e]));
      }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // a power of two at or below the largest element (1 where that is 0, tiny or not finite)
    const uint32_t eb = __float_as_uint(most) & 0x7f800000u;
    const float unit = eb >= 0x01000000u && eb <= 0x7e000000u ? __uint_as_float(eb) : 1.f;
    const float inv = 1.f / unit;
    #pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      qf[j][0] = pack_half2(x[j][0] * inv, x[j][1] * inv);
      qf[j][1] = pack_half2(x[j][2] * inv, x[j][3] * inv);
    }
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = 2 * c + i, r = TILES == 1 ? col & 3 : col;
      col_scale[i] = __shfl_sync(0xffffffffu, unit, r * 4) * p.scale_log2;
      col_pos[i] = qoff + m0 + r;
    }
  }

  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  float acc[TILES][KSTEPS][4];
  #pragma unroll
  for (int t = 0; t < TILES; ++t)
    #pragma unroll
    for (int i = 0; i < KSTEPS; ++i)
      #pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][i][e] = 0.f;

  const uint8_t* kb = p.k + (int64_t)b * p.k_stride_b + (int64_t)h * p.k_stride_h + (D == 128 ? 16 : KB) * c;
  const uint8_t* vb = p.v + (int64_t)b * p.v_stride_b + (int64_t)h * p.v_stride_h + VB * g;
  const float* ks = p.k_scale + (int64_t)b * p.ks_stride_b + (int64_t)h * p.ks_stride_h;
  const float* vs = p.v_scale + (int64_t)b * p.vs_stride_b + (int64_t)h * p.vs_stride_h;
  // keys behind the last visible one of the last row are never touched
  const int last_pos = qoff + min(m0 + ROWS, p.M) - 1;
  const int n_end = p.causal ? min(kv_len, max(last_pos + 1, 0)) : kv_len;
  const int blocks = (n_end + BLOCK - 1) / BLOCK;

  for (int blk = rank * WARPS + warp; blk < blocks; blk += C * WARPS) {
    const float k_scale = __ldg(ks + blk), v_scale = __ldg(vs + blk);
    const int n0 = blk * BLOCK;
    const bool whole = n0 + BLOCK <= n_end && (!p.causal || n0 + BLOCK - 1 <= qoff + m0);
    // every key of the block beyond the largest distance from every row: one bias value
    const bool before = n0 + BLOCK - 1 - (qoff + m0) <= -md;
    const bool far = has_bias && (before || n0 - last_pos >= md);
    const float far_bias = far ? lut[before ? 0 : 2 * md] : 0.f;
    #pragma unroll
    for (int half = 0; half < 4 / SUB; ++half) {
      const int nb = n0 + half * SUB * 16;
      if (half > 0 && nb >= n_end) break;
      uint32_t kw[SUB][2][KW], vw[SUB][4][VW];
      #pragma unroll
      for (int t = 0; t < SUB; ++t)
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = nb + t * 16 + g + 8 * i;
          #pragma unroll
          for (int w = 0; w < KW; ++w) kw[t][i][w] = 0;
          if (whole || n < n_end) load_bytes<KB>(kb + (int64_t)n * D, kw[t][i]);
        }
      #pragma unroll
      for (int t = 0; t < SUB; ++t)
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = nb + t * 16 + 2 * c + (i & 1) + 8 * (i >> 1);
          #pragma unroll
          for (int w = 0; w < VW; ++w) vw[t][i][w] = 0;
          if (whole || n < n_end) load_bytes<VB>(vb + (int64_t)n * D, vw[t][i]);
        }
      // ---- scores of SUB x 16 keys
      float s[SUB][4];
      #pragma unroll
      for (int t = 0; t < SUB; ++t) {
        #pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
        #pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
          mma_16816(s[t], half2_of_e4m3x2(kw[t][0][j] & 0xffffu), half2_of_e4m3x2(kw[t][1][j] & 0xffffu),
                    half2_of_e4m3x2(kw[t][0][j] >> 16), half2_of_e4m3x2(kw[t][1][j] >> 16), qf[j][0], qf[j][1]);
      }
      const float f0 = col_scale[0] * k_scale, f1 = col_scale[1] * k_scale;
      float mx[2] = {-INFINITY, -INFINITY};
      #pragma unroll
      for (int t = 0; t < SUB; ++t)
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = nb + t * 16 + g + 8 * (e >> 1);
          float bias = far_bias;
          if (has_bias && !far) bias = lut[min(max(n - col_pos[e & 1] + md, 0), 2 * md)];
          s[t][e] = fmaf(s[t][e], e & 1 ? f1 : f0, bias);
          if (!whole && (n >= n_end || (p.causal && n > col_pos[e & 1]))) s[t][e] = -INFINITY;
          mx[e & 1] = fmaxf(mx[e & 1], s[t][e]);
        }
      // ---- running maximum, weights
      float alpha[2], ref[2];
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 4));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 8));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 16));
        const float m_new = fmaxf(m_run[i], mx[i]);
        ref[i] = m_new == -INFINITY ? 0.f : m_new;
        alpha[i] = fast_exp2(m_run[i] - ref[i]);
        m_run[i] = m_new;
        l_run[i] *= alpha[i];
      }
      float part[TILES][KSTEPS][4];
      #pragma unroll
      for (int t = 0; t < TILES; ++t)
        #pragma unroll
        for (int i = 0; i < KSTEPS; ++i)
          #pragma unroll
          for (int e = 0; e < 4; ++e) part[t][i][e] = 0.f;
      #pragma unroll
      for (int t = 0; t < SUB; ++t) {
        float w[4], lo[4];
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = fast_exp2(s[t][e] - ref[e & 1]);
          l_run[e & 1] += w[e];
          lo[e] = w[e] - __half2float(__float2half_rn(w[e]));
        }
        uint32_t b0, b1, c0 = 0, c1 = 0;
        if (TILES == 1) {                // columns 0 .. 3 hi, 4 .. 7 lo
          const bool low = c >= 2;
          b0 = transpose_8x8(pack_half2(low ? lo[0] : w[0], low ? lo[1] : w[1]));
          b1 = transpose_8x8(pack_half2(low ? lo[2] : w[2], low ? lo[3] : w[3]));
        } else {
          b0 = transpose_8x8(pack_half2(w[0], w[1]));
          b1 = transpose_8x8(pack_half2(w[2], w[3]));
          c0 = transpose_8x8(pack_half2(lo[0], lo[1]));
          c1 = transpose_8x8(pack_half2(lo[2], lo[3]));
        }
        #pragma unroll
        for (int i = 0; i < KSTEPS; ++i) {
          // rows g and g + 8 of tile i: bytes 2i and 2i + 1 of this lane's piece; pairs of keys (0, 1) and (2, 3)
          const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
          const uint32_t x = __byte_perm(vw[t][0][i / 2], vw[t][1][i / 2], sel);
          const uint32_t y = __byte_perm(vw[t][2][i / 2], vw[t][3][i / 2], sel);
          const uint32_t a0 = half2_of_e4m3x2(x & 0xffffu), a1 = half2_of_e4m3x2(x >> 16);
          const uint32_t a2 = half2_of_e4m3x2(y & 0xffffu), a3 = half2_of_e4m3x2(y >> 16);
          mma_16816(part[0][i], a0, a1, a2, a3, b0, b1);
          if (TILES == 2) mma_16816(part[TILES - 1][i], a0, a1, a2, a3, c0, c1);
        }
      }
      #pragma unroll
      for (int t = 0; t < TILES; ++t)
        #pragma unroll
        for (int i = 0; i < KSTEPS; ++i)
          #pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][i][e] = fmaf(part[t][i][e], v_scale, acc[t][i][e] * alpha[e & 1]);
    }
  }

  // ---- the warp's result: hi + lo, sums over the lanes that share a column
  #pragma unroll
  for (int i = 0; i < 2; ++i) {
    l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 4);
    l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 8);
    l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 16);
    if (g == 0) { sm_m[warp][2 * c + i] = m_run[i]; sm_l[warp][2 * c + i] = l_run[i]; }
  }
  #pragma unroll
  for (int i = 0; i < KSTEPS; ++i)
    #pragma unroll
    for (int e = 0; e < 4; ++e) {
      float o = acc[0][i][e];
      if (TILES == 1) o += __shfl_xor_sync(0xffffffffu, o, 2);          // column + 4
      else o += acc[TILES - 1][i][e];
      const int row = 2 * c + (e & 1);
      if (row < ROWS) sm_o[warp][row][VB * g + 2 * i + (e >> 1)] = o;
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
      o += sm_o[w][r][d] * f;
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

static int cluster_blocks(int64_t heads, int N) {
  // as many blocks per head as fill the GPU a few times over, each with at least a block of 64 keys per warp
  const int64_t most = (N + WARPS * BLOCK - 1) / (WARPS * BLOCK);
  int C = 1;
  while (C < MAX_CLUSTER && heads * C < 8 * 148 && C * 2 <= most) C *= 2;
  return C;
}

template <typename T, int D, int TILES>
static int launch(const Params& p, const BucketSpec& spec, size_t smem, cudaStream_t stream) {
  const int C = cluster_blocks((int64_t)p.B * p.H * p.row_groups, p.N);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)C, (unsigned)p.H, (unsigned)(p.B * p.row_groups));
  cfg.blockDim = dim3(THREADS); cfg.stream = stream; cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, decode_quantized_kernel<T, D, TILES>, p, spec) == cudaSuccess ? T5B_OK : T5B_ERR_LAUNCH;
}

template <typename T, int D>
static int launch_rows(Params& p, const BucketSpec& spec, size_t smem, cudaStream_t stream) {
  p.row_groups = p.M <= 4 ? 1 : (p.M + 7) / 8;
  if ((int64_t)p.B * p.row_groups > 65535) return T5B_ERR_SHAPE;
  return p.M <= 4 ? launch<T, D, 1>(p, spec, smem, stream) : launch<T, D, 2>(p, spec, smem, stream);
}

template <typename T>
static int launch_type(Params& p, int D, const BucketSpec& spec, size_t smem, cudaStream_t stream) {
  switch (D) {
    case 16: return launch_rows<T, 16>(p, spec, smem, stream);
    case 32: return launch_rows<T, 32>(p, spec, smem, stream);
    case 64: return launch_rows<T, 64>(p, spec, smem, stream);
    case 128: return launch_rows<T, 128>(p, spec, smem, stream);
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
  if (a->B < 0 || a->H < 0 || a->M < 0 || a->N < 0 || a->H > 65535) return T5B_ERR_SHAPE;
  if (a->B == 0 || a->H == 0 || a->M == 0) return T5B_OK;
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
  const size_t smem = a->table ? (size_t)(2 * spec.max_distance + 1) * 4 : 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == T5B_F16) return decq::launch_type<__half>(p, a->D, spec, smem, st);
  return decq::launch_type<__nv_bfloat16>(p, a->D, spec, smem, st);
}
