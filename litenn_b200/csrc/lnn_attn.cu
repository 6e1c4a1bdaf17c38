// Attention with a sliding window and sinks on the FP32 pipe, forward and backward, and the single-token step over a
// cache.  One pass over the visible tiles of keys, the running maximum and sum of the softmax in registers; the
// backward pass recomputes the probabilities from the stored denominators, once for the rows of dq and once for those
// of dk and dv, so that every sum has one owner and a fixed order (no atomics).
//
// The tiles are for sequences of one tile, heads of more than 128 values and heads that the split form does not hold: bound
// by shared-memory reads (a float4 per two rows or columns and four multiply-adds of each), 16 rows and columns of threads
// with 4 x 4 products each.  37 positions of 4 heads of 64 values: 9 us of which 4 are the launch.
// The step is bound by HBM: the cache is read once, 64 sequences of 4096 slots with 8 heads of 128 values (2.15 GB) in
// 330 us, 6.5 TB/s.
#include <cooperative_groups.h>
#include <math_constants.h>
#include <float.h>
#include <algorithm>
#include <type_traits>
#include "lnn_attn.cuh"
#include "lnn_tc_dev.cuh"

namespace {

namespace cg = cooperative_groups;
using lnn::AttnArgs;
using lnn::exp2_fast;
using lnn::min_or_nan;

constexpr int kThreads = 256;           // 16 x 16

// rows [r0, r0 + B) of a [len][dim] matrix into shared memory with pitch DP + 4, zeros outside
template <int B, int DP>
__device__ __forceinline__ void load_rows(float* dst, const float* src, int r0, int len, int dim) {
  for (int i = threadIdx.x; i < B * DP; i += kThreads) {
    const int r = i / DP, c = i % DP;
    dst[r * (DP + 4) + c] = r0 + r < len && c < dim ? __ldg(src + (int64_t)(r0 + r) * dim + c) : 0.0f;
  }
}
// s[r][c] = row (ty + 16 r) of A times row (tx + 16 c) of Bm
template <int B, int DP>
__device__ __forceinline__ void tile_product(float (&s)[B / 16][B / 16], const float* A, const float* Bm, int ty, int tx) {
  constexpr int R = B / 16, PITCH = DP + 4;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < R; ++c) s[r][c] = 0.0f;
  for (int d = 0; d < DP; d += 4) {
    float4 a[R], b[R];
#pragma unroll
    for (int r = 0; r < R; ++r) a[r] = *reinterpret_cast<const float4*>(A + (ty + 16 * r) * PITCH + d);
#pragma unroll
    for (int c = 0; c < R; ++c) b[c] = *reinterpret_cast<const float4*>(Bm + (tx + 16 * c) * PITCH + d);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < R; ++c)
        s[r][c] = fmaf(a[r].w, b[c].w, fmaf(a[r].z, b[c].z, fmaf(a[r].y, b[c].y, fmaf(a[r].x, b[c].x, s[r][c]))));
  }
}
// o[r][..] += sum_j W[ty + 16 r][j] X[j][..]; a weight of zero leaves out what X holds there (it may not be finite)
template <int B, int DP>
__device__ __forceinline__ void tile_weighted(float (&o)[B / 16][DP / 16], const float* W, const float* X, int ty, int tx) {
  constexpr int R = B / 16, PITCH = DP + 4;
  for (int j = 0; j < B; ++j) {
    float x[DP / 16];
#pragma unroll
    for (int u = 0; u < DP / 16; ++u) x[u] = X[j * PITCH + tx + 16 * u];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float w = W[(ty + 16 * r) * (B + 1) + j];
      if (w != 0.0f)
#pragma unroll
        for (int u = 0; u < DP / 16; ++u) o[r][u] = fmaf(w, x[u], o[r][u]);
    }
  }
}
__device__ __forceinline__ float row_max(float v) {        // over the 16 threads of a row
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <int B, int DP>
__global__ void __launch_bounds__(kThreads)
simt_fwd_kernel(const AttnArgs a) {
  constexpr int R = B / 16, PITCH = DP + 4;
  extern __shared__ __align__(16) float smem[];
  float *Q = smem, *K = Q + B * PITCH, *V = K + B * PITCH, *P = V + B * PITCH;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  if (a.beside) lnn::start_next();
  else lnn::wait_for_previous();
  const bool left = !a.info || lnn::any_group_left(a);
  const int tiles_q = (a.q_len + B - 1) / B, past = a.kv_len - a.q_len;
  for (int64_t work = blockIdx.x; left && work < (int64_t)tiles_q * a.q_heads * a.batch; work += gridDim.x) {
    const int h = (int)(work / tiles_q % a.q_heads), b = (int)(work / tiles_q / a.q_heads);
    const int i0 = (int)(work % tiles_q) * B;
    if (a.info && lnn::group_ok(a, b, h / (a.q_heads / a.kv_heads))) continue;
    __syncthreads();
    const int len = lnn::attn_length(a.lengths, b, a.kv_len, a.status);
    const int64_t head = (int64_t)b * a.q_heads + h;
    const int64_t kv = ((int64_t)b * a.kv_heads + h / (a.q_heads / a.kv_heads)) * a.kv_len * a.dim;
    const float factor = fabsf(a.scale) * lnn::kLog2e, sign = a.scale < 0.0f ? -1.0f : 1.0f;
    float o[R][DP / 16], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -CUDART_INF_F;
      l[r] = 0.0f;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u) o[r][u] = 0.0f;
    }
    const int p_hi = min(min(i0 + B, a.q_len) - 1 + past, len - 1);
    if (p_hi >= i0 + past) {
      load_rows<B, DP>(Q, a.q + head * a.q_len * a.dim, i0, a.q_len, a.dim);
      const lnn::KeyTiles tiles(i0 + past, p_hi, a.window, a.sinks, B);
      for (int t = 0; t < tiles.count; ++t) {
        const int j0 = tiles.at(t) * B;
        __syncthreads();
        load_rows<B, DP>(K, a.k + kv, j0, a.kv_len, a.dim);
        load_rows<B, DP>(V, a.v + kv, j0, a.kv_len, a.dim);
        __syncthreads();
        float s[R][R];
        tile_product<B, DP>(s, Q, K, ty, tx);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int p = i0 + ty + 16 * r + past;
          float top = -CUDART_INF_F;
#pragma unroll
          for (int c = 0; c < R; ++c) {
            s[r][c] = p <= p_hi && lnn::attn_visible(p, j0 + tx + 16 * c, a.window, a.sinks) ? __fmul_rn(s[r][c], sign) : -CUDART_INF_F;
            top = fmaxf(top, s[r][c]);
          }
          top = fmaxf(m[r], row_max(top));
          const float base = top == -CUDART_INF_F ? 0.0f : top;
          // (differences of scores before the factor, which may be 0)
          const float keep = m[r] == -CUDART_INF_F ? 0.0f : exp2_fast(__fmul_rn(__fsub_rn(m[r], base), factor));
          float sum = 0.0f;
#pragma unroll
          for (int c = 0; c < R; ++c) {
            const float e = s[r][c] == -CUDART_INF_F ? 0.0f : exp2_fast(__fmul_rn(__fsub_rn(s[r][c], base), factor));
            sum = __fadd_rn(sum, e);
            P[(ty + 16 * r) * (B + 1) + tx + 16 * c] = __fmul_rn(e, a.down);
          }
          l[r] = __fadd_rn(__fmul_rn(l[r], keep), row_sum(sum));
          m[r] = top;
#pragma unroll
          for (int u = 0; u < DP / 16; ++u) o[r][u] = __fmul_rn(o[r][u], keep);
        }
        __syncthreads();
        tile_weighted<B, DP>(o, P, V, ty, tx);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = i0 + ty + 16 * r;
      if (i >= a.q_len) continue;
      const bool empty = i + past > p_hi;
      const float inv = empty ? 0.0f : __fdiv_rn(1.0f, l[r]);
      float* to = a.o + (head * a.q_len + i) * a.dim;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u)
        if (tx + 16 * u < a.dim) to[tx + 16 * u] = empty ? 0.0f : __fmul_rn(__fmul_rn(o[r][u], inv), a.up);
      if (tx == 0)
        reinterpret_cast<float2*>(a.lse)[head * a.q_len + i] = empty ? make_float2(CUDART_INF_F, 0.0f) : lnn::log_sum(m[r], factor, l[r]);
    }
  }
  if (a.beside) lnn::wait_at_end();
}

// 2^(factor s - lse), 1 at most whatever rounding says
__device__ __forceinline__ float weight(float s, float factor, float2 lse) {
  return exp2_fast(min_or_nan(__fsub_rn(fmaf(s, factor, -lse.x), lse.y), 0.0f));
}
// P = 2^(factor S - lse) and dS = scale P (dP + delta) of a tile: rows are queries (KEYS false) or keys (true)
template <int B, int DP>
__global__ void __launch_bounds__(kThreads)
simt_dq_kernel(const AttnArgs a) {
  constexpr int R = B / 16, PITCH = DP + 4;
  extern __shared__ __align__(16) float smem[];
  float *Q = smem, *D = Q + B * PITCH, *K = D + B * PITCH, *V = K + B * PITCH, *S = V + B * PITCH;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  if (a.beside) lnn::start_next();
  else lnn::wait_for_previous();
  const bool left = !a.info || lnn::any_group_left(a);
  const int tiles_q = (a.q_len + B - 1) / B, past = a.kv_len - a.q_len;
  for (int64_t work = blockIdx.x; left && work < (int64_t)tiles_q * a.q_heads * a.batch; work += gridDim.x) {
    const int h = (int)(work / tiles_q % a.q_heads), b = (int)(work / tiles_q / a.q_heads);
    const int i0 = (int)(work % tiles_q) * B;
    if (a.info && lnn::group_ok(a, b, h / (a.q_heads / a.kv_heads))) continue;
    __syncthreads();
    const int len = lnn::attn_length(a.lengths, b, a.kv_len, a.status);
    const int64_t head = (int64_t)b * a.q_heads + h;
    const int64_t kv = ((int64_t)b * a.kv_heads + h / (a.q_heads / a.kv_heads)) * a.kv_len * a.dim;
    const float factor = a.scale * lnn::kLog2e;
    float g[R][DP / 16], delta[R];
    float2 lse[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = i0 + ty + 16 * r;
      lse[r] = i < a.q_len ? __ldg(reinterpret_cast<const float2*>(a.lse) + head * a.q_len + i) : make_float2(CUDART_INF_F, 0.0f);
      delta[r] = i < a.q_len ? a.delta[head * a.delta_pitch + i] : 0.0f;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u) g[r][u] = 0.0f;
    }
    const int p_hi = min(min(i0 + B, a.q_len) - 1 + past, len - 1);
    if (p_hi >= i0 + past) {
      load_rows<B, DP>(Q, a.q + head * a.q_len * a.dim, i0, a.q_len, a.dim);
      load_rows<B, DP>(D, a.dout + head * a.q_len * a.dim, i0, a.q_len, a.dim);
      const lnn::KeyTiles tiles(i0 + past, p_hi, a.window, a.sinks, B);
      for (int t = 0; t < tiles.count; ++t) {
        const int j0 = tiles.at(t) * B;
        __syncthreads();
        load_rows<B, DP>(K, a.k + kv, j0, a.kv_len, a.dim);
        load_rows<B, DP>(V, a.v + kv, j0, a.kv_len, a.dim);
        __syncthreads();
        float s[R][R], dp[R][R];
        tile_product<B, DP>(s, Q, K, ty, tx);
        tile_product<B, DP>(dp, D, V, ty, tx);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < R; ++c) {
            const int p = i0 + ty + 16 * r + past;
            const bool seen = p <= p_hi && lnn::attn_visible(p, j0 + tx + 16 * c, a.window, a.sinks);
            const float e = weight(s[r][c], factor, lse[r]);
            S[(ty + 16 * r) * (B + 1) + tx + 16 * c] = seen ? __fmul_rn(__fmul_rn(e, __fadd_rn(dp[r][c], delta[r])), a.scale) : 0.0f;
          }
        __syncthreads();
        tile_weighted<B, DP>(g, S, K, ty, tx);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = i0 + ty + 16 * r;
      if (i >= a.q_len) continue;
      float* to = a.dq + (head * a.q_len + i) * a.dim;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u)
        if (tx + 16 * u < a.dim) to[tx + 16 * u] = a.acc_q ? __fadd_rn(to[tx + 16 * u], g[r][u]) : g[r][u];
    }
  }
  if (a.beside) lnn::wait_at_end();
}

template <int B, int DP>
__global__ void __launch_bounds__(kThreads)
simt_dkv_kernel(const AttnArgs a) {
  constexpr int R = B / 16, PITCH = DP + 4;
  extern __shared__ __align__(16) float smem[];
  float *Q = smem, *D = Q + B * PITCH, *K = D + B * PITCH, *V = K + B * PITCH, *P = V + B * PITCH, *S = P + B * (B + 1);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  if (a.beside) lnn::start_next();
  else lnn::wait_for_previous();
  const bool left = !a.info || lnn::any_group_left(a);
  const int tiles_k = (a.kv_len + B - 1) / B, past = a.kv_len - a.q_len, group = a.q_heads / a.kv_heads;
  for (int64_t work = blockIdx.x; left && work < (int64_t)tiles_k * a.kv_heads * a.batch; work += gridDim.x) {
    const int hk = (int)(work / tiles_k % a.kv_heads), b = (int)(work / tiles_k / a.kv_heads);
    const int j0 = (int)(work % tiles_k) * B;
    if (a.info && lnn::group_ok(a, b, hk)) continue;
    __syncthreads();
    const int len = lnn::attn_length(a.lengths, b, a.kv_len, a.status);
    const int64_t kv = ((int64_t)b * a.kv_heads + hk) * a.kv_len * a.dim;
    const float factor = a.scale * lnn::kLog2e;
    float gk[R][DP / 16], gv[R][DP / 16];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < DP / 16; ++u) gk[r][u] = gv[r][u] = 0.0f;
    const lnn::QuerySpan span(j0, min(j0 + B, a.kv_len) - 1, a.window, a.sinks, past, len);
    if (span.hi >= span.lo) {
      load_rows<B, DP>(K, a.k + kv, j0, a.kv_len, a.dim);
      load_rows<B, DP>(V, a.v + kv, j0, a.kv_len, a.dim);
      for (int h = hk * group; h < (hk + 1) * group; ++h) {
        const int64_t head = (int64_t)b * a.q_heads + h;
        for (int i0 = (span.lo - past) / B * B; i0 + past <= span.hi; i0 += B) {
          __syncthreads();
          load_rows<B, DP>(Q, a.q + head * a.q_len * a.dim, i0, a.q_len, a.dim);
          load_rows<B, DP>(D, a.dout + head * a.q_len * a.dim, i0, a.q_len, a.dim);
          __syncthreads();
          float s[R][R], dp[R][R];
          tile_product<B, DP>(s, K, Q, ty, tx);
          tile_product<B, DP>(dp, V, D, ty, tx);
#pragma unroll
          for (int c = 0; c < R; ++c) {
            const int i = i0 + tx + 16 * c, p = i + past;
            const float2 lse = i < a.q_len ? __ldg(reinterpret_cast<const float2*>(a.lse) + head * a.q_len + i) : make_float2(CUDART_INF_F, 0.0f);
            const float delta = i < a.q_len ? __ldg(a.delta + head * a.delta_pitch + i) : 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const bool seen = i < a.q_len && p < len && lnn::attn_visible(p, j0 + ty + 16 * r, a.window, a.sinks);
              const float e = seen ? weight(s[r][c], factor, lse) : 0.0f;
              P[(ty + 16 * r) * (B + 1) + tx + 16 * c] = e;
              S[(ty + 16 * r) * (B + 1) + tx + 16 * c] = seen ? __fmul_rn(__fmul_rn(e, __fadd_rn(dp[r][c], delta)), a.scale) : 0.0f;
            }
          }
          __syncthreads();
          tile_weighted<B, DP>(gv, P, D, ty, tx);
          tile_weighted<B, DP>(gk, S, Q, ty, tx);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = j0 + ty + 16 * r;
      if (j >= a.kv_len) continue;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u) {
        const int c = tx + 16 * u;
        if (c >= a.dim) continue;
        const int64_t at = kv + (int64_t)j * a.dim + c;
        if (a.dk) a.dk[at] = a.acc_k ? __fadd_rn(a.dk[at], gk[r][u]) : gk[r][u];
        if (a.dv) a.dv[at] = a.acc_v ? __fadd_rn(a.dv[at], gv[r][u]) : gv[r][u];
      }
    }
  }
  if (a.beside) lnn::wait_at_end();
}

// one warp per row
__global__ void __launch_bounds__(kThreads)
attn_delta_kernel(float* __restrict__ delta, const float* __restrict__ dout, const float* __restrict__ o, int64_t rows, int dim) {
  lnn::wait_for_previous();
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  float s = 0.0f;
  for (int c = threadIdx.x & 31; c < dim; c += 32) s = fmaf(__ldg(dout + row * dim + c), __ldg(o + row * dim + c), s);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, x));
  if ((threadIdx.x & 31) == 0) delta[row] = -s;
}

template <int B, int DP, class Kernel>
int launch_simt(lnn::Device* d, Kernel* kernel, int matrices, int tiles, int64_t works, const AttnArgs& a) {
  const unsigned grid = (unsigned)std::min<int64_t>(works, a.info ? d->sm_count : 1 << 30);
  const size_t bytes = (size_t)(matrices * B * (DP + 4) + tiles * B * (B + 1)) * 4;
  LNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  LNN_CUDA(lnn::launch_chained(d, kernel, grid, kThreads, bytes, a));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

template <int B, int DP>
int simt_fwd(lnn::Device* d, const AttnArgs& a) {
  return launch_simt<B, DP>(d, simt_fwd_kernel<B, DP>, 3, 1,
                            lnn_ceil_div(a.q_len, B) * a.q_heads * a.batch, a);
}
template <int B, int DP>
int simt_bwd(lnn::Device* d, AttnArgs a) {
  int rc = LNN_OK;
  if (a.dq)
    rc = launch_simt<B, DP>(d, simt_dq_kernel<B, DP>, 4, 1,
                            lnn_ceil_div(a.q_len, B) * a.q_heads * a.batch, a);
  a.beside = a.beside || a.dq;
  if (!rc && (a.dk || a.dv))
    rc = launch_simt<B, DP>(d, simt_dkv_kernel<B, DP>, 4, 2,
                            lnn_ceil_div(a.kv_len, B) * a.kv_heads * a.batch, a);
  return rc;
}

// ---- the cache -----------------------------------------------------------------------------------
// Slots of a sequence: the first `sinks` positions keep theirs, the later ones go round the other `window`.  A
// position p that a query at the newest one sees is in slot p (p < sinks) or sinks + (p - sinks) % window, and
// all slots below min(length, sinks + window) hold such positions: attention over the cache needs no mask.
constexpr float kMaxLength = 16777216.0f;      // lengths are exact in fp32 up to 2^24

// a sequence's length; below zero: the slot of the batch is not in use
__device__ __forceinline__ int cache_length(float x, int b, int* status) {
  if (x < 0.0f) return -1;
  if (!(x < kMaxLength) || x != floorf(x)) {
    if (atomicCAS(status, 0, LNN_E_INVALID) == 0) { status[1] = 5; status[2] = b; status[3] = (int)x; }
    return -1;
  }
  return (int)x;
}

// A row of threads per slot, columns in units of T.  Bound by its launch and one dependent load: 4 heads of 1028 slots of 128
// values in 5 us.
template <class T>
__global__ void __launch_bounds__(kThreads)
cache_store_kernel(T* __restrict__ ck, T* __restrict__ cv, float* __restrict__ lengths_out, const T* __restrict__ k,
                   const T* __restrict__ v, const float* __restrict__ lengths, int heads, int kv_len, int units, int window,
                   int sinks, int* status) {
  lnn::wait_for_previous();
  const int b = blockIdx.z, h = blockIdx.y, slots = window + sinks;
  if (lengths && __ldg(lengths + b) < 0.0f) return;               // this slot of the batch stays as it is
  const int len = lnn::attn_length(lengths, b, kv_len, status);
  if (blockIdx.x == 0 && h == 0 && threadIdx.x + threadIdx.y == 0) lengths_out[b] = (float)len;
  const int64_t src = ((int64_t)b * heads + h) * kv_len * units, dst = ((int64_t)b * heads + h) * slots * units;
  const int used = min(len, slots);
  for (int slot = blockIdx.x * blockDim.y + threadIdx.y; slot < used; slot += gridDim.x * blockDim.y) {
    // the latest position that lives in this slot
    const int p = slot < sinks ? slot : slot + (len - 1 - slot) / window * window;
    const int64_t from = src + (int64_t)p * units, to = dst + (int64_t)slot * units;
    for (int c = threadIdx.x; c < units; c += blockDim.x) {
      const T x = k[from + c], y = v[from + c];
      ck[to + c] = x;
      cv[to + c] = y;
    }
  }
}

template <class T>
int cache_store(lnn::Device* d, uint64_t CK, uint64_t CV, uint64_t LEN_OUT, uint64_t K, uint64_t V, uint64_t LEN, int batch, int heads,
                int kv_len, int units, int window, int sinks) {
  unsigned x = 1;
  while (x < 64 && x < (unsigned)units) x *= 2;
  const dim3 block(x, kThreads / x);
  const int64_t blocks = std::min<int64_t>(lnn_ceil_div(std::min(kv_len, window + sinks), block.y),
                                           std::max<int64_t>(1, (int64_t)d->sm_count * 16 / ((int64_t)batch * heads)));
  LNN_CUDA(lnn::launch_chained(d, cache_store_kernel<T>, dim3((unsigned)blocks, (unsigned)heads, (unsigned)batch), block, 0,
                               (T*)(uintptr_t)CK, (T*)(uintptr_t)CV, (float*)(uintptr_t)LEN_OUT, (const T*)(uintptr_t)K,
                               (const T*)(uintptr_t)V, (const float*)(uintptr_t)LEN, heads, kv_len, units, window, sinks, d->status_dev));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

constexpr int kMaxStages = 8, kMaxSplits = 8;

struct StepArgs {
  float* o;
  const float *q, *k, *v;                // [batch][q_heads][dim], [batch][kv_heads][dim]
  float *ck, *cv;                        // [batch][kv_heads][sinks + window][dim]
  const float* lengths;
  float* lengths_out;
  int batch, q_heads, kv_heads, dim, window, sinks, splits, group_chunks;
  int stage_slots, stages;
  float scale;
  float down, up;                        // powers of two, down * up = 1: see StepSums
  int* status;
};

// Eight lanes share a key: each holds 4 NV of its values, and of the outputs of GC heads.  A warp takes four keys at a time,
// and every group of eight lanes has a softmax of its own, which meet at the end: within the warp by shuffles, in the
// block through shared memory and over the blocks of a cluster (the slots of one sequence and head, cut into contiguous
// shares) through distributed shared memory.  The new key and value are read from the arguments while one block writes
// them into the cache.
constexpr int kStepWarps = kThreads / 32;
// A warp has two heads at most (their queries and sums in registers; one of more than 128 values): where a block has
// more, its warps are teams.
template <int GC, int NV> constexpr int kStepHeads = GC > 1 && NV <= 4 ? 2 : 1;
template <int GC, int NV> constexpr int kStepTeams = GC / kStepHeads<GC, NV>;
template <int GC, int NV> constexpr int kStepKeys = kStepHeads<GC, NV> * NV <= 8 && NV <= 4 ? 2 : 1;      // that a group of lanes takes at a time
template <int NV> constexpr int kStepRow = NV * 32 + 2;        // values, maximum and sum of a partial result

struct StepPlace {
  int rank, hk, chunk, b, h0, heads, len, fresh, n, begin, end;
  int64_t oq, okv, oc;
  bool idle;
  __device__ __forceinline__ StepPlace(const StepArgs& a, int gc) {
    rank = blockIdx.x;                                            // the cluster runs along x
    hk = blockIdx.y / a.group_chunks; chunk = blockIdx.y % a.group_chunks; b = blockIdx.z;
    const int group = a.q_heads / a.kv_heads, slots = a.window + a.sinks;
    h0 = hk * group + chunk * gc;
    heads = min(gc, group - chunk * gc);
    const float length = __ldg(a.lengths + b);
    len = cache_length(length, b, a.status);
    if (rank == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.lengths_out[b] = len < 0 ? length : (float)(len + 1);
    oq = ((int64_t)b * a.q_heads + h0) * a.dim;
    okv = ((int64_t)b * a.kv_heads + hk) * a.dim;
    oc = okv * slots;
    idle = len < 0;                                               // the same for the whole cluster
    if (idle) {
      if (rank == 0)
        for (int i = threadIdx.x; i < heads * a.dim; i += kThreads) a.o[oq + i] = 0.0f;
      return;
    }
    fresh = len < a.sinks ? len : a.sinks + (len - a.sinks) % a.window;
    n = min(len + 1, slots);
    const int per = ((n + a.splits - 1) / a.splits + 31) / 32 * 32;
    begin = min(rank * per, n);
    end = min(begin + per, n);
  }
};

// The softmax of a group of eight lanes over the keys it has seen, for GC heads.  m is no maximum but a score that no other
// is more than kSlack above: short streams would move a maximum all the time.  Weights of up to 2^kSlack meet the values
// times `down`, a power of two for which the sum over all slots is below half of the largest value: an average of finite
// values is finite.  (The other end: a term is off by 2^-149 / down at most, which is below the normal numbers up to 2^14 slots.)
constexpr int kSlackBits = 8;
constexpr float kSlack = (float)kSlackBits;
template <int GC, int NV>
struct StepSums {
  uint64_t o[GC][2 * NV];                                        // pairs of values
  float m[GC], l[GC];
  __device__ __forceinline__ StepSums() {
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      m[g] = -FLT_MAX;
      l[g] = 0.0f;
#pragma unroll
      for (int u = 0; u < 2 * NV; ++u) o[g][u] = 0;
    }
  }
  // scores s[g][k] (the same in all eight lanes) of KEYS keys, of which the first `real` are there, and their values
  template <int KEYS>
  __device__ __forceinline__ void take(const float (&s)[GC][KEYS], int real, const uint64_t (&v)[KEYS][2 * NV], float down) {
    bool far = false;
#pragma unroll
    for (int g = 0; g < GC; ++g)
#pragma unroll
      for (int k = 0; k < KEYS; ++k) far = far || (k < real && s[g][k] > m[g] + kSlack);
    if (__any_sync(0xffffffffu, far)) {
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        float top = m[g];
#pragma unroll
        for (int k = 0; k < KEYS; ++k) top = k < real ? fmaxf(top, s[g][k]) : top;
        const float keep = exp2_fast(__fsub_rn(m[g], top));
        const uint64_t keep2 = lnn_tc::pack2(keep, keep);
        m[g] = top;
        l[g] = __fmul_rn(l[g], keep);
#pragma unroll
        for (int u = 0; u < 2 * NV; ++u) o[g][u] = lnn_tc::mul2(o[g][u], keep2);
      }
    }
#pragma unroll
    for (int g = 0; g < GC; ++g)
#pragma unroll
      for (int k = 0; k < KEYS; ++k) {
        const float e = k < real ? exp2_fast(__fsub_rn(s[g][k], m[g])) : 0.0f;
        const float low = __fmul_rn(e, down);
        const uint64_t e2 = lnn_tc::pack2(low, low);
        l[g] = __fadd_rn(l[g], e);
#pragma unroll
        for (int u = 0; u < 2 * NV; ++u) o[g][u] = lnn_tc::fma2(e2, v[k][u], o[g][u]);
      }
  }
};
// this lane's share of q . k
template <int NV>
__device__ __forceinline__ float step_dot(const uint64_t (&q)[2 * NV], const uint64_t (&k)[2 * NV]) {
  uint64_t s = 0;
#pragma unroll
  for (int u = 0; u < 2 * NV; ++u) s = lnn_tc::fma2(q[u], k[u], s);
  float x, y;
  lnn_tc::unpack2(s, x, y);
  return __fadd_rn(x, y);
}

// The sums of all threads of the cluster into the output.  smem: kStepWarps * kStepHeads + GC rows.
template <int GC, int NV>
__device__ __forceinline__ void step_finish(const StepArgs& a, const StepPlace& p, StepSums<kStepHeads<GC, NV>, NV>& t, float* smem) {
  constexpr int kRow = kStepRow<NV>, TEAMS = kStepTeams<GC, NV>, HEADS = kStepHeads<GC, NV>, WARPS = kStepWarps / TEAMS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane & 7, sub = lane >> 3;
  float* mine = smem + warp * HEADS * kRow;
  float* block = smem + kStepWarps * HEADS * kRow;
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    float top = fmaxf(t.m[g], __shfl_xor_sync(0xffffffffu, t.m[g], 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float w = exp2_fast(__fsub_rn(t.m[g], top));
    float sum = __fmul_rn(t.l[g], w);
    sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 8));
    sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 16));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      float x[4];
      lnn_tc::unpack2(t.o[g][2 * u], x[0], x[1]);
      lnn_tc::unpack2(t.o[g][2 * u + 1], x[2], x[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __fmul_rn(x[i], w);
        x[i] = __fadd_rn(x[i], __shfl_xor_sync(0xffffffffu, x[i], 8));
        x[i] = __fadd_rn(x[i], __shfl_xor_sync(0xffffffffu, x[i], 16));
        if (sub == 0) mine[g * kRow + u * 32 + part * 4 + i] = x[i];
      }
    }
    if (lane == 0) {
      mine[g * kRow + NV * 32] = top;
      mine[g * kRow + NV * 32 + 1] = sum;
    }
  }
  __syncthreads();
  // column c of COUNT partial results (those from `count` on have no weight), or with c = NV * 32 + 1 the sum of the sums;
  // and their maximum.  All are loaded at once: the ones of other blocks are far away.
  const auto join = [&](auto&& from, auto most, int count, int c) {
    constexpr int COUNT = decltype(most)::value;
    float top = -FLT_MAX, m[COUNT], x[COUNT];
#pragma unroll
    for (int w = 0; w < COUNT; ++w) {
      m[w] = w < count ? from(w)[NV * 32] : -FLT_MAX;
      x[w] = w < count ? from(w)[c] : 0.0f;
    }
#pragma unroll
    for (int w = 0; w < COUNT; ++w) top = fmaxf(top, m[w]);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < COUNT; ++w) sum = fmaf(exp2_fast(__fsub_rn(m[w], top)), x[w], sum);
    return make_float2(sum, top);
  };
  for (int i = threadIdx.x; i < GC * (NV * 32 + 1); i += kThreads) {
    const int g = i / (NV * 32 + 1), c = i % (NV * 32 + 1);
    const auto of_warp = [&](int w) { return smem + ((g / HEADS * WARPS + w) * HEADS + g % HEADS) * kRow; };
    const float2 r = join(of_warp, std::integral_constant<int, WARPS>(), WARPS, c < NV * 32 ? c : NV * 32 + 1);
    if (c < NV * 32) block[g * kRow + c] = r.x;
    else { block[g * kRow + NV * 32] = r.y; block[g * kRow + NV * 32 + 1] = r.x; }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (a.splits > 1) cluster.sync();
  else __syncthreads();
  for (int i = p.rank * kThreads + threadIdx.x; i < p.heads * a.dim; i += a.splits * kThreads) {
    const int g = i / a.dim, c = i % a.dim;
    const auto of_rank = [&](int r) { return (a.splits > 1 ? cluster.map_shared_rank(block, r) : block) + g * kRow; };
    constexpr std::integral_constant<int, kMaxSplits> most{};
    const float sum = join(of_rank, most, a.splits, NV * 32 + 1).x;
    a.o[p.oq + i] = __fmul_rn(__fdiv_rn(join(of_rank, most, a.splits, c).x, sum), a.up);
  }
  if (a.splits > 1) cluster.sync();                      // nobody leaves while its shared memory is being read
}
// One block per cluster and key head writes the new row: nobody reads it from the cache in this launch.
__device__ __forceinline__ void step_append(const StepArgs& a, const StepPlace& p) {
  if (p.rank == 0 && p.chunk == 0)
    for (int i = threadIdx.x; i < a.dim; i += kThreads) {
      a.ck[p.oc + (int64_t)p.fresh * a.dim + i] = a.k[p.okv + i];
      a.cv[p.oc + (int64_t)p.fresh * a.dim + i] = a.v[p.okv + i];
    }
}

// Rows of any alignment, straight from global memory.
template <int GC, int NV>
__global__ void __launch_bounds__(kThreads)
step_kernel(const StepArgs a) {
  extern __shared__ __align__(16) float smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane & 7, sub = lane >> 3, dim = a.dim;
  lnn::wait_for_previous();
  const StepPlace p(a, GC);
  if (p.idle) return;
  const auto load = [&](const float* row, uint64_t (&x)[2 * NV], float times) {
#pragma unroll
    for (int u = 0; u < 2 * NV; ++u) {
      const int c = u / 2 * 32 + part * 4 + u % 2 * 2;
      x[u] = lnn_tc::pack2(c < dim ? __fmul_rn(__ldg(row + c), times) : 0.0f, c + 1 < dim ? __fmul_rn(__ldg(row + c + 1), times) : 0.0f);
    }
  };
  constexpr int HEADS = kStepHeads<GC, NV>, WARPS = kStepWarps / kStepTeams<GC, NV>;
  const int team = warp / WARPS, turn = warp % WARPS;
  uint64_t q[HEADS][2 * NV];
#pragma unroll
  for (int g = 0; g < HEADS; ++g) load(a.q + p.oq + min(team * HEADS + g, p.heads - 1) * dim, q[g], a.scale * lnn::kLog2e);
  StepSums<HEADS, NV> t;
  for (int s0 = p.begin; s0 < p.end; s0 += 4 * WARPS) {
    const int slot = s0 + turn * 4 + sub, from = min(slot, p.end - 1);
    uint64_t k[2 * NV], v[1][2 * NV];
    load(from == p.fresh ? a.k + p.okv : a.ck + p.oc + (int64_t)from * dim, k, 1.0f);
    load(from == p.fresh ? a.v + p.okv : a.cv + p.oc + (int64_t)from * dim, v[0], 1.0f);
    float s[HEADS][1];
#pragma unroll
    for (int g = 0; g < HEADS; ++g) {
      s[g][0] = step_dot<NV>(q[g], k);
#pragma unroll
      for (int x = 4; x > 0; x >>= 1) s[g][0] = __fadd_rn(s[g][0], __shfl_xor_sync(0xffffffffu, s[g][0], x));
    }
    t.template take<1>(s, slot < p.end ? 1 : 0, v, a.down);
  }
  step_append(a, p);
  step_finish<GC, NV>(a, p, t, smem);
}

// Bound by HBM (figures at the top).  Rows of 16-byte units: the slots of a share are one piece of memory, which bulk copies
// bring into a ring of stages in shared memory; two blocks per SM have up to 192 KB on the way.  FULL: dim = 32 NV.
template <int GC, int NV, bool FULL>
__global__ void __launch_bounds__(kThreads, 2)
step_bulk_kernel(const StepArgs a) {
  extern __shared__ __align__(16) float smem[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ int abort_flag_smem;
  constexpr int HEADS = kStepHeads<GC, NV>, WARPS = kStepWarps / kStepTeams<GC, NV>, KEYS = kStepKeys<GC, NV>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane & 7, sub = lane >> 3;
  const int team = warp / WARPS, turn = warp % WARPS, dim = FULL ? NV * 32 : a.dim;
  lnn::wait_for_previous();
  const StepPlace p(a, GC);
  if (p.idle) return;
  const int per_stage = a.stage_slots, steps = (p.end - p.begin + per_stage - 1) / per_stage;
  const int stage_floats = 2 * per_stage * dim;
  const auto fetch = [&](int i, int stage) {                     // by one thread: K and V of step i
    const int first = p.begin + i * per_stage, count = min(per_stage, p.end - first);
    const uint32_t bar = lnn_tc::smem_u32(&full[stage]), bytes = (uint32_t)(count * dim * 4);
    const uint32_t dst = lnn_tc::smem_u32(smem + stage * stage_floats);
    lnn_tc::mbar_expect_tx(bar, 2 * bytes);
    lnn_tc::bulk_load(dst, a.ck + p.oc + (int64_t)first * dim, bytes, bar);
    lnn_tc::bulk_load(dst + per_stage * dim * 4, a.cv + p.oc + (int64_t)first * dim, bytes, bar);
  };
  if (threadIdx.x == 0) {
    abort_flag_smem = 0;
    for (int i = 0; i < a.stages; ++i) {
      lnn_tc::mbar_init(lnn_tc::smem_u32(&full[i]), 1);
      lnn_tc::mbar_init(lnn_tc::smem_u32(&empty[i]), kStepWarps);
    }
    lnn_tc::fence_barrier_init();
    for (int i = 0; i < min(a.stages, steps); ++i) fetch(i, i);
  }
  const float factor = a.scale * lnn::kLog2e;
  uint64_t q[HEADS][2 * NV];
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    const float* from = a.q + p.oq + min(team * HEADS + g, p.heads - 1) * dim + part * 4;      // (a head too many is not stored)
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const float4 v = FULL || u * 32 + part * 4 < dim ? __ldg(reinterpret_cast<const float4*>(from + u * 32)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      q[g][2 * u] = lnn_tc::pack2(v.x * factor, v.y * factor);
      q[g][2 * u + 1] = lnn_tc::pack2(v.z * factor, v.w * factor);
    }
  }
  __syncthreads();
  StepSums<HEADS, NV> t;
  bool ok = true;
  int stage = 0, before = 0;
  uint32_t phase = 0, phase_before = 0;
  for (int i = 0; i < steps; ++i) {
    const int first = p.begin + i * per_stage, count = min(per_stage, p.end - first), fresh = p.fresh - first;
    if (warp == 0 && i > 0 && i - 1 + a.stages < steps) {         // the stage before this one is filled again
      ok = lnn_tc::mbar_wait(lnn_tc::smem_u32(&empty[before]), phase_before, &abort_flag_smem, a.status, 41, i);
      if (ok && lane == 0) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (a new row was written by ordinary stores)
        fetch(i - 1 + a.stages, before);
      }
    }
    float* K = smem + stage * stage_floats;
    float* V = K + per_stage * dim;
    ok = ok && lnn_tc::mbar_wait(lnn_tc::smem_u32(&full[stage]), phase, &abort_flag_smem, a.status, 40, i);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    // KEYS keys of a group at a time, 4 apart: the warps of a team take pieces of 4 KEYS slots
    for (int base = turn * 4 * KEYS; base < count; base += 4 * KEYS * WARPS) {
      const int at = base + sub, real = KEYS == 2 && at + 4 < count ? 2 : (at < count ? 1 : 0);
      if (fresh >= base && fresh < base + 4 * KEYS) {             // the row's place in the cache is being written
        for (int c = lane; c < dim; c += 32) {
          K[fresh * dim + c] = __ldg(a.k + p.okv + c);           // (each team writes it: the same values)
          V[fresh * dim + c] = __ldg(a.v + p.okv + c);
        }
        __syncwarp();
      }
      // (what is not there is read from the last slot that is, and has no weight)
      uint64_t x[KEYS][2 * NV];
      const auto load = [&](const float* rows) {
#pragma unroll
        for (int k = 0; k < KEYS; ++k) {
          const float* r = rows + min(at + 4 * k, count - 1) * dim + part * 4;
#pragma unroll
          for (int u = 0; u < NV; ++u) {
            const ulonglong2 v = FULL || u * 32 + part * 4 < dim ? *reinterpret_cast<const ulonglong2*>(r + u * 32) : make_ulonglong2(0, 0);
            x[k][2 * u] = v.x; x[k][2 * u + 1] = v.y;
          }
        }
      };
      load(K);
      float s[HEADS][KEYS];
#pragma unroll
      for (int g = 0; g < HEADS; ++g)
#pragma unroll
        for (int k = 0; k < KEYS; ++k) s[g][k] = step_dot<NV>(q[g], x[k]);
      load(V);
#pragma unroll
      for (int y = 4; y > 0; y >>= 1)
#pragma unroll
        for (int g = 0; g < HEADS; ++g)
#pragma unroll
          for (int k = 0; k < KEYS; ++k) s[g][k] = __fadd_rn(s[g][k], __shfl_xor_sync(0xffffffffu, s[g][k], y));
      t.template take<KEYS>(s, real, x, a.down);
    }
    __syncwarp();
    if (lane == 0) lnn_tc::mbar_arrive(lnn_tc::smem_u32(&empty[stage]));
    before = stage;
    phase_before = phase;
    if (++stage == a.stages) { stage = 0; phase ^= 1u; }
  }
  if (__syncthreads_or(!ok)) {
    // copies that are still on their way must not land in what comes next
    const long long t0 = clock64();
    while (clock64() - t0 < lnn_tc::kAbortDelay) { }
  }
  __syncthreads();
  step_append(a, p);
  step_finish<GC, NV>(a, p, t, smem);
}

template <int GC, int NV>
int launch_step(lnn::Device* d, StepArgs& a, bool vec) {
  const int group = a.q_heads / a.kv_heads, slots = a.window + a.sinks;
  a.group_chunks = (group + GC - 1) / GC;
  const int64_t clusters = (int64_t)a.batch * a.kv_heads * a.group_chunks;
  a.splits = 1;
  while (a.splits < kMaxSplits && clusters * a.splits < 2 * d->sm_count && slots >= a.splits * 2 * 64) a.splits *= 2;
  LNN_REQUIRE((int64_t)a.kv_heads * a.group_chunks < 65536, "too many heads");
  const size_t join = (size_t)(kStepWarps * kStepHeads<GC, NV> + GC) * kStepRow<NV> * 4;
  size_t bytes = join;
  void (*kernel)(const StepArgs) = step_kernel<GC, NV>;
  if (vec) {
    // stages of 32 KB or less, a turn of a team's warps at least, as many as two blocks per SM have room for or the share has slots for
    const int share = (slots + a.splits - 1) / a.splits;
    a.stage_slots = 4 * kStepKeys<GC, NV> * kStepWarps / kStepTeams<GC, NV>;
    while (a.stage_slots * 2 * a.dim * 8 <= 32768 && a.stage_slots < share) a.stage_slots *= 2;
    const int stage = a.stage_slots * a.dim * 8;
    a.stages = std::max(1, std::min({kMaxStages, 104 * 1024 / stage, (share + a.stage_slots - 1) / a.stage_slots}));
    bytes = std::max(join, (size_t)a.stages * stage);
    kernel = a.dim == NV * 32 ? step_bulk_kernel<GC, NV, true> : step_bulk_kernel<GC, NV, false>;
  }
  if (bytes > 47 * 1024)                                         // (barriers come on top)
    LNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.splits, (unsigned)(a.kv_heads * a.group_chunks), (unsigned)a.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = d->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.splits > 1 ? 2 : 1;
  LNN_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}
template <int NV>
int launch_step(lnn::Device* d, StepArgs& a, bool vec) {
  const int group = a.q_heads / a.kv_heads;
  if (group == 1) return launch_step<1, NV>(d, a, vec);
  if (group == 2) return launch_step<2, NV>(d, a, vec);
  return launch_step<4, NV>(d, a, vec);
}

const float* in(uint64_t p) { return (const float*)(uintptr_t)p; }
float* out(uint64_t p) { return (float*)(uintptr_t)p; }

int check_geom(const lnn_attn_geom* g) {
  LNN_REQUIRE(g && g->batch > 0 && g->q_heads > 0 && g->kv_heads > 0 && g->q_len > 0 && g->kv_len > 0 && g->dim > 0, "bad geometry");
  LNN_REQUIRE(g->q_heads % g->kv_heads == 0, "%d query heads over %d key heads", g->q_heads, g->kv_heads);
  LNN_REQUIRE(g->q_len <= g->kv_len, "%d queries over %d keys", g->q_len, g->kv_len);
  LNN_REQUIRE(g->dim <= 256, "heads of %d values: at most 256", g->dim);
  LNN_REQUIRE(g->window > 0 && g->sinks >= 0, "window %d, sinks %d", g->window, g->sinks);
  LNN_REQUIRE(g->batch < 65536 && g->q_heads < 65536 && g->kv_len <= (1 << 24), "geometry too large");
  return LNN_OK;
}

AttnArgs attn_args(lnn::Device* d, const lnn_attn_geom* g, uint64_t Q, uint64_t K, uint64_t V, uint64_t LEN) {
  AttnArgs a = {};
  a.q = in(Q); a.k = in(K); a.v = in(V); a.lengths = in(LEN);
  a.batch = g->batch; a.q_heads = g->q_heads; a.kv_heads = g->kv_heads; a.q_len = g->q_len; a.kv_len = g->kv_len;
  a.dim = g->dim; a.scale = g->scale;
  a.window = g->window < g->kv_len ? g->window : g->kv_len;       // (positions end there: no sum below passes 2^31)
  a.sinks = g->sinks < g->kv_len ? g->sinks : g->kv_len;
  int bits = 1;
  while ((1 << (bits - 1)) < g->kv_len) ++bits;
  a.up = (float)(1 << bits); a.down = 1.0f / a.up;
  a.status = d->status_dev;
  return a;
}

}  // namespace

namespace lnn {

// Few tiles: of 32 rows instead of 64, twice as many blocks of which each has half the way to go (us for 4 and 64 heads of 64
// positions of 64 values: 12.7 -> 10.1 and 13.1 -> 12.3, with gradients 35.5 -> 29.4 and 40.5 -> 35.8; of 16 rows: 13.8, 17.4).
int attn_simt_fwd(Device* d, const AttnArgs& a) {
  const bool few = !a.info && lnn_ceil_div(a.q_len, 64) * a.q_heads * a.batch * 2 <= d->sm_count;
  if (few && a.dim <= 32) return simt_fwd<32, 32>(d, a);
  if (few && a.dim <= 64) return simt_fwd<32, 64>(d, a);
  if (few && a.dim <= 128) return simt_fwd<32, 128>(d, a);
  if (a.dim <= 32) return simt_fwd<64, 32>(d, a);
  if (a.dim <= 64) return simt_fwd<64, 64>(d, a);
  if (a.dim <= 128) return simt_fwd<64, 128>(d, a);
  return simt_fwd<32, 256>(d, a);
}

int attn_simt_bwd(Device* d, const AttnArgs& a) {
  const bool few = !a.info && lnn_ceil_div(a.kv_len, 64) * a.kv_heads * a.batch * 2 <= d->sm_count;
  if (few && a.dim <= 32) return simt_bwd<32, 32>(d, a);
  if (few && a.dim <= 64) return simt_bwd<32, 64>(d, a);
  if (few && a.dim <= 128) return simt_bwd<32, 128>(d, a);
  if (a.dim <= 32) return simt_bwd<64, 32>(d, a);
  if (a.dim <= 64) return simt_bwd<64, 64>(d, a);
  if (a.dim <= 128) return simt_bwd<64, 128>(d, a);
  return simt_bwd<32, 256>(d, a);
}

int attn_delta(Device* d, float* delta, const float* dout, const float* o, int64_t rows, int dim) {
  LNN_CUDA(launch_chained(d, attn_delta_kernel, (unsigned)lnn_ceil_div(rows, kThreads / 32), kThreads, 0, delta, dout, o, rows, dim));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

}  // namespace lnn

extern "C" {

int lnn_sink_attn_fwd(int dev, uint64_t O, uint64_t LSE, uint64_t Q, uint64_t K, uint64_t V, uint64_t LEN, const lnn_attn_geom* g) {
  LNN_DEV(d, dev);
  int rc = check_geom(g);
  if (rc) return rc;
  LNN_REQUIRE(O && LSE && LSE % 8 == 0 && Q && K && V, "bad arguments");
  AttnArgs a = attn_args(d, g, Q, K, V, LEN);
  a.o = out(O); a.lse = out(LSE);
  return lnn::attn_tc_applicable(a) ? lnn::attn_tc_fwd(d, a) : lnn::attn_simt_fwd(d, a);
}

int lnn_sink_attn_bwd(int dev, uint64_t dQ, uint64_t dK, uint64_t dV, uint64_t Q, uint64_t K, uint64_t V, uint64_t O, uint64_t LSE,
                      uint64_t LEN, uint64_t dO, const lnn_attn_geom* g, int acc_q, int acc_k, int acc_v) {
  LNN_DEV(d, dev);
  int rc = check_geom(g);
  if (rc) return rc;
  LNN_REQUIRE(Q && K && V && O && LSE && LSE % 8 == 0 && dO, "bad arguments");
  AttnArgs a = attn_args(d, g, Q, K, V, LEN);
  a.o = out(O); a.lse = out(LSE); a.dout = in(dO);
  a.dq = out(dQ); a.dk = out(dK); a.dv = out(dV);
  a.acc_q = acc_q; a.acc_k = acc_k; a.acc_v = acc_v;
  if (lnn::attn_tc_applicable(a)) return lnn::attn_tc_bwd(d, a);
  const int64_t rows = (int64_t)g->batch * g->q_heads * g->q_len;
  lnn::Scratch delta(d);
  rc = delta.get((uint64_t)rows * 4);
  if (!rc) rc = lnn::attn_delta(d, delta.as<float>(), in(dO), in(O), rows, g->dim);
  if (rc) return rc;
  a.delta = delta.as<float>(); a.delta_pitch = g->q_len;
  return lnn::attn_simt_bwd(d, a);
}

int lnn_sink_cache_store(int dev, uint64_t CK, uint64_t CV, uint64_t LEN_OUT, uint64_t K, uint64_t V, uint64_t LEN, int batch,
                         int heads, int kv_len, int dim, int window, int sinks) {
  LNN_DEV(d, dev);
  LNN_REQUIRE(CK && CV && LEN_OUT && LEN_OUT != LEN && K && V && batch > 0 && heads > 0 && kv_len > 0 && dim > 0 && window > 0 && sinks >= 0,
              "bad arguments");
  LNN_REQUIRE(batch < 65536 && heads < 65536 && kv_len <= (1 << 24) && (int64_t)window + sinks <= (1 << 24), "geometry too large");
  if (dim % 4 == 0 && ((CK | CV | K | V) & 15) == 0)
    return cache_store<float4>(d, CK, CV, LEN_OUT, K, V, LEN, batch, heads, kv_len, dim / 4, window, sinks);
  return cache_store<float>(d, CK, CV, LEN_OUT, K, V, LEN, batch, heads, kv_len, dim, window, sinks);
}

int lnn_sink_attn_step(int dev, uint64_t O, uint64_t Q, uint64_t K, uint64_t V, uint64_t CK, uint64_t CV, uint64_t LEN,
                       uint64_t LEN_OUT, int batch, int q_heads, int kv_heads, int dim, int window, int sinks, float scale) {
  LNN_DEV(d, dev);
  LNN_REQUIRE(O && Q && K && V && CK && CV && LEN && LEN_OUT && LEN != LEN_OUT, "bad arguments");
  LNN_REQUIRE(batch > 0 && q_heads > 0 && kv_heads > 0 && dim > 0 && window > 0 && sinks >= 0 && q_heads % kv_heads == 0,
              "bad arguments");
  LNN_REQUIRE(dim <= 256, "heads of %d values: at most 256", dim);
  LNN_REQUIRE(batch < 65536 && (int64_t)window + sinks <= (1 << 24), "geometry too large");
  StepArgs a = {};
  a.o = out(O); a.q = in(Q); a.k = in(K); a.v = in(V); a.ck = out(CK); a.cv = out(CV);
  a.lengths = in(LEN); a.lengths_out = out(LEN_OUT);
  a.batch = batch; a.q_heads = q_heads; a.kv_heads = kv_heads; a.dim = dim; a.window = window; a.sinks = sinks;
  a.scale = scale; a.status = d->status_dev;
  int bits = kSlackBits + 1;
  while ((1 << (bits - kSlackBits - 1)) < window + sinks) ++bits;
  a.up = (float)(1ll << bits); a.down = 1.0f / a.up;
  const bool vec = dim % 4 == 0 && ((Q | K | V | CK | CV) & 15) == 0;
  if (dim <= 32) return launch_step<1>(d, a, vec);
  if (dim <= 64) return launch_step<2>(d, a, vec);
  if (dim <= 96) return launch_step<3>(d, a, vec);
  if (dim <= 128) return launch_step<4>(d, a, vec);
  return launch_step<8>(d, a, vec);
}

}  // extern "C"
