// Operators on tokens: rows of a table and their gradient, the logarithm of a token's probability, the clipped
// policy loss.  Token numbers are whole numbers in fp32 (exact to 2^24); one below zero marks a padded place, which
// gives zeros and no gradient.  Anything else that is no row of the table is treated as padding and leaves
// LNN_E_INVALID in the device status, so that the next read of a result raises.
//
// All of them are bound by HBM.
#include <cooperative_groups.h>
#include <float.h>
#include <math_constants.h>
#include <algorithm>
#include "lnn_common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;

// ---- token numbers -----------------------------------------------------------------------------
// The row a token stands for, or -1.
__device__ __forceinline__ int token_row(float id, int vocab, int64_t at, int what, int* status) {
  if (id < 0.0f) return -1;
  if (!(id < (float)vocab) || id != floorf(id)) {
    if (atomicCAS(status, 0, LNN_E_INVALID) == 0) {
      status[1] = what;
      status[2] = (int)at;
      status[3] = (int)id;
    }
    return -1;
  }
  return (int)id;
}

// ---- embedding ---------------------------------------------------------------------------------
template <class T> __device__ __forceinline__ T scaled(T v, float s);
template <> __device__ __forceinline__ float scaled(float v, float s) { return __fmul_rn(v, s); }
template <> __device__ __forceinline__ float4 scaled(float4 v, float s) {
  return make_float4(__fmul_rn(v.x, s), __fmul_rn(v.y, s), __fmul_rn(v.z, s), __fmul_rn(v.w, s));
}
template <class T> __device__ __forceinline__ T plus(T a, T b);
template <> __device__ __forceinline__ float plus(float a, float b) { return __fadd_rn(a, b); }
template <> __device__ __forceinline__ float4 plus(float4 a, float4 b) {
  return make_float4(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y), __fadd_rn(a.z, b.z), __fadd_rn(a.w, b.w));
}
template <class T> __device__ __forceinline__ T nothing();
template <> __device__ __forceinline__ float nothing() { return 0.0f; }
template <> __device__ __forceinline__ float4 nothing() { return make_float4(0.0f, 0.0f, 0.0f, 0.0f); }

// A sum of values T with what its additions have rounded off beside it (Knuth's two-sum): a frequent token's row has
// thousands of terms in pieces.
template <class T> struct Sum;
template <> struct Sum<float> {
  float v = 0.0f, rest = 0.0f;
  __device__ __forceinline__ void add(float x) {
    const float s = __fadd_rn(v, x), b = __fsub_rn(s, v);
    rest = __fadd_rn(rest, __fadd_rn(__fsub_rn(v, __fsub_rn(s, b)), __fsub_rn(x, b)));
    v = s;
  }
  // (a sum that is not finite leaves nothing to add)
  __device__ __forceinline__ float rounded(float scale) const { return __fmul_rn(fabsf(v) <= FLT_MAX ? __fadd_rn(v, rest) : v, scale); }
};
template <> struct Sum<float4> {
  Sum<float> x, y, z, w;
  __device__ __forceinline__ void add(float4 v) { x.add(v.x); y.add(v.y); z.add(v.z); w.add(v.w); }
  __device__ __forceinline__ float4 rounded(float s) const { return make_float4(x.rounded(s), y.rounded(s), z.rounded(s), w.rounded(s)); }
};

// One row of threads (blockDim.x) per token, columns in units of T.  Bound by HBM: 16384 tokens of 768 values, 100 MB in 18.6 us,
// 5.4 TB/s.
template <class T>
__global__ void __launch_bounds__(kThreads)
embedding_fwd_kernel(T* __restrict__ Y, const T* __restrict__ table, const float* __restrict__ ids, int64_t tokens,
                     int vocab, int64_t units, float scale, int* status) {
  lnn::wait_for_previous();
  for (int64_t n = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; n < tokens; n += (int64_t)gridDim.x * blockDim.y) {
    const int row = token_row(__ldg(ids + n), vocab, n, 1, status);
    for (int64_t c = threadIdx.x; c < units; c += blockDim.x)
      Y[n * units + c] = row < 0 ? nothing<T>() : scaled(__ldg(table + row * units + c), scale);
  }
}

// ---- gradient of the table ---------------------------------------------------------------------
// Tokens are sorted by row, stably (radix sort, 8 bits a pass), so that the terms of a row are added in the order
// of the tokens whatever the launch looks like: no atomics on values.  One cluster of eight blocks sorts: its passes are
// short chains of dependent steps, which meet in distributed shared memory instead of at the ends of kernels (16384 tokens of
// 50001 rows: four launches took 32 us), and the other clusters write the zeros of the rows without tokens meanwhile: 154 MB in
// 27 us, 5.7 TB/s, behind which the sort is over.
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kSortBlocks = 8;
constexpr int kSortKeys = 4;                       // per lane at a time

struct SortArgs {
  const float* ids;
  uint32_t *keys[2], *at[2];                       // by turns; the last pass leaves its result in keys[(passes - 1) & 1]
  int64_t n;
  int vocab, passes;
  float4* zeros;                                   // the table in 16-byte units, and the floats in front and behind
  int64_t quads;
  float *lead, *tail;
  int leads, tails;
  int* status;
};
constexpr uint32_t kNoKey = 0xffffffffu;

// The lanes whose key has this lane's digit; none for a lane without a key.  Eight votes take a fraction of the time of one
// __match_any_sync.
__device__ __forceinline__ uint32_t same_digit(uint32_t key, int shift) {
  uint32_t same = __ballot_sync(0xffffffffu, key != kNoKey);
#pragma unroll
  for (int bit = 0; bit < 8; ++bit) {
    const bool one = (key >> (shift + bit)) & 1u;
    const uint32_t ones = __ballot_sync(0xffffffffu, one);
    same &= one ? ones : ~ones;
  }
  return key == kNoKey ? 0u : same;
}

__global__ void __launch_bounds__(kSortThreads, 2) __cluster_dims__(kSortBlocks, 1, 1)
sort_tokens_kernel(const __grid_constant__ SortArgs a) {
  __shared__ uint32_t count[kSortWarps][256];
  __shared__ uint32_t hist[256], warp_total[8];
  lnn::wait_for_previous();
  if (blockIdx.x >= kSortBlocks) {
    const int64_t first = (int64_t)(blockIdx.x - kSortBlocks) * kSortThreads + threadIdx.x;
    const int64_t stride = (int64_t)(gridDim.x - kSortBlocks) * kSortThreads;
    for (int64_t i = first; i < a.quads; i += stride) a.zeros[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (first < a.leads) a.lead[first] = 0.0f;
    if (first < a.tails) a.tail[first] = 0.0f;
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block = blockIdx.x;
  // a contiguous strip of the tokens per warp, in the order of the warps
  const int64_t per = ((a.n + kSortBlocks * kSortWarps - 1) / (kSortBlocks * kSortWarps) + 31) / 32 * 32;
  const int64_t begin = min((int64_t)(block * kSortWarps + warp) * per, a.n), end = min(begin + per, a.n);
  const bool once = per <= kSortKeys * 32;                       // a strip's keys stay in registers
  uint32_t key[kSortKeys], same[kSortKeys];
  for (int pass = 0; pass < a.passes; ++pass) {
    const uint32_t *keys = a.keys[(pass + 1) & 1], *from = a.at[(pass + 1) & 1];
    uint32_t *out_keys = a.keys[pass & 1], *out_at = a.at[pass & 1];
    const int shift = 8 * pass;
    const auto load = [&](int64_t i0) {
#pragma unroll
      for (int u = 0; u < kSortKeys; ++u) {
        const int64_t i = i0 + u * 32 + lane;
        key[u] = kNoKey;
        if (i < end) {
          if (pass > 0) {
            key[u] = __ldcg(keys + i);                           // (written by other blocks of this kernel)
          } else {
            const int row = token_row(__ldg(a.ids + i), a.vocab, i, 2, a.status);
            key[u] = row < 0 ? (uint32_t)a.vocab : (uint32_t)row;      // padding comes last
          }
        }
      }
    };
    for (int i = threadIdx.x; i < kSortWarps * 256; i += kSortThreads) (&count[0][0])[i] = 0;
    load(begin);
    __syncthreads();
    for (int64_t i0 = begin; i0 < end; i0 += kSortKeys * 32) {
      if (i0 > begin) load(i0);
#pragma unroll
      for (int u = 0; u < kSortKeys; ++u) {
        if (i0 + u * 32 >= end) break;
        same[u] = same_digit(key[u], shift);
        if (lane == __ffs(same[u]) - 1) count[warp][(key[u] >> shift) & 255u] += __popc(same[u]);
        __syncwarp();
      }
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      uint32_t total = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) total += count[w][threadIdx.x];
      hist[threadIdx.x] = total;
    }
    cluster.sync();
    // where this block's tokens of digit threadIdx.x begin: all smaller digits, then the blocks before this one
    uint32_t before = 0, total = 0, scan = 0;
    if (threadIdx.x < 256) {
      uint32_t h[kSortBlocks];
#pragma unroll
      for (int b = 0; b < kSortBlocks; ++b) h[b] = cluster.map_shared_rank(hist, b)[threadIdx.x];
#pragma unroll
      for (int b = 0; b < kSortBlocks; ++b) {
        if (b < block) before += h[b];
        total += h[b];
      }
      scan = total;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
      }
      if (lane == 31) warp_total[warp] = scan;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      for (int w = 0; w < warp; ++w) scan += warp_total[w];
      uint32_t base = scan - total + before;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w][threadIdx.x];
        count[w][threadIdx.x] = base;
        base += c;
      }
    }
    __syncthreads();
    for (int64_t i0 = begin; i0 < end; i0 += kSortKeys * 32) {
      if (!once) load(i0);
#pragma unroll
      for (int u = 0; u < kSortKeys; ++u) {
        if (i0 + u * 32 >= end) break;
        const int64_t i = i0 + u * 32 + lane;
        const uint32_t digit = (key[u] >> shift) & 255u;
        if (!once) same[u] = same_digit(key[u], shift);
        uint32_t to = 0;
        if (same[u]) to = count[warp][digit] + __popc(same[u] & ((1u << lane) - 1u));
        __syncwarp();
        if (same[u]) {
          if (lane == __ffs(same[u]) - 1) count[warp][digit] += __popc(same[u]);
          __stcg(out_keys + to, key[u]);
          __stcg(out_at + to, pass > 0 ? __ldcg(from + i) : (uint32_t)i);
        }
        __syncwarp();
      }
    }
    __threadfence();
    cluster.sync();                                              // the next pass reads what all have written; hist is free
  }
}

// Sums of the sorted tokens, kPiece of them per row of threads.  What a piece holds of a row that starts in an earlier
// piece goes to head[piece], the beginning of one that goes on behind it to tail[piece]; table_join_kernel adds those.
// Bound by waiting more than by bytes: 16384 tokens of 768 values, 50 MB read, 28 of rows and 3 of parts written, in 18 us (4.4 TB/s;
// the lookup has 5.4) for 512 blocks of four batches of loads each, and 10 us for the joins, of which the most frequent token's (a
// thousand of 16384) is a chain of five.
constexpr int kPiece = 32;

template <class T>
__global__ void __launch_bounds__(kThreads)
table_grad_kernel(T* __restrict__ dtable, const T* __restrict__ dy, const uint32_t* __restrict__ keys,
                  const uint32_t* __restrict__ at, T* __restrict__ head, T* __restrict__ tail, int64_t tokens, int vocab,
                  int64_t units, float scale, int accumulate) {
  // the block's sorted tokens, read once: the sums then wait for one load, not for three that depend on one another
  __shared__ uint32_t key_of[kThreads / 32 * kPiece], token_of[kThreads / 32 * kPiece];
  lnn::wait_for_previous();
  const int64_t pieces = (tokens + kPiece - 1) / kPiece;
  const int64_t piece = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t lo = piece * kPiece, hi = min(lo + kPiece, tokens);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = tid; i < (int)blockDim.y * kPiece; i += kThreads) {
    const int64_t e = (int64_t)blockIdx.x * blockDim.y * kPiece + i;
    if (e < tokens) {
      key_of[i] = __ldg(keys + e);
      token_of[i] = __ldg(at + e);
    }
  }
  const uint32_t before = lo > 0 && lo < tokens ? __ldg(keys + lo - 1) : (uint32_t)vocab;
  const uint32_t behind = hi < tokens ? __ldg(keys + hi) : (uint32_t)vocab;
  __syncthreads();
  if (piece >= pieces) return;
  const uint32_t *key = key_of + threadIdx.y * kPiece, *token = token_of + threadIdx.y * kPiece;
  const int n = (int)(hi - lo);
  for (int64_t c = threadIdx.x + (int64_t)blockIdx.y * blockDim.x; c < units; c += (int64_t)gridDim.y * blockDim.x) {
    uint32_t cur = key[0];
    bool continued = before == cur;
    T sum = nothing<T>();
    for (int e0 = 0; e0 < n; e0 += 8) {
      T v[8];
      uint32_t k[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const bool in = e0 + u < n;
        k[u] = in ? key[e0 + u] : cur;
        v[u] = in && k[u] < (uint32_t)vocab ? __ldg(dy + (int64_t)token[e0 + u] * units + c) : nothing<T>();
      }
      if (e0 + 8 <= n && k[0] == cur && k[7] == cur) {            // (sorted: all eight) pairs of pairs: fewer roundings
        sum = plus(sum, plus(plus(plus(v[0], v[1]), plus(v[2], v[3])), plus(plus(v[4], v[5]), plus(v[6], v[7]))));
        continue;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (e0 + u < n) {
          if (k[u] != cur) {
            if (continued) {
              head[piece * units + c] = sum;
            } else {
              T* o = dtable + cur * units + c;
              *o = accumulate ? plus(*o, scaled(sum, scale)) : scaled(sum, scale);
            }
            cur = k[u];
            continued = false;
            sum = v[u];
          } else {
            sum = plus(sum, v[u]);
          }
        }
      }
    }
    if (cur >= (uint32_t)vocab) continue;
    if (continued) {
      head[piece * units + c] = sum;
    } else if (behind == cur) {
      tail[piece * units + c] = sum;
    } else {
      T* o = dtable + cur * units + c;
      *o = accumulate ? plus(*o, scaled(sum, scale)) : scaled(sum, scale);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
table_join_kernel(T* __restrict__ dtable, const uint32_t* __restrict__ keys, const T* __restrict__ head,
                  const T* __restrict__ tail, int64_t tokens, int vocab, int64_t units, float scale, int accumulate) {
  lnn::wait_for_previous();
  const int64_t pieces = (tokens + kPiece - 1) / kPiece;
  const int64_t piece = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (piece + 1 >= pieces) return;
  const int64_t lo = piece * kPiece, hi = lo + kPiece;
  const uint32_t row = keys[hi - 1];
  if (row >= (uint32_t)vocab || keys[hi] != row) return;                    // nothing goes on behind this piece
  if (keys[lo] == row && lo > 0 && keys[lo - 1] == row) return;             // it began earlier
  // the last piece that has some of the row: it begins with it.  Eight pieces are looked at at once, further apart each time.
  int64_t last = piece + 1, step = 1;
  const auto advance = [&]() {
    int found = 0;
#pragma unroll
    for (int u = 1; u <= 8; ++u) {
      const int64_t p = last + u * step;
      found += p < pieces && __ldg(keys + p * kPiece) == row ? 1 : 0;
    }
    last += found * step;
    return found;
  };
  while (advance() == 8) step *= 8;
  for (step /= 8; step > 0; step /= 8) advance();
  for (int64_t c = threadIdx.x + (int64_t)blockIdx.y * blockDim.x; c < units; c += (int64_t)gridDim.y * blockDim.x) {
    Sum<T> sum;
    sum.add(tail[piece * units + c]);
    for (int64_t p0 = piece + 1; p0 <= last; p0 += 16) {
      T v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = p0 + u <= last ? __ldg(head + (p0 + u) * units + c) : nothing<T>();
#pragma unroll
      for (int u = 0; u < 16; ++u)
        if (p0 + u <= last) sum.add(v[u]);
    }
    T* o = dtable + row * units + c;
    *o = accumulate ? plus(*o, sum.rounded(scale)) : sum.rounded(scale);
  }
}

// Threads along the columns of a row and rows per block.
dim3 row_block(int64_t units, unsigned x = 1) {
  while (x < kThreads && x < units) x *= 2;
  return dim3(x, kThreads / x);
}

bool aligned16(const void* a, const void* b, int64_t cols) {
  return cols % 4 == 0 && (((uintptr_t)a | (uintptr_t)b) & 15) == 0;
}

template <class T>
int embedding_bwd(lnn::Device* d, T* dtable, const T* dy, const float* ids, int64_t tokens, int vocab, int64_t units,
                  float scale, int accumulate) {
  const int64_t pieces = lnn_ceil_div(tokens, kPiece);
  lnn::Scratch keys(d), parts(d);
  const int64_t pad = (tokens + 3) / 4 * 4;
  int rc = keys.get((uint64_t)(4 * pad) * 4);
  if (!rc && pieces > 1) rc = parts.get((uint64_t)pieces * units * sizeof(T) * 2);
  if (rc) return rc;
  uint32_t* buf = keys.as<uint32_t>();
  SortArgs a = {};
  for (int i = 0; i < 2; ++i) { a.keys[i] = buf + i * pad; a.at[i] = buf + (2 + i) * pad; }
  a.ids = ids; a.n = tokens; a.vocab = vocab; a.status = d->status_dev;
  a.passes = 1;
  while (((int64_t)vocab >> (8 * a.passes)) != 0) ++a.passes;             // (keys go up to vocab)
  const int64_t floats = accumulate ? 0 : (int64_t)vocab * units * (int64_t)(sizeof(T) / 4);
  float* table = reinterpret_cast<float*>(dtable);
  a.lead = table;
  a.leads = (int)std::min<int64_t>((4 - (((uintptr_t)table >> 2) & 3)) & 3, floats);
  a.zeros = reinterpret_cast<float4*>(table + a.leads);
  a.quads = (floats - a.leads) / 4;
  a.tail = table + a.leads + a.quads * 4;
  a.tails = (int)(floats - a.leads - a.quads * 4);
  // a block writes 64 KB of zeros: small enough to even out over SMs of which a cluster of eight leaves some free (as many blocks as
  // SMs: 39 us for 154 MB, small ones: 30)
  const int64_t fill = lnn_ceil_div(floats, kSortThreads * 32);
  const unsigned blocks = (unsigned)(kSortBlocks + lnn_ceil_div(fill, kSortBlocks) * kSortBlocks);
  LNN_CUDA(lnn::launch_chained(d, sort_tokens_kernel, blocks, kSortThreads, 0, a));
  LNN_CHECK_LAUNCH(d);
  const uint32_t *src_k = a.keys[(a.passes - 1) & 1], *src_at = a.at[(a.passes - 1) & 1];
  const dim3 block = row_block(units, 32);
  const dim3 grid((unsigned)lnn_ceil_div(pieces, block.y), (unsigned)std::min<int64_t>(lnn_ceil_div(units, block.x), 64));
  T *head = parts.as<T>(), *tail = head + pieces * units;
  LNN_CUDA(lnn::launch_chained(d, table_grad_kernel<T>, grid, block, 0, dtable, dy, src_k, src_at, head, tail, tokens, vocab, units, scale, accumulate));
  LNN_CHECK_LAUNCH(d);
  if (pieces > 1) {
    LNN_CUDA(lnn::launch_chained(d, table_join_kernel<T>, grid, block, 0, dtable, src_k, head, tail, tokens, vocab, units, scale, accumulate));
    LNN_CHECK_LAUNCH(d);
  }
  return LNN_OK;
}

// ---- rows of logits ----------------------------------------------------------------------------
// lse(z) = m + log(sum exp(z - m)) in one pass: every thread keeps the maximum and the sum of what it has seen and
// rescales the sum when the maximum moves; the pairs meet through shuffles, shared memory and, where a row is cut over
// a cluster, distributed shared memory, always in the same order.  Bound by HBM: 4096 rows of 32003 (524 MB) in 90 us, 5.8 TB/s,
// 2048 of 131072 (1.07 GB) in 165 us, 6.5 TB/s; the gradient's pass over the latter (2.15 GB) in 326 us, 6.6 TB/s.
struct MaxSum { float m, s; };

__device__ __forceinline__ MaxSum joined(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  const float base = m == -CUDART_INF_F ? 0.0f : m;               // nothing but -inf so far: the sum is 0
  return {m, __fadd_rn(__fmul_rn(a.s, expf(a.m - base)), __fmul_rn(b.s, expf(b.m - base)))};
}
__device__ __forceinline__ void take(MaxSum& a, float m, float v0, float v1, float v2, float v3) {
  if (m > a.m) {
    a.s = __fmul_rn(a.s, expf(a.m - m));
    a.m = m;
  }
  const float base = a.m == -CUDART_INF_F ? 0.0f : a.m;
  a.s = __fadd_rn(a.s, __fadd_rn(__fadd_rn(expf(v0 - base), expf(v1 - base)), __fadd_rn(expf(v2 - base), expf(v3 - base))));
}

struct PolicyArgs {
  const float *old, *adv, *ref;     // old null: the logarithm itself is wanted; ref may be null
  float low, high, kl;
};

constexpr int kLogitQuads = 4;                      // loads of a thread at a time
// out[row] = log p(id) or the policy loss; stats[row] = {max, 1 / sum, d out / d log p}
__global__ void __launch_bounds__(kThreads)
token_logit_kernel(float* __restrict__ out, float* __restrict__ stats, const float* __restrict__ logits,
                   const float* __restrict__ ids, int64_t vocab, int splits, PolicyArgs a, int* status) {
  lnn::wait_for_previous();
  const int64_t row = blockIdx.x / (unsigned)splits;
  const int rank = (int)(blockIdx.x - row * splits);
  const float* z = logits + row * vocab;
  __shared__ MaxSum part[kThreads / 32];
  __shared__ MaxSum block_part;
  const int id = token_row(__ldg(ids + row), (int)vocab, row, 3, status);     // the same in all blocks of the row
  if (id < 0) {
    if (rank == 0 && threadIdx.x == 0) {
      out[row] = 0.0f;
      if (stats) { stats[row * 3] = 0.0f; stats[row * 3 + 1] = 0.0f; stats[row * 3 + 2] = 0.0f; }
    }
    return;
  }
  MaxSum t = {-CUDART_INF_F, 0.0f};
  const int64_t lead = min((int64_t)((4 - (((uintptr_t)z >> 2) & 3)) & 3), vocab);   // up to the first 16-byte boundary
  const int64_t quads = (vocab - lead) >> 2;
  const float4* z4 = reinterpret_cast<const float4*>(z + lead);
  const int64_t begin = quads * rank / splits, end = quads * (rank + 1) / splits;
  for (int64_t i = begin + threadIdx.x; i < end; i += kThreads * kLogitQuads) {
    float4 v[kLogitQuads];
#pragma unroll
    for (int u = 0; u < kLogitQuads; ++u)
      v[u] = i + u * kThreads < end ? __ldg(z4 + i + u * kThreads) : make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
    float top = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < kLogitQuads; ++u) top = fmaxf(top, fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w)));
#pragma unroll
    for (int u = 0; u < kLogitQuads; ++u) take(t, top, v[u].x, v[u].y, v[u].z, v[u].w);
  }
  if (rank == 0 && threadIdx.x < 8) {                         // up to three values in front, up to three behind
    const int64_t j = threadIdx.x < 4 ? (int64_t)threadIdx.x : lead + (quads << 2) + threadIdx.x - 4;
    if (threadIdx.x < 4 ? j < lead : j < vocab) take(t, z[j], z[j], -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const MaxSum b = {__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o)};
    t = joined(t, b);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = t;
  __syncthreads();
  // the first lanes hold the parts of the warps, then those of the blocks of the cluster
  const auto of_lanes = [&](MaxSum x) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      const MaxSum b = {__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.s, o)};
      x = joined(x, b);
    }
    return x;
  };
  if (threadIdx.x < 32) {
    t = of_lanes(part[threadIdx.x & 7]);
    if (threadIdx.x == 0) block_part = t;
  }
  if (splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0 && threadIdx.x < 32) {
      const int r = threadIdx.x & 7;
      t = MaxSum{-CUDART_INF_F, 0.0f};
      if (r < splits) t = *cluster.map_shared_rank(&block_part, r);
      t = of_lanes(t);
    }
    cluster.sync();
  }
  if (rank == 0 && threadIdx.x == 0) {
    // 64 bits for the row's own numbers: whether a ratio is clipped is decided next to a border
    const double logp = (double)z[id] - (double)t.m - log((double)t.s);
    double value = logp, slope = 1.0;
    if (a.old) {
      const double adv = a.adv[row], r = exp(logp - (double)a.old[row]), plain = r * adv;
      const double lo = 1.0 - (double)a.low, hi = 1.0 + (double)a.high;
      value = -fmin(plain, fmin(fmax(r, lo), hi) * adv);
      slope = (adv >= 0.0 ? r <= hi : r >= lo) ? -plain : 0.0;
      if (plain != plain) value = slope = plain;           // (fmin and comparisons drop a NaN)
      if (a.ref) {
        const double u = (double)a.ref[row] - logp, e = exp(u);
        value += (double)a.kl * (e - u - 1.0);
        slope += (double)a.kl * (1.0 - e);
      }
    }
    out[row] = (float)value;
    if (stats) { stats[row * 3] = t.m; stats[row * 3 + 1] = (float)(1.0 / (double)t.s); stats[row * 3 + 2] = (float)slope; }
  }
}

// dz[j] (+)= c (delta - exp(z - m) / s) with c = d out / d log p times the gradient of out: one pass over z and dz.
constexpr int kGradQuads = 4;                      // per thread
__global__ void __launch_bounds__(kThreads)
token_logit_grad_kernel(float* __restrict__ dlogits, const float* __restrict__ logits, const float* __restrict__ stats,
                        const float* __restrict__ ids, const float* __restrict__ dout, int64_t vocab, int chunks,
                        int accumulate) {
  lnn::wait_for_previous();
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int chunk = (int)(blockIdx.x - row * chunks);
  const float m = __ldg(stats + row * 3), inv = __ldg(stats + row * 3 + 1);
  const float slope = __ldg(stats + row * 3 + 2);
  const float c = slope == 0.0f ? 0.0f : __fmul_rn(slope, __ldg(dout + row));
  const float idf = __ldg(ids + row);
  const int64_t id = c != 0.0f ? (int64_t)idf : -1;
  const float* z = logits + row * vocab;
  float* dz = dlogits + row * vocab;
  const auto grad = [&](float v, int64_t j) {
    return __fmul_rn(c, __fsub_rn(j == id ? 1.0f : 0.0f, __fmul_rn(expf(v - m), inv)));
  };
  const int64_t lead = min((int64_t)((4 - (((uintptr_t)z >> 2) & 3)) & 3), vocab);
  const bool vec = (((uintptr_t)z ^ (uintptr_t)dz) & 15) == 0;
  const int64_t quads = vec ? (vocab - lead) >> 2 : 0;
  const int64_t q0 = (int64_t)chunk * (kThreads * kGradQuads) + threadIdx.x;
  const float4* z4 = reinterpret_cast<const float4*>(z + lead);
  float4* dz4 = reinterpret_cast<float4*>(dz + lead);
#pragma unroll
  for (int u = 0; u < kGradQuads; ++u) {
    const int64_t q = q0 + u * kThreads;
    if (q < quads) {
      float4 g = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c != 0.0f) {
        const float4 v = __ldg(z4 + q);
        const int64_t j = lead + (q << 2);
        g = make_float4(grad(v.x, j), grad(v.y, j + 1), grad(v.z, j + 2), grad(v.w, j + 3));
      }
      dz4[q] = accumulate ? plus(dz4[q], g) : g;
    }
  }
  // what no aligned group of four covers: the ends of the row, or all of it
  const auto one = [&](int64_t j) {
    const float g = c != 0.0f ? grad(z[j], j) : 0.0f;
    dz[j] = accumulate ? __fadd_rn(dz[j], g) : g;
  };
  if (vec) {
    if (chunk == 0 && threadIdx.x < 8) {
      const int64_t j = threadIdx.x < 4 ? (int64_t)threadIdx.x : lead + (quads << 2) + threadIdx.x - 4;
      if (threadIdx.x < 4 ? j < lead : j < vocab) one(j);
    }
  } else {
    const int64_t end = min((int64_t)(chunk + 1) * (kThreads * kGradQuads * 4), vocab);
    for (int64_t j = (int64_t)chunk * (kThreads * kGradQuads * 4) + threadIdx.x; j < end; j += kThreads) one(j);
  }
}

const float* in(uint64_t p) { return (const float*)(uintptr_t)p; }
float* out(uint64_t p) { return (float*)(uintptr_t)p; }

int token_logit(int dev, uint64_t OUT, uint64_t STATS, uint64_t X, uint64_t IDS, int64_t rows, int64_t vocab, PolicyArgs a) {
  LNN_DEV(d, dev);
  LNN_REQUIRE(OUT && X && IDS && rows > 0 && vocab > 0, "bad arguments");
  LNN_REQUIRE(vocab <= (1 << 24), "a vocabulary of %lld: token numbers are exact in fp32 up to 2^24", (long long)vocab);
  LNN_REQUIRE(rows <= (1 << 27), "too many rows");
  // a row goes over a cluster of blocks where the rows alone do not fill the device
  int splits = 1;
  static_assert(kThreads / 32 == 8, "parts of a block, blocks of a cluster: eight");
  while (splits < 8 && rows * splits < 4 * d->sm_count && vocab >= (int64_t)splits * 2 * kThreads * 16) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = d->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  LNN_CUDA(cudaLaunchKernelEx(&cfg, token_logit_kernel, out(OUT), out(STATS), in(X), in(IDS), vocab, splits, a, d->status_dev));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

}  // namespace

extern "C" {

int lnn_embedding_fwd(int dev, uint64_t Y, uint64_t TABLE, uint64_t IDS, int64_t tokens, int64_t vocab, int64_t dim,
                      float scale) {
  LNN_DEV(d, dev);
  LNN_REQUIRE(Y && TABLE && IDS && tokens > 0 && vocab > 0 && dim > 0, "bad arguments");
  LNN_REQUIRE(vocab <= (1 << 24), "a table of %lld rows: token numbers are exact in fp32 up to 2^24", (long long)vocab);
  const bool vec = aligned16(out(Y), in(TABLE), dim);
  const int64_t units = vec ? dim / 4 : dim;
  const dim3 block = row_block(units);
  const unsigned grid = (unsigned)std::min<int64_t>(lnn_ceil_div(tokens, block.y), (int64_t)d->sm_count * 64);
  if (vec)
    LNN_CUDA(lnn::launch_chained(d, embedding_fwd_kernel<float4>, grid, block, 0, (float4*)out(Y), (const float4*)in(TABLE), in(IDS),
                                 tokens, (int)vocab, units, scale, d->status_dev));
  else
    LNN_CUDA(lnn::launch_chained(d, embedding_fwd_kernel<float>, grid, block, 0, out(Y), in(TABLE), in(IDS), tokens, (int)vocab, units,
                                 scale, d->status_dev));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

int lnn_embedding_bwd_acc(int dev, uint64_t dTABLE, uint64_t dY, uint64_t IDS, int64_t tokens, int64_t vocab, int64_t dim,
                          float scale, int accumulate) {
  LNN_DEV(d, dev);
  LNN_REQUIRE(dTABLE && dY && IDS && tokens > 0 && vocab > 0 && dim > 0, "bad arguments");
  LNN_REQUIRE(vocab <= (1 << 24), "a table of %lld rows: token numbers are exact in fp32 up to 2^24", (long long)vocab);
  LNN_REQUIRE(tokens < (1ll << 31), "too many tokens");
  if (aligned16(out(dTABLE), in(dY), dim))
    return embedding_bwd<float4>(d, (float4*)out(dTABLE), (const float4*)in(dY), in(IDS), tokens, (int)vocab, dim / 4, scale,
                                 accumulate);
  return embedding_bwd<float>(d, out(dTABLE), in(dY), in(IDS), tokens, (int)vocab, dim, scale, accumulate);
}

int lnn_token_log_prob_fwd(int dev, uint64_t LOGP, uint64_t STATS, uint64_t X, uint64_t IDS, int64_t rows, int64_t vocab) {
  return token_logit(dev, LOGP, STATS, X, IDS, rows, vocab, PolicyArgs{});
}

int lnn_policy_loss_fwd(int dev, uint64_t LOSS, uint64_t STATS, uint64_t X, uint64_t IDS, uint64_t OLD, uint64_t ADV,
                        uint64_t REF, int64_t rows, int64_t vocab, float clip_low, float clip_high, float kl) {
  LNN_REQUIRE(OLD && ADV, "bad arguments");
  LNN_REQUIRE(clip_low >= 0.0f && clip_low <= 1.0f && clip_high >= 0.0f, "clip range 1 - %g .. 1 + %g", clip_low, clip_high);
  return token_logit(dev, LOSS, STATS, X, IDS, rows, vocab, PolicyArgs{in(OLD), in(ADV), in(REF), clip_low, clip_high, kl});
}

int lnn_token_logit_bwd_acc(int dev, uint64_t dX, uint64_t X, uint64_t STATS, uint64_t IDS, uint64_t dOUT, int64_t rows,
                            int64_t vocab, int accumulate) {
  LNN_DEV(d, dev);
  LNN_REQUIRE(dX && X && STATS && IDS && dOUT && rows > 0 && vocab > 0 && vocab <= (1 << 24), "bad arguments");
  const int64_t chunks = lnn_ceil_div(vocab, kThreads * kGradQuads * 4);
  LNN_REQUIRE(rows * chunks < (1ll << 31), "too many rows");
  LNN_CUDA(lnn::launch_chained(d, token_logit_grad_kernel, (unsigned)(rows * chunks), kThreads, 0, out(dX), in(X), in(STATS), in(IDS),
                               in(dOUT), vocab, (int)chunks, accumulate));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

}  // extern "C"
