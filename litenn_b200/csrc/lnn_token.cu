// Operators on tokens: rows of a table and their gradient, the logarithm of a token's probability, the clipped
// policy loss.  Token numbers are whole numbers in fp32 (exact to 2^24); one below zero marks a padded place, which
// gives zeros and no gradient.  Anything else that is no row of the table is treated as padding and leaves
// LNN_E_INVALID in the device status, so that the next read of a result raises.
//
// All of them are bound by HBM.
#include <cooperative_groups.h>
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

// One row of threads (blockDim.x) per token, columns in units of T.
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
// of the tokens whatever the launch looks like: no atomics on values.
constexpr int kSortWarps = kThreads / 32;
constexpr int kMaxSortBlocks = 64;
constexpr int kSortKeys = 4;                       // per lane at a time

// Sorting is a chain of short dependent steps; rows without tokens have to become zero.  Blocks behind the first
// `sort_blocks` of every launch write a share of the zeros meanwhile.
struct SortArgs {
  const float* ids;                                // the first pass reads these, the later ones keys and at
  const uint32_t *keys, *at;
  uint32_t *out_keys, *out_at, *hist;              // hist [sort_blocks][256]
  int64_t n;
  int vocab, shift, sort_blocks;
  float4* zeros;                                   // [zero_begin, zero_end) of the table in 16-byte units, and its odd floats
  int64_t zero_begin, zero_end;
  float* odd;
  int odds;
  int* status;
};
__device__ __forceinline__ void write_zeros(const SortArgs& a) {
  const int64_t stride = (int64_t)(gridDim.x - a.sort_blocks) * kThreads;
  const int64_t first = (int64_t)(blockIdx.x - a.sort_blocks) * kThreads + threadIdx.x;
  for (int64_t i = a.zero_begin + first; i < a.zero_end; i += stride) a.zeros[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (first < a.odds) a.odd[first] = 0.0f;
}

// The share of a block, cut into one contiguous strip per warp, which takes kSortKeys * 32 tokens of it at a time.
struct SortStrip {
  int64_t begin, end;
  __device__ __forceinline__ explicit SortStrip(const SortArgs& a) {
    const int64_t per = ((a.n + a.sort_blocks - 1) / a.sort_blocks + kThreads - 1) / kThreads * 32;      // tokens per warp
    begin = min(((int64_t)blockIdx.x * kSortWarps + (threadIdx.x >> 5)) * per, a.n);
    end = min(begin + per, a.n);
  }
};
constexpr uint32_t kNoKey = 0xffffffffu;
__device__ __forceinline__ void load_keys(const SortArgs& a, int64_t i0, int64_t end, uint32_t (&key)[kSortKeys]) {
#pragma unroll
  for (int u = 0; u < kSortKeys; ++u) {
    const int64_t i = i0 + u * 32 + (threadIdx.x & 31);
    key[u] = kNoKey;
    if (i < end) {
      if (a.keys) {
        key[u] = __ldg(a.keys + i);
      } else {
        const int row = token_row(__ldg(a.ids + i), a.vocab, i, 2, a.status);
        key[u] = row < 0 ? (uint32_t)a.vocab : (uint32_t)row;    // padding comes last
      }
    }
  }
}
__device__ __forceinline__ uint32_t digit_of(uint32_t key, int shift) { return key == kNoKey ? 256u : (key >> shift) & 255u; }
__device__ __forceinline__ void count_digits(uint32_t* count, const uint32_t (&key)[kSortKeys], int shift) {
#pragma unroll
  for (int u = 0; u < kSortKeys; ++u) {
    const uint32_t digit = digit_of(key[u], shift);
    const uint32_t same = __match_any_sync(0xffffffffu, digit);
    if (digit < 256u && (threadIdx.x & 31) == __ffs(same) - 1) count[digit] += __popc(same);
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kThreads)
sort_count_kernel(const __grid_constant__ SortArgs a) {
  __shared__ uint32_t count[kSortWarps][256];
  lnn::wait_for_previous();
  if ((int)blockIdx.x >= a.sort_blocks) { write_zeros(a); return; }
  for (int i = threadIdx.x; i < kSortWarps * 256; i += kThreads) (&count[0][0])[i] = 0;
  const SortStrip s(a);
  uint32_t key[kSortKeys];
  load_keys(a, s.begin, s.end, key);
  __syncthreads();
  for (int64_t i0 = s.begin; i0 < s.end; i0 += kSortKeys * 32) {
    if (i0 > s.begin) load_keys(a, i0, s.end, key);
    count_digits(count[threadIdx.x >> 5], key, a.shift);
  }
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) total += count[w][threadIdx.x];
  a.hist[blockIdx.x * 256 + threadIdx.x] = total;
}

__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(const __grid_constant__ SortArgs a) {
  __shared__ uint32_t count[kSortWarps][256];
  __shared__ uint32_t warp_total[kSortWarps];
  lnn::wait_for_previous();
  if ((int)blockIdx.x >= a.sort_blocks) { write_zeros(a); return; }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kSortWarps * 256; i += kThreads) (&count[0][0])[i] = 0;
  const SortStrip s(a);
  const bool once = s.end - s.begin <= kSortKeys * 32;           // the strip's keys stay in registers
  uint32_t key[kSortKeys];
  load_keys(a, s.begin, s.end, key);
  // where this block's tokens of digit threadIdx.x begin: all smaller digits, then the blocks before this one
  uint32_t before = 0, total = 0;
#pragma unroll 16
  for (int b = 0; b < a.sort_blocks; ++b) {
    const uint32_t c = __ldg(a.hist + b * 256 + threadIdx.x);
    if (b < (int)blockIdx.x) before += c;
    total += c;
  }
  __syncthreads();
  for (int64_t i0 = s.begin; i0 < s.end; i0 += kSortKeys * 32) {
    if (i0 > s.begin) load_keys(a, i0, s.end, key);
    count_digits(count[warp], key, a.shift);
  }
  uint32_t scan = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  for (int w = 0; w < warp; ++w) scan += warp_total[w];
  uint32_t base = scan - total + before;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) {
    const uint32_t c = count[w][threadIdx.x];
    count[w][threadIdx.x] = base;
    base += c;
  }
  __syncthreads();
  for (int64_t i0 = s.begin; i0 < s.end; i0 += kSortKeys * 32) {
    if (!once) load_keys(a, i0, s.end, key);
#pragma unroll
    for (int u = 0; u < kSortKeys; ++u) {
      const int64_t i = i0 + u * 32 + lane;
      const uint32_t digit = digit_of(key[u], a.shift);
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      uint32_t to = 0;
      if (digit < 256u) to = count[warp][digit] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (digit < 256u) {
        if (lane == __ffs(same) - 1) count[warp][digit] += __popc(same);
        a.out_keys[to] = key[u];
        a.out_at[to] = a.at ? __ldg(a.at + i) : (uint32_t)i;
      }
      __syncwarp();
    }
  }
}

// Sums of the sorted tokens, kPiece of them per row of threads.  What a piece holds of a row that starts in an earlier
// piece goes to head[piece], the beginning of one that goes on behind it to tail[piece]; table_join_kernel adds those.
constexpr int kPiece = 32;

template <class T>
__global__ void __launch_bounds__(kThreads)
table_grad_kernel(T* __restrict__ dtable, const T* __restrict__ dy, const uint32_t* __restrict__ keys,
                  const uint32_t* __restrict__ at, T* __restrict__ head, T* __restrict__ tail, int64_t tokens, int vocab,
                  int64_t units, float scale, int accumulate) {
  lnn::wait_for_previous();
  const int64_t pieces = (tokens + kPiece - 1) / kPiece;
  const int64_t piece = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (piece >= pieces) return;
  const int64_t lo = piece * kPiece, hi = min(lo + kPiece, tokens);
  for (int64_t c = threadIdx.x + (int64_t)blockIdx.y * blockDim.x; c < units; c += (int64_t)gridDim.y * blockDim.x) {
    uint32_t cur = keys[lo];
    bool continued = lo > 0 && keys[lo - 1] == cur;
    T sum = nothing<T>();
    for (int64_t e0 = lo; e0 < hi; e0 += 8) {
      T v[8];
      uint32_t k[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const bool in = e0 + u < hi;
        k[u] = in ? keys[e0 + u] : cur;
        v[u] = in && k[u] < (uint32_t)vocab ? __ldg(dy + at[e0 + u] * units + c) : nothing<T>();
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (e0 + u < hi) {
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
    } else if (hi < tokens && keys[hi] == cur) {
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
  // the last piece that has some of the row: it begins with it (steps that double, then halve)
  const auto begins = [&](int64_t p) { return p < pieces && __ldg(keys + p * kPiece) == row; };
  int64_t last = piece + 1, step = 1;
  while (begins(last + step)) { last += step; step *= 2; }
  for (; step > 0; step >>= 1)
    if (begins(last + step)) last += step;
  for (int64_t c = threadIdx.x + (int64_t)blockIdx.y * blockDim.x; c < units; c += (int64_t)gridDim.y * blockDim.x) {
    T sum = tail[piece * units + c];
#pragma unroll 8
    for (int64_t p = piece + 1; p <= last; ++p) sum = plus(sum, __ldg(head + p * units + c));
    T* o = dtable + row * units + c;
    *o = accumulate ? plus(*o, scaled(sum, scale)) : scaled(sum, scale);
  }
}

// Threads along the columns of a row and rows per block.
dim3 row_block(int64_t units) {
  unsigned x = 1;
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
  SortArgs a = {};
  a.sort_blocks = (int)std::min<int64_t>(kMaxSortBlocks, lnn_ceil_div(tokens, kSortKeys * kThreads));
  const int64_t pad = (tokens + 3) / 4 * 4;
  int rc = keys.get((uint64_t)(4 * pad + a.sort_blocks * 256) * 4);
  if (!rc) rc = parts.get((uint64_t)pieces * units * sizeof(T) * 2);
  if (rc) return rc;
  uint32_t* buf = keys.as<uint32_t>();
  uint32_t *k[2] = {buf, buf + pad}, *at[2] = {buf + 2 * pad, buf + 3 * pad};
  a.hist = buf + 4 * pad;
  a.ids = ids; a.n = tokens; a.vocab = vocab; a.status = d->status_dev;
  int passes = 1;
  while ((vocab >> (8 * passes)) != 0) ++passes;                 // (keys go up to vocab)
  // the zeros, a share with each launch
  const int64_t floats = accumulate ? 0 : (int64_t)vocab * units * (int64_t)(sizeof(T) / 4);
  float* table = reinterpret_cast<float*>(dtable);
  const int64_t lead = std::min<int64_t>((4 - (((uintptr_t)table >> 2) & 3)) & 3, floats), quads = (floats - lead) / 4;
  a.zeros = reinterpret_cast<float4*>(table + lead);
  const int64_t fill_blocks = std::min<int64_t>((int64_t)d->sm_count * 4, lnn_ceil_div(quads, 2 * passes * kThreads * 4));
  int launch = 0;
  const auto next = [&]() {                                      // a share of the zeros for the next launch; its grid
    a.zero_begin = quads * launch / (2 * passes);
    a.zero_end = quads * (launch + 1) / (2 * passes);
    a.odds = 0;
    if (launch == 0) { a.odd = table; a.odds = (int)lead; }
    if (launch == 1) { a.odd = table + lead + quads * 4; a.odds = (int)(floats - lead - quads * 4); }
    ++launch;
    return (unsigned)(a.sort_blocks + std::max<int64_t>(fill_blocks, a.odds > 0));
  };
  for (int pass = 0; pass < passes; ++pass) {
    a.shift = 8 * pass;
    a.keys = pass ? k[(pass - 1) & 1] : nullptr;
    a.at = pass ? at[(pass - 1) & 1] : nullptr;
    a.out_keys = k[pass & 1];
    a.out_at = at[pass & 1];
    unsigned blocks = next();
    LNN_CUDA(lnn::launch_chained(d, sort_count_kernel, blocks, kThreads, 0, a));
    LNN_CHECK_LAUNCH(d);
    blocks = next();
    LNN_CUDA(lnn::launch_chained(d, sort_scatter_kernel, blocks, kThreads, 0, a));
    LNN_CHECK_LAUNCH(d);
  }
  const uint32_t *src_k = a.out_keys, *src_at = a.out_at;
  const dim3 block = row_block(units);
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
// a cluster, distributed shared memory, always in the same order.
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
      const double adv = a.adv[row], r = exp(logp - (double)a.old[row]);
      const double lo = 1.0 - (double)a.low, hi = 1.0 + (double)a.high;
      value = -fmin(r * adv, fmin(fmax(r, lo), hi) * adv);
      slope = (adv >= 0.0 ? r <= hi : r >= lo) ? -adv * r : 0.0;
      if (a.ref) {
        const double u = (double)a.ref[row] - logp, e = exp(u);
        value += (double)a.kl * (e - u - 1.0);
        slope += (double)a.kl * (1.0 - e);
      }
      if (logp != logp) value = slope = logp;              // (fmin and comparisons drop a NaN)
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
