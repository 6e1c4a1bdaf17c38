// Attention with a sliding window and sinks on the tensor cores (tcgen05, TMEM, TMA), forward and backward, for heads of up
// to 128 values.
//
// fp32 accuracy comes from the split that the other contractions use: x 2^-e = hi + lo in fp16 with an exact power of two
// per head, and lo hi + hi lo + hi hi into one fp32 accumulator.  The accumulator truncates (measured: 1.6 10^-8 of the
// result per instruction, so a chain of 768 is 1.2 10^-5 low), so the small products go first, no accumulator lives
// longer than one tile, and the tiles are added up in registers with rounding.
//
// One kernel serves four passes over tiles of 128 stationary rows against a stream of BN rows:
//   FWD  rows are queries:  S = Q K^T, P = softmax (running maximum and sum), O += P V
//   DQ   rows are queries:  S, dP = dO V^T, dS = P (dP - delta), dQ += dS K
//   DV   rows are keys:     S^T = K Q^T, P^T, dV += P^T dO
//   DK   rows are keys:     S^T, dP^T = V dO^T, dS^T, dK += dS^T Q
// Scores of 10^7 and more are as good as others: weights come from differences of scores (FWD), or from scores that are those of
// FWD to the bit and a logarithm of the denominator that is kept in two floats.
// Each sum has one owner: no atomics, results do not change from run to run.  dV and dK are separate passes (S^T is computed
// twice) because 128 stationary rows of K and V of 128 values leave room in shared memory for two tiles of Q and one
// of dO, not for two of both.
//
// What bounds it, for heads of 128 values: waiting, not a rate.  Counters of 8 heads over 2 of 4096 positions, window 1024 (of the
// clocks in which an SM is active): tensor pipe FWD 47, DV 56, DQ 44, DK 48 %, issue slots 33 to 39 %; of their peaks L1 28 to 33 %, L2 9
// to 21 %, DRAM 5 to 7 %.  FWD and DV have one slot each for K and V (Q and dO), whose next load begins when the products of the last
// are over; DQ and DK have gaps between dependent products; and a tile of rows begins with its first loads and ends with
// 64 KB of results (two to three steps).  Under load the SMs run at 1.6 of their 1.9 GHz.  8192 positions, 16 heads, window
// 1024: 199 us, 325 TFLOP/s (three products each: 551 is the most); 8 heads over 2, window 2048: FWD 166, DQ 304, DV 187, DK 337 us.
//
// A persistent CTA of 576 threads per SM: warp 0 loads (TMA), one thread of warp 1 issues the MMAs, warps 2-17 (four per
// quarter of the TMEM lanes, a fourth of the columns each) turn scores into weights, write them back to TMEM as the A operand
// of the second product (hi and lo in the columns that the scores were in), and keep the running sums in registers.
// The MMA stream is one step ahead: S(g + 1) runs while the weights of step g are computed.
#include <algorithm>
#include "lnn_attn.cuh"
#include "lnn_tc_dev.cuh"

namespace {

using namespace lnn_tc;
using lnn::AttnArgs;
using lnn::HeadInfo;
using lnn::exp2_fast;

enum { FWD = 0, DV = 1, DQ = 2, DK = 3 };

constexpr int kComputeWarps = 16, kParts = kComputeWarps / 4;
constexpr int kAttnThreads = 32 * (2 + kComputeWarps);
constexpr int kBoxRows = 32;                     // rows of a TMA box
constexpr int kRowsM = 128;                      // stationary rows

// ---- preparation -----------------------------------------------------------------------------------
// One pass over each operand: split, row norms (what bounds dS), and for dO the rows of dO * O and the denominators
// with a padded pitch.  Bound by HBM, with about 5 us of dependent latencies in front and behind (24 heads of 8192 rows
// of 128 values, 200 MB: 35 us).  Eight values to a lane: half the address arithmetic and shuffles of four.
// The scale of a head is guessed from 32 of its rows, so that the largest value of them is in [2^8, 2^9); the true
// maximum may be 2^7 times that before fp16 overflows.  A head beyond it, or with values that are not finite, is
// marked and goes to the FP32-pipe kernels: a scale for such an outlier would cost the others their low bits.  Where the 32 rows
// are zero (dO of a loss on few tokens), the last row is asked, and where that is zero too and others are not, the block that
// ends last splits the head once more with the scale of its true maximum (8 heads of 8192 rows of 128 values: 0.3 ms more).
constexpr int kPrepThreads = 256;
constexpr int kPrepRows = 64;                    // a block takes a multiple of them
constexpr int kPrepBlocksPerSm = 4;
constexpr int kSampleRows = 32;

struct PrepTensor {
  const float* src;
  __half* hi;                    // [heads][rows][width]; lo behind all heads
  float* norms;                  // [heads][rows]: squares of the rows' norms after scaling, or null
  int heads, per_batch, rows;
  int first, sinks;              // keys: rows below `first` that are no sinks are seen by no query
  int past;                      // queries: row i is at position i + past
  float sign;
};
struct PrepArgs {
  PrepTensor t[4];
  int tensors, dim, width, batch;        // width: dim rounded up to the 16 values of an MMA
  const float* lengths;
  int kv_len;
  HeadInfo* info;                // [all heads of all tensors]
  float* block_max;              // [head][blocks]: largest magnitudes, +inf: not finite
  float* block_norm;
  int blocks, block_rows;        // row blocks of the longest tensor, rows of a block
  unsigned int* counters;        // one per head, zero between launches
  // the last tensor is dO
  const float *o, *lse;
  float *lse_p, *delta_p;        // lse_p: -hi, -hi, 14 - lo, 14 - lo of two rows
  int pitch;
  int* taken;                    // [4] works that have been taken, of each pass
  int* status;
};

struct Eight { float4 a, b; };
// hi of a row's logarithm, lo is two floats behind: two rows are read together
__device__ __forceinline__ int64_t lse_at(int64_t head, int pitch, int row) { return head * 2 * pitch + (row >> 1) * 4 + (row & 1); }

// VEC: rows of whole, aligned quads
template <int DP, bool VEC>
__global__ void __launch_bounds__(kPrepThreads, kPrepBlocksPerSm)
attn_prep_kernel(const __grid_constant__ PrepArgs a) {
  constexpr int LANES = DP / 8, ROWS = 32 / LANES;              // eight values per lane; rows that a warp takes at once
  constexpr int kWarps = kPrepThreads / 32, STRIDE = kWarps * ROWS, BATCH = 2;
  __shared__ float red[kWarps], red_norm[kWarps];
  __shared__ int last_block;
  __shared__ float head_max;
  lnn::wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES, c = lane % LANES * 8;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 4) a.taken[threadIdx.x] = 0;
  int head = blockIdx.y, ti = 0;
  while (head >= a.t[ti].heads) head -= a.t[ti++].heads;
  const PrepTensor& t = a.t[ti];
  const int blocks = (t.rows + a.block_rows - 1) / a.block_rows;
  if ((int)blockIdx.x >= blocks) return;
  const int len = lnn::attn_length(a.lengths, head / t.per_batch, a.kv_len, a.status);
  const int end = min(t.rows, len - t.past), dim = a.dim, first = t.first, sinks = t.sinks;      // rows from `end` on are padding
  const bool is_do = a.o != nullptr && ti == a.tensors - 1, with_norms = t.norms != nullptr;
  const float* src = t.src + (int64_t)head * t.rows * dim + c;
  const float* src_o = a.o + (int64_t)head * t.rows * dim + c;
  const auto quad = [&](const float* p, int c) {
    if (VEC) return c < dim ? __ldg(reinterpret_cast<const float4*>(p)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(c < dim ? __ldg(p) : 0.0f, c + 1 < dim ? __ldg(p + 1) : 0.0f, c + 2 < dim ? __ldg(p + 2) : 0.0f,
                       c + 3 < dim ? __ldg(p + 3) : 0.0f);
  };
  const auto load = [&](const float* p) { return Eight{quad(p, c), quad(p + 4, c + 4)}; };      // (p: this lane's values)
  const auto largest = [](const Eight& v) {
    return fmaxf(fmaxf(fmaxf(fabsf(v.a.x), fabsf(v.a.y)), fmaxf(fabsf(v.a.z), fabsf(v.a.w))),
                 fmaxf(fmaxf(fabsf(v.b.x), fabsf(v.b.y)), fmaxf(fabsf(v.b.z), fabsf(v.b.w))));
  };
  const auto row_total = [&](float v) {                          // over the lanes of a row
#pragma unroll
    for (int s = LANES / 2; s > 0; s >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, s));
    return v;
  };
  const auto warp_max = [&](float v) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
    return v;
  };
  Eight x[BATCH], y[BATCH];
  const auto fetch = [&](int r0) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int r = r0 + u * STRIDE;
      const bool real = r < end && (r >= first || r < sinks);
      x[u].a = x[u].b = y[u].a = y[u].b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (real) x[u] = load(src + (int64_t)r * dim);
      if (is_do && real) y[u] = load(src_o + (int64_t)r * dim);
    }
  };
  int r_first = blockIdx.x * a.block_rows + warp * ROWS + sub, r_end = min((int)(blockIdx.x + 1) * a.block_rows, t.rows);
  fetch(r_first);
  // the scale, from rows spread over those that are real (the same ones in every block of the head; what is not a number is
  // left out here and found below)
  float top = 0.0f;
  const int span = end - first;
  if (span > 0) {
#pragma unroll
    for (int i = warp * ROWS + sub; i < kSampleRows; i += STRIDE) {
      top = fmaxf(top, largest(load(src + (int64_t)(first + (int)((int64_t)i * span / kSampleRows)) * dim)));
    }
  }
  top = warp_max(top);
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red[w]);
  if (top == 0.0f && span > 0) top = warp_max(largest(load(src + (int64_t)(end - 1) * dim)));
  const int ebits = (int)(__float_as_uint(top) >> 23);
  int e = top == 0.0f || ebits == 255 ? 0 : ebits - 127 - 8;
  const bool nothing = top == 0.0f;                               // the sample says
  const uint64_t minus = pack2(-1.0f, -1.0f);
  __syncthreads();

  __half* hi = t.hi + (int64_t)head * t.rows * a.width + c;
  __half* lo = hi + (int64_t)t.heads * t.rows * a.width;
  for (bool again = false;; again = true) {
    const float factor = t.sign * pow2f_int(max(-126, min(127, -e)));     // (|e| > 100 is not taken anyway)
    const uint64_t factor2 = pack2(factor, factor);
    float top_norm = 0.0f;
    bool number = true;
    top = 0.0f;
    for (int r0 = r_first; r0 - sub < r_end; r0 += BATCH * STRIDE) {      // (the same turns for both rows of a warp)
      if (r0 != r_first) fetch(r0);
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int r = r0 + u * STRIDE;
        const bool in = r < r_end;
        if (is_do) {
          const float half = fmaf(x[u].a.w, y[u].a.w, fmaf(x[u].a.z, y[u].a.z, fmaf(x[u].a.y, y[u].a.y, __fmul_rn(x[u].a.x, y[u].a.x))));
          const float delta = row_total(fmaf(x[u].b.w, y[u].b.w, fmaf(x[u].b.z, y[u].b.z, fmaf(x[u].b.y, y[u].b.y, fmaf(x[u].b.x, y[u].b.x, half)))));
          if (c == 0 && in) a.delta_p[(int64_t)head * a.pitch + r] = -delta;
        }
        uint32_t h[4], l[4];
        float norm = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4& w = k < 2 ? x[u].a : x[u].b;
          top = fmaxf(top, k & 1 ? fmaxf(fabsf(w.z), fabsf(w.w)) : fmaxf(fabsf(w.x), fabsf(w.y)));
          const uint64_t v = mul2(k & 1 ? pack2(w.z, w.w) : pack2(w.x, w.y), factor2);
          float p, q;
          unpack2(v, p, q);
          norm = fmaf(q, q, fmaf(p, p, norm));
          const __half2 hh = __floats2half2_rn(p, q);
          const float2 f = __half22float2(hh);
          unpack2(fma2(pack2(f.x, f.y), minus, v), p, q);
          const __half2 ll = __floats2half2_rn(p, q);
          h[k] = *reinterpret_cast<const uint32_t*>(&hh);
          l[k] = *reinterpret_cast<const uint32_t*>(&ll);
        }
        number = number && norm == norm;
        if (in && c < a.width) {
          *reinterpret_cast<uint4*>(hi + (int64_t)r * a.width) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(lo + (int64_t)r * a.width) = make_uint4(l[0], l[1], l[2], l[3]);
        }
        if (with_norms) {
          norm = row_total(norm);
          top_norm = fmaxf(top_norm, norm);
          if (c == 0 && in) t.norms[(int64_t)head * t.rows + r] = norm;
        }
      }
    }
    if (is_do && !again) {
      const auto put_lse = [&](int r, float2 v) {
        float* to = a.lse_p + lse_at(head, a.pitch, r);
        to[0] = -v.x;
        to[2] = 14.0f - v.y;
      };
      for (int r = blockIdx.x * a.block_rows + threadIdx.x; r < r_end; r += kPrepThreads)
        put_lse(r, r < end ? __ldg(reinterpret_cast<const float2*>(a.lse) + (int64_t)head * t.rows + r) : make_float2(CUDART_INF_F, 0.0f));
      if ((int)blockIdx.x == blocks - 1)                           // columns that exist in no head
        for (int r = t.rows + threadIdx.x; r < a.pitch; r += kPrepThreads) {
          a.delta_p[(int64_t)head * a.pitch + r] = 0.0f;
          put_lse(r, make_float2(CUDART_INF_F, 0.0f));
        }
    }
    top = __all_sync(0xffffffffu, number) ? warp_max(top) : CUDART_INF_F;
    top_norm = warp_max(top_norm);
    if (lane == 0) { red[warp] = top; red_norm[warp] = top_norm; }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) { top = fmaxf(top, red[w]); top_norm = fmaxf(top_norm, red_norm[w]); }
      if (again) {
        a.info[blockIdx.y] = HeadInfo{e, 1, sqrtf(top_norm)};
        last_block = 0;
      } else {
        const int64_t at = (int64_t)blockIdx.y * a.blocks;
        __stcg(a.block_max + at + blockIdx.x, top);
        __stcg(a.block_norm + at + blockIdx.x, top_norm);
        __threadfence();
        last_block = atomicAdd(a.counters + blockIdx.y, 1u) == (unsigned)blocks - 1;
      }
    }
    __syncthreads();
    if (!last_block) return;
    if (warp == 0) {
      __threadfence();
      top = 0.0f;
      top_norm = 0.0f;
      for (int i = lane; i < blocks; i += 32) {
        top = fmaxf(top, __ldcg(a.block_max + (int64_t)blockIdx.y * a.blocks + i));
        top_norm = fmaxf(top_norm, __ldcg(a.block_norm + (int64_t)blockIdx.y * a.blocks + i));
      }
      top = warp_max(top);
      top_norm = warp_max(top_norm);
      if (lane == 0) {
        const float scaled = __fmul_rn(top, fabsf(factor));
        a.info[blockIdx.y] = HeadInfo{e, top == 0.0f || (scaled >= 4.0f && scaled < 65000.0f), sqrtf(top_norm)};
        a.counters[blockIdx.y] = 0;
        head_max = top;
      }
    }
    if (!nothing) return;
    __syncthreads();
    top = head_max;
    if (top == 0.0f || !(top < CUDART_INF_F)) return;
    e = (int)(__float_as_uint(top) >> 23) - 127 - 14;              // the largest in [2^14, 2^15)
    r_first = warp * ROWS + sub;
    r_end = t.rows;
    fetch(r_first);
  }
}

// ---- the passes ----------------------------------------------------------------------------------------
struct TcArgs {
  AttnArgs a;
  const float *lse_p, *delta_p;  // [q head][2 pitch] (see PrepArgs), [q head][pitch]
  const float* norms;            // squares, DQ: of dO's rows, DK: of V's
  int pitch, width;
  int works;
  int* taken;                    // works that CTAs have taken so far
  int beside;                    // runs beside the pass in front of it, which shares only operands with it
  const uint32_t* x2;            // DQ: dO, DK: V, split
  // FWD, DQ: the works from `whole` on are cut into `splits` each (few tiles, or few in the last round of the SMs)
  int whole;
  float2* stats;                 // FWD: [part][128] maximum (of what was accumulated) and sum of a row
  // DV, DK: keys below sinks take `splits_sink` works per tile of rows, the others `splits`
  int tiles, sink_tiles, splits_sink, splits;
  float* parts;                  // [part][128][DP] of the tiles that have several works
};

template <int MODE, int DP> struct Shape {
  static constexpr bool TWO = MODE == DQ || MODE == DK, KEYS = MODE == DV || MODE == DK;
  static constexpr int BN = TWO ? 64 : 128;
  static constexpr int SLABS = DP / 64;                          // 64 values (128 bytes) wide
  static constexpr uint32_t X_PART = kRowsM * DP * 2, X_BYTES = 2 * X_PART;
  static constexpr uint32_t Y_PART = BN * DP * 2, Y_BYTES = 2 * Y_PART;
  // ring depths: see the order of the MMAs
  static constexpr int NY = TWO ? 3 : (DP == 128 ? 1 : 2), NZ = TWO ? 2 : (DP == 128 ? 1 : 2);
  static constexpr int NS = TWO ? 2 : 3;                         // score buffers (and of dP)
  static constexpr int NO = TWO ? NY : NZ;                       // steps that a completed result is told apart over
  static constexpr uint32_t TILES = X_BYTES + (NY + NZ) * Y_BYTES;
  // TMEM columns: DQ and DK keep their second stationary operand (dO, V) there, which leaves shared memory for a third
  // stream tile and makes its products faster (33 instead of 50 clocks for 64 columns)
  static constexpr uint32_t T_DP = NS * BN, T_OUT = T_DP + (TWO ? NS * BN : 0), T_X2 = T_OUT + DP;
  static_assert(T_X2 + (TWO ? DP : 0) <= 512, "TMEM");
};

// Tiles with one work only write their results themselves: their places are behind the others' and are not there where
// only the tiles with sinks are cut.
__device__ __forceinline__ int64_t parts_per_head(const TcArgs& t) {
  return (int64_t)t.sink_tiles * t.splits_sink + (t.splits > 1 ? (int64_t)(t.tiles - t.sink_tiles) * t.splits : 0);
}

constexpr float kWeightUnit = 1.0f / 16384.0f;      // weights are 2^14 times what they stand for

// Accumulated scores times this are scores to the base two.  (2^-126 in place of 0: masked scores stay -inf)
__device__ __forceinline__ float score_factor(const AttnArgs& a, int eq, int ek) {
  return fmaxf(__fmul_rn(__fmul_rn(fabsf(a.scale), lnn::kLog2e), pow2f_int(eq + ek)), 1.17549435e-38f);
}

// A tile of 128 stationary rows and the steps of its stream.  The loading warp works it out (divisions, the sequence's
// length, the scales) and hands it to the others through shared memory, ahead of the tile's turn.
struct Work {
  int b, hk, h, row0, steps;
  int p_hi, lowest, sink_n, sink_steps;  // queries: positions
  int s0;                                // queries: first step
  int i_lo, nq, q_hi, hq0, q0;           // keys: first query, tiles of queries per head, position of the last query; first step
  int split_up;                          // one of several works of its rows
  int skip;                              // the FP32 pipe's
  int end;                               // there is none: the last was taken
  int part;                              // its place among the parts
  int ek, ev, eq, eo;                    // exponents of the scales (eq, eo: of query head h)
  float norm_v, norm_do;
};

template <int MODE, int DP>
__device__ __forceinline__ void make_work(Work& k, const TcArgs& t, int w, bool some_left) {
  using S = Shape<MODE, DP>;
  const AttnArgs& a = t.a;
  const int past = a.kv_len - a.q_len, group = a.q_heads / a.kv_heads;
  k.steps = 0;
  k.split_up = 0;
  if (!S::KEYS) {
    // the last tiles first: they see most, and the short ones fill up what is left
    int split = 0, splits = 1;
    k.part = w - t.whole;
    if (w >= t.whole) {
      splits = t.splits;
      split = k.part % splits;
      w = t.whole + k.part / splits;
    }
    const int heads = a.batch * a.q_heads, turn = w / heads, head = w - turn * heads;
    k.b = head / a.q_heads; k.h = head - k.b * a.q_heads; k.hk = k.h / group;
    const int len = lnn::attn_length(a.lengths, k.b, a.kv_len, a.status);
    k.row0 = (t.tiles - 1 - turn) * kRowsM;
    k.p_hi = min(min(k.row0 + kRowsM, a.q_len) - 1 + past, len - 1);
    if (k.p_hi >= k.row0 + past) {
      k.lowest = max(k.row0 + past - a.window + 1, 0);
      k.sink_n = min(a.sinks, k.lowest);
      k.sink_steps = (k.sink_n + S::BN - 1) / S::BN;
      const int all = k.sink_steps + (k.p_hi - k.lowest) / S::BN + 1;
      k.s0 = (int)((int64_t)all * split / splits);
      k.steps = (int)((int64_t)all * (split + 1) / splits) - k.s0;
    }
    k.split_up = splits > 1;
  } else {
    // the first tiles first: most queries see them
    const int heads = a.batch * a.kv_heads;
    int r = w / heads, split, splits, tile;
    const int head = w - r * heads;
    k.b = head / a.kv_heads; k.hk = head - k.b * a.kv_heads; k.h = k.hk * group;
    k.part = (int)(head * parts_per_head(t) + r);
    if (r < t.sink_tiles * t.splits_sink) {
      splits = t.splits_sink; tile = r / splits; split = r - tile * splits;
    } else {
      r -= t.sink_tiles * t.splits_sink;
      splits = t.splits; tile = r / splits; split = r - tile * splits; tile += t.sink_tiles;
    }
    k.split_up = splits > 1;
    const int len = lnn::attn_length(a.lengths, k.b, a.kv_len, a.status);
    k.row0 = tile * kRowsM;
    const lnn::QuerySpan span(k.row0, min(k.row0 + kRowsM, a.kv_len) - 1, a.window, a.sinks, past, len);
    if (span.hi >= span.lo) {
      k.q_hi = span.hi;
      k.i_lo = (span.lo - past) & ~7;                        // (the denominators are read in vectors)
      k.nq = (span.hi - past - k.i_lo) / S::BN + 1;
      const int all = k.nq * group;
      const int first = (int)((int64_t)all * split / splits);
      k.steps = (int)((int64_t)all * (split + 1) / splits) - first;
      k.hq0 = first / k.nq; k.q0 = first - k.hq0 * k.nq;
    }
  }
  k.skip = some_left && !lnn::group_ok(a, k.b, k.hk);
  const int qh = k.b * a.q_heads + k.h;
  const HeadInfo ik = lnn::info_of(a, 1, k.b * a.kv_heads + k.hk), iv = lnn::info_of(a, 2, k.b * a.kv_heads + k.hk);
  k.ek = ik.e; k.ev = iv.e; k.norm_v = iv.norm;
  k.eq = lnn::info_of(a, 0, qh).e;
  if (MODE != FWD) {
    const HeadInfo io = lnn::info_of(a, 3, qh);
    k.eo = io.e; k.norm_do = io.norm;
  }
}

// The steps of a work one after another: rows [r, r + n) of head `head` of the stream.
template <int MODE, int DP>
struct Steps {
  int head, r, n, s, q;
  __device__ __forceinline__ Steps(const TcArgs& t, const Work& k) : s(0) {
    if (!Shape<MODE, DP>::KEYS) { head = k.b * t.a.kv_heads + k.hk; q = 0; s = k.s0; }
    else { head = k.b * t.a.q_heads + k.h + k.hq0; q = k.q0; }
    at(t, k);
  }
  __device__ __forceinline__ void at(const TcArgs& t, const Work& k) {
    constexpr int BN = Shape<MODE, DP>::BN;
    if (!Shape<MODE, DP>::KEYS) {
      if (s < k.sink_steps) { r = s * BN; n = min(BN, k.sink_n - r); }
      else { r = k.lowest + (s - k.sink_steps) * BN; n = min(BN, k.p_hi + 1 - r); }
    } else {
      r = k.i_lo + q * BN;
      n = min(BN, k.q_hi - (t.a.kv_len - t.a.q_len) + 1 - r);
    }
  }
  __device__ __forceinline__ void next(const TcArgs& t, const Work& k) {
    ++s;
    if (Shape<MODE, DP>::KEYS && ++q == k.nq) { q = 0; ++head; }
    at(t, k);
  }
};

// One lane of a converged warp.  The warps that load and issue run as whole warps with this lane doing the asynchronous
// instructions: addresses and descriptors then live in uniform registers (with a single running thread every MMA waited
// for its descriptors to be moved there, 100 to 140 clocks an instruction).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Descriptors as two words: the upper one is the same for all tiles of a layout.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A whole warp's wait: all lanes go on or all give up (what follows is done by whole warps).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int role, int step) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, role, step));
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// 16 weights as fp16, two to a column: 8 columns of hi, 8 of lo
__device__ __forceinline__ void store_split(uint32_t at, const uint64_t* w) {
  uint32_t x[16];
  const uint64_t minus = pack2(-1.0f, -1.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    unpack2(w[i], a, b);
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    unpack2(fma2(pack2(f.x, f.y), minus, w[i]), a, b);           // (exact)
    const __half2 l = __floats2half2_rn(a, b);
    x[i] = *reinterpret_cast<const uint32_t*>(&h);
    x[8 + i] = *reinterpret_cast<const uint32_t*>(&l);
  }
  tmem_st16(at, x);
}
// bits 0 .. n of a word
__device__ __forceinline__ uint32_t bits_to(int n) { return n < 0 ? 0u : (n >= 31 ? 0xffffffffu : (2u << n) - 1u); }

template <int MODE, int DP>
__global__ void __launch_bounds__(kAttnThreads, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapY,
               const __grid_constant__ CUtensorMap mapZ, const __grid_constant__ TcArgs t) {
  using S = Shape<MODE, DP>;
  constexpr int BN = S::BN, NY = S::NY, NZ = S::NZ, NS = S::NS, NO = S::NO;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_x_full, bar_x_empty, bar_y_full[NY], bar_z_full[NZ];
  __shared__ uint64_t bar_s_full[NS], bar_p_full[NS], bar_o_full[NO], bar_x2_full;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag_smem;
  __shared__ float exchange[3][kComputeWarps][32];
  constexpr int NW = 3;                                          // works handed over
  __shared__ uint64_t bar_w_full[NW], bar_w_empty[NW];
  __shared__ Work works[NW];
  // What goes with the columns of a pass over keys, loaded with the rows of their step.  A slot is free when its step's weights
  // are complete: DK, when its Y slot is (OUT(g) is over); DV, when Y(g + 4) is loaded: S(g + 4 - NY) waited for them.
  constexpr int NC = S::TWO ? NY : 4;
  __shared__ uint64_t bar_c_full[NC];
  __shared__ __align__(16) float col_lse[S::KEYS ? NC : 1][2 * BN], col_delta[MODE == DK ? NC : 1][BN];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_flag_smem;
  int* status = t.a.status;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sX = base, sY = sX + S::X_BYTES, sZ = sY + NY * S::Y_BYTES;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar_x_full), 1);
    mbar_init(smem_u32(&bar_x_empty), 1);
    for (int i = 0; i < NY; ++i) mbar_init(smem_u32(&bar_y_full[i]), 1);
    for (int i = 0; i < NZ; ++i) mbar_init(smem_u32(&bar_z_full[i]), 1);
    for (int i = 0; i < NS; ++i) { mbar_init(smem_u32(&bar_s_full[i]), 1); mbar_init(smem_u32(&bar_p_full[i]), kComputeWarps); }
    for (int i = 0; i < NW; ++i) { mbar_init(smem_u32(&bar_w_full[i]), 1); mbar_init(smem_u32(&bar_w_empty[i]), 1 + kComputeWarps); }
    for (int i = 0; i < NO; ++i) mbar_init(smem_u32(&bar_o_full[i]), 1);
    mbar_init(smem_u32(&bar_x2_full), kComputeWarps);
    for (int i = 0; i < NC; ++i) mbar_init(smem_u32(&bar_c_full[i]), 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base_smem), 512);
    tmem_relinquish();
  }
  if (t.beside) lnn::start_next();
  else lnn::wait_for_previous();
  // an earlier kernel gave up, or the tiles have no place: leave as a whole CTA (the decision must be uniform)
  if (threadIdx.x == 0) {
    uint32_t dynamic;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dynamic));
    const bool fits = base + S::TILES <= smem_u32(smem_raw) + dynamic;
    if (!fits) report_expired_wait(status, 36, (int)blockIdx.x, 0);
    abort_flag_smem = !fits || wait_expired(status) ? 2 : 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (abort_flag_smem == 2) {
    if (warp == 1) tmem_dealloc(tmem_base_smem, 512);
    if (t.beside) lnn::wait_at_end();
    return;
  }
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
  const bool some_left = lnn::any_group_left(t.a);               // work for the FP32 pipe

  if (warp == 0) {
    // ---- loads ------------------------------------------------------------------------------------
    const int x_part = (S::KEYS ? t.a.batch * t.a.kv_heads : t.a.batch * t.a.q_heads);     // heads in front of lo
    const int y_part = (S::KEYS ? t.a.batch * t.a.q_heads : t.a.batch * t.a.kv_heads);
    const auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, uint32_t part_bytes, uint32_t slab_bytes, int head,
                          int parts, int row, int boxes) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int s = 0; s < S::SLABS; ++s)
          for (int i = 0; i < boxes; ++i)
            tma_load_3d(dst + p * part_bytes + s * slab_bytes + i * (kBoxRows * 128), map, bar, s * 64, row + i * kBoxRows,
                        head + p * parts);
    };
    bool ok = true;
    int g = 0, nw = 0, nr = 0;
    // What goes with a step's weights in FWD and DV is loaded one step behind the rows of its scores: the order of use.
    // A slot is free when the products of the step that used it are over, which the barriers of their results tell (each
    // batch of MMAs has one commit: a second one cost 50 clocks of a stream that has few to spare).
    struct Pending { int head, r, boxes, g; bool any; } late = {0, 0, 0, 0, false};
    const auto load_z = [&](const Pending& z) {
      const int slot = z.g % NZ;
      // its last reader: OUT(g - NZ) (FWD, DV); dP(g - NZ), complete with S(g - NZ) (DQ, DK)
      if (z.g >= NZ) {
        const int before = z.g - NZ;
        if (!warp_wait(S::TWO ? smem_u32(&bar_s_full[before % NS]) : smem_u32(&bar_o_full[before % NO]),
                       (before / (S::TWO ? NS : NO)) & 1, abort_flag, status, 10, z.g)) return false;
      }
      if (elect_one()) {
        // DQ, DK: Y and Z of a step are waited for together
        const uint32_t bar = S::TWO ? smem_u32(&bar_y_full[z.g % NY]) : smem_u32(&bar_z_full[slot]);
        if (!S::TWO) mbar_expect_tx(bar, (uint32_t)(2 * S::SLABS * z.boxes * kBoxRows * 128));
        load(&mapZ, sZ + slot * S::Y_BYTES, bar, S::Y_PART, BN * 128, z.head, y_part, z.r, z.boxes);
      }
      __syncwarp();
      return true;
    };
    // Works are taken one by one, the longest first, so that SMs that come late or meet short ones even out.  Results do not
    // depend on who takes what.  A work is made out while the one before it is loaded: its rows are asked for the moment
    // that their place is free.
    const auto take = [&]() {
      int w = 0;
      if (lane == 0) w = atomicAdd(t.taken, 1);
      return __shfl_sync(0xffffffffu, w, 0);
    };
    Work k = {}, ahead = {};
    const auto take_ahead = [&]() {
      const int w = take();
      ahead = Work{};
      if (w < t.works) make_work<MODE, DP>(ahead, t, w, some_left);
      else ahead.end = 1;
    };
    take_ahead();
    for (; ok; ++nr) {
      k = ahead;
      if (k.end && !S::TWO && late.any && !load_z(late)) { ok = false; break; }
      if (!warp_wait(smem_u32(&bar_w_empty[nr % NW]), ((nr / NW) & 1) ^ 1, abort_flag, status, 13, nr)) { ok = false; break; }
      if (lane == 0) {
        works[nr % NW] = k;
        mbar_arrive(smem_u32(&bar_w_full[nr % NW]));
      }
      __syncwarp();
      if (k.end) break;
      // (what the work before still needs must not wait for the next one with steps: that one's place among the works may be
      // free only when the one before is finished)
      if (k.steps == 0 || k.skip) {
        if (!S::TWO && late.any && !load_z(late)) { ok = false; break; }
        late.any = false;
        take_ahead();
        continue;
      }
      if (!warp_wait(smem_u32(&bar_x_empty), (nw & 1) ^ 1, abort_flag, status, 11, nr)) { ok = false; break; }
      if (elect_one()) {
        const int xh = S::KEYS ? k.b * t.a.kv_heads + k.hk : k.b * t.a.q_heads + k.h;
        const uint32_t bx = smem_u32(&bar_x_full);
        mbar_expect_tx(bx, S::X_BYTES);
        load(&mapX, sX, bx, S::X_PART, kRowsM * 128, xh, x_part, k.row0, kRowsM / kBoxRows);
      }
      __syncwarp();
      Steps<MODE, DP> step(t, k);
      for (int s = 0; s < k.steps; ++s, ++g) {
        const Pending z = {step.head, step.r, (step.n + kBoxRows - 1) / kBoxRows, g, true};
        const int slot = g % NY;
        // its last reader: S(g - NY) (FWD, DV), OUT(g - NY) (DQ, DK)
        if (g >= NY) {
          const int before = g - NY;
          if (!warp_wait(S::TWO ? smem_u32(&bar_o_full[before % NO]) : smem_u32(&bar_s_full[before % NS]),
                         (before / (S::TWO ? NO : NS)) & 1, abort_flag, status, 12, g)) { ok = false; break; }
        }
        if (elect_one()) {
          const uint32_t bar = smem_u32(&bar_y_full[slot]);
          mbar_expect_tx(bar, (uint32_t)((S::TWO ? 4 : 2) * S::SLABS * z.boxes * kBoxRows * 128));
          load(&mapY, sY + slot * S::Y_BYTES, bar, S::Y_PART, BN * 128, z.head, y_part, z.r, z.boxes);
          if (S::KEYS) {
            const int64_t at = (int64_t)z.head * t.pitch + z.r;
            const uint32_t bc = smem_u32(&bar_c_full[g % NC]);
            mbar_expect_tx(bc, (MODE == DK ? 3 : 2) * BN * 4);
            bulk_load(smem_u32(&col_lse[g % NC][0]), t.lse_p + 2 * at, 2 * BN * 4, bc);
            if (MODE == DK) bulk_load(smem_u32(&col_delta[g % NC][0]), t.delta_p + at, BN * 4, bc);
          }
        }
        __syncwarp();
        if (S::TWO) {
          if (!load_z(z)) { ok = false; break; }
        } else {
          if (late.any && !load_z(late)) { ok = false; break; }
          late = z;
        }
        step.next(t, k);
        if (s == 0) take_ahead();
      }
      ++nw;
    }
  } else if (warp == 1) {
    // ---- MMAs -------------------------------------------------------------------------------------
    // K-major tiles of 128-byte rows (128-byte swizzle); the same bytes are an MN-major operand when the rows are K:
    // 64 values of MN to a row, slabs of 64 BN rows apart.  Lower words: address and the leading offset, in 16 bytes.
    constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
    constexpr uint32_t K_LO = 1u << 16, MN_LO = (BN * 128u >> 4) << 16;
    const int ksteps = t.width / 16;
    const auto scores = [&](uint32_t d, uint32_t ax, uint32_t by, uint32_t id) {
      const uint32_t a = K_LO + (ax >> 4), b = K_LO + (by >> 4);
#pragma unroll
      for (int pr = 0; pr < 3; ++pr)      // q's lo k's hi, hi lo, hi hi: in this order in all passes, whose scores are the same to the bit
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
          if (ks < ksteps) mma_ss(d, a + (pr == (S::KEYS ? 1 : 0) ? S::X_PART / 16 : 0) + (ks / 4) * (kRowsM * 128 / 16) + (ks % 4) * 2,
                 b + (pr == (S::KEYS ? 0 : 1) ? S::Y_PART / 16 : 0) + (ks / 4) * (BN * 128 / 16) + (ks % 4) * 2, DESC_HI, id, pr + ks > 0);
    };
    const auto second_scores = [&](uint32_t d, uint32_t by, uint32_t id) {      // dO or V from TMEM: DP / 2 columns of hi, then of lo
      const uint32_t a = tmem + S::T_X2, b = K_LO + (by >> 4);
#pragma unroll
      for (int pr = 0; pr < 3; ++pr)
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
          if (ks < ksteps) mma_ts(d, a + (pr == 0 ? DP / 2 : 0) + ks * 8, b + (pr == 1 ? S::Y_PART / 16 : 0) + (ks / 4) * (BN * 128 / 16) + (ks % 4) * 2,
                 DESC_HI, id, pr + ks > 0);
    };
    const auto weighted = [&](uint32_t d, uint32_t p, uint32_t bz, int n16) {      // 16 scores became 8 columns of hi and 8 of lo
      const uint32_t id = (1u << 4) | (1u << 16) | ((uint32_t)(t.width >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t b = MN_LO + (bz >> 4);
      if (n16 == BN) {
#pragma unroll
        for (int pr = 0; pr < 3; ++pr)
#pragma unroll
          for (int ks = 0; ks < BN / 16; ++ks)
            mma_ts(d, p + (pr == 0 ? 8 : 0) + ks * 16, b + (pr == 1 ? S::Y_PART / 16 : 0) + ks * (16 * 128 / 16), DESC_HI, id, pr + ks > 0);
      } else {
        for (int pr = 0; pr < 3; ++pr)
          for (int ks = 0; ks < n16 / 16; ++ks)
            mma_ts(d, p + (pr == 0 ? 8 : 0) + ks * 16, b + (pr == 1 ? S::Y_PART / 16 : 0) + ks * (16 * 128 / 16), DESC_HI, id, pr + ks > 0);
      }
    };
    bool ok = true;
    int g = 0, nw = 0, nr = 0;
    struct Pending { int g, n16; bool any; } late = {0, 0, false};
    const auto out = [&](const Pending& q) {
      if (!warp_wait(smem_u32(&bar_p_full[q.g % NS]), (q.g / NS) & 1, abort_flag, status, 20, q.g)) return false;
      uint32_t bz = sY + (q.g % NY) * S::Y_BYTES;
      if (!S::TWO) {
        if (!warp_wait(smem_u32(&bar_z_full[q.g % NZ]), (q.g / NZ) & 1, abort_flag, status, 22, q.g)) return false;
        bz = sZ + (q.g % NZ) * S::Y_BYTES;
      }
      tc_fence_after();
      if (elect_one()) {
        weighted(tmem + S::T_OUT, tmem + (q.g % NS) * BN, bz, q.n16);
        umma_commit(smem_u32(&bar_o_full[q.g % NO]));
      }
      __syncwarp();
      return true;
    };
    for (; ok; ++nr) {
      if (!warp_wait(smem_u32(&bar_w_full[nr % NW]), (nr / NW) & 1, abort_flag, status, 27, nr)) { ok = false; break; }
      const Work k = works[nr % NW];
      if (k.end) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_w_empty[nr % NW]));
      if (k.steps == 0 || k.skip) {
        if (late.any && !out(late)) { ok = false; break; }
        late.any = false;
        continue;
      }
      if (!warp_wait(smem_u32(&bar_x_full), nw & 1, abort_flag, status, 23, nr)) { ok = false; break; }
      Steps<MODE, DP> step(t, k);
      int n16 = (step.n + 15) & ~15;
      const int steps = k.steps;
      for (int s = 0; s < steps; ++s, ++g) {
        const uint32_t id = (1u << 4) | ((uint32_t)(n16 >> 3) << 17) | ((128u >> 4) << 24);
        const uint32_t at = tmem + (g % NS) * BN;
        const uint32_t y = sY + (g % NY) * S::Y_BYTES, z = sZ + (g % NZ) * S::Y_BYTES;
        if (S::TWO) {
          // dP(g), S(g), OUT(g - 1).  The last readers of these buffers: the weights of step g - 2 are complete
          // (OUT(g - 2) waited for them), and OUT(g - 2) itself has to be over; dP(g) keeps the tensor cores busy meanwhile.
          if (s == 0) {
            // (whoever brings the second operand first finishes the work before: its last step cannot wait for this one)
            if (late.any && !out(late)) { ok = false; break; }
            late.any = false;
            if (!warp_wait(smem_u32(&bar_x2_full), nw & 1, abort_flag, status, 28, nr)) { ok = false; break; }
          }
          if (!warp_wait(smem_u32(&bar_y_full[g % NY]), (g / NY) & 1, abort_flag, status, 26, g)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) second_scores(at + S::T_DP, z, id);
          __syncwarp();
          // (a first step has nothing to wait for: OUT(g - 1), in front of it, waited until OUT(g - 2) had been read)
          if (s > 0 && g >= 2 && !warp_wait(smem_u32(&bar_o_full[(g - 2) % NO]), ((g - 2) / NO) & 1, abort_flag, status, 25, g)) { ok = false; break; }
        } else {
          // S(g), OUT(g - 1); the weights of step g - 3 were in this buffer, and OUT(g - 2) waited until OUT(g - 3) was read
          if (!warp_wait(smem_u32(&bar_y_full[g % NY]), (g / NY) & 1, abort_flag, status, 24, g)) { ok = false; break; }
        }
        tc_fence_after();
        if (elect_one()) {
          scores(at, sX, y, id);
          umma_commit(smem_u32(&bar_s_full[g % NS]));
          if (s == steps - 1) umma_commit(smem_u32(&bar_x_empty));
        }
        __syncwarp();
        const Pending now = {g, n16, true};
        step.next(t, k);                                         // while the scores run
        n16 = (step.n + 15) & ~15;
        if (late.any && !out(late)) { ok = false; break; }
        late = now;
      }
      ++nw;
    }
    if (ok && late.any) out(late);
  } else {
    // ---- weights and sums -------------------------------------------------------------------------
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    constexpr int COLS = BN / kParts, OUT = DP / kParts;
    const AttnArgs& a = t.a;
    const int past = a.kv_len - a.q_len, row_in = quarter * 32 + lane;
    bool ok = true;
    int g = 0, buf = 0;
    uint32_t buf_phase = 0;
    // The warps of a quarter hold parts of the same rows: one value of each row from every warp to every other.  The barrier
    // itself has no limit, so a warp that gives up arrives once more on its way out (below), and those it lets go look
    // whether somebody has given up.
    const auto share = [&](float (*buffer)[32], float mine, float (&all)[kParts]) {
      buffer[quarter * kParts + part][lane] = mine;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + quarter), "n"(32 * kParts) : "memory");
      if (__any_sync(0xffffffffu, *abort_flag)) return false;
#pragma unroll
      for (int i = 0; i < kParts; ++i) all[i] = buffer[quarter * kParts + i][lane];
      return true;
    };
    // The running sums of a tile are finished during the first step of the next one: its first weights are computed (and the
    // second product of this tile started) before this tile's results are stored.
    uint64_t sums[OUT / 2];
    float m = -CUDART_INF_F, l = 0.0f, times = 1.0f;             // FWD: maximum and sum; DQ: what the sums are multiplied by
    float keep_before = 1.0f, factor_before = 1.0f;
    int pending = -1;                                              // the slot of the work that is not finished
#pragma unroll
    for (int i = 0; i < OUT / 2; ++i) sums[i] = 0;
    const int rows = S::KEYS ? a.kv_len : a.q_len;
    // sums = sums * keep + tile (FWD), or sums + tile * factor, with what belonged to step gd
    const auto drain = [&](int gd) {
      if (!warp_wait(smem_u32(&bar_o_full[gd % NO]), (gd / NO) & 1, abort_flag, status, 30, gd)) return false;
      tc_fence_after();
      uint32_t v[OUT];
#pragma unroll
      for (int q = 0; q < OUT / 16; ++q) tmem_ld16(tmem + lanes + S::T_OUT + part * OUT + q * 16, v + q * 16);
      tmem_ld_wait();
      const float f = MODE == FWD ? keep_before : factor_before;
      const uint64_t f2 = pack2(f, f);
#pragma unroll
      for (int i = 0; i < OUT / 2; ++i) {
        const uint64_t x = pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        sums[i] = MODE == FWD ? fma2(sums[i], f2, x) : fma2(x, f2, sums[i]);
      }
      return true;
    };
    // The results of the work in `slot`, whose maximum, sum and factor are given; the sums are zero after it.
    const auto finish = [&](int slot, float top, float sum, float factor_of) {
      const Work& k = works[slot];
      const int row = k.row0 + row_in, steps = k.steps;
      const int xh = S::KEYS ? k.b * a.kv_heads + k.hk : k.b * a.q_heads + k.h;
      float* dst;
      int accumulate = 0, limit = rows, pitch_cols = a.dim;
      float mul = 1.0f;
      bool empty = false;
      int64_t at = ((int64_t)xh * rows + row) * a.dim;
      if (MODE == FWD) {
        if (steps > 0) {
          float all[kParts];
          if (!share(exchange[2], sum, all)) return false;
          sum = __fadd_rn(__fadd_rn(all[0], all[1]), __fadd_rn(all[2], all[3]));
        }
        empty = steps == 0 || row + past > k.p_hi;
        mul = __fmul_rn(__fdiv_rn(1.0f, sum), pow2f_int(k.ev));
        if (k.split_up) {
          mul = 1.0f;
          if (part == 0) t.stats[(int64_t)k.part * kRowsM + row_in] = make_float2(empty ? -CUDART_INF_F : top, empty ? 0.0f : sum);
        } else if (part == 0 && row < rows)
          reinterpret_cast<float2*>(a.lse)[(int64_t)xh * rows + row] =
              empty ? make_float2(CUDART_INF_F, 0.0f) : lnn::log_sum(top, score_factor(a, k.eq, k.ek), __fmul_rn(sum, kWeightUnit));
        dst = a.o;
      } else if (MODE == DQ) {
        mul = factor_of;
        dst = a.dq; accumulate = a.acc_q;
      } else {
        if (MODE == DK) mul = fabsf(a.scale);
        dst = MODE == DK ? a.dk : a.dv;
        accumulate = MODE == DK ? a.acc_k : a.acc_v;
      }
      if (k.split_up) {
        dst = t.parts; accumulate = 0; limit = k.row0 + kRowsM;
        at = ((int64_t)k.part * kRowsM + row_in) * DP;
        pitch_cols = DP;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_w_empty[slot]));
      const uint64_t mul2x = pack2(mul, mul);
      const bool vec = pitch_cols % 8 == 0 && (((uintptr_t)dst) & 31) == 0;
      // A lane has one row of the warp's columns, in pieces of 32 bytes.  The lanes of a group change pieces, so that they
      // hold one piece each of as many rows and store 128 bytes of a row together (a tile of 64 KB in
      // 4000 clocks; in pieces of 32 bytes 6000).
      constexpr int G = OUT / 8;
#pragma unroll
      for (int i = 0; i < OUT / 2; ++i) sums[i] = MODE == FWD && empty ? 0 : mul2(sums[i], mul2x);
      if (vec) {
#pragma unroll
        for (int bit = 1; bit < G; bit <<= 1) {
          const bool up = lane & bit;
#pragma unroll
          for (int i = 0; i < G; ++i) {
            if (i & bit) continue;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint64_t &x = sums[i * 4 + u], &y = sums[(i | bit) * 4 + u];
              const uint64_t got = __shfl_xor_sync(0xffffffffu, up ? x : y, bit);
              if (up) x = got; else y = got;
            }
          }
        }
        const int piece = part * OUT + lane % G * 8, row_first = row - lane % G;
        float* to = dst + at - (int64_t)(lane % G) * pitch_cols + piece;
#pragma unroll
        for (int i = 0; i < G; ++i) {
          if (row_first + i < limit && piece < pitch_cols) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; u += 2) unpack2(sums[i * 4 + u / 2], x[u], x[u + 1]);
            float* o = to + (int64_t)i * pitch_cols;
            if (MODE != FWD && accumulate) {
              const float4 y0 = *reinterpret_cast<const float4*>(o), y1 = *reinterpret_cast<const float4*>(o + 4);
              const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
              for (int u = 0; u < 8; ++u) x[u] = __fadd_rn(y[u], x[u]);
            }
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
                         "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                         : "memory");
          }
        }
      } else {
        float* to = dst + at + part * OUT;
        const int cols = row < limit ? pitch_cols - part * OUT : 0;  // of this warp's part
#pragma unroll
        for (int i = 0; i < OUT; i += 2) {
          float x[2];
          unpack2(sums[i / 2], x[0], x[1]);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (i + u < cols) to[i + u] = MODE != FWD && accumulate ? __fadd_rn(to[i + u], x[u]) : x[u];
        }
      }
#pragma unroll
      for (int i = 0; i < OUT / 2; ++i) sums[i] = 0;
      return true;
    };
    int nr = 0, nw = 0;
    for (; ok; ++nr) {
      const int slot = nr % NW;
      if (!warp_wait(smem_u32(&bar_w_full[slot]), (nr / NW) & 1, abort_flag, status, 33, nr)) { ok = false; break; }
      const Work& k = works[slot];
      if (k.end) break;
      const int steps = k.steps, row0 = k.row0;
      if (k.skip || steps == 0) {
        // (behind the results that are still to be stored)
        if (pending >= 0 && (!drain(g - 1) || !finish(pending, m, l, times))) { ok = false; break; }
        pending = -1;
        if (!k.skip) {
          // nothing is seen: zeros
          if (!finish(slot, 0.0f, 1.0f, 1.0f)) { ok = false; break; }
        } else {
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_w_empty[slot]));
        }
        continue;
      }
      const int row = row0 + row_in;
      const int xh = S::KEYS ? k.b * a.kv_heads + k.hk : k.b * a.q_heads + k.h;
      const float m_old = m, l_old = l, times_old = times;
      m = -CUDART_INF_F;
      l = 0.0f;
      float row_hi = -CUDART_INF_F, row_up = 0.0f, row_less = 0.0f;      // DQ: see PrepArgs
      int row_exp = 0;                                             // DQ, DK: dS is scaled by 2^row_exp
      float norm = 0.0f;
      if (S::TWO && row < rows) norm = sqrtf(__ldg(t.norms + (int64_t)xh * rows + row));
      if (MODE == DQ && row < rows) {
        row_hi = __ldg(t.lse_p + lse_at(xh, t.pitch, row));
        row_up = __ldg(t.lse_p + lse_at(xh, t.pitch, row) + 2);
        row_less = __ldg(t.delta_p + (int64_t)xh * t.pitch + row);
      }
      if (S::TWO) {
        // The second stationary operand into TMEM, once the products of the work before are over: this warp's fourth of
        // the columns of its rows, hi and lo (what is no row of the tensor is zero).
        if (!warp_wait(smem_u32(&bar_x_empty), (nw & 1) ^ 1, abort_flag, status, 34, nr)) { ok = false; break; }
        const int64_t lo_at = (int64_t)(S::KEYS ? a.batch * a.kv_heads : a.batch * a.q_heads) * rows * (t.width / 2);
        const uint32_t* src = t.x2 + ((int64_t)xh * rows + row) * (t.width / 2) + part * (DP / 8);
        tc_fence_after();
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t x[DP / 8];
#pragma unroll
          for (int i = 0; i < DP / 8; i += 4) {
            const uint4 v = row < rows && part * (DP / 8) + i < t.width / 2 ? __ldg(reinterpret_cast<const uint4*>(src + p * lo_at + i)) : make_uint4(0, 0, 0, 0);
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
          }
          const uint32_t to = tmem + lanes + S::T_X2 + p * (DP / 2) + part * (DP / 8);
          if (DP == 128) tmem_st16(to, x);
          else tmem_st8(to, x);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_x2_full));
        ++nw;
      }
      int cur_head = -1;
      float c = 0.0f, cdp = 0.0f, factor = 1.0f;
      Steps<MODE, DP> step(t, k);
      for (int s = 0; s < steps; ++s, ++g, buf_phase ^= buf == NS - 1, buf = buf == NS - 1 ? 0 : buf + 1, step.next(t, k)) {
        const int r0 = step.r, n = step.n, qh = S::KEYS ? step.head : xh;
        if (qh != cur_head) {                                      // the scales that go with a query head
          int eq = k.eq, eo = k.eo;
          float norm_do = k.norm_do;
          if (S::KEYS && (cur_head >= 0 || k.hq0 > 0)) {
            const HeadInfo io = lnn::info_of(a, 3, qh);
            eq = lnn::info_of(a, 0, qh).e; eo = io.e; norm_do = io.norm;
          }
          cur_head = qh;
          c = score_factor(a, eq, k.ek);
          if (MODE == DV) factor = pow2f_int(eo - 14);
          if (S::TWO) {
            cdp = pow2f_int(eo + k.ev);
            // |dP| <= |dO| |V|, and |delta| <= |dO| times the largest |V| of the head: below 2^15 after scaling
            const float bound = fmaxf(MODE == DK ? norm_do * (norm + k.norm_v) : 2.0f * norm * k.norm_v, 0.0009765625f);
            row_exp = 14 - ((int)(__float_as_uint(bound) >> 23) - 127) - (eo + k.ev);
            if (MODE == DK) factor = pow2f_int(eq - row_exp);
          }
        }
        // which columns of the tile this row sees: [lo, hi], and those up to hi that are below `always`
        const int col0 = part * COLS;
        bool all;
        uint32_t seen = 0xffffffffu;
        if (!S::KEYS) {
          const int p = row + past;
          all = n == BN && r0 + BN - 1 <= row0 + past && (k.p_hi - r0 < a.window || r0 + BN <= a.sinks);
          if (!all) seen = bits_to(min(p - r0, n - 1) - col0) & (~bits_to(p - a.window - r0 - col0) | bits_to(a.sinks - 1 - r0 - col0));
        } else {
          all = n == BN && r0 + past >= row0 + kRowsM - 1 &&
                (r0 + past + BN - 1 < row0 + a.window || row0 + kRowsM <= a.sinks);
          const int last = row < a.sinks ? k.q_hi : (int)min((int64_t)row + a.window - 1, (int64_t)k.q_hi);
          if (!all) seen = bits_to(min(last - past - r0, n - 1) - col0) & ~bits_to(row - past - r0 - 1 - col0);
        }
        const uint32_t ts = tmem + lanes + buf * BN + col0;
        if (S::KEYS && !warp_wait(smem_u32(&bar_c_full[g % NC]), (g / NC) & 1, abort_flag, status, 35, g)) { ok = false; break; }
        if (!warp_wait(smem_u32(&bar_s_full[buf]), buf_phase, abort_flag, status, 31, g)) { ok = false; break; }
        tc_fence_after();
        if (MODE == FWD) {
          // (the scores are read twice, 16 at a time: registers)
          float top = -CUDART_INF_F;
          if (col0 < n) {
#pragma unroll
            for (int q = 0; q < COLS / 16; ++q) {
              uint32_t v[16];
              tmem_ld16(ts + q * 16, v);
              tmem_ld_wait();
              if (!all) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (!(seen >> (q * 16 + i) & 1u)) v[i] = 0xff800000u;
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) top = fmaxf(top, __uint_as_float(v[i]));
            }
          }
          float tops[kParts];
          if (!share(exchange[g & 1], top, tops)) { ok = false; break; }
          top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          // (differences of scores before the factor: exact near the maximum, whose weight is 2^14 however large the scores are)
          const float now = fmaxf(m, top);
          const float at = now == -CUDART_INF_F ? 0.0f : now;
          const float keep = exp2_fast(__fmul_rn(__fsub_rn(m, at), c));
          const uint64_t c2 = pack2(c, c), less = pack2(-at, -at), shift = pack2(14.0f, 14.0f);
          uint64_t sum = 0;
          if (col0 < n) {
#pragma unroll
            for (int q = 0; q < COLS / 16; ++q) {
              uint32_t v[16];
              uint64_t wt[8];
              tmem_ld16(ts + q * 16, v);
              tmem_ld_wait();
              if (!all) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (!(seen >> (q * 16 + i) & 1u)) v[i] = 0xff800000u;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float x, y;
                unpack2(fma2(add2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), less), c2, shift), x, y);
                wt[i] = pack2(exp2_fast(x), exp2_fast(y));
                sum = add2(sum, wt[i]);
              }
              store_split(ts + q * 16, wt);
            }
          }
          float s0, s1;
          unpack2(sum, s0, s1);
          l = fmaf(l, keep, __fadd_rn(s0, s1));
          m = now;
          if ((s > 0 || pending >= 0) && !drain(g - 1)) { ok = false; break; }
          keep_before = keep;
        } else {
          if (col0 < n) {
            const float exponent = S::TWO ? (float)row_exp : 14.0f, more = exponent - 14.0f;
            const uint64_t c2 = pack2(c, c), cdp2 = pack2(cdp, cdp), more2 = pack2(more, more);
            uint64_t hi = pack2(row_hi, row_hi), up = pack2(row_up + more, row_up + more), less = pack2(row_less, row_less);
            const float* cl = &col_lse[S::KEYS ? g % NC : 0][S::KEYS ? 2 * col0 : 0];
            const float* cd = &col_delta[MODE == DK ? g % NC : 0][MODE == DK ? col0 : 0];
#pragma unroll
            for (int q = 0; q < COLS / 16; ++q) {
              uint32_t v[16], d[16];
              uint64_t wt[8];
              tmem_ld16(ts + q * 16, v);
              if (S::TWO) tmem_ld16(ts + S::T_DP + q * 16, d);
              tmem_ld_wait();
              if (!all) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (!(seen >> (q * 16 + i) & 1u)) v[i] = 0xff800000u;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (S::KEYS) {                                     // (a warp reads one address)
                  const float4 l4 = *reinterpret_cast<const float4*>(cl + (q * 16 + 2 * i) * 2);
                  hi = pack2(l4.x, l4.y);
                  up = S::TWO ? add2(pack2(l4.z, l4.w), more2) : pack2(l4.z, l4.w);
                  if (S::TWO) {
                    const float2 d2 = *reinterpret_cast<const float2*>(cd + q * 16 + 2 * i);
                    less = pack2(d2.x, d2.y);
                  }
                }
                float x, y;
                unpack2(add2(fma2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), c2, hi), up), x, y);
                // (1 at most but for the last bits: the scores are those of FWD to the bit, the logarithm has no step of its own)
                wt[i] = pack2(exp2_fast(x), exp2_fast(y));
                if (S::TWO)
                  wt[i] = mul2(wt[i], fma2(pack2(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])), cdp2, less));
              }
              store_split(ts + q * 16, wt);
            }
          }
          if ((s > 0 || pending >= 0) && !drain(g - 1)) { ok = false; break; }
          factor_before = factor;
        }
        // the weights are there, and OUT(g - 1) has been read: OUT(g) may start
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_p_full[buf]));
        if (pending >= 0) {
          if (!finish(pending, m_old, l_old, times_old)) { ok = false; break; }
          pending = -1;
        }
      }
      if (!ok) break;
      if (MODE == DQ) times = __fmul_rn(a.scale, pow2f_int(k.ek - row_exp));
      pending = slot;
    }
    if (ok && pending >= 0) ok = drain(g - 1) && finish(pending, m, l, times);
    if (!ok) asm volatile("bar.arrive %0, %1;" ::"r"(1 + quarter), "n"(32 * kParts) : "memory");
  }

  // ---- tear-down ------------------------------------------------------------------------------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // copies issued before the abort may still be landing in this CTA's shared memory
    const long long t0 = clock64();
    while (clock64() - t0 < kAbortDelay) { }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (t.beside) lnn::wait_at_end();
}

// dK and dV of the tiles that several works shared: their parts in order.
constexpr int kPartBlocks = 8;                   // blocks per tile
template <int DP>
__global__ void __launch_bounds__(256)
attn_parts_kernel(const __grid_constant__ TcArgs tk, const __grid_constant__ TcArgs tv, int blocks_k) {
  lnn::wait_for_previous();
  const bool values = (int)blockIdx.x >= blocks_k;               // blocks of dK first, if any
  const TcArgs& t = values ? tv : tk;
  const AttnArgs& a = t.a;
  constexpr int ROWS = kRowsM / kPartBlocks;
  const int block = values ? blockIdx.x - blocks_k : blockIdx.x;
  const int tile = block / kPartBlocks, first = block % kPartBlocks * ROWS, hk = blockIdx.y, b = blockIdx.z;
  const int splits = tile < t.sink_tiles ? t.splits_sink : t.splits;
  if (splits == 1 || !lnn::group_ok(a, b, hk)) return;
  float* __restrict__ dst = values ? a.dv : a.dk;
  const float* __restrict__ parts = t.parts;
  const bool accumulate = values ? a.acc_v : a.acc_k;
  const int64_t w0 = (int64_t)(b * a.kv_heads + hk) * parts_per_head(t) +
                     (tile < t.sink_tiles ? tile * t.splits_sink : t.sink_tiles * t.splits_sink + (tile - t.sink_tiles) * t.splits);
  for (int i = threadIdx.x; i < ROWS * DP / 4; i += 256) {
    const int row = tile * kRowsM + first + i / (DP / 4), col = i % (DP / 4) * 4;
    if (row >= a.kv_len || col >= a.dim) continue;
    const float4* from = reinterpret_cast<const float4*>(parts + w0 * kRowsM * DP + first * DP) + i;
    float4 s = __ldg(from);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
      const float4 x = __ldg(from + (int64_t)k * (kRowsM * DP / 4));
      s = make_float4(__fadd_rn(s.x, x.x), __fadd_rn(s.y, x.y), __fadd_rn(s.z, x.z), __fadd_rn(s.w, x.w));
    }
    float* to = dst + ((int64_t)(b * a.kv_heads + hk) * a.kv_len + row) * a.dim + col;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (col + u < a.dim) to[u] = accumulate ? __fadd_rn(to[u], v[u]) : v[u];
  }
}

// O or dQ of the tiles of queries that several works shared.
template <int MODE, int DP>
__global__ void __launch_bounds__(256)
attn_merge_kernel(const __grid_constant__ TcArgs t) {
  lnn::wait_for_previous();
  constexpr int ROWS = kRowsM / kPartBlocks;
  const AttnArgs& a = t.a;
  const int work = blockIdx.x / kPartBlocks, first = blockIdx.x % kPartBlocks * ROWS;
  const int heads = a.batch * a.q_heads, w = t.whole + work, turn = w / heads, head = w - turn * heads;
  const int b = head / a.q_heads, hk = (head - b * a.q_heads) / (a.q_heads / a.kv_heads), row0 = (t.tiles - 1 - turn) * kRowsM;
  if (!lnn::group_ok(a, b, hk)) return;
  const int past = a.kv_len - a.q_len, len = lnn::attn_length(a.lengths, b, a.kv_len, a.status);
  const float scale_v = MODE == FWD ? pow2f_int(lnn::info_of(a, 2, b * a.kv_heads + hk).e) : 1.0f;
  const float c = MODE == FWD ? score_factor(a, lnn::info_of(a, 0, head).e, lnn::info_of(a, 1, b * a.kv_heads + hk).e) : 1.0f;
  const int64_t part0 = (int64_t)work * t.splits;
  for (int i = threadIdx.x; i < ROWS * DP / 4; i += 256) {
    const int r = first + i / (DP / 4), col = i % (DP / 4) * 4, row = row0 + r;
    if (row >= a.q_len || col >= a.dim) continue;
    const float4* from = reinterpret_cast<const float4*>(t.parts + (part0 * kRowsM + r) * DP + col);
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float top = -CUDART_INF_F, total = 0.0f;
    if (MODE == FWD)
      for (int k = 0; k < t.splits; ++k) top = fmaxf(top, __ldg(t.stats + (part0 + k) * kRowsM + r).x);
    const float base = top == -CUDART_INF_F ? 0.0f : top;
#pragma unroll 4
    for (int k = 0; k < t.splits; ++k) {
      const float4 x = __ldg(from + (int64_t)k * (kRowsM * DP / 4));
      float f = 1.0f;
      if (MODE == FWD) {
        const float2 st = __ldg(t.stats + (part0 + k) * kRowsM + r);
        f = exp2_fast(__fmul_rn(__fsub_rn(st.x, base), c));
        total = fmaf(f, st.y, total);
      }
      s = make_float4(fmaf(x.x, f, s.x), fmaf(x.y, f, s.y), fmaf(x.z, f, s.z), fmaf(x.w, f, s.w));
    }
    const int64_t at = ((int64_t)head * a.q_len + row) * a.dim + col;
    float v[4] = {s.x, s.y, s.z, s.w};
    if (MODE == FWD) {
      const bool empty = row + past >= len;
      const float mul = empty ? 0.0f : __fmul_rn(__fdiv_rn(1.0f, total), scale_v);
      if (col == 0)
        reinterpret_cast<float2*>(a.lse)[(int64_t)head * a.q_len + row] =
            empty ? make_float2(CUDART_INF_F, 0.0f) : lnn::log_sum(top, c, __fmul_rn(total, kWeightUnit));
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (col + u < a.dim) a.o[at + u] = empty ? 0.0f : __fmul_rn(v[u], mul);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (col + u < a.dim) a.dq[at + u] = a.acc_q ? __fadd_rn(a.dq[at + u], v[u]) : v[u];
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------
// [2 heads][rows][width] fp16: lo behind hi; the boxes are 64 wide (zeros behind the width)
int operand_map(CUtensorMap* tm, const void* base, int width, int rows, int64_t heads) {
  const uint64_t dims[3] = {(uint64_t)width, (uint64_t)rows, (uint64_t)(2 * heads)};
  const uint64_t strides[2] = {(uint64_t)width * 2, (uint64_t)rows * width * 2};
  const uint32_t box[3] = {64, kBoxRows, 1}, es[3] = {1, 1, 1};
  return lnn_tc::encode_half_map(tm, base, 3, dims, strides, box, es);
}

template <int MODE, int DP>
int launch_pass(lnn::Device* d, const CUtensorMap* x, const CUtensorMap* y, const CUtensorMap* z, const TcArgs& t) {
  using S = Shape<MODE, DP>;
  // The tiles begin at a multiple of 1024, for which there is that much room where the block has it; DK at 128 values leaves 256
  // bytes: enough behind what the kernel declares itself, and the kernel looks whether it is.
  static size_t declared = 0;
  if (declared == 0) {
    cudaFuncAttributes attr;
    LNN_CUDA(cudaFuncGetAttributes(&attr, attn_tc_kernel<MODE, DP>));
    declared = attr.sharedSizeBytes;
  }
  const size_t bytes = std::min<size_t>(S::TILES + 1024, 227 * 1024 - declared);
  LNN_CUDA(cudaFuncSetAttribute(attn_tc_kernel<MODE, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  LNN_CUDA(lnn::launch_chained(d, attn_tc_kernel<MODE, DP>, std::min(t.works, d->sm_count), kAttnThreads, bytes, *x, *y, *z, t));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

// What a work costs beside its steps (its first loads, its results), in steps; the traffic of one part; a launch.
constexpr double kWorkCost = 3.0, kPartCost = 0.011, kMergeCost = 1.5;

// Works of a pass over keys: how often a tile's steps are cut, so that the rounds of the SMs come out even.
template <int MODE, int DP>
void plan_keys(const lnn::Device* d, TcArgs& t) {
  constexpr int BN = Shape<MODE, DP>::BN;
  const AttnArgs& a = t.a;
  const int64_t group = a.q_heads / a.kv_heads, heads = (int64_t)a.batch * a.kv_heads;
  t.tiles = (a.kv_len + kRowsM - 1) / kRowsM;
  t.sink_tiles = std::min(t.tiles, (a.sinks + kRowsM - 1) / kRowsM);
  const int64_t most = group * ((a.q_len + BN - 1) / BN + 1);                      // steps of a tile that sees all queries
  const int64_t some = std::min<int64_t>(most, group * ((std::min<int64_t>((int64_t)a.window + kRowsM, a.q_len) + BN - 1) / BN + 1));
  double best = 0.0;
  for (int splits = 1; splits <= 32 && splits <= some; ++splits) {
    const int64_t length = (some + splits - 1) / splits, sink = std::min<int64_t>(64, (most + length - 1) / length);
    const int64_t works = heads * (t.sink_tiles * sink + (t.tiles - t.sink_tiles) * splits);
    const int64_t parts = heads * ((sink > 1 ? t.sink_tiles * sink : 0) + (splits > 1 ? (t.tiles - t.sink_tiles) * splits : 0));
    const double cost = (double)((works + d->sm_count - 1) / d->sm_count) * (double)(std::max(length, (most + sink - 1) / sink) + kWorkCost) +
                        kPartCost * (double)parts + (parts ? kMergeCost : 0.0);
    if (splits == 1 || cost < best) {
      best = cost;
      t.splits = splits; t.splits_sink = (int)sink; t.works = (int)works;
    }
  }
}

// Works of a pass over queries: those of the last round of the SMs, or all where they are few, may be cut.  A pass beside
// others fills their gaps with whole ones (8192 positions of 8 heads with gradients: 1080 us with DQ's last round cut, 1073).
template <int MODE, int DP>
void plan_queries(const lnn::Device* d, TcArgs& t, bool alone) {
  constexpr int BN = Shape<MODE, DP>::BN;
  const AttnArgs& a = t.a;
  t.tiles = (a.q_len + kRowsM - 1) / kRowsM;
  const int64_t all = (int64_t)a.batch * a.q_heads * t.tiles, full = all / d->sm_count, rest = all - full * d->sm_count;
  // steps of the first work of the last round, the longest of them
  const int64_t row0 = (t.tiles - 1 - full * d->sm_count / ((int64_t)a.batch * a.q_heads)) * kRowsM, past = a.kv_len - a.q_len;
  const int64_t p_hi = std::min<int64_t>(row0 + kRowsM, a.q_len) - 1 + past, lowest = std::max<int64_t>(row0 + past - a.window + 1, 0);
  const int64_t steps = rest > 0 ? (std::min<int64_t>(a.sinks, lowest) + BN - 1) / BN + (p_hi - lowest) / BN + 1 : 0;
  double best = (rest > 0 ? 1.0 : 0.0) * ((double)steps + kWorkCost);
  t.splits = 1;
  for (int splits = 2; splits <= 32 && splits <= steps && rest > 0 && (alone || full == 0); ++splits) {
    const double cost = (double)((rest * splits + d->sm_count - 1) / d->sm_count) * ((double)((steps + splits - 1) / splits) + kWorkCost) +
                        kPartCost * (double)(rest * splits) + kMergeCost;
    if (cost < best) { best = cost; t.splits = splits; }
  }
  t.whole = t.splits > 1 ? (int)(full * d->sm_count) : (int)all;
  t.works = t.whole + (int)(t.splits > 1 ? rest * t.splits : 0);
}

struct Operands {
  lnn::Scratch halves, small;
  PrepArgs p = {};
  CUtensorMap map[4];
  explicit Operands(lnn::Device* d) : halves(d), small(d) {}
};

// q, k, v and (backward) dO into their split form
template <int DP>
int prepare(lnn::Device* d, AttnArgs& a, Operands& op, bool backward) {
  PrepArgs& p = op.p;
  const int past = a.kv_len - a.q_len, first = std::max(0, past - a.window + 1);
  const int64_t nq = (int64_t)a.batch * a.q_heads, nk = (int64_t)a.batch * a.kv_heads;
  p.width = (a.dim + 15) / 16 * 16;
  const int64_t sq = nq * a.q_len * p.width, sk = nk * a.kv_len * p.width;
  int rc = op.halves.get((uint64_t)(2 * (sq + 2 * sk + (backward ? sq : 0))) * 2);
  if (rc) return rc;
  __half* h = op.halves.as<__half>();
  __half* at[4] = {h, h + 2 * sq, h + 2 * sq + 2 * sk, h + 2 * sq + 4 * sk};
  p.tensors = backward ? 4 : 3;
  p.dim = a.dim; p.batch = a.batch; p.lengths = a.lengths; p.kv_len = a.kv_len; p.status = a.status;
  // one round of blocks: each has about 5 us of latencies (the sample, the last block's turn) to hide behind its rows
  const auto row_blocks = [&](int rows) { return ((int64_t)rows + p.block_rows - 1) / p.block_rows; };
  p.block_rows = kPrepRows;
  while ((backward ? 2 : 1) * nq * row_blocks(a.q_len) + 2 * nk * row_blocks(a.kv_len) > kPrepBlocksPerSm * d->sm_count && p.block_rows < 1024)
    p.block_rows += kPrepRows;
  p.blocks = (int)row_blocks(a.kv_len);
  p.pitch = (a.q_len + 7) / 8 * 8 + kRowsM;
  const int64_t heads = 2 * nk + (backward ? 2 : 1) * nq;
  const int64_t norm_words = backward ? nk * a.kv_len + nq * a.q_len : 0, col_words = backward ? 3 * nq * p.pitch : 0;
  const int64_t info_words = (heads * (int64_t)sizeof(HeadInfo) / 4 + 3) / 4 * 4;
  rc = op.small.get((uint64_t)(4 + info_words + (col_words + 3) / 4 * 4 + 2 * heads * p.blocks + norm_words) * 4);
  if (rc) return rc;
  float* s = op.small.as<float>();
  p.taken = (int*)s; s += 4;
  p.info = (HeadInfo*)s; s += info_words;
  p.lse_p = s; p.delta_p = s + 2 * nq * p.pitch; s += (col_words + 3) / 4 * 4;       // (16-byte aligned: the pitch is a multiple of 8)
  p.block_max = s; s += heads * p.blocks;
  p.block_norm = s; s += heads * p.blocks;
  float *norm_v = backward ? s : nullptr, *norm_do = backward ? s + nk * a.kv_len : nullptr;
  p.counters = d->tile_counters;
  p.t[0] = {a.q, at[0], nullptr, (int)nq, a.q_heads, a.q_len, 0, 0, past, a.scale < 0.0f ? -1.0f : 1.0f};
  p.t[1] = {a.k, at[1], nullptr, (int)nk, a.kv_heads, a.kv_len, first, a.sinks, 0, 1.0f};
  p.t[2] = {a.v, at[2], norm_v, (int)nk, a.kv_heads, a.kv_len, first, a.sinks, 0, 1.0f};
  p.t[3] = {a.dout, at[3], norm_do, (int)nq, a.q_heads, a.q_len, 0, 0, past, 1.0f};
  if (backward) { p.o = a.o; p.lse = a.lse; }
  a.info = p.info;
  a.backward = backward;
  for (int i = 0; i < p.tensors; ++i) {
    rc = operand_map(&op.map[i], at[i], p.width, p.t[i].rows, p.t[i].heads);
    if (rc) return rc;
  }
  const bool vec = a.dim % 4 == 0 && (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (backward ? (uintptr_t)a.dout | (uintptr_t)a.o : 0)) & 15) == 0;
  const dim3 grid((unsigned)p.blocks, (unsigned)heads);
  if (vec) LNN_CUDA(lnn::launch_chained(d, attn_prep_kernel<DP, true>, grid, kPrepThreads, 0, p));
  else LNN_CUDA(lnn::launch_chained(d, attn_prep_kernel<DP, false>, grid, kPrepThreads, 0, p));
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

// A pass over queries, and the launch that joins its parts.
template <int MODE, int DP>
struct QueriesPass {
  lnn::Scratch parts;
  TcArgs t;
  int64_t n = 0;
  QueriesPass(lnn::Device* d, const TcArgs& args) : parts(d), t(args) {}
  int run(lnn::Device* d, const Operands& op, bool alone) {
    plan_queries<MODE, DP>(d, t, alone);
    n = t.works - t.whole;
    if (n > 0) {
      const int rc = parts.get((uint64_t)n * kRowsM * (DP * 4 + (MODE == FWD ? 8 : 0)));
      if (rc) return rc;
      t.parts = parts.as<float>();
      t.stats = reinterpret_cast<float2*>(t.parts + n * kRowsM * DP);
    }
    return launch_pass<MODE, DP>(d, &op.map[0], &op.map[1], &op.map[2], t);
  }
  int join(lnn::Device* d) {
    if (n == 0) return LNN_OK;
    LNN_CUDA(lnn::launch_chained(d, attn_merge_kernel<MODE, DP>, (unsigned)(n / t.splits * kPartBlocks), 256, 0, t));
    LNN_CHECK_LAUNCH(d);
    return LNN_OK;
  }
};

template <int DP>
int tc_fwd(lnn::Device* d, AttnArgs a) {
  Operands op(d);
  int rc = prepare<DP>(d, a, op, false);
  if (rc) return rc;
  TcArgs t = {};
  t.a = a;
  t.width = op.p.width;
  t.taken = op.p.taken;
  QueriesPass<FWD, DP> pass(d, t);
  a.beside = 1;
  if ((rc = pass.run(d, op, true)) || (rc = lnn::attn_simt_fwd(d, a))) return rc;      // (the latter: the heads that were marked)
  return pass.join(d);
}

template <int MODE, int DP>
struct KeysPass {
  lnn::Scratch parts;
  TcArgs t;
  bool cut = false;
  KeysPass(lnn::Device* d, const TcArgs& args) : parts(d), t(args) {}
  int run(lnn::Device* d, const Operands& op) {
    plan_keys<MODE, DP>(d, t);
    cut = t.splits > 1 || t.splits_sink > 1;
    const int64_t n = cut ? (int64_t)t.a.batch * t.a.kv_heads * ((int64_t)t.sink_tiles * t.splits_sink +
                                                                 (t.splits > 1 ? (int64_t)(t.tiles - t.sink_tiles) * t.splits : 0)) : 0;
    const int rc = n ? parts.get((uint64_t)n * kRowsM * DP * 4) : LNN_OK;
    if (rc) return rc;
    t.parts = parts.as<float>();
    return launch_pass<MODE, DP>(d, &op.map[1], &op.map[0], &op.map[3], t);
  }
};

// The three passes read the same operands and write memory of their own: the SMs that are done with one begin the next.
template <int DP>
int tc_bwd(lnn::Device* d, AttnArgs a) {
  Operands op(d);
  int rc = prepare<DP>(d, a, op, true);
  if (rc) return rc;
  TcArgs t = {};
  t.a = a;
  t.lse_p = op.p.lse_p; t.delta_p = op.p.delta_p; t.pitch = op.p.pitch; t.width = op.p.width;
  QueriesPass<DQ, DP> q(d, t);
  KeysPass<DV, DP> v(d, t);
  KeysPass<DK, DP> k(d, t);
  k.t.taken = op.p.taken;
  v.t.taken = op.p.taken + 1;
  q.t.taken = op.p.taken + 2;
  q.t.norms = op.p.t[3].norms;
  q.t.x2 = (const uint32_t*)op.p.t[3].hi;
  k.t.norms = op.p.t[2].norms;
  k.t.x2 = (const uint32_t*)op.p.t[2].hi;
  // the pass of the longest works first, that of the shortest last
  v.t.beside = a.dk != nullptr;
  q.t.beside = a.dk || a.dv;
  if (a.dk && (rc = k.run(d, op))) return rc;
  if (a.dv && (rc = v.run(d, op))) return rc;
  if (a.dq && (rc = q.run(d, op, !a.dk && !a.dv))) return rc;
  a.delta = op.p.delta_p;
  a.delta_pitch = op.p.pitch;
  a.beside = 1;
  if ((rc = lnn::attn_simt_bwd(d, a)) || (rc = q.join(d))) return rc;
  if (k.cut || v.cut) {
    const int tiles = (a.kv_len + kRowsM - 1) / kRowsM, blocks_k = k.cut ? tiles * kPartBlocks : 0, blocks_v = v.cut ? tiles * kPartBlocks : 0;
    LNN_CUDA(lnn::launch_chained(d, attn_parts_kernel<DP>,
                                 dim3((unsigned)(blocks_k + blocks_v), (unsigned)a.kv_heads, (unsigned)a.batch), 256, 0, k.t, v.t, blocks_k));
    LNN_CHECK_LAUNCH(d);
  }
  return LNN_OK;
}

}  // namespace

namespace lnn {

// Short sequences are the FP32-pipe kernels': one launch in place of three, or three in place of five, and a tile of 128 rows would
// be half empty.  us for 32 heads, FP32 pipe / tensor cores: of 64 values, 64 positions 10.3 / 15.2, 96 positions 17.5 / 15.5, with
// gradients 32.5 / 40.0 and 46.5 / 39.6; of 128 values, 32 positions 9.9 / 16.8, 64 positions 16.5 / 18.2, 96 positions 22.8 / 19.4,
// with gradients 32.6 / 41.1, 55.4 / 45.9 and 78.8 / 49.4.  (The same for both directions: the gradients' scores are to
// be those that the denominators were made of.  Only a head whose dO the split form does not hold goes back by the other way.)
bool attn_tc_applicable(const AttnArgs& a) {
  const int64_t heads = 2ll * a.batch * (a.q_heads + a.kv_heads);
  if (a.kv_len <= (a.dim <= 64 ? 64 : 32)) return false;
  return a.dim <= 128 && heads <= kTileCounters && heads < 65536;
}
int attn_tc_fwd(Device* d, const AttnArgs& a) { return a.dim <= 64 ? tc_fwd<64>(d, a) : tc_fwd<128>(d, a); }
int attn_tc_bwd(Device* d, const AttnArgs& a) { return a.dim <= 64 ? tc_bwd<64>(d, a) : tc_bwd<128>(d, a); }

}  // namespace lnn
