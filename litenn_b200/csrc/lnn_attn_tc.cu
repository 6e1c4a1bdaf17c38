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
// Each sum has one owner: no atomics, results do not change from run to run.  dV and dK are separate passes (S^T is computed
// twice) because 128 stationary rows of K and V of 128 values leave room in shared memory for two tiles of Q and one
// of dO, not for two of both.
//
// A persistent CTA of 320 threads per SM: warp 0 loads (TMA), one thread of warp 1 issues the MMAs, warps 2-9 (two per
// quarter of the TMEM lanes, half of the columns each) turn scores into weights, write them back to TMEM as the A operand
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

constexpr int kComputeWarps = 8;
constexpr int kAttnThreads = 32 * (2 + kComputeWarps);
constexpr int kBoxRows = 32;                     // rows of a TMA box
constexpr int kRowsM = 128;                      // stationary rows

// ---- preparation -----------------------------------------------------------------------------------
// One pass over each operand: split, row norms (what bounds dS), and for dO the rows of dO * O and the denominators
// with a padded pitch.  The scale of a head is guessed from 32 of its rows, so that the largest value of them is in
// [2^8, 2^9); the true maximum may be 2^7 times that before fp16 overflows.  A head beyond it, or with values that are
// not finite, is marked and goes to the FP32-pipe kernels.
constexpr int kPrepThreads = 256;
constexpr int kPrepRows = 64;
constexpr int kSampleRows = 32;

struct PrepTensor {
  const float* src;
  __half* hi;                    // [heads][rows][DP]; lo behind all heads
  float* norms;                  // [heads][rows], or null
  int heads, per_batch, rows;
  int first, sinks;              // keys: rows below `first` that are no sinks are seen by no query
  int past;                      // queries: row i is at position i + past
  float sign;
};
struct PrepArgs {
  PrepTensor t[4];
  int tensors, dim, batch;
  const float* lengths;
  int kv_len;
  HeadInfo* info;                // [all heads of all tensors]
  uint32_t* block_max;           // [head][blocks]: largest magnitudes after scaling
  float* block_norm;
  int blocks;                    // row blocks of the longest tensor
  unsigned int* counters;        // one per head, zero between launches
  // the last tensor is dO
  const float *o, *lse;
  float *lse_p, *delta_p;
  int pitch;
  int* status;
};

template <int DP>
__global__ void __launch_bounds__(kPrepThreads)
attn_prep_kernel(const __grid_constant__ PrepArgs a) {
  constexpr int E = DP / 32;                                    // elements per lane
  __shared__ uint32_t red[kPrepThreads / 32];
  __shared__ float redn[kPrepThreads / 32];
  __shared__ int last_block;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int head = blockIdx.y, ti = 0;
  while (head >= a.t[ti].heads) head -= a.t[ti++].heads;
  const PrepTensor& t = a.t[ti];
  const int blocks = (t.rows + kPrepRows - 1) / kPrepRows;
  if ((int)blockIdx.x >= blocks) return;
  const int len = lnn::attn_length(a.lengths, head / t.per_batch, a.kv_len, a.status);
  const int end = min(t.rows, len - t.past), dim = a.dim;        // rows from here on are padding
  const float* src = t.src + (int64_t)head * t.rows * dim;
  const bool vec = E == 4 && dim == DP && (((uintptr_t)t.src) & 15) == 0;
  const auto load = [&](const float* base, int r, float (&x)[E]) {
    const float* p = base + (int64_t)r * dim + lane * E;
    if (vec) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p));
      x[0] = v.x; x[1] = v.y; x[E - 2] = v.z; x[E - 1] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = lane * E + i < dim ? __ldg(p + i) : 0.0f;
    }
  };
  // the scale, from rows spread over those that are real (the same ones in every block of the head)
  uint32_t m = 0;
  const int span = end - t.first;
  if (span > 0)
    for (int i = warp; i < kSampleRows; i += kPrepThreads / 32) {
      float x[E];
      load(src, t.first + (int)((int64_t)i * span / kSampleRows), x);
#pragma unroll
      for (int k = 0; k < E; ++k) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu);
    }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int w = 1; w < kPrepThreads / 32; ++w) m = max(m, red[w]);
  const int ebits = (int)(m >> 23);
  const int e = m == 0u || ebits == 255 ? 0 : max(ebits, 1) - 127 - 8;
  const Pow2Scale scale(-e);
  __syncthreads();

  __half* hi = t.hi + (int64_t)head * t.rows * DP;
  __half* lo = hi + (int64_t)t.heads * t.rows * DP;
  const bool is_do = a.o != nullptr && ti == a.tensors - 1;
  uint32_t top = 0;
  float top_norm = 0.0f;
  const int r_end = min((int)(blockIdx.x + 1) * kPrepRows, t.rows);
  for (int r = blockIdx.x * kPrepRows + warp; r < r_end; r += kPrepThreads / 32) {
    const bool real = r < end && (r >= t.first || r < t.sinks);
    float x[E];
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = 0.0f;
    if (real) load(src, r, x);
    float delta = 0.0f;
    if (is_do) {
      if (real) {
        float y[E];
        load(a.o + (int64_t)head * t.rows * dim, r, y);
#pragma unroll
        for (int k = 0; k < E; ++k) delta = fmaf(x[k], y[k], delta);
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) delta = __fadd_rn(delta, __shfl_xor_sync(0xffffffffu, delta, s));
      if (lane == 0) {
        a.delta_p[(int64_t)head * a.pitch + r] = delta;
        a.lse_p[(int64_t)head * a.pitch + r] = real ? a.lse[(int64_t)head * t.rows + r] : CUDART_INF_F;
      }
    }
    __half h[E], l[E];
    float norm = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float xs = scale(__fmul_rn(x[k], t.sign));
      top = max(top, __float_as_uint(xs) & 0x7fffffffu);
      norm = fmaf(xs, xs, norm);
      split_half(xs, h[k], l[k]);
    }
    if (E == 4) {
      reinterpret_cast<uint2*>(hi + (int64_t)r * DP)[lane] = *reinterpret_cast<uint2*>(h);
      reinterpret_cast<uint2*>(lo + (int64_t)r * DP)[lane] = *reinterpret_cast<uint2*>(l);
    } else {
      reinterpret_cast<uint32_t*>(hi + (int64_t)r * DP)[lane] = *reinterpret_cast<uint32_t*>(h);
      reinterpret_cast<uint32_t*>(lo + (int64_t)r * DP)[lane] = *reinterpret_cast<uint32_t*>(l);
    }
    if (t.norms) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) norm = __fadd_rn(norm, __shfl_xor_sync(0xffffffffu, norm, s));
      norm = sqrtf(norm);
      top_norm = fmaxf(top_norm, norm);
      if (lane == 0) t.norms[(int64_t)head * t.rows + r] = norm;
    }
  }
  if (is_do && (int)blockIdx.x == blocks - 1)                    // columns that exist in no head
    for (int r = t.rows + threadIdx.x; r < a.pitch; r += kPrepThreads) {
      a.delta_p[(int64_t)head * a.pitch + r] = 0.0f;
      a.lse_p[(int64_t)head * a.pitch + r] = CUDART_INF_F;
    }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) { red[warp] = top; redn[warp] = top_norm; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPrepThreads / 32; ++w) { top = max(top, red[w]); top_norm = fmaxf(top_norm, redn[w]); }
    const int64_t at = (int64_t)blockIdx.y * a.blocks;
    __stcg(a.block_max + at + blockIdx.x, top);
    __stcg(a.block_norm + at + blockIdx.x, top_norm);
    __threadfence();
    last_block = atomicAdd(a.counters + blockIdx.y, 1u) == (unsigned)blocks - 1;
  }
  __syncthreads();
  if (!last_block || warp != 0) return;
  __threadfence();
  top = 0;
  top_norm = 0.0f;
  for (int i = lane; i < blocks; i += 32) {
    top = max(top, __ldcg(a.block_max + (int64_t)blockIdx.y * a.blocks + i));
    top_norm = fmaxf(top_norm, __ldcg(a.block_norm + (int64_t)blockIdx.y * a.blocks + i));
  }
  top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top_norm = fmaxf(top_norm, __shfl_xor_sync(0xffffffffu, top_norm, s));
  if (lane == 0) {
    const float largest = __uint_as_float(top);
    a.info[blockIdx.y] = HeadInfo{e, top == 0u || (largest >= 4.0f && largest < 65000.0f), top_norm};
    a.counters[blockIdx.y] = 0;
  }
}

// ---- the passes ----------------------------------------------------------------------------------------
struct TcArgs {
  AttnArgs a;
  const float *lse_p, *delta_p;  // [q head][pitch]
  const float* norms;            // DQ: of dO's rows, DK: of V's
  int pitch;
  int works;
  // DV, DK: keys below sinks take `splits_sink` works per tile of rows, the others `splits`
  int tiles, sink_tiles, splits_sink, splits;
  float* parts;                  // [part][128][DP] of the tiles that have several works
};

template <int MODE, int DP> struct Shape {
  static constexpr bool TWO = MODE == DQ || MODE == DK, KEYS = MODE == DV || MODE == DK;
  static constexpr int BN = TWO && DP == 128 ? 64 : 128;
  static constexpr int SLABS = DP / 64;                          // 64 values (128 bytes) wide
  static constexpr uint32_t X_PART = kRowsM * DP * 2, X_BYTES = 2 * X_PART;
  static constexpr uint32_t Y_PART = BN * DP * 2, Y_BYTES = 2 * Y_PART;
  // ring depths: see the order of the MMAs
  static constexpr int NY = TWO ? 2 : (DP == 128 ? 1 : 2), NZ = TWO ? 1 : (DP == 128 ? 1 : 2);
  static constexpr int NS = TWO ? 2 : 3;                         // score buffers
  static constexpr uint32_t SMEM = (TWO ? 2 : 1) * X_BYTES + (NY + NZ) * Y_BYTES + 1024;
  // TMEM columns
  static constexpr uint32_t T_DP = NS * BN, T_OUT = T_DP + (TWO ? BN : 0);
  static_assert(T_OUT + DP <= 512, "TMEM");
};

// Tiles with one work only write their results themselves: their places are behind the others' and are not there where
// only the tiles with sinks are cut.
__device__ __forceinline__ int64_t parts_per_head(const TcArgs& t) {
  return (int64_t)t.sink_tiles * t.splits_sink + (t.splits > 1 ? (int64_t)(t.tiles - t.sink_tiles) * t.splits : 0);
}

// a tile of 128 stationary rows and the steps of its stream
template <int MODE, int DP>
struct Work {
  int b, hk, h, row0, steps, first;      // h: the query head of a pass over queries
  int len, p_hi, lowest, sink_n, sink_steps;         // queries: positions
  int i_lo, nq, q_hi;                    // keys: first query, tiles of queries per head, position of the last query
  int tile, split, splits;
  int64_t part;                          // its place among the parts
  __device__ __forceinline__ Work(const TcArgs& t, int w) {
    using S = Shape<MODE, DP>;
    const AttnArgs& a = t.a;
    const int past = a.kv_len - a.q_len, group = a.q_heads / a.kv_heads;
    first = 0;
    if (!S::KEYS) {
      tile = w % t.tiles;
      const int head = w / t.tiles;
      b = head / a.q_heads; h = head % a.q_heads; hk = h / group;
      split = 0; splits = 1;
      len = lnn::attn_length(a.lengths, b, a.kv_len, a.status);
      row0 = tile * kRowsM;
      p_hi = min(min(row0 + kRowsM, a.q_len) - 1 + past, len - 1);
      steps = 0;
      if (p_hi >= row0 + past) {
        lowest = max(row0 + past - a.window + 1, 0);
        sink_n = min(a.sinks, lowest);
        sink_steps = (sink_n + S::BN - 1) / S::BN;
        steps = sink_steps + (p_hi - lowest) / S::BN + 1;
      }
    } else {
      const int per = t.sink_tiles * t.splits_sink + (t.tiles - t.sink_tiles) * t.splits;
      int r = w % per;
      const int head = w / per;
      b = head / a.kv_heads; hk = head % a.kv_heads; h = hk * group;
      part = (int64_t)head * parts_per_head(t) + r;
      if (r < t.sink_tiles * t.splits_sink) {
        tile = r / t.splits_sink; split = r % t.splits_sink; splits = t.splits_sink;
      } else {
        r -= t.sink_tiles * t.splits_sink;
        tile = t.sink_tiles + r / t.splits; split = r % t.splits; splits = t.splits;
      }
      len = lnn::attn_length(a.lengths, b, a.kv_len, a.status);
      row0 = tile * kRowsM;
      const lnn::QuerySpan span(row0, min(row0 + kRowsM, a.kv_len) - 1, a.window, a.sinks, past, len);
      steps = 0;
      if (span.hi >= span.lo) {
        q_hi = span.hi;
        i_lo = (span.lo - past) & ~7;                        // (the denominators are read in vectors)
        nq = (span.hi - past - i_lo) / S::BN + 1;
        const int all = nq * group;
        first = (int)((int64_t)all * split / splits);
        steps = (int)((int64_t)all * (split + 1) / splits) - first;
      }
    }
  }
  // step s: stream rows [r, r + n) of head `head` (of the stream's operands)
  __device__ __forceinline__ void step(const TcArgs& t, int s, int& head, int& r, int& n) const {
    using S = Shape<MODE, DP>;
    if (!S::KEYS) {
      head = b * t.a.kv_heads + hk;
      if (s < sink_steps) { r = s * S::BN; n = min(S::BN, sink_n - r); }
      else { r = lowest + (s - sink_steps) * S::BN; n = min(S::BN, p_hi + 1 - r); }
    } else {
      const int at = first + s, hq = at / nq;
      head = b * t.a.q_heads + h + hq;
      r = i_lo + (at - hq * nq) * S::BN;
      n = min(S::BN, q_hi - (t.a.kv_len - t.a.q_len) + 1 - r);
    }
  }
};

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum)
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
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A whole warp's wait: all lanes go on or all give up (what follows is done by whole warps).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int role, int step) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, role, step));
}

// 32 weights as fp16, two to a column: 16 columns of hi, 16 of lo
__device__ __forceinline__ void store_split(uint32_t at, const float* w) {
  uint32_t hi[16], lo[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const __half2 h = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(__fsub_rn(w[2 * i], f.x), __fsub_rn(w[2 * i + 1], f.y));
    hi[i] = *reinterpret_cast<const uint32_t*>(&h);
    lo[i] = *reinterpret_cast<const uint32_t*>(&l);
  }
  tmem_st16(at, hi);
  tmem_st16(at + 16, lo);
}

__device__ __forceinline__ uint32_t idesc_f16(int n, int b_major) {
  return (1u << 4) | ((uint32_t)b_major << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

template <int MODE, int DP>
__global__ void __launch_bounds__(kAttnThreads, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapX2,
               const __grid_constant__ CUtensorMap mapY, const __grid_constant__ CUtensorMap mapZ,
               const __grid_constant__ TcArgs t) {
  using S = Shape<MODE, DP>;
  constexpr int BN = S::BN, NY = S::NY, NZ = S::NZ, NS = S::NS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_x_full, bar_x_empty, bar_y_full[NY], bar_y_empty[NY], bar_z_full[NZ], bar_z_empty[NZ];
  __shared__ uint64_t bar_s_full[NS], bar_p_full[NS], bar_o_full, bar_o_empty, bar_pair[4];
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag_smem;
  __shared__ float exchange[3][kComputeWarps][32];

  // an earlier kernel gave up: leave as a whole CTA (the decision must be uniform)
  if (threadIdx.x == 0) abort_flag_smem = (*(volatile int*)t.a.status == LNN_E_TIMEOUT) ? 2 : 0;
  __syncthreads();
  if (abort_flag_smem == 2) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_flag_smem;
  int* status = t.a.status;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sX = base, sX2 = sX + S::X_BYTES, sY = sX2 + (S::TWO ? S::X_BYTES : 0u), sZ = sY + NY * S::Y_BYTES;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar_x_full), 1);
    mbar_init(smem_u32(&bar_x_empty), 1);
    for (int i = 0; i < NY; ++i) { mbar_init(smem_u32(&bar_y_full[i]), 1); mbar_init(smem_u32(&bar_y_empty[i]), 1); }
    for (int i = 0; i < NZ; ++i) { mbar_init(smem_u32(&bar_z_full[i]), 1); mbar_init(smem_u32(&bar_z_empty[i]), 1); }
    for (int i = 0; i < NS; ++i) { mbar_init(smem_u32(&bar_s_full[i]), 1); mbar_init(smem_u32(&bar_p_full[i]), kComputeWarps); }
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&bar_pair[i]), 2);
    mbar_init(smem_u32(&bar_o_full), 1);
    mbar_init(smem_u32(&bar_o_empty), kComputeWarps);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base_smem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_smem;

  if (warp == 0) {
    // ---- loads ------------------------------------------------------------------------------------
    if (lane == 0) {
      const int x_part = (S::KEYS ? t.a.batch * t.a.kv_heads : t.a.batch * t.a.q_heads);     // heads in front of lo
      const int y_part = (S::KEYS ? t.a.batch * t.a.q_heads : t.a.batch * t.a.kv_heads);
      const auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int part_bytes, int slab_bytes, int head,
                            int parts, int row, int boxes) {
        for (int p = 0; p < 2; ++p)
          for (int s = 0; s < S::SLABS; ++s)
            for (int i = 0; i < boxes; ++i)
              tma_load_3d(dst + p * part_bytes + s * slab_bytes + i * (kBoxRows * 128), map, bar, s * 64, row + i * kBoxRows,
                          head + p * parts);
      };
      bool ok = true;
      int g = 0, nw = 0;
      // what goes with a step's weights in FWD and DV is loaded one step behind the rows of its scores: the order of use
      struct Pending { int head, r, boxes, g; bool any; } late = {0, 0, 0, 0, false};
      const auto load_z = [&](const Pending& z) {
        const int slot = z.g % NZ;
        if (!mbar_wait(smem_u32(&bar_z_empty[slot]), ((z.g / NZ) & 1) ^ 1, abort_flag, status, 10, z.g)) return false;
        const uint32_t bar = smem_u32(&bar_z_full[slot]);
        mbar_expect_tx(bar, (uint32_t)(2 * S::SLABS * z.boxes * kBoxRows * 128));
        load(&mapZ, sZ + slot * S::Y_BYTES, bar, S::Y_PART, BN * 128, z.head, y_part, z.r, z.boxes);
        return true;
      };
      for (int w = blockIdx.x; ok && w < t.works; w += gridDim.x) {
        const Work<MODE, DP> k(t, w);
        if (k.steps == 0 || !lnn::group_ok(t.a, k.b, k.hk)) continue;
        if (!mbar_wait(smem_u32(&bar_x_empty), (nw & 1) ^ 1, abort_flag, status, 11, w)) { ok = false; break; }
        const int xh = S::KEYS ? k.b * t.a.kv_heads + k.hk : k.b * t.a.q_heads + k.h;
        const uint32_t bx = smem_u32(&bar_x_full);
        mbar_expect_tx(bx, (S::TWO ? 2u : 1u) * S::X_BYTES);
        load(&mapX, sX, bx, S::X_PART, kRowsM * 128, xh, x_part, k.row0, kRowsM / kBoxRows);
        if (S::TWO) load(&mapX2, sX2, bx, S::X_PART, kRowsM * 128, xh, x_part, k.row0, kRowsM / kBoxRows);
        for (int s = 0; s < k.steps; ++s, ++g) {
          Pending z;
          int n;
          k.step(t, s, z.head, z.r, n);
          z.boxes = (n + kBoxRows - 1) / kBoxRows;
          z.g = g;
          z.any = true;
          const int slot = g % NY;
          if (!mbar_wait(smem_u32(&bar_y_empty[slot]), ((g / NY) & 1) ^ 1, abort_flag, status, 12, g)) { ok = false; break; }
          const uint32_t bar = smem_u32(&bar_y_full[slot]);
          mbar_expect_tx(bar, (uint32_t)(2 * S::SLABS * z.boxes * kBoxRows * 128));
          load(&mapY, sY + slot * S::Y_BYTES, bar, S::Y_PART, BN * 128, z.head, y_part, z.r, z.boxes);
          if (S::TWO) {
            if (!load_z(z)) { ok = false; break; }
          } else {
            if (late.any && !load_z(late)) { ok = false; break; }
            late = z;
          }
        }
        ++nw;
      }
      if (ok && !S::TWO && late.any) load_z(late);
    }
  } else if (warp == 1) {
    // ---- MMAs -------------------------------------------------------------------------------------
    if (lane == 0) {
      // K-major tiles of 128-byte rows (128-byte swizzle); the same bytes are an MN-major operand when the rows are K:
      // 64 values of MN to a row, slabs of 64 BN rows apart
      const uint64_t dk0 = make_smem_desc(0u, 16u, 1024u, 2u);
      const uint64_t dm0 = make_smem_desc(0u, BN * 128u, 1024u, 2u);
      const auto scores = [&](uint32_t d, uint32_t ax, uint32_t by, int n16) {
        const uint32_t id = idesc_f16(n16, 0);
        uint32_t accum = 0;
#pragma unroll
        for (int pr = 0; pr < 3; ++pr) {                          // lo hi, hi lo, hi hi
          const uint64_t a0 = dk0 + ((ax + (pr == 0 ? S::X_PART : 0u)) >> 4), b0 = dk0 + ((by + (pr == 1 ? S::Y_PART : 0u)) >> 4);
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks) {
            umma_f16(d, a0 + (ks / 4) * (kRowsM * 128 / 16) + (ks % 4) * 2, b0 + (ks / 4) * (BN * 128 / 16) + (ks % 4) * 2, id, accum);
            accum = 1;
          }
        }
      };
      const auto weighted = [&](uint32_t d, uint32_t p, uint32_t bz, int n16) {
        const uint32_t id = idesc_f16(DP, 1);
        uint32_t accum = 0;
        for (int pr = 0; pr < 3; ++pr) {
          const uint64_t b0 = dm0 + ((bz + (pr == 1 ? S::Y_PART : 0u)) >> 4);
          const uint32_t a0 = p + (pr == 0 ? 16 : 0);             // 32 scores became 16 columns of hi and 16 of lo
          for (int ks = 0; ks < n16 / 16; ++ks) {
            umma_f16_ts(d, a0 + (ks / 2) * 32 + (ks % 2) * 8, b0 + ks * (16 * 128 / 16), id, accum);
            accum = 1;
          }
        }
      };
      bool ok = true;
      int g = 0, nw = 0;
      struct Pending { int g, n16; bool any; } late = {0, 0, false};
      const auto out = [&](const Pending& q) {
        if (!mbar_wait(smem_u32(&bar_p_full[q.g % NS]), (q.g / NS) & 1, abort_flag, status, 20, q.g)) return false;
        if (!mbar_wait(smem_u32(&bar_o_empty), (q.g & 1) ^ 1, abort_flag, status, 21, q.g)) return false;
        uint32_t bz = sY + (q.g % NY) * S::Y_BYTES;
        if (!S::TWO) {
          if (!mbar_wait(smem_u32(&bar_z_full[q.g % NZ]), (q.g / NZ) & 1, abort_flag, status, 22, q.g)) return false;
          bz = sZ + (q.g % NZ) * S::Y_BYTES;
        }
        tc_fence_after();
        weighted(tmem + S::T_OUT, tmem + (q.g % NS) * BN, bz, q.n16);
        umma_commit(smem_u32(&bar_o_full));
        umma_commit(S::TWO ? smem_u32(&bar_y_empty[q.g % NY]) : smem_u32(&bar_z_empty[q.g % NZ]));
        return true;
      };
      for (int w = blockIdx.x; ok && w < t.works; w += gridDim.x) {
        const Work<MODE, DP> k(t, w);
        if (k.steps == 0 || !lnn::group_ok(t.a, k.b, k.hk)) continue;
        if (!mbar_wait(smem_u32(&bar_x_full), nw & 1, abort_flag, status, 23, w)) { ok = false; break; }
        for (int s = 0; s < k.steps; ++s, ++g) {
          int head, r, n;
          k.step(t, s, head, r, n);
          const int n16 = (n + 15) & ~15;
          if (!mbar_wait(smem_u32(&bar_y_full[g % NY]), (g / NY) & 1, abort_flag, status, 24, g)) { ok = false; break; }
          // The scores of step g - NS were in this buffer, and its weights behind them.  FWD, DV: OUT(g - 2) waited for
          // the drain of OUT(g - 3).  DQ, DK: OUT(g - 2) has to be over, in front of dP(g - 1) in the stream.
          if (S::TWO && g >= 2 && !mbar_wait(smem_u32(&bar_o_full), g & 1, abort_flag, status, 25, g)) { ok = false; break; }
          tc_fence_after();
          scores(tmem + (g % NS) * BN, sX, sY + (g % NY) * S::Y_BYTES, n16);
          if (!S::TWO) {
            umma_commit(smem_u32(&bar_s_full[g % NS]));
            umma_commit(smem_u32(&bar_y_empty[g % NY]));
            if (s == k.steps - 1) umma_commit(smem_u32(&bar_x_empty));
          }
          if (late.any && !out(late)) { ok = false; break; }
          late = {g, n16, true};
          if (S::TWO) {
            // (its buffer: the weights of step g - 1 are complete, OUT(g - 1) waited for them)
            if (!mbar_wait(smem_u32(&bar_z_full[g % NZ]), (g / NZ) & 1, abort_flag, status, 26, g)) { ok = false; break; }
            tc_fence_after();
            scores(tmem + S::T_DP, sX2, sZ + (g % NZ) * S::Y_BYTES, n16);
            umma_commit(smem_u32(&bar_s_full[g % NS]));
            umma_commit(smem_u32(&bar_z_empty[g % NZ]));
            if (s == k.steps - 1) umma_commit(smem_u32(&bar_x_empty));
          }
        }
        ++nw;
      }
      if (ok && late.any) out(late);
    }
  } else {
    // ---- weights and sums -------------------------------------------------------------------------
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    constexpr int COLS = BN / 2, CHUNKS = COLS / 32, OUT = DP / 2;
    const AttnArgs& a = t.a;
    const int past = a.kv_len - a.q_len, row_in = quarter * 32 + lane;
    bool ok = true;
    int g = 0;
    // the two warps of a quarter hold halves of the same rows: one value of each row to the other warp and back (a bounded
    // wait, like all others: a warp that gives up must not leave its partner behind)
    uint32_t pairs = 0;
    const auto swapped = [&](float* buffer, float mine, float& other) {
      buffer[(quarter + 4 * half) * 32 + lane] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_pair[quarter]));
      if (!warp_wait(smem_u32(&bar_pair[quarter]), pairs & 1u, abort_flag, status, 32, g)) return false;
      ++pairs;
      other = buffer[(quarter + 4 * (half ^ 1)) * 32 + lane];
      return true;
    };
    for (int w = blockIdx.x; ok && w < t.works; w += gridDim.x) {
      const Work<MODE, DP> k(t, w);
      if (!lnn::group_ok(a, k.b, k.hk)) continue;
      const int row = k.row0 + row_in;
      const int xh = S::KEYS ? k.b * a.kv_heads + k.hk : k.b * a.q_heads + k.h;
      const int kvh = k.b * a.kv_heads + k.hk;
      float acc[OUT];
#pragma unroll
      for (int i = 0; i < OUT; ++i) acc[i] = 0.0f;
      float m = -CUDART_INF_F, l = 0.0f, keep_before = 1.0f;      // FWD
      float row_lse = CUDART_INF_F, row_delta = 0.0f;              // DQ
      int row_exp = 0;                                             // DQ, DK: dS is scaled by 2^row_exp
      const int ek = lnn::info_of(a, 1, kvh).e, ev = lnn::info_of(a, 2, kvh).e;
      const int rows = S::KEYS ? a.kv_len : a.q_len;
      float norm = 0.0f, other_norm = 0.0f;
      if (S::TWO && row < rows) norm = __ldg(t.norms + (int64_t)xh * rows + row);
      if (MODE == DQ) {
        if (row < rows) {
          row_lse = __ldg(t.lse_p + (int64_t)xh * t.pitch + row);
          row_delta = __ldg(t.delta_p + (int64_t)xh * t.pitch + row);
        }
        other_norm = lnn::info_of(a, 2, kvh).norm;
      }
      int cur_head = -1;
      float c = 0.0f, cdp = 0.0f, factor = 1.0f, factor_before = 1.0f;
      const auto drain = [&](int gd, float old_times, float tile_times) {
        if (!warp_wait(smem_u32(&bar_o_full), gd & 1, abort_flag, status, 30, gd)) return false;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < OUT / 32; ++q) {
          uint32_t v[32];
          tmem_ld32(tmem + lanes + S::T_OUT + half * OUT + q * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (MODE == FWD) acc[q * 32 + i] = fmaf(acc[q * 32 + i], old_times, __uint_as_float(v[i]));
            else acc[q * 32 + i] = fmaf(__uint_as_float(v[i]), tile_times, acc[q * 32 + i]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_o_empty));
        return true;
      };
      for (int s = 0; s < k.steps; ++s, ++g) {
        int head, r0, n;
        k.step(t, s, head, r0, n);
        const int qh = S::KEYS ? head : xh;
        if (qh != cur_head) {                                      // the scales that go with a query head
          cur_head = qh;
          const int eq = lnn::info_of(a, 0, qh).e;
          // (2^-126 in place of 0: masked scores stay -inf)
          c = fmaxf(__fmul_rn(__fmul_rn(fabsf(a.scale), lnn::kLog2e), pow2f_int(eq + ek)), 1.17549435e-38f);
          if (MODE == DV) factor = pow2f_int(lnn::info_of(a, 3, qh).e - 14);
          if (S::TWO) {
            const int eo = lnn::info_of(a, 3, qh).e;
            cdp = pow2f_int(eo + ev);
            if (MODE == DK) other_norm = lnn::info_of(a, 3, qh).norm;
            // |dP - delta| <= 2 |dO| |V|: below 2^15 after scaling
            const float bound = fmaxf(2.0f * norm * other_norm, 0.0009765625f);
            row_exp = 14 - ((int)(__float_as_uint(bound) >> 23) - 127) - (eo + ev);
            if (MODE == DK) factor = pow2f_int(eq - row_exp);
          }
        }
        // which columns of the tile this row sees: [lo, hi], or up to `always`
        int lo, hi, always;
        bool all;
        if (!S::KEYS) {
          const int p = row + past;
          lo = p - a.window + 1 - r0; hi = min(p - r0, n - 1); always = a.sinks - r0;
          all = n == BN && r0 + BN - 1 <= k.row0 + past &&
                (k.p_hi - r0 < a.window || r0 + BN <= a.sinks);
        } else {
          const int last = row < a.sinks ? k.q_hi : (int)min((int64_t)row + a.window - 1, (int64_t)k.q_hi);
          lo = row - past - r0; hi = min(last - past - r0, n - 1); always = 0;
          all = n == BN && r0 + past >= k.row0 + kRowsM - 1 &&
                (r0 + past + BN - 1 < k.row0 + a.window || k.row0 + kRowsM <= a.sinks);
        }
        const int buf = g % NS;
        const uint32_t ts = tmem + lanes + buf * BN + half * COLS;
        const int col0 = half * COLS;
        if (!warp_wait(smem_u32(&bar_s_full[buf]), (g / NS) & 1, abort_flag, status, 31, g)) { ok = false; break; }
        tc_fence_after();
        if (MODE == FWD) {
          uint32_t v[COLS];
          float sc[COLS];
          float top = -CUDART_INF_F;
          if (col0 < n) {
#pragma unroll
            for (int q = 0; q < CHUNKS; ++q) tmem_ld32(ts + q * 32, v + q * 32);
            tmem_ld_wait();
            if (all) {
#pragma unroll
              for (int i = 0; i < COLS; ++i) { sc[i] = __uint_as_float(v[i]); top = fmaxf(top, sc[i]); }
            } else {
#pragma unroll
              for (int i = 0; i < COLS; ++i) {
                const int col = col0 + i;
                sc[i] = col <= hi && (col >= lo || col < always) ? __uint_as_float(v[i]) : -CUDART_INF_F;
                top = fmaxf(top, sc[i]);
              }
            }
          }
          float other;
          if (!swapped(&exchange[g & 1][0][0], top, other)) { ok = false; break; }
          top = fmaxf(top, other);
          const float now = fmaxf(m, __fmul_rn(top, c));
          const float at = now == -CUDART_INF_F ? 0.0f : now;
          const float keep = exp2_fast(__fsub_rn(m, at));
          const float shift = 14.0f - at;
          float sum = 0.0f;
          if (col0 < n) {
#pragma unroll
            for (int q = 0; q < CHUNKS; ++q) {
              float part = 0.0f;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                sc[q * 32 + i] = exp2_fast(fmaf(sc[q * 32 + i], c, shift));
                part = __fadd_rn(part, sc[q * 32 + i]);
              }
              sum = __fadd_rn(sum, part);
              store_split(ts + q * 32, sc + q * 32);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_p_full[buf]));
          l = fmaf(l, keep, sum);
          m = now;
          if (s > 0 && !drain(g - 1, keep_before, 1.0f)) { ok = false; break; }
          keep_before = keep;
        } else {
          if (col0 < n) {
#pragma unroll
            for (int q = 0; q < CHUNKS; ++q) {
              uint32_t v[32], d[32];
              float wt[32];
              tmem_ld32(ts + q * 32, v);
              if (S::TWO) tmem_ld32(tmem + lanes + S::T_DP + col0 + q * 32, d);
              const float* cl = t.lse_p + (int64_t)qh * t.pitch + r0 + col0 + q * 32;
              const float* cd = t.delta_p + (int64_t)qh * t.pitch + r0 + col0 + q * 32;
              tmem_ld_wait();
#pragma unroll
              for (int i0 = 0; i0 < 32; i0 += 4) {
                float4 l4 = make_float4(row_lse, row_lse, row_lse, row_lse), d4 = make_float4(row_delta, row_delta, row_delta, row_delta);
                if (S::KEYS) {
                  l4 = __ldg(reinterpret_cast<const float4*>(cl + i0));
                  if (S::TWO) d4 = __ldg(reinterpret_cast<const float4*>(cd + i0));
                }
                const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, ds[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  const int i = i0 + u, col = col0 + q * 32 + i;
                  const float up = (S::TWO ? (float)row_exp : 14.0f) - ls[u];
                  float x = exp2_fast(fmaf(__uint_as_float(v[i]), c, up));
                  if (S::TWO) x = __fmul_rn(x, fmaf(__uint_as_float(d[i]), cdp, -ds[u]));
                  wt[i] = all || (col <= hi && (col >= lo || col < always)) ? x : 0.0f;
                }
              }
              store_split(ts + q * 32, wt);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_p_full[buf]));
          if (s > 0 && !drain(g - 1, 1.0f, factor_before)) { ok = false; break; }
          factor_before = factor;
        }
      }
      if (!ok) break;
      if (k.steps > 0 && !drain(g - 1, keep_before, factor_before)) { ok = false; break; }

      // ---- results ----
      float* dst;
      int accumulate = 0, limit = rows;
      float times = 1.0f;
      int64_t at = ((int64_t)xh * rows + row) * a.dim;
      int pitch_cols = a.dim;
      if (MODE == FWD) {
        if (k.steps > 0) {
          float other;
          if (!swapped(&exchange[2][0][0], l, other)) { ok = false; break; }
          l = __fadd_rn(l, other);
        }
        const bool empty = k.steps == 0 || row + past > k.p_hi;
        times = empty ? 0.0f : __fmul_rn(__fdiv_rn(1.0f, l), pow2f_int(ev));
        if (half == 0 && row < rows)
          a.lse[(int64_t)xh * rows + row] = empty ? CUDART_INF_F : __fadd_rn(m, __fsub_rn(log2f(l), 14.0f));
        if (empty) {
#pragma unroll
          for (int i = 0; i < OUT; ++i) acc[i] = 0.0f;
        }
        dst = a.o;
      } else if (MODE == DQ) {
        times = __fmul_rn(a.scale, pow2f_int(ek - row_exp));
        dst = a.dq; accumulate = a.acc_q;
      } else {
        if (MODE == DK) times = fabsf(a.scale);
        dst = MODE == DK ? a.dk : a.dv;
        accumulate = MODE == DK ? a.acc_k : a.acc_v;
        if (k.splits > 1) {
          dst = t.parts; accumulate = 0; limit = k.row0 + kRowsM;
          at = (k.part * kRowsM + row_in) * DP;
          pitch_cols = DP;
        }
      }
      if (row < limit) {
        float* to = dst + at;
        const bool vec = pitch_cols % 4 == 0 && (((uintptr_t)dst) & 15) == 0;
#pragma unroll
        for (int i = 0; i < OUT; i += 4) {
          const int col = half * OUT + i;
          if (vec) {
            if (col < pitch_cols) {
              float4 x = make_float4(__fmul_rn(acc[i], times), __fmul_rn(acc[i + 1], times), __fmul_rn(acc[i + 2], times),
                                     __fmul_rn(acc[i + 3], times));
              if (accumulate) {
                const float4 y = *reinterpret_cast<const float4*>(to + col);
                x = make_float4(__fadd_rn(y.x, x.x), __fadd_rn(y.y, x.y), __fadd_rn(y.z, x.z), __fadd_rn(y.w, x.w));
              }
              *reinterpret_cast<float4*>(to + col) = x;
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (col + u < pitch_cols) {
                const float x = __fmul_rn(acc[i + u], times);
                to[col + u] = accumulate ? __fadd_rn(to[col + u], x) : x;
              }
          }
        }
      }
    }
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
}

// dK or dV of the tiles that several works shared: their parts in order.
template <int DP>
__global__ void __launch_bounds__(256)
attn_parts_kernel(float* __restrict__ dst, const float* __restrict__ parts, const TcArgs t, int accumulate) {
  const AttnArgs& a = t.a;
  const int tile = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int splits = tile < t.sink_tiles ? t.splits_sink : t.splits;
  if (splits == 1 || !lnn::group_ok(a, b, hk)) return;
  const int64_t w0 = (int64_t)(b * a.kv_heads + hk) * parts_per_head(t) +
                     (tile < t.sink_tiles ? tile * t.splits_sink : t.sink_tiles * t.splits_sink + (tile - t.sink_tiles) * t.splits);
  for (int i = threadIdx.x; i < kRowsM * DP / 4; i += 256) {
    const int row = tile * kRowsM + i / (DP / 4), col = i % (DP / 4) * 4;
    if (row >= a.kv_len || col >= a.dim) continue;
    float4 s = __ldg(reinterpret_cast<const float4*>(parts + w0 * kRowsM * DP) + i);
    for (int k = 1; k < splits; ++k) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(parts + (w0 + k) * kRowsM * DP) + i);
      s = make_float4(__fadd_rn(s.x, x.x), __fadd_rn(s.y, x.y), __fadd_rn(s.z, x.z), __fadd_rn(s.w, x.w));
    }
    float* to = dst + ((int64_t)(b * a.kv_heads + hk) * a.kv_len + row) * a.dim + col;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (col + u < a.dim) to[u] = accumulate ? __fadd_rn(to[u], v[u]) : v[u];
  }
}

// ---- host ------------------------------------------------------------------------------------------------
// [2 heads][rows][DP] fp16: lo behind hi
int operand_map(CUtensorMap* tm, const void* base, int dp, int rows, int64_t heads) {
  const uint64_t dims[3] = {(uint64_t)dp, (uint64_t)rows, (uint64_t)(2 * heads)};
  const uint64_t strides[2] = {(uint64_t)dp * 2, (uint64_t)rows * dp * 2};
  const uint32_t box[3] = {64, kBoxRows, 1}, es[3] = {1, 1, 1};
  return lnn_tc::encode_half_map(tm, base, 3, dims, strides, box, es);
}

template <int MODE, int DP>
int launch_pass(lnn::Device* d, const CUtensorMap* x, const CUtensorMap* x2, const CUtensorMap* y, const CUtensorMap* z, const TcArgs& t) {
  using S = Shape<MODE, DP>;
  static_assert(S::SMEM + 2048 <= 227 * 1024, "shared memory");
  LNN_CUDA(cudaFuncSetAttribute(attn_tc_kernel<MODE, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
  attn_tc_kernel<MODE, DP><<<std::min(t.works, d->sm_count), kAttnThreads, S::SMEM, d->stream>>>(*x, *x2, *y, *z, t);
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

// Works of a pass over keys: a tile's steps are cut so that there are about three works per SM and none is longer than that.
template <int MODE, int DP>
void plan_keys(const lnn::Device* d, TcArgs& t) {
  constexpr int BN = Shape<MODE, DP>::BN;
  const AttnArgs& a = t.a;
  const int64_t group = a.q_heads / a.kv_heads, heads = (int64_t)a.batch * a.kv_heads;
  t.tiles = (a.kv_len + kRowsM - 1) / kRowsM;
  t.sink_tiles = std::min(t.tiles, (a.sinks + kRowsM - 1) / kRowsM);
  const int64_t most = group * ((a.q_len + BN - 1) / BN + 1);
  const int64_t some = std::min<int64_t>(most, group * ((std::min<int64_t>((int64_t)a.window + kRowsM, a.q_len) + BN - 1) / BN + 1));
  const int64_t total = heads * (t.sink_tiles * most + (t.tiles - t.sink_tiles) * some);
  const int64_t length = std::max<int64_t>(6, total / (d->sm_count * 3));
  t.splits_sink = (int)std::min<int64_t>(64, (most + length - 1) / length);
  t.splits = (int)std::min<int64_t>(64, (some + length - 1) / length);
  t.works = (int)(heads * (t.sink_tiles * t.splits_sink + (t.tiles - t.sink_tiles) * t.splits));
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
  const int64_t sq = nq * a.q_len * DP, sk = nk * a.kv_len * DP;
  int rc = op.halves.get((uint64_t)(2 * (sq + 2 * sk + (backward ? sq : 0))) * 2);
  if (rc) return rc;
  __half* h = op.halves.as<__half>();
  __half* at[4] = {h, h + 2 * sq, h + 2 * sq + 2 * sk, h + 2 * sq + 4 * sk};
  p.tensors = backward ? 4 : 3;
  p.dim = a.dim; p.batch = a.batch; p.lengths = a.lengths; p.kv_len = a.kv_len; p.status = a.status;
  p.blocks = (a.kv_len + kPrepRows - 1) / kPrepRows;
  p.pitch = (a.q_len + 7) / 8 * 8 + kRowsM;
  const int64_t heads = 2 * nk + (backward ? 2 : 1) * nq;
  const int64_t norm_words = backward ? nk * a.kv_len + nq * a.q_len : 0, col_words = backward ? 2 * nq * p.pitch : 0;
  const int64_t info_words = (heads * (int64_t)sizeof(HeadInfo) / 4 + 3) / 4 * 4;
  rc = op.small.get((uint64_t)(info_words + (col_words + 3) / 4 * 4 + 2 * heads * p.blocks + norm_words) * 4);
  if (rc) return rc;
  float* s = op.small.as<float>();
  p.info = (HeadInfo*)s; s += info_words;
  p.lse_p = s; p.delta_p = s + col_words / 2; s += (col_words + 3) / 4 * 4;       // (16-byte aligned: the pitch is a multiple of 8)
  p.block_max = (uint32_t*)s; s += heads * p.blocks;
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
    rc = operand_map(&op.map[i], at[i], DP, p.t[i].rows, p.t[i].heads);
    if (rc) return rc;
  }
  attn_prep_kernel<DP><<<dim3((unsigned)p.blocks, (unsigned)heads), kPrepThreads, 0, d->stream>>>(p);
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

template <int DP>
int tc_fwd(lnn::Device* d, AttnArgs a) {
  Operands op(d);
  int rc = prepare<DP>(d, a, op, false);
  if (rc) return rc;
  TcArgs t = {};
  t.a = a;
  t.tiles = (a.q_len + kRowsM - 1) / kRowsM;
  t.works = a.batch * a.q_heads * t.tiles;
  rc = launch_pass<FWD, DP>(d, &op.map[0], &op.map[0], &op.map[1], &op.map[2], t);
  return rc ? rc : lnn::attn_simt_fwd(d, a);                     // the heads that were marked
}

template <int MODE, int DP>
int keys_pass(lnn::Device* d, TcArgs t, Operands& op, float* dst, int accumulate) {
  plan_keys<MODE, DP>(d, t);
  lnn::Scratch parts(d);
  const bool cut = t.splits > 1 || t.splits_sink > 1;
  if (cut) {
    const int64_t n = (int64_t)t.a.batch * t.a.kv_heads *
                      ((int64_t)t.sink_tiles * t.splits_sink + (t.splits > 1 ? (int64_t)(t.tiles - t.sink_tiles) * t.splits : 0));
    int rc = n ? parts.get((uint64_t)n * kRowsM * DP * 4) : LNN_OK;
    if (rc) return rc;
    t.parts = parts.as<float>();
  }
  int rc = launch_pass<MODE, DP>(d, &op.map[1], &op.map[2], &op.map[0], &op.map[3], t);
  if (rc || !cut) return rc;
  attn_parts_kernel<DP><<<dim3((unsigned)t.tiles, (unsigned)t.a.kv_heads, (unsigned)t.a.batch), 256, 0, d->stream>>>(
      dst, t.parts, t, accumulate);
  LNN_CHECK_LAUNCH(d);
  return LNN_OK;
}

template <int DP>
int tc_bwd(lnn::Device* d, AttnArgs a) {
  Operands op(d);
  int rc = prepare<DP>(d, a, op, true);
  if (rc) return rc;
  TcArgs t = {};
  t.a = a;
  t.lse_p = op.p.lse_p; t.delta_p = op.p.delta_p; t.pitch = op.p.pitch;
  if (a.dq) {
    TcArgs q = t;
    q.norms = op.p.t[3].norms;
    q.tiles = (a.q_len + kRowsM - 1) / kRowsM;
    q.works = a.batch * a.q_heads * q.tiles;
    rc = launch_pass<DQ, DP>(d, &op.map[0], &op.map[3], &op.map[1], &op.map[2], q);
    if (rc) return rc;
  }
  if (a.dv) {
    rc = keys_pass<DV, DP>(d, t, op, a.dv, a.acc_v);
    if (rc) return rc;
  }
  if (a.dk) {
    t.norms = op.p.t[2].norms;
    rc = keys_pass<DK, DP>(d, t, op, a.dk, a.acc_k);
    if (rc) return rc;
  }
  a.delta = op.p.delta_p;
  a.delta_pitch = op.p.pitch;
  return lnn::attn_simt_bwd(d, a);
}

}  // namespace

namespace lnn {

bool attn_tc_applicable(const AttnArgs& a) {
  const int64_t heads = 2ll * a.batch * (a.q_heads + a.kv_heads);
  return a.dim <= 128 && heads <= kTileCounters && heads < 65536;
}
int attn_tc_fwd(Device* d, const AttnArgs& a) { return a.dim <= 64 ? tc_fwd<64>(d, a) : tc_fwd<128>(d, a); }
int attn_tc_bwd(Device* d, const AttnArgs& a) { return a.dim <= 64 ? tc_bwd<64>(d, a) : tc_bwd<128>(d, a); }

}  // namespace lnn
