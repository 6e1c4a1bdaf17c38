// Causal attention with a sliding window and a few first tokens ("sinks") that stay visible: what its translation
// units share.
//
// Query i of q_len sits at position p = i + kv_len - q_len of its sequence, and sees key j when
//   p < length,  j <= p  and  (p - j < window  or  j < sinks).
// Rows that see nothing (padding behind a sequence's length) give zeros and receive and pass on no gradient.
#pragma once
#include <float.h>
#include <math_constants.h>
#include "lnn_common.cuh"

namespace lnn {

// What is known about a head after its split into fp16 hi and lo.
struct HeadInfo {
  int e;                         // x 2^-e was split
  int ok;                        // finite, and inside fp16's range with that scale
  float norm;                    // the largest norm of a row, scaled
};

struct AttnArgs {
  const float *q, *k, *v;        // [batch][q_heads][q_len][dim], [batch][kv_heads][kv_len][dim]
  const float* lengths;          // [batch] whole numbers, or null: kv_len everywhere
  float* o;
  float* lse;                    // [batch][q_heads][q_len][2]: log2 of the softmax' denominator, see log_sum; +inf, 0 where nothing is seen
  const float* dout;             // gradient of o
  const float* delta;            // [batch][q_heads][delta_pitch]: - rows of dout * o summed
  int64_t delta_pitch;
  float *dq, *dk, *dv;
  int acc_q, acc_k, acc_v;
  int batch, q_heads, kv_heads, q_len, kv_len, dim;
  int window, sinks;
  float scale;
  float down, up;                // powers of two, down * up = 1: kv_len weights times any value times `down` stay below the largest
  int* status;
  const HeadInfo* info;          // of q's, k's, v's and (backward) dout's heads, or null: see group_ok
  int backward;
  int beside;                    // FP32 pipe: runs beside the kernel in front of it, which shares only operands with it
};

constexpr float kLog2e = 1.4426950408889634f;

// The tiles of keys that a tile of queries sees: those of the first tokens, then those of the window.
struct KeyTiles {
  int sink_tiles, first, count;
  // queries at positions [p_lo, p_hi]
  __host__ __device__ KeyTiles(int p_lo, int p_hi, int window, int sinks, int tile) {
    const int lowest = p_lo - window + 1 > 0 ? p_lo - window + 1 : 0;
    first = lowest / tile;
    const int s = (sinks + tile - 1) / tile;
    sink_tiles = s < first ? s : first;
    count = sink_tiles + p_hi / tile - first + 1;
  }
  __host__ __device__ int at(int t) const { return t < sink_tiles ? t : first + t - sink_tiles; }
};

// The positions of queries that see some of the keys [j_lo, j_hi].
struct QuerySpan {
  int lo, hi;                    // hi < lo: none
  __host__ __device__ QuerySpan(int j_lo, int j_hi, int window, int sinks, int past, int length) {
    lo = j_lo > past ? j_lo : past;
    hi = length - 1;
    if (j_lo >= sinks && (int64_t)j_hi + window - 1 < hi) hi = j_hi + window - 1;
  }
};

__host__ __device__ inline bool attn_visible(int p, int j, int window, int sinks) {
  return j <= p && (p - j < window || j < sinks);
}

#ifdef __CUDACC__
// The length of a sequence: whole, not above kv_len; below zero counts as zero.
__device__ __forceinline__ int attn_length(const float* lengths, int b, int kv_len, int* status) {
  if (!lengths) return kv_len;
  const float x = __ldg(lengths + b);
  if (x < 0.0f) return 0;
  if (!(x <= (float)kv_len) || x != floorf(x)) {
    if (atomicCAS(status, 0, LNN_E_INVALID) == 0) { status[1] = 4; status[2] = b; status[3] = (int)x; }
    return 0;
  }
  return (int)x;
}

__device__ __forceinline__ HeadInfo info_of(const AttnArgs& a, int tensor, int head) {
  const int nq = a.batch * a.q_heads, nk = a.batch * a.kv_heads;
  const int* p = reinterpret_cast<const int*>(a.info + (tensor == 0 ? 0 : nq + (tensor - 1) * nk) + head);
  return {__ldg(p), __ldg(p + 1), __int_as_float(__ldg(p + 2))};
}
// Whether the tensor cores take the query heads of key head hk: all of its operands were split without loss and the
// products of their scales stay far inside fp32's range.  The FP32-pipe kernels take the others.
__device__ __forceinline__ bool group_ok(const AttnArgs& a, int b, int hk) {
  const int group = a.q_heads / a.kv_heads, kvh = b * a.kv_heads + hk;
  const HeadInfo k = info_of(a, 1, kvh), v = info_of(a, 2, kvh);
  bool ok = k.ok && v.ok && abs(k.e) <= 100 && abs(v.e) <= 100;
  for (int i = 0; i < group; ++i) {
    const int h = b * a.q_heads + hk * group + i;
    const HeadInfo q = info_of(a, 0, h);
    ok = ok && q.ok && abs(q.e) <= 100 && abs(q.e + k.e) <= 100;
    if (a.backward) {
      const HeadInfo o = info_of(a, 3, h);
      // (weights times 2^row_exp, 2^-26 2^-(o.e + v.e) or more, are above fp32's smallest down to 2^-44: what is left of 2^-40 in fp16)
      ok = ok && o.ok && abs(o.e) <= 100 && o.e + v.e >= -100 && o.e + v.e <= 56 && abs(q.e + o.e + v.e) <= 90 && abs(k.e + o.e + v.e) <= 90;
    }
  }
  return ok;
}
// For a whole block: whether any of its work is left to the FP32 pipe.
__device__ __forceinline__ bool any_group_left(const AttnArgs& a) {
  int left = 0;
  for (int i = threadIdx.x; i < a.batch * a.kv_heads; i += blockDim.x) left |= !group_ok(a, i / a.kv_heads, i % a.kv_heads);
  return __syncthreads_or(left) != 0;
}

// The smaller of the two, or NaN where one of them is (fminf would drop it, and a weight of NaN would become one of 1).
__device__ __forceinline__ float min_or_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// log2 of a softmax' denominator, c top + log2(sum) where sum is of 2^(c (s - top)), as the sum of two floats: 24 bits of it
// would leave a weight 2^(c s - log_sum) nothing to go by once scores are large (half a step is 2^-11 at 10^4 and 1 at 10^7).  The
// difference fma(c, s, -hi) is rounded at its own size.  NaN where the scores themselves are past fp32's range.
__device__ __forceinline__ float2 log_sum(float top, float c, float sum) {
  const float p = __fmul_rn(top, c), q = log2f(sum);
  if (!(fabsf(p) <= FLT_MAX)) return make_float2(CUDART_NAN_F, 0.0f);
  const float hi = __fadd_rn(p, q), b = __fsub_rn(hi, p);
  return make_float2(hi, __fadd_rn(fmaf(top, c, -p), __fadd_rn(__fsub_rn(p, __fsub_rn(hi, b)), __fsub_rn(q, b))));
}
// 2^x with a relative error of 2^-22, 0 below the normal numbers
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
#endif

// On the FP32 pipe; with `info`, only the heads that the tensor cores have left.  Gradients: those that are not null.
int attn_simt_fwd(Device* d, const AttnArgs& a);
int attn_simt_bwd(Device* d, const AttnArgs& a);
bool attn_tc_applicable(const AttnArgs& a);
int attn_tc_fwd(Device* d, const AttnArgs& a);
int attn_tc_bwd(Device* d, const AttnArgs& a);
int attn_delta(Device* d, float* delta, const float* dout, const float* o, int64_t rows, int dim);

}  // namespace lnn
