// Causal attention with a sliding window and a few first tokens ("sinks") that stay visible: what its translation
// units share.
//
// Query i of q_len sits at position p = i + kv_len - q_len of its sequence, and sees key j when
//   p < length,  j <= p  and  (p - j < window  or  j < sinks).
// Rows that see nothing (padding behind a sequence's length) give zeros and receive and pass on no gradient.
#pragma once
#include "lnn_common.cuh"

namespace lnn {

struct AttnArgs {
  const float *q, *k, *v;        // [batch][q_heads][q_len][dim], [batch][kv_heads][kv_len][dim]
  const float* lengths;          // [batch] whole numbers, or null: kv_len everywhere
  float* o;
  float* lse;                    // [batch][q_heads][q_len]: log2 of the softmax' denominator, +inf where nothing is seen
  const float* dout;             // gradient of o
  const float* delta;            // [batch][q_heads][q_len]: rows of dout * o summed
  float *dq, *dk, *dv;
  int acc_q, acc_k, acc_v;
  int batch, q_heads, kv_heads, q_len, kv_len, dim;
  int window, sinks;
  float scale;
  int* status;
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

// 2^x with a relative error of 2^-22, 0 below the normal numbers
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
#endif

int attn_simt_fwd(Device* d, const AttnArgs& a);
int attn_simt_bwd(Device* d, const AttnArgs& a);       // the gradients that are not null
int attn_delta(Device* d, float* delta, const float* dout, const float* o, int64_t rows, int dim);

}  // namespace lnn
