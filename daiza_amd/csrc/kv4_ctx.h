// kv4_ctx.h — attention inputs of a context whose key/value cache is held in 4 bits (kv4.h).
#pragma once
#include "batch_kernels.h"
#include "kv4.h"
#include "model_kernels.h"

namespace dz {

// Column col of token t's attention in-projection: the product itself (n-token forward), ...
struct ProjRows {
  const float* y;
  int64_t ld;
  __device__ __forceinline__ float scale() const { return 1.f; }
  __device__ __forceinline__ float at(int t, int64_t col, float) const { return y[(size_t)t * ld + col]; }
};
// ... or one token's split-K partials, times 1/rms of its input.
template <int NP>
struct ProjPartials {
  const float* p;
  int np;
  int64_t ldp;
  const float* ss;
  int nss;
  int64_t H;
  float eps;
  __device__ __forceinline__ float scale() const { return inv_rms_from(ss, nss, H, eps); }
  __device__ __forceinline__ float at(int, int64_t col, float s) const { return sum_strided<NP>(p, ldp, np, col) * s; }
};

// bt_attn_prep_kernel with the cache rows written in 4 bits: per q-head RMSNorm, partial RoPE and 1/sqrt(256) -> qb[t][h],
// the gate half -> gate[t][h]; per kv-head the same for k (no scale), k and v quantised into row row0 + t of the cache,
// whose weight (where weights are kept) starts at 0.  Position pos0 + t.  Grid (n, nq + nkv), 256 threads, one dim each.
template <class Src>
__global__ __launch_bounds__(256) void kv4_prep_kernel(Src src, int nq, int nkv, const float* __restrict__ q_norm,
                                                       const float* __restrict__ k_norm, float eps, const float* __restrict__ rope,
                                                       int rope_dim, int pos0, int row0, float* __restrict__ qb,
                                                       float* __restrict__ gate, Kv4View c, float* __restrict__ weights, int64_t ldw) {
  constexpr int HD = 256, T = HD / 32;
  __shared__ float xs[HD];
  __shared__ float red[4];
  __shared__ uint8_t code[2][HD];
  const int t = blockIdx.x, hh = blockIdx.y;
  const unsigned tid = threadIdx.x;
  const bool isq = hh < nq;
  const int kvh = hh - nq;
  const float sc = src.scale();
  const float raw = src.at(t, isq ? (int64_t)hh * 2 * HD + tid : (int64_t)nq * 2 * HD + (int64_t)kvh * HD + tid, sc);
  // the gate (q-head) or v (kv-head) value of this dim, the norm weight and the RoPE factors, requested with raw
  const float other =
      src.at(t, isq ? (int64_t)hh * 2 * HD + HD + tid : (int64_t)nq * 2 * HD + (int64_t)nkv * HD + (int64_t)kvh * HD + tid, sc);
  const float nwt = isq ? q_norm[tid] : k_norm[tid];
  const int half = rope_dim / 2;
  const int dd = (int)tid < half ? (int)tid : (int)tid - half;
  const bool rot = (int)tid < rope_dim;
  const float* cs = rope + (size_t)(pos0 + t) * rope_dim;
  const float co = rot ? cs[dd] : 0.f, sn = rot ? cs[half + dd] : 0.f;
  const float s = wave_sum(raw * raw);
  if ((tid & 63u) == 0) red[tid >> 6] = s;
  __syncthreads();
  const float ssum = (red[0] + red[1]) + (red[2] + red[3]);
  const float in = 1.0f / sqrtf(ssum / (float)HD + eps);
  xs[tid] = (raw * in) * nwt;
  __syncthreads();
  float v = xs[tid];
  if (rot) {
    const float x1 = xs[dd], x2 = xs[dd + half];
    v = (int)tid < half ? __builtin_fmaf(x1, co, x2 * sn) : __builtin_fmaf(x2, co, x1 * sn);
  }
  if (isq) {
    qb[((size_t)t * nq + hh) * HD + tid] = v * (1.0f / sqrtf((float)HD));
    gate[((size_t)t * nq + hh) * HD + tid] = other;
    return;
  }
  const int64_t r = (int64_t)row0 + t;
  const size_t ch = (size_t)kvh * c.code_head(), sh = (size_t)kvh * c.scale_head();
  const float both[2] = {v, other};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    unsigned big = __float_as_uint(both[i]) & 0x7FFFFFFFu;  // as whole numbers: a NaN is larger than every number
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) big = max(big, (unsigned)__shfl_xor((int)big, o));
    const int sb = kv4_scale_byte(__uint_as_float(big));
    code[i][tid] = (uint8_t)kv4_code(both[i], sb);
    if ((tid & 31u) == 0) {
      (i ? c.vs : c.ks)[sh + (size_t)r * T + tid / 32] = (uint8_t)sb;
      if (sb == 255) c.bad[(size_t)kvh * (c.cap / kKv4Tile) + r / kKv4Tile] = 1;
    }
  }
  __syncthreads();
  if (tid < HD / 8) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (unsigned)code[0][8 * tid + i] << (4 * i);
    *reinterpret_cast<unsigned*>(c.kc + ch + (size_t)r * (HD / 2) + 4 * tid) = w;
  } else if (tid < HD / 8 + 16) {
    const int ln = (int)tid - HD / 8;
    u32x2 w{0, 0};
#pragma unroll
    for (int b = 0; b < T; ++b)
      w[b / 4] |= (unsigned)(code[1][32 * b + 2 * ln] | code[1][32 * b + 2 * ln + 1] << 4) << (8 * (b % 4));
    *reinterpret_cast<u32x2*>(c.vc + ch + kv4_value_offset<HD>(r, ln)) = w;
  } else if (tid == 255 && weights) {
    weights[(size_t)kvh * ldw + r] = 0.f;
  }
}

}  // namespace dz
