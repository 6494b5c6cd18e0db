// logprobs.hip — log probabilities of given tokens, entropies and the best alternatives of rows of logits.
#include <math.h>

#include "elem.h"
#include "topk.h"

namespace dz {

constexpr int kLogprobTop = 64;

// A logit and its id as one word whose unsigned order is "larger value first, then lower id", NaN below -inf.
__device__ __forceinline__ uint64_t logit_key(float v, int i) {
  const uint64_t id = (unsigned)~(unsigned)i;
  return v != v ? id : (cand_key(v, i) & 0xFFFFFFFF00000000ull) | id;
}

template <class E>
__global__ __launch_bounds__(1024) void logprobs_simple_kernel(const E* __restrict__ x, int64_t ld, int vocab,
                                                               const int32_t* __restrict__ tokens, int top,
                                                               float* __restrict__ logp, float* __restrict__ entropy,
                                                               int32_t* __restrict__ top_ids, float* __restrict__ top_logp) {
  __shared__ float red[2][16];
  __shared__ uint64_t kred[16];
  const int i = blockIdx.x, tid = threadIdx.x;
  x += (size_t)i * ld;
  float m = -INFINITY;
  for (int c = tid; c < vocab; c += 1024) m = fmaxf(m, to_f32(x[c]));
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) red[0][tid >> 6] = m;
  __syncthreads();
  for (int w = 0; w < 16; ++w) m = fmaxf(m, red[0][w]);
  __syncthreads();
  float z = 0.f, a = 0.f;
  for (int c = tid; c < vocab; c += 1024) {
    const float d = to_f32(x[c]) - m, e = expf(d);
    z += e;
    a += d == -INFINITY ? 0.f : e * d;
  }
  z = wave_sum(z);
  a = wave_sum(a);
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = z;
    red[1][tid >> 6] = a;
  }
  __syncthreads();
  z = a = 0.f;
  for (int w = 0; w < 16; ++w) {
    z += red[0][w];
    a += red[1][w];
  }
  const float lz = logf(z);
  if (tid == 0) {
    if (logp) {
      const int t = tokens[i];
      logp[i] = t < 0 || t >= vocab ? __builtin_nanf("") : (to_f32(x[t]) - m) - lz;
    }
    if (entropy) entropy[i] = lz - a / z;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int c = tid; c < vocab; c += 1024) {
      const uint64_t key = logit_key(to_f32(x[c]), c);
      if (key < last && key > best) best = key;
    }
    best = wave_max_key(best);
    __syncthreads();
    if ((tid & 63) == 0) kred[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < 16; ++w) best = kred[w] > best ? kred[w] : best;
    last = best;
    if (tid == 0) {
      const int id = (int)~(unsigned)best;
      top_ids[(size_t)i * top + k] = id;
      if (top_logp) top_logp[(size_t)i * top + k] = (to_f32(x[id]) - m) - lz;
    }
  }
}

size_t logprobs_work(int n, int64_t vocab, int top) { return 16; }

int logprobs(const void* logits, int64_t ld, int type, int n, int vocab, const int32_t* tokens, int top, float* logp, float* entropy,
             int32_t* top_ids, float* top_logp, void* work, hipStream_t s) {
  return with_type(type, [&](auto* e) -> int {
    using E = std::remove_pointer_t<decltype(e)>;
    logprobs_simple_kernel<E><<<(unsigned)n, 1024, 0, s>>>((const E*)logits, ld, vocab, tokens, top, logp, entropy, top_ids, top_logp);
    DZ_HIP_CHECK(hipGetLastError());
    return DZ_OK;
  });
}

}  // namespace dz

using namespace dz;

extern "C" {

size_t dz_logprobs_work_bytes(int n, int64_t vocab, int top) {
  return n < 1 || vocab < 1 || top < 0 || top > kLogprobTop ? 0 : logprobs_work(n, vocab, top);
}

int dz_logprobs_dev(const void* logits, int64_t ld, int type, int n, int64_t vocab, const int32_t* tokens, int top, float* logp,
                    float* entropy, int32_t* top_ids, float* top_logp, void* work, void* stream) {
  if (int rc = check_type(type)) return rc;
  if (n < 0 || vocab < 1 || vocab > (int64_t)1 << 30) return set_error(DZ_ERR_TENSOR, "logprobs: %d rows of %lld", n, (long long)vocab);
  if (ld < vocab) return set_error(DZ_ERR_TENSOR, "logprobs: row stride %lld under %lld", (long long)ld, (long long)vocab);
  if (top < 0 || top > kLogprobTop || top > vocab)
    return set_error(DZ_ERR_UNSUPPORTED, "logprobs: %d alternatives of %lld (at most %d)", top, (long long)vocab, kLogprobTop);
  if (n == 0) return DZ_OK;
  if (!logits || !work || (top && !top_ids) || (logp && !tokens)) return set_error(DZ_ERR_MODEL, "null argument");
  int rc = ensure_device(), dev = 0;
  if (rc) return rc;
  DZ_HIP_CHECK(hipGetDevice(&dev));
  if ((rc = check_array(logits, type_size(type), dev, "logits")) || (rc = check_array(work, 16, dev, "work")) ||
      (logp && ((rc = check_array(tokens, 4, dev, "tokens")) || (rc = check_array(logp, 4, dev, "logp")))) ||
      (entropy && (rc = check_array(entropy, 4, dev, "entropy"))) || (top && (rc = check_array(top_ids, 4, dev, "top_ids"))) ||
      (top && top_logp && (rc = check_array(top_logp, 4, dev, "top_logp"))))
    return rc;
  return logprobs(logits, ld, type, n, (int)vocab, tokens, top, logp, entropy, top_ids, top_logp, work, static_cast<hipStream_t>(stream));
}

}  // extern "C"
