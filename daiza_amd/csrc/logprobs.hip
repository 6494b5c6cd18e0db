// logprobs.hip — log probabilities of given tokens, entropies and the best alternatives of rows of logits.
#include <math.h>

#include <algorithm>

#include "elem.h"
#include "logprobs.h"
#include "topk.h"

namespace dz {

constexpr int kLogprobTop = 64;     // most alternatives
constexpr int kLpThreads = 256;
constexpr int kLpVals = 16;         // logits of a thread and step
constexpr int kLpStep = kLpThreads * kLpVals;
constexpr int kLpMaxSplits = 64;    // parts of a row
constexpr int kLpCand = kLogprobTop * kLpVals + 2 * kLogprobTop;  // candidates in LDS (see logprobs_kernel)

// A logit and its id as one word whose unsigned order is "larger value first, then lower id", NaN below -inf.
__device__ __forceinline__ uint64_t logit_key(float v, int i) {
  const uint64_t id = (unsigned)~(unsigned)i;
  return v != v ? id : (cand_key(v, i) & 0xFFFFFFFF00000000ull) | id;
}

// Σ e^(x-m) (z) and Σ e^(x-m) (x-m) (a) over some logits whose largest is m.
struct LogitSums {
  float m, z, a;
};
constexpr float kLpFar = -1e4f;  // e^ of it is 0, its products with sums are finite
// The sums at a maximum M >= s.m.
__device__ __forceinline__ LogitSums at_maximum(const LogitSums& s, float M) {
  if (s.m == -INFINITY) return LogitSums{M, s.z, s.a};  // no terms yet (or NaN, which stays)
  const float d = fmaxf(s.m - M, kLpFar), f = expf(d);
  return LogitSums{M, s.z * f, f * __builtin_fmaf(d, s.z, s.a)};
}
__device__ __forceinline__ LogitSums join(const LogitSums& x, const LogitSums& y) {
  const float M = fmaxf(x.m, y.m);
  const LogitSums p = at_maximum(x, M), q = at_maximum(y, M);
  return LogitSums{M, p.z + q.z, p.a + q.a};
}

// N consecutive elements from an address of the element's own alignment.
template <class E, int N>
__device__ __forceinline__ void load_elems(const E* p, float (&x)[N]) {
  struct __attribute__((packed, aligned(sizeof(E)))) Raw {
    E e[N];
  };
  const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f32(r.e[i]);
}

// The `top` largest of the cnt (>= top) distinct keys in c, in order, to c[0 .. top): every key counts the larger ones.
// The workgroup's threads call it together; cnt <= kLpCand.
__device__ __forceinline__ void prune(uint64_t* c, int cnt, int top, int tid) {
  constexpr int N = (kLpCand + kLpThreads - 1) / kLpThreads;
  uint64_t mine[N];
  int rank[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = tid + k * kLpThreads;
    rank[k] = kLpCand;
    if (i < cnt) {
      mine[k] = c[i];
      int r = 0;
      for (int j = 0; j < cnt; ++j) r += c[j] > mine[k] ? 1 : 0;
      rank[k] = r;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (rank[k] < top) c[rank[k]] = mine[k];
  __syncthreads();
}

// One part of a row: its sums and its `top` best keys.  A pass over the logits, 4096 a step: each thread keeps its own
// running maximum and sums; keys above the part's top-th best so far go to a list in LDS.  A step in which more than 64
// threads have such a key (the first one; rows that keep rising) first raises the bound to the top-th largest of the threads'
// own best keys of the step: only threads whose best is above it can then add any, so that a step adds at most
// 64 x 16 keys to the 64 that a pruned list holds.
// Grid (parts, n), 256 threads.  part -> sums[row][part], keys[row][part][top].
template <class E, bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(const E* __restrict__ x, int64_t ld, int vocab, int per, int top,
                                                              LogitSums* __restrict__ sums, uint64_t* __restrict__ keys) {
  __shared__ uint64_t cand[TOP ? kLpCand : 1], best[TOP ? kLpThreads : 1];
  __shared__ int s_cnt, s_n;
  __shared__ uint64_t s_bound;
  __shared__ LogitSums red[kLpThreads / 64];
  const int tid = threadIdx.x, part = blockIdx.x, parts = gridDim.x;
  const size_t row = blockIdx.y;
  x += row * (size_t)ld;
  const int beg = part * per, end = min(vocab, beg + per);
  LogitSums s{-INFINITY, 0.f, 0.f};
  uint64_t bound = 0;  // keys up to this one are not among the part's best
  if (TOP && tid == 0) s_cnt = 0;
  float v[kLpVals];
  auto load = [&](int c0) {
    // a thread's logits: runs of 16 bytes, the workgroup's runs one after another
    constexpr int R = 16 / sizeof(E);
#pragma unroll
    for (int k = 0; k < kLpVals / R; ++k) {
      const int c = c0 + (k * kLpThreads + tid) * R;
      float r[R];
      if (c + R <= end) {
        load_elems(x + c, r);
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) r[i] = c + i < end ? to_f32(x[c + i]) : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) v[k * R + i] = r[i];
    }
  };
  auto index = [&](int c0, int i) {
    constexpr int R = 16 / sizeof(E);
    return c0 + ((i / R) * kLpThreads + tid) * R + i % R;
  };
  for (int c0 = beg; c0 < end; c0 += kLpStep) {
    load(c0);
    float vm = v[0];
#pragma unroll
    for (int i = 1; i < kLpVals; ++i) vm = fmaxf(vm, v[i]);
    const float M = fmaxf(s.m, vm);
    if (M > s.m) s = at_maximum(s, M);
    const float base = M == -INFINITY ? 0.f : M;
    float z = 0.f, a = 0.f;
#pragma unroll
    for (int i = 0; i < kLpVals; ++i) {
      // e^d by the hardware's 2^x: the product's rounding is d 2^-24 of a term that is e^d
      const float d = v[i] - base, e = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      z += e;
      a = __builtin_fmaf(e, fmaxf(d, kLpFar), a);  // a logit of -inf adds nothing; NaN comes in by e
    }
    s.z += z;
    s.a += a;
    if constexpr (TOP) {
      uint64_t top_key = 0;
#pragma unroll
      for (int i = 0; i < kLpVals; ++i) {
        const int c = index(c0, i);
        const uint64_t k = c < end ? logit_key(v[i], c) : 0;
        top_key = k > top_key ? k : top_key;
      }
      if (tid == 0) s_n = 0;
      __syncthreads();  // also: the list is whole
      const unsigned long long over = __ballot(top_key > bound);
      if ((tid & 63) == 0 && over) atomicAdd(&s_n, __popcll(over));
      __syncthreads();
      const int n = s_n;
      if (n == 0) continue;
      if (n > kLogprobTop) {
        best[tid] = top_key;
        if (tid == 0) s_bound = bound;
        __syncthreads();
        int r = 0;
        for (int j = 0; j < kLpThreads; ++j) r += best[j] > top_key ? 1 : 0;
        // threads without a logit share the key 0: no rank is top - 1 then, and the bound stays
        if (r == top - 1 && top_key > bound) s_bound = top_key - 1;
        __syncthreads();
        bound = s_bound;
      }
#pragma unroll
      for (int i = 0; i < kLpVals; ++i) {
        const int c = index(c0, i);
        const uint64_t k = c < end ? logit_key(v[i], c) : 0;
        if (k > bound) cand[atomicAdd(&s_cnt, 1)] = k;
      }
      __syncthreads();
      const int cnt = s_cnt;
      if (cnt >= top) {
        prune(cand, cnt, top, tid);
        bound = cand[top - 1];
        if (tid == 0) s_cnt = top;
      }
    }
  }
  // the threads' sums, lanes and then waves in a fixed order
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const LogitSums y{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.a, o)};
    s = join(s, y);
  }
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    s = join(join(red[0], red[1]), join(red[2], red[3]));
    sums[row * parts + part] = s;
  }
  if constexpr (TOP) {
    const int cnt = s_cnt;
    if (tid < top) keys[(row * parts + part) * top + tid] = tid < cnt ? cand[tid] : 0;  // a part of fewer logits than top: unordered
  }
}

// The parts of a row as its results.  Grid (n), 256 threads.
template <class E>
__global__ __launch_bounds__(kLpThreads) void logprobs_join_kernel(const E* __restrict__ x, int64_t ld, int vocab, int parts, int top,
                                                                   const LogitSums* __restrict__ sums,
                                                                   const uint64_t* __restrict__ keys,
                                                                   const int32_t* __restrict__ tokens, float* __restrict__ logp,
                                                                   float* __restrict__ entropy, int32_t* __restrict__ top_ids,
                                                                   float* __restrict__ top_logp) {
  __shared__ uint64_t cand[kLpCand];
  __shared__ LogitSums sh;
  const int tid = threadIdx.x;
  const size_t row = blockIdx.x;
  x += row * (size_t)ld;
  if (tid < 64) {
    LogitSums s{-INFINITY, 0.f, 0.f};
    if (tid < parts) s = sums[row * parts + tid];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const LogitSums y{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.a, o)};
      s = join(s, y);
    }
    if (tid == 0) sh = s;
  }
  // the parts' best keys, as many parts at a time as the list holds beside those kept so far
  int cnt = 0;
  if (top) {
    const uint64_t* kr = keys + row * (size_t)parts * top;
    const int total = parts * top;
    for (int at = 0; at < total;) {
      const int take = min(total - at, kLpCand - cnt);
      for (int i = tid; i < take; i += kLpThreads) cand[cnt + i] = kr[at + i];
      at += take;
      cnt += take;
      __syncthreads();
      prune(cand, cnt, top, tid);
      cnt = top;
    }
  }
  __syncthreads();
  const LogitSums s = sh;
  const float lz = s.m == -INFINITY ? __builtin_nanf("") : logf(s.z);
  if (tid == 0) {
    if (logp) {
      const int t = tokens[row];
      logp[row] = t < 0 || t >= vocab ? __builtin_nanf("") : (to_f32(x[t]) - s.m) - lz;
    }
    if (entropy) entropy[row] = lz - s.a / s.z;
  }
  if (tid < top) {
    const int id = (int)~(unsigned)cand[tid];
    top_ids[row * top + tid] = id;
    if (top_logp) top_logp[row * top + tid] = (to_f32(x[id]) - s.m) - lz;
  }
}

// Parts of a row: whole steps, as many workgroups as fill the device a few times over.
static int logprob_parts(int n, int64_t vocab, int* per) {
  const int64_t steps = (vocab + kLpStep - 1) / kLpStep;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({steps, kLpMaxSplits, 2048 / n}));
  const int64_t p = (steps + want - 1) / want;
  *per = (int)(p * kLpStep);
  return (int)((steps + p - 1) / p);
}

size_t logprobs_work(int n, int64_t vocab, int top) {
  int per;
  const size_t parts = (size_t)n * logprob_parts(n, vocab, &per);
  return parts * ((size_t)top * sizeof(uint64_t)) + parts * sizeof(LogitSums) + 16;
}

int logprobs(const void* logits, int64_t ld, int type, int n, int vocab, const int32_t* tokens, int top, float* logp, float* entropy,
             int32_t* top_ids, float* top_logp, void* work, hipStream_t s) {
  int per;
  const int parts = logprob_parts(n, vocab, &per);
  uint64_t* keys = static_cast<uint64_t*>(work);
  LogitSums* sums = reinterpret_cast<LogitSums*>(keys + (size_t)n * parts * top);
  return with_type(type, [&](auto* e) -> int {
    using E = std::remove_pointer_t<decltype(e)>;
    const E* x = static_cast<const E*>(logits);
    // rows beyond the grid's second dimension go in further launches
    for (int r0 = 0; r0 < n; r0 += 65535) {
      const dim3 g((unsigned)parts, (unsigned)std::min(65535, n - r0));
      const size_t at = (size_t)r0 * parts;
      if (top) logprobs_kernel<E, true><<<g, kLpThreads, 0, s>>>(x + (size_t)r0 * ld, ld, vocab, per, top, sums + at, keys + at * top);
      else logprobs_kernel<E, false><<<g, kLpThreads, 0, s>>>(x + (size_t)r0 * ld, ld, vocab, per, top, sums + at, keys);
      DZ_HIP_CHECK(hipGetLastError());
    }
    logprobs_join_kernel<E><<<(unsigned)n, kLpThreads, 0, s>>>(x, ld, vocab, parts, top, sums, keys, tokens, logp, entropy, top_ids,
                                                                top_logp);
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
