// logprobs.hip — log probabilities of given tokens, entropies and the best alternatives of rows of logits.
#include <math.h>

#include <algorithm>

#include "elem.h"
#include "logprobs.h"
#include "topk.h"

namespace dz {

constexpr int kLogprobTop = 64;   // most alternatives: a wave's lanes
constexpr int kLpVals = 16;       // logits of a lane and step
constexpr int kLpStep = 64 * kLpVals;
constexpr int kLpMaxParts = 256;  // parts of a row: the join's threads
constexpr int kLpKeep = 2 * kLogprobTop + 16;       // a longer list is cut to the best
constexpr int kLpCand = kLpKeep + kLpStep;          // ... which one step can outgrow by this much

// A logit and its id as one word whose unsigned order is "larger value first, then lower id", NaN below -inf.
__device__ __forceinline__ uint64_t logit_key(float v, int i) {
  const unsigned u = __float_as_uint(v + 0.f), o = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
  return (uint64_t)(v != v ? 0u : o) << 32 | (unsigned)~(unsigned)i;
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

// 16 bytes from an address of the element's own alignment, and the values that they are.
template <class E>
__device__ __forceinline__ u32x4 load16(const E* p) {
  struct __attribute__((packed, aligned(sizeof(E)))) Raw {
    u32x4 w;
  };
  return reinterpret_cast<const Raw*>(p)->w;
}
template <class E, int R>
__device__ __forceinline__ void values_of(u32x4 w, float* x) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if constexpr (R == 4) x[i] = __uint_as_float(w[i]);
    else x[i] = to_f32(__builtin_bit_cast(E, (uint16_t)(w[i / 2] >> (16 * (i & 1)))));
  }
}

// Wave-wide (one wave a workgroup, so LDS needs no barrier but the compiler's).
__device__ __forceinline__ void lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The `top` largest of the cnt (>= top) distinct keys in c, in order, to c[0 .. top): every key counts the larger ones.
__device__ __forceinline__ void prune(uint64_t* c, int cnt, int top, int lane) {
  // in rounds of 64: a key's rank is known before any is moved, so the best of all go to a second place first
  uint64_t best = 0;  // lane r: the key of rank r
  __shared__ uint64_t out[kLogprobTop];
  for (int i0 = 0; i0 < cnt; i0 += 64) {
    const uint64_t mine = i0 + lane < cnt ? c[i0 + lane] : 0;
    int r = mine ? 0 : kLogprobTop;
    for (int j = 0; j < cnt; ++j) r += c[j] > mine ? 1 : 0;
    if (r < top) out[r] = mine;
  }
  lds_fence();
  if (lane < top) best = out[lane];
  if (lane < top) c[lane] = best;
  lds_fence();
}

// One part of a row by one wave: its sums and its `top` best keys in order.  A pass over the logits, 1024 a step, the next
// step's on their way: each lane keeps its own running maximum and sums.  Keys above the part's top-th best so far
// (`bound`) go to a list in LDS; a lane looks at its keys only where the largest of its logits reaches the bound's value.
// Where more than 32 lanes do (the first step; rows that keep rising) the bound first rises to the top-th largest of the
// lanes' own best keys: only lanes whose best is above it can then add any.
// Bound by the loads at many rows: 16 exponentials and about 120 other instructions a lane and step of 4 KB of f32.
// Grid (parts, n), 64 threads.
template <class E, bool TOP>
__global__ __launch_bounds__(64) void logprobs_kernel(const E* __restrict__ x, int64_t ld, int vocab, int per, int top,
                                                      LogitSums* __restrict__ sums, uint64_t* __restrict__ keys) {
  constexpr int R = 16 / sizeof(E);  // a lane's logits: runs of 16 bytes, the wave's runs one after another
  __shared__ uint64_t cand[TOP ? kLpCand : 1];
  const int lane = threadIdx.x, part = blockIdx.x, parts = gridDim.x;
  const size_t row = blockIdx.y;
  x += row * (size_t)ld;
  const int beg = part * per, end = min(vocab, beg + per);
  LogitSums s{-INFINITY, 0.f, 0.f};
  uint64_t bound = 0;  // keys up to this one are not among the part's best
  float floor = 0.f;   // only larger logits have keys above it, where it is that of a number
  bool any = true;     // it is none: every key is looked at
  int cnt = 0;
  auto raise = [&](uint64_t key) {
    bound = key;
    floor = cand_of(key).v;
    any = key <= (uint64_t)0x00800000u << 32;  // NaN, nothing, or -inf
  };
  // the logits of the step at c0
  auto step = [&](int c0, const float (&v)[kLpVals]) {
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
      const unsigned long long over = __ballot(any || vm > floor);
      if (over) {
        auto key_at = [&](int i) {
          const int c = c0 + ((i / R) * 64 + lane) * R + i % R;
          return c < end ? logit_key(v[i], c) : (uint64_t)0;
        };
        if (__popcll(over) > 32) {
          uint64_t best = 0;
#pragma unroll
          for (int i = 0; i < kLpVals; ++i) {
            const uint64_t k = key_at(i);
            best = k > best ? k : best;
          }
          cand[cnt + lane] = best;  // behind the list
          lds_fence();
          int r = best > bound ? 0 : 64;
#pragma unroll 8
          for (int j = 0; j < 64; ++j) r += cand[cnt + j] > best ? 1 : 0;
          lds_fence();
          const unsigned long long at = __ballot(r == top - 1);  // none where fewer lanes than top are above the bound
          if (at) {
            const int l = __builtin_ctzll(at);
            const uint64_t k = ((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(best >> 32), l) << 32) |
                               (unsigned)__builtin_amdgcn_readlane((int)(unsigned)best, l);
            raise(k - 1);
            // an equal logit of a lower id in this step is above the bound: the next number down (below 0, past -0)
            floor = floor == 0.f ? -__uint_as_float(1u) : cand_of(bound - ((uint64_t)1 << 32)).v;
          }
        }
#pragma unroll
        for (int i = 0; i < kLpVals; ++i) {
          if (!__ballot(any || v[i] > floor)) continue;
          const uint64_t k = key_at(i);
          const unsigned long long in = __ballot(k > bound);
          if (k > bound) cand[cnt + __popcll(in & ((1ull << lane) - 1))] = k;
          cnt += __popcll(in);
        }
        lds_fence();
        if (cnt > kLpKeep || (any && cnt >= top)) {
          prune(cand, cnt, top, lane);
          cnt = top;
          raise(cand[top - 1]);
        } else if (!any) {
          floor = cand_of(bound).v;  // later ids do not win ties
        }
      }
    }
  };
  // whole steps, whose loads need no bounds and are requested a step ahead; then what is left
  const int whole = beg + (end - beg) / kLpStep * kLpStep;
  if (beg < whole) {
    const E* p = x + lane * R;
    u32x4 next[kLpVals / R];
#pragma unroll
    for (int k = 0; k < kLpVals / R; ++k) next[k] = load16(p + beg + k * 64 * R);
    for (int c0 = beg; c0 < whole; c0 += kLpStep) {
      float v[kLpVals];
#pragma unroll
      for (int k = 0; k < kLpVals / R; ++k) values_of<E, R>(next[k], v + k * R);
      const int cn = min(c0 + kLpStep, whole - kLpStep);
#pragma unroll
      for (int k = 0; k < kLpVals / R; ++k) next[k] = load16(p + cn + k * 64 * R);
      step(c0, v);
    }
  }
  if (whole < end) {
    float v[kLpVals];
#pragma unroll
    for (int i = 0; i < kLpVals; ++i) {
      const int c = whole + ((i / R) * 64 + lane) * R + i % R;
      const float u = to_f32(x[min(c, end - 1)]);
      v[i] = c < end ? u : -INFINITY;
    }
    step(whole, v);
  }
  // the lanes' sums in a fixed order
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const LogitSums y{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.a, o)};
    s = join(s, y);
  }
  if (lane == 0) sums[row * parts + part] = s;
  if constexpr (TOP) {
    // a part of fewer logits than top keeps what it has, in order, and zeros
    for (int i = cnt + lane; i < top; i += 64) cand[i] = 0;
    lds_fence();
    prune(cand, max(cnt, top), top, lane);
    if (lane < top) keys[(row * parts + part) * top + lane] = lane < cnt ? cand[lane] : 0;
  }
}

// The parts of a row as its results.  Of the parts' lists, each in order, only those whose first key is among the `top`
// largest first keys can hold one of the row's best, and only keys not below the last of those: they are gathered
// in LDS (at most top x top of them, a few more than top as a rule) and ranked by counting the larger ones.
// Grid (n), 256 threads, thread p for part p.
template <class E>
__global__ __launch_bounds__(256) void logprobs_join_kernel(const E* __restrict__ x, int64_t ld, int vocab, int parts, int top,
                                                            const LogitSums* __restrict__ sums, const uint64_t* __restrict__ keys,
                                                            const int32_t* __restrict__ tokens, float* __restrict__ logp,
                                                            float* __restrict__ entropy, int32_t* __restrict__ top_ids,
                                                            float* __restrict__ top_logp) {
  __shared__ uint64_t cand[kLogprobTop * kLogprobTop], first[256], out[kLogprobTop];
  __shared__ LogitSums red[4];
  __shared__ uint64_t s_bound;
  __shared__ int s_cnt;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const size_t row = blockIdx.x;
  x += row * (size_t)ld;
  if (tid < top) out[tid] = 0;
  const bool has = tid < parts;
  const int t = logp ? tokens[row] : -1;
  LogitSums s{-INFINITY, 0.f, 0.f};
  if (has) s = sums[row * parts + tid];
  const uint64_t* list = keys + (row * (size_t)parts + (has ? tid : 0)) * top;
  constexpr int N = 4;  // of its list, requested with the sums
  uint64_t k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = has && i < top ? list[min(i, top - 1)] : 0;
  const float xt = t >= 0 && t < vocab ? to_f32(x[t]) : __builtin_nanf("");
  if (tid == 0) {
    s_cnt = 0;
    s_bound = 1;  // fewer parts than top: every key
  }
  first[tid] = k[0];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const LogitSums y{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.a, o)};
    s = join(s, y);
  }
  if (lane == 0) red[w] = s;
  __syncthreads();
  if (parts >= top && top && 64 * w < parts) {
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < parts; ++j) r += first[j] > k[0] ? 1 : 0;
    if (k[0] && r == top - 1) s_bound = k[0];
  }
  __syncthreads();
  const uint64_t bound = s_bound;
  for (int i = 0; i < top; ++i) {
    const uint64_t key = i == 0 ? k[0] : i == 1 ? k[1] : i == 2 ? k[2] : i == 3 ? k[3] : has ? list[i] : 0;
    const bool in = key >= bound;
    if (!__ballot(in)) break;
    if (in) cand[atomicAdd(&s_cnt, 1)] = key;
  }
  __syncthreads();
  const int cnt = s_cnt;
  for (int i = tid; i < cnt; i += 256) {
    const uint64_t mine = cand[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < cnt; ++j) r += cand[j] > mine ? 1 : 0;
    if (r < top) out[r] = mine;
  }
  __syncthreads();
  s = join(join(red[0], red[1]), join(red[2], red[3]));
  const float lz = s.m == -INFINITY ? __builtin_nanf("") : logf(s.z);
  if (tid == 0) {
    if (logp) logp[row] = (xt - s.m) - lz;
    if (entropy) entropy[row] = lz - s.a / s.z;
  }
  if (tid < top) {
    const uint64_t key = out[tid];
    const int id = (int)min(~(unsigned)key, (unsigned)(vocab - 1));
    top_ids[row * top + tid] = id;
    if (top_logp) top_logp[row * top + tid] = (to_f32(x[id]) - s.m) - lz;
  }
}

// Parts of a row: whole steps, enough waves to fill the device.
static int logprob_parts(int n, int64_t vocab, int* per) {
  const int64_t steps = (vocab + kLpStep - 1) / kLpStep;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({steps, kLpMaxParts, 4096 / n}));
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
      if (top) logprobs_kernel<E, true><<<g, 64, 0, s>>>(x + (size_t)r0 * ld, ld, vocab, per, top, sums + at, keys + at * top);
      else logprobs_kernel<E, false><<<g, 64, 0, s>>>(x + (size_t)r0 * ld, ld, vocab, per, top, sums + at, keys);
      DZ_HIP_CHECK(hipGetLastError());
    }
    logprobs_join_kernel<E><<<(unsigned)n, 256, 0, s>>>(x, ld, vocab, parts, top, sums, keys, tokens, logp, entropy, top_ids, top_logp);
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
