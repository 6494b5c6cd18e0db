// logprobs.hip — log probabilities of given tokens, entropies and the best alternatives of rows of logits.
#include <math.h>

#include <algorithm>

#include "elem.h"
#include "logprobs.h"
#include "topk.h"

namespace dz {

constexpr int kLpVals = 16;      // logits of a lane and step
constexpr int kLpStep = 64 * kLpVals;
constexpr int kLpGroups = 4;     // groups of a step: the 16 lanes of a DPP row
constexpr int kLpMaxParts = 256; // parts of a row
constexpr int kLpCand = kLogprobTop * kLpVals + 2 * kLogprobTop;  // candidates in LDS (see logprobs_join_kernel)
constexpr int kLpJoin = 512;     // threads of the join
constexpr int kLpListed = 1024;  // groups looked through at a time

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

// Logits 16 lanes of a step hold: a lane's are runs of 16 bytes, the wave's runs one after another.
template <class E>
__device__ __forceinline__ int logit_at(int step, int lane, int i) {
  constexpr int R = 16 / sizeof(E);
  return step * kLpStep + ((i / R) * 64 + lane) * R + i % R;
}
// ... of a step that ends behind the row: -inf there.
template <class E>
__device__ __forceinline__ void load_ragged(const E* __restrict__ x, int step, int lane, int vocab, float (&v)[kLpVals]) {
#pragma unroll
  for (int i = 0; i < kLpVals; ++i) {
    const int c = logit_at<E>(step, lane, i);
    const float u = to_f32(x[min(c, vocab - 1)]);
    v[i] = c < vocab ? u : -INFINITY;
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false)));
}

// One part of a row by one wave: its sums, and the largest logit of every group of 256 (for the alternatives; gmax null:
// none wanted).  A pass over the logits, 1024 a step, the next step's on their way; each lane keeps its own running maximum
// and sums.  Bound by the loads: 1024 rows of 248320 bf16 logits at the rate of a copy (5.2 TB/s).  Keys and ids take no part
// here: a list of best keys kept during the pass cost 40% of it at 20 alternatives.
// Grid (parts, n), 64 threads.
template <class E>
__global__ __launch_bounds__(64) void logprobs_kernel(const E* __restrict__ x, int64_t ld, int vocab, int per,
                                                      LogitSums* __restrict__ sums, float* __restrict__ gmax) {
  constexpr int R = 16 / sizeof(E);
  const int lane = threadIdx.x, part = blockIdx.x, parts = gridDim.x;
  const size_t row = blockIdx.y;
  const int steps = (vocab + kLpStep - 1) / kLpStep;
  x += row * (size_t)ld;
  if (gmax) gmax += row * (size_t)steps * kLpGroups + (lane >> 4);
  const int beg = part * per, end = min(steps, beg + per);
  LogitSums s{-INFINITY, 0.f, 0.f};
  auto take = [&](int step, const float (&v)[kLpVals]) {
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
    if (gmax) {
      float g = vm;
      g = dpp_max<0xB1>(g);
      g = dpp_max<0x4E>(g);
      g = dpp_max<0x141>(g);
      g = dpp_max<0x140>(g);
      if ((lane & 15) == 0) gmax[step * kLpGroups] = g;
    }
  };
  // whole steps, whose loads need no bounds and are requested a step ahead; then what is left
  const int whole = min(end, vocab / kLpStep);
  if (beg < whole) {
    const E* p = x + lane * R;
    u32x4 next[kLpVals / R];
#pragma unroll
    for (int k = 0; k < kLpVals / R; ++k) next[k] = load16(p + (size_t)beg * kLpStep + k * 64 * R);
    for (int c = beg; c < whole; ++c) {
      float v[kLpVals];
#pragma unroll
      for (int k = 0; k < kLpVals / R; ++k) values_of<E, R>(next[k], v + k * R);
      const int cn = min(c + 1, whole - 1);
#pragma unroll
      for (int k = 0; k < kLpVals / R; ++k) next[k] = load16(p + (size_t)cn * kLpStep + k * 64 * R);
      take(c, v);
    }
  }
  if (whole < end) {
    float v[kLpVals];
    load_ragged(x, whole, lane, vocab, v);
    take(whole, v);
  }
  // the lanes' sums in a fixed order
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const LogitSums y{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.a, o)};
    s = join(s, y);
  }
  if (lane == 0) sums[row * parts + part] = s;
}

// The `top` largest of the cnt distinct keys in c, in order, to c[0 .. min(top, cnt)): every key counts the larger ones.
__device__ __forceinline__ void prune(uint64_t* c, int cnt, int top, int tid) {
  constexpr int N = (kLpCand + kLpJoin - 1) / kLpJoin;
  uint64_t mine[N];
  int rank[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = tid + kLpJoin * k;
    rank[k] = kLpCand;
    if (i < cnt) {
      mine[k] = c[i];
      int r = 0;
#pragma unroll 8
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

// A row's results.  Alternatives: the groups' maxima are dealt to 256 threads, and the top-th largest of what each thread holds
// is a value that at least `top` logits reach, so that only groups that reach it (a few more than top of them) hold any
// of the best; those are read again, 32 at a time, and their keys not below it gathered in LDS and ranked by counting the
// larger ones.  Where more keys come than the list holds (rows full of ties), the bound first rises to the top-th
// largest of the threads' own best keys of the batch: at most top threads, of 16 logits each, then have any above it.
// Grid (n), 512 threads, thread p for part p.
template <class E>
__global__ __launch_bounds__(kLpJoin) void logprobs_join_kernel(const E* __restrict__ x, int64_t ld, int vocab, int parts, int top,
                                                                const LogitSums* __restrict__ sums,
                                                                const float* __restrict__ gmax, const int32_t* __restrict__ tokens,
                                                                float* __restrict__ logp, float* __restrict__ entropy,
                                                                int32_t* __restrict__ top_ids, float* __restrict__ top_logp) {
  constexpr int R = 16 / sizeof(E), kHeld = 4;
  __shared__ uint64_t cand[kLpCand], best[kLpJoin];
  __shared__ __align__(16) unsigned order[256];
  __shared__ int group[kLpListed];
  __shared__ LogitSums red[kLpMaxParts / 64];
  __shared__ uint64_t s_bound;
  __shared__ unsigned s_least;
  __shared__ int s_cnt, s_n;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const size_t row = blockIdx.x;
  x += row * (size_t)ld;
  const int t = logp ? tokens[row] : -1;
  LogitSums s{-INFINITY, 0.f, 0.f};
  if (tid < parts) s = sums[row * parts + tid];
  const int groups = (vocab + kLpStep - 1) / kLpStep * kLpGroups;
  if (top) gmax += row * (size_t)groups;
  float held[kHeld], gm = -INFINITY;  // the groups tid + 256 i of the first 1024, and the largest of all of the thread's
  if (top && tid < 256) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = gmax[min(tid + 256 * i, groups - 1)];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) gm = tid + 256 * i < groups ? fmaxf(gm, held[i]) : gm;
    for (int g = tid + 256 * kHeld; g < groups; g += 256) gm = fmaxf(gm, gmax[g]);
    order[tid] = (unsigned)(cand_key(gm, 0) >> 32);
  }
  const float xt = t >= 0 && t < vocab ? to_f32(x[t]) : __builtin_nanf("");
  if (tid == 0) {
    s_cnt = s_n = 0;
    s_least = ~0u;
  }
  if (w < kLpMaxParts / 64) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const LogitSums y{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.a, o)};
      s = join(s, y);
    }
    if (lane == 0) red[w] = s;
  }
  __syncthreads();
  s = join(join(red[0], red[1]), join(red[2], red[3]));
  const float lz = s.m == -INFINITY ? __builtin_nanf("") : logf(s.z);
  if (tid == 0) {
    if (logp) logp[row] = (xt - s.m) - lz;
    if (entropy) entropy[row] = lz - s.a / s.z;
  }
  if (top == 0) return;
  // the smallest of the values with fewer than top larger ones is the top-th largest
  const int holders = min(groups, 256);
  if (tid < holders) {
    const unsigned mine = order[tid];
    int r = 0;
    for (int j = 0; j + 4 <= holders; j += 4) {  // groups come in fours
      const u32x4 o = *reinterpret_cast<const u32x4*>(order + j);
      r += (o[0] > mine) + (o[1] > mine) + (o[2] > mine) + (o[3] > mine);
    }
    if (r < top) atomicMin(&s_least, mine);
  }
  __syncthreads();
  // every key where fewer than top groups hold a logit above -inf
  const bool any = holders < top || s_least < 0x00800000u;
  const float least = any ? -INFINITY : cand_of((uint64_t)s_least << 32).v;
  uint64_t bound = 0;
  int cnt = 0;
  for (int g0 = 0; g0 < groups; g0 += kLpListed) {
    if (g0) {
      __syncthreads();
      if (tid == 0) s_n = 0;
      __syncthreads();
    }
    if (tid < 256) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int g = g0 + tid + 256 * i;
        const float m = g0 == 0 ? held[i] : gmax[min(g, groups - 1)];
        if (g < groups && (any || m >= least)) group[atomicAdd(&s_n, 1)] = g;
      }
    }
    __syncthreads();
    const int listed = s_n;
    for (int b = 0; b < listed; b += kLpJoin / 16) {
      const int at = b + (tid >> 4), g = group[min(at, listed - 1)], step = g / kLpGroups, ln = (g % kLpGroups) * 16 + (tid & 15);
      float v[kLpVals];
      if ((step + 1) * kLpStep <= vocab) {
#pragma unroll
        for (int k = 0; k < kLpVals / R; ++k) values_of<E, R>(load16(x + logit_at<E>(step, ln, k * R)), v + k * R);
      } else {
        load_ragged(x, step, ln, vocab, v);
      }
      uint64_t key[kLpVals], top_key = 0;
      int mine = 0;
#pragma unroll
      for (int i = 0; i < kLpVals; ++i) {
        const int c = logit_at<E>(step, ln, i);
        key[i] = at < listed && c < vocab && (any || v[i] >= least) ? logit_key(v[i], c) : 0;
        if (key[i] <= bound) key[i] = 0;
        mine += key[i] ? 1 : 0;
        top_key = key[i] > top_key ? key[i] : top_key;
      }
      __syncthreads();  // s_n has been read
      if (tid == 0) {
        s_n = 0;
        s_bound = bound;
      }
      best[tid] = top_key;
      __syncthreads();
      if (mine) atomicAdd(&s_n, mine);
      __syncthreads();
      const int all = s_n;
      if (all == 0) continue;
      if (cnt + all > kLpCand) {
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < kLpJoin; ++j) r += best[j] > top_key ? 1 : 0;
        if (top_key && r == top - 1) s_bound = top_key - 1;
        __syncthreads();
        bound = s_bound;
      }
#pragma unroll
      for (int i = 0; i < kLpVals; ++i)
        if (key[i] > bound) cand[atomicAdd(&s_cnt, 1)] = key[i];
      __syncthreads();
      cnt = s_cnt;
      if (cnt > 2 * kLogprobTop) {
        prune(cand, cnt, top, tid);
        cnt = top;
        bound = cand[top - 1];
        if (tid == 0) s_cnt = top;
      }
    }
  }
  __syncthreads();
  prune(cand, cnt, top, tid);
  if (tid < top) {
    const SpecCand c = cand_of(cand[tid]);
    top_ids[row * top + tid] = c.i;
    if (top_logp) top_logp[row * top + tid] = (c.v - s.m) - lz;
  }
}

// Parts of a row, `per` steps each: enough waves to fill the device.
static int logprob_parts(int n, int64_t vocab, int* per) {
  const int64_t steps = (vocab + kLpStep - 1) / kLpStep;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({steps, kLpMaxParts, 8192 / n}));
  const int64_t p = (steps + want - 1) / want;
  *per = (int)p;
  return (int)((steps + p - 1) / p);
}

size_t logprobs_work(int n, int64_t vocab, int top) {
  int per;
  const size_t parts = (size_t)n * logprob_parts(n, vocab, &per);
  const size_t groups = top ? (size_t)n * ((vocab + kLpStep - 1) / kLpStep) * kLpGroups : 0;
  return groups * sizeof(float) + parts * sizeof(LogitSums) + 16;
}

int logprobs(const void* logits, int64_t ld, int type, int n, int vocab, const int32_t* tokens, int top, float* logp, float* entropy,
             int32_t* top_ids, float* top_logp, void* work, hipStream_t s) {
  int per;
  const int parts = logprob_parts(n, vocab, &per);
  const size_t groups = (size_t)((vocab + kLpStep - 1) / kLpStep) * kLpGroups;
  LogitSums* sums = static_cast<LogitSums*>(work);
  float* gmax = reinterpret_cast<float*>(sums + (size_t)n * parts);
  return with_type(type, [&](auto* e) -> int {
    using E = std::remove_pointer_t<decltype(e)>;
    const E* x = static_cast<const E*>(logits);
    // rows beyond the grid's second dimension go in further launches
    for (int r0 = 0; r0 < n; r0 += std::min(65535, n - r0)) {
      logprobs_kernel<E><<<dim3((unsigned)parts, (unsigned)std::min(65535, n - r0)), 64, 0, s>>>(
          x + (size_t)r0 * ld, ld, vocab, per, sums + (size_t)r0 * parts, top ? gmax + r0 * groups : nullptr);
      DZ_HIP_CHECK(hipGetLastError());
    }
    // nor does a launch have 2^32 threads
    constexpr int kRows = 1 << 22;
    for (int r0 = 0; r0 < n; r0 += std::min(kRows, n - r0)) {
      const size_t t0 = (size_t)r0 * top;
      logprobs_join_kernel<E><<<(unsigned)std::min(kRows, n - r0), kLpJoin, 0, s>>>(
          x + (size_t)r0 * ld, ld, vocab, parts, top, sums + (size_t)r0 * parts, top ? gmax + r0 * groups : nullptr,
          logp ? tokens + r0 : nullptr, logp ? logp + r0 : nullptr, entropy ? entropy + r0 : nullptr, top ? top_ids + t0 : nullptr,
          top_logp ? top_logp + t0 : nullptr);
      DZ_HIP_CHECK(hipGetLastError());
    }
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
