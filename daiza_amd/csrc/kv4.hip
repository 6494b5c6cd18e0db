// kv4.hip — the key/value cache held in 4 bits (kv4.h): rows in and out, attention over it and eviction from it.
#include <math.h>

#include <algorithm>
#include <new>

#include "elem.h"
#include "kv4.h"

struct dz_kv4 {
  dz::Kv4View v;
  uint8_t* base = nullptr;
  int device = 0;
  int rows = 0;  // capacity asked for
  int len = 0;
};

namespace dz {

template <class F>
static int with_head_dim(int hd, F&& f) {
  switch (hd) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    default: return set_error(DZ_ERR_UNSUPPORTED, "4-bit cache: head_dim %d (64, 128 or 256)", hd);
  }
}

// ---------------------------------------------------------------- rows in and out

// One row of one head of keys (z = 0) or values (z = 1) per workgroup, a thread per dim: a block's 32 threads find its
// largest value, the codes meet in LDS and leave in the layout's words.  Grid (n, nkv, 2), HD threads.
template <int HD, class E>
__global__ __launch_bounds__(HD) void kv4_append_kernel(Kv4View c, int row0, const E* __restrict__ k, int64_t ldk,
                                                        const E* __restrict__ v, int64_t ldv) {
  constexpr int T = HD / 32;
  __shared__ uint8_t code[HD];
  const int d = threadIdx.x, g = blockIdx.y;
  const int64_t r = (int64_t)row0 + blockIdx.x;
  const bool values = blockIdx.z != 0;
  const float x = to_f32((values ? v + (size_t)blockIdx.x * ldv : k + (size_t)blockIdx.x * ldk)[(size_t)g * HD + d]);
  unsigned big = __float_as_uint(x) & 0x7FFFFFFFu;  // as whole numbers: a NaN is larger than every number
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) big = max(big, (unsigned)__shfl_xor((int)big, o));
  const int sb = kv4_scale_byte(__uint_as_float(big));
  code[d] = (uint8_t)kv4_code(x, sb);
  if ((d & 31) == 0) (values ? c.vs : c.ks)[g * c.scale_head() + (size_t)r * T + d / 32] = (uint8_t)sb;
  __syncthreads();
  if (!values) {
    if (d < HD / 8) {
      const int lk = d / T, b = d % T;
      unsigned w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= (unsigned)code[32 * b + 8 * lk + i] << (4 * i);
      *reinterpret_cast<unsigned*>(c.kc + g * c.code_head() + (size_t)r * (HD / 2) + 4 * d) = w;
    }
  } else if (d < 16) {
    uint8_t* p = c.vc + g * c.code_head() + kv4_value_offset<HD>(r, d);
    unsigned short* w = reinterpret_cast<unsigned short*>(p);
#pragma unroll
    for (int t = 0; t < T; t += 2) {
      const unsigned a = code[32 * t + 2 * d] | (unsigned)code[32 * t + 2 * d + 1] << 4;
      const unsigned b = code[32 * t + 32 + 2 * d] | (unsigned)code[32 * t + 33 + 2 * d] << 4;
      w[t / 2] = (unsigned short)(a | b << 8);
    }
  }
}

__device__ __forceinline__ float kv4_grid(unsigned code) {
  constexpr unsigned kHalves = 0xC8643210u;  // 0, 1, 2, 3, 4, 6, 8, 12 halves
  const float a = 0.5f * (float)((kHalves >> (4 * (code & 7u))) & 15u);
  return code & 8u ? -a : a;
}

// The values of rows start + blockIdx.x, f32 [kv head][n][HD].  Grid (n, nkv, 2), HD threads.
template <int HD>
__global__ __launch_bounds__(HD) void kv4_read_kernel(Kv4View c, int start, int n, float* __restrict__ k, float* __restrict__ v) {
  constexpr int T = HD / 32;
  const int d = threadIdx.x, g = blockIdx.y, t = d / 32, in = d % 32;
  const int64_t r = (int64_t)start + blockIdx.x;
  const bool values = blockIdx.z != 0;
  float* out = values ? v : k;
  if (!out) return;
  const size_t ch = g * c.code_head();
  unsigned byte;
  if (values) byte = c.vc[ch + kv4_value_offset<HD>(r, in / 2) + t];
  else byte = c.kc[ch + (size_t)r * (HD / 2) + 4 * ((in / 8) * T + t) + (in % 8) / 2];
  const unsigned code = (byte >> (4 * (d & 1))) & 15u;
  const unsigned sb = (values ? c.vs : c.ks)[g * c.scale_head() + (size_t)r * T + t];
  out[((size_t)g * n + blockIdx.x) * HD + d] = kv4_grid(code) * kv4_scale(sb);
}

int kv4_append(const Kv4View& c, int row0, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, int n, hipStream_t s) {
  return with_head_dim(c.hd, [&](auto D) {
    constexpr int HD = decltype(D)::value;
    return with_type(type, [&](auto* e) -> int {
      using E = std::remove_pointer_t<decltype(e)>;
      kv4_append_kernel<HD, E><<<dim3((unsigned)n, (unsigned)c.nkv, 2), HD, 0, s>>>(c, row0, (const E*)k, ldk, (const E*)v, ldv);
      DZ_HIP_CHECK(hipGetLastError());
      return DZ_OK;
    });
  });
}

int kv4_read(const Kv4View& c, int start, int n, float* k, float* v, hipStream_t s) {
  return with_head_dim(c.hd, [&](auto D) -> int {
    constexpr int HD = decltype(D)::value;
    kv4_read_kernel<HD><<<dim3((unsigned)n, (unsigned)c.nkv, 2), HD, 0, s>>>(c, start, n, k, v);
    DZ_HIP_CHECK(hipGetLastError());
    return DZ_OK;
  });
}

// ---------------------------------------------------------------- attention

// A (token, query head) per workgroup: tiles of 256 rows, a thread per row for the scores and per dim for the sums.
template <int HD, class E>
__global__ __launch_bounds__(256) void kv4_attend_simple_kernel(Kv4View c, int len, const E* __restrict__ q, int64_t ldq, int nq,
                                                                int n, float scale, float2* __restrict__ stats,
                                                                E* __restrict__ out, int64_t ldo) {
  constexpr int T = HD / 32;
  __shared__ float qs[HD], ps[256], red[4];
  const int i = blockIdx.x, h = blockIdx.y, g = h / (nq / c.nkv), tid = threadIdx.x;
  if (tid < HD) qs[tid] = to_f32(q[(size_t)i * ldq + (size_t)h * HD + tid]) * scale;
  const int seen = len - n + i + 1;
  const size_t ch = g * c.code_head(), sh = g * c.scale_head();
  float m = -INFINITY, l = 0.f, o = 0.f;
  __syncthreads();
  for (int p0 = 0; p0 < seen; p0 += 256) {
    const int r = p0 + tid;
    float sc = -INFINITY;
    if (r < seen) {
      sc = 0.f;
      const unsigned* kr = reinterpret_cast<const unsigned*>(c.kc + ch + (size_t)r * (HD / 2));
      for (int b = 0; b < T; ++b) {
        float a = 0.f;
        for (int lk = 0; lk < 4; ++lk) {
          const unsigned w = kr[lk * T + b];
          for (int j = 0; j < 8; ++j) a = __builtin_fmaf(kv4_grid((w >> (4 * j)) & 15u), qs[32 * b + 8 * lk + j], a);
        }
        sc = __builtin_fmaf(a, kv4_scale(c.ks[sh + (size_t)r * T + b]), sc);
      }
    }
    float bm = sc;
    for (int x = 1; x < 64; x <<= 1) bm = fmaxf(bm, __shfl_xor(bm, x));
    if ((tid & 63) == 0) red[tid >> 6] = bm;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float al = m == -INFINITY ? 0.f : expf(m - mn);
    const float p = r < seen ? expf(sc - mn) : 0.f;
    ps[tid] = p;
    float sum = wave_sum(p);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    l = l * al + ((red[0] + red[1]) + (red[2] + red[3]));
    m = mn;
    if (tid < HD) {
      const int t = tid / 32, in = tid % 32;
      o *= al;
      for (int j = 0; j < min(256, seen - p0); ++j) {
        const unsigned byte = c.vc[ch + kv4_value_offset<HD>(p0 + j, in / 2) + t];
        const float x = kv4_grid((byte >> (4 * (tid & 1))) & 15u) * kv4_scale(c.vs[sh + (size_t)(p0 + j) * T + t]);
        o = __builtin_fmaf(ps[j], x, o);
      }
    }
    __syncthreads();
  }
  if (tid < HD) out[(size_t)i * ldo + (size_t)h * HD + tid] = from_f32<E>(o / l);
  if (stats && tid == 0) stats[(size_t)i * nq + h] = make_float2(m, l);
}

// weights[g][r] += the softmax weights that row r received, a thread per row, queries and heads in order.
template <int HD, class E>
__global__ __launch_bounds__(256) void kv4_weights_simple_kernel(Kv4View c, int len, const E* __restrict__ q, int64_t ldq, int nq,
                                                                 int n, float scale, const float2* __restrict__ stats,
                                                                 float* __restrict__ weights, int64_t ldw) {
  constexpr int T = HD / 32;
  __shared__ float qs[HD];
  const int g = blockIdx.y, grp = nq / c.nkv, tid = threadIdx.x, r = (int)blockIdx.x * 256 + tid;
  const size_t ch = g * c.code_head(), sh = g * c.scale_head();
  float acc = 0.f;
  for (int i = 0; i < n; ++i)
    for (int h = g * grp; h < (g + 1) * grp; ++h) {
      __syncthreads();
      if (tid < HD) qs[tid] = to_f32(q[(size_t)i * ldq + (size_t)h * HD + tid]) * scale;
      __syncthreads();
      if (r <= len - n + i) {
        float sc = 0.f;
        const unsigned* kr = reinterpret_cast<const unsigned*>(c.kc + ch + (size_t)r * (HD / 2));
        for (int b = 0; b < T; ++b) {
          float a = 0.f;
          for (int lk = 0; lk < 4; ++lk) {
            const unsigned w = kr[lk * T + b];
            for (int j = 0; j < 8; ++j) a = __builtin_fmaf(kv4_grid((w >> (4 * j)) & 15u), qs[32 * b + 8 * lk + j], a);
          }
          sc = __builtin_fmaf(a, kv4_scale(c.ks[sh + (size_t)r * T + b]), sc);
        }
        const float2 st = stats[(size_t)i * nq + h];
        acc += expf(sc - st.x) / st.y;
      }
    }
  if (r < len) weights[(size_t)g * ldw + r] += acc;
}

size_t kv4_attend_work(int hd, int n_head, int n) { return (size_t)n * n_head * sizeof(float2); }

int kv4_attend(const Kv4View& c, int len, const void* q, int64_t ldq, int type, int n_head, int n, float scale, float* weights,
               int64_t ldw, void* out, int64_t ldo, void* work, hipStream_t s) {
  return with_head_dim(c.hd, [&](auto D) {
    constexpr int HD = decltype(D)::value;
    return with_type(type, [&](auto* e) -> int {
      using E = std::remove_pointer_t<decltype(e)>;
      float2* stats = static_cast<float2*>(work);
      kv4_attend_simple_kernel<HD, E><<<dim3((unsigned)n, (unsigned)n_head), 256, 0, s>>>(
          c, len, (const E*)q, ldq, n_head, n, scale, weights ? stats : nullptr, (E*)out, ldo);
      DZ_HIP_CHECK(hipGetLastError());
      if (weights) {
        kv4_weights_simple_kernel<HD, E><<<dim3((unsigned)((len + 255) / 256), (unsigned)c.nkv), 256, 0, s>>>(
            c, len, (const E*)q, ldq, n_head, n, scale, stats, weights, ldw);
        DZ_HIP_CHECK(hipGetLastError());
      }
      return DZ_OK;
    });
  });
}

// ---------------------------------------------------------------- eviction

// Weights as unsigned words in their order: NaN below every number, the zeros of either sign alike.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// kept[g] of head g: the `take` rows of [0, old) with the largest keys (the lower row first among equal ones), then the rows
// [old, old + recent), in ascending order.  The key of the take-th largest is found byte by byte from the top
// (a histogram of the keys that share the bytes found so far); then every wave counts and writes its span in order.
// Grid (nkv), 1024 threads.
__global__ __launch_bounds__(1024) void kv4_select_kernel(const float* __restrict__ w, int64_t ldw, int old, int take, int recent,
                                                          int32_t* __restrict__ kept) {
  __shared__ unsigned hist[256], wsum[16][2], s_prefix, s_left;
  const unsigned tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
  const int g = blockIdx.x, m = take + recent;
  w += (size_t)g * ldw;
  kept += (size_t)g * m;
  for (int i = (int)tid; i < recent; i += 1024) kept[take + i] = old + i;
  if (take == 0) return;
  unsigned prefix = 0, left = (unsigned)take;  // the key's bytes so far; how many rows come from the keys that share them
  for (int sh = 24; sh >= 0; sh -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = (int)tid; i < old; i += 1024) {
      const unsigned k = weight_key(w[i]);
      if (sh == 24 || (k >> (sh + 8)) == (prefix >> (sh + 8))) atomicAdd(&hist[(k >> sh) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned b = 255, seen = 0;
      while (seen + hist[b] < left) seen += hist[b--];
      s_prefix = prefix | b << sh;
      s_left = left - seen;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    __syncthreads();
  }
  // rows above the key, and the first `left` rows at it
  const int span = (old + 1023) / 1024 * 64, b0 = (int)wv * span, b1 = min(old, b0 + span);
  unsigned above = 0, at = 0;
  for (int i = b0; i < b1; i += 64) {
    const int r = i + (int)lane;
    const unsigned k = r < b1 ? weight_key(w[r]) : 0u;
    above += (unsigned)__popcll(__ballot(r < b1 && k > prefix));
    at += (unsigned)__popcll(__ballot(r < b1 && k == prefix));
  }
  if (lane == 0) {
    wsum[wv][0] = above;
    wsum[wv][1] = at;
  }
  __syncthreads();
  above = at = 0;
  for (unsigned i = 0; i < wv; ++i) {
    above += wsum[i][0];
    at += wsum[i][1];
  }
  for (int i = b0; i < b1; i += 64) {
    const int r = i + (int)lane;
    const unsigned k = r < b1 ? weight_key(w[r]) : 0u;
    const unsigned long long ba = __ballot(r < b1 && k > prefix), bt = __ballot(r < b1 && k == prefix);
    const unsigned long long below = (1ull << lane) - 1;
    const unsigned ra = above + (unsigned)__popcll(ba & below), rt = at + (unsigned)__popcll(bt & below);
    if (r < b1 && (k > prefix || (k == prefix && rt < left))) kept[ra + min(rt, left)] = r;
    above += (unsigned)__popcll(ba);
    at += (unsigned)__popcll(bt);
  }
}

// Row kept[g][i] of c -> row i of dst, with its weight.  Grid (ceil(m / 4), nkv), 256 threads, a wave per row.
template <int HD>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Kv4View c, Kv4View dst, const int32_t* __restrict__ kept, int m,
                                                         const float* __restrict__ w, int64_t ldw, float* __restrict__ dw,
                                                         int64_t ld_dw) {
  constexpr int T = HD / 32;
  const int g = blockIdx.y, i = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= m) return;
  const int64_t r = kept[(size_t)g * m + i];
  typedef uint8_t bytes __attribute__((ext_vector_type(T)));
  if (lane < HD / 8)
    reinterpret_cast<unsigned*>(dst.kc + g * dst.code_head() + (size_t)i * (HD / 2))[lane] =
        reinterpret_cast<const unsigned*>(c.kc + g * c.code_head() + (size_t)r * (HD / 2))[lane];
  else if (lane < HD / 8 + 16) {
    const int ln = lane - HD / 8;
    *reinterpret_cast<bytes*>(dst.vc + g * dst.code_head() + kv4_value_offset<HD>(i, ln)) =
        *reinterpret_cast<const bytes*>(c.vc + g * c.code_head() + kv4_value_offset<HD>(r, ln));
  } else if (lane == 48)
    *reinterpret_cast<bytes*>(dst.ks + g * dst.scale_head() + (size_t)i * T) =
        *reinterpret_cast<const bytes*>(c.ks + g * c.scale_head() + (size_t)r * T);
  else if (lane == 49)
    *reinterpret_cast<bytes*>(dst.vs + g * dst.scale_head() + (size_t)i * T) =
        *reinterpret_cast<const bytes*>(c.vs + g * c.scale_head() + (size_t)r * T);
  else if (lane == 50 && dw)
    dw[(size_t)g * ld_dw + i] = w[(size_t)g * ldw + r];
}

int kv4_evict(const Kv4View& c, int len, const float* weights, int64_t ldw, int keep, int recent, const Kv4View& dst,
              float* dst_weights, int64_t ld_dst, int32_t* kept, hipStream_t s) {
  const int m = std::min(keep, len);
  if (m == 0) return DZ_OK;
  recent = std::min(recent, len);
  kv4_select_kernel<<<dim3((unsigned)c.nkv), 1024, 0, s>>>(weights, ldw, len - recent, m - recent, recent, kept);
  DZ_HIP_CHECK(hipGetLastError());
  return with_head_dim(c.hd, [&](auto D) -> int {
    constexpr int HD = decltype(D)::value;
    kv4_gather_kernel<HD><<<dim3((unsigned)((m + 3) / 4), (unsigned)c.nkv), 256, 0, s>>>(c, dst, kept, m, weights, ldw,
                                                                                          dst_weights, ld_dst);
    DZ_HIP_CHECK(hipGetLastError());
    return DZ_OK;
  });
}

// Makes a cache's device current while a call runs.
struct OnDevice {
  int was = -1;
  int rc = DZ_OK;
  explicit OnDevice(int device) { rc = enter(device); }
  int enter(int device) {
    int cur = 0;
    DZ_HIP_CHECK(hipGetDevice(&cur));
    if (cur == device) return DZ_OK;
    DZ_HIP_CHECK(hipSetDevice(device));
    was = cur;
    return DZ_OK;
  }
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

}  // namespace dz

// ---------------------------------------------------------------- C ABI

using namespace dz;

extern "C" {

int dz_kv4_create(int kv_heads, int head_dim, int capacity, dz_kv4** out) {
  if (!out) return set_error(DZ_ERR_MODEL, "null argument");
  if (kv_heads < 1 || kv_heads > 4096) return set_error(DZ_ERR_TENSOR, "4-bit cache: %d kv heads", kv_heads);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(DZ_ERR_UNSUPPORTED, "4-bit cache: head_dim %d (64, 128 or 256)", head_dim);
  if (capacity < 1 || capacity > (1 << 30)) return set_error(DZ_ERR_TENSOR, "4-bit cache: capacity %d", capacity);
  if (int rc = ensure_device()) return rc;
  dz_kv4* c = new (std::nothrow) dz_kv4();
  if (!c) return set_error(DZ_ERR_MODEL, "out of memory");
  const int cap = (capacity + kKv4Tile - 1) / kKv4Tile * kKv4Tile;
  const size_t bytes = kv4_bytes(kv_heads, head_dim, cap);
  hipError_t e = hipGetDevice(&c->device);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&c->base), bytes);
  // zeros: a tile's rows past the last one are read (and masked), so they must stand for numbers
  if (e == hipSuccess) e = hipMemset(c->base, 0, bytes);
  if (e == hipSuccess) e = hipDeviceSynchronize();
  if (e != hipSuccess) {
    if (c->base) (void)hipFree(c->base);
    delete c;
    return set_error(DZ_ERR_DEVICE, "4-bit cache of %zu bytes: %s", bytes, hipGetErrorString(e));
  }
  c->v = kv4_carve(c->base, kv_heads, head_dim, cap);
  c->rows = capacity;
  *out = c;
  return DZ_OK;
}

int dz_kv4_free(dz_kv4* c) {
  if (!c) return DZ_OK;
  OnDevice on(c->device);
  (void)hipFree(c->base);  // waits for the work on it
  delete c;
  return DZ_OK;
}

int dz_kv4_len(const dz_kv4* c) { return c ? c->len : -1; }

int dz_kv4_truncate(dz_kv4* c, int len) {
  if (!c) return set_error(DZ_ERR_MODEL, "null cache");
  if (len >= c->len) return DZ_OK;
  if (len < 0) return set_error(DZ_ERR_TENSOR, "truncate to %d", len);
  c->len = len;
  return DZ_OK;
}

int dz_kv4_append_dev(dz_kv4* c, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, int n, void* stream) {
  if (!c || (n && (!k || !v))) return set_error(DZ_ERR_MODEL, "null argument");
  if (n < 0) return set_error(DZ_ERR_TENSOR, "append of %d rows", n);
  const int64_t row = (int64_t)c->v.nkv * c->v.hd;
  if (ldk < row || ldv < row) return set_error(DZ_ERR_TENSOR, "append: row strides %lld, %lld under a row's %lld", (long long)ldk,
                                               (long long)ldv, (long long)row);
  if (n > c->rows - c->len) return set_error(DZ_ERR_TENSOR, "append: cache full (%d + %d > %d rows)", c->len, n, c->rows);
  int rc = check_type(type);
  if (rc || n == 0) return rc;
  OnDevice on(c->device);
  if ((rc = on.rc) || (rc = check_array(k, type_size(type), c->device, "k")) || (rc = check_array(v, type_size(type), c->device, "v")))
    return rc;
  rc = kv4_append(c->v, c->len, k, ldk, v, ldv, type, n, static_cast<hipStream_t>(stream));
  if (rc == DZ_OK) c->len += n;
  return rc;
}

int dz_kv4_read_dev(const dz_kv4* c, int start, int n, float* k, float* v, void* stream) {
  if (!c) return set_error(DZ_ERR_MODEL, "null cache");
  if (start < 0 || n < 0 || n > c->len - start)
    return set_error(DZ_ERR_TENSOR, "read of rows [%d, %d + %d) of %d", start, start, n, c->len);
  if (n == 0 || (!k && !v)) return DZ_OK;
  OnDevice on(c->device);
  int rc = on.rc;
  if (rc || (k && (rc = check_array(k, 4, c->device, "k"))) || (v && (rc = check_array(v, 4, c->device, "v")))) return rc;
  return kv4_read(c->v, start, n, k, v, static_cast<hipStream_t>(stream));
}

size_t dz_kv4_attend_work_bytes(const dz_kv4* c, int n_head, int n) {
  return !c || n_head < 1 || n < 1 ? 0 : kv4_attend_work(c->v.hd, n_head, n);
}

int dz_kv4_attend_dev(const dz_kv4* c, const void* q, int64_t ldq, int type, int n_head, int n, float scale, float* weights,
                      int64_t ldw, void* out, int64_t ldo, void* work, void* stream) {
  if (!c || !q || !out || !work) return set_error(DZ_ERR_MODEL, "null argument");
  if (n_head < 1 || n_head > 65535 || n_head % c->v.nkv)
    return set_error(DZ_ERR_TENSOR, "attend: %d heads on %d kv heads", n_head, c->v.nkv);
  if (n < 1 || n > c->len) return set_error(DZ_ERR_TENSOR, "attend: %d queries over %d rows", n, c->len);
  int rc = check_type(type);
  if (rc) return rc;
  const int64_t row = (int64_t)n_head * c->v.hd;
  if (ldq < row || ldo < row) return set_error(DZ_ERR_TENSOR, "attend: row strides %lld, %lld under a row's %lld", (long long)ldq,
                                               (long long)ldo, (long long)row);
  if (weights && ldw < c->len) return set_error(DZ_ERR_TENSOR, "attend: weights of %lld rows, %d held", (long long)ldw, c->len);
  OnDevice on(c->device);
  if ((rc = on.rc) || (rc = check_array(q, type_size(type), c->device, "q")) ||
      (rc = check_array(out, type_size(type), c->device, "out")) || (rc = check_array(work, 16, c->device, "work")) ||
      (weights && (rc = check_array(weights, 4, c->device, "weights"))))
    return rc;
  return kv4_attend(c->v, c->len, q, ldq, type, n_head, n, scale, weights, ldw, out, ldo, work, static_cast<hipStream_t>(stream));
}

int dz_kv4_evict_dev(const dz_kv4* c, const float* weights, int64_t ldw, int keep, int recent, dz_kv4* dst, float* dst_weights,
                     int64_t ld_dst, int32_t* kept, void* stream) {
  if (!c || !dst) return set_error(DZ_ERR_MODEL, "null argument");
  if (c == dst) return set_error(DZ_ERR_TENSOR, "evict: the rows that stay go to another cache");
  if (c->v.nkv != dst->v.nkv || c->v.hd != dst->v.hd || c->device != dst->device)
    return set_error(DZ_ERR_TENSOR, "evict: the caches' shapes or devices differ");
  if (recent < 0 || keep < recent) return set_error(DZ_ERR_TENSOR, "evict: keep %d, of which %d recent", keep, recent);
  const int m = std::min(keep, c->len);
  if (m && (!weights || !kept)) return set_error(DZ_ERR_MODEL, "null argument");
  if (m > dst->rows) return set_error(DZ_ERR_TENSOR, "evict: %d rows into a cache for %d", m, dst->rows);
  if (m && (ldw < c->len || (dst_weights && ld_dst < m))) return set_error(DZ_ERR_TENSOR, "evict: weights' row stride under the rows held");
  OnDevice on(c->device);
  int rc = on.rc;
  if (m && (rc || (rc = check_array(weights, 4, c->device, "weights")) || (rc = check_array(kept, 4, c->device, "kept")) ||
            (dst_weights && (rc = check_array(dst_weights, 4, c->device, "dst_weights")))))
    return rc;
  rc = kv4_evict(c->v, c->len, weights, ldw, keep, recent, dst->v, dst_weights, ld_dst, kept, static_cast<hipStream_t>(stream));
  if (rc == DZ_OK) dst->len = m;
  return rc;
}

}  // extern "C"
