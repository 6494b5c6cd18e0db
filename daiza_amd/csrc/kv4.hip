// kv4.hip — the key/value cache held in 4 bits (kv4.h): rows in and out, attention over it and eviction from it.
#include <math.h>

#include <algorithm>
#include <mutex>
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

// Four consecutive elements from an address of the element's own alignment.
template <class E>
__device__ __forceinline__ void load4(const E* p, float (&x)[4]) {
  struct __attribute__((packed, aligned(sizeof(E)))) Raw {
    E e[4];
  };
  const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32(r.e[i]);
}

constexpr int kKv4RowThreads = 256;
template <int HD>
constexpr int kv4_wg_rows() { return kKv4RowThreads / (HD / 4); }

// Rows of keys (z = 0) or values (z = 1) of a head into the cache, a thread per four dims: the eight threads of a block
// find its largest value; a thread's four codes are half a word of keys, or a byte of values for each of two lanes.
// Bound by the rows read, at 4 x 256: 1024 rows 5.1 us (8.4 MB in, 1.1 MB out), 32768 rows 89 us (3.4 TB/s; the codes are
// stores of one and two bytes); one row 2.9 us, a launch.
// Grid (ceil(n / kv4_wg_rows), nkv, 2), 256 threads.
template <int HD, class E>
__global__ __launch_bounds__(kKv4RowThreads) void kv4_append_kernel(Kv4View c, int row0, int n, const E* __restrict__ k, int64_t ldk,
                                                                    const E* __restrict__ v, int64_t ldv) {
  constexpr int T = HD / 32, D4 = HD / 4;
  const int a = (int)threadIdx.x % D4, g = blockIdx.y, b = a / 8;
  const int64_t i = (int64_t)blockIdx.x * kv4_wg_rows<HD>() + threadIdx.x / D4, r = row0 + i;
  if (i >= n) return;  // all lanes of a block at once
  const bool values = blockIdx.z != 0;
  float x[4];
  load4((values ? v + (size_t)i * ldv : k + (size_t)i * ldk) + (size_t)g * HD + 4 * a, x);
  unsigned big = 0;  // as whole numbers: a NaN is larger than every number
#pragma unroll
  for (int j = 0; j < 4; ++j) big = max(big, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) big = max(big, (unsigned)__shfl_xor((int)big, o));
  const int sb = kv4_scale_byte(__uint_as_float(big));
  unsigned code = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) code |= kv4_code(x[j], sb) << (4 * j);
  if (a % 8 == 0) {
    (values ? c.vs : c.ks)[g * c.scale_head() + (size_t)r * T + b] = (uint8_t)sb;
    if (sb == 255) c.bad[(size_t)g * (c.cap / kKv4Tile) + r / kKv4Tile] = 1;
  }
  if (!values) {
    uint8_t* p = c.kc + g * c.code_head() + (size_t)r * (HD / 2) + 2 * a;
    *reinterpret_cast<unsigned short*>(p) = (unsigned short)code;
  } else {
    uint8_t* p = c.vc + g * c.code_head() + kv4_value_offset<HD>(r, 2 * (a % 8)) + b;
    p[0] = (uint8_t)code;
    p[16] = (uint8_t)(code >> 8);
  }
}

__device__ __forceinline__ float kv4_grid(unsigned code) {
  constexpr unsigned kHalves = 0xC8643210u;  // 0, 1, 2, 3, 4, 6, 8, 12 halves
  const float a = 0.5f * (float)((kHalves >> (4 * (code & 7u))) & 15u);
  return code & 8u ? -a : a;
}

// The values of rows start .. start + n, f32 [kv head][n][HD], a thread per four dims.  Bound by the stores: 8192 rows of 4 x 256
// 15.2 us (67 MB, 4.4 TB/s).
// Grid (ceil(n / kv4_wg_rows), nkv, 2), 256 threads.
template <int HD>
__global__ __launch_bounds__(kKv4RowThreads) void kv4_read_kernel(Kv4View c, int start, int n, float* __restrict__ k,
                                                                  float* __restrict__ v) {
  constexpr int T = HD / 32, D4 = HD / 4;
  const int a = (int)threadIdx.x % D4, g = blockIdx.y, b = a / 8;
  const int64_t i = (int64_t)blockIdx.x * kv4_wg_rows<HD>() + threadIdx.x / D4, r = start + i;
  const bool values = blockIdx.z != 0;
  float* out = values ? v : k;
  if (!out || i >= n) return;
  unsigned code;
  if (values) {
    const uint8_t* p = c.vc + g * c.code_head() + kv4_value_offset<HD>(r, 2 * (a % 8)) + b;
    code = p[0] | (unsigned)p[16] << 8;
  } else {
    code = *reinterpret_cast<const unsigned short*>(c.kc + g * c.code_head() + (size_t)r * (HD / 2) + 2 * a);
  }
  const float s = kv4_scale((values ? c.vs : c.ks)[g * c.scale_head() + (size_t)r * T + b]);
  struct __attribute__((packed, aligned(4))) Four {
    float x[4];
  };
  Four y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y.x[j] = kv4_grid((code >> (4 * j)) & 15u) * s;
  *reinterpret_cast<Four*>(out + ((size_t)g * n + i) * HD + 4 * a) = y;
}

int kv4_append(const Kv4View& c, int row0, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, int n, hipStream_t s) {
  return with_head_dim(c.hd, [&](auto D) {
    constexpr int HD = decltype(D)::value, W = kv4_wg_rows<HD>();
    return with_type(type, [&](auto* e) -> int {
      using E = std::remove_pointer_t<decltype(e)>;
      kv4_append_kernel<HD, E><<<dim3((unsigned)((n + W - 1) / W), (unsigned)c.nkv, 2), kKv4RowThreads, 0, s>>>(
          c, row0, n, (const E*)k, ldk, (const E*)v, ldv);
      DZ_HIP_CHECK(hipGetLastError());
      return DZ_OK;
    });
  });
}

int kv4_read(const Kv4View& c, int start, int n, float* k, float* v, hipStream_t s) {
  return with_head_dim(c.hd, [&](auto D) -> int {
    constexpr int HD = decltype(D)::value, W = kv4_wg_rows<HD>();
    kv4_read_kernel<HD><<<dim3((unsigned)((n + W - 1) / W), (unsigned)c.nkv, 2), kKv4RowThreads, 0, s>>>(c, start, n, k, v);
    DZ_HIP_CHECK(hipGetLastError());
    return DZ_OK;
  });
}

// ---------------------------------------------------------------- attention

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A query is carried as a sum of bf16 values that holds every bit of its type; a probability as enough of them that what
// is lost lies beneath the rounding of the output: 24 bits for f32, 16 for the 16-bit types (2^-17 against 2^-11 and 2^-8).
template <class E>
struct Parts;
template <>
struct Parts<float> {
  static constexpr int q = 3, p = 3;
};
template <>
struct Parts<__half> {
  static constexpr int q = 2, p = 2;
};
template <>
struct Parts<__hip_bfloat16> {
  static constexpr int q = 1, p = 2;
};

// The high halves of two words as one (a in the low half): two bf16 values cut from two f32.
__device__ __forceinline__ unsigned high_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// x minus its high 16 bits, exact.
__device__ __forceinline__ float rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }

// The nearest bf16 values of two f32.
__device__ __forceinline__ unsigned near_halves(float a, float b) {
  typedef float f32x2v __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2v{a, b}, bf16x2));
}

// Eight f32 values as N bf16 operands whose sum they are to 8 N bits: the last part takes the nearest value, so that where
// bits are lost (probabilities as two parts) the errors are of either sign.  Cut instead, all of a row's probabilities were too
// small beside their sum, and f16 outputs with them by 5.4e-6 (2^-17.5) on average; the times are the same.
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&out)[N]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[k][i] = N == 2 && k == 1 ? near_halves(r[2 * i], r[2 * i + 1]) : high_halves(r[2 * i], r[2 * i + 1]);
    if (k + 1 < N)
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = rest(r[i]);
  }
}

// Scale byte `i` of a word as the f32 operand of the conversions, which take its exponent bits alone.
__device__ __forceinline__ float scale_of(unsigned w, int i) {
  return __uint_as_float(i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1);
}
template <int SEL>
__device__ __forceinline__ unsigned fp4_pair(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
__device__ __forceinline__ unsigned fp4_pair(unsigned w, float scale, int sel) {
  switch (sel) {
    case 0: return fp4_pair<0>(w, scale);
    case 1: return fp4_pair<1>(w, scale);
    case 2: return fp4_pair<2>(w, scale);
    default: return fp4_pair<3>(w, scale);
  }
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A lane's words of a tile of 32 rows.
template <int HD>
struct KeyWords {
  static constexpr int T = HD / 32, G = T >= 4 ? T / 4 : 1;  // words; blocks that the lane has a part of (half of one at 64)
  unsigned code[2][T];  // rows 16h + ln: dims lk·HD/4 + 8b .. +7
  unsigned scale[2];    // their blocks' bytes
  __device__ __forceinline__ void load(const uint8_t* kc, const uint8_t* ks, int64_t row, int ln, int lk) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t r = row + 16 * h + ln;
      const unsigned* p = reinterpret_cast<const unsigned*>(kc + (size_t)r * (HD / 2) + 4 * T * lk);
#pragma unroll
      for (int b = 0; b < T; ++b) code[h][b] = p[b];
      const uint8_t* q = ks + (size_t)r * T + (T >= 4 ? lk * G : lk / 2);
      scale[h] = G == 2 ? *reinterpret_cast<const unsigned short*>(q) : *q;
    }
  }
  // Part b of the rows 16h + ln as a bf16 operand: a lane's dims lk·HD/4 + 8b .. +7, for the 16x16x32 instruction.
  __device__ __forceinline__ u32x4 operand(int h, int b) const {
    const float s = scale_of(scale[h], b / 4);
    const unsigned w = code[h][b];
    return u32x4{fp4_pair<0>(w, s), fp4_pair<1>(w, s), fp4_pair<2>(w, s), fp4_pair<3>(w, s)};
  }
  // Bit r of the result: row 16h + r has a block that is not a number.
  __device__ __forceinline__ unsigned bad_rows(int h) const {
    const unsigned long long m = __ballot((scale[h] & 255u) == 255u || (G == 2 && scale[h] >> 8 == 255u));
    const unsigned v = (unsigned)m | (unsigned)(m >> 32);
    return (v | v >> 16) & 0xFFFFu;  // the four lanes of a row have a quarter each
  }
};
template <int HD>
struct ValueWords {
  static constexpr int T = HD / 32;
  unsigned code[2 * T];      // byte j·T + t
  unsigned scale[2][T];      // rows 16h + 4lk + i: byte i·T + t
  __device__ __forceinline__ void load(const uint8_t* vc, const uint8_t* vs, int64_t row, int lane) {
    const uint8_t* p = vc + (size_t)row * (HD / 2) + 16 * lane;
#pragma unroll
    for (int c = 0; c < T / 2; ++c) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(p + 1024 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) code[4 * c + i] = w[i];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned* q = reinterpret_cast<const unsigned*>(vs + (size_t)(row + 16 * h + 4 * (lane >> 4)) * T);
#pragma unroll
      for (int i = 0; i < T; ++i) scale[h][i] = q[i];
    }
  }
  // Dims 32t + 2ln and + 1 of slot j's row.
  __device__ __forceinline__ unsigned pair(int j, int t) const {
    const int o = j * T + t, s = (j & 3) * T + t;
    return fp4_pair(code[o / 4], scale_of(scale[j >> 2][s / 4], s % 4), o % 4);
  }
  // The operands of dims 32t + 2ln (lo) and 32t + 2ln + 1 (hi) over the lane's eight slots.
  __device__ __forceinline__ void operands(int t, u32x4& lo, u32x4& hi) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned a = pair(2 * i, t), b = pair(2 * i + 1, t);
      lo[i] = __builtin_amdgcn_perm(b, a, 0x05040100u);
      hi[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    }
  }
  // Blocks that are not numbers count as zeros from here on (their codes are zeros); first[t] becomes the first row of
  // the tile, at `row`, with such a block t, if that is earlier.
  __device__ __forceinline__ void take_bad(int row, int lk, int (&first)[T]) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      int at = 0x7FFFFFFF;
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        const int s = (j & 3) * T + t;
        if (((scale[j >> 2][s / 4] >> (8 * (s % 4))) & 255u) == 255u) at = row + 16 * (j >> 2) + 4 * lk + (j & 3);
      }
      at = min(at, __shfl_xor(at, 16));
      at = min(at, __shfl_xor(at, 32));
      first[t] = min(first[t], at);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < T; ++i)  // bytes of 255 become 127
        scale[h][i] ^= ((scale[h][i] & 0x7F7F7F7Fu) + 0x01010101u) & scale[h][i] & 0x80808080u;
  }
};

// The query rows of a workgroup, row ρ = token · grp + head of the group, as operands in LDS: [row tile][b][part]
// [lane][16 B], lane 16·lk + ln holding dims lk·HD/4 + 8b .. +7 of the tile's row ln.  Requested and stored apart, for
// other loads to be on their way in between.
template <int HD, class E, int TILES, int NT>
struct QueryStage {
  static constexpr int T = HD / 32, QP = Parts<E>::q, N = (TILES * T * 64 + NT - 1) / NT;
  E x[N][8];
  __device__ __forceinline__ void load(const E* __restrict__ q, int64_t ldq, int head0, int grp, int row0, int rows, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = tid + i * NT, lane = u & 63, b = (u >> 6) % T, tile = (u >> 6) / T;
      const int rho = min(row0 + 16 * tile + (lane & 15), rows - 1);  // a row past the last is the last one again: not used
      struct __attribute__((packed, aligned(sizeof(E)))) Raw {
        E e[8];
      };
      const Raw r = *reinterpret_cast<const Raw*>(q + (size_t)(rho / grp) * ldq + (size_t)(head0 + rho % grp) * HD +
                                                  (HD / 4) * (lane >> 4) + 8 * b);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = r.e[j];
    }
  }
  __device__ __forceinline__ void store(u32x4* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = tid + i * NT, lane = u & 63, b = (u >> 6) % T, tile = (u >> 6) / T;
      if (N * NT != TILES * T * 64 && u >= TILES * T * 64) break;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32(x[i][j]);
      u32x4 part[QP];
      split8<QP>(v, part);
#pragma unroll
      for (int k = 0; k < QP; ++k) lds[((tile * T + b) * QP + k) * 64 + lane] = part[k];
    }
  }
};

constexpr float kLog2e = 1.4426950408889634f;

// Where a call's results go: the output itself (nch = 1) or a record (m, l, o[HD]) per row and chunk of positions.
struct AttendOut {
  float* rec = nullptr;         // [n][nq][nch][2 + HD]
  float2* stats = nullptr;      // [n][nq] (m, l), or null
  const float* gate = nullptr;  // [n][nq][HD]: the output times its sigmoid, or null
  float* scores = nullptr;      // [n][nq][cap]: the scores (few rows, for the weights), or null
  // Element d of row `row` (HD elements each).
  template <class E, int HD>
  __device__ __forceinline__ E value(float o, float l, size_t row, int d) const {
    float y = o / l;
    if (gate) y *= 1.0f / (1.0f + expf(-gate[row * HD + d]));
    return from_f32<E>(y);
  }
};

// M matrix instructions with V vector instructions spread among them.
template <int M, int V>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, (V + M - 1) / M, 0);
  }
}

// The largest (sum) of x over the four lanes ln, ln + 16, ln + 32, ln + 48.
__device__ __forceinline__ float max_over_lk(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_over_lk(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Causal attention of the n·grp query rows of a key/value head on the matrix cores, in one pass with the running maximum m and
// sum l of each row's softmax.  Scores as S^T = K · Q^T, the operand of the queries from LDS; lane (ln, lk) gets the scores of
// row ln at positions 4lk + i and 16 + 4lk + i of the tile, which are, in that order, its part of the operand P of O += P · V.
// Dequantising is exact, queries and probabilities are sums of bf16 operands (Parts): products are those of f32 values, and
// the sums f32.
//
// A workgroup has RT tiles of 16 rows and PS waves for each, which take the chunk's tiles of 32 positions in turn, each a
// tile ahead with its loads; their results meet in LDS at the end.  Two waves a SIMD, so that one's dequantising runs beside
// the other's matrix instructions.  At 24 heads on 4 x 256, f32:
//   RT = 1 (up to 192 rows)  bound by latency to about 16384 positions (one token behind 4096: 8.0 us and the merge's 2.7)
//                            and by the cache's bytes beyond (262144: 62 us, 4.6 TB/s, of 285 MB)
//   RT = 4                   bound by the vector instructions (of which a wave dequantises its values with about 190 a tile, 32
//                            positions) and the matrix instructions (96 of 6.7 ns a tile: three parts of Q, three of P) that
//                            do not run beside each other well enough: 1.7 us a tile.  333 tokens behind 7000 positions, 59
//                            GFLOP, 182 to 190 us.  f32 queries as six 6-bit digits of the 16x16x128 instruction, which take the keys
//                            as they stand, took 169 us, but hold a query to 2^-29 of the largest of each 32 dims: beside
//                            an outlier that meets keys of 0 the other dims lose bits that an f32 product has.
// Tiles with blocks that are not numbers, and calls that keep their scores, take loops of their own: in the common one
// the bookkeeping cost 40 registers that it does not have.
// Grid: row tiles x key/value heads x chunks; 64 RT PS threads.
// Row tiles of a wave, and threads of a workgroup.  Two tiles share the values' dequantising, where registers hold two and the
// other wave of the SIMD stays: 1024 tokens of 32 heads on 8 x 128 bf16 behind 8192 positions 290 us for 350, 333 tokens 121
// for 190 (16-bit types).  f32 gains as much there but loses on short calls (300 tokens behind 3700 positions 52 us for 45);
// at 256 dims two tiles leave one wave a SIMD, and 1024 f32 tokens took 745 us for 659.
template <int HD, class E, int RT>
constexpr int attend_wave_tiles() { return RT == 4 && HD <= 128 && sizeof(E) == 2 ? 2 : 1; }
template <int HD, class E, int RT, int PS>
constexpr int attend_threads() { return 64 * RT / attend_wave_tiles<HD, E, RT>() * PS; }
template <int HD, class E, int RT, int PS>
__global__ __launch_bounds__((attend_threads<HD, E, RT, PS>()), 2) void kv4_attend_kernel(Kv4View c, int len, const E* __restrict__ q, int64_t ldq, int nq,
                                                                     int n, float scale, int csz, int nch, AttendOut dst,
                                                                     E* __restrict__ out, int64_t ldo) {
  constexpr int T = HD / 32, QP = Parts<E>::q, PP = Parts<E>::p, QT = attend_wave_tiles<HD, E, RT>(),
                NT = attend_threads<HD, E, RT, PS>();
  extern __shared__ __align__(16) uint8_t smem[];
  u32x4* qs = reinterpret_cast<u32x4*>(smem);
  const int grp = nq / c.nkv, rows = n * grp, ntile = (rows + 16 * RT - 1) / (16 * RT);
  const int pairs = c.nkv * nch, pair = (int)blockIdx.x % pairs;
  const int tile = ntile - 1 - (int)blockIdx.x / pairs, g = pair % c.nkv, z = pair / c.nkv;
  const unsigned tid = threadIdx.x, lane = tid & 63u;
  const int w = __builtin_amdgcn_readfirstlane((int)(tid >> 6)), rt = w % (RT / QT) * QT, turn = w / (RT / QT);
  const int ln = (int)(lane & 15u), lk = (int)(lane >> 4);
  const int row0 = 16 * RT * tile, wrow = row0 + 16 * rt;
  const int before = len - n;
  // the positions that any row of the workgroup (of the wave) sees in the chunk
  const int last_row = min(row0 + 16 * RT, rows) - 1, wlast = min(wrow + 16 * QT, rows) - 1;
  const int pbeg = z * csz, pend = min(min((z + 1) * csz, len), before + last_row / grp + 1);
  const int wend = wrow < rows ? min(pend, before + wlast / grp + 1) : pbeg;
  const int wmin = wrow < rows ? before + wrow / grp + 1 : 0;  // what the wave's first row sees
  int rho[QT], ctx[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    rho[u] = wrow + 16 * u + ln;
    ctx[u] = rho[u] < rows ? before + rho[u] / grp + 1 : 0;
  }
  const uint8_t *kc = c.kc + g * c.code_head(), *vc = c.vc + g * c.code_head();
  const uint8_t *ks = c.ks + g * c.scale_head(), *vs = c.vs + g * c.scale_head();
  const uint8_t* bad = c.bad + (size_t)g * (c.cap / kKv4Tile);
  constexpr int step = 32 * PS;
  const int p_first = pbeg + 32 * turn;
  KeyWords<HD> kw;
  ValueWords<HD> vw;
  QueryStage<HD, E, RT, NT> queries;
  queries.load(q, ldq, g * grp, grp, row0, rows, (int)tid);
  // whether a tile of the chunk may hold blocks that are not numbers: such chunks take a loop of their own
  unsigned flag = 0;
  for (int p = pbeg + 32 * (int)lane; p < pend; p += 32 * 64) flag |= bad[p >> 5];
  if (p_first < wend) {
    kw.load(kc, ks, p_first, ln, lk);
    vw.load(vc, vs, p_first, (int)lane);
  }
  queries.store(qs, (int)tid);
  __syncthreads();
  f32x4 o[QT][2 * T];
  float m[QT], l[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
#pragma unroll
    for (int t = 0; t < 2 * T; ++t) o[u][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[u] = -INFINITY;
    l[u] = 0.f;
  }
  int first[T];  // first position seen whose value block t is not a number
#pragma unroll
  for (int t = 0; t < T; ++t) first[t] = 0x7FFFFFFF;
  unsigned qoff = (unsigned)(rt * T * QP * 64) + lane;
  auto tiles = [&](auto Odd, auto Keep) {
    for (int p0 = p_first; p0 < wend; p0 += step) {
      constexpr bool odd = decltype(Odd)::value;
      const int pn = p0 + step < wend ? p0 + step : p0;  // past the last tile: not used
      // the queries are read from LDS anew for every tile: in registers they would cost the second wave its place
      asm volatile("" : "+v"(qoff));
      f32x4 s[QT][2];
#pragma unroll
      for (int u = 0; u < QT; ++u) s[u][0] = s[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      // matrix instructions of block b among the next block's dequantising
      u32x4 k0 = kw.operand(0, 0), k1 = kw.operand(1, 0), qq[QT][QP];
#pragma unroll
      for (int u = 0; u < QT; ++u)
#pragma unroll
        for (int k = 0; k < QP; ++k) qq[u][k] = qs[qoff + (u * T * QP + k) * 64];
#pragma unroll
      for (int b = 0; b < T; ++b) {
        u32x4 n0 = k0, n1 = k1, qn[QT][QP];
        if (b + 1 < T) {
#pragma unroll
          for (int u = 0; u < QT; ++u)
#pragma unroll
            for (int k = 0; k < QP; ++k) qn[u][k] = qs[qoff + ((u * T + b + 1) * QP + k) * 64];
          n0 = kw.operand(0, b + 1);
          n1 = kw.operand(1, b + 1);
        }
#pragma unroll
        for (int k = 0; k < QP; ++k)
#pragma unroll
          for (int u = 0; u < QT; ++u) {
            s[u][0] = mfma(k0, qq[u][k], s[u][0]);
            s[u][1] = mfma(k1, qq[u][k], s[u][1]);
          }
        interleave<2 * QP * QT, 10>();
        __builtin_amdgcn_sched_barrier(0);
        k0 = n0;
        k1 = n1;
#pragma unroll
        for (int u = 0; u < QT; ++u)
#pragma unroll
          for (int k = 0; k < QP; ++k) qq[u][k] = qn[u][k];
      }
      unsigned b0 = 0, b1 = 0;
      if constexpr (odd) {
        b0 = kw.bad_rows(0);
        b1 = kw.bad_rows(1);
      }
      kw.load(kc, ks, pn, ln, lk);
      u32x4 pp[QT][PP];
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[u][j >> 2][j & 3] * scale;
        if constexpr (odd) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (((j < 4 ? b0 : b1) >> (4 * lk + (j & 3))) & 1u) x[j] = __builtin_nanf("");
        }
        if (p0 + 32 > wmin) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (p0 + 16 * (j >> 2) + 4 * lk + (j & 3) >= ctx[u]) x[j] = -INFINITY;
        }
        if constexpr (decltype(Keep)::value) {
          // every position up to the last row's is in some wave's tile, so that the rows are written whole
          if (dst.scores && rho[u] < rows) {
            float* y = dst.scores + ((size_t)(rho[u] / grp) * nq + g * grp + rho[u] % grp) * c.cap + p0 + 4 * lk;
            *reinterpret_cast<f32x4*>(y) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(y + 16) = f32x4{x[4], x[5], x[6], x[7]};
          }
        }
        const float bm = max_over_lk(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))));
        const float mn = fmaxf(m[u], bm);
        // a row that has seen nothing keeps m = -inf: its factor is 1 by definition, and its probabilities 0
        const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[u] - mn) * kLog2e);
        const float base = mn == -INFINITY ? 0.f : mn;
        float p[8], ps = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f((x[j] - base) * kLog2e);
          ps += p[j];
        }
        l[u] = l[u] * al + sum_over_lk(ps);
        m[u] = mn;
        // the O rows of this lane are 4lk + i: their factors live in lanes 4lk + i
        if (__ballot(al != 1.f)) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = __shfl(al, 4 * lk + i);
#pragma unroll
            for (int t = 0; t < 2 * T; ++t) o[u][t][i] *= a;
          }
        }
        split8<PP>(p, pp[u]);
      }
      if constexpr (odd) vw.take_bad(p0, lk, first);
      u32x4 lo, hi;
      vw.operands(0, lo, hi);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        u32x4 nlo = lo, nhi = hi;
        if (t + 1 < T) vw.operands(t + 1, nlo, nhi);
#pragma unroll
        for (int k = 0; k < PP; ++k)
#pragma unroll
          for (int u = 0; u < QT; ++u) {
            o[u][2 * t] = mfma(pp[u][k], lo, o[u][2 * t]);
            o[u][2 * t + 1] = mfma(pp[u][k], hi, o[u][2 * t + 1]);
          }
        interleave<2 * PP * QT, 24>();
        __builtin_amdgcn_sched_barrier(0);
        lo = nlo;
        hi = nhi;
      }
      vw.load(vc, vs, pn, (int)lane);
    }
  };
  if (__ballot(flag != 0)) {
    tiles(std::true_type{}, std::integral_constant<bool, RT == 1>{});
    // rows that see a value which is not a number
#pragma unroll
    for (int u = 0; u < QT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ci = __shfl(ctx[u], 4 * lk + i);
#pragma unroll
        for (int t = 0; t < T; ++t)
          if (first[t] < ci) o[u][2 * t][i] = o[u][2 * t + 1][i] = __builtin_nanf("");
      }
  } else if (RT == 1 && dst.scores) {
    tiles(std::false_type{}, std::integral_constant<bool, RT == 1>{});
  } else {
    tiles(std::false_type{}, std::false_type{});
  }
  if constexpr (RT == 1) {
    // the waves' results of the rows that there are, [wave][row][HD + 8] (the rows of a store in different banks), over
    // the queries, which every wave has read; then each row's largest maximum and the sums at it, four dims a thread
    constexpr int LD = HD + 8;
    const int nr = min(16, rows - row0);
    float* ms = reinterpret_cast<float*>(smem);  // m [PS][16], l [PS][16]
    float* os = ms + 32 * PS;
    __syncthreads();
    if (lk == 0) {
      ms[16 * w + ln] = m[0];
      ms[16 * PS + 16 * w + ln] = l[0];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * lk + i < nr)
#pragma unroll
        for (int t = 0; t < T; ++t)
          *reinterpret_cast<float2*>(os + (size_t)(w * nr + 4 * lk + i) * LD + 32 * t + 2 * ln) = make_float2(o[0][2 * t][i], o[0][2 * t + 1][i]);
    __syncthreads();
    for (int u = (int)tid; u < nr * (HD / 4); u += NT) {
      const int q = u / (HD / 4), r = row0 + q, d = 4 * (u % (HD / 4));
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < PS; ++k) M = fmaxf(M, ms[16 * k + q]);
      f32x4 O{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < PS; ++k) {
        const float e = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((ms[16 * k + q] - M) * kLog2e);
        L = __builtin_fmaf(ms[16 * PS + 16 * k + q], e, L);
        O += *reinterpret_cast<const f32x4*>(os + (size_t)(k * nr + q) * LD + d) * e;
      }
      const size_t row = (size_t)(r / grp) * nq + g * grp + r % grp;
      if (nch == 1) {
        E* y = out + (size_t)(r / grp) * ldo + (size_t)(g * grp + r % grp) * HD + d;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = dst.value<E, HD>(O[j], L, row, d + j);
        if (dst.stats && d == 0) dst.stats[row] = make_float2(M, L);
      } else {
        float* rr = dst.rec + (row * nch + z) * (2 + HD);
        if (d == 0) *reinterpret_cast<float2*>(rr) = make_float2(M, L);
        *reinterpret_cast<float2*>(rr + 2 + d) = make_float2(O[0], O[1]);
        *reinterpret_cast<float2*>(rr + 4 + d) = make_float2(O[2], O[3]);
      }
    }
    return;
  }
  // the waves of a row tile: the later half's results go to the earlier half's, until one has all
  f32x4* os = reinterpret_cast<f32x4*>(smem);  // [slot][2T][lane], over the queries, which every wave has read
  float2* mls = reinterpret_cast<float2*>(smem + (size_t)(RT * PS / 2) * 2 * T * 1024);  // [slot][lane]
#pragma unroll
  for (int half = PS / 2; half > 0; half /= 2) {
    __syncthreads();
    if (turn >= half && turn < 2 * half) {
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const int slot = (turn - half) * RT + rt + u;
#pragma unroll
        for (int t = 0; t < 2 * T; ++t) os[(slot * 2 * T + t) * 64 + lane] = o[u][t];
        mls[slot * 64 + lane] = make_float2(m[u], l[u]);
      }
    }
    __syncthreads();
    if (turn < half) {
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const int from = turn * RT + rt + u;
        const float2 ml = mls[from * 64 + lane];
        const float M = fmaxf(m[u], ml.x);
        const float ea = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[u] - M) * kLog2e);
        const float eb = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((ml.x - M) * kLog2e);
        l[u] = l[u] * ea + ml.y * eb;
        m[u] = M;
        float fa[4], fb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fa[i] = __shfl(ea, 4 * lk + i);
          fb[i] = __shfl(eb, 4 * lk + i);
        }
#pragma unroll
        for (int t = 0; t < 2 * T; ++t) {
          const f32x4 v = os[(from * 2 * T + t) * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[u][t][i] = o[u][t][i] * fa[i] + v[i] * fb[i];
        }
      }
    }
  }
  if (turn) return;
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    if (lk == 0 && rho[u] < rows) {
      const size_t row = (size_t)(rho[u] / grp) * nq + g * grp + rho[u] % grp;
      if (nch > 1) *reinterpret_cast<float2*>(dst.rec + (row * nch + z) * (2 + HD)) = make_float2(m[u], l[u]);
      else if (dst.stats) dst.stats[row] = make_float2(m[u], l[u]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = wrow + 16 * u + 4 * lk + i;
      const float li = __shfl(l[u], 4 * lk + i);
      if (r >= rows) continue;
      const size_t row = (size_t)(r / grp) * nq + g * grp + r % grp;
      if (nch == 1) {
        E* y = out + (size_t)(r / grp) * ldo + (size_t)(g * grp + r % grp) * HD + 2 * ln;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          y[32 * t] = dst.value<E, HD>(o[u][2 * t][i], li, row, 32 * t + 2 * ln);
          y[32 * t + 1] = dst.value<E, HD>(o[u][2 * t + 1][i], li, row, 32 * t + 2 * ln + 1);
        }
      } else {
        float* rr = dst.rec + (row * nch + z) * (2 + HD) + 2 + 2 * ln;
#pragma unroll
        for (int t = 0; t < T; ++t) *reinterpret_cast<float2*>(rr + 32 * t) = make_float2(o[u][2 * t][i], o[u][2 * t + 1][i]);
      }
    }
  }
}

// The chunks' records of a row (query blockIdx.x, head blockIdx.y) as 64 dims (blockIdx.z) of its output, and its
// statistics: 256 threads, wave w for the w-th quarter of the chunks, N of its records requested at a time.  A chunk whose
// positions the row does not see has l = 0, m = -inf and zeros.  Bound by latency: one token of 24 heads in 64 chunks 2.5 us.
template <int HD, class E, int N>
__global__ __launch_bounds__(256) void kv4_merge_kernel(AttendOut src, int nch, int nq, E* __restrict__ out, int64_t ldo) {
  __shared__ float fac[kKv4MaxChunks], red[4][65], mx[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, d = (int)blockIdx.z * 64 + lane;
  const size_t row = (size_t)blockIdx.x * nq + blockIdx.y;
  const float* rec = src.rec + row * nch * (2 + HD);
  const int q4 = (nch + 3) / 4, z0 = w * q4, z1 = min(nch, z0 + q4);
  float v[N];
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = rec[(size_t)min(z0 + k, nch - 1) * (2 + HD) + 2 + d];
  const float2 ml = *reinterpret_cast<const float2*>(rec + (size_t)min(tid, nch - 1) * (2 + HD));
  float m = ml.x;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
  if (lane == 0) mx[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  const float e = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((ml.x - m) * kLog2e);
  if (tid < nch) fac[tid] = e;
  float l = tid < nch ? ml.y * e : 0.f;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) l += __shfl_xor(l, k);
  if (lane == 0) red[w][64] = l;
  __syncthreads();
  float o = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (z0 + k < z1) o = __builtin_fmaf(v[k], fac[z0 + k], o);
  for (int z = z0 + N; z < z1; z += N) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = rec[(size_t)min(z + k, nch - 1) * (2 + HD) + 2 + d];
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (z + k < z1) o = __builtin_fmaf(v[k], fac[z + k], o);
  }
  red[w][lane] = o;
  __syncthreads();
  if (w) return;
  l = (red[0][64] + red[1][64]) + (red[2][64] + red[3][64]);
  o = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
  out[(size_t)blockIdx.x * ldo + (size_t)blockIdx.y * HD + d] = src.value<E, HD>(o, l, row, d);
  if (src.stats && d == 0) src.stats[row] = make_float2(m, l);
}

// The same of at most 4 chunks (many rows): four dims a thread and no LDS.  333 tokens of 24 heads in two chunks: 7.6 us against
// 26.6 by the kernel above.  Grid (ceil(n · nq · HD/4 / 256)), 256 threads.
template <int HD, class E>
__global__ __launch_bounds__(256) void kv4_merge_few_kernel(AttendOut src, int nch, int nq, int64_t rows, E* __restrict__ out,
                                                            int64_t ldo) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, row = u / (HD / 4);
  const int d = 4 * (int)(u % (HD / 4));
  if (row >= rows) return;
  const float* rec = src.rec + (size_t)row * nch * (2 + HD);
  float2 ml[4], a[4], b[4];
#pragma unroll
  for (int z = 0; z < 4; ++z) {
    const float* r = rec + (size_t)min(z, nch - 1) * (2 + HD);
    ml[z] = *reinterpret_cast<const float2*>(r);
    a[z] = *reinterpret_cast<const float2*>(r + 2 + d);
    b[z] = *reinterpret_cast<const float2*>(r + 4 + d);
  }
  const float m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int z = 0; z < 4; ++z) {
    if (z >= nch) break;
    const float e = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((ml[z].x - m) * kLog2e);
    l = __builtin_fmaf(ml[z].y, e, l);
    o[0] = __builtin_fmaf(a[z].x, e, o[0]);
    o[1] = __builtin_fmaf(a[z].y, e, o[1]);
    o[2] = __builtin_fmaf(b[z].x, e, o[2]);
    o[3] = __builtin_fmaf(b[z].y, e, o[3]);
  }
  E* y = out + (size_t)(row / nq) * ldo + (size_t)(row % nq) * HD + d;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = src.value<E, HD>(o[j], l, (size_t)row, d + j);
  if (src.stats && d == 0) src.stats[row] = make_float2(m, l);
}

// weights[g][r] += Σ exp(s_ρr - m_ρ) / l_ρ over the group's query rows ρ in order, from the scores that the attention left
// (few rows): four positions a thread.  Bound by the launch: 32768 positions of 24 heads 5.1 us (3.1 MB).  Grid (ceil(len / 1024), nkv), 256 threads.
__global__ __launch_bounds__(256) void kv4_few_weights_kernel(const float* __restrict__ scores, int cap, int len, int nq, int grp,
                                                              int rows, const float2* __restrict__ stats,
                                                              float* __restrict__ weights, int64_t ldw) {
  const int before = len - rows / grp;
  const int g = blockIdx.y, r = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
  if (r >= len) return;
  f32x4 s[16];
  float2 st[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int rho = min(k, rows - 1);
    const size_t row = (size_t)(rho / grp) * nq + g * grp + rho % grp;
    s[k] = *reinterpret_cast<const f32x4*>(scores + row * cap + r);  // cap is a multiple of 32
    st[k] = stats[row];
  }
  f32x4 a{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (k < rows) {
      const float inv = 1.f / st[k].y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f((s[k][i] - st[k].x) * kLog2e) * inv;
        a[i] += r + i <= before + k / grp ? p : 0.f;  // what a row does not see gets nothing though the row's sum be a NaN
      }
    }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r + i < len) weights[(size_t)g * ldw + r + i] += a[i];
}

// Bytes of a row tile of the operands that the weights' pass takes ready.
template <int HD, class E>
constexpr int ready_bytes() { return HD / 32 * Parts<E>::q * 1024; }

// The query rows of a key/value head as operands, a tile of 16 rows per workgroup: [kv head][row tile].  500 tiles of f32
// rows 9 us.
// Grid (row tiles, nkv), 256 threads.
template <int HD, class E>
__global__ __launch_bounds__(256) void kv4_split_kernel(const E* __restrict__ q, int64_t ldq, int nkv, int nq, int n,
                                                        uint8_t* __restrict__ split) {
  const int g = blockIdx.y, grp = nq / nkv;
  uint8_t* to = split + ((size_t)g * gridDim.x + blockIdx.x) * ready_bytes<HD, E>();
  QueryStage<HD, E, 1, 256> queries;
  queries.load(q, ldq, g * grp, grp, 16 * (int)blockIdx.x, n * grp, (int)threadIdx.x);
  queries.store(reinterpret_cast<u32x4*>(to), (int)threadIdx.x);
}

// weights[g][r] += Σ over the group's query rows ρ of exp(s_ρr - m_ρ) / l_ρ: a wave holds the operands of 16·PT rows of keys and
// walks the query rows 16 at a time, in LDS for the workgroup's four waves, a lane adding up its four positions
// of each 16 over the query rows ln, in order; the sixteen lanes of a position are summed at the end.
// READY: the queries come as operands (kv4_split_kernel), the next tile's requested ahead and LDS in two halves, one
// barrier a tile, and the row tiles may be spread over gridDim.z workgroups whose sums kv4_join_weights_kernel adds; else
// the workgroup forms them (few rows, where a launch more would cost more).
// Bound by the matrix instructions (96 of 6.7 ns a wave and tile with f32 queries and PT = 4) and the vector ones (about
// 350, 0.7 us), which add up to the 2.9 us that a tile of two waves a SIMD takes; a tile's exponentials among the next
// one's matrix instructions measured the same.
// Grid (ceil(len / 64PT), nkv, parts), 256 threads.
template <int HD, class E, int PT, bool READY>
__global__ __launch_bounds__(256, 1) void kv4_weights_kernel(Kv4View c, int len, const E* __restrict__ q, int64_t ldq, int nq, int n,
                                                             float scale, const u32x4* __restrict__ split,
                                                             const float2* __restrict__ stats, float* __restrict__ weights,
                                                             int64_t ldw, float* __restrict__ parts) {
  constexpr int T = HD / 32, QP = Parts<E>::q, TILE = T * QP * 64, N = (TILE + 255) / 256;
  __shared__ u32x4 qs[(READY ? 2 : 1) * TILE];
  const int g = blockIdx.y, grp = nq / c.nkv, rows = n * grp, before = len - n;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int ln = lane & 15, lk = lane >> 4;
  const int pblk = (int)blockIdx.x * 64 * PT, pw = pblk + 16 * PT * w;  // the workgroup's and the wave's first position
  const uint8_t *kc = c.kc + g * c.code_head(), *ks = c.ks + g * c.scale_head();
  u32x4 kop[PT][T];
  unsigned nan[PT];
#pragma unroll
  for (int u = 0; u < PT; u += (PT == 1 ? 1 : 2)) {
    KeyWords<HD> kw;
    // whole tiles of 32 rows; past the last one (a wave with nothing to do, or half a tile) the first is read instead
    const int r = pw + 16 * u, base = r < len ? r & ~31 : 0;
    kw.load(kc, ks, base, ln, lk);
    const int h0 = r < len ? (r >> 4) & 1 : 0;
#pragma unroll
    for (int b = 0; b < T; ++b) {
      if constexpr (PT == 1) {
        kop[u][b] = h0 ? kw.operand(1, b) : kw.operand(0, b);
      } else {
        kop[u][b] = kw.operand(0, b);
        kop[u + 1][b] = kw.operand(1, b);
      }
    }
    if constexpr (PT == 1) {
      nan[u] = h0 ? kw.bad_rows(1) : kw.bad_rows(0);
    } else {
      nan[u] = kw.bad_rows(0);
      nan[u + 1] = kw.bad_rows(1);
    }
  }
  unsigned any_nan = 0;
#pragma unroll
  for (int u = 0; u < PT; ++u) any_nan |= nan[u];
  float acc[PT][4];
#pragma unroll
  for (int u = 0; u < PT; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[u][i] = 0.f;
  // from the tile of the first query row that sees the workgroup's first position
  const int ts = max(0, pblk - before) * grp / 16, tn = (rows + 15) / 16;
  const int z = READY ? (int)blockIdx.z : 0, nz = READY ? (int)gridDim.z : 1;
  const int t0 = ts + (int)((int64_t)(tn - ts) * z / nz), te = ts + (int)((int64_t)(tn - ts) * (z + 1) / nz);
  u32x4 next[READY ? N : 1];
  float2 st_next = make_float2(0.f, 1.f);
  const u32x4* tiles = split + (size_t)g * tn * TILE;
  auto stat = [&](int t) {
    const int rho = min(16 * t + ln, rows - 1);
    return stats[(size_t)(rho / grp) * nq + g * grp + rho % grp];
  };
  auto request = [&](int t) {
    if constexpr (READY)
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = tiles[(size_t)t * TILE + (TILE % 256 ? min(tid + 256 * i, TILE - 1) : tid + 256 * i)];
    st_next = stat(t);
  };
  if (t0 < te) request(t0);
  for (int t = t0; t < te; ++t) {
    const u32x4* qt = qs;
    if constexpr (READY) {
      u32x4* to = qs + (t & 1) * TILE;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (TILE % 256 == 0 || tid + 256 * i < TILE) to[tid + 256 * i] = next[i];
      qt = to;
    } else {
      QueryStage<HD, E, 1, 256> queries;
      queries.load(q, ldq, g * grp, grp, 16 * t, rows, tid);
      __syncthreads();
      queries.store(qs, tid);
    }
    const float2 st = st_next;
    __syncthreads();
    request(min(t + 1, te - 1));
    const int rho = 16 * t + ln;
    const int ctx = rho < rows ? before + rho / grp + 1 : 0;
    f32x4 s[PT];
#pragma unroll
    for (int u = 0; u < PT; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < T; ++b)
#pragma unroll
      for (int k = 0; k < QP; ++k) {
        const u32x4 qq = qt[(b * QP + k) * 64 + lane];
#pragma unroll
        for (int u = 0; u < PT; ++u) s[u] = mfma(kop[u][b], qq, s[u]);
      }
    const float inv = 1.f / st.y;
    if (any_nan) {
#pragma unroll
      for (int u = 0; u < PT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((nan[u] >> (4 * lk + i)) & 1u) s[u][i] = __builtin_nanf("");
    }
    // the tile's first row sees the fewest positions; a tile past the last row has rows that count for nothing
    const bool whole = 16 * t + 16 <= rows && before + 16 * t / grp + 1 >= pw + 16 * PT;
#pragma unroll
    for (int u = 0; u < PT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f((s[u][i] * scale - st.x) * kLog2e) * inv;
        acc[u][i] += whole || pw + 16 * u + 4 * lk + i < ctx ? p : 0.f;
      }
  }
#pragma unroll
  for (int u = 0; u < PT; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = acc[u][i];
      a += __shfl_xor(a, 1);
      a += __shfl_xor(a, 2);
      a += __shfl_xor(a, 4);
      a += __shfl_xor(a, 8);
      const int r = pw + 16 * u + 4 * lk + i;
      if (ln != 0 || r >= len) continue;
      if (READY && nz > 1) parts[((size_t)(g * gridDim.x + blockIdx.x) * nz + z) * (64 * PT) + (r - pblk)] = a;
      else weights[(size_t)g * ldw + r] += a;
    }
}

// weights[g][r] += the sums of its nz parts [kv head][block of 64 PT positions][part][64 PT], in order.
// Grid (ceil(len / 64PT), nkv), 64 PT threads.
__global__ __launch_bounds__(256) void kv4_join_weights_kernel(const float* __restrict__ parts, int nz, int len,
                                                               float* __restrict__ weights, int64_t ldw) {
  const int g = blockIdx.y, n = (int)blockDim.x, r = (int)blockIdx.x * n + (int)threadIdx.x;
  if (r >= len) return;
  const float* p = parts + (size_t)(g * gridDim.x + blockIdx.x) * nz * n + threadIdx.x;
  float a = 0.f;
  for (int z = 0; z < nz; z += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[(size_t)min(z + i, nz - 1) * n];
#pragma unroll
    for (int i = 0; i < 8; ++i) a += z + i < nz ? v[i] : 0.f;
  }
  weights[(size_t)g * ldw + r] += a;
}

// The form of the kernel that a call takes: row tiles of a workgroup (rt), and the waves of a row tile (ps).  Four row tiles
// read the cache once between them; up to 192 rows one tile a workgroup, each with its own pass over the cache but more
// waves on the same chunk, is faster.  Behind 8192 positions, one tile against four, us:
//   rows            48           192          288          384
//   24/4 x 256 f32  17.7 : 24.5  34.6 : 42.0  44.5 : 52.9  57.8 : 60.7
//   32/8 x 128 bf16 14.6 : 18.9  30.9 : 33.0  43.5 : 42.7  47.2 : 48.8
//   16/4 x 64 bf16   9.6 : 12.7  15.1 : 18.7  19.2 : 22.5  23.7 : 24.8
// With one key/value head (8/1 x 256 f32: 24.0 : 31.9 at 384 rows) it would still be ahead beyond the line, whose work memory
// and cache traffic grow with the rows.  It takes eight waves, or four while 256 workgroups of four have no more than a tile
// each: fewer results to join (one token, four against eight: 24/4 x 256 f32 10.8 : 12.2 us at 4096 positions, 14.6 : 15.1 at
// 16384, 18.3 : 18.1 at 32768; 8/1 x 128 f16 8.2 : 8.9 at 4096, 12.7 : 11.1 at 32768).
struct AttendForm {
  int rt, ps;
};
static AttendForm attend_form(int rows, int nkv, int len) {
  if (rows > 192) return AttendForm{4, 2};
  return AttendForm{1, (int64_t)len * nkv * ((rows + 15) / 16) <= 256 * 128 ? 4 : 8};
}
template <class F>
static int with_form(AttendForm form, F&& f) {
  if (form.rt == 4) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
  if (form.ps == 8) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
}
// Chunks of positions that a call's row tiles are spread over: as many workgroups as are resident at once (one a compute unit, of
// two waves a SIMD; two where a wave has two row tiles and each gets 512 positions, below which 16 tiles behind 4000
// positions took 16.7 us for 13.4); or, where that leaves a good part of them idle in the last round, up to three chunks, if
// each is long enough to be worth a merge (1024 tokens of 24 heads on 4 behind 8192 positions, 384 row tiles: 581 us in two
// chunks, 659 in one).  len = 0: the most chunks that any length takes.
constexpr int kKv4LongChunk = 2048;
static int attend_chunks(int n, int n_head, int nkv, bool pairs, int len) {
  const int rows = n * (n_head / nkv), rt = attend_form(rows, nkv, 0).rt;
  const int64_t tiles = (int64_t)((rows + 16 * rt - 1) / (16 * rt)) * nkv;
  const int resident = pairs && rt == 4 && (len == 0 || len * tiles >= 512 * 512) ? 512 : 256;
  int best = (int)std::max<int64_t>(1, std::min<int64_t>(kKv4MaxChunks, resident / tiles));
  if (tiles >= 4 * resident) return best;  // the last round is a small part of the work, the chunks' records would be large
  if (len == 0) return std::max(best, 3);
  auto rounds = [&](int k) { return (tiles * k + resident - 1) / resident; };
  for (int k = best + 1; k <= 3 && len / k >= kKv4LongChunk; ++k)
    if (10 * rounds(k) * best < 9 * rounds(best) * k) best = k;
  return best;
}

// From this many tiles of 16 query rows on the weights' pass takes its queries as operands formed once.  Attention and pass, formed
// once against by every workgroup, us:
//   rows                   80           96           128          192
//   24/4 x 256 f32   600   24.9 : 22.5  25.4 : 24.0  26.3 : 27.9  28.3 : 35.0
//                   8192   39.6 : 35.2  42.6 : 39.2  44.3 : 44.2  55.6 : 60.2
//   32/8 x 128 bf16  600   19.9 : 16.1  20.2 : 16.9  20.6 : 18.8  22.7 : 22.5
//                   8192   32.5 : 29.5  34.2 : 31.8  36.6 : 35.6  47.5 : 48.8
//   8/1 x 256 f32   8192   27.4 : 24.9  27.9 : 26.7  29.0 : 31.0  32.6 : 38.4
constexpr int kKv4SplitTiles = 8;
// It has 4 tiles of 16 positions a wave then, and its query rows over as many workgroups as make up this number (attention and
// pass of 2000 rows behind 2000 and 7333 positions: 24/4 x 256 f32 106 and 276 us, with all the rows in each workgroup 291
// and 408; 16/4 x 64 bf16 46 and 100, 137 and 168; 8/1 x 128 f16 38 and 60, 161 and 181).
constexpr int kKv4WeightGroups = 512, kKv4WeightTiles = 4;

size_t kv4_attend_work(const Kv4View& c, int n_head, int n, bool weights) {
  const size_t rows = (size_t)n * n_head, nch = (size_t)attend_chunks(n, n_head, c.nkv, c.hd <= 128, 0);
  const size_t rec = nch > 1 ? (rows * nch * (size_t)(2 + c.hd) * sizeof(float) + 15) / 16 * 16 : 0;
  const int tiles = (n * (n_head / c.nkv) + 15) / 16;
  const size_t stats = (rows * sizeof(float2) + 15) / 16 * 16;
  if (!weights) return stats + rec;
  if (tiles == 1) return stats + rec + rows * (size_t)c.cap * sizeof(float);  // the scores
  // over the records; the f32 queries' are the largest
  const size_t ready = (size_t)(c.hd / 32) * Parts<float>::q * 1024;
  const size_t split = tiles >= kKv4SplitTiles ? (size_t)tiles * c.nkv * ready + kKv4WeightGroups * 64 * kKv4WeightTiles * sizeof(float) : 0;
  return stats + std::max(rec, split);
}

// Dynamic LDS of a workgroup for a call of `rows` rows a key/value head.
template <int HD, class E, int RT, int PS>
constexpr size_t attend_lds(int rows) {
  const size_t queries = (size_t)RT * (HD / 32 * Parts<E>::q * 1024);
  const size_t join = RT == 1 ? (size_t)PS * (128 + (rows < 16 ? rows : 16) * (HD + 8) * 4) : (size_t)(RT * PS / 2) * (HD / 32 * 2 * 1024 + 512);
  return queries > join ? queries : join;
}

// Dynamic-LDS limits, set once for each device before any launch or capture.
int prepare_kv4_kernels() {
  static std::mutex mu;
  static bool done[64];
  std::lock_guard<std::mutex> lock(mu);
  int dev = 0;
  DZ_HIP_CHECK(hipGetDevice(&dev));
  if (dev < 64 && done[dev]) return DZ_OK;
  for (int hd : {64, 128, 256})
    for (int type : {DZ_F32, DZ_F16, DZ_BF16})
      for (AttendForm form : {AttendForm{1, 4}, AttendForm{1, 8}, AttendForm{4, 2}}) {
        const int rc = with_head_dim(hd, [&](auto D) {
          return with_type(type, [&](auto* e) {
            return with_form(form, [&](auto R, auto P) -> int {
              using E = std::remove_pointer_t<decltype(e)>;
              constexpr int HD = decltype(D)::value, RT = decltype(R)::value, PS = decltype(P)::value;
              DZ_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kv4_attend_kernel<HD, E, RT, PS>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)attend_lds<HD, E, RT, PS>(16)));
              return DZ_OK;
            });
          });
        });
        if (rc) return rc;
      }
  if (dev < 64) done[dev] = true;
  return DZ_OK;
}

int kv4_attend(const Kv4View& c, int len, const void* q, int64_t ldq, int type, int n_head, int n, float scale, float* weights,
               int64_t ldw, void* out, int64_t ldo, void* work, hipStream_t s, const float* gate) {
  const int rows = n * (n_head / c.nkv);
  const AttendForm form = attend_form(rows, c.nkv, len);
  const int unit = 32 * form.ps;  // a tile for every wave
  const bool pairs = c.hd <= 128 && type != DZ_F32;
  const int most = attend_chunks(n, n_head, c.nkv, pairs, len);
  const int csz = ((len + most - 1) / most + unit - 1) / unit * unit, nch = (int)(((int64_t)len + csz - 1) / csz);
  return with_head_dim(c.hd, [&](auto D) {
    constexpr int HD = decltype(D)::value;
    return with_type(type, [&](auto* e) -> int {
      using E = std::remove_pointer_t<decltype(e)>;
      AttendOut dst;
      float2* stats = static_cast<float2*>(work);
      dst.stats = weights ? stats : nullptr;
      dst.gate = gate;
      dst.rec = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + ((size_t)n * n_head * sizeof(float2) + 15) / 16 * 16);
      // behind the records
      dst.scores = weights && rows <= 16 ? dst.rec + (nch > 1 ? ((size_t)n * n_head * nch * (2 + HD) + 3) / 4 * 4 : 0) : nullptr;
      const int rc = with_form(form, [&](auto R, auto P) -> int {
        constexpr int RT = decltype(R)::value, PS = decltype(P)::value;
        const unsigned wgs = (unsigned)((rows + 16 * RT - 1) / (16 * RT) * c.nkv * nch);
        kv4_attend_kernel<HD, E, RT, PS><<<dim3(wgs), attend_threads<HD, E, RT, PS>(), attend_lds<HD, E, RT, PS>(rows), s>>>(
            c, len, (const E*)q, ldq, n_head, n, scale, csz, nch, dst, (E*)out, ldo);
        DZ_HIP_CHECK(hipGetLastError());
        return DZ_OK;
      });
      if (rc) return rc;
      if (nch > 1) {
        const dim3 grid((unsigned)n, (unsigned)n_head, HD / 64);
        const int64_t all = (int64_t)n * n_head;
        if (nch <= 4)
          kv4_merge_few_kernel<HD, E><<<dim3((unsigned)((all * (HD / 4) + 255) / 256)), 256, 0, s>>>(dst, nch, n_head, all, (E*)out, ldo);
        else if (nch <= 16) kv4_merge_kernel<HD, E, 4><<<grid, 256, 0, s>>>(dst, nch, n_head, (E*)out, ldo);
        else kv4_merge_kernel<HD, E, 16><<<grid, 256, 0, s>>>(dst, nch, n_head, (E*)out, ldo);
        DZ_HIP_CHECK(hipGetLastError());
      }
      if (weights && dst.scores) {
        kv4_few_weights_kernel<<<dim3((unsigned)((len + 1023) / 1024), (unsigned)c.nkv), 256, 0, s>>>(
            dst.scores, c.cap, len, n_head, n_head / c.nkv, rows, stats, weights, ldw);
        DZ_HIP_CHECK(hipGetLastError());
      } else if (weights) {
        const int row_tiles = (rows + 15) / 16;
        u32x4* split = row_tiles >= kKv4SplitTiles ? reinterpret_cast<u32x4*>(dst.rec) : nullptr;
        auto run = [&](auto P, auto R, int parts_n, float* parts) {
          constexpr int PT = decltype(P)::value;
          kv4_weights_kernel<HD, E, PT, decltype(R)::value>
              <<<dim3((unsigned)((len + 64 * PT - 1) / (64 * PT)), (unsigned)c.nkv, (unsigned)parts_n), 256, 0, s>>>(
                  c, len, (const E*)q, ldq, n_head, n, scale, split, stats, weights, ldw, parts);
        };
        if (split) {
          constexpr int PT = kKv4WeightTiles;
          kv4_split_kernel<HD, E><<<dim3((unsigned)row_tiles, (unsigned)c.nkv), 256, 0, s>>>((const E*)q, ldq, c.nkv, n_head, n,
                                                                                          reinterpret_cast<uint8_t*>(split));
          DZ_HIP_CHECK(hipGetLastError());
          const int blocks = (len + 64 * PT - 1) / (64 * PT);
          const int nz = (int)std::max<int64_t>(1, std::min<int64_t>(row_tiles, kKv4WeightGroups / ((int64_t)blocks * c.nkv)));
          float* parts = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(split) + (size_t)row_tiles * c.nkv * ready_bytes<HD, E>());
          run(std::integral_constant<int, PT>{}, std::true_type{}, nz, parts);
          if (nz > 1) {
            DZ_HIP_CHECK(hipGetLastError());
            kv4_join_weights_kernel<<<dim3((unsigned)blocks, (unsigned)c.nkv), 64 * PT, 0, s>>>(parts, nz, len, weights, ldw);
          }
        } else {
          // as many rows of keys a wave as leave about a workgroup for each compute unit
          const int64_t units = ((int64_t)len + 63) / 64 * c.nkv;
          if (units >= 4 * 200) run(std::integral_constant<int, 4>{}, std::false_type{}, 1, nullptr);
          else if (units >= 2 * 200) run(std::integral_constant<int, 2>{}, std::false_type{}, 1, nullptr);
          else run(std::integral_constant<int, 1>{}, std::false_type{}, 1, nullptr);
        }
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

// n plus the number of set bits of m below the lane's own.
__device__ __forceinline__ unsigned lanes_below(unsigned long long m, unsigned n) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, n));
}

constexpr int kKv4Held = 32;  // keys a thread of the selection holds

// kept[g] of head g: the `take` rows of [0, old) with the largest keys (the lower row first among equal ones), then the rows
// [old, old + recent), in ascending order.  Each wave has a span of the rows; the key of the take-th largest is
// found 11, 11 and 10 bits at a time from the top, by a histogram of the keys that share the bits found so far; then every
// wave counts and writes its span in order.  HELD: the keys stay in registers (old <= 32768), else they are read anew.
// Bound by latency, one workgroup a head: 32768 rows 24.6 us, 1100 rows 9.3 us.  The rows whose key is that of 0 are counted
// by the wave: where most rows are such, one bin took 35 us of atomics.  Grid (nkv), 1024 threads.
template <bool HELD>
__global__ __launch_bounds__(1024) void kv4_select_kernel(const float* __restrict__ w, int64_t ldw, int old, int take, int recent,
                                                          int32_t* __restrict__ kept) {
  __shared__ unsigned hist[2048], wsum[16][2], wtot[16], s_prefix, s_left;
  const unsigned tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
  const int g = blockIdx.x, m = take + recent;
  w += (size_t)g * ldw;
  kept += (size_t)g * m;
  for (int i = (int)tid; i < recent; i += 1024) kept[take + i] = old + i;
  if (take == 0) return;
  const int span = (old + 1023) / 1024 * 64, b0 = (int)wv * span, b1 = min(old, b0 + span);
  unsigned held[HELD ? kKv4Held : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kKv4Held; ++j) {
      const int r = b0 + 64 * j + (int)lane;
      held[j] = r < b1 ? __float_as_uint(w[r]) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kKv4Held; ++j) held[j] = weight_key(__uint_as_float(held[j]));
  }
  // f(row, key, whether there is one) for the wave's rows, 64 at a time, in order
  auto rows = [&](auto&& f) {
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < kKv4Held; ++j) {
        if (b0 + 64 * j >= b1) break;
        const int r = b0 + 64 * j + (int)lane;
        f(r, held[j], r < b1);
      }
    } else {
      for (int i = b0; i < b1; i += 256) {
        unsigned k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = weight_key(w[min(i + 64 * j + (int)lane, b1 - 1)]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = i + 64 * j + (int)lane;
          f(r, k[j], r < b1);
        }
      }
    }
  };
  unsigned prefix = 0, left = (unsigned)take;  // the key's bits so far; how many rows come from the keys that share them
  constexpr unsigned kZero = 0x80000000u;      // the key of 0
  int zeros = 0;                               // how many the wave has
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, up = pass == 0 ? 32 : pass == 1 ? 21 : 10;
    hist[tid] = hist[1024 + tid] = 0;
    __syncthreads();
    // keys of 0 (rows never attended to, often many) are counted by the wave, not one after another in their bin
    rows([&](int, unsigned k, bool has) {
      if (pass == 0) zeros += __popcll(__ballot(has && k == kZero));
      if (has && (pass == 0 || (k >> (up & 31)) == (prefix >> (up & 31))) && k != kZero)
        atomicAdd(&hist[(k >> sh) & (pass == 2 ? 1023u : 2047u)], 1u);
    });
    if (zeros && lane == 0 && (pass == 0 || (kZero >> (up & 31)) == (prefix >> (up & 31)))) atomicAdd(&hist[(kZero >> sh) & (pass == 2 ? 1023u : 2047u)], (unsigned)zeros);
    __syncthreads();
    // how many keys lie in the bins above a thread's two, from the top
    const unsigned hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid], own = hi + lo;
    unsigned up_to = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned v = (unsigned)__shfl_up((int)up_to, o);
      if ((int)lane >= o) up_to += v;
    }
    if (lane == 63) wtot[wv] = up_to;
    __syncthreads();
    unsigned above = up_to - own;
    for (unsigned i = 0; i < wv; ++i) above += wtot[i];
    if (above < left && above + own >= left) {
      const bool h = above + hi >= left;
      s_prefix = prefix | (h ? 2047u - 2 * tid : 2046u - 2 * tid) << sh;
      s_left = left - above - (h ? 0u : hi);
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
  }
  // rows above the key, and the first `left` rows at it
  unsigned above = 0, at = 0;  // of the lane's rows, then of the wave's
  rows([&](int, unsigned k, bool has) {
    above += has && k > prefix;
    at += has && k == prefix;
  });
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    above += (unsigned)__shfl_xor((int)above, o);
    at += (unsigned)__shfl_xor((int)at, o);
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
  rows([&](int r, unsigned k, bool has) {
    const unsigned long long ba = __ballot(has && k > prefix), bt = __ballot(has && k == prefix);
    const unsigned ra = lanes_below(ba, above);
    if (bt) {
      const unsigned rt = lanes_below(bt, at);
      if (has && (k > prefix || (k == prefix && rt < left))) kept[ra + min(rt, left)] = r;
      at += (unsigned)__popcll(bt);
    } else if (has && k > prefix) {
      kept[ra + min(at, left)] = r;
    }
    above += (unsigned)__popcll(ba);
  });
}

// Rows kept[g] of c -> the rows of dst, with their weights: a tile of 32 rows of dst per workgroup, its loads all under way
// at once.  Bound by latency of two dependent loads: 8192 rows of 4 x 256 6.6 us (18 MB read and written, 2.7 TB/s).
// Grid (ceil(m / 32), nkv), 256 threads.
template <int HD>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Kv4View c, Kv4View dst, const int32_t* __restrict__ kept, int m,
                                                         const float* __restrict__ w, int64_t ldw, float* __restrict__ dw,
                                                         int64_t ld_dw) {
  constexpr int T = HD / 32, KU = HD / 32, NK = 32 * KU / 256 > 0 ? 32 * KU / 256 : 1;  // KU: 16-byte units of a row's keys
  typedef uint8_t bytes __attribute__((ext_vector_type(T)));
  __shared__ int src[32];
  const int g = blockIdx.y, i0 = (int)blockIdx.x * 32, tid = threadIdx.x, nr = min(32, m - i0);
  if (tid < 32) src[tid] = kept[(size_t)g * m + min(i0 + tid, m - 1)];
  __syncthreads();
  const uint8_t *kc = c.kc + g * c.code_head(), *vc = c.vc + g * c.code_head();
  uint8_t *dkc = dst.kc + g * dst.code_head(), *dvc = dst.vc + g * dst.code_head();
  u32x4 kk[NK];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    const int u = tid + 256 * j, q = min(u / KU, nr - 1);
    kk[j] = *reinterpret_cast<const u32x4*>(kc + (size_t)src[q] * (HD / 2) + 16 * (u % KU));
  }
  bytes vv[2];  // of row (tid + 256 j) / 16, lane tid % 16
#pragma unroll
  for (int j = 0; j < 2; ++j)
    vv[j] = *reinterpret_cast<const bytes*>(vc + kv4_value_offset<HD>(src[min((tid + 256 * j) / 16, nr - 1)], tid % 16));
  const int q = tid & 31, what = tid >> 5;  // 0: the keys' scales, 1: the values', 2: the weight
  if (q < nr && what < 2) {
    const bytes e = *reinterpret_cast<const bytes*>((what ? c.vs : c.ks) + g * c.scale_head() + (size_t)src[q] * T);
    *reinterpret_cast<bytes*>((what ? dst.vs : dst.ks) + g * dst.scale_head() + (size_t)(i0 + q) * T) = e;
    bool bad = false;
#pragma unroll
    for (int t = 0; t < T; ++t) bad |= e[t] == 255;
    if (bad) dst.bad[(size_t)g * (dst.cap / kKv4Tile) + (i0 + q) / kKv4Tile] = 1;
  }
  if (q < nr && what == 2 && dw) dw[(size_t)g * ld_dw + i0 + q] = w[(size_t)g * ldw + src[q]];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    const int u = tid + 256 * j;
    if (u / KU < nr) *reinterpret_cast<u32x4*>(dkc + (size_t)(i0 + u / KU) * (HD / 2) + 16 * (u % KU)) = kk[j];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = (tid + 256 * j) / 16;
    if (r < nr) *reinterpret_cast<bytes*>(dvc + kv4_value_offset<HD>(i0 + r, tid % 16)) = vv[j];
  }
}

int kv4_evict(const Kv4View& c, int len, const float* weights, int64_t ldw, int keep, int recent, const Kv4View& dst,
              float* dst_weights, int64_t ld_dst, int32_t* kept, hipStream_t s) {
  const int m = std::min(keep, len);
  if (m == 0) return DZ_OK;
  recent = std::min(recent, len);
  const int old = len - recent;
  if (old <= 1024 * kKv4Held)
    kv4_select_kernel<true><<<dim3((unsigned)c.nkv), 1024, 0, s>>>(weights, ldw, old, m - recent, recent, kept);
  else
    kv4_select_kernel<false><<<dim3((unsigned)c.nkv), 1024, 0, s>>>(weights, ldw, old, m - recent, recent, kept);
  DZ_HIP_CHECK(hipGetLastError());
  return with_head_dim(c.hd, [&](auto D) -> int {
    constexpr int HD = decltype(D)::value;
    kv4_gather_kernel<HD><<<dim3((unsigned)((m + 31) / 32), (unsigned)c.nkv), 256, 0, s>>>(c, dst, kept, m, weights, ldw,
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
  int rc = ensure_device();
  if (rc || (rc = prepare_kv4_kernels())) return rc;
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

static size_t attend_work_bytes(const dz_kv4* c, int n_head, int n, bool weights) {
  if (!c || n_head < 1 || n < 1 || n_head % c->v.nkv || (int64_t)n * n_head > 1 << 30) return 0;  // refused calls
  return kv4_attend_work(c->v, n_head, n, weights);
}
size_t dz_kv4_attend_work_bytes(const dz_kv4* c, int n_head, int n) { return attend_work_bytes(c, n_head, n, true); }
size_t dz_kv4_attend_only_work_bytes(const dz_kv4* c, int n_head, int n) { return attend_work_bytes(c, n_head, n, false); }

int dz_kv4_attend_dev(const dz_kv4* c, const void* q, int64_t ldq, int type, int n_head, int n, float scale, float* weights,
                      int64_t ldw, void* out, int64_t ldo, void* work, void* stream) {
  if (!c || !q || !out || !work) return set_error(DZ_ERR_MODEL, "null argument");
  if (n_head < 1 || n_head > 65535 || n_head % c->v.nkv)
    return set_error(DZ_ERR_TENSOR, "attend: %d heads on %d kv heads", n_head, c->v.nkv);
  if (n < 1 || n > c->len) return set_error(DZ_ERR_TENSOR, "attend: %d queries over %d rows", n, c->len);
  if ((int64_t)n * n_head > 1 << 30) return set_error(DZ_ERR_UNSUPPORTED, "attend: %d queries of %d heads", n, n_head);
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
  return kv4_attend(c->v, c->len, q, ldq, type, n_head, n, scale, weights, ldw, out, ldo, work, static_cast<hipStream_t>(stream), nullptr);
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
