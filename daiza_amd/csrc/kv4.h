// kv4.h — key/value cache held in 4 bits: layout, element access and the launches shared with the contexts.
//
// A row's head is head_dim/32 blocks of 32 values, each value a 4-bit float (sign, two exponent bits, one mantissa bit)
// and each block a byte e: value = code · 2^(e - 127), e = 255 for a block with an infinity or a NaN.  The scale is a
// power of two, so that a value converts exactly to bf16 (v_cvt_scalef32_pk_bf16_fp4), the operand type of the matrix
// instructions, and a row's codes do not depend on how a division rounds.  It is the smallest power at which the largest
// value of the block does not round past 6: against the one below it wherever that value's mantissa is under 2, whose
// largest values are cut to 6, the error of a block of normal values is 11.2% instead of 11.5%, and the mean size
// of what is stored 99% instead of 98%.
//
// Layout, per key/value head and tile of 32 rows, T = head_dim/32 blocks (lane = 16·lk + ln of a wave):
//   keys    row r at r·head_dim/2, its dims in nibble order.  Lane (ln, lk) takes the quarter lk of row ln's dims: its part of
//           the matrix operands, dims in an order that the queries share
//   values  the lane's slots j = 0..7 are rows 4lk + j (j < 4) and 16 + 4lk + j - 4, the rows whose probabilities the
//           score product leaves in that lane; byte (j, t) of its 8·T bytes holds dims 32t + 2ln (low nibble) and
//           32t + 2ln + 1; the bytes come in chunks of 16, chunk c of all lanes one after another
//   scales  T bytes a row, for keys and for values
#pragma once
#include "common.h"

namespace dz {

constexpr int kKv4Tile = 32;  // rows of a tile
constexpr int kKv4MaxChunks = 256;  // a thread of the merge each
constexpr int kKv4MinExp = -120, kKv4MaxExp = 125;  // 6 · 2^125 is the largest f32 of the format

struct Kv4View {
  uint8_t *kc = nullptr, *vc = nullptr;  // codes  [kv head][cap · hd/2]
  uint8_t *ks = nullptr, *vs = nullptr;  // scales [kv head][cap · hd/32]
  uint8_t* bad = nullptr;                // [kv head][cap/32]: not 0 where a row of the tile has (or had) a scale byte of 255
  int nkv = 0, hd = 0, cap = 0;          // cap: rows, a multiple of 32
  __host__ __device__ size_t code_head() const { return (size_t)cap * (size_t)(hd / 2); }
  __host__ __device__ size_t scale_head() const { return (size_t)cap * (size_t)(hd / 32); }
};
inline size_t kv4_bytes(int nkv, int hd, int cap) {
  return (size_t)nkv * ((size_t)cap * (size_t)(hd / 2 + hd / 32) * 2 + (size_t)(cap / kKv4Tile));
}
// A view of kv4_bytes(nkv, hd, cap) bytes at base (16-byte aligned).
inline Kv4View kv4_carve(uint8_t* base, int nkv, int hd, int cap) {
  Kv4View v;
  v.nkv = nkv;
  v.hd = hd;
  v.cap = cap;
  v.kc = base;
  v.vc = v.kc + nkv * v.code_head();
  v.ks = v.vc + nkv * v.code_head();
  v.vs = v.ks + nkv * v.scale_head();
  v.bad = v.vs + nkv * v.scale_head();
  return v;
}

// One key/value head of a view.
inline Kv4View kv4_head(Kv4View v, int h) {
  v.kc += h * v.code_head();
  v.vc += h * v.code_head();
  v.ks += h * v.scale_head();
  v.vs += h * v.scale_head();
  v.bad += (size_t)h * (v.cap / kKv4Tile);
  v.nkv = 1;
  return v;
}

// Offset of the T bytes of value row r that lane ln (dims 32t + 2ln, +1) holds.
template <int HD>
__device__ __forceinline__ size_t kv4_value_offset(int64_t r, int ln) {
  constexpr int T = HD / 32;
  const int q = (int)(r & 31), lk = (q & 15) >> 2, j = (q & 3) + ((q >> 4) << 2);
  const int off = j * T;
  return (size_t)(r >> 5) * (16 * HD) + (size_t)((off >> 4) * 1024 + (16 * lk + ln) * 16 + (off & 15));
}

// The scale byte of a block whose largest absolute value is big, and the value's 4-bit code at that scale.
__device__ __forceinline__ int kv4_scale_byte(float big) {
  const unsigned u = __float_as_uint(big);
  const int e = (int)(u >> 23) - 127;  // big is not negative; subnormals lie far below the least scale
  if (e == 128) return 255;
  return min(max(e - 2 + ((u & 0x7FFFFFu) >= 0x600000u ? 1 : 0), kKv4MinExp), kKv4MaxExp) + 127;
}
__device__ __forceinline__ unsigned kv4_code(float x, int scale_byte) {
  // 2^-(e) as two factors, each in range; both products are exact but where the result is far below the first step
  const int n = 127 - scale_byte, h = n / 2;
  const float a = (fabsf(x) * __uint_as_float((unsigned)(127 + h) << 23)) * __uint_as_float((unsigned)(127 + n - h) << 23);
  unsigned c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  if (scale_byte == 255) c = 0;
  return c | (x < 0.f && c ? 8u : 0u);
}
__device__ __forceinline__ float kv4_scale(unsigned byte) {
  return byte == 255u ? __builtin_nanf("") : __uint_as_float(byte << 23);
}

// Rows k, v -> rows [row0, row0 + n) of the cache.
int kv4_append(const Kv4View& c, int row0, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, int n, hipStream_t s);
int kv4_read(const Kv4View& c, int start, int n, float* k, float* v, hipStream_t s);
int prepare_kv4_kernels();
// weights: for calls that add to the rows' weights.
size_t kv4_attend_work(const Kv4View& c, int n_head, int n, bool weights);
// gate: see AttendOut (f32 [n][n_head][head_dim]).
int kv4_attend(const Kv4View& c, int len, const void* q, int64_t ldq, int type, int n_head, int n, float scale, float* weights,
               int64_t ldw, void* out, int64_t ldo, void* work, hipStream_t s, const float* gate);
int kv4_evict(const Kv4View& c, int len, const float* weights, int64_t ldw, int keep, int recent, const Kv4View& dst,
              float* dst_weights, int64_t ld_dst, int32_t* kept, hipStream_t s);

}  // namespace dz
