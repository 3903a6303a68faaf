// Shared pieces of the 8-bit KV cache and of the attention kernels over it and
// over uncompressed keys and values: element conversions, parameters, and the
// list of 64-token tiles a group of queries has to read.
#pragma once

#include <math.h>

#include "tq_common.h"

namespace tq {
namespace kv {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int TILE = 64;     // tokens per tile (and per transposed tile of value codes)
constexpr int HALF = TILE / 2;
constexpr int DEC_WAVES = 4, DEC_ROWS = 16;            // tq_kv_decode.h: waves and most rows per workgroup
constexpr int DENSE = -1;    // format of uncompressed keys and values (else TQ_KV8_*)
// The reference of the softmax's weights, in base 2: this far below the running
// maximum. fp16 weights then reach 2^14, which leaves those down to 2^-28 of the
// largest normal, and smaller ones 2^-39 apart; bf16 weights stay below 2^-12,
// so that sums over 2^12 tokens of bf16's largest values stay finite.
template <bool BF>
constexpr float W_SHIFT = BF ? -20.f : 13.f;
// The chunk kernel moves its reference only when a weight would grow past this
// (in base 2) above what W_SHIFT allows: few tiles do after the first ones.
template <bool BF>
constexpr float W_SLACK = BF ? 8.f : 1.f;
constexpr float QMAX_INT8 = 127.f, QMAX_E4M3 = 448.f;
constexpr float TINY = 0x1p-110f;  // blocks below are stored as 0: QMAX / a stays finite

// Four int8 codes to two dwords of exact fp16: with the sign bit flipped, byte
// u = code + 128 under 0x64 is the fp16 number 1024 + u, and 1152 comes off.
__device__ inline u2 int8x4_f16(uint32_t w) {
  w ^= 0x80808080u;
  const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
  const h2 lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
  const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
  return u2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// Four int8 codes to two dwords of exact bf16 (7 significant bits): the upper
// halves of their float32 values. One instruction per code, which the compiler
// makes two of.
template <int BYTE>
__device__ inline uint32_t int8_f32(uint32_t w) {
  uint32_t r;
  if constexpr (BYTE == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(r) : "v"(w));
  if constexpr (BYTE == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(r) : "v"(w));
  if constexpr (BYTE == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(r) : "v"(w));
  if constexpr (BYTE == 3) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(r) : "v"(w));
  return r;
}
__device__ inline u2 int8x4_bf16(uint32_t w) {
  return u2{__builtin_amdgcn_perm(int8_f32<1>(w), int8_f32<0>(w), 0x07060302u),
            __builtin_amdgcn_perm(int8_f32<3>(w), int8_f32<2>(w), 0x07060302u)};
}

// Four codes of format FMT to two dwords of exact fp16 (BF: bf16).
template <int FMT, bool BF>
__device__ inline u2 codes4(uint32_t w) {
  if constexpr (FMT == TQ_KV8_INT8) {
    return BF ? int8x4_bf16(w) : int8x4_f16(w);
  } else if constexpr (BF) {
    return u2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
  } else {
    return u2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
  }
}

// One code as float32.
template <int FMT>
__device__ inline float code_value(uint32_t byte) {
  if constexpr (FMT == TQ_KV8_INT8)
    return (float)(int8_t)byte;
  else
    return __builtin_amdgcn_cvt_f32_fp8(byte, 0);
}

// Element bits of a 16-bit type <-> float32 (to the nearest, ties to even).
template <bool BF>
__device__ inline float elem(uint32_t h) {
  if constexpr (BF)
    return __uint_as_float(h << 16);
  else
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <bool BF>
__device__ inline uint32_t bits2(float a, float b) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
  else
    return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
}

// Values that are infinite or NaN: taken out of the product (0 x inf would reach
// rows that do not see them, and the remainders of split weights are 0) and
// counted in one of their own, marks x seen: 1 for inf, 128 for -inf, 2^14 for
// NaN (at most 64 of each per tile: exact), which gives what the rows that see
// them get.
// The larger of two pairs of 16-bit magnitudes (signs off), half by half; whether
// either is that of an infinity or NaN.
__device__ inline uint32_t top16(uint32_t a, uint32_t x) {
  typedef uint16_t s2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s2, a), __builtin_bit_cast(s2, x & 0x7fff7fffu)));
}
template <bool BF>
__device__ inline bool odd16(uint32_t top) {
  constexpr uint32_t ex = BF ? 0x7f80u : 0x7c00u;
  return (top & 0xffffu) >= ex || top >> 16 >= ex;
}
template <bool BF>
__device__ inline uint32_t mark16(uint32_t h) {
  constexpr uint32_t ex = BF ? 0x7f80u : 0x7c00u;
  if ((h & ex) != ex) return 0u;
  if (h & 0x7fffu & ~ex) return BF ? 0x4680u : 0x7400u;  // 16384
  return h & 0x8000u ? (BF ? 0x4300u : 0x5800u) : (BF ? 0x3f80u : 0x3c00u);  // 128, 1
}
template <bool BF>
__device__ inline u4 marks(u4& v) {
  u4 m;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = mark16<BF>(v[i] & 0xffffu), hi = mark16<BF>(v[i] >> 16);
    m[i] = lo | hi << 16;
    v[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
  }
  return m;
}
__device__ inline float marked(float c) {
  const uint32_t n = (uint32_t)c;
  const float up = n & 127u ? INFINITY : 0.f, down = n & 127u << 7 ? -INFINITY : 0.f;
  return n >> 14 ? NAN : up + down;
}
// Bit i: the row at position pos sees token t + i (i < count <= 16): t + i <
// end, <= pos, and > low or < sinks.
__device__ inline uint32_t seen_bits(int t, int count, int end, int pos, int low, int sinks) {
  const auto below = [&](int x) { return (1u << min(max(x - t, 0), count)) - 1u; };  // tokens before x
  return below(min(end, pos + 1)) & (~below(low + 1) | below(sinks));
}
// x where bit k is set, else -inf (a bit field and a merge).
__device__ inline float seen_or(uint32_t bits, int k, float x) {
  const uint32_t m = __builtin_amdgcn_sbfe(bits, k, 1);
  return __uint_as_float((__float_as_uint(x) & m) | (0xff800000u & ~m));
}
// 1.0 in the halves whose token is seen (bits 0 and 1)
template <bool BF>
__device__ inline uint32_t seen2(uint32_t bits) {
  constexpr uint32_t one = BF ? 0x3f80u : 0x3c00u;
  return (bits & 1u ? one : 0u) | (bits & 2u ? one << 16 : 0u);
}

// acc plus both elements.
template <bool BF>
__device__ inline float add2(uint32_t x, float acc) {
  if constexpr (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, x), b2{(__bf16)1.f, (__bf16)1.f}, acc, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{(_Float16)1.f, (_Float16)1.f}, acc, false);
}

template <bool BF>
__device__ inline f4 mma16(u4 a, u4 b, f4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ inline f16v mma32(u4 a, u4 b, f16v c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Reductions over a wave without trips through LDS: rotations within rows of 16
// lanes, then exchanges of rows and of halves. Every lane gets the result.
template <int N>
__device__ inline uint32_t row_rotated(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x120 + N, 0xf, 0xf, true);
}
template <typename F>
__device__ inline uint32_t rows_joined(uint32_t x, F f) {  // over the lanes that differ in bits 4 and 5
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(b[0], b[1]);
}
template <typename F>
__device__ inline uint32_t wave_joined(uint32_t x, F f) {
  x = f(x, row_rotated<8>(x));
  x = f(x, row_rotated<4>(x));
  x = f(x, row_rotated<2>(x));
  x = f(x, row_rotated<1>(x));
  return rows_joined(x, f);
}
__device__ inline uint32_t max_bits(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
__device__ inline uint32_t sum_bits(uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }
__device__ inline float wave_max(float x) { return __uint_as_float(wave_joined(__float_as_uint(x), max_bits)); }
__device__ inline float wave_sum(float x) { return __uint_as_float(wave_joined(__float_as_uint(x), sum_bits)); }

// The maximum over the lanes that differ in bits 4 and 5 (16) or 5 (32) of their
// number.
template <int FROM>
__device__ inline float lanes_max(float x) {
  if constexpr (FROM == 16) return __uint_as_float(rows_joined(__float_as_uint(x), max_bits));
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Rows of an operand: element (b, h, t, i) at p[b * sb + h * sh + t * st + i].
struct Rows {
  const void* p;
  int64_t sb, sh, st;
};

struct Params {
  Rows q, out, k, v;  // k, v: uncompressed keys and values
  const uint8_t *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  const uint16_t *k_tail, *v_tail;
  int64_t cap;
  const int32_t* len_b;
  float* ws;              // partials: (M, m, l, -) per slot, then O (slots, D)
  int64_t o_off;          // floats before the O part
  int32_t batch, hkv, group, n_q, rows;  // rows = group * n_q per kv head, row = i * group + head
  int32_t max_len, block_shift, window, sinks;
  int32_t wgs;            // decode: workgroups that share the list of all tiles; 0: one per (sequence, kv head)
  int32_t splits, chunk;  // chunk kernel: a split is `chunk` consecutive tiles
  int32_t tile_rows, row_tiles;  // chunk kernel: rows per workgroup (128, 256), and how many such per kv head
  int32_t out_f32;
  float scale;            // times log2 e: scores are kept in base 2
};

// The tiles that queries at positions pmin .. pmax have to read: the first
// `sinks` of a windowed call, those from the first query's window on, and the
// tail of an 8-bit cache as the last one.
struct Tiles {
  int main_len;       // tokens held in whole tiles (codes, or all of them)
  int sink_tiles;     // tiles before the gap
  int first;          // first tile after the gap
  int n_main, n;      // tiles without / with the tail
  __device__ int at(int i) const { return i < sink_tiles ? i : first + i - sink_tiles; }
};

__device__ inline Tiles tiles_of(int len, bool cached, int block_shift, int pmin, int pmax, int window, int sinks) {
  Tiles t;
  t.main_len = cached ? (len >> block_shift) << block_shift : len;
  const int hi = max(0, min(pmax + 1, t.main_len));
  const int hi_t = (hi + TILE - 1) / TILE;
  const int lo = window ? max(0, pmin - window + 1) : 0;
  t.sink_tiles = window ? min(hi_t, (sinks + TILE - 1) / TILE) : 0;
  t.first = min(max(lo / TILE, t.sink_tiles), hi_t);
  t.n_main = t.sink_tiles + hi_t - t.first;
  t.n = t.n_main + (cached && len > t.main_len && pmax >= t.main_len ? 1 : 0);
  return t;
}

__device__ inline int length_of(const Params& p, int b) {
  return p.len_b ? min(max(p.len_b[b], 0), p.max_len) : p.max_len;
}

// Decode's list of tiles: those of (sequence 0, kv head 0), (0, 1), ... Each of
// p.wgs workgroups takes `per` consecutive ones, whatever sequences they belong
// to, so that sequences of any lengths load the chip evenly. The part of
// (sequence, kv head) unit u that workgroup w holds goes to partial slot w + u:
// along the list each step is to the next w or the next u, so slots are distinct.
// In the list a unit's tiles are filled up to a multiple of DEC_WAVES (places
// without a tile): as many as its waves take at once, so that short shares hold
// no parts of two units, which would take twice as long.
struct Share {
  int total, per;   // places in the list, places per workgroup
};

__device__ inline int decode_places(const Params& p, bool cached, int b) {
  const int len = length_of(p, b);
  const int n = tiles_of(len, cached, p.block_shift, len - p.n_q, len - 1, p.window, p.sinks).n;
  return (n + DEC_WAVES - 1) / DEC_WAVES * DEC_WAVES;
}

// Inclusive sums over the wave's lanes: within rows of 16, then the rows before.
__device__ inline int wave_scan(int n) {
  n += __builtin_amdgcn_update_dpp(0, n, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  n += __builtin_amdgcn_update_dpp(0, n, 0x112, 0xf, 0xf, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x114, 0xf, 0xf, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x118, 0xf, 0xf, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3, :31 to 2 and 3
  return n + __builtin_amdgcn_update_dpp(0, n, 0x143, 0xc, 0xf, false);
}

// The share, and for workgroup `wg` (>= 0) the sequence that its first tile
// belongs to (b; -1: no tiles) or for sequence b: the tiles before it.
__device__ inline Share share_of(const Params& p, bool cached, int wg, int& b, int& before) {
  const int lane = threadIdx.x & 63;
  Share s;
  const auto per_of = [&](int total) {
    s.total = total;
    s.per = max(DEC_WAVES, ((total + p.wgs - 1) / p.wgs + DEC_WAVES - 1) / DEC_WAVES * DEC_WAVES);
  };
  if (p.len_b == nullptr) {
    const int n = decode_places(p, cached, 0) * p.hkv;
    per_of(n * p.batch);
    if (wg >= 0) b = wg * s.per < s.total ? wg * s.per / n : -1;
    before = b * n;
    return s;
  }
  int n = lane < p.batch ? decode_places(p, cached, lane) * p.hkv : 0;
  int sum = wave_scan(n);  // of the first 64 sequences
  int total = __builtin_amdgcn_readlane(sum, 63);
  for (int b0 = 64; b0 < p.batch; b0 += 64)
    total += __builtin_amdgcn_readlane(wave_scan(b0 + lane < p.batch ? decode_places(p, cached, b0 + lane) * p.hkv : 0), 63);
  per_of(total);
  const int at = wg * s.per;
  if (wg >= 0 && at >= s.total) {
    b = -1;
    return s;
  }
  int base = 0;
  for (int b0 = 0;; b0 += 64) {
    int l = -1;
    if (wg >= 0) {
      const uint64_t past = __ballot(base + sum > at);
      if (past) l = __builtin_ctzll(past);
    } else if (b < b0 + 64) {
      l = b - b0;
    }
    if (l >= 0) {
      before = base + (l > 0 ? __builtin_amdgcn_readlane(sum, l - 1) : 0);
      b = b0 + l;
      return s;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
    n = b0 + 64 + lane < p.batch ? decode_places(p, cached, b0 + 64 + lane) * p.hkv : 0;
    sum = wave_scan(n);
  }
}

// Kernels by head dim (one source file each): FMT of DENSE / TQ_KV8_*.
template <int D>
hipError_t launch_decode(const Params& p, bool bf16, int fmt, hipStream_t stream);
template <int D>
hipError_t launch_chunk(const Params& p, bool bf16, int fmt, hipStream_t stream);

}  // namespace kv
}  // namespace tq
