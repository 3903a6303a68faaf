// Shared pieces of the 8-bit KV cache and of the attention kernels over it and
// over uncompressed keys and values: element conversions, parameters, and the
// list of 64-token tiles a group of queries has to read.
#pragma once

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
constexpr int DEC_WAVES = 4, DEC_ROWS = 16;            // tq_kv_decode.h: waves and most rows per workgroup
constexpr int CH_WAVES = 4, CH_ROWS = CH_WAVES * 32;   // tq_kv_chunk.h
constexpr int DENSE = -1;    // format of uncompressed keys and values (else TQ_KV8_*)
// The reference of the softmax's weights is kept this far (in base 2) below the
// running maximum: weights up to 2^14 in fp16, which leaves those down to 2^-28
// of the largest normal, and smaller ones 2^-39 apart.
constexpr float W_SHIFT = 14.f;
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
// halves of their float32 values.
__device__ inline u2 int8x4_bf16(uint32_t w) {
  const float a = (float)(int8_t)w, b = (float)(int8_t)(w >> 8), c = (float)(int8_t)(w >> 16), d = (float)(int8_t)(w >> 24);
  return u2{__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u),
            __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x07060302u)};
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
  float* ws;              // partials: ML (units, splits, 4), then O (units, splits, D)
  int64_t o_off;          // floats before the O part
  int32_t batch, hkv, group, n_q, rows;  // rows = group * n_q per kv head, row = i * group + head
  int32_t max_len, block_shift, window, sinks;
  int32_t splits, chunk;  // a split is `chunk` consecutive tiles
  int32_t row_tiles;      // row tiles of a kv head (chunk kernel)
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

// Kernels by head dim (one source file each): FMT of DENSE / TQ_KV8_*.
template <int D>
hipError_t launch_decode(const Params& p, bool bf16, int fmt, hipStream_t stream);
template <int D>
hipError_t launch_chunk(const Params& p, bool bf16, int fmt, hipStream_t stream);

}  // namespace kv
}  // namespace tq
