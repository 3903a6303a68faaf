// 8-bit KV cache: quantising keys and values as they are written, and reading
// them back. Both are bound by memory: 2 bytes in and 1 out per element (and
// back). One workgroup takes one 64-token tile of one (row, side), whose value
// codes are 64 whole bytes per dim.
//
// Write: the tile stays in registers between its blocks' maxima and its codes.
// Maxima are taken on the absolute values' bits, which order 16-bit floats and
// put infinities and NaN on top; a wave's loads lie in one group of 16 tokens.
// Codes are x * (QMAX / a) in float32, one rounding (v_rndne / v_cvt_pk_fp8, ties
// to even). Value codes turn in LDS, 4 x 4 bytes at a time. The workgroup of a
// call's first tile also moves the incomplete block: it has read the tail before
// it writes there.
//
// Measured, 8 kv heads, head dim 128, bf16, int8: 8192 tokens written in 13.3 us
// (3.8 TB/s; 2.8 us for one token), 32,768 read back in 32.0 us (6.3 TB/s).

#include "tq_kv8.h"

namespace tq {
namespace kv {
namespace {

constexpr int WT = 256;

struct WriteParams {
  tq_kv8_store s;
  Rows k, v;
  const int32_t *start_b, *n_new_b;
  int32_t start, n_new, slots, shift;
};

// Bytes of four dwords, as rows and columns exchanged.
__device__ inline void turn4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

template <int D, int BLOCK, bool BF>
__global__ __launch_bounds__(WT) void write_kernel(const WriteParams p) {
  constexpr int PER = TILE * D / 8 / WT;   // pieces of 8 elements per thread
  constexpr int PARTS = D / 32;            // maxima of a group of 16 tokens
  constexpr int LP = D + 4;                // LDS row pitch of codes, bytes
  __shared__ __align__(16) uint8_t lt[TILE * LP];
  __shared__ uint32_t part[4][PARTS];

  const int side = blockIdx.x & 1;
  const int j = (blockIdx.x >> 1) % p.slots, bh = (blockIdx.x >> 1) / p.slots;
  const int b = bh / p.s.heads, h = bh - b * p.s.heads;
  const int start = p.start_b ? p.start_b[b] : p.start;
  const int n = p.n_new_b ? p.n_new_b[b] : p.n_new;
  if (n <= 0 || n > p.n_new || start < 0 || start > p.s.cap - n) return;
  const int end = start + n;
  const int t0 = (start / TILE + j) * TILE;
  const int first = max(t0, start / BLOCK * BLOCK), last = min(t0 + TILE, end / BLOCK * BLOCK);  // of completed blocks

  const Rows& src = side ? p.v : p.k;
  const uint16_t* x0 = (const uint16_t*)src.p + (int64_t)b * src.sb + (int64_t)h * src.sh;
  uint16_t* tail = (uint16_t*)(side ? p.s.v_tail : p.s.k_tail) + (int64_t)bh * BLOCK * D;

  if (first < last) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int vec = i * WT + threadIdx.x, t = t0 + vec / (D / 8), c = vec % (D / 8);
      x[i] = u4{0, 0, 0, 0};
      if (t >= first && t < last) x[i] = t < start ? *(const u4*)(tail + t % BLOCK * D + c * 8) : *(const u4*)(x0 + (int64_t)(t - start) * src.st + c * 8);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = top16(top, x[i][k]);
      top = max(top & 0xffffu, top >> 16);
      top = wave_joined(top, [](uint32_t a, uint32_t b) { return max(a, b); });
      const int w = i * (WT / 64) + wave;  // 64 pieces; 2 D of them are 16 tokens
      if (lane == 0) part[w / PARTS][w % PARTS] = top;
    }
    __syncthreads();
    const float qmax = p.s.fmt == TQ_KV8_INT8 ? QMAX_INT8 : QMAX_E4M3;
    float inv[TILE / BLOCK];
#pragma unroll
    for (int g = 0; g < TILE / BLOCK; ++g) {
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < BLOCK / 16 * PARTS; ++k) top = max(top, part[g * (BLOCK / 16) + k / PARTS][k % PARTS]);
      const float a = elem<BF>(top);
      const bool finite = top < (BF ? 0x7f80u : 0x7c00u), codes = finite && a >= TINY;
      inv[g] = codes ? qmax / a : 0.f;
      const int t = t0 + g * BLOCK;
      if (threadIdx.x == 0 && t >= first && t < last)
        (side ? p.s.v_scales : p.s.k_scales)[(int64_t)bh * (p.s.cap >> p.shift) + t / BLOCK] = codes ? a / qmax : finite ? 0.f : NAN;
    }

    uint8_t* kc = p.s.k_codes + ((int64_t)bh * p.s.cap + t0) * D;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int vec = i * WT + threadIdx.x, t = vec / (D / 8), c = vec % (D / 8);
      float f = inv[0];
#pragma unroll
      for (int g = 1; g < TILE / BLOCK; ++g) f = t / BLOCK == g ? inv[g] : f;
      u2 w = {0, 0};
      if (f > 0.f) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float c0 = elem<BF>(x[i][2 * k] & 0xffff) * f, c1 = elem<BF>(x[i][2 * k] >> 16) * f;
          const float c2 = elem<BF>(x[i][2 * k + 1] & 0xffff) * f, c3 = elem<BF>(x[i][2 * k + 1] >> 16) * f;
          if (p.s.fmt == TQ_KV8_INT8) {
            w[k] = ((uint32_t)(int)rintf(c0) & 0xff) | ((uint32_t)(int)rintf(c1) & 0xff) << 8 | ((uint32_t)(int)rintf(c2) & 0xff) << 16 |
                   (uint32_t)(int)rintf(c3) << 24;
          } else {
            w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(c0, c1, 0, false);
            w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(c2, c3, w[k], true);
          }
        }
      }
      if (side == 0) {
        if (t0 + t >= first && t0 + t < last) *(u2*)(kc + vec * 8) = w;
      } else {
        *(uint32_t*)(lt + t * LP + c * 8) = w.x;
        *(uint32_t*)(lt + t * LP + c * 8 + 4) = w.y;
      }
    }
    if (side == 1) {
      __syncthreads();
      uint8_t* vc = p.s.v_codes + ((int64_t)bh * p.s.cap + t0) * D;
#pragma unroll
      for (int i = threadIdx.x; i < D / 4 * (TILE / 8); i += WT) {  // 4 dims x 8 tokens
        const int c = i % (TILE / 8), dim = i / (TILE / 8) * 4, t = t0 + c * 8;
        if (t < first || t >= last) continue;
        uint32_t w[2][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k / 4][k % 4] = *(const uint32_t*)(lt + (c * 8 + k) * LP + dim);
        turn4(w[0]);
        turn4(w[1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) *(u2*)(vc + (dim + k) * TILE + c * 8) = u2{w[0][k], w[1][k]};
      }
    }
  }

  if (j == 0) {  // the incomplete block's tokens (what the tail held has been read)
    __syncthreads();
    const int at = max(start, end / BLOCK * BLOCK);
    for (int i = threadIdx.x; i < (end - at) * (D / 8); i += WT) {
      const int t = at + i / (D / 8), c = i % (D / 8);
      *(u4*)(tail + t % BLOCK * D + c * 8) = *(const u4*)(x0 + (int64_t)(t - start) * src.st + c * 8);
    }
  }
}

struct ReadParams {
  tq_kv8_store s;
  const int32_t* len_b;
  int32_t len, start, n, shift, tiles;
  void *k, *v;
};

// 8 values to out (element offset at), rounded once.
template <int OUT>
__device__ inline void put8(void* out, int64_t at, const float (&x)[8]) {
  if constexpr (OUT == TQ_F32) {
    float* o = (float*)out + at;
    *(f4*)o = f4{x[0], x[1], x[2], x[3]};
    *(f4*)(o + 4) = f4{x[4], x[5], x[6], x[7]};
  } else {
    constexpr bool B = OUT == TQ_BF16;
    *(u4*)((uint16_t*)out + at) = u4{bits2<B>(x[0], x[1]), bits2<B>(x[2], x[3]), bits2<B>(x[4], x[5]), bits2<B>(x[6], x[7])};
  }
}

template <int D, int FMT, int OUT>
__global__ __launch_bounds__(WT) void read_kernel(const ReadParams p) {
  constexpr int LP = D + 4;
  __shared__ __align__(16) uint8_t lt[TILE * LP];
  const int side = blockIdx.x & 1;
  const int tile = p.start / TILE + (blockIdx.x >> 1) % p.tiles, bh = (blockIdx.x >> 1) / p.tiles;
  const int len = p.len_b ? min((int64_t)max(p.len_b[bh / p.s.heads], 0), p.s.cap) : p.len;
  const int held = len >> p.shift << p.shift, t0 = tile * TILE;
  const float* scales = (side ? p.s.v_scales : p.s.k_scales) + (int64_t)bh * (p.s.cap >> p.shift);
  const uint16_t* tail = (const uint16_t*)(side ? p.s.v_tail : p.s.k_tail) + ((int64_t)bh << p.shift) * D;
  void* out = side ? p.v : p.k;
  const uint8_t* kc = p.s.k_codes + ((int64_t)bh * p.s.cap + t0) * D;

  if (side && t0 < held) {
    const uint8_t* vc = p.s.v_codes + ((int64_t)bh * p.s.cap + t0) * D;
    for (int i = threadIdx.x; i < D * TILE / 16; i += WT) {
      const int dim = i / (TILE / 16), c = i % (TILE / 16);
      const u4 w = *(const u4*)(vc + dim * TILE + c * 16);
#pragma unroll
      for (int k = 0; k < 16; ++k) lt[(c * 16 + k) * LP + dim] = (uint8_t)(w[k / 4] >> 8 * (k % 4));
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < TILE * D / 8; i += WT) {
    const int t = i / (D / 8), c = i % (D / 8), at = t0 + t;
    if (at < p.start || at >= p.start + p.n) continue;
    float x[8];
    if (at < held) {
      const u2 w = side ? u2{*(const uint32_t*)(lt + t * LP + c * 8), *(const uint32_t*)(lt + t * LP + c * 8 + 4)}
                        : *(const u2*)(kc + t * D + c * 8);
      const float s = scales[at >> p.shift];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = code_value<FMT>(w[k / 4] >> 8 * (k % 4) & 0xff) * s;
    } else if (at < len) {
      const u4 w = *(const u4*)(tail + (at - held) * D + c * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t e = k & 1 ? w[k / 2] >> 16 : w[k / 2] & 0xffff;
        x[k] = p.s.kv_dtype == TQ_BF16 ? elem<true>(e) : elem<false>(e);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = 0.f;
    }
    put8<OUT>(out, ((int64_t)bh * p.n + at - p.start) * D + c * 8, x);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int D, int BLOCK>
void launch_write(const WriteParams& p, uint32_t wgs, hipStream_t s) {
  if (p.s.kv_dtype == TQ_BF16)
    write_kernel<D, BLOCK, true><<<wgs, WT, 0, s>>>(p);
  else
    write_kernel<D, BLOCK, false><<<wgs, WT, 0, s>>>(p);
}
template <int D>
void launch_write(const WriteParams& p, uint32_t wgs, hipStream_t s) {
  if (p.s.block == 16)
    launch_write<D, 16>(p, wgs, s);
  else if (p.s.block == 32)
    launch_write<D, 32>(p, wgs, s);
  else
    launch_write<D, 64>(p, wgs, s);
}
template <int D, int FMT>
void launch_read(const ReadParams& p, int out, uint32_t wgs, hipStream_t s) {
  if (out == TQ_F16)
    read_kernel<D, FMT, TQ_F16><<<wgs, WT, 0, s>>>(p);
  else if (out == TQ_BF16)
    read_kernel<D, FMT, TQ_BF16><<<wgs, WT, 0, s>>>(p);
  else
    read_kernel<D, FMT, TQ_F32><<<wgs, WT, 0, s>>>(p);
}
template <int D>
void launch_read(const ReadParams& p, int out, uint32_t wgs, hipStream_t s) {
  if (p.s.fmt == TQ_KV8_INT8)
    launch_read<D, TQ_KV8_INT8>(p, out, wgs, s);
  else
    launch_read<D, TQ_KV8_E4M3>(p, out, wgs, s);
}

}  // namespace

int check_store(const tq_kv8_store* s) {
  if (s == nullptr) return set_error(TQ_ERR_INVALID, "kv8: NULL store");
  if (s->fmt != TQ_KV8_INT8 && s->fmt != TQ_KV8_E4M3) return set_error(TQ_ERR_UNSUPPORTED, "kv8: unknown format %d", s->fmt);
  if (s->d != 64 && s->d != 96 && s->d != 128 && s->d != 256)
    return set_error(TQ_ERR_UNSUPPORTED, "kv8: head_dim %d: use 64, 96, 128 or 256", s->d);
  if (s->block != 16 && s->block != 32 && s->block != 64)
    return set_error(TQ_ERR_UNSUPPORTED, "kv8: blocks of %d tokens: use 16, 32 or 64", s->block);
  if (s->kv_dtype != TQ_F16 && s->kv_dtype != TQ_BF16) return set_error(TQ_ERR_UNSUPPORTED, "kv8: keys and values are fp16 or bf16");
  if (s->batch < 0 || s->heads < 1) return set_error(TQ_ERR_INVALID, "kv8: batch %d, heads %d", s->batch, s->heads);
  if ((int64_t)s->batch * s->heads >= (int64_t)1 << 31) return set_error(TQ_ERR_UNSUPPORTED, "kv8: too many sequences and heads");
  if (s->cap < 0 || s->cap % TILE || s->cap >= (int64_t)1 << 31)
    return set_error(TQ_ERR_INVALID, "kv8: room for %lld tokens: a multiple of 64 below 2^31", (long long)s->cap);
  if (s->batch == 0 || s->cap == 0) return TQ_OK;
  const void* const p[] = {s->k_codes, s->v_codes, s->k_scales, s->v_scales, s->k_tail, s->v_tail};
  for (const void* q : p)
    if (q == nullptr) return set_error(TQ_ERR_INVALID, "kv8: NULL array in the store");
  if (!aligned16(s->k_codes) || !aligned16(s->v_codes) || !aligned16(s->k_tail) || !aligned16(s->v_tail))
    return set_error(TQ_ERR_INVALID, "kv8: codes and tails need 16-byte alignment");
  return TQ_OK;
}

int check_rows(const tq_rows4& r, const char* what) {
  if (r.p == nullptr) return set_error(TQ_ERR_INVALID, "%s: NULL", what);
  if (!aligned16(r.p)) return set_error(TQ_ERR_INVALID, "%s: needs 16-byte alignment", what);
  if (r.sb % 8 || r.sh % 8 || r.st % 8) return set_error(TQ_ERR_INVALID, "%s: strides must be multiples of 8 elements", what);
  return TQ_OK;
}

}  // namespace kv
}  // namespace tq

using namespace tq;

extern "C" int tq_kv8_write(const tq_kv8_store* store, const tq_rows4* k, const tq_rows4* v, const int32_t* start_b, int32_t start,
                            const int32_t* n_new_b, int32_t n_new, void* stream) {
  if (int rc = kv::check_store(store)) return rc;
  if (k == nullptr || v == nullptr) return set_error(TQ_ERR_INVALID, "kv8 write: NULL keys or values");
  if (n_new < 0) return set_error(TQ_ERR_INVALID, "kv8 write: %d tokens", n_new);
  if (n_new == 0 || store->batch == 0) return TQ_OK;
  if (n_new > store->cap || (start_b == nullptr && (start < 0 || start > store->cap - n_new)))
    return set_error(TQ_ERR_INVALID, "kv8 write: tokens %d .. %lld past the room for %lld", start, (long long)start + n_new - 1,
                     (long long)store->cap);
  if (int rc = kv::check_rows(*k, "kv8 write: keys")) return rc;
  if (int rc = kv::check_rows(*v, "kv8 write: values")) return rc;
  kv::WriteParams p{};
  p.s = *store;
  p.k = {k->p, k->sb, k->sh, k->st};
  p.v = {v->p, v->sb, v->sh, v->st};
  p.start_b = start_b;
  p.n_new_b = n_new_b;
  p.start = start;
  p.n_new = n_new;
  p.slots = (n_new + kv::TILE - 2) / kv::TILE + 1;  // tiles that n_new tokens touch at most, wherever they start
  if (start_b == nullptr) p.slots = (start + n_new - 1) / kv::TILE - start / kv::TILE + 1;
  p.shift = store->block == 16 ? 4 : store->block == 32 ? 5 : 6;
  const int64_t wgs = (int64_t)store->batch * store->heads * p.slots * 2;
  if (wgs >= (int64_t)1 << 31) return set_error(TQ_ERR_UNSUPPORTED, "kv8 write: too many blocks in one call");
  hipStream_t s = (hipStream_t)stream;
  if (store->d == 64)
    kv::launch_write<64>(p, (uint32_t)wgs, s);
  else if (store->d == 96)
    kv::launch_write<96>(p, (uint32_t)wgs, s);
  else if (store->d == 128)
    kv::launch_write<128>(p, (uint32_t)wgs, s);
  else
    kv::launch_write<256>(p, (uint32_t)wgs, s);
  TQ_LAUNCH_CHECK("kv8 write");
  return TQ_OK;
}

extern "C" int tq_kv8_read(const tq_kv8_store* store, const int32_t* len_b, int32_t len, int32_t start, int32_t n,
                           int32_t out_dtype, void* k_out, void* v_out, void* stream) {
  if (int rc = kv::check_store(store)) return rc;
  if (out_dtype != TQ_F16 && out_dtype != TQ_BF16 && out_dtype != TQ_F32)
    return set_error(TQ_ERR_UNSUPPORTED, "kv8 read: unknown output type %d", out_dtype);
  if (n < 0 || start < 0 || start > store->cap - n)
    return set_error(TQ_ERR_INVALID, "kv8 read: tokens %d .. %lld past the room for %lld", start, (long long)start + n - 1,
                     (long long)store->cap);
  if (len_b == nullptr && (len < 0 || len > store->cap)) return set_error(TQ_ERR_INVALID, "kv8 read: length %d", len);
  if (n == 0 || store->batch == 0) return TQ_OK;
  if (k_out == nullptr || v_out == nullptr || !kv::aligned16(k_out) || !kv::aligned16(v_out))
    return set_error(TQ_ERR_INVALID, "kv8 read: outputs need 16-byte alignment");
  kv::ReadParams p{};
  p.s = *store;
  p.len_b = len_b;
  p.len = len;
  p.start = start;
  p.n = n;
  p.shift = store->block == 16 ? 4 : store->block == 32 ? 5 : 6;
  p.tiles = (start + n - 1) / kv::TILE - start / kv::TILE + 1;
  p.k = k_out;
  p.v = v_out;
  const int64_t wgs = (int64_t)store->batch * store->heads * p.tiles * 2;
  if (wgs >= (int64_t)1 << 31) return set_error(TQ_ERR_UNSUPPORTED, "kv8 read: too many tokens in one call");
  hipStream_t s = (hipStream_t)stream;
  if (store->d == 64)
    kv::launch_read<64>(p, out_dtype, (uint32_t)wgs, s);
  else if (store->d == 96)
    kv::launch_read<96>(p, out_dtype, (uint32_t)wgs, s);
  else if (store->d == 128)
    kv::launch_read<128>(p, out_dtype, (uint32_t)wgs, s);
  else
    kv::launch_read<256>(p, out_dtype, (uint32_t)wgs, s);
  TQ_LAUNCH_CHECK("kv8 read");
  return TQ_OK;
}
