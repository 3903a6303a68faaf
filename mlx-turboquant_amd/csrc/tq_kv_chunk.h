// Causal attention of many query rows per kv head (a chunk of query tokens
// times the query heads of the kv head) over an 8-bit KV cache or uncompressed
// 16-bit keys and values.
//
// A workgroup of 4 waves takes 128 rows, 32 per wave, row = token * group +
// head, and goes over the 64-token tiles that they see; K and V pass through
// LDS in 16 bits, V transposed. MFMA 32x32x16 bounds it (4 D multiply-adds per
// pair), then the softmax's exponentials.
//
// Scores, transposed: S^T = K q^T. Key row m of a 32-token half tile is token m
// with bits 2 and 3 swapped, so that lane (column n, half h) holds, register by
// register, tokens 16k + 8h + 0 .. 7: the B operand of O^T = V^T P^T as it is.
//
// Codes are exact in both 16-bit types. Key scales multiply the scores. Value
// scales multiply the weights before these are rounded: for bf16 by the whole
// scale on exact codes; for fp16 (whose range the weights need) by scale / 2^e
// in [1, 2), with 2^e taken into V, exactly unless the block's largest value
// is below 2^-17 (then off by at most 2^-25, half the smallest fp16).
// Both are the same for 16 tokens, so uniform over a wave.
//
// Infinite and NaN values of 16-bit tiles are left out of the products, where
// they would reach rows that do not see them (0 x inf), and joined at the end
// (marks()).
#pragma once

#include <math.h>

#include "tq_kv8.h"

namespace tq {
namespace kv {

constexpr int CH_THREADS = CH_WAVES * 64;

template <int D, bool BF, int FMT>
struct Chunk {
  static constexpr bool CACHED = FMT != DENSE;
  static constexpr int KP = D + 8, VP = TILE + 8;  // row pitches: reads of 16 lanes hit 64 banks
  static constexpr int BUF = TILE * KP + D * VP;   // elements of a tile's K and V
  static constexpr int LDS = 2 * BUF * 2;
  // what a thread loads of a tile: pieces of 16 codes, or of 8 elements
  static constexpr int NK = (TILE * D / (CACHED ? 16 : 8) + CH_THREADS - 1) / CH_THREADS;
  static constexpr int NV = CACHED ? NK : (TILE / 4 * (D / 8) + CH_THREADS - 1) / CH_THREADS * 4;

  u4 kx[NK], vx[NV];  // on their way from memory

  // key row of token t of a tile: bits 2 and 3 swapped
  static __device__ int krow(int t) { return (t & ~12) | (t & 4) << 1 | (t & 8) >> 1; }

  // ------------------------------------------------------- a tile of codes
  __device__ void load8(const uint8_t* kc, const uint8_t* vc, int tile) {
    const u4* k = (const u4*)(kc + (int64_t)tile * (TILE * D));
    const u4* v = (const u4*)(vc + (int64_t)tile * (TILE * D));
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int i = j * CH_THREADS + threadIdx.x;
      if (TILE * D / 16 % CH_THREADS == 0 || i < TILE * D / 16) kx[j] = k[i], vx[j] = v[i];
    }
  }
  __device__ void store8(const Params& p, const float* vsc, int t0, int main_len, uint16_t* kl, uint16_t* vl) const {
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int i = j * CH_THREADS + threadIdx.x;
      if (TILE * D / 16 % CH_THREADS != 0 && i >= TILE * D / 16) break;
      const int t = i / (D / 16), c = i % (D / 16);
      uint16_t* d = kl + krow(t) * KP + c * 16;
      const u4 x = kx[j];
      const u2 a = codes4<FMT, BF>(x.x), b = codes4<FMT, BF>(x.y), e = codes4<FMT, BF>(x.z), f = codes4<FMT, BF>(x.w);
      *(u4*)d = u4{a.x, a.y, b.x, b.y};
      *(u4*)(d + 8) = u4{e.x, e.y, f.x, f.y};
    }
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int i = j * CH_THREADS + threadIdx.x;
      if (TILE * D / 16 % CH_THREADS != 0 && i >= TILE * D / 16) break;
      const int dim = i / (TILE / 16), c = i % (TILE / 16);
      uint16_t* d = vl + dim * VP + c * 16;
      const u4 x = vx[j];
      const u2 a = codes4<FMT, BF>(x.x), b = codes4<FMT, BF>(x.y), e = codes4<FMT, BF>(x.z), f = codes4<FMT, BF>(x.w);
      u4 lo = {a.x, a.y, b.x, b.y}, hi = {e.x, e.y, f.x, f.y};
      if constexpr (!BF) {
        const float s = value_power(vsc[(t0 + c * 16) >> p.block_shift]);
        const h8 sc = {(_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s};
        lo = __builtin_bit_cast(u4, __builtin_bit_cast(h8, lo) * sc);
        hi = __builtin_bit_cast(u4, __builtin_bit_cast(h8, hi) * sc);
      }
      *(u4*)d = lo;
      *(u4*)(d + 8) = hi;
    }
    if (t0 + TILE > main_len) {  // tokens not written yet: any bytes
      for (int i = threadIdx.x; i < TILE * D / 16; i += CH_THREADS) {
        uint16_t* d = vl + i / (TILE / 16) * VP + i % (TILE / 16) * 16;
        if (t0 + i % (TILE / 16) * 16 >= main_len) *(u4*)d = *(u4*)(d + 8) = u4{0, 0, 0, 0};
      }
    }
  }

  // 2^e of the value scale that fp16 values carry: codes * 2^e stay in fp16's range
  static __device__ float value_power(float s) {
    if (!(s > 0.f)) return 1.f;
    return ldexpf(1.f, min(max(ilogbf(s), -24), FMT == TQ_KV8_INT8 ? 9 : 7));
  }
  // what the weights carry (codes of a scale of 0 are 0: any weight will do)
  static __device__ float value_factor(float s) {
    if (s == 0.f) return 1.f;
    return BF ? s : s * (1.f / value_power(s));
  }

  // ------------------------------------------------- a tile of 16-bit tokens
  // nv tokens at rows 0 .. of kb, vb; zeros after them. Values as 4 tokens x 8
  // dims per thread, to be paired by tokens.
  static constexpr int KPIECES = TILE * D / 8, VTASKS = TILE / 4 * (D / 8);
  static __device__ u4 k_piece(const uint16_t* kb, int64_t kst, int nv, int i) {
    const int t = i / (D / 8), c = i % (D / 8);
    return i < KPIECES && t < nv ? *(const u4*)(kb + (int64_t)t * kst + c * 8) : u4{0, 0, 0, 0};
  }
  static __device__ void k_put(u4 x, int i, uint16_t* kl) {
    if (KPIECES % CH_THREADS == 0 || i < KPIECES) *(u4*)(kl + krow(i / (D / 8)) * KP + i % (D / 8) * 8) = x;
  }
  static __device__ u4 v_piece(const uint16_t* vb, int64_t vst, int nv, int i, int u) {
    const int c = i % (D / 8), t = i / (D / 8) * 4 + u;
    return i < VTASKS && t < nv ? *(const u4*)(vb + (int64_t)t * vst + c * 8) : u4{0, 0, 0, 0};
  }
  // Infinite and NaN values go in as 0; returns whether there were any. MARKS:
  // their marks go in, and 0 for the others.
  template <bool MARKS>
  static __device__ bool v_put(u4 (&x)[4], int i, uint16_t* vl) {
    if (VTASKS % CH_THREADS != 0 && i >= VTASKS) return false;
    const int c = i % (D / 8), t = i / (D / 8) * 4;
    uint32_t odd = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) odd |= odd16<BF>(x[u][k]);
    if (MARKS || odd & ODD_BITS) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const u4 mk = marks<BF>(x[u]);
        if (MARKS) x[u] = mk;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t sel = k & 1 ? 0x07060302u : 0x05040100u;
      *(u2*)(vl + (c * 8 + k) * VP + t) =
          u2{__builtin_amdgcn_perm(x[1][k / 2], x[0][k / 2], sel), __builtin_amdgcn_perm(x[3][k / 2], x[2][k / 2], sel)};
    }
    return odd & ODD_BITS;
  }
  __device__ void load16(const uint16_t* kb, int64_t kst, const uint16_t* vb, int64_t vst, int nv) {
#pragma unroll
    for (int j = 0; j < NK; ++j) kx[j] = k_piece(kb, kst, nv, j * CH_THREADS + threadIdx.x);
#pragma unroll
    for (int j = 0; j < NV; ++j) vx[j] = v_piece(vb, vst, nv, j / 4 * CH_THREADS + threadIdx.x, j % 4);
  }
  __device__ bool store16(uint16_t* kl, uint16_t* vl) const {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < NK; ++j) k_put(kx[j], j * CH_THREADS + threadIdx.x, kl);
#pragma unroll
    for (int j = 0; j < NV; j += 4) {
      u4 x[4] = {vx[j], vx[j + 1], vx[j + 2], vx[j + 3]};
      odd |= v_put<false>(x, j / 4 * CH_THREADS + threadIdx.x, vl);
    }
    return odd;
  }
  // at once: the tail of an 8-bit cache, or any tile's marks (no keys)
  template <bool MARKS>
  static __device__ bool stage16(const uint16_t* kb, int64_t kst, const uint16_t* vb, int64_t vst, int nv, uint16_t* kl, uint16_t* vl) {
    bool odd = false;
    if (!MARKS)
      for (int i = threadIdx.x; i < KPIECES; i += CH_THREADS) k_put(k_piece(kb, kst, nv, i), i, kl);
    for (int i = threadIdx.x; i < VTASKS; i += CH_THREADS) {
      u4 x[4] = {v_piece(vb, vst, nv, i, 0), v_piece(vb, vst, nv, i, 1), v_piece(vb, vst, nv, i, 2), v_piece(vb, vst, nv, i, 3)};
      odd |= v_put<MARKS>(x, i, vl);
    }
    return odd;
  }
};

template <int D, bool BF, int FMT>
__global__ __launch_bounds__(CH_THREADS, D > 128 ? 1 : 2) void chunk_kernel(const Params p) {
  using C = Chunk<D, BF, FMT>;
  constexpr bool CACHED = FMT != DENSE;
  constexpr int NS = D / 16, NO = D / 32;
  extern __shared__ __align__(16) uint16_t lds[];

  // workgroups of one kv head on one XCD (ids go round the 8 XCDs): they share
  // its keys and values in that XCD's L2
  const int per = gridDim.x >> 3;
  const int id = blockIdx.x < per * 8 ? (blockIdx.x & 7) * per + (blockIdx.x >> 3) : blockIdx.x;
  const int split = id % p.splits;
  const int bh = id / p.splits / p.row_tiles;
  const int rt = p.row_tiles - 1 - id / p.splits % p.row_tiles;  // those that see most first
  const int b = bh / p.hkv, h = bh - b * p.hkv;
  const int len = length_of(p, b);
  const int row0 = rt * CH_ROWS;
  const int pmin = len - p.n_q + row0 / p.group;
  const int pmax = len - p.n_q + min(p.rows - 1, row0 + CH_ROWS - 1) / p.group;
  const Tiles tl = tiles_of(len, CACHED, p.block_shift, pmin, pmax, p.window, p.sinks);
  const int first = split * p.chunk, last = min(tl.n, first + p.chunk);
  if (p.splits > 1 && first >= tl.n) return;  // the merge kernel counts the same tiles

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;
  const int row = row0 + wave * 32 + n;
  const bool live = row < p.rows;
  const int qi = row / p.group, head = row - qi * p.group;
  const int pos = live ? len - p.n_q + qi : -1;
  const int low = p.window ? pos - p.window : -1;
  // the wave's own span of positions
  const int wpmin = len - p.n_q + (row0 + wave * 32) / p.group;
  const int wpmax = min(pmax, len - p.n_q + (row0 + wave * 32 + 31) / p.group);
  const bool wave_live = row0 + wave * 32 < p.rows;

  const uint8_t *kc = nullptr, *vc = nullptr;
  const float *ksc = nullptr, *vsc = nullptr;
  const uint16_t *kb = nullptr, *vb = nullptr;
  if constexpr (CACHED) {
    kc = p.k_codes + (int64_t)bh * p.cap * D;
    vc = p.v_codes + (int64_t)bh * p.cap * D;
    ksc = p.k_scales + (int64_t)bh * (p.cap >> p.block_shift);
    vsc = p.v_scales + (int64_t)bh * (p.cap >> p.block_shift);
    kb = p.k_tail + ((int64_t)bh << p.block_shift) * D;
    vb = p.v_tail + ((int64_t)bh << p.block_shift) * D;
  } else {
    kb = (const uint16_t*)p.k.p + (int64_t)b * p.k.sb + (int64_t)h * p.k.sh;
    vb = (const uint16_t*)p.v.p + (int64_t)b * p.v.sb + (int64_t)h * p.v.sh;
  }

  C c;
  // a tile's memory into registers (not the tail of an 8-bit cache)
  const auto load = [&](int it) {
    if (it >= last || it >= tl.n_main) return;
    const int tile = tl.at(it);
    if constexpr (CACHED)
      c.load8(kc, vc, tile);
    else
      c.load16(kb + (int64_t)tile * TILE * p.k.st, p.k.st, vb + (int64_t)tile * TILE * p.v.st, p.v.st, len - tile * TILE);
  };
  load(first);

  // scores of a positive scale: their maximum is taken before it multiplies
  const float scale = p.scale == 0.f ? 1.f : fabsf(p.scale);
  u4 q[NS];
  {
    const uint16_t* qp = (const uint16_t*)p.q.p + (int64_t)b * p.q.sb + (int64_t)(h * p.group + head) * p.q.sh + (int64_t)qi * p.q.st;
    const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;
    const bool none = !live || p.scale == 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) q[i] = none ? u4{0, 0, 0, 0} : *(const u4*)(qp + i * 16 + hf * 8) ^ sign;
  }
  f16v o[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) o[i][k] = 0.f;
  float m = -INFINITY, l = 0.f;
  bool odd = false;  // this thread met an infinite or NaN value

  for (int it = first, buf = 0; it < last; ++it, buf ^= 1) {
    uint16_t *kl = lds + buf * C::BUF, *vl = kl + TILE * C::KP;
    const bool codes = CACHED && it < tl.n_main;
    const int t0 = codes || !CACHED ? tl.at(it) * TILE : tl.main_len;
    const int nv = min(TILE, (codes ? tl.main_len : len) - t0);
    // 16 tokens each: what multiplies scores, log2 of what multiplies weights,
    // and its inverse for their sum (a scale of 0 has codes of 0 only: 1 will do)
    float sc[4], lf[4], rf[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      sc[g] = scale, lf[g] = 0.f, rf[g] = 1.f;
      if (codes) {
        const int blk = (t0 + 16 * g) >> p.block_shift;
        const float ks = ksc[blk], f = C::value_factor(vsc[blk]);
        sc[g] = ks == 0.f ? scale : scale * ks;
        lf[g] = __builtin_amdgcn_logf(f);
        rf[g] = f == f ? __builtin_amdgcn_rcpf(f) : 1.f;
      }
    }
    if constexpr (CACHED) {
      if (codes)
        c.store8(p, vsc, t0, tl.main_len, kl, vl);
      else
        odd |= C::template stage16<false>(kb, D, vb, D, nv, kl, vl);
    } else {
      odd |= c.store16(kl, vl);
    }
    load(it + 1);
    // One barrier per tile: a wave that is past it writes the other buffer, which
    // everyone has read before coming here.
    __syncthreads();
    // nothing of the tile is seen by this wave
    if (!wave_live || t0 > wpmax || (p.window && t0 + TILE - 1 <= wpmin - p.window && t0 >= p.sinks)) continue;

    // scores
    f16v s[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int k = 0; k < 16; ++k) s[sub][k] = 0.f;
      const uint16_t* kp = kl + (sub * 32 + n) * C::KP + hf * 8;
#pragma unroll
      for (int i = 0; i < NS; ++i) s[sub] = mma32<BF>(*(const u4*)(kp + i * 16), q[i], s[sub]);
    }
    const bool masked = nv < TILE || t0 + TILE - 1 > wpmin || (p.window && t0 <= wpmax - p.window && t0 + TILE > p.sinks);
    if (masked) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t seen = seen_bits(t0 + 16 * g + 8 * hf, 8, t0 + nv, pos, low, p.sinks);
        // a block without a finite scale: NaN where it is seen only
        const float bad = sc[g] + lf[g], nan = bad == bad ? 0.f : bad;
        if (bad != bad) sc[g] = scale, lf[g] = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float x = s[g >> 1][(g & 1) * 8 + k] + nan;
          s[g >> 1][(g & 1) * 8 + k] = seen >> k & 1 ? x : -INFINITY;
        }
      }
    }
    // softmax
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x = s[g >> 1][(g & 1) * 8];
#pragma unroll
      for (int k = 1; k < 8; ++k) x = fmaxf(x, s[g >> 1][(g & 1) * 8 + k]);
      top = fmaxf(top, x * sc[g]);
    }
    top = lanes_max<32>(top) - W_SHIFT<BF>;
    if (__any(top > m + W_SLACK<BF>)) {
      const float mn = fmaxf(m, top);
      const float a = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= a;
      l *= a;
      m = mn;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    u4 pw[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float w[8], sum = 0.f;
      const float off = lf[g] - ref;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = s[g >> 1][(g & 1) * 8 + k];
        w[k] = __builtin_amdgcn_exp2f(fmaf(x, sc[g], off));
        sum += w[k];
      }
      l = fmaf(sum, rf[g], l);
#pragma unroll
      for (int k = 0; k < 4; ++k) pw[g][k] = bits2<BF>(w[2 * k], w[2 * k + 1]);
    }
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      const uint16_t* vp = vl + (i * 32 + n) * C::VP + hf * 8;
#pragma unroll
      for (int g = 0; g < 4; ++g) o[i] = mma32<BF>(*(const u4*)(vp + g * 16), pw[g], o[i]);
    }
  }

  // Infinite and NaN values, left out so far: what the rows that see them get.
  if (__syncthreads_or(odd)) {
    for (int it = CACHED ? max(first, tl.n_main) : first; it < last; ++it) {
      const int t0 = CACHED ? tl.main_len : tl.at(it) * TILE;
      const int nv = min(TILE, len - t0);
      const uint16_t* vt = CACHED ? vb : vb + (int64_t)t0 * p.v.st;
      const bool some = C::template stage16<true>(nullptr, 0, vt, CACHED ? (int64_t)D : p.v.st, nv, nullptr, lds);
      if (__syncthreads_or(some)) {
        u4 ones[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t seen = seen_bits(t0 + 16 * g + 8 * hf, 8, t0 + nv, pos, low, p.sinks);
#pragma unroll
          for (int u = 0; u < 4; ++u) ones[g][u] = seen2<BF>(seen >> 2 * u);
        }
#pragma unroll
        for (int i = 0; i < NO; ++i) {
          const uint16_t* vp = lds + (i * 32 + n) * C::VP + hf * 8;
          f16v x;
#pragma unroll
          for (int k = 0; k < 16; ++k) x[k] = 0.f;
#pragma unroll
          for (int g = 0; g < 4; ++g) x = mma32<BF>(*(const u4*)(vp + g * 16), ones[g], x);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[i][k] += marked(x[k]);
        }
      }
      __syncthreads();
    }
  }

  l += __shfl_xor(l, 32);
  if (!live) return;
  if (p.splits > 1) {
    const int64_t u = ((int64_t)bh * p.rows + row) * p.splits + split;
    if (hf == 0) p.ws[u * 4] = m, p.ws[u * 4 + 1] = m, p.ws[u * 4 + 2] = l;
    float* d = p.ws + p.o_off + u * D;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *(f4*)(d + i * 32 + k * 8 + hf * 4) = f4{o[i][4 * k], o[i][4 * k + 1], o[i][4 * k + 2], o[i][4 * k + 3]};
    return;
  }
  const int64_t at = (int64_t)b * p.out.sb + (int64_t)(h * p.group + head) * p.out.sh + (int64_t)qi * p.out.st;
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int dim = i * 32 + k * 8 + hf * 4;
      f4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = pos < 0 ? 0.f : o[i][4 * k + j] / l;
      if (p.out_f32)
        *(f4*)((float*)p.out.p + at + dim) = x;
      else
        *(u2*)((uint16_t*)p.out.p + at + dim) = u2{bits2<BF>(x[0], x[1]), bits2<BF>(x[2], x[3])};
    }
}

template <int D, bool BF, int FMT>
hipError_t launch_chunk_as(const Params& p, hipStream_t stream) {
  constexpr int bytes = Chunk<D, BF, FMT>::LDS;
  static_assert(bytes + 16 <= 160 * 1024, "LDS");
  auto kern = chunk_kernel<D, BF, FMT>;
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
  }
  kern<<<(uint32_t)(p.splits * p.row_tiles * p.batch * p.hkv), CH_THREADS, bytes, stream>>>(p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_chunk(const Params& p, bool bf16, int fmt, hipStream_t stream) {
  if (fmt == DENSE) return bf16 ? launch_chunk_as<D, true, DENSE>(p, stream) : launch_chunk_as<D, false, DENSE>(p, stream);
  if (fmt == TQ_KV8_INT8)
    return bf16 ? launch_chunk_as<D, true, TQ_KV8_INT8>(p, stream) : launch_chunk_as<D, false, TQ_KV8_INT8>(p, stream);
  return bf16 ? launch_chunk_as<D, true, TQ_KV8_E4M3>(p, stream) : launch_chunk_as<D, false, TQ_KV8_E4M3>(p, stream);
}

}  // namespace kv
}  // namespace tq
