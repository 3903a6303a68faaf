// Causal attention of many query rows per kv head (a chunk of query tokens
// times the query heads of the kv head) over an 8-bit KV cache or uncompressed
// 16-bit keys and values.
//
// A workgroup of 4 or 8 waves takes 32 rows per wave, row = token * group +
// head, and goes over the 64-token tiles that they see; K and V pass through
// LDS in 16 bits, V transposed. MFMA 32x32x16 (4 D multiply-adds per pair) and the
// vector instructions bound it together: on this chip their times add up but for
// about two vector instructions per product. So each step has as few of them as
// could be found, spread between the products: per wave and tile of codes at
// head dim 128, 32 products and 244 others, 32 of them exponentials.
//
// Measured: 2048 queries of 32 heads on 8 over 32,768 tokens, head dim 128, bf16,
// int8: 1028 us, 1.04 PFLOP/s (a large bf16 product reaches 1.22); 8192 queries
// over 16-bit keys and values, window 1024: 188 us, 0.69 PFLOP/s of what is seen.
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


template <int D, bool BF, int FMT, int WAVES>
struct Chunk {
  static constexpr int CH_THREADS = WAVES * 64;
  static constexpr bool CACHED = FMT != DENSE;
  static constexpr int KP = D + 8, VP = TILE + 8;  // row pitches: reads of 16 lanes hit 64 banks
  static constexpr int BUF = TILE * KP + D * VP;   // elements of a tile's K and V
  static constexpr int LDS = 2 * BUF * 2;
  // what a thread loads of a tile: pieces of 16 codes, or of 8 elements
  static constexpr int NK = (TILE * D / (CACHED ? 16 : 8) + CH_THREADS - 1) / CH_THREADS;
  static constexpr int VTOK = WAVES == 8 ? 2 : 4;  // 16-bit values: tokens that a thread pairs
  static constexpr int NV = CACHED ? NK : (TILE / VTOK * (D / 8) + CH_THREADS - 1) / CH_THREADS * VTOK;

  u4 kx[NK], vx[NV];  // on their way from memory

  // key row of token t of a tile: bits 2 and 3 swapped
  static __device__ int krow(int t) { return (t & ~12) | (t & 4) << 1 | (t & 8) >> 1; }

  // ------------------------------------------------------- a tile of codes
  static constexpr int PIECES = TILE * D / 16;
  static constexpr bool EVEN = PIECES % CH_THREADS == 0;

  static __device__ void load8(u4 (&x)[NK], const uint8_t* codes, int tile) {
    const u4* v = (const u4*)(codes + (int64_t)tile * (TILE * D));
#pragma unroll
    for (int j = 0; j < NK; ++j) x[j] = v[EVEN ? j * CH_THREADS + threadIdx.x : min(j * CH_THREADS + (int)threadIdx.x, PIECES - 1)];
  }
  static __device__ void put16(u4 x, uint16_t* d) {
    const u2 a = codes4<FMT, BF>(x.x), b = codes4<FMT, BF>(x.y), e = codes4<FMT, BF>(x.z), f = codes4<FMT, BF>(x.w);
    *(u4*)d = u4{a.x, a.y, b.x, b.y};
    *(u4*)(d + 8) = u4{e.x, e.y, f.x, f.y};
  }
  __device__ void store_k8(uint16_t* kl, int j) const {
    const int i = j * CH_THREADS + threadIdx.x;
    if (EVEN || i < PIECES) put16(kx[j], kl + krow(i / (D / 16)) * KP + i % (D / 16) * 16);
  }
  // fp16: times `power`, the power of two of this lane's 16 tokens (lane & 3)
  __device__ void store_v8(float power, uint16_t* vl, int j) const {
    const int i = j * CH_THREADS + threadIdx.x;
    if (!EVEN && i >= PIECES) return;
    uint16_t* d = vl + i / (TILE / 16) * VP + i % (TILE / 16) * 16;
    if constexpr (BF) {
      put16(vx[j], d);
    } else {
      const u4 x = vx[j];
      const u2 a = codes4<FMT, BF>(x.x), b = codes4<FMT, BF>(x.y), e = codes4<FMT, BF>(x.z), f = codes4<FMT, BF>(x.w);
      const _Float16 s = (_Float16)power;
      const h8 sc = {s, s, s, s, s, s, s, s};
      *(u4*)d = __builtin_bit_cast(u4, __builtin_bit_cast(h8, u4{a.x, a.y, b.x, b.y}) * sc);
      *(u4*)(d + 8) = __builtin_bit_cast(u4, __builtin_bit_cast(h8, u4{e.x, e.y, f.x, f.y}) * sc);
    }
  }
  // values of tokens from `nv` on, which no write has reached: any bytes
  static __device__ void clear_v8(int nv, uint16_t* vl) {
    for (int i = threadIdx.x; i < PIECES; i += CH_THREADS) {
      uint16_t* d = vl + i / (TILE / 16) * VP + i % (TILE / 16) * 16;
      if (i % (TILE / 16) * 16 >= nv) *(u4*)d = *(u4*)(d + 8) = u4{0, 0, 0, 0};
    }
  }

  // e of the power of two of a value scale that fp16 values carry: codes * 2^e
  // stay in fp16's range
  static __device__ int value_exponent(float s) {
    return min(max((int)(__float_as_uint(s) >> 23 & 255) - 127, -24), FMT == TQ_KV8_INT8 ? 9 : 7);
  }
  static __device__ float value_power(float s) { return __uint_as_float((uint32_t)(127 + value_exponent(s)) << 23); }
  // what the weights carry (codes of a scale of 0 are 0: any weight will do)
  static __device__ float value_factor(float s) {
    const float f = BF ? s : s * __uint_as_float((uint32_t)(127 - value_exponent(s)) << 23);
    return s == 0.f ? 1.f : f;
  }

  // ------------------------------------------------- a tile of 16-bit tokens
  // nv tokens at rows 0 .. of kb, vb. Values as VTOK tokens x 8 dims per thread, to
  // be paired by tokens; tokens go along the lanes, so that they meet LDS's banks
  // in turn.
  static constexpr int KPIECES = TILE * D / 8, VSPAN = TILE / VTOK, VTASKS = VSPAN * (D / 8);
  // rows past nv repeat the last one: no weight reaches them
  static __device__ u4 k_piece(const uint16_t* kb, int64_t kst, int nv, int i) {
    return *(const u4*)(kb + min(i / (D / 8), nv - 1) * kst + i % (D / 8) * 8);
  }
  static __device__ void k_put(u4 x, int i, uint16_t* kl) {
    if (KPIECES % CH_THREADS == 0 || i < KPIECES) *(u4*)(kl + krow(i / (D / 8)) * KP + i % (D / 8) * 8) = x;
  }
  static __device__ u4 v_piece(const uint16_t* vb, int64_t vst, int nv, int i, int u) {
    return *(const u4*)(vb + min(i % VSPAN * VTOK + u, nv - 1) * vst + i / VSPAN * 8);
  }
  // FINITE: infinite and NaN values go in as 0; MARKS: their marks go in, and 0
  // for the others. Returns top16() of the values.
  enum { AS_IS, FINITE, MARKS };
  template <int HOW>
  static __device__ uint32_t v_put(const u4 (&v)[VTOK], int i, uint16_t* vl) {
    if (VTASKS % CH_THREADS != 0 && i >= VTASKS) return 0;
    const int c = i / VSPAN, t = i % VSPAN * VTOK;
    uint32_t top = 0;
    u4 x[VTOK];
#pragma unroll
    for (int u = 0; u < VTOK; ++u) {
      x[u] = v[u];
#pragma unroll
      for (int k = 0; k < 4; ++k) top = top16(top, x[u][k]);
      if (HOW != AS_IS) {
        const u4 mk = marks<BF>(x[u]);
        if (HOW == MARKS) x[u] = mk;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t sel = k & 1 ? 0x07060302u : 0x05040100u;
      const uint32_t lo = __builtin_amdgcn_perm(x[1][k / 2], x[0][k / 2], sel);
      uint16_t* d = vl + (c * 8 + k) * VP + t;
      if constexpr (VTOK == 4)
        *(u2*)d = u2{lo, __builtin_amdgcn_perm(x[3][k / 2], x[2][k / 2], sel)};
      else
        *(uint32_t*)d = lo;
    }
    return top;
  }
  // A thread's pieces are whole rows apart (D = 96: not): its own offset, and
  // uniform ones.
  static constexpr int ROWS = CH_THREADS / (D / 8);
  static constexpr bool APART = CH_THREADS % (D / 8) == 0;
  int64_t k_off, v_off;
  __device__ void offsets(int64_t kst, int64_t vst) {
    k_off = (int64_t)(threadIdx.x / (D / 8)) * kst + threadIdx.x % (D / 8) * 8;
    v_off = (int64_t)(threadIdx.x % VSPAN * VTOK) * vst + threadIdx.x / VSPAN * 8;
  }
  __device__ void load_k16(const uint16_t* kb, int64_t kst, int nv) {
    if (APART && nv >= TILE) {
#pragma unroll
      for (int j = 0; j < NK; ++j) kx[j] = *(const u4*)(kb + j * ROWS * kst + k_off);
    } else {
#pragma unroll
      for (int j = 0; j < NK; ++j) kx[j] = k_piece(kb, kst, nv, j * CH_THREADS + threadIdx.x);
    }
  }
  __device__ void load_v16(const uint16_t* vb, int64_t vst, int nv) {
    if (nv >= TILE) {
      if (VTASKS % CH_THREADS == 0 || threadIdx.x < VTASKS) {
#pragma unroll
        for (int j = 0; j < NV; ++j) vx[j] = *(const u4*)(vb + j % VTOK * vst + v_off + j / VTOK * (CH_THREADS / VSPAN * 8));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) vx[j] = v_piece(vb, vst, nv, min(j / VTOK * CH_THREADS + (int)threadIdx.x, VTASKS - 1), j % VTOK);
    }
  }
  __device__ void store_k16(uint16_t* kl, int j) const { k_put(kx[j], j * CH_THREADS + threadIdx.x, kl); }
  template <int HOW>
  __device__ uint32_t store_v16(uint16_t* vl, int j) const {
    u4 x[VTOK];
#pragma unroll
    for (int u = 0; u < VTOK; ++u) x[u] = vx[VTOK * j + u];
    return v_put<HOW>(x, j * CH_THREADS + threadIdx.x, vl);
  }
  // pieces of a thread's part of a tile to LDS
  static constexpr int PK = NK, PV = CACHED ? NK : NV / VTOK;
  // at once: the tail of an 8-bit cache, or any tile's marks (no keys)
  template <int HOW>
  static __device__ bool stage16(const uint16_t* kb, int64_t kst, const uint16_t* vb, int64_t vst, int nv, uint16_t* kl, uint16_t* vl) {
    uint32_t top = 0;
    if (HOW != MARKS)
      for (int i = threadIdx.x; i < KPIECES; i += CH_THREADS) k_put(k_piece(kb, kst, nv, i), i, kl);
    for (int i = threadIdx.x; i < VTASKS; i += CH_THREADS) {
      u4 x[VTOK];
#pragma unroll
      for (int u = 0; u < VTOK; ++u) x[u] = v_piece(vb, vst, nv, i, u);
      top = top16(top, v_put<HOW>(x, i, vl));
    }
    return odd16<BF>(top);
  }
};

template <int D, bool BF, int FMT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, D > 128 ? 1 : 2) void chunk_kernel(const Params p) {
  using C = Chunk<D, BF, FMT, WAVES>;
  constexpr int CH_ROWS = WAVES * 32;
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

  // What 16 tokens of codes each have: sc multiplies scores, lf is log2 of what
  // multiplies weights, rf its inverse for their sum (a scale of 0 has codes of 0
  // only: 1 will do). Lane & 3 has the scales of its 16 tokens; they become
  // uniform only here.
  struct Scales {
    float sc[4], lf[4], rf[4];
  };
  const auto scales_of = [&](bool codes, float ks, float vs) {
    Scales x;
    if (codes) {
      const float f = C::value_factor(vs);
      const float sc = ks == 0.f ? scale : scale * ks, lf = __builtin_amdgcn_logf(f);
      const float rf = f == f ? __builtin_amdgcn_rcpf(f) : 1.f;
      const auto at = [](float y, int g) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(y), g)); };
#pragma unroll
      for (int g = 0; g < 4; ++g) x.sc[g] = at(sc, g), x.lf[g] = at(lf, g), x.rf[g] = at(rf, g);
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g) x.sc[g] = scale, x.lf[g] = 0.f, x.rf[g] = 1.f;
    }
    return x;
  };
  // Hides what the rows do not see of tokens t0 .. t0 + nv - 1 and moves the
  // reference m where it has to.
  const auto before = [&](f16v (&s)[2], Scales& x, int t0, int nv) {
    if (nv < TILE || t0 + TILE - 1 > wpmin || (p.window && t0 <= wpmax - p.window && t0 + TILE > p.sinks)) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t seen = seen_bits(t0 + 16 * g + 8 * hf, 8, t0 + nv, pos, low, p.sinks);
        // a block without a finite scale: NaN where it is seen only
        float nan = 0.f;
        if constexpr (CACHED) {
          const float bad = x.sc[g] + x.lf[g];
          if (bad != bad) nan = bad, x.sc[g] = scale, x.lf[g] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float y = s[g >> 1][(g & 1) * 8 + k];
          s[g >> 1][(g & 1) * 8 + k] = seen_or(seen, k, CACHED ? y + nan : y);
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float y = s[g >> 1][(g & 1) * 8];
#pragma unroll
      for (int k = 1; k < 8; ++k) y = fmaxf(y, s[g >> 1][(g & 1) * 8 + k]);
      top = fmaxf(top, y * x.sc[g]);
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
  };
  // Weights of 16 tokens (8 of them this lane's). Their sum is that of the rounded
  // ones: a weight's rounding then moves the output by its distance from that
  // token's value only (a lone weight cancels), and two are added at once.
  const auto weights = [&](const f16v (&s)[2], const Scales& x, int g) {
    const float off = x.lf[g] - (m == -INFINITY ? 0.f : m);
    float sum = 0.f;
    u4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = (g & 1) * 8 + 2 * k;
      w[k] = bits2<BF>(__builtin_amdgcn_exp2f(fmaf(s[g >> 1][i], x.sc[g], off)), __builtin_amdgcn_exp2f(fmaf(s[g >> 1][i + 1], x.sc[g], off)));
      sum = add2<BF>(w[k], sum);
    }
    l = fmaf(sum, x.rf[g], l);
    return w;
  };
  // Other work goes between the products, a few instructions each: what runs
  // under a product (they do not run beside another wave's).
  const auto between = [](int n) {
    for (int i = 0; i < n; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // MFMA
      __builtin_amdgcn_sched_group_barrier(0x2, 7, 0);  // VALU
    }
  };
  // A tile's scores, with `beside` among them; operands are on their way from LDS
  // during the products before.
  const auto scores = [&](f16v (&s)[2], const uint16_t* kl, auto beside) {
    const uint16_t* kp = kl + n * C::KP + hf * 8;
    u4 f[2][4];  // two steps of both halves
    const auto read = [&](u4 (&f)[4], int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = *(const u4*)(kp + k % 2 * 32 * C::KP + (i + k / 2) * 16);
    };
    read(f[0], 0);
#pragma unroll
    for (int k = 0; k < 16; ++k) s[0][k] = s[1][k] = 0.f;
#pragma unroll
    for (int i = 0; i < NS; i += 2) {
      if (i + 2 < NS) read(f[i / 2 + 1 & 1], i + 2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k % 2] = mma32<BF>(f[i / 2 & 1][k], q[i + k / 2], s[k % 2]);
      beside(i / 2);
      between(4);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // A tile's part of the output: the products of 16 tokens while the next 16
  // weights are computed.
  const auto output = [&](const f16v (&s)[2], const Scales& x, const uint16_t* vl) {
    const uint16_t* vp = vl + n * C::VP + hf * 8;
    u4 f[2][NO];
    const auto read = [&](u4 (&f)[NO], int g) {
#pragma unroll
      for (int i = 0; i < NO; ++i) f[i] = *(const u4*)(vp + i * 32 * C::VP + g * 16);
    };
    read(f[0], 0);
    u4 w = weights(s, x, 0);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g < 3) read(f[g + 1 & 1], g + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] = mma32<BF>(f[g & 1][i], w, o[i]);
      if (g < 3) w = weights(s, x, g + 1);
      between(NO);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // The tiles but the tail of an 8-bit cache, j = 0 .. count - 1. While step j
  // computes tile j's scores, tile j + 1 goes to LDS and tile j + 2 comes from
  // memory. Past the last tile that happens with the last one again, for nobody.
  // One barrier per step: what a step writes to LDS the step before has read.
  const int count = min(last, tl.n_main) - first;
  if (count > 0) {
    C c;
    if constexpr (!CACHED) c.offsets(p.k.st, p.v.st);
    const auto tile_at = [&](int j) { return tl.at(first + min(j, count - 1)); };
    const auto load_k = [&](int j) {
      const int t = tile_at(j);
      if constexpr (CACHED)
        C::load8(c.kx, kc, t);
      else
        c.load_k16(kb + (int64_t)t * TILE * p.k.st, p.k.st, len - t * TILE);
    };
    const auto load_v = [&](int j) {
      const int t = tile_at(j);
      if constexpr (CACHED)
        C::load8(c.vx, vc, t);
      else
        c.load_v16(vb + (int64_t)t * TILE * p.v.st, p.v.st, len - t * TILE);
    };
    const auto k_at = [&](int j) { return lds + (j & 1) * C::BUF; };
    const auto v_at = [&](int j) { return lds + (j & 1) * C::BUF + TILE * C::KP; };
    // the scales of this lane's 16 tokens of tiles j and j + 1
    float ks = 1.f, vs = 1.f, ks1 = 1.f, vs1 = 1.f;
    const auto load_scales = [&](int j) {
      if constexpr (CACHED) {
        const int blk = (tile_at(j) * TILE + 16 * (lane & 3)) >> p.block_shift;
        ks1 = ksc[blk];
        vs1 = vsc[blk];
      }
    };
    // piece i of the C::PK + C::PV of tile j's keys and values
    const auto store = [&](int j, int i) -> uint32_t {
      if constexpr (CACHED) {
        if (i < C::PK)
          c.store_k8(k_at(j), i);
        else
          c.store_v8(C::value_power(vs1), v_at(j), i - C::PK);
        return 0;
      } else {
        if (i < C::PK) {
          c.store_k16(k_at(j), i);
          return 0;
        }
        return c.template store_v16<C::AS_IS>(v_at(j), i - C::PK);
      }
    };
    // what store left: apart from its straight line of code
    const auto mend_v = [&](int j, uint32_t found) {
      if constexpr (CACHED) {
        const int nv = tl.main_len - tile_at(j) * TILE;
        if (nv < TILE) C::clear_v8(nv, v_at(j));
      } else if (odd16<BF>(found)) {
        odd = true;
#pragma unroll
        for (int i = 0; i < C::PV; ++i) c.template store_v16<C::FINITE>(v_at(j), i);
      }
    };
    uint32_t found = 0;
    load_scales(0);
    load_k(0);
    load_v(0);
#pragma unroll
    for (int i = 0; i < C::PK + C::PV; ++i) found = top16(found, store(0, i));
    ks = ks1;
    vs = vs1;
    load_scales(1);
    load_k(1);
    mend_v(0, found);
    load_v(1);
    for (int j = 0; j < count; ++j) {
      const int t0 = tile_at(j) * TILE;
      Scales x = scales_of(CACHED, ks, vs);
      __syncthreads();
      f16v s[2];
      found = 0;
      scores(s, k_at(j), [&](int r) {  // the pieces spread over the NS / 2 groups of products
#pragma unroll
        for (int i = 0; i < C::PK + C::PV; ++i)
          if (i * (NS / 2) / (C::PK + C::PV) == r) found = top16(found, store(j + 1, i));
      });
      ks = ks1;
      vs = vs1;
      load_scales(j + 2);
      load_k(j + 2);
      mend_v(j + 1, found);
      load_v(j + 2);
      before(s, x, t0, (CACHED ? tl.main_len : len) - t0);
      output(s, x, v_at(j));
    }
    __syncthreads();
  }
  if (CACHED && last > tl.n_main) {  // the tail
    const int nv = len - tl.main_len;
    uint16_t* vl = lds + TILE * C::KP;
    odd |= C::template stage16<C::FINITE>(kb, D, vb, D, nv, lds, vl);
    __syncthreads();
    f16v s[2];
    scores(s, lds, [](int) {});
    Scales x = scales_of(false, 1.f, 1.f);
    before(s, x, tl.main_len, nv);
    output(s, x, vl);
  }

  // Infinite and NaN values, left out so far: what the rows that see them get.
  if (__syncthreads_or(odd)) {
    for (int it = CACHED ? max(first, tl.n_main) : first; it < last; ++it) {
      const int t0 = CACHED ? tl.main_len : tl.at(it) * TILE;
      const int nv = min(TILE, len - t0);
      const uint16_t* vt = CACHED ? vb : vb + (int64_t)t0 * p.v.st;
      const bool some = C::template stage16<C::MARKS>(nullptr, 0, vt, CACHED ? (int64_t)D : p.v.st, nv, nullptr, lds);
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
  const float inv = 1.f / l;
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int dim = i * 32 + k * 8 + hf * 4;
      f4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = pos < 0 ? 0.f : o[i][4 * k + j] * inv;
      if (p.out_f32)
        *(f4*)((float*)p.out.p + at + dim) = x;
      else
        *(u2*)((uint16_t*)p.out.p + at + dim) = u2{bits2<BF>(x[0], x[1]), bits2<BF>(x[2], x[3])};
    }
}

template <int D, bool BF, int FMT, int WAVES>
hipError_t launch_chunk_as(const Params& p, hipStream_t stream) {
  constexpr int bytes = Chunk<D, BF, FMT, WAVES>::LDS;
  static_assert(bytes <= 160 * 1024, "LDS");
  auto kern = chunk_kernel<D, BF, FMT, WAVES>;
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
  }
  kern<<<(uint32_t)(p.splits * p.row_tiles * p.batch * p.hkv), WAVES * 64, bytes, stream>>>(p);
  return hipGetLastError();
}

template <int D, bool BF>
hipError_t launch_chunk_of(const Params& p, int fmt, hipStream_t stream) {
  if constexpr (D <= 128)
    if (p.tile_rows == 256)
      return fmt == DENSE ? launch_chunk_as<D, BF, DENSE, 8>(p, stream)
             : fmt == TQ_KV8_INT8 ? launch_chunk_as<D, BF, TQ_KV8_INT8, 8>(p, stream) : launch_chunk_as<D, BF, TQ_KV8_E4M3, 8>(p, stream);
  return fmt == DENSE ? launch_chunk_as<D, BF, DENSE, 4>(p, stream)
         : fmt == TQ_KV8_INT8 ? launch_chunk_as<D, BF, TQ_KV8_INT8, 4>(p, stream) : launch_chunk_as<D, BF, TQ_KV8_E4M3, 4>(p, stream);
}

template <int D>
hipError_t launch_chunk(const Params& p, bool bf16, int fmt, hipStream_t stream) {
  return bf16 ? launch_chunk_of<D, true>(p, fmt, stream) : launch_chunk_of<D, false>(p, fmt, stream);
}

}  // namespace kv
}  // namespace tq
