// Attention of at most 16 query rows per kv head (the query heads of one or a
// few tokens) over an 8-bit KV cache or uncompressed 16-bit keys and values.
//
// A workgroup of 4 waves takes `chunk` consecutive 64-token tiles of one
// (sequence, kv head), each wave every fourth of them; the waves combine in
// LDS, the workgroups of one kv head through the merge kernel. What bounds it
// is reading the cache once; nothing of it passes through LDS:
//
// Scores, transposed: S^T = K q^T with MFMA 16x16x32, A = 16 tokens x 32 dims,
// B = 32 dims x 16 query rows. Row 4a + i of the s-th product of a tile is
// token 16a + 4s + i, so lane (column n, group g) ends up with the scores of
// the 16 consecutive tokens 16g .. 16g + 15: one scale of keys and one of
// values per lane and tile (blocks are multiples of 16 tokens), and exactly the
// k-slots that O^T = V^T P^T takes as its B operand. The A operand there is 16
// dims x 32 tokens: from the transposed value codes one 16-byte load per lane
// gives two of them. 16-bit tiles are loaded by rows and paired by v_perm.
//
// Codes are exact in fp16, so the 8-bit products run in fp16 on the codes; bf16
// queries are brought into fp16's range by one power of two per row (elements
// 2^29 below their row's largest lose bits). Key scales multiply the float32
// scores. Value scales join the exponent: with s' = s + log2(scale) the weights
// exp2(s' - M), M the running maximum of s' less 13, are at most 2^13
// whatever the scales, and are rounded to fp16 for the product (2^-11 relative); the sum l of
// exp2(s - m) has its own maximum m. 16-bit tiles of bf16 take the weights as
// two bf16 parts.
//
// Measured: 32 sequences of 8432 tokens on average, 8 kv heads, head dim 128,
// int8, bf16 queries of 32 heads: 107 us, 5.2 TB/s of codes; one sequence of
// 131,072 tokens in e4m3, fp16: 52 us, 5.2 TB/s; 16-bit keys and values, 16
// sequences, window 4096: 52 us, 4.5 TB/s. Short calls are bound by a wave's
// own tiles, one after the other: 2.3 us each at head dim 128, 1.5 at 64, 4.6 at
// 256.
//
// Masked scores are -inf and their weights 0; infinite and NaN values in 16-bit
// tiles are taken apart (marks()).
#pragma once

#include <math.h>

#include "tq_kv8.h"

namespace tq {
namespace kv {

template <int D, bool BF, int FMT>
struct Decode {
  static constexpr bool CACHED = FMT != DENSE;
  static constexpr int NS = D / 32;   // products per 16 tokens of scores
  static constexpr int NO = D / 16;   // 16-dim tiles of the output
  static constexpr int NC = D / 64;   // 64-byte pieces of a code row
  static constexpr bool ODD = D % 64 != 0;
  static constexpr bool AHEAD = D <= 128;

  const Params& p;
  int n, g;           // query row (column of S^T), lane group
  int pos, low;       // the row sees tokens t <= pos with t > low or t < sinks
  int pmin, pmax, lowmax;
  float cn, cx;       // scale * log2 e, times the power of two taken off q in two parts
  u4 q[NS];
  f4 o[NO];
  float M, m, l;

  __device__ explicit Decode(const Params& pp) : p(pp) {}

  // first of the 8 dims that lane group gg holds at step st of the scores
  static __device__ int kdim(int st, int gg) {
    if (!CACHED) return st * 32 + gg * 8;
    return st < 2 * NC ? (st >> 1) * 64 + gg * 16 + (st & 1) * 8 : NC * 64 + gg * 8;
  }

  __device__ void load_q(const uint16_t* qp, bool live, u4 (&f)[NS]) const {
#pragma unroll
    for (int st = 0; st < NS; ++st) f[st] = live ? *(const u4*)(qp + kdim(st, g)) : u4{0, 0, 0, 0};
  }

  // bf16 rows to fp16: times 2^e, the row's largest element to [2^14, 2^15)
  __device__ void to_f16(u4 (&f)[NS]) {
    float top = 0.f;
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, fabsf(elem<true>(f[st][i] & 0xffff)));
        top = fmaxf(top, fabsf(elem<true>(f[st][i] >> 16)));
      }
    top = lanes_max<16>(top);
    int e = 0;
    if (top > 0.f && top < INFINITY) e = 15 - (ilogbf(top) + 1);
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[st][i] = bits2<false>(ldexpf(elem<true>(f[st][i] & 0xffff), e), ldexpf(elem<true>(f[st][i] >> 16), e));
    // both normal numbers; a key scale comes between them
    cn *= ldexpf(1.f, -e / 2);
    cx = ldexpf(1.f, -(e - e / 2));
  }

  // Scores (masked: -inf) to weights, and the running maxima and sum.
  template <bool TWO, int N>
  __device__ void weights(const float (&s)[N], float lv, bool masked, float (&w)[N]) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, s[i]);
    const float Mn = fmaxf(M, lanes_max<16>(TWO ? mx + lv : mx) - W_SHIFT<!TWO && BF>);
    const float ref = Mn == -INFINITY ? 0.f : Mn;
    if (__any(Mn > M)) {
      const float a = __builtin_amdgcn_exp2f(M - ref);
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= a;
      if (!TWO) l *= a;
      M = Mn;
    }
    // one exponential per score, against the lane's own largest of the tile
    // where two references are needed: both are then a factor
    const float near = TWO ? (mx == -INFINITY ? 0.f : mx) : ref;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = __builtin_amdgcn_exp2f(s[i] - near);
      sum += w[i];
    }
    if (TWO) {
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(mx + lv - ref);
      const float mref = mn == -INFINITY ? 0.f : mn;
      l = l * __builtin_amdgcn_exp2f(m - mref) + sum * __builtin_amdgcn_exp2f(mx - mref);
      m = mn;
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] *= f;
    } else {
      l += sum;
    }
    if (TWO && masked) {  // a block without a finite scale is NaN where it is seen only
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = s[i] == -INFINITY ? 0.f : w[i];
    }
  }

  // Whether every row sees all of tokens t0 .. t0 + count - 1.
  __device__ bool whole(int t0, int count, int len) const {
    return t0 + count <= len && t0 + count - 1 <= pmin && (t0 > lowmax || t0 + count <= p.sinks);
  }

  // --------------------------------------------------------- a tile of codes
  // In registers as loaded. The next tile's keys are loaded when the scores have
  // taken this one's, its values when the output has, so that a wave always has
  // half a tile on the way.
  u4 kr[4][NC];
  u2 kx[4];
  u4 vr[NO];
  float ks, vs;

  __device__ void load_k(const uint8_t* kc, const float* ksc, int tile) {
    // a uniform base per tile, one lane offset for all of them
    const uint8_t* kp = kc + (int64_t)tile * (TILE * D);
    const uint32_t row = (16 * (n >> 2) + (n & 3)) * D, at = row + g * 16, ax = row + NC * 64 + g * 8;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int c = 0; c < NC; ++c) kr[s][c] = *(const u4*)(kp + (at + s * 4 * D + c * 64));
      if constexpr (ODD) kx[s] = *(const u2*)(kp + (ax + s * 4 * D));
    }
    ks = ksc[(tile * TILE + 16 * g) >> p.block_shift];
  }
  __device__ void load_v(const uint8_t* vc, const float* vsc, int tile) {
    const uint8_t* vp = vc + (int64_t)tile * (D * TILE);
    const uint32_t at = NO * n * TILE + g * 16;
#pragma unroll
    for (int i = 0; i < NO; ++i) vr[i] = *(const u4*)(vp + (at + i * TILE));
    vs = vsc[(tile * TILE + 16 * g) >> p.block_shift];
  }

  // The tile in registers; `next` (< 0: none) is loaded behind it.
  __device__ void tile8(const uint8_t* kc, const uint8_t* vc, const float* ksc, const float* vsc, int tile, int next, int main_len) {
    const int t0 = tile * TILE;
    if (!AHEAD) load_k(kc, ksc, tile);
    float s[16], w[16];
    const float cs = BF ? cn * ks * cx : cn * ks;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const u2 a = codes4<FMT, false>(kr[t][c].x), b = codes4<FMT, false>(kr[t][c].y);
        acc = mma16<false>(u4{a.x, a.y, b.x, b.y}, q[2 * c], acc);
        const u2 e = codes4<FMT, false>(kr[t][c].z), f = codes4<FMT, false>(kr[t][c].w);
        acc = mma16<false>(u4{e.x, e.y, f.x, f.y}, q[2 * c + 1], acc);
      }
      if constexpr (ODD) {
        const u2 a = codes4<FMT, false>(kx[t].x), b = codes4<FMT, false>(kx[t].y);
        acc = mma16<false>(u4{a.x, a.y, b.x, b.y}, q[NS - 1], acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i] * cs;
      if (!AHEAD) __builtin_amdgcn_sched_barrier(0);  // no conversions ahead: registers
    }
    if (AHEAD && next >= 0) load_k(kc, ksc, next);
    if (!AHEAD) {
      __builtin_amdgcn_sched_barrier(0);  // the values' registers are the keys'
      load_v(vc, vsc, tile);
    }
    const bool masked = !whole(t0, TILE, main_len);
    if (masked) {
      const uint32_t seen = seen_bits(t0 + 16 * g, 16, main_len, pos, low, p.sinks);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = seen_or(seen, i, s[i]);
      if (t0 + 16 * g >= main_len) {  // not written yet: any bytes
#pragma unroll
        for (int i = 0; i < NO; ++i) vr[i] = u4{0, 0, 0, 0};
      }
    }
    weights<true, 16>(s, __builtin_amdgcn_logf(vs), masked, w);
    u4 pw[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) pw[t][i] = bits2<false>(w[8 * t + 2 * i], w[8 * t + 2 * i + 1]);
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      const u2 a = codes4<FMT, false>(vr[i].x), b = codes4<FMT, false>(vr[i].y);
      o[i] = mma16<false>(u4{a.x, a.y, b.x, b.y}, pw[0], o[i]);
      const u2 e = codes4<FMT, false>(vr[i].z), f = codes4<FMT, false>(vr[i].w);
      o[i] = mma16<false>(u4{e.x, e.y, f.x, f.y}, pw[1], o[i]);
      if (!AHEAD && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    if (AHEAD && next >= 0) load_v(vc, vsc, next);
  }

  // ------------------------------------------- half a tile of 16-bit tokens
  // 32 tokens: row 4a + i of the s-th product is token 8a + 4s + i, and a lane
  // has the scores of tokens 8g .. 8g + 7, one k-step of the output. Of nv
  // tokens at rows 0 .. of kb, vb; rows past nv repeat the last one, which no
  // query sees there. The next half is loaded as the next tile is in tile8.
  u4 k16[2][NS];
  uint32_t v16[8][NO / 2];  // dims NO n .. NO n + NO - 1 of 8 tokens

  __device__ void load_k16(const uint16_t* kb, int64_t kst, int nv) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint16_t* kp = kb + (int64_t)min(8 * (n >> 2) + 4 * s + (n & 3), nv - 1) * kst;
#pragma unroll
      for (int st = 0; st < NS; ++st) k16[s][st] = *(const u4*)(kp + kdim(st, g));
    }
  }
  __device__ void load_v16(const uint16_t* vb, int64_t vst, int nv) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint16_t* vp = vb + (int64_t)min(8 * g + u, nv - 1) * vst + NO * n;
      if constexpr (NO % 8 == 0) {
#pragma unroll
        for (int i = 0; i < NO / 8; ++i) {
          const u4 x = *(const u4*)(vp + 8 * i);
          v16[u][4 * i] = x.x, v16[u][4 * i + 1] = x.y, v16[u][4 * i + 2] = x.z, v16[u][4 * i + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NO / 2; ++i) v16[u][i] = *(const uint32_t*)(vp + 2 * i);
      }
    }
  }

  // Tokens t0 .. t0 + nv - 1 (nv <= 32 of them count) in registers; nn > 0: the
  // next half, of nn tokens at kn, vn, is loaded behind it.
  __device__ void half16(const u4 (&qf)[NS], float c, int t0, int nv, const uint16_t* kn, int64_t kst, const uint16_t* vn,
                         int64_t vst, int nn) {
    if (!AHEAD) load_k16(kn, kst, nv);
    float s[8], w[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < NS; ++st) acc = mma16<BF>(k16[t][st], qf[st], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i] * c;
    }
    if (AHEAD && nn > 0) load_k16(kn, kst, nn);
    if (!AHEAD) {
      __builtin_amdgcn_sched_barrier(0);
      load_v16(vn, vst, nv);
    }
    const bool masked = !whole(t0, HALF, t0 + nv);
    uint32_t seen = 0xff;
    if (masked) {
      seen = seen_bits(t0 + 8 * g, 8, t0 + nv, pos, low, p.sinks);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = seen_or(seen, i, s[i]);
    }
    weights<CACHED, 8>(s, 0.f, masked, w);
    u4 pw, px;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pw[i] = bits2<BF>(w[2 * i], w[2 * i + 1]);
      if constexpr (BF) px[i] = bits2<true>(w[2 * i] - elem<true>(pw[i] & 0xffff), w[2 * i + 1] - elem<true>(pw[i] >> 16));
    }
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < NO / 2; ++i) top = top16(top, v16[u][i]);
    const bool apart = __any(odd16<BF>(top));
    const u4 ones = {seen2<BF>(seen), seen2<BF>(seen >> 2), seen2<BF>(seen >> 4), seen2<BF>(seen >> 6)};
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      u4 vf;  // 8 tokens of dim NO n + i
#pragma unroll
      for (int u = 0; u < 4; ++u)
        vf[u] = __builtin_amdgcn_perm(v16[2 * u + 1][i / 2], v16[2 * u][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
      if (apart) {
        const f4 m = mma16<BF>(marks<BF>(vf), ones, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] += marked(m[k]);
      }
      o[i] = mma16<BF>(vf, pw, o[i]);
      if constexpr (BF) o[i] = mma16<BF>(vf, px, o[i]);
      if (!AHEAD && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    if (AHEAD && nn > 0) load_v16(vn, vst, nn);
  }
};

// One (sequence, kv head): places first .. last - 1 of its list (those past its
// tiles hold none), to the output (slot < 0) or to partial slot `slot`.
template <int D, bool BF, int FMT>
__device__ inline void decode_unit(const Params& p, int b, int h, int first, int last, int slot) {
  constexpr bool CACHED = FMT != DENSE, AHEAD = Decode<D, BF, FMT>::AHEAD;
  constexpr int PASS = D > 128 ? 2 : 1;      // of the output through LDS
  constexpr int NO = D / 16, NP = NO / PASS;
  __shared__ float os[DEC_WAVES][DEC_ROWS][NP * 16 + 4];
  __shared__ float ml[DEC_WAVES][DEC_ROWS][4];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = b * p.hkv + h;
  const int len = length_of(p, b);
  const int pmin = len - p.n_q, pmax = len - 1;
  const Tiles tl = tiles_of(len, CACHED, p.block_shift, pmin, pmax, p.window, p.sinks);

  last = min(last, tl.n);

  Decode<D, BF, FMT> w(p);
  w.n = lane & 15;
  w.g = lane >> 4;
  const int qi = w.n / p.group, head = w.n - qi * p.group;
  const bool live = w.n < p.rows;
  w.pos = live ? pmin + qi : -1;
  w.low = p.window ? w.pos - p.window : -1;
  w.pmin = pmin;
  w.pmax = pmax;
  w.lowmax = p.window ? pmax - p.window : -1;
  w.M = w.m = -INFINITY;
  w.l = 0.f;
#pragma unroll
  for (int i = 0; i < NO; ++i) w.o[i] = f4{0.f, 0.f, 0.f, 0.f};
  const uint16_t* qp = (const uint16_t*)p.q.p + (int64_t)b * p.q.sb + (int64_t)(h * p.group + head) * p.q.sh + (int64_t)qi * p.q.st;
  w.cn = p.scale;

  if constexpr (CACHED) {
    const int64_t row = bh;
    const uint8_t* kc = p.k_codes + row * p.cap * D;
    const uint8_t* vc = p.v_codes + row * p.cap * D;
    const float* ksc = p.k_scales + row * (p.cap >> p.block_shift);
    const float* vsc = p.v_scales + row * (p.cap >> p.block_shift);
    const int end = min(last, tl.n_main);
    int i = first + wave;
    if (AHEAD && i < end) {
      w.load_k(kc, ksc, tl.at(i));
      w.load_v(vc, vsc, tl.at(i));
    }
    w.load_q(qp, live, w.q);
    if constexpr (BF) w.to_f16(w.q);
    for (; i < end; i += DEC_WAVES)
      w.tile8(kc, vc, ksc, vsc, tl.at(i), i + DEC_WAVES < end ? tl.at(i + DEC_WAVES) : -1, tl.main_len);
    if (i < last) {  // the tail
      u4 qt[D / 32];
      w.load_q(qp, live, qt);
      const uint16_t *kt = p.k_tail + (row << p.block_shift) * D, *vt = p.v_tail + (row << p.block_shift) * D;
      const int nt = len - tl.main_len;
      if constexpr (AHEAD) {
        w.load_k16(kt, D, nt);
        w.load_v16(vt, D, nt);
      }
      for (int t = 0; t < nt; t += HALF) {
        const int at = AHEAD ? t + HALF : t;
        w.half16(qt, p.scale, tl.main_len + t, min(nt - t, HALF), kt + at * D, D, vt + at * D, D, nt - t - HALF);
      }
    }
  } else {
    w.load_q(qp, live, w.q);
    const uint16_t* kb = (const uint16_t*)p.k.p + (int64_t)b * p.k.sb + (int64_t)h * p.k.sh;
    const uint16_t* vb = (const uint16_t*)p.v.p + (int64_t)b * p.v.sb + (int64_t)h * p.v.sh;
    // halves of the wave's tiles, in order: the tokens from `t0` on
    int i = first + wave;
    if (i < last) {
      int t0 = tl.at(i) * TILE;
      if constexpr (AHEAD) {
        w.load_k16(kb + (int64_t)t0 * p.k.st, p.k.st, len - t0);
        w.load_v16(vb + (int64_t)t0 * p.v.st, p.v.st, len - t0);
      }
      for (;;) {
        int next = t0 + HALF;
        if (!(t0 & HALF) && next < len) {
          // the tile's other half
        } else {
          i += DEC_WAVES;
          next = i < last ? tl.at(i) * TILE : len;
        }
        const int64_t at = AHEAD ? next : t0;
        w.half16(w.q, p.scale, t0, min(HALF, len - t0), kb + at * p.k.st, p.k.st, vb + at * p.v.st, p.v.st, len - next);
        if (next >= len) break;
        t0 = next;
      }
    }
  }

  // the row's sum over its four lanes
  if constexpr (CACHED) {
    const float mt = lanes_max<16>(w.m);
    w.l *= __builtin_amdgcn_exp2f(w.m - (mt == -INFINITY ? 0.f : mt));
    w.m = mt;
  } else {
    w.m = w.M;
  }
  w.l += __shfl_xor(w.l, 16);
  w.l += __shfl_xor(w.l, 32);
  if (w.g == 0) ml[wave][w.n][0] = w.M, ml[wave][w.n][1] = w.m, ml[wave][w.n][2] = w.l;

  const int orow = threadIdx.x >> 4, oi = orow / p.group, oh = orow - oi * p.group;
  float M = 0.f, m = 0.f, l = 0.f, f[DEC_WAVES];
  for (int ps = 0; ps < PASS; ++ps) {
    if (ps) __syncthreads();
#pragma unroll
    for (int i = 0; i < NO; ++i)
      if (i / NP == ps)
#pragma unroll
        for (int k = 0; k < 4; ++k) os[wave][w.n][(i - ps * NP) * 16 + 4 * w.g + k] = w.o[i][k];
    __syncthreads();
    if (ps == 0) {
      M = m = -INFINITY;
      for (int v = 0; v < DEC_WAVES; ++v) M = fmaxf(M, ml[v][orow][0]), m = fmaxf(m, ml[v][orow][1]);
      const float Mr = M == -INFINITY ? 0.f : M, mr = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int v = 0; v < DEC_WAVES; ++v) {
        f[v] = __builtin_amdgcn_exp2f(ml[v][orow][0] - Mr);
        l += ml[v][orow][2] * __builtin_amdgcn_exp2f(ml[v][orow][1] - mr);
      }
      if (slot >= 0 && orow < p.rows && (threadIdx.x & 15) == 0) {
        float* d = p.ws + ((int64_t)slot * p.rows + orow) * 4;
        d[0] = M, d[1] = m, d[2] = l;
      }
    }
    if (orow >= p.rows) continue;
    const float Mr = M == -INFINITY ? 0.f : M, mr = m == -INFINITY ? 0.f : m;
    const float fin = (CACHED ? __builtin_amdgcn_exp2f(Mr - mr) : 1.f) / l;
    for (int k = threadIdx.x & 15; k < NP * 16; k += 16) {
      const int i = k % NP, r = k / NP, dim = NO * r + ps * NP + i;  // in the order of the dims
      float x = 0.f;
#pragma unroll
      for (int v = 0; v < DEC_WAVES; ++v) x += os[v][orow][i * 16 + r] * f[v];
      if (slot >= 0) {
        p.ws[p.o_off + ((int64_t)slot * p.rows + orow) * D + dim] = x;
      } else {
        x = pmin + oi < 0 ? 0.f : x * fin;
        const int64_t at = (int64_t)b * p.out.sb + (int64_t)(h * p.group + oh) * p.out.sh + (int64_t)oi * p.out.st + dim;
        if (p.out_f32)
          ((float*)p.out.p)[at] = x;
        else
          ((uint16_t*)p.out.p)[at] = bits2<BF>(x, 0.f) & 0xffff;
      }
    }
  }
}

template <int D, bool BF, int FMT>
__global__ __launch_bounds__(DEC_WAVES * 64, 2) void decode_kernel(const Params p) {
  constexpr bool CACHED = FMT != DENSE;
  int b, h, n, i = 0;      // sequence, kv head, its places, the first one to do
  int at = 0, end;         // of the list
  if (p.wgs == 0) {
    b = blockIdx.x / p.hkv;
    h = blockIdx.x - b * p.hkv;
    end = n = decode_places(p, CACHED, b);
  } else {
    int before;
    const Share s = share_of(p, CACHED, blockIdx.x, b, before);
    if (b < 0) return;
    at = blockIdx.x * s.per;
    end = min(s.total, at + s.per);
    n = decode_places(p, CACHED, b);
    h = (at - before) / n;
    i = at - before - h * n;
  }
  for (;;) {
    const int last = min(n, i + end - at);
    decode_unit<D, BF, FMT>(p, b, h, i, last, p.wgs == 0 ? -1 : blockIdx.x + b * p.hkv + h);
    at += last - i;
    if (at >= end) return;
    i = 0;
    if (++h == p.hkv) {
      h = 0;
      do n = decode_places(p, CACHED, ++b);
      while (n == 0);  // ends: the list has places left
    }
    __syncthreads();  // the last unit's reads of LDS
  }
}

template <int D, bool BF, int FMT>
hipError_t launch_decode_as(const Params& p, hipStream_t stream) {
  decode_kernel<D, BF, FMT><<<(uint32_t)(p.wgs ? p.wgs : p.batch * p.hkv), DEC_WAVES * 64, 0, stream>>>(p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_decode(const Params& p, bool bf16, int fmt, hipStream_t stream) {
  if (fmt == DENSE) return bf16 ? launch_decode_as<D, true, DENSE>(p, stream) : launch_decode_as<D, false, DENSE>(p, stream);
  if (fmt == TQ_KV8_INT8)
    return bf16 ? launch_decode_as<D, true, TQ_KV8_INT8>(p, stream) : launch_decode_as<D, false, TQ_KV8_INT8>(p, stream);
  return bf16 ? launch_decode_as<D, true, TQ_KV8_E4M3>(p, stream) : launch_decode_as<D, false, TQ_KV8_E4M3>(p, stream);
}

}  // namespace kv
}  // namespace tq
