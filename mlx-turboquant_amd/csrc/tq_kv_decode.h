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
// exp2(s' - M), M the running maximum of s' less W_SHIFT, are at most 2^14
// whatever the scales, and are rounded to fp16 for the product (2^-11 relative); the sum l of
// exp2(s - m) has its own maximum m. 16-bit tiles of bf16 take the weights as
// two bf16 parts.
//
// Masked scores are -inf and their weights 0. In 16-bit tiles that some rows
// see only in part, a value that is infinite or NaN would reach the rows that
// do not see it (0 x inf): such tiles are done row by row.
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

  const Params& p;
  int n, g;           // query row (column of S^T), lane group
  int pos, low;       // the row sees tokens t <= pos with t > low or t < sinks
  int pmin, pmax, lowmax;
  float cn;           // scale * log2 e (times the power of two taken off q)
  u4 q[NS];
  f4 o[NO];
  float M, m, l;

  __device__ explicit Decode(const Params& pp) : p(pp) {}

  // first of the 8 dims that lane group gg holds at step st of the scores
  static __device__ int kdim(int st, int gg) {
    if (!CACHED) return st * 32 + gg * 8;
    return st < 2 * NC ? (st >> 1) * 64 + gg * 16 + (st & 1) * 8 : NC * 64 + gg * 8;
  }
  __device__ bool sees(int t, int at, int lw) const { return t <= at && (t > lw || t < p.sinks); }

  __device__ void load_q(const uint16_t* qp, bool live, u4 (&f)[NS]) const {
#pragma unroll
    for (int st = 0; st < NS; ++st) f[st] = live ? *(const u4*)(qp + kdim(st, g)) : u4{0, 0, 0, 0};
  }

  // bf16 rows to fp16: times 2^e, the row's largest element to [2^14, 2^15)
  __device__ float to_f16(u4 (&f)[NS]) const {
    float top = 0.f;
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, fabsf(elem<true>(f[st][i] & 0xffff)));
        top = fmaxf(top, fabsf(elem<true>(f[st][i] >> 16)));
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int e = 0;
    if (top > 0.f && top < INFINITY) e = 15 - (ilogbf(top) + 1);
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[st][i] = bits2<false>(ldexpf(elem<true>(f[st][i] & 0xffff), e), ldexpf(elem<true>(f[st][i] >> 16), e));
    return ldexpf(1.f, -e);
  }

  // Scores (masked: -inf) to weights, and the running maxima and sum.
  template <bool TWO>
  __device__ void weights(const float (&s)[16], float lv, bool masked, float (&w)[16]) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    float top = TWO ? mx + lv : mx;
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float Mn = fmaxf(M, top - W_SHIFT);
    const float ref = Mn == -INFINITY ? 0.f : Mn;
    if (__any(Mn > M)) {
      const float a = __builtin_amdgcn_exp2f(M - ref);
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= a;
      if (!TWO) l *= a;
      M = Mn;
    }
    const float off = TWO ? lv - ref : -ref;
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(s[i] + off);
    if (masked) {  // a block without a finite scale is NaN where it is seen only
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = s[i] == -INFINITY ? 0.f : w[i];
    }
    float sum = 0.f;
    if (TWO) {
      const float mn = fmaxf(m, mx);
      const float mref = mn == -INFINITY ? 0.f : mn;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(s[i] - mref);
      l = l * __builtin_amdgcn_exp2f(m - mref) + sum;
      m = mn;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += w[i];
      l += sum;
    }
  }

  // Whether every row sees all of tokens t0 .. t0 + 63.
  __device__ bool whole(int t0, int len) const {
    return t0 + TILE <= len && t0 + TILE - 1 <= pmin && (t0 > lowmax || t0 + TILE <= p.sinks);
  }

  // --------------------------------------------------------- a tile of codes
  __device__ void tile8(const uint8_t* kc, const uint8_t* vc, const float* ksc, const float* vsc, int tile, int main_len) {
    const int t0 = tile * TILE, r = n;
    u4 kr[4][NC > 0 ? NC : 1];
    u2 kx[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint8_t* kp = kc + (int64_t)(t0 + 16 * (r >> 2) + 4 * s + (r & 3)) * D;
#pragma unroll
      for (int c = 0; c < NC; ++c) kr[s][c] = *(const u4*)(kp + c * 64 + g * 16);
      if constexpr (ODD) kx[s] = *(const u2*)(kp + NC * 64 + g * 8);
    }
    const int blk = (t0 + 16 * g) >> p.block_shift;
    const float ks = ksc[blk], vs = vsc[blk];
    u4 vr[NO];
    const uint8_t* vp = vc + ((int64_t)tile * D + r) * TILE + g * 16;
#pragma unroll
    for (int i = 0; i < NO; ++i) vr[i] = *(const u4*)(vp + i * 16 * TILE);

    float s[16], w[16];
    const float cs = cn * ks;
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
    }
    const bool masked = !whole(t0, main_len);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = t0 + 16 * g + i;
        s[i] = t < main_len && sees(t, pos, low) ? s[i] : -INFINITY;
      }
      if (t0 + 16 * g >= main_len) {  // not written yet: any bytes
#pragma unroll
        for (int i = 0; i < NO; ++i) vr[i] = u4{0, 0, 0, 0};
      }
    }
    weights<true>(s, __builtin_amdgcn_logf(vs), masked, w);
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
    }
  }

  // ------------------------------------------------- a tile of 16-bit tokens
  // Tokens t0 .. t0 + nv - 1 (1 <= nv <= 64) at rows 0 .. of kb, vb. Rows past
  // nv repeat the last one; no query sees them.
  __device__ void tile16(const u4 (&qf)[NS], float c, const uint16_t* kb, int64_t kst, const uint16_t* vb, int64_t vst,
                         int t0, int nv) {
    const int r = n;
    float s[16], w[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint16_t* kp = kb + (int64_t)min(16 * (r >> 2) + 4 * t + (r & 3), nv - 1) * kst;
      u4 kr[NS];
#pragma unroll
      for (int st = 0; st < NS; ++st) kr[st] = *(const u4*)(kp + kdim(st, g));
      f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < NS; ++st) acc = mma16<BF>(kr[st], qf[st], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i] * c;
    }
    const bool masked = nv < TILE || !whole(t0, t0 + nv);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = 16 * g + i;
        s[i] = t < nv && sees(t0 + t, pos, low) ? s[i] : -INFINITY;
      }
    }
    weights<CACHED>(s, 0.f, masked, w);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u4 pw, px;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = w[8 * t + 2 * i], b = w[8 * t + 2 * i + 1];
        pw[i] = bits2<BF>(a, b);
        if constexpr (BF) px[i] = bits2<true>(a - elem<true>(pw[i] & 0xffff), b - elem<true>(pw[i] >> 16));
      }
      u4 vf[NO];  // 8 tokens of one dim each
      if constexpr (CACHED) {
        // the output's dims as tile8 has them: dim 16 i + r
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint16_t* v0 = vb + (int64_t)min(16 * g + 8 * t + 2 * u, nv - 1) * vst + i * 16 + r;
            const uint16_t* v1 = vb + (int64_t)min(16 * g + 8 * t + 2 * u + 1, nv - 1) * vst + i * 16 + r;
            vf[i][u] = (uint32_t)*v0 | (uint32_t)*v1 << 16;
          }
      } else {
        // dims NO r .. NO r + NO - 1 of 8 tokens, paired by tokens: dim NO r + i
        uint32_t vr[8][NO / 2];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const uint16_t* vp = vb + (int64_t)min(16 * g + 8 * t + u, nv - 1) * vst + NO * r;
          if constexpr (NO % 8 == 0) {
#pragma unroll
            for (int i = 0; i < NO / 8; ++i) {
              const u4 x = *(const u4*)(vp + 8 * i);
              vr[u][4 * i] = x.x, vr[u][4 * i + 1] = x.y, vr[u][4 * i + 2] = x.z, vr[u][4 * i + 3] = x.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < NO / 2; ++i) vr[u][i] = *(const uint32_t*)(vp + 2 * i);
          }
        }
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            vf[i][u] = __builtin_amdgcn_perm(vr[2 * u + 1][i / 2], vr[2 * u][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
      }
      bool odd = false;
      if (masked) {  // an infinite or NaN value among the tile's?
        const uint32_t ex = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            odd |= (vf[i][u] & ex) == ex || (vf[i][u] & ex << 16) == ex << 16;
      }
      if (__any(odd)) {
#pragma unroll
        for (int i = 0; i < NO; ++i) {
#pragma unroll 1
          for (int row = 0; row < DEC_ROWS; ++row) {
            const int at = __shfl(pos, row), lw = __shfl(low, row);
            u4 v = vf[i];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int k = 16 * g + 8 * t + 2 * u;
              v[u] &= (k < nv && sees(t0 + k, at, lw) ? 0xffffu : 0u) | (k + 1 < nv && sees(t0 + k + 1, at, lw) ? 0xffff0000u : 0u);
            }
            f4 x = mma16<BF>(v, pw, f4{0.f, 0.f, 0.f, 0.f});
            if constexpr (BF) x = mma16<BF>(finite(v), px, x);
            o[i] = n == row ? o[i] + x : o[i];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NO; ++i) {
          o[i] = mma16<BF>(vf[i], pw, o[i]);
          if constexpr (BF) o[i] = mma16<BF>(vf[i], px, o[i]);
        }
      }
    }
  }
  // infinite and NaN values as 0: the weights' remainders may be 0
  static __device__ u4 finite(u4 v) {
    const uint32_t ex = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if ((v[u] & ex) == ex) v[u] &= 0xffff0000u;
      if ((v[u] & ex << 16) == ex << 16) v[u] &= 0xffffu;
    }
    return v;
  }
};

template <int D, bool BF, int FMT>
__global__ __launch_bounds__(DEC_WAVES * 64) void decode_kernel(const Params p) {
  constexpr bool CACHED = FMT != DENSE;
  constexpr int PASS = D > 128 ? 2 : 1;      // of the output through LDS
  constexpr int NO = D / 16, NP = NO / PASS;
  __shared__ float os[DEC_WAVES][DEC_ROWS][NP * 16 + 4];
  __shared__ float ml[DEC_WAVES][DEC_ROWS][4];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int split = blockIdx.x % p.splits, bh = blockIdx.x / p.splits;
  const int b = bh / p.hkv, h = bh - b * p.hkv;
  const int len = length_of(p, b);
  const int pmin = len - p.n_q, pmax = len - 1;
  const Tiles tl = tiles_of(len, CACHED, p.block_shift, pmin, pmax, p.window, p.sinks);
  const int first = split * p.chunk, last = min(tl.n, first + p.chunk);
  if (p.splits > 1 && first >= tl.n) return;  // the merge kernel counts the same tiles

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
  for (int i = 0; i < NO; ++i) w.o[i] = f4{0.f, 0.f, 0.f, 0.f};

  const uint16_t* qp = (const uint16_t*)p.q.p + (int64_t)b * p.q.sb + (int64_t)(h * p.group + head) * p.q.sh + (int64_t)qi * p.q.st;
  w.load_q(qp, live, w.q);
  w.cn = p.scale;
  if constexpr (CACHED && BF) w.cn *= w.to_f16(w.q);

  if constexpr (CACHED) {
    const int64_t row = bh;
    const uint8_t* kc = p.k_codes + row * p.cap * D;
    const uint8_t* vc = p.v_codes + row * p.cap * D;
    const float* ksc = p.k_scales + row * (p.cap >> p.block_shift);
    const float* vsc = p.v_scales + row * (p.cap >> p.block_shift);
    for (int i = first + wave; i < last; i += DEC_WAVES) {
      if (i < tl.n_main) {
        w.tile8(kc, vc, ksc, vsc, tl.at(i), tl.main_len);
      } else {
        u4 qt[D / 32];
        w.load_q(qp, live, qt);
        w.tile16(qt, p.scale, p.k_tail + (row << p.block_shift) * D, D, p.v_tail + (row << p.block_shift) * D, D,
                 tl.main_len, len - tl.main_len);
      }
    }
  } else {
    const uint16_t* kb = (const uint16_t*)p.k.p + (int64_t)b * p.k.sb + (int64_t)h * p.k.sh;
    const uint16_t* vb = (const uint16_t*)p.v.p + (int64_t)b * p.v.sb + (int64_t)h * p.v.sh;
    for (int i = first + wave; i < last; i += DEC_WAVES) {
      const int t0 = tl.at(i) * TILE;
      w.tile16(w.q, p.scale, kb + (int64_t)t0 * p.k.st, p.k.st, vb + (int64_t)t0 * p.v.st, p.v.st, t0, min(TILE, len - t0));
    }
  }

  // the row's sum over its four lanes
  if constexpr (CACHED) {
    float mt = fmaxf(w.m, __shfl_xor(w.m, 16));
    mt = fmaxf(mt, __shfl_xor(mt, 32));
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
      if (p.splits > 1 && orow < p.rows && (threadIdx.x & 15) == 0) {
        float* d = p.ws + (((int64_t)bh * p.rows + orow) * p.splits + split) * 4;
        d[0] = M, d[1] = m, d[2] = l;
      }
    }
    if (orow >= p.rows) continue;
    const float Mr = M == -INFINITY ? 0.f : M, mr = m == -INFINITY ? 0.f : m;
    const float fin = CACHED ? __builtin_amdgcn_exp2f(Mr - mr) : 1.f;
    for (int k = threadIdx.x & 15; k < NP * 16; k += 16) {
      // column k in the order of the output's dims
      const int i = CACHED ? k >> 4 : k % NP, r = CACHED ? k & 15 : k / NP;
      const int dim = CACHED ? (ps * NP + i) * 16 + r : NO * r + ps * NP + i;
      float x = 0.f;
#pragma unroll
      for (int v = 0; v < DEC_WAVES; ++v) x += os[v][orow][i * 16 + r] * f[v];
      if (p.splits > 1) {
        p.ws[p.o_off + (((int64_t)bh * p.rows + orow) * p.splits + split) * D + dim] = x;
      } else {
        x = pmin + oi < 0 ? 0.f : x / l * fin;
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
hipError_t launch_decode_as(const Params& p, hipStream_t stream) {
  decode_kernel<D, BF, FMT><<<(uint32_t)(p.splits * p.batch * p.hkv), DEC_WAVES * 64, 0, stream>>>(p);
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
