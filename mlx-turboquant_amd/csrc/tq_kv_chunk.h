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
// Infinite and NaN values in 16-bit tiles that some rows see only in part are
// taken apart (marks()).
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
  static constexpr int LDS = (TILE * KP + D * VP) * 2;

  // key row of token t of a tile: bits 2 and 3 swapped
  static __device__ int krow(int t) { return (t & ~12) | (t & 4) << 1 | (t & 8) >> 1; }

  // One tile of codes to LDS.
  static __device__ void stage8(const Params& p, const uint8_t* kc, const uint8_t* vc, const float* vsc, int tile, int main_len,
                                uint16_t* kl, uint16_t* vl) {
    const int t0 = tile * TILE;
    for (int i = threadIdx.x; i < TILE * D / 16; i += CH_THREADS) {
      const int t = i / (D / 16), c = i % (D / 16);
      const u4 x = *(const u4*)(kc + (int64_t)(t0 + t) * D + c * 16);
      uint16_t* d = kl + krow(t) * KP + c * 16;
      const u2 a = codes4<FMT, BF>(x.x), b = codes4<FMT, BF>(x.y), e = codes4<FMT, BF>(x.z), f = codes4<FMT, BF>(x.w);
      *(u4*)d = u4{a.x, a.y, b.x, b.y};
      *(u4*)(d + 8) = u4{e.x, e.y, f.x, f.y};
    }
    for (int i = threadIdx.x; i < D * TILE / 16; i += CH_THREADS) {
      const int dim = i / (TILE / 16), c = i % (TILE / 16);
      u4 x = *(const u4*)(vc + ((int64_t)tile * D + dim) * TILE + c * 16);
      uint16_t* d = vl + dim * VP + c * 16;
      u2 a = codes4<FMT, BF>(x.x), b = codes4<FMT, BF>(x.y), e = codes4<FMT, BF>(x.z), f = codes4<FMT, BF>(x.w);
      u4 lo = {a.x, a.y, b.x, b.y}, hi = {e.x, e.y, f.x, f.y};
      if constexpr (!BF) {
        const float s = value_power(vsc[(t0 + c * 16) >> p.block_shift]);
        const h8 sc = {(_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s, (_Float16)s};
        lo = __builtin_bit_cast(u4, __builtin_bit_cast(h8, lo) * sc);
        hi = __builtin_bit_cast(u4, __builtin_bit_cast(h8, hi) * sc);
      }
      if (t0 + c * 16 >= main_len) lo = hi = u4{0, 0, 0, 0};  // not written yet: any bytes
      *(u4*)d = lo;
      *(u4*)(d + 8) = hi;
    }
  }

  // 2^e of the value scale that fp16 values carry: codes * 2^e stay in fp16's range
  static __device__ float value_power(float s) {
    if (!(s > 0.f)) return 1.f;
    return ldexpf(1.f, min(max(ilogbf(s), -24), FMT == TQ_KV8_INT8 ? 9 : 7));
  }
  static __device__ float value_factor(float s) { return BF ? s : s * (1.f / value_power(s)); }

  // nv 16-bit tokens (rows of kb, vb) to LDS, zeros after them. Returns whether
  // this thread met an infinite or NaN value.
  static __device__ bool stage16(const uint16_t* kb, int64_t kst, const uint16_t* vb, int64_t vst, int nv, uint16_t* kl,
                                 uint16_t* vl) {
    for (int i = threadIdx.x; i < TILE * D / 8; i += CH_THREADS) {
      const int t = i / (D / 8), c = i % (D / 8);
      u4 x = {0, 0, 0, 0};
      if (t < nv) x = *(const u4*)(kb + (int64_t)t * kst + c * 8);
      *(u4*)(kl + krow(t) * KP + c * 8) = x;
    }
    uint32_t odd = 0;
    // 4 tokens x 8 dims per thread, paired by tokens
    for (int i = threadIdx.x; i < TILE / 4 * (D / 8); i += CH_THREADS) {
      const int c = i % (D / 8), t = i / (D / 8) * 4;
      u4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[u] = u4{0, 0, 0, 0};
        if (t + u < nv) x[u] = *(const u4*)(vb + (int64_t)(t + u) * vst + c * 8);
#pragma unroll
        for (int k = 0; k < 4; ++k) odd |= odd16<BF>(x[u][k]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t sel = k & 1 ? 0x07060302u : 0x05040100u;
        *(u2*)(vl + (c * 8 + k) * VP + t) =
            u2{__builtin_amdgcn_perm(x[1][k / 2], x[0][k / 2], sel), __builtin_amdgcn_perm(x[3][k / 2], x[2][k / 2], sel)};
      }
    }
    return odd & ODD_BITS;
  }
};

template <int D, bool BF, int FMT>
__global__ __launch_bounds__(CH_THREADS, D > 128 ? 1 : 2) void chunk_kernel(const Params p) {
  using C = Chunk<D, BF, FMT>;
  constexpr bool CACHED = FMT != DENSE;
  constexpr int NS = D / 16, NO = D / 32;
  extern __shared__ __align__(16) uint16_t lds[];
  __shared__ int odd_tile;
  uint16_t* kl = lds;
  uint16_t* vl = lds + TILE * C::KP;

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

  u4 q[NS];
  {
    const uint16_t* qp = (const uint16_t*)p.q.p + (int64_t)b * p.q.sb + (int64_t)(h * p.group + head) * p.q.sh + (int64_t)qi * p.q.st;
#pragma unroll
    for (int i = 0; i < NS; ++i) q[i] = live ? *(const u4*)(qp + i * 16 + hf * 8) : u4{0, 0, 0, 0};
  }
  f16v o[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) o[i][k] = 0.f;
  float m = -INFINITY, l = 0.f;

  for (int it = first; it < last; ++it) {
    __syncthreads();  // the last tile's reads
    if (threadIdx.x == 0) odd_tile = 0;
    __syncthreads();
    const bool codes = CACHED && it < tl.n_main;
    int t0, nv;
    const float *ksc = nullptr, *vsc = nullptr;
    if (codes) {
      if constexpr (CACHED) {
        const int tile = tl.at(it);
        t0 = tile * TILE;
        nv = min(TILE, tl.main_len - t0);
        ksc = p.k_scales + (int64_t)bh * (p.cap >> p.block_shift);
        vsc = p.v_scales + (int64_t)bh * (p.cap >> p.block_shift);
        C::stage8(p, p.k_codes + (int64_t)bh * p.cap * D, p.v_codes + (int64_t)bh * p.cap * D, vsc, tile, tl.main_len, kl, vl);
      }
    } else {
      bool odd;
      if constexpr (CACHED) {
        t0 = tl.main_len;
        nv = len - t0;
        odd = C::stage16(p.k_tail + ((int64_t)bh << p.block_shift) * D, D, p.v_tail + ((int64_t)bh << p.block_shift) * D, D, nv,
                         kl, vl);
      } else {
        t0 = tl.at(it) * TILE;
        nv = min(TILE, len - t0);
        const uint16_t* kb = (const uint16_t*)p.k.p + (int64_t)b * p.k.sb + (int64_t)h * p.k.sh;
        const uint16_t* vb = (const uint16_t*)p.v.p + (int64_t)b * p.v.sb + (int64_t)h * p.v.sh;
        odd = C::stage16(kb + (int64_t)t0 * p.k.st, p.k.st, vb + (int64_t)t0 * p.v.st, p.v.st, nv, kl, vl);
      }
      if (odd) odd_tile = 1;
    }
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
    float f[4] = {1.f, 1.f, 1.f, 1.f};
#pragma unroll
    for (int grp = 0; grp < 4; ++grp) {
      float c = p.scale;
      if (codes) {
        const int blk = (t0 + 16 * grp) >> p.block_shift;
        c *= ksc[blk];
        f[grp] = C::value_factor(vsc[blk]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s[grp >> 1][(grp & 1) * 8 + k] *= c;
    }
    const bool masked = nv < TILE || t0 + TILE - 1 > wpmin || (p.window && t0 <= wpmax - p.window && t0 + TILE > p.sinks);
    uint32_t seen[4];
    if (masked) {
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        seen[grp] = seen_bits(t0 + 16 * grp + 8 * hf, 8, t0 + nv, pos, low, p.sinks);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float x = s[grp >> 1][(grp & 1) * 8 + k];
          s[grp >> 1][(grp & 1) * 8 + k] = seen[grp] >> k & 1 ? x : -INFINITY;
        }
      }
    }
    // softmax
    float top = -INFINITY;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int k = 0; k < 16; ++k) top = fmaxf(top, s[sub][k]);
    top = lanes_max<32>(top);
    const float mn = fmaxf(m, top - W_SHIFT);
    const float ref = mn == -INFINITY ? 0.f : mn;
    if (__any(mn > m)) {
      const float a = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= a;
      l *= a;
      m = mn;
    }
    float sum = 0.f;
    u4 pw[4];
#pragma unroll
    for (int grp = 0; grp < 4; ++grp) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = s[grp >> 1][(grp & 1) * 8 + k];
        w[k] = __builtin_amdgcn_exp2f(x - ref);
        sum += w[k];
        if (CACHED) {
          w[k] *= f[grp];
          // a block whose scale is not finite is NaN where it is seen only
          if (masked) w[k] = x == -INFINITY ? 0.f : w[k];
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) pw[grp][k] = bits2<BF>(w[2 * k], w[2 * k + 1]);
    }
    l += sum;
    if (masked && odd_tile) {
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const uint16_t* vp = vl + (i * 32 + n) * C::VP + hf * 8;
        f16v x;
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = 0.f;
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) {
          u4 v = *(const u4*)(vp + grp * 16);
          const u4 ones = {seen2<BF>(seen[grp]), seen2<BF>(seen[grp] >> 2), seen2<BF>(seen[grp] >> 4), seen2<BF>(seen[grp] >> 6)};
          x = mma32<BF>(marks<BF>(v), ones, x);
          o[i] = mma32<BF>(v, pw[grp], o[i]);
          __builtin_amdgcn_sched_barrier(0);  // one at a time: this is rare, registers are not
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) o[i][k] += marked(x[k]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const uint16_t* vp = vl + (i * 32 + n) * C::VP + hf * 8;
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) o[i] = mma32<BF>(*(const u4*)(vp + grp * 16), pw[grp], o[i]);
      }
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
