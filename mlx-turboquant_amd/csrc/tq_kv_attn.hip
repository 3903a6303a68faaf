// Attention over 8-bit and uncompressed KV caches: checks, the split of the
// tiles over workgroups, and the merge of the splits' partials.

#include <math.h>

#include <algorithm>

#include "tq_kv8.h"

namespace tq {
namespace kv {

int check_store(const tq_kv8_store* s);
int check_rows(const tq_rows4& r, const char* what);

extern template hipError_t launch_decode<64>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_decode<96>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_decode<128>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_decode<256>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_chunk<64>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_chunk<96>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_chunk<128>(const Params&, bool, int, hipStream_t);
extern template hipError_t launch_chunk<256>(const Params&, bool, int, hipStream_t);

namespace {

constexpr int MT = 256;
// Up to so many splits of a chunk, several rows per workgroup join theirs. One row
// per workgroup against that, us, 32 heads of head dim 128 over 4096 tokens: 1024
// queries in 2 splits 147 / 92, 128 in 8 splits 37.1 / 32.4, 32 in 8 splits 25.9 /
// 26.4, in 16 splits 22.1 / 24.7.
constexpr int ROWS_SPLITS = 8;
// Workgroups that share the tiles in decode: two per CU, what their registers
// allow.
constexpr int STREAM_WGS = 512;
// One workgroup per (sequence, kv head) and no merge instead, up to so many
// tiles (the incomplete block's among them) times head dim. Split and merged
// against that, us, one sequence of 8 kv heads, bf16, int8: head dim 64, 1024
// tokens 9.4 / 8.4, 1536 9.4 / 10.6; 128, 512 tokens 11.4 / 9.1, 1024 11.4 /
// 13.1; 256, 256 tokens 16.8 / 12.8, 512 17.1 / 18.4; 8 sequences alike.
constexpr int DIRECT_WORK = 1536;

// Where a query row's partials (M, m, l, O) lie, O in units of 2^M, l in units of
// 2^m; joined they give out = 2^(M - m) O / l.
struct MergeRow {
  int b, h, qi, head, len;
  int count;           // partials
  int64_t slot, step;  // first partial, distance of the next
};

// A row of chunks that are split: its own slots, one after the other.
__device__ inline MergeRow chunk_row(const Params& p, bool cached, int unit) {
  MergeRow r;
  const int bh = unit / p.rows, row = unit - bh * p.rows;
  r.b = bh / p.hkv, r.h = bh - r.b * p.hkv;
  r.qi = row / p.group, r.head = row - r.qi * p.group;
  r.len = length_of(p, r.b);
  const int r0 = row / p.tile_rows * p.tile_rows;
  const int pmin = r.len - p.n_q + r0 / p.group, pmax = r.len - p.n_q + min(p.rows - 1, r0 + p.tile_rows - 1) / p.group;
  r.count = (tiles_of(r.len, cached, p.block_shift, pmin, pmax, p.window, p.sinks).n + p.chunk - 1) / p.chunk;
  r.slot = (int64_t)unit * p.splits;
  r.step = 1;
  return r;
}

// A row of decode, whose slots lie one for each workgroup that shares its unit.
__device__ inline MergeRow shared_row(const Params& p, bool cached, int unit) {
  MergeRow r;
  const int bh = unit / p.rows, row = unit - bh * p.rows;
  r.b = bh / p.hkv, r.h = bh - r.b * p.hkv;
  r.qi = row / p.group, r.head = row - r.qi * p.group;
  r.len = length_of(p, r.b);
  int seq = r.b, before;
  const Share sh = share_of(p, cached, -1, seq, before);
  const int n = decode_places(p, cached, r.b), at = before + r.h * n;
  r.count = n ? (at + n - 1) / sh.per - at / sh.per + 1 : 0;
  r.slot = (int64_t)(at / sh.per + bh) * p.rows + row;
  r.step = p.rows;
  return r;
}

// 4 dims of the row: the partials' sums x and l.
template <bool BF>
__device__ inline void put_row(const Params& p, const MergeRow& r, int c, f4 x, float l, float Mr, float mr) {
  const float inv = 1.f / l, f = __builtin_amdgcn_exp2f(Mr - mr);  // apart: their product can be subnormal
  x = r.len - p.n_q + r.qi < 0 ? f4{0.f, 0.f, 0.f, 0.f} : x * inv * f;
  const int64_t at = (int64_t)r.b * p.out.sb + (int64_t)(r.h * p.group + r.head) * p.out.sh + (int64_t)r.qi * p.out.st + c * 4;
  if (p.out_f32)
    *(f4*)((float*)p.out.p + at) = x;
  else
    *(u2*)((uint16_t*)p.out.p + at) = u2{bits2<BF>(x[0], x[1]), bits2<BF>(x[2], x[3])};
}

// Rows of chunks in few splits: D / 4 threads per row, one partial after another,
// two at a time on their way. Bound by the partials' bytes.
template <int D, bool BF>
__global__ __launch_bounds__(MT) void merge_rows_kernel(const Params p, bool cached, int units) {
  constexpr int L = D / 4, R = MT / L;
  const int c = threadIdx.x % L, i0 = threadIdx.x / L;
  const int64_t unit = (int64_t)blockIdx.x * R + i0;
  if (i0 >= R || unit >= units) return;
  const MergeRow r = chunk_row(p, cached, (int)unit);
  const f4* ml = (const f4*)p.ws + r.slot;
  const f4* o = (const f4*)(p.ws + p.o_off) + r.slot * L + c;
  float M = -INFINITY, m = -INFINITY;
  for (int i = 0; i < r.count; ++i) M = fmaxf(M, ml[i].x), m = fmaxf(m, ml[i].y);
  const float Mr = M == -INFINITY ? 0.f : M, mr = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int i = 0; i < r.count; ++i) {
    l += ml[i].z * __builtin_amdgcn_exp2f(ml[i].y - mr);
    x += o[(int64_t)i * L] * __builtin_amdgcn_exp2f(ml[i].x - Mr);
  }
  put_row<BF>(p, r, c, x, l, Mr, mr);
}

// One query row per workgroup.
template <int D, bool BF>
__global__ __launch_bounds__(MT) void merge_kernel(const Params p, bool cached) {
  // Lanes of 4 dims, groups of partials (D = 96: some threads idle). Latency bounds
  // it, so every wave works out the weights of PASS partials by itself, one to a lane,
  // while a thread's N pieces of them are on their way. Threads (MT) 64 / 128 / 256 /
  // 512, us of the calls as a whole: 131072 tokens, 8 kv heads 64.8 / 63.3 / 62.7 /
  // 62.8; 4 tokens to each of 8 sequences of up to 4K, head dim 256, 28.3 / 27.7 / 27.3
  // / 27.4; 32 sequences of up to 16K, where a row has two or three partials, 118.4 /
  // 118.7 / 119.5 / 121.1.
  constexpr int L = D / 4, G = MT / L, PASS = G < 8 ? 8 * G : 64, N = (PASS + G - 1) / G;
  __shared__ f4 os[G][L];
  const MergeRow r = p.wgs ? shared_row(p, cached, blockIdx.x) : chunk_row(p, cached, blockIdx.x);
  const int count = r.count;
  const float* ml = p.ws + r.slot * 4;
  const int64_t step = r.step * 4;

  const int lane = threadIdx.x & 63, c = threadIdx.x % L, grp = threadIdx.x / L;
  float M = -INFINITY, m = -INFINITY;
  const float* o = p.ws + p.o_off + r.slot * D + c * 4;
  float Mr = 0.f, mr = 0.f, l = 0.f;
  f4 x = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < count; i0 += PASS) {
    const int n = min(PASS, count - i0);
    f4 y[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (grp + j * G < n) y[j] = *(const f4*)(o + step / 4 * (i0 + grp + j * G) * D);
    if (i0 == 0) {
      for (int i = lane; i < count; i += 64) M = fmaxf(M, ml[step * i]), m = fmaxf(m, ml[step * i + 1]);
      M = wave_max(M);
      m = wave_max(m);
      Mr = M == -INFINITY ? 0.f : M, mr = m == -INFINITY ? 0.f : m;
    }
    float f = 0.f;
    if (lane < n) {
      const float* q = ml + step * (i0 + lane);
      f = __builtin_amdgcn_exp2f(q[0] - Mr);
      l += q[2] * __builtin_amdgcn_exp2f(q[1] - mr);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float w = __shfl(f, (grp + j * G) & 63);
      if (grp + j * G < n) x += y[j] * w;
    }
  }
  if (grp < G) os[grp][c] = x;
  l = wave_sum(l);
  __syncthreads();
  if (threadIdx.x >= L) return;
#pragma unroll
  for (int i = 1; i < G; ++i) x += os[i][c];
  put_row<BF>(p, r, c, x, l, Mr, mr);
}

template <int D>
hipError_t launch_merge(const Params& p, bool bf16, bool cached, hipStream_t s) {
  const uint32_t units = (uint32_t)(p.batch * p.hkv * p.rows);
  if (p.wgs == 0 && p.splits <= ROWS_SPLITS) {
    constexpr int R = MT / (D / 4);
    const uint32_t wgs = (units + R - 1) / R;
    if (bf16)
      merge_rows_kernel<D, true><<<wgs, MT, 0, s>>>(p, cached, (int)units);
    else
      merge_rows_kernel<D, false><<<wgs, MT, 0, s>>>(p, cached, (int)units);
  } else if (bf16) {
    merge_kernel<D, true><<<units, MT, 0, s>>>(p, cached);
  } else {
    merge_kernel<D, false><<<units, MT, 0, s>>>(p, cached);
  }
  return hipGetLastError();
}

// Rows per workgroup of the chunk kernel, 128 (4 waves, two workgroups per CU up to
// head dim 128) or 256 (8 waves, which share each tile's way through LDS), and in how
// many parts a row tile's key tiles go to workgroups of their own: the pair of the
// least estimated time. Workgroups run in rounds of one or two per CU; a round takes
// as long as its share of tiles, and as 4 more for its beginning and end; parts are
// written and read again. Times are in those of a tile of 128 rows alone on a CU,
// 0.37 + 0.0066 head dim us: 1.5 for two beside each other, 1.45 for one of 256 rows.
//
// Candidates are the most parts that fill one to four rounds. us, 32 heads on 8, bf16,
// int8, head dim 128, 128 rows unsplit / 128 rows in 2 to 4 parts / 256 rows unsplit /
// 256 rows in parts that fill two or three rounds: 768 queries over 32,768 tokens 681 /
// 417 / - / 391, 1280 queries 993 / 684 / 901 / 626, 1536 994 / 806 / 900 / 721, 2048
// 995 / 1019 / 902 / 930; 1024 over 4096 92 / 88 / 122 / 83. 8192 queries over 16-bit
// keys and values, unsplit: window 1024 192 / - / 197, 2048 327 / - / 316. Over the 28 shapes that
// were timed the choice is 0.8% off the best on average, 8% at most.
template <typename F>
void choose_chunks(int64_t heads, int64_t rows, int d, const F& most_tiles, int& tile_rows, int& splits) {
  constexpr int CUS = 256;
  const double tile_us = 0.37 + 0.0066 * d;
  double best = INFINITY;
  for (int r = 128; r <= (d <= 128 ? 256 : 128); r *= 2) {
    const bool two = r == 128 && d <= 128;
    const int64_t tiles = most_tiles(r), base = std::max<int64_t>(1, heads * ((rows + r - 1) / r));
    for (int round = 0; round <= 4; ++round) {
      const int64_t want = round ? std::min(CUS * round / base, (tiles + 3) / 4) : 1;
      if (want < 1 || (round && want == 1)) continue;
      const int64_t chunk = (tiles + want - 1) / want, parts = (tiles + chunk - 1) / chunk;
      const int64_t wgs = base * parts, full = wgs / (two ? 2 * CUS : CUS), rest = wgs % (two ? 2 * CUS : CUS);
      const double time = two ? 1.5 * (full + (rest > CUS)) + (rest > 0 && rest <= CUS) : (r == 256 ? 1.45 : 1.0) * (full + (rest > 0));
      double us = time * (chunk + 4) * tile_us;
      if (parts > 1) us += 4 + 8e-6 / 5 * (d + 4) * (double)(heads * rows * parts);  // the merge; bytes at 5 TB/s
      if (us < best) best = us, tile_rows = r, splits = (int)parts;
    }
  }
}

// Shapes of a call; fills what the launch needs but the pointers.
int plan(const tq_kv8_store* s, const tq_kv_attn_desc* d, Params& p, bool& decode, size_t& bytes) {
  if (d == nullptr) return set_error(TQ_ERR_INVALID, "attention: NULL descriptor");
  if (d->d != 64 && d->d != 96 && d->d != 128 && d->d != 256)
    return set_error(TQ_ERR_UNSUPPORTED, "attention: head_dim %d: use 64, 96, 128 or 256", d->d);
  if (d->dtype != TQ_F16 && d->dtype != TQ_BF16) return set_error(TQ_ERR_UNSUPPORTED, "attention: fp16 or bf16 only");
  if (d->out_dtype != d->dtype && d->out_dtype != TQ_F32)
    return set_error(TQ_ERR_UNSUPPORTED, "attention: the output is of the queries' type or float32");
  if (d->batch < 0 || d->hq < 1 || d->hkv < 1 || d->n_q < 0 || d->hq % d->hkv)
    return set_error(TQ_ERR_INVALID, "attention: batch %d, %d query heads on %d, %d queries", d->batch, d->hq, d->hkv, d->n_q);
  if (d->window < 0 || d->sinks < 0 || d->max_len < 0)
    return set_error(TQ_ERR_INVALID, "attention: window %d, sinks %d, max_len %d", d->window, d->sinks, d->max_len);
  if (d->max_len > 0x7fffffff - 4096 || d->n_q > 0x7fffffff - 4096 || (int64_t)d->n_q * (d->hq / d->hkv) > 0x7fffffff - 4096)
    return set_error(TQ_ERR_UNSUPPORTED, "attention: too many tokens");
  if (s != nullptr) {
    if (int rc = check_store(s)) return rc;
    if (s->d != d->d || s->batch != d->batch || s->heads != d->hkv || s->kv_dtype != d->dtype)
      return set_error(TQ_ERR_INVALID, "attention: the cache is of other shapes or another type than the queries");
    if (d->max_len > s->cap) return set_error(TQ_ERR_INVALID, "attention: length %d > the cache's room for %lld", d->max_len, (long long)s->cap);
  }
  p.batch = d->batch;
  p.hkv = d->hkv;
  p.group = d->hq / d->hkv;
  p.n_q = d->n_q;
  p.rows = p.group * p.n_q;
  p.max_len = d->max_len;
  p.block_shift = s == nullptr ? 0 : s->block == 16 ? 4 : s->block == 32 ? 5 : 6;
  // a window of at least max_len hides nothing, and so no sinks matter
  p.window = d->window >= d->max_len ? 0 : d->window;
  p.sinks = p.window ? (d->sinks < d->max_len ? d->sinks : d->max_len) : 0;
  p.out_f32 = d->out_dtype == TQ_F32;
  p.scale = d->scale * 1.44269504088896340736f;
  decode = p.rows <= DEC_ROWS;
  const int64_t heads = (int64_t)p.batch * p.hkv;
  if (heads >= (int64_t)1 << 31) return set_error(TQ_ERR_UNSUPPORTED, "attention: too many sequences and heads");
  // tiles that a group of rows reads at most, the tail among them
  const auto most_tiles = [&](int64_t rows) {
    int64_t tiles = ((int64_t)d->max_len + TILE - 1) / TILE;
    if (p.window) {
      const int64_t span = std::min<int64_t>(p.n_q, rows / p.group + 2);
      tiles = std::min<int64_t>(tiles, (p.sinks + TILE - 1) / TILE + (p.window + span + TILE - 1) / TILE + 1);
    }
    return std::max<int64_t>(1, tiles + (s != nullptr));
  };
  p.tile_rows = 128;
  p.splits = 1;
  if (!decode) choose_chunks(heads, p.rows, d->d, most_tiles, p.tile_rows, p.splits);
  p.row_tiles = decode ? 1 : (p.rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t tiles = most_tiles(decode ? p.rows : p.tile_rows);
  const int64_t units = heads, base = units * p.row_tiles;
  if (base >= (int64_t)1 << 31 || units * p.rows >= (int64_t)1 << 31 || units * tiles >= (int64_t)1 << 30)
    return set_error(TQ_ERR_UNSUPPORTED, "attention: too many rows or tokens in one call");
  int64_t slots = 0;
  if (decode) {
    p.wgs = 0;
    // also where units of one length fill the chip evenly: 64 sequences of 4096
    // tokens, head dim 128: 94.6 us against 102.8
    const bool even = d->len_b == nullptr && units % STREAM_WGS == 0;
    if (tiles * d->d > DIRECT_WORK && !even) p.wgs = (int)std::min<int64_t>(STREAM_WGS, units * ((tiles + DEC_WAVES - 1) / DEC_WAVES));
    if (p.wgs) slots = (p.wgs + units) * p.rows;
  } else {
    p.chunk = (int)((tiles + p.splits - 1) / p.splits);
    p.splits = (int)((tiles + p.chunk - 1) / p.chunk);
    if (base * p.splits >= (int64_t)1 << 31) return set_error(TQ_ERR_UNSUPPORTED, "attention: too many rows in one call");
    if (p.splits > 1) slots = units * p.rows * p.splits;
  }
  p.o_off = slots * 4;
  bytes = (size_t)(slots * (4 + d->d)) * sizeof(float);
  return TQ_OK;
}

int attention(const tq_kv8_store* s, const tq_kv_attn_desc* d, void* ws, size_t ws_bytes, hipStream_t stream) {
  Params p{};
  bool decode;
  size_t need;
  if (int rc = plan(s, d, p, decode, need)) return rc;
  if (p.batch == 0 || p.rows == 0) return TQ_OK;
  if (int rc = check_rows(d->q, "attention: queries")) return rc;
  if (int rc = check_rows(d->out, "attention: output")) return rc;
  if (s == nullptr && d->max_len > 0) {
    if (int rc = check_rows(d->k, "attention: keys")) return rc;
    if (int rc = check_rows(d->v, "attention: values")) return rc;
  }
  if (need > 0 && (ws == nullptr || ws_bytes < need))
    return set_error(TQ_ERR_WORKSPACE, "attention: workspace of %zu bytes, %zu needed", ws == nullptr ? (size_t)0 : ws_bytes, need);
  if (need > 0 && ((uintptr_t)ws & 15)) return set_error(TQ_ERR_INVALID, "attention: the workspace needs 16-byte alignment");
  p.q = {d->q.p, d->q.sb, d->q.sh, d->q.st};
  p.out = {d->out.p, d->out.sb, d->out.sh, d->out.st};
  p.k = {d->k.p, d->k.sb, d->k.sh, d->k.st};
  p.v = {d->v.p, d->v.sb, d->v.sh, d->v.st};
  p.len_b = d->len_b;
  p.ws = (float*)ws;
  int fmt = DENSE;
  if (s != nullptr) {
    fmt = s->fmt;
    p.k_codes = s->k_codes;
    p.v_codes = s->v_codes;
    p.k_scales = s->k_scales;
    p.v_scales = s->v_scales;
    p.k_tail = (const uint16_t*)s->k_tail;
    p.v_tail = (const uint16_t*)s->v_tail;
    p.cap = s->cap;
  }
  const bool bf = d->dtype == TQ_BF16;
  hipError_t e;
  if (decode)
    e = d->d == 64 ? launch_decode<64>(p, bf, fmt, stream) : d->d == 96 ? launch_decode<96>(p, bf, fmt, stream)
        : d->d == 128 ? launch_decode<128>(p, bf, fmt, stream) : launch_decode<256>(p, bf, fmt, stream);
  else
    e = d->d == 64 ? launch_chunk<64>(p, bf, fmt, stream) : d->d == 96 ? launch_chunk<96>(p, bf, fmt, stream)
        : d->d == 128 ? launch_chunk<128>(p, bf, fmt, stream) : launch_chunk<256>(p, bf, fmt, stream);
  if (e == hipSuccess && need > 0) {
    const bool c = s != nullptr;
    e = d->d == 64 ? launch_merge<64>(p, bf, c, stream) : d->d == 96 ? launch_merge<96>(p, bf, c, stream)
        : d->d == 128 ? launch_merge<128>(p, bf, c, stream) : launch_merge<256>(p, bf, c, stream);
  }
  if (e != hipSuccess) return set_error(TQ_ERR_LAUNCH, "attention launch failed: %s", hipGetErrorString(e));
  return TQ_OK;
}

size_t workspace(const tq_kv8_store* s, const tq_kv_attn_desc* d) {
  Params p{};
  bool decode;
  size_t need = 0;
  return plan(s, d, p, decode, need) == TQ_OK && p.batch > 0 && p.rows > 0 ? need : 0;
}

}  // namespace
}  // namespace kv
}  // namespace tq

extern "C" size_t tq_kv8_attention_workspace_bytes(const tq_kv8_store* store, const tq_kv_attn_desc* desc) {
  return store == nullptr ? 0 : tq::kv::workspace(store, desc);
}
extern "C" int tq_kv8_attention(const tq_kv8_store* store, const tq_kv_attn_desc* desc, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (store == nullptr) return tq::set_error(TQ_ERR_INVALID, "kv8: NULL store");
  return tq::kv::attention(store, desc, workspace, workspace_bytes, (hipStream_t)stream);
}
extern "C" size_t tq_window_attention_workspace_bytes(const tq_kv_attn_desc* desc) { return tq::kv::workspace(nullptr, desc); }
extern "C" int tq_window_attention(const tq_kv_attn_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
  return tq::kv::attention(nullptr, desc, workspace, workspace_bytes, (hipStream_t)stream);
}
