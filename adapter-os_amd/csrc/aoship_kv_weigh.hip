/*
 * aoship_kv_weigh.hip — the attention weight that each position of the paged cache gets from a batch's rows.
 *
 * For key/value head h of a sequence, over its rows r (new token and query head of the group) that see position j:
 *
 *   w_j = prior_j + sum_r e^(s_rj - m_r) / l_r,   s_rj = scale q_r . k_j,  m_r = max_j s_rj,  l_r = sum_j e^(s_rj - m_r)
 *
 * A weight needs its rows' sums over all positions first. Sequences of up to 32 rows (a token, a few) read their keys
 * once: the scores go to memory as they are formed (4 bytes for a row's position), with the rows' maxima and sums over
 * pieces of the sequence, and a second launch makes weights of them. With more rows the scores would be more than the
 * keys: they are formed twice, for the sums and for the weights. Scores, sums and weights are float32, added in one order.
 *
 * Matrix instructions' registers (aoship_device.h): every accumulator register is read, so results need no hold; operands are
 * not held, as in the attention over the cache, and the tests check the outputs with the whole chip multiplying and
 * converting at once, in every format, against float64 and run to run, bit for bit.
 */
#include "aoship_internal.h"
#include "aoship_kv.h"
#include <hip/hip_ext.h>

using namespace kv;

namespace {

constexpr int FEW = AOS_KV_WEIGH_FEW;      /* rows of a sequence whose scores are kept */
constexpr int KB = AOS_KV_WEIGH_BLOCK;     /* positions of a workgroup: a tile of 64 a wave */
constexpr int RT = 64;                     /* rows of a stage */

/* A tile's keys of 32 positions a block, as the matrix instructions take them: lane l has the quarter of position
 * l % 32 (through `at`) that half l / 32 of the dimensions makes, undecoded. */
template <int FMT, int HDP>
struct Keys {
  static constexpr int UNITS = HDP * bits<FMT>() / 256; /* 16-byte units of a lane and block */
  static constexpr int SB = FMT == AOS_KV_BF16 ? 0 : HDP / 64;
  static constexpr int W8 = bits<FMT>() / 4; /* words of 8 codes */
  uint32_t w[2][UNITS * 4];
  uint32_t sb[2][SB ? SB : 1];
  /* at: the position of this lane's row within a block */
  __device__ __forceinline__ void load(const unsigned char *t, int at, int half) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int pos = 32 * b + at;
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        const u32x4 x = aos_gld16(t + ((half * UNITS + i) * TILE + pos) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[b][4 * i + j] = x[j];
      }
      if constexpr (SB > 0)
#pragma unroll
        for (int i = 0; i < SB; ++i)
          sb[b][i] = *(const __attribute__((address_space(1))) unsigned char *)(t + ks_off<FMT, HDP>() + (half * SB + i) * TILE + ks_index(pos));
    }
  }
  /* step e of a block: 8 dimensions from half * HDP / 2 + 8 e on */
  __device__ __forceinline__ u32x4 operand(int b, int e) const {
    return decode8<FMT>(&w[b][e * W8], FMT == AOS_KV_BF16 ? 1.0f : byte_scale(sb[b][SB ? e / 4 : 0], 0));
  }
};

/* a sequence's visible span, as row (token) t sees it: [lo, hi] */
struct Span {
  int p0, window;
  __host__ __device__ __forceinline__ int hi(int t) const { return p0 + t; }
  __host__ __device__ __forceinline__ int lo(int t) const { return window > 0 && p0 + t - window + 1 > 0 ? p0 + t - window + 1 : 0; }
};

__device__ __forceinline__ float score_factor(float scale) { /* (a scale of zero stays above it: masks keep -infinity) */
  return fmaxf(fabsf(scale) * LOG2E, 1.17549435e-38f);
}

/* Workgroups go to the XCDs in turn: which part of a sequence each has turns with the sequence (or chunk), so that no XCD
 * has the parts that short sequences, or rows before them, do not reach. */
__device__ __forceinline__ int turned(int i, int by, int n) {
  return (int)(((uint32_t)i + (uint32_t)by) % (uint32_t)n);
}

/* ---- few rows -------------------------------------------------------------------------------- */

/* Grid: pieces of `tiles` position tiles, key/value heads, sequences. S^T = K . Q^T by v_mfma_f32_32x32x16_bf16: row
 * 16 s + 8 a + 4 c + i of a block of 32 keys is position 16 c + 8 s + 4 a + i, so that a lane's 16 scores are 16
 * consecutive positions of its row. The waves take a piece's tiles in turn.
 *
 * Bound by memory: 64 streams of up to 16001 positions, 28/4 heads of 128, 16 bits: 147 us for 682 MB fetched and 75
 * written (5.1 TB/s; a large copy 4.7), then 29 us to read the scores and make weights of them. One stream of 512: 5 and 4
 * us, latencies. */
template <int FMT, int HDP>
__global__ void __launch_bounds__(256, 2) aos_kv_scores_kernel(aos_kv_weigh_params p) {
  constexpr int KS = HDP / 16;
  __shared__ float ml[4][2][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const uint32_t wg = p.wg0 + blockIdx.x;
  const int sh = (int)(wg / (uint32_t)p.pieces);
  const int piece = turned((int)(wg - (uint32_t)sh * (uint32_t)p.pieces), sh, p.pieces);
  const int s = sh / p.b.nkv, h = sh - s * p.b.nkv;
  const Seq q = seq_at(p.b, s);
  const int g = p.nh / p.b.nkv, rows = q.count * g;
  const Span v = {q.len - q.count, p.window};
  if (rows == 0 || q.len == 0) return;
  const int first = v.lo(0) / TILE, end = (q.len + TILE - 1) / TILE; /* tiles that some row sees */
  int t0 = piece * p.tiles, t1 = t0 + p.tiles < end ? t0 + p.tiles : end;
  if (t0 < first) t0 = first;
  if (t0 >= t1) return;

  const int rr = col < rows ? col : rows - 1, t = rr / g, hh = h * g + rr - t * g;
  const int hi = v.hi(t), lo = v.lo(t), lo_max = v.lo(q.count - 1), hi_min = v.hi(0);
  const float cs = score_factor(p.scale);
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
  u32x4 qf[KS];
  const uint16_t *qr = p.q + (long long)(q.row0 + t) * p.q_ld + hh * p.b.hd;
#pragma unroll
  for (int e = 0; e < KS; ++e) {
    const int d = half * (HDP / 2) + 8 * e;
    qf[e] = d < p.b.hd && col < rows ? aos_gld16(qr + d) : u32x4{};
#pragma unroll
    for (int i = 0; i < 4; ++i) qf[e][i] ^= flip;
  }
  const int at = ((col & 4) << 2) | ((col & 16) >> 1) | ((col & 8) >> 1) | (col & 3);
  float *out = p.scores + ((long long)sh * p.rows + col) * p.lpad + 16 * half;
  float m = NINF, l = 0.0f;
  for (int i = t0 + wave; i < t1; i += 4) {
    const int tb = i * TILE, page = page_of(p.b, s, tb);
    Keys<FMT, HDP> k;
    k.load(tile_ptr<FMT, HDP>(p.b, page < 0 ? 0 : page, h, tb), at, half);
    f32x16 sc[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int e = 0; e < KS; ++e)
#pragma unroll
      for (int b = 0; b < 2; ++b) sc[b] = mfma32(k.operand(b, e), qf[e], sc[b]);
    if (page < 0 || tb < lo_max || tb + TILE - 1 > hi_min) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int pos = tb + 32 * b + 16 * half + j;
          if (page < 0 || pos < lo || pos > hi) sc[b][j] = NINF;
        }
    }
    float mx = NINF;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[b][j]);
    mx = half_max(mx) * cs;
    if (page >= 0 && lo < tb + TILE && hi >= tb) mx = fmaxf(mx, LEAST);
    const float top = fmaxf(m, mx), ms = safe_max(top);
    l = l * ex2(m - ms);
    m = top;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) l = l + ex2(fmaf(sc[b][j], cs, -ms));
    if (col < rows)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *(f32x4 *)(out + tb + 32 * b + j) = f32x4{sc[b][j], sc[b][j + 1], sc[b][j + 2], sc[b][j + 3]};
  }
  l = half_sum(l);
  if (half == 0) {
    ml[wave][0][col] = m;
    ml[wave][1][col] = l;
  }
  __syncthreads();
  if (tid < rows) {
    float top = NINF, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][0][tid]);
    const float ms = safe_max(top);
#pragma unroll
    for (int w = 0; w < 4; ++w) sum = sum + ml[w][1][tid] * ex2(ml[w][0][tid] - ms);
    float *part = p.part + (((long long)sh * p.pieces + piece) * p.rows + tid) * 2;
    part[0] = top;
    part[1] = sum;
  }
}

/* four weights at a position (a multiple of 4): prior + x, of positions below len */
__device__ __forceinline__ void store4(const aos_kv_weigh_params &p, int s, int h, int pos, int len, const float *x) {
  float *w = p.w + (long long)s * p.w_seq + (long long)h * p.w_head + pos;
  const float *o = p.prior ? p.prior + (long long)s * p.prior_seq + (long long)h * p.prior_head + pos : nullptr;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (pos + i < len) w[i] = o ? o[i] + x[i] : x[i];
}

/* Grid: pieces of 1024 positions, key/value heads, sequences: the kept scores made weights. A thread has four positions. */
constexpr int WB = 1024;
__global__ void __launch_bounds__(256) aos_kv_weights_kernel(aos_kv_weigh_params p, int blocks) {
  __shared__ float red[8][2][FEW], base[FEW], inv[FEW];
  const int tid = threadIdx.x;
  const uint32_t wg = p.wg0 + blockIdx.x;
  const int blk = (int)(wg % (uint32_t)blocks), sh = (int)(wg / (uint32_t)blocks);
  const int s = sh / p.b.nkv, h = sh - s * p.b.nkv;
  const Seq q = seq_at(p.b, s);
  const int rows = q.count * (p.nh / p.b.nkv), pos = blk * WB + 4 * tid;
  if (blk * WB >= q.len) return;
  const Span v = {q.len - q.count, p.window};
  bool odd = false;                            /* some row has no distribution */
  const int first = rows ? v.lo(0) / TILE : 0; /* the scores of earlier tiles were not formed */
  if (rows) {
    /* the rows' maxima and sums over the pieces, eight threads a row */
    const int c0 = first / p.tiles, c1 = ((q.len - 1) / TILE) / p.tiles, r = tid % FEW, k = tid / FEW;
    const float2 *part = (const float2 *)p.part + (long long)sh * p.pieces * p.rows + r;
    float m = NINF, l = 0.0f;
    if (r < rows)
      for (int c = c0 + k; c <= c1; c += 32) { /* (four on their way together) */
        float2 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = c + 8 * i <= c1 ? part[(long long)(c + 8 * i) * p.rows] : make_float2(NINF, 0.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float top = fmaxf(m, y[i].x), ms = safe_max(top);
          l = l * ex2(m - ms) + y[i].y * ex2(y[i].x - ms);
          m = top;
        }
      }
    red[k][0][r] = m;
    red[k][1][r] = l;
    __syncthreads();
    if (tid < FEW) {
      float top = NINF, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, red[i][0][tid]);
      const float ms = safe_max(top);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = sum + red[i][1][tid] * ex2(red[i][0][tid] - ms);
      base[tid] = ms;
      inv[tid] = inverse(sum, top);
    }
    odd = __syncthreads_or(tid < FEW && inv[tid] != inv[tid]) != 0;
  }
  if (pos >= q.len) return;
  float x[4] = {};
  if (rows && pos + 3 >= first * TILE) {
    const float cs = score_factor(p.scale);
    const float *sc = p.scores + (long long)sh * p.rows * p.lpad + pos;
    for (int r0 = 0; r0 < rows; r0 += 8) { /* (eight on their way together) */
      f32x4 y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        y[k] = r0 + k < rows ? *(const f32x4 *)(sc + (long long)(r0 + k) * p.lpad) : f32x4{NINF, NINF, NINF, NINF};
#pragma unroll
      for (int k = 0; k < 8; ++k) /* (rows past the last have factors of zero) */
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fmaf(ex2(fmaf(y[k][i], cs, -base[r0 + k])), inv[r0 + k], x[i]);
    }
    if (odd) { /* rows without a distribution: what they do not see has no part of them */
      const bool there = page_of(p.b, s, pos) >= 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = 0.0f;
        for (int r = 0; r < rows; ++r) {
          const int t = r / (p.nh / p.b.nkv);
          if (!there || pos + i < v.lo(t) || pos + i > v.hi(t)) continue;
          x[i] = fmaf(ex2(fmaf(sc[(long long)r * p.lpad + i], cs, -base[r])), inv[r], x[i]);
        }
      }
    }
  }
  store4(p, s, h, pos, q.len, x);
}

/* a kernel's wgs workgroups, in as many launches as they take */
template <class Launch>
int in_pieces(const aos_kv_weigh_params *p, uint32_t wgs, Launch &&launch) {
  aos_kv_weigh_params a = *p;
  for (a.wg0 = 0; a.wg0 < wgs; a.wg0 += AOS_LAUNCH_PIECE(wgs - a.wg0)) {
    launch(a, AOS_LAUNCH_PIECE(wgs - a.wg0));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

template <int FMT, int HDP>
int launch_few(const aos_kv_weigh_params *p, const aos_launch_ctx *ctx) {
  const uint32_t sh = (uint32_t)p->b.n_seqs * (uint32_t)p->b.nkv;
  const int blocks = (p->b.max_len + WB - 1) / WB;
  int e = in_pieces(p, sh * (uint32_t)p->pieces, [&](const aos_kv_weigh_params &a, uint32_t n) {
    AOS_LAUNCH(ctx, (aos_kv_scores_kernel<FMT, HDP>), dim3(n), dim3(256), 0, a);
  });
  if (!e)
    e = in_pieces(p, sh * (uint32_t)blocks, [&](const aos_kv_weigh_params &a, uint32_t n) {
      AOS_LAUNCH(ctx, aos_kv_weights_kernel, dim3(n), dim3(256), 0, a, blocks);
    });
  return e;
}

/* ---- many rows ------------------------------------------------------------------------------- */

/* The rows of a sequence that see some of the positions k0 .. k1 - 1: [ra, rb) */
struct Rows {
  int ra, rb;
};
__host__ __device__ __forceinline__ Rows rows_of(const Seq &q, const Span &v, int g, int k0, int k1) {
  Rows r;
  const int ta = k0 - v.p0; /* the first that is not before them, and the last whose window reaches them */
  const long long far = v.window > 0 ? (long long)k1 - 1 + v.window - 1 - v.p0 : q.count - 1;
  /* (-1: none; a block's distance before the rows, 2^30 at most, passes 2^31 times g) */
  const int tb = far < -1 ? -1 : far < q.count - 1 ? (int)far : q.count - 1;
  r.ra = (ta > 0 ? ta : 0) * g;
  r.rb = (tb + 1) * g;
  return r;
}

/* The rows of a head are dealt out in shares of `unit`, one or more a sequence: `each` of every sequence, or (each 0) as
 * many as its own rows need and one at most to spare, sequence s's from number (first row) / unit + s on. The second,
 * whose shares follow the batch's rows, is for batches of which the first would make more than twice as many, like single
 * tokens beside a prompt (63 and one of 4001, up to 16000 positions, 28/4 heads of 128: 454 us and 107 MB, 1933 us and
 * 979 MB by the first; prompts of 900, 400, 1200 and 700, whose sequences it has to search for, 70 us, 66 by the first). */
struct Shares {
  int unit, each;
  __host__ __device__ __forceinline__ long long base(int g, int s, int row0) const {
    return each ? (long long)s * each : (long long)row0 * g / unit + s;
  }
};
/* how many there are of each kind */
inline double shares_of_each(const aos_kv_batch &b, long long g, int unit) {
  return (double)((b.max_new * g + unit - 1) / unit) * b.n_seqs;
}
inline double shares_of_own(const aos_kv_batch &b, long long g, int unit) {
  return (double)(b.n_tokens * g / unit + b.n_seqs);
}

/* Share number x of head h of sequence s is its part-th; s -1: none. From the number i of a head's share (of all of a
 * sequence's, head by head, where each sequence has as many). Uniform: each wave searches for the sequence, 64 at a time. */
struct Share {
  int s, h;
  long long part, x;
};
__device__ __forceinline__ Share share_at(const aos_kv_batch &b, const Shares &d, int g, uint32_t i, int lane) {
  Share o;
  if (d.each) {
    const int sh = (int)(i / (uint32_t)d.each);
    o.part = (int)(i - (uint32_t)sh * (uint32_t)d.each);
    o.s = sh / b.nkv;
    o.h = sh - o.s * b.nkv;
    o.x = (long long)o.s * d.each + o.part;
    return o;
  }
  const uint32_t x = i / (uint32_t)b.nkv;
  o.h = (int)(i - x * (uint32_t)b.nkv);
  o.x = x;
  int at = 0, n = b.n_seqs; /* the last of at .. at + n - 1 whose shares begin at or before x (where starts fall, any) */
  for (;;) {
    const int step = (n + 63) / 64, k = lane * step;
    const bool yes = k < n && d.base(g, at + k, b.starts[at + k]) <= x;
    const int c = (int)__popcll(__ballot(yes));
    if (c == 0) {
      o.s = -1;
      return o;
    }
    at += (c - 1) * step;
    n = n - (c - 1) * step < step ? n - (c - 1) * step : step;
    if (step == 1) break;
  }
  o.s = __builtin_amdgcn_readfirstlane(at);
  o.part = o.x - d.base(g, o.s, b.starts[o.s]);
  if (o.part < 0) o.s = -1; /* (only where starts fall) */
  return o;
}

/* Whether the batch's starts fall somewhere (noted): its sequences' rows may then be the same, and none of them is served. */
__device__ __forceinline__ bool refused(const aos_kv_batch &b, bool fall, int tid) {
  if (!__syncthreads_or(fall ? 1 : 0)) return false;
  if (tid == 0) note(b.faults, AOS_KV_FAULT_BATCH);
  return true;
}

/* A stage: 64 rows' queries, [unit of 8 dimensions][row], a unit's rows 16 bytes more apart than they take (a row's
 * units, which 16 lanes write, then lie in different banks), with the rows' maxima and factors or positions. */
template <int HDP>
struct Stage {
  static constexpr int UNITS = HDP / 8, LD = RT * 16 + 16, N = UNITS * RT / 256;
  unsigned char q[UNITS * LD];
  long long next[RT]; /* where the queries of the stage after this one begin (elements; past the last row: that row's) */
  int hi[RT];         /* the last position that a row sees; -1 past the last row */
  float m[RT], f[RT];
};

/* A workgroup has the keys of KB positions in registers, a tile a wave, and the rows of one chunk (p.rc of them) that see
 * some of them go by in stages of 64 through LDS.
 *   SUM false: each row's maximum and sum over the block's positions, to part[head][block][row].
 *   SUM true: the weights of the block's positions from the chunk's rows, to scores[chunk][head][position].
 * Grid: blocks, shares (chunks) of the rows.
 *
 * Prompt of 4001, 28/4 heads of 128, 16 bits: 93 and 90 us for 57 GFLOP each, more than any one unit's part of it: a SIMD has 34 us
 * of vector instructions (12 and 10 of them to a matrix one), 17 of the exponentials' lower rate and 23 of matrix
 * instructions. They overlap little: both position blocks' products end in the same step, so that a wave has no exponentials
 * to form while its products run, and registers leave three waves a SIMD (heads wider than 128: one, two where the weights of
 * quantised keys are formed); waves wait for 35% of their cycles. 32 tokens over up to 8132 positions, 12 sequences, 24/8 heads, 8
 * bits: 30 us either way. Queries' fragments read four ahead of the matrix instructions were within the runs' spread (the prompt
 * 209 and 205 us for 213 and 207 in all), with a wave fewer a SIMD slower (216 and 219; the 32 tokens 79 us for 72 and 73). */
template <int FMT, int HDP, bool SUM>
__global__ void __launch_bounds__(256, HDP == 256 ? 1 : 3) aos_kv_weigh_kernel(aos_kv_weigh_params p) {
  constexpr int KS = HDP / 16, N = Stage<HDP>::N, LD = Stage<HDP>::LD, UNITS = Stage<HDP>::UNITS;
  __shared__ __attribute__((aligned(16))) Stage<HDP> st[2];
  __shared__ float red[SUM ? 1 : 2][4][2][SUM ? 1 : RT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const uint32_t wg = p.wg0 + blockIdx.x;
  const int x = (int)(wg / (uint32_t)p.blocks), b0 = (int)(wg - (uint32_t)x * (uint32_t)p.blocks);
  const int blk = turned(b0, x, p.blocks), g = p.nh / p.b.nkv;
  const Share chunk = share_at(p.b, Shares{p.rc, p.chunks}, g, (uint32_t)x, lane);
  const int s = chunk.s, h = chunk.h;
  if (s < 0) return;
  const Seq q = seq_at(p.b, s);
  const int k0 = blk * KB, k1 = k0 + KB < q.len ? k0 + KB : q.len;
  if (q.count == 0 || k0 >= q.len) return;
  const Span v = {q.len - q.count, p.window};
  const Rows vis = rows_of(q, v, g, k0, k1);
  if (chunk.part * p.rc >= vis.rb) return; /* (a share to spare) */
  const int r1 = (int)chunk.part * p.rc;
  const int ra = vis.ra > r1 ? vis.ra / RT * RT : r1, rb = vis.rb < r1 + p.rc ? vis.rb : r1 + p.rc;
  if (ra >= rb) return;

  const int tb = k0 + TILE * wave; /* this wave's keys */
  const int page = tb < q.len ? page_of(p.b, s, tb) : -1;
  const float cs = score_factor(p.scale);
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
  const long long total = (long long)p.b.n_tokens * g; /* rows of a head */
  const float2 *stat = (const float2 *)p.stat + h * total + (long long)q.row0 * g;
  auto token = [&](int r) { return (int)(((uint64_t)(uint32_t)r * p.g_mul) >> p.g_shift); }; /* r / g */

  /* a thread's pieces of a stage: rows tid / UNITS + i * 256 / UNITS, unit tid % UNITS */
  constexpr int STEP = 256 / UNITS;
  const int unit = tid % UNITS, row1 = tid / UNITS;
  const bool real = 8 * unit < p.b.hd; /* (zeros past head_dim) */
  auto place = [&](int r) {
    const int x = r < rb ? r : rb - 1, t = token(x);
    return (long long)(q.row0 + t) * p.q_ld + (long long)(h * g + x - t * g) * p.b.hd;
  };
  const uint16_t *qu = p.q + (real ? 8 * unit : 0);
  u32x4 fq[N];
  float2 fs = {0.0f, 0.0f};
  int fh = 0;
  auto fetch = [&](int r0, auto &&at) { /* the queries of a stage's rows, at(i) from qu, and what goes with them */
#pragma unroll
    for (int i = 0; i < N; ++i) fq[i] = aos_gld16(qu + at(row1 + i * STEP));
    if (tid < RT) {
      const int r = r0 + tid;
      fh = r < rb ? v.hi(token(r)) : -1;
      if (SUM && r < rb) fs = stat[r];
    }
  };
  auto put = [&](Stage<HDP> &d, int r0) {
#pragma unroll
    for (int i = 0; i < N; ++i) *(u32x4 *)(d.q + unit * LD + (row1 + i * STEP) * 16) = real ? fq[i] : u32x4{};
    if (tid < RT) {
      d.hi[tid] = fh;
      if (SUM) {
        d.m[tid] = fs.x;
        d.f[tid] = fs.y;
      }
    } else if (tid < 2 * RT) {
      d.next[tid - RT] = place(r0 + RT + tid - RT);
    }
  };
  fetch(ra, [&](int i) { return place(ra + i); }); /* (on their way with the keys) */
  const bool fall = starts_fall(p.b, tid, 256);
  u32x4 kf[2][KS];
  {
    Keys<FMT, HDP> k;
    k.load(tile_ptr<FMT, HDP>(p.b, page < 0 ? 0 : page, h, tb), col, half);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        kf[b][e] = k.operand(b, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) kf[b][e][j] ^= flip; /* a negative scale: negated keys */
      }
  }
  float acc[2] = {0.0f, 0.0f};
  put(st[0], ra);
  if (refused(p.b, fall, tid)) return;
  int i = 0;
  for (int r0 = ra; r0 < rb; r0 += RT, ++i) {
    const Stage<HDP> &d = st[i & 1];
    if (r0 + RT < rb) fetch(r0 + RT, [&](int i) { return d.next[i]; });
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      float m = NINF, l = 0.0f;
      /* what the 32 rows see of the tile: something, and whether all of them all of it */
      const int rs = r0 + 32 * sub, re = rs + 32 < rb ? rs + 32 : rb;
      const int ta = token(rs), tz = token(re - 1); /* (no rows: not used) */
      const bool any = page >= 0 && rs < rb && tb <= v.hi(tz) && tb + TILE > v.lo(ta);
      const bool edge = tb < v.lo(tz) || tb + TILE - 1 > v.hi(ta) || re < rs + 32;
      if (any) { /* uniform */
        f32x16 sc[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          const u32x4 qf = *(const u32x4 *)(d.q + (half * KS + e) * LD + (32 * sub + col) * 16);
#pragma unroll
          for (int b = 0; b < 2; ++b) sc[b] = SUM ? mfma32(qf, kf[b][e], sc[b]) : mfma32(kf[b][e], qf, sc[b]);
        }
        if constexpr (!SUM) {
          const int hi = d.hi[32 * sub + col], lo = v.lo(hi - v.p0);
          if (edge) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int pos = tb + 32 * b + 8 * (j >> 2) + 4 * half + (j & 3);
                if (pos < lo || pos > hi) sc[b][j] = NINF;
              }
          }
          float mx = NINF;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[b][j]);
          mx = half_max(mx) * cs;
          if (lo < tb + TILE && hi >= tb) mx = fmaxf(mx, LEAST);
          m = mx;
          const float ms = safe_max(m);
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) l = l + ex2(fmaf(sc[b][j], cs, -ms));
          l = half_sum(l);
        } else {
#pragma unroll
          for (int j4 = 0; j4 < 4; ++j4) {
            const int at = 32 * sub + 8 * j4 + 4 * half; /* rows at .. at + 3 of the stage */
            const f32x4 rm = *(const f32x4 *)(d.m + at), rf = *(const f32x4 *)(d.f + at);
            if (edge) {
              const int4 hi = *(const int4 *)(d.hi + at);
              const int his[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int pos = tb + 32 * b + col;
                  const float e = fmaf(ex2(fmaf(sc[b][4 * j4 + j], cs, -rm[j])), rf[j], acc[b]);
                  acc[b] = pos >= v.lo(his[j] - v.p0) && pos <= his[j] ? e : acc[b];
                }
            } else {
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[b] = fmaf(ex2(fmaf(sc[b][4 * j4 + j], cs, -rm[j])), rf[j], acc[b]);
            }
          }
        }
      }
      if constexpr (!SUM) {
        if (half == 0) {
          red[i & 1][wave][0][32 * sub + col] = m;
          red[i & 1][wave][1][32 * sub + col] = l;
        }
      }
    }
    if (r0 + RT < rb) put(st[(i + 1) & 1], r0 + RT);
    __syncthreads();
    if constexpr (!SUM) {
      if (tid < RT && r0 + tid < rb) {
        float top = NINF, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, red[i & 1][w][0][tid]);
        const float ms = safe_max(top);
#pragma unroll
        for (int w = 0; w < 4; ++w) sum = sum + red[i & 1][w][1][tid] * ex2(red[i & 1][w][0][tid] - ms);
        float2 *part = (float2 *)p.part + ((long long)h * p.blocks + blk) * total + (long long)q.row0 * g + r0 + tid;
        *part = make_float2(top, sum);
      }
    }
  }
  if constexpr (SUM) {
    float *out = p.scores + (chunk.x * p.b.nkv + h) * p.lpad + tb;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float sum = half_sum(acc[b]);
      if (half == 0 && tb < q.len) out[32 * b + col] = sum;
    }
  }
}

/* Grid: shares of 256 rows: a row's maximum and the inverse of its sum over all blocks. */
__global__ void __launch_bounds__(256) aos_kv_weigh_rows_kernel(aos_kv_weigh_params p) {
  if (refused(p.b, starts_fall(p.b, (int)threadIdx.x, 256), (int)threadIdx.x)) return;
  const int g = p.nh / p.b.nkv;
  const Share piece = share_at(p.b, Shares{256, p.row_pieces}, g, p.wg0 + blockIdx.x, (int)threadIdx.x & 63);
  const int s = piece.s, h = piece.h;
  if (s < 0) return;
  const Seq q = seq_at(p.b, s);
  if (piece.part * 256 + (int)threadIdx.x >= (long long)q.count * g) return;
  const int r = (int)piece.part * 256 + (int)threadIdx.x;
  const Span v = {q.len - q.count, p.window};
  const int t = r / g, hi = v.hi(t), lo = v.lo(t);
  const long long total = (long long)p.b.n_tokens * g, at = (long long)q.row0 * g + r;
  const float2 *part = (const float2 *)p.part + (long long)h * p.blocks * total + at;
  float m = NINF, l = 0.0f;
  const int k1 = hi < 0 ? -1 : hi / KB;
  for (int k0 = lo / KB; k0 <= k1; k0 += 8) { /* (eight on their way together) */
    float2 y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = k0 + i <= k1 ? part[(long long)(k0 + i) * total] : make_float2(NINF, 0.0f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float top = fmaxf(m, y[i].x), ms = safe_max(top);
      l = l * ex2(m - ms) + y[i].y * ex2(y[i].x - ms);
      m = top;
    }
  }
  ((float2 *)p.stat)[h * total + at] = make_float2(safe_max(m), inverse(l, m));
}

/* Grid: blocks of KB positions, key/value heads, sequences: the chunks' weights added in order. */
__global__ void __launch_bounds__(64) aos_kv_weigh_sum_kernel(aos_kv_weigh_params p) {
  if (refused(p.b, starts_fall(p.b, (int)threadIdx.x, 64), (int)threadIdx.x)) return;
  const uint32_t wg = p.wg0 + blockIdx.x;
  const int blk = (int)(wg % (uint32_t)p.blocks), sh = (int)(wg / (uint32_t)p.blocks);
  const int s = sh / p.b.nkv, h = sh - s * p.b.nkv;
  const Seq q = seq_at(p.b, s);
  const int g = p.nh / p.b.nkv, k0 = blk * KB, k1 = k0 + KB < q.len ? k0 + KB : q.len, pos = k0 + 4 * (int)threadIdx.x;
  if (pos >= q.len) return;
  float x[4] = {};
  if (q.count) {
    const Span v = {q.len - q.count, p.window};
    const Rows vis = rows_of(q, v, g, k0, k1);
    const long long step = (long long)p.b.nkv * p.lpad; /* from a chunk to the next */
    const float *in = p.scores + Shares{p.rc, p.chunks}.base(g, s, q.row0) * step + (long long)h * p.lpad + pos;
    const int c1 = (vis.rb + p.rc - 1) / p.rc;
    for (int c0 = vis.ra / p.rc; c0 < c1; c0 += 8) {
      f32x4 y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = c0 + j < c1 ? *(const f32x4 *)(in + (c0 + j) * step) : f32x4{};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = x[i] + y[j][i];
    }
  }
  store4(p, s, h, pos, q.len, x);
}

template <int FMT, int HDP>
int launch_many(const aos_kv_weigh_params *p, const aos_launch_ctx *ctx) {
  const uint32_t sh = (uint32_t)p->b.n_seqs * (uint32_t)p->b.nkv;
  const uint32_t wgs = (uint32_t)p->slots * (uint32_t)p->b.nkv * (uint32_t)p->blocks;
  int e = in_pieces(p, wgs, [&](const aos_kv_weigh_params &a, uint32_t n) {
    AOS_LAUNCH(ctx, (aos_kv_weigh_kernel<FMT, HDP, false>), dim3(n), dim3(256), 0, a);
  });
  if (!e)
    e = in_pieces(p, (uint32_t)p->row_slots * (uint32_t)p->b.nkv, [&](const aos_kv_weigh_params &a, uint32_t n) {
      AOS_LAUNCH(ctx, aos_kv_weigh_rows_kernel, dim3(n), dim3(256), 0, a);
    });
  if (!e)
    e = in_pieces(p, wgs, [&](const aos_kv_weigh_params &a, uint32_t n) {
      AOS_LAUNCH(ctx, (aos_kv_weigh_kernel<FMT, HDP, true>), dim3(n), dim3(256), 0, a);
    });
  if (!e)
    e = in_pieces(p, sh * (uint32_t)p->blocks, [&](const aos_kv_weigh_params &a, uint32_t n) {
      AOS_LAUNCH(ctx, aos_kv_weigh_sum_kernel, dim3(n), dim3(64), 0, a);
    });
  return e;
}

template <int FMT, int HDP>
int weigh(const aos_kv_weigh_params *p, const aos_launch_ctx *ctx) {
  return p->few ? launch_few<FMT, HDP>(p, ctx) : launch_many<FMT, HDP>(p, ctx);
}

}  // namespace

/* The shape of a batch's launches and the workspace they need (which grows with each of the batch's sizes). */
extern "C" int aos_kv_weigh_shape(aos_kv_weigh_params *p, size_t *bytes) {
  const aos_kv_batch &b = p->b;
  const long long g = p->nh / b.nkv, rows = b.max_new * g, sh = (long long)b.n_seqs * b.nkv;
  const long long blocks = b.max_len > 0 ? ((long long)b.max_len + KB - 1) / KB : 1;
  if (rows > (1ll << 30) || sh > 0x7fffffff) return 0;
  p->rows = (int)rows;
  p->blocks = (int)blocks;
  /* r / g for r < 2^30: r M >> 31 + s with 2^s >= g, M = 2^(31 + s) / g rounded up: off by less than 2^30 g / 2^(31 + s) < 1 / 2
   * of the least distance to the next whole number */
  int sh2 = 0;
  while ((1ll << sh2) < g) ++sh2;
  p->g_mul = (uint32_t)(((1ull << (31 + sh2)) + (uint64_t)g - 1) / (uint64_t)g);
  p->g_shift = 31 + sh2;
  p->lpad = p->blocks * KB;
  /* few rows: pieces of a block where there are few, of up to eight, so that the sums of pieces stay few (64 streams of up
   * to 16001 positions, 16128 blocks: 181 us in pieces of one, 186 of three, 200 of seven, whose last round is half empty) */
  long long span = sh * blocks / 8192;
  span = span < 1 ? 1 : span > 8 ? 8 : span;
  p->tiles = (int)span * (KB / TILE);
  p->pieces = (int)((blocks + span - 1) / span);
  /* many rows: chunks of 64 where there are few, of up to 512 (prompt of 4001, 28 heads: 198 to 201 us; chunks of 256 take as
   * long, 201 to 202, and leave twice as many weights to add up) */
  const double one = shares_of_each(b, g, RT), own = shares_of_own(b, g, RT);
  const bool each = one <= 2 * own;
  const double heads = b.nkv * (double)blocks, units = (each ? one : own) * heads;
  const int k = units < 4096 ? 1 : units > 16384 ? 8 : (int)(units / 2048);
  p->rc = RT * k;
  p->chunks = each ? (int)((rows + p->rc - 1) / p->rc) : 0;
  p->row_pieces = each ? (int)((rows + 255) / 256) : 0;
  const double slots = each ? shares_of_each(b, g, p->rc) : shares_of_own(b, g, p->rc);
  const double row_slots = each ? shares_of_each(b, g, 256) : shares_of_own(b, g, 256);
  const double kept = (double)sh * rows * (4.0 * p->lpad + 8.0 * blocks);
  p->few = rows <= FEW && kept <= AOS_KV_WEIGH_KEEP && !p->no_few;
  double need = kept, wgs = (double)sh * blocks;
  if (!p->few) {
    /* (chunks times blocks are at most units / 8 or 4096, and one more for each sequence's head and block; units are at
     * most those of `most`, which grow with each of the batch's sizes, whichever way is taken) */
    const double most = fmin(one, 2 * own) * heads;
    need = 8.0 * b.n_tokens * p->nh * (blocks + 1) + 4.0 * KB * ((most > 32768 ? most / 8 : 4096) + (double)sh * blocks);
    const double work = slots * (double)blocks;
    wgs = fmax(wgs, b.nkv * fmax(work, row_slots));
  }
  if (need > AOS_KV_WEIGH_MOST || wgs > 2e9) return 0;
  p->slots = p->few ? 0 : (int)slots;
  p->row_slots = p->few ? 0 : (int)row_slots;
  *bytes = (size_t)need;
  return 1;
}

/* What every batch within these sizes needs, whichever way it goes; 0 where this batch cannot be counted. */
extern "C" size_t aos_kv_weigh_most(const aos_kv_weigh_params *p) {
  aos_kv_weigh_params a = *p;
  a.no_few = 1;
  size_t many = 0, few = 0;
  if (!aos_kv_weigh_shape(&a, &many)) return 0;
  a.no_few = 0;
  if (a.b.max_new * (a.nh / a.b.nkv) > FEW) a.b.max_new = FEW / (a.nh / a.b.nkv);
  if (a.b.max_new > 0 && aos_kv_weigh_shape(&a, &few) && !a.few) few = (size_t)AOS_KV_WEIGH_KEEP;
  return many > few ? many : few;
}

/* the parts of a workspace of that many bytes */
extern "C" void aos_kv_weigh_parts(aos_kv_weigh_params *p, void *ws) {
  const size_t sh = (size_t)p->b.n_seqs * p->b.nkv, total = (size_t)p->b.n_tokens * p->nh;
  p->scores = (float *)ws;
  p->part = p->scores + (p->few ? sh * (size_t)p->rows : (size_t)p->slots * p->b.nkv) * (size_t)p->lpad;
  p->stat = p->few ? nullptr : p->part + 2 * total * (size_t)p->blocks;
}

/* Diagnostic, for tests without a device: the rows (heads of a group times `count` new tokens) of a sequence of `len` positions
 * that see some of the positions k0 .. k1 - 1, as the kernels of many rows find them: [out[0], out[1]). */
extern "C" void aoship_internal_kv_weigh_rows(int g, int window, int count, int len, int k0, int k1, int *out) {
  const Rows r = rows_of(Seq{0, count, len}, Span{len - count, window}, g, k0, k1);
  out[0] = r.ra;
  out[1] = r.rb;
}

/* The launches of a batch, for tests without a device: out = {few, rows of a chunk, chunks of each sequence (0: their own),
 * chunks, 256-row pieces of each, pieces, padded length}; returns the workspace's bytes, 0 for a batch too large. */
extern "C" size_t aoship_internal_kv_weigh_shape(int nkv, int nh, int n_seqs, int n_tokens, int max_new, int max_len, int *out) {
  aos_kv_weigh_params p = {};
  p.b.nkv = nkv;
  p.b.n_seqs = n_seqs;
  p.b.n_tokens = n_tokens;
  p.b.max_new = max_new < n_tokens ? max_new : n_tokens;
  p.b.max_len = max_len;
  p.nh = nh;
  size_t bytes = 0;
  if (!aos_kv_weigh_shape(&p, &bytes)) return 0;
  const int got[7] = {p.few, p.rc, p.chunks, p.slots, p.row_pieces, p.row_slots, p.lpad};
  for (int i = 0; i < 7; ++i) out[i] = got[i];
  return bytes;
}
/* number of sequence s's first share */
extern "C" long long aoship_internal_kv_weigh_share(int unit, int each, int g, int s, int row0) {
  return Shares{unit, each}.base(g, s, row0);
}

#define KV_DISPATCH(fn, fmt, hdp, ...)                                       \
  ((hdp) == 64 ? ((fmt) == AOS_KV_BF16    ? fn<AOS_KV_BF16, 64>(__VA_ARGS__)    \
                  : (fmt) == AOS_KV_MXFP8 ? fn<AOS_KV_MXFP8, 64>(__VA_ARGS__)   \
                                          : fn<AOS_KV_MXFP4, 64>(__VA_ARGS__))  \
   : (hdp) == 128 ? ((fmt) == AOS_KV_BF16    ? fn<AOS_KV_BF16, 128>(__VA_ARGS__)   \
                     : (fmt) == AOS_KV_MXFP8 ? fn<AOS_KV_MXFP8, 128>(__VA_ARGS__)  \
                                             : fn<AOS_KV_MXFP4, 128>(__VA_ARGS__)) \
                  : ((fmt) == AOS_KV_BF16    ? fn<AOS_KV_BF16, 256>(__VA_ARGS__)   \
                     : (fmt) == AOS_KV_MXFP8 ? fn<AOS_KV_MXFP8, 256>(__VA_ARGS__)  \
                                             : fn<AOS_KV_MXFP4, 256>(__VA_ARGS__)))

extern "C" int aos_launch_kv_weigh(const aos_kv_weigh_params *p, const aos_launch_ctx *ctx) {
  return KV_DISPATCH(weigh, p->b.format, p->b.hdp, p, ctx);
}
