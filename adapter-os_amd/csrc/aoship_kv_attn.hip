/*
 * aoship_kv_attn.hip — attention of each sequence's new tokens over the paged key/value cache.
 *
 * For query head h of a token at position p, with the keys k_j and values v_j of its key/value head:
 *
 *   s_j = scale q . k_j,  j <= p (and j > p - window);   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max s_j
 *
 * in one pass over the tiles of 64 positions with the running m and sum in float32. The new tokens of a sequence
 * and the query heads that share a key/value head are one list of rows (token, head), so a tile is read once for
 * all of them.
 *
 * Matrix instructions' registers (aoship_device.h): every accumulator register is read, so results need no hold. Operands,
 * some of which vector instructions have just converted, are not held until the results are read: that would take
 * registers which the kernels do not have (256 of 256 and no private memory). The tests check the outputs with the whole
 * chip multiplying and converting at once, in every format, against float64 and run to run, bit for bit.
 */
#include "aoship_internal.h"
#include "aoship_kv.h"
#include <hip/hip_ext.h>

#include <type_traits>

using namespace kv;

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int SC1 = 16; /* buffer cache policy: device-coherent (sc1) */
constexpr float LOG2E = 1.44269504f;
constexpr float NINF = -__builtin_inff();
/* Running maximum of a row that has seen positions, whose scores were all minus infinity: its sum of zero makes it NaN,
 * that of a row that has seen nothing (NINF) zeros. */
constexpr float LEAST = -3.40282347e38f;
/* The running maximum of a row follows its scores only once they pass it by 2^SLACK (probabilities up to 256, an exact
 * power of two from what the true maximum would give): the accumulators are hardly ever rescaled. */
constexpr float SLACK = 8.0f;

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { /* round to nearest even */
  bf16x2 r;
  r[0] = (__bf16)a;
  r[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

/* the four lanes l % 16 + 16 j combined; every lane gets the result */
__device__ __forceinline__ float quad_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float y = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  const uint32_t v = __builtin_bit_cast(uint32_t, y);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float y = __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
  const uint32_t v = __builtin_bit_cast(uint32_t, y);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_bit_cast(float, (uint32_t)b[0]) + __builtin_bit_cast(float, (uint32_t)b[1]);
}
__device__ __forceinline__ float inverse(float sum, float m) {
  return sum != 0.0f ? 1.0f / sum : m == NINF ? 0.0f : __builtin_nanf("");
}
/* exponent base of a running maximum: a row that has seen nothing yet keeps its zero sum free of inf - inf */
__device__ __forceinline__ float safe_max(float m) { return m == NINF ? 0.0f : m; }

/* eight consecutive codes (of W words each 8) as the bfloat16 operand of a matrix instruction */
template <int FMT>
__device__ __forceinline__ u32x4 decode8(const uint32_t *w, float scale) {
  if constexpr (FMT == AOS_KV_BF16) {
    return u32x4{w[0], w[1], w[2], w[3]};
  } else if constexpr (FMT == AOS_KV_MXFP8) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, true))};
  } else {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 3))};
  }
}
/* Scale byte j of a word (constant once unrolled) as its power of two; 255 gives infinity, which times its zero codes is
 * NaN. Plain operations, two where one that selects a byte would do (24 streams of 32768 at 4 bits: 126 us and 124):
 * beside matrix instructions the compiler places wait states for what it knows, not for an asm statement. */
__device__ __forceinline__ float byte_scale(uint32_t w, int j) {
  return __builtin_bit_cast(float, (w >> 8 * j & 255u) << 23);
}

/* Infinities and NaNs among the values. In a tile that a row sees only in part, the product of such a value with a
 * probability of zero would reach rows that do not see it. Once one has entered the cache (a word that append sets), the
 * kernels look for them in such tiles: the matrix product gets zeros in their place, another one counts for each row and
 * dimension those that the row sees, by class, and the output takes them at the end (OddMarks). Quantised values need
 * this only where they pass through LDS as bfloat16: else a block's not-a-number scale is met by a probability that is
 * set to zero after scaling. */
/* The word with infinities and NaNs as zeros (cls < 0), or 1.0 where it holds +infinity (cls 0), -infinity (1) or a
 * NaN (2) and zeros elsewhere. */
__device__ __forceinline__ uint32_t odd_part(uint32_t w, int cls) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = (w >> (16 * i)) & 0xffffu;
    const bool odd = (h & 0x7f80u) == 0x7f80u;
    const int c = (h & 0x7fu) ? 2 : (int)(h >> 15);
    const uint32_t x = cls < 0 ? (odd ? 0u : h) : (odd && c == cls ? 0x3f80u : 0u);
    r |= x << (16 * i);
  }
  return r;
}
__device__ __forceinline__ u32x4 odd_part(u32x4 w, int cls) {
  return u32x4{odd_part(w[0], cls), odd_part(w[1], cls), odd_part(w[2], cls), odd_part(w[3], cls)};
}
/* N accumulator elements' marks, a bit each for +infinity, -infinity and NaN seen */
template <int N>
struct OddMarks {
  uint32_t bit[3][(N + 31) / 32];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < 3; ++c)
#pragma unroll
      for (int i = 0; i < (N + 31) / 32; ++i) bit[c][i] = 0u;
  }
  __device__ __forceinline__ void set(int cls, int i, uint32_t bits) { /* cls need not be constant */
    bit[0][i] |= cls == 0 ? bits : 0u;
    bit[1][i] |= cls == 1 ? bits : 0u;
    bit[2][i] |= cls == 2 ? bits : 0u;
  }
  __device__ __forceinline__ float apply(int i, float x) const {
    if (bit[0][i / 32] >> (i % 32) & 1) x = x + __builtin_inff();
    if (bit[1][i / 32] >> (i % 32) & 1) x = x - __builtin_inff();
    if (bit[2][i / 32] >> (i % 32) & 1) x = x + __builtin_nanf("");
    return x;
  }
};
/* Weight of a piece whose maximum is m in a sum whose maximum is ms. Zero would turn an infinity that the row sees into a
 * NaN, and a weight kept at 2^-126 would let values near 2^128 count: where there are infinities (MARK), a weight below
 * that is 2^-126 twice, which leaves less than 2^-123 of anything finite. */
template <bool MARK>
struct Weight {
  float f, g;
  __device__ __forceinline__ Weight(float m, float ms) : f(ex2(m - ms)), g(1.0f) {
    constexpr float TINY = 1.17549435e-38f;
    if (MARK && f < TINY) f = g = TINY;
  }
  __device__ __forceinline__ float operator()(float x) const { return MARK ? x * f * g : x * f; }
};

/* ---- sharing the work ------------------------------------------------------------------------ */

/* What of a sequence the attention walks: rows (token, head) in row tiles of R, each over nt tiles from tile t0 on.
 * A sequence with rows but no positions has one tile, in which nothing is visible; one of more than `few` rows is the
 * other kernel's. */
struct Work {
  Seq q;
  int rows, rts, t0, nt;
};
template <int R>
__device__ __forceinline__ Work work_of(const aos_kv_attn_params &p, int few, const Seq &q) {
  Work w;
  w.q = q;
  w.rows = q.count * (p.nh / p.b.nkv);
  w.rts = w.rows > few ? 0 : (w.rows + R - 1) / R;
  const int first = q.len - q.count - p.window + 1; /* first position that the first row sees */
  w.t0 = p.window > 0 && first > 0 ? first / TILE : 0;
  w.nt = (q.len + TILE - 1) / TILE - w.t0;
  if (w.nt < 1) w.nt = 1;
  return w;
}

__device__ __forceinline__ int wave_scan(int x, int lane) { /* inclusive sum over lanes */
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = (int)aos_shfl((uint32_t)x, lane - d);
    if (lane >= d) x += y;
  }
  return x;
}

/* Shares are of weights: a row tile's position tiles and, for its beginning and end (its queries, its first tile's
 * latency, the joining of its waves, its output), as many more as they take the time of. A border that would cut fewer
 * than SNAP tiles off a row tile moves to the row tile's end. */
constexpr int SNAP = 3;

/* ---- few rows: 16 to a wave, the cache streamed through registers ------------------------------ */

/* A workgroup takes an even share of all (sequence, key/value head, row tile, tile of positions); its four waves
 * take the tiles of a row tile in turn. Scores S^T[position][row] = K . Q^T, output O^T[dimension][row] = V^T . P^T
 * by v_mfma_f32_16x16x32_bf16: the accumulator of block b (of four 16-position blocks) holds rows 4 quad + i, and
 * the row 4 j + i of block b is made position 16 j + 4 b + i, so a lane's scores are the 16 consecutive positions
 * 16 quad ..+15, which is what the value units hold: the probabilities never cross lanes. Probabilities are rounded
 * to bfloat16 for the second product (half a unit of 8 bits each, like the output's own rounding); sums are float32.
 * In the quantised formats the value scales multiply the probabilities (exactly: powers of two).
 *
 * Bound by reading the cache once, by latency where that is little. Keys and values go straight to registers, the next
 * tile's on their way while one is worked on: a tile is used by one workgroup's one or two matrix instructions a block,
 * which LDS would not speed up. 64 streams of up to 16001 positions, 28/4 heads of 128: 16 bits 228 us, 5.7 TB/s; 32 of up
 * to 8191, 24/8 heads, 8 bits: 73 us, 4.6 TB/s; 24 of 32768, 40/8 heads, 4 bits: 122 us, 4.7 TB/s. The quantised ones wait
 * half of the waves' time with half as many bytes on their way (67 KB a CU for 128): not memory's limit, which 16 bits
 * come nearer, nor the vector instructions' (a quarter fewer of a decoded tile's 470: 1%). */
template <int FMT, int HDP>
struct Tile { /* a tile's keys and values in registers */
  static constexpr int KW = HDP * bits<FMT>() / 128; /* words of a key row's quarter */
  static constexpr int VW = bits<FMT>() / 2;         /* words of a value unit */
  static constexpr int DB = HDP / 16, NBLK = HDP / 32;
  static constexpr int KB = HDP == 256 ? 2 : 1; /* key scale blocks of a lane */
  uint32_t k[4][KW];
  uint32_t v[DB][VW];
  uint32_t ks[KB];
  u32x4 vs[FMT == AOS_KV_BF16 ? 1 : NBLK];

  __device__ __forceinline__ void load_k(const unsigned char *t, int lane) {
    const int r = lane & 15, quad = lane >> 4;
    const __attribute__((address_space(1))) unsigned char *g = (const __attribute__((address_space(1))) unsigned char *)t;
    if constexpr (FMT == AOS_KV_MXFP4 && HDP == 64) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int pos = 16 * (r >> 2) + 4 * b + (r & 3);
        const u32x2 w = *(const __attribute__((address_space(1))) u32x2 *)(g + ((quad >> 1) * TILE + pos) * 16 + 8 * (quad & 1));
        k[b][0] = w.x;
        k[b][1] = w.y;
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int pos = 16 * (r >> 2) + 4 * b + (r & 3);
#pragma unroll
        for (int i = 0; i < KW / 4; ++i) {
          const u32x4 w = aos_gld16(t + ((quad * (KW / 4) + i) * TILE + pos) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) k[b][4 * i + j] = w[j];
        }
      }
    }
    if constexpr (FMT != AOS_KV_BF16) {
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        const int blk = HDP == 64 ? quad >> 1 : quad * KB + i;
        ks[i] = *(const __attribute__((address_space(1))) uint32_t *)(g + ks_off<FMT, HDP>() + blk * TILE + 16 * (r >> 2) + 4 * (r & 3));
      }
    }
  }
  __device__ __forceinline__ void load_v(const unsigned char *t, int lane) {
    const int r = lane & 15, quad = lane >> 4;
    const unsigned char *g = t + v_off<FMT, HDP>();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if constexpr (FMT == AOS_KV_MXFP4) {
        const u32x2 w = *(const __attribute__((address_space(1))) u32x2 *)(g + (quad * HDP + 16 * d + r) * 8);
        v[d][0] = w.x;
        v[d][1] = w.y;
      } else {
#pragma unroll
        for (int i = 0; i < VW / 4; ++i) {
          const u32x4 w = aos_gld16(g + (((VW / 4) * quad + i) * HDP + 16 * d + r) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[d][4 * i + j] = w[j];
        }
      }
    }
    if constexpr (FMT != AOS_KV_BF16) {
#pragma unroll
      for (int i = 0; i < NBLK; ++i) vs[i] = aos_gld16(t + vs_off<FMT, HDP>() + i * TILE + 16 * quad);
    }
  }
};

template <int HDP, int NB>
constexpr int part_floats() { /* of a piece: maxima and sums [NB][2][16], then the output accumulators */
  return NB * (32 + 16 * HDP);
}

template <int HDP, int NB>
struct RowsShared {
  float red[2][NB * HDP / 4][64]; /* accumulators of two waves */
  float mls[4][2][NB][64];        /* the waves' maxima and sums */
  uint32_t last;
};

constexpr int ROWS_SETUP = 5; /* weight of a row tile beside its position tiles */

/* LEAN: a tile's keys and values are loaded as their turn comes, not a tile ahead (half the registers) */

template <int FMT, int HDP, int NB, bool MARK, bool LEAN>
__device__ __forceinline__ void rows_body(const aos_kv_attn_params &p, int few, int min_share, RowsShared<HDP, NB> &sh) {
  constexpr int R = 16 * NB, DB = HDP / 16, KS = HDP / 32, W8 = bits<FMT>() / 4; /* W8: words of 8 codes */
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int G = gridDim.x, w = blockIdx.x;
  const int g = p.nh / p.b.nkv;

  /* The sequences go by 64 at a time, one a lane: all weights, this workgroup's share [u, u1) of them, and the
   * sequence that u falls in. */
  int c0 = 0; /* the first sequence that the lanes hold */
  Seq held;
  auto hold = [&](int s0) {
    c0 = s0;
    held = s0 + lane < p.b.n_seqs ? seq_at(p.b, s0 + lane) : Seq{0, 0, 0};
    const Work x = work_of<R>(p, few, held);
    return p.b.nkv * x.rts * (x.nt + ROWS_SETUP);
  };
  int mine = hold(0), upto = wave_scan(mine, lane);
  int total = __builtin_amdgcn_readlane(upto, 63);
  for (int s0 = 64; s0 < p.b.n_seqs; s0 += 64) total += __builtin_amdgcn_readlane(wave_scan(hold(s0), lane), 63);
  int share = (total + G - 1) / G;
  if (share < min_share) share = min_share;
  const int u = w * share;
  if (u >= total) return;
  const int u1 = u + share < total ? u + share : total;
  int base = 0; /* weights before sequence s */
  if (c0) {
    mine = hold(0);
    upto = wave_scan(mine, lane);
  }
  while (__builtin_amdgcn_readlane(upto, 63) + base <= u) { /* (u < total) */
    base += __builtin_amdgcn_readlane(upto, 63);
    mine = hold(c0 + 64);
    upto = wave_scan(mine, lane);
  }
  int s;
  {
    const int l = __builtin_ctzll(__ballot(upto + base > u));
    s = c0 + l;
    base += __builtin_amdgcn_readlane(upto - mine, l);
  }

  /* (a scale of zero stays above it, so that what a row does not see keeps -infinity) */
  const float cs = fmaxf(fabsf(p.scale) * LOG2E, 1.17549435e-38f);
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u; /* a negative scale: negated queries */
  for (int place = -1, seg = 0; place < u1;) { /* place: where row tile seg of sequence s begins among the weights */
    if (s >= c0 + 64) (void)hold(s);
    Seq sq;
    sq.row0 = __builtin_amdgcn_readlane(held.row0, s - c0);
    sq.count = __builtin_amdgcn_readlane(held.count, s - c0);
    sq.len = __builtin_amdgcn_readlane(held.len, s - c0);
    const Work x = work_of<R>(p, few, sq);
    const int weight = x.nt + ROWS_SETUP;
    if (place < 0) { /* the first: the border may be anywhere in it */
      seg = (u - base) / weight;
      place = base + seg * weight;
    }
    if (seg >= p.b.nkv * x.rts) { /* the next sequence's */
      if (++s >= p.b.n_seqs) break;
      seg = 0;
      continue;
    }
    auto cut = [&](int at) { /* the tile before which a border at weight `at` cuts this row tile */
      const int t = at - place - ROWS_SETUP;
      return t < SNAP ? 0 : x.nt - t < SNAP ? x.nt : t;
    };
    const int j = u > place ? cut(u) : 0, je = u1 < place + weight ? cut(u1) : x.nt, n = je - j;
    const int h = seg / x.rts, rt = seg - h * x.rts, at0 = place;
    ++seg;
    place += weight;
    if (n <= 0) continue;
    const int r0 = rt * R, nrows = x.rows - r0 < R ? x.rows - r0 : R;
    const int p0 = x.q.len - x.q.count; /* position of the sequence's first new token */

    /* this lane's rows: query, and the positions [lo, hi] that it sees */
    u32x4 qf[NB][KS];
    int lo[NB], hi[NB];
    long long orow[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int rr = 16 * b + col < nrows ? 16 * b + col : nrows - 1, row = r0 + rr;
      const int t = row / g, hh = h * g + row - t * g;
      hi[b] = p0 + t;
      lo[b] = p.window > 0 && hi[b] - p.window + 1 > 0 ? hi[b] - p.window + 1 : 0;
      const uint16_t *qr = p.q + (long long)(x.q.row0 + t) * p.q_ld + hh * p.b.hd;
      orow[b] = (long long)(x.q.row0 + t) * p.out_ld + hh * p.b.hd;
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        const int d = quad * (HDP / 4) + 8 * e;
        qf[b][e] = d < p.b.hd && 16 * b + col < nrows ? aos_gld16(qr + d) : u32x4{};
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[b][e][i] ^= flip;
      }
    }
    const int t_first = r0 / g, t_last = (r0 + nrows - 1) / g;
    const int hi_min = p0 + t_first, hi_max = p0 + t_last;
    const int lo_max = p.window > 0 && p0 + t_last - p.window + 1 > 0 ? p0 + t_last - p.window + 1 : 0;

    f32x4 o[NB][DB];
    float m[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b] = NINF;
      l[b] = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[b][d] = f32x4{};
    }

    OddMarks<NB * DB * 4> marks;
    if constexpr (MARK) marks.clear();

    /* tiles of this wave: j + wave, j + wave + 4, ..., up to the last that the row tile sees */
    const int sees = hi_max / TILE - x.t0 + 1 - j, mine = ((sees < n && hi_max >= 0 ? sees : n) - wave + 3) / 4;
    for (int i0 = 0; i0 < mine; i0 += 64) {
      const int cnt = mine - i0 < 64 ? mine - i0 : 64;
      /* the pages of the next 64 tiles, one a lane */
      int pg = -1;
      {
        const int pos = (x.t0 + j + wave + 4 * (i0 + lane)) * TILE;
        if (lane < cnt && pos < x.q.len) pg = page_of(p.b, s, pos);
      }
      Tile<FMT, HDP> tl;
      auto ptr = [&](int i) {
        const int page = __builtin_amdgcn_readlane(pg, i);
        return tile_ptr<FMT, HDP>(p.b, page < 0 ? 0 : page, h, (x.t0 + j + wave + 4 * (i0 + i)) * TILE);
      };
      {
        const unsigned char *t = ptr(0);
        if (!LEAN) tl.load_k(t, lane);
        if (!LEAN) tl.load_v(t, lane);
      }
      for (int i = 0; i < cnt; ++i) {
        const int tb = (x.t0 + j + wave + 4 * (i0 + i)) * TILE;
        const bool there = __builtin_amdgcn_readlane(pg, i) >= 0;
        const unsigned char *next = ptr(i + 1 < cnt ? i + 1 : i), *here = ptr(i);
        if (LEAN) tl.load_k(here, lane);
        f32x4 sc[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int k = 0; k < 4; ++k) sc[b][k] = f32x4{};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < KS; ++e) {
            const float ksc = FMT == AOS_KV_BF16 ? 1.0f : byte_scale(tl.ks[e * Tile<FMT, HDP>::KB / KS], k);
            const u32x4 a = decode8<FMT>(&tl.k[k][e * W8], ksc);
#pragma unroll
            for (int b = 0; b < NB; ++b) sc[b][k] = mfma16(a, qf[b][e], sc[b][k]);
          }
        if (!LEAN && i + 1 < cnt) tl.load_k(next, lane);
        if (LEAN) tl.load_v(here, lane);

        const bool edge = !there || tb < lo_max || tb + TILE - 1 > hi_min; /* uniform */
        /* most tiles need no masks: two copies where the registers allow it, else one that asks as it goes */
        auto work = [&](auto copy) {
          constexpr int COPY = decltype(copy)::value; /* 0: without masks, 1: with them, 2: either */
          const bool masks = COPY == 1 || (COPY == 2 && edge);
          uint32_t seen[NB]; /* bit 4 b + i: the row sees position 16 quad + 4 b + i of the tile */
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            seen[b] = 0xffffu;
            if (masks) {
              const int at = tb + 16 * quad;
              seen[b] = 0;
#pragma unroll
              for (int k = 0; k < 16; ++k)
                if (there && at + k >= lo[b] && at + k <= hi[b]) seen[b] |= 1u << k;
            }
          }
          u32x4 pf[NB][2]; /* probabilities: operand of the second product */
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float mx = NINF;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (masks && !(seen[b] >> k & 1)) sc[b][k >> 2][k & 3] = NINF;
              mx = fmaxf(mx, sc[b][k >> 2][k & 3]);
            }
            mx = quad_max(mx) * cs;
            if (!masks || (there && lo[b] < tb + TILE && hi[b] >= tb)) mx = fmaxf(mx, LEAST);
            if (__ballot(mx > m[b] + SLACK)) {
              const float top = fmaxf(m[b], mx), alpha = ex2(m[b] - safe_max(top));
              l[b] = l[b] * alpha;
#pragma unroll
              for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[b][d][k] = o[b][d][k] * alpha;
              m[b] = top;
            }
            const float ms = safe_max(m[b]);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float e = ex2(fmaf(sc[b][k >> 2][k & 3], cs, -ms));
              l[b] = l[b] + e;
              sc[b][k >> 2][k & 3] = e;
            }
            if constexpr (FMT == AOS_KV_BF16) {
#pragma unroll
              for (int t = 0; t < 2; ++t)
                pf[b][t] = u32x4{pack_bf16(sc[b][2 * t][0], sc[b][2 * t][1]), pack_bf16(sc[b][2 * t][2], sc[b][2 * t][3]),
                                 pack_bf16(sc[b][2 * t + 1][0], sc[b][2 * t + 1][1]),
                                 pack_bf16(sc[b][2 * t + 1][2], sc[b][2 * t + 1][3])};
            }
          }
          if (MARK && masks) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
#pragma unroll 1
              for (int cls = 0; cls < 3; ++cls)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                  f32x4 c = {};
#pragma unroll
                  for (int t = 0; t < 2; ++t) {
                    u32x4 a, sf;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                      a[k] = odd_part(tl.v[d][(4 * t + k) % Tile<FMT, HDP>::VW], cls);
                      sf[k] = (seen[b] >> (8 * t + 2 * k) & 1 ? 0x3f80u : 0u) |
                              (seen[b] >> (8 * t + 2 * k + 1) & 1 ? 0x3f800000u : 0u);
                    }
                    c = mfma16(a, sf, c);
                  }
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const int e = (b * DB + d) * 4 + k;
                    marks.set(cls, e / 32, c[k] > 0.0f ? 1u << (e % 32) : 0u);
                  }
                }
#pragma unroll
              for (int k = 0; k < Tile<FMT, HDP>::VW; ++k) tl.v[d][k] = odd_part(tl.v[d][k], -1);
            }
          }
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            if constexpr (FMT != AOS_KV_BF16) {
              if (d % 2 == 0) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                  for (int t = 0; t < 2; ++t) {
                    float y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                      y[k] = sc[b][2 * t + (k >> 2)][k & 3] * byte_scale(tl.vs[d / 2][2 * t + (k >> 2)], k & 3);
                      /* (a scale that is not a number, of a position that the row does not see) */
                      if (masks) y[k] = seen[b] >> (8 * t + k) & 1 ? y[k] : 0.0f;
                    }
                    pf[b][t] = u32x4{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]),
                                     pack_bf16(y[6], y[7])};
                  }
              }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const u32x4 a = decode8<FMT>(&tl.v[d][t * W8], 1.0f);
#pragma unroll
              for (int b = 0; b < NB; ++b) o[b][d] = mfma16(a, pf[b][t], o[b][d]);
            }
          }
        };
        if constexpr (FMT == AOS_KV_BF16 || NB > 1 || HDP == 256)
          work(std::integral_constant<int, 2>{});
        else if (edge)
          work(std::integral_constant<int, 1>{});
        else
          work(std::integral_constant<int, 0>{});
        if (!LEAN && i + 1 < cnt) tl.load_v(next, lane);
      }
    }

    if constexpr (MARK)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[b][d][k] = marks.apply((b * DB + d) * 4 + k, o[b][d][k]);

    /* the waves' pieces into wave 0's: one maximum, then their sums two by two */
    auto join_waves = [&]() {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        sh.mls[wave][0][b][lane] = m[b];
        sh.mls[wave][1][b][lane] = l[b];
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float top = NINF;
#pragma unroll
        for (int v = 0; v < 4; ++v) top = fmaxf(top, sh.mls[v][0][b][lane]);
        const float ms = safe_max(top);
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; ++v) sum = sum + Weight<MARK>(sh.mls[v][0][b][lane], ms)(sh.mls[v][1][b][lane]);
        const Weight<MARK> f(m[b], ms);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[b][d][k] = f(o[b][d][k]);
        m[b] = top;
        l[b] = sum;
      }
#pragma unroll
      for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int k = 0; k < 4; ++k) sh.red[wave - half][(b * DB + d) * 4 + k][lane] = o[b][d][k];
        __syncthreads();
        if (wave < half)
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int k = 0; k < 4; ++k) o[b][d][k] = o[b][d][k] + sh.red[wave][(b * DB + d) * 4 + k][lane];
        __syncthreads();
      }
    };
#pragma unroll
    for (int b = 0; b < NB; ++b) l[b] = quad_sum(l[b]);
    if (n > 1) join_waves(); /* (one tile is wave 0's) */

    auto put = [&](int b, int d, f32x4 y, float inv) {
      const int at = 16 * d + 4 * quad;
      if (16 * b + col < nrows && at < p.b.hd)
        *(u32x2 *)(p.out + orow[b] + at) = u32x2{pack_bf16(y[0] * inv, y[1] * inv), pack_bf16(y[2] * inv, y[3] * inv)};
    };
    bool done = n == x.nt;
    if (!done) {
      /* a cut row tile: borders wf .. wl cut it, its pieces lie in slots of workgroups wf - 1 .. wl (2 w: the piece that w
       * begins with, 2 w + 1: the one that it ends with), and the last to arrive joins them: each of its waves every
       * fourth, several in flight */
      constexpr int PF = part_floats<HDP, NB>(), FLY = 4 / NB;
      const int wf = (at0 + ROWS_SETUP + SNAP + share - 1) / share, wl = (at0 + ROWS_SETUP + x.nt - SNAP) / share;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)p.part, (short)0, 0x7fffffff, 0x00020000);
      if (wave == 0) {
        const int slot = (2 * w + (j > 0 ? 0 : 1)) * PF;
        if (quad == 0)
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            aos_publish(p.part + slot + 32 * b + col, m[b]);
            aos_publish(p.part + slot + 32 * b + 16 + col, l[b]);
          }
#pragma unroll
        for (int b = 0; b < NB; ++b)
          if (16 * b + col < nrows)
#pragma unroll
            for (int d = 0; d < DB; ++d)
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[b][d]), rs,
                                                     (slot + 32 * NB + ((b * DB + d) * 64 + lane) * 4) * 4, 0, SC1);
        aos_mem_wait();
        if (lane == 0) {
          const uint32_t old = aos_arrive(p.counters + wf);
          if (old == (uint32_t)(wl - wf + 1)) aos_reset(p.counters + wf);
          sh.last = old == (uint32_t)(wl - wf + 1) ? 1u : 0u;
        }
      }
      __syncthreads();
      done = sh.last != 0;
      if (done) {
        const int np = wl - wf + 2;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          m[b] = NINF;
          l[b] = 0.0f;
#pragma unroll
          for (int d = 0; d < DB; ++d) o[b][d] = f32x4{};
        }
        for (int k0 = wave; k0 < np; k0 += 4 * FLY) {
          float pm[FLY][NB], pl[FLY][NB];
          f32x4 y[FLY][NB][DB];
#pragma unroll
          for (int i = 0; i < FLY; ++i) {
            const int k = k0 + 4 * i < np ? k0 + 4 * i : k0; /* (past the end: the first again, with no weight) */
            const int slot = (k == 0 ? 2 * wf - 1 : 2 * (wf + k - 1)) * PF;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              pm[i][b] = aos_collect(p.part + slot + 32 * b + col);
              pl[i][b] = aos_collect(p.part + slot + 32 * b + 16 + col);
#pragma unroll
              for (int d = 0; d < DB; ++d)
                y[i][b][d] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                           rs, (slot + 32 * NB + ((b * DB + d) * 64 + lane) * 4) * 4, 0, SC1));
            }
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float top = m[b];
#pragma unroll
            for (int i = 0; i < FLY; ++i) top = fmaxf(top, pm[i][b]);
            const float ms = safe_max(top);
            const Weight<MARK> f0(m[b], ms);
            l[b] = f0(l[b]);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[b][d][e] = f0(o[b][d][e]);
#pragma unroll
            for (int i = 0; i < FLY; ++i) {
              if (k0 + 4 * i >= np) continue; /* uniform */
              const Weight<MARK> f(pm[i][b], ms);
              l[b] = l[b] + f(pl[i][b]);
#pragma unroll
              for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][d][e] = o[b][d][e] + f(y[i][b][d][e]);
            }
            m[b] = top;
          }
        }
        join_waves();
      }
      __syncthreads(); /* sh.last is free again */
    }
    if (done && wave == 0)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float inv = inverse(l[b], m[b]);
#pragma unroll
        for (int d = 0; d < DB; ++d) put(b, d, o[b][d], inv);
      }
  }
}

/* waves per SIMD that the registers of a tile in flight and the accumulators leave room for */
constexpr int rows_waves(int fmt, int hdp, int nb) {
  return nb > 1 || hdp == 256 || (fmt == AOS_KV_BF16 && hdp == 128) ? 1 : 2;
}

/* two bodies, so that the registers of the rare one (infinities or NaNs in the cache) stay out of the other's way */
template <int FMT, int HDP, int NB>
__global__ void __launch_bounds__(256, rows_waves(FMT, HDP, NB)) aos_kv_rows_kernel(aos_kv_attn_params p, int few, int min_share) {
  __shared__ RowsShared<HDP, NB> sh;
  if constexpr (FMT == AOS_KV_BF16) {
    if (*p.b.nonfinite) {
      rows_body<FMT, HDP, NB, true, FMT == AOS_KV_BF16 && HDP == 256>(p, few, min_share, sh);
      return;
    }
  }
  rows_body<FMT, HDP, NB, false, FMT == AOS_KV_BF16 && HDP == 256>(p, few, min_share, sh);
}

/* ---- many rows: tiles of 128, keys and values through LDS ------------------------------------- */

/* Four waves of 32 rows walk a row tile's positions 64 at a time. A tile of the cache goes to LDS once for all of
 * them, as bfloat16 in the cache's own order (a bfloat16 tile as it lies, straight from memory; quantised ones
 * through registers), while the one before it is worked on: two stages, 64 KB for 128 dimensions, two workgroups a
 * CU, so that one's exponentials run under the other's matrix instructions.
 *
 * S^T = K . Q^T and O^T = V^T . P^T by v_mfma_f32_32x32x16_bf16. Row 16 s + 8 a + 4 c + i of a block of 32 keys is
 * position 16 c + 8 s + 4 a + i, which puts the 16 consecutive positions 16 c ..+15 on half c of the lanes, register
 * by register: what the value pieces hold, so the probabilities never cross lanes here either.
 *
 * The workgroups share all (key/value head, row tile, position tile) evenly; where a row tile is cut, its pieces meet
 * as in the kernel above. Neighbouring shares, which read the same keys, go to one XCD.
 *
 * Bound by the matrix cores. Prompt of 4076 tokens, 28/4 heads of 128, 16 bits: 142 us, 840 TFLOP/s (16304 tokens 1890 us,
 * 1010; a large library product 1140 on the same card); 512 tokens over 15872, 40/8 heads, 8 bits: 202 us, 830 TFLOP/s.
 * Other cards took up to 155 and 215 us. With fragments read from LDS just before each matrix instruction 200 us for 151,
 * with row tiles dealt whole 210. */
constexpr int TR = 128;         /* rows of a row tile */
constexpr int tiles_per_cu(int hdp) { return hdp == 256 ? 1 : 2; }

template <int HDP>
constexpr int tile_part_floats() { /* of a piece: maxima and sums [4 waves][2][32], then the accumulators */
  return 4 * 64 + TR * HDP;
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float half_max(float x) { /* with the lane 32 away */
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
}

/* Four positions of two dimensions (a word of 8-bit codes each, or the low halves of words of 4-bit ones) as bfloat16
 * pairs of positions {dimension 0: 01, 23, dimension 1: 01, 23}: the codes of a position side by side, so that one
 * conversion applies its scale to both, then the positions side by side. */
template <int FMT>
__device__ __forceinline__ u32x4 decode4x2(uint32_t w0, uint32_t w1, const float *scale) {
  uint32_t x[4];
  if constexpr (FMT == AOS_KV_MXFP8) {
    const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400u), hi = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
    x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale[0], false));
    x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale[1], true));
    x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale[2], false));
    x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale[3], true));
  } else { /* nibbles of positions 0 .. 3: even ones (position 0, 2) and odd ones (1, 3), a byte a position */
    const uint32_t even = (w0 & 0x0f0fu) | ((w1 << 4) & 0xf0f0u), odd = ((w0 >> 4) & 0x0f0fu) | (w1 & 0xf0f0u);
    x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(even, scale[0], 0));
    x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(odd, scale[1], 0));
    x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(even, scale[2], 1));
    x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(odd, scale[3], 1));
  }
  return u32x4{__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
               __builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
}

/* A tile on its way to LDS (keys at `dst`, values TILE * HDP * 2 bytes after them). fetch() starts it, put() (of the
 * quantised formats) writes what fetch() loaded; the caller waits and synchronises. */
template <int FMT, int HDP>
struct Stage {
  static constexpr int KU = HDP * bits<FMT>() / 128 * TILE / 256; /* key units of a thread */
  static constexpr int VPAIRS = 4 * HDP / 2; /* pairs of value units: dimensions d and d + 16 of a block of 32 */
  static constexpr int VP = (VPAIRS + 255) / 256;
  static constexpr int VW = bits<FMT>() / 2;
  static __device__ __forceinline__ bool has(int tid, int i) { return tid + 256 * i < VPAIRS; }
  static __device__ __forceinline__ int unit(int tid, int i) { return (tid + 256 * i) / (HDP / 2); }
  static __device__ __forceinline__ int dim(int tid, int i) {
    const int c = (tid + 256 * i) % (HDP / 2);
    return (c & ~15) * 2 + (c & 15);
  }
  static constexpr bool Q = FMT != AOS_KV_BF16;
  u32x4 k[Q ? (KU ? KU : 1) : 1];
  uint32_t v[Q ? VP : 1][2][Q ? VW : 1];
  u32x4 vs[Q ? VP : 1];
  uint32_t ks[Q ? (KU ? KU : 1) : 1];

  __device__ __forceinline__ void fetch(const unsigned char *t, unsigned char *dst, int tid) {
    if constexpr (!Q) {
      const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      constexpr int N = 4 * TILE * HDP / 1024 / 4;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)t, (short)0, 4 * TILE * HDP, 0x00020000);
#pragma unroll
      for (int i = 0; i < N; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void *)(dst + (4 * i + wave) * 1024), 16, lane * 16, (4 * i + wave) * 1024, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < (KU ? KU : 1); ++i) {
        const int c = tid + 256 * i, pos = c & 63, u = c >> 6;
        if (KU == 0 && u >= HDP * bits<FMT>() / 128) break;
        k[i] = aos_gld16(t + (u * TILE + pos) * 16);
        ks[i] = *(const __attribute__((address_space(1))) unsigned char *)(t + ks_off<FMT, HDP>() +
                                                                          (u * (128 / bits<FMT>()) / 32) * TILE + ks_index(pos));
      }
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        if (!has(tid, i)) break;
        const int d = dim(tid, i), u = unit(tid, i);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned char *g = t + v_off<FMT, HDP>() + (u * HDP + d + 16 * e) * (4 * VW);
          if constexpr (FMT == AOS_KV_MXFP8) {
            const u32x4 w = aos_gld16(g);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][e][j % VW] = w[j];
          } else {
            const u32x2 w = *(const __attribute__((address_space(1))) u32x2 *)g;
            v[i][e][0] = w.x;
            v[i][e][1] = w.y;
          }
        }
        vs[i] = aos_gld16(t + vs_off<FMT, HDP>() + (d >> 5) * TILE + 16 * u);
      }
    }
  }
  __device__ __forceinline__ void put(unsigned char *dst, int tid) {
    if constexpr (Q) {
#pragma unroll
      for (int i = 0; i < (KU ? KU : 1); ++i) {
        const int c = tid + 256 * i, pos = c & 63, u = c >> 6;
        if (KU == 0 && u >= HDP * bits<FMT>() / 128) break;
        constexpr int PER = 16 / bits<FMT>(); /* 16-byte bfloat16 units of a unit of codes */
        uint32_t w[4] = {k[i][0], k[i][1], k[i][2], k[i][3]};
#pragma unroll
        for (int j = 0; j < PER; ++j)
          *(u32x4 *)(dst + ((u * PER + j) * TILE + pos) * 16) = decode8<FMT>(&w[j * (4 / PER)], byte_scale(ks[i], 0));
      }
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        if (!has(tid, i)) break;
        const int d = dim(tid, i), u = unit(tid, i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u32x4 r[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) { /* positions 8 j + 4 k ..+3 */
            float sc[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[e] = byte_scale(vs[i][2 * j + k], e);
            const uint32_t w0 = FMT == AOS_KV_MXFP8 ? v[i][0][(2 * j + k) % VW] : v[i][0][j % VW] >> (16 * k);
            const uint32_t w1 = FMT == AOS_KV_MXFP8 ? v[i][1][(2 * j + k) % VW] : v[i][1][j % VW] >> (16 * k);
            const u32x4 x = decode4x2<FMT>(w0, w1, sc);
            r[0][2 * k] = x[0], r[0][2 * k + 1] = x[1], r[1][2 * k] = x[2], r[1][2 * k + 1] = x[3];
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) *(u32x4 *)(dst + TILE * HDP * 2 + ((2 * u + j) * HDP + d + 16 * e) * 16) = r[e];
        }
      }
    }
  }
};

/* Row tile slots of a batch: sequence s, whose rows begin at `start`, has its row tiles from slot_base() on, fewer than the
 * next one's base. Starts outside the batch's rows (of sequences that do not fit) count as its ends, so that the bases
 * ascend wherever the starts do; the kernel takes no batch whose starts fall: which sequence a slot belongs to would depend
 * on where a walk comes from, and workgroups that share a row tile would expect other arrivals than come. */
__host__ __device__ __forceinline__ int slot_base(const aos_kv_batch &b, int start, int g, int s) {
  start = start < 0 ? 0 : start > b.n_tokens ? b.n_tokens : start;
  return (int)((long long)start * g / TR) + s;
}
/* whether the starts of every n-th sequence from the first-th on fall */
__host__ __device__ __forceinline__ bool starts_fall(const aos_kv_batch &b, int first, int n) {
  bool fall = false;
  for (int s = first; s < b.n_seqs; s += n) fall |= b.starts[s + 1] < b.starts[s];
  return fall;
}

/* Where a walk over the slots is: sequence s, which has the slots base .. next - 1. */
struct Cursor {
  Seq q;
  int s, base, next;
};
__host__ __device__ __forceinline__ void open(const aos_kv_batch &b, int g, int s, Cursor &c) {
  const int r0 = b.starts[s], r1 = b.starts[s + 1];
  c.s = s;
  c.q = seq_of(b, r0, r1, b.lens[s]);
  c.base = slot_base(b, r0, g, s);
  c.next = s + 1 < b.n_seqs ? slot_base(b, r1, g, s + 1) : 0x7fffffff;
}
__host__ __device__ __forceinline__ void seek(const aos_kv_batch &b, int g, int slot, Cursor &c) {
  int lo = 0, hi = b.n_seqs; /* the last sequence whose slots begin at or before `slot` */
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (slot_base(b, b.starts[mid], g, mid) <= slot)
      lo = mid;
    else
      hi = mid;
  }
  open(b, g, lo, c);
}

/* (for a wave whose lanes all hold the same: kept in scalar registers) */
__host__ __device__ __forceinline__ void uniform(Cursor &c) {
#ifdef __HIP_DEVICE_COMPILE__
  c.q.row0 = __builtin_amdgcn_readfirstlane(c.q.row0);
  c.q.count = __builtin_amdgcn_readfirstlane(c.q.count);
  c.q.len = __builtin_amdgcn_readfirstlane(c.q.len);
  c.s = __builtin_amdgcn_readfirstlane(c.s);
  c.base = __builtin_amdgcn_readfirstlane(c.base);
  c.next = __builtin_amdgcn_readfirstlane(c.next);
#endif
}

/* A row tile: rows r0 .. r0 + rows - 1 of its sequence and the position tiles t0 .. t0 + nt - 1 that they see (at least
 * one). nt 0: no such row tile, or one of a sequence of few rows. */
struct RowTile {
  int r0, rows, t0, nt;
};
__host__ __device__ __forceinline__ RowTile row_tile(const aos_kv_attn_params &p, int g, int few, const Cursor &c, int slot) {
  RowTile o = {};
  const int all = c.q.count * g, r = slot - c.base;
  if (all <= few || r < 0 || r > (all - 1) / TR) return o; /* (slots times TR may pass 32 bits) */
  o.r0 = r * TR;
  o.rows = all - o.r0 < TR ? all - o.r0 : TR;
  const int p0 = c.q.len - c.q.count;
  const int first = p0 + o.r0 / g, last = p0 + (o.r0 + o.rows - 1) / g;
  const int low = p.window > 0 && first - p.window + 1 > 0 ? first - p.window + 1 : 0;
  o.t0 = low / TILE;
  o.nt = (last < 0 ? 0 : last / TILE) - o.t0 + 1;
  return o;
}

constexpr int SETUP = 4; /* weight of a row tile beside its position tiles */

/* The weights of a key/value head are counted in runs of slots, each from a cursor at the run's first slot on: a run's sum,
 * and where a border at weight v of it falls: a slot and the position tile of its row tile that the border cuts off (0:
 * the border is at the row tile's beginning). */
__host__ __device__ __forceinline__ int run_weight(const aos_kv_attn_params &p, int g, int few, Cursor c, int first, int end) {
  int sum = 0;
  for (int x = first; x < end; ++x) {
    while (x >= c.next) open(p.b, g, c.s + 1, c);
    const int nt = row_tile(p, g, few, c, x).nt;
    sum += nt ? nt + SETUP : 0;
  }
  return sum;
}
__host__ __device__ __forceinline__ void run_border(const aos_kv_attn_params &p, int g, int few, Cursor &c, int first,
                                                    int end, int v, int &slot, int &j) {
  for (int x = first; x < end; ++x) {
    while (x >= c.next) open(p.b, g, c.s + 1, c);
    const int nt = row_tile(p, g, few, c, x).nt, weight = nt ? nt + SETUP : 0;
    if (v < weight) {
      const int t = v - SETUP;
      slot = nt - t < SNAP ? x + 1 : x;
      j = t < SNAP || nt - t < SNAP ? 0 : t;
      return;
    }
    v -= weight;
  }
}

/* A workgroup's walk: at position tile j of head h's slot, up to position tile j1 of head h1's slot1. */
struct Walk {
  int h, slot, j, h1, slot1, j1;
};
/* Goes on to the next row tile, from the slot that the walk is at; false where its share ends. */
__host__ __device__ __forceinline__ bool next_row_tile(const aos_kv_attn_params &p, int g, int few, int slots, Walk &k,
                                                       Cursor &c, RowTile &x) {
  for (;; ++k.slot, k.j = 0) {
    if (k.slot >= slots) {
      if (++k.h >= p.b.nkv) return false;
      k.slot = 0;
      seek(p.b, g, 0, c);
      uniform(c);
    }
    if (k.h > k.h1 || (k.h == k.h1 && k.slot >= k.slot1 && (k.slot > k.slot1 || k.j1 == 0))) return false;
    while (k.slot >= c.next) {
      open(p.b, g, c.s + 1, c);
      uniform(c);
    }
    x = row_tile(p, g, few, c, k.slot);
    if (x.nt) return true;
  }
}
/* Borders wf .. wl cut the row tile of nt position tiles of which workgroup w has j .. je - 1 (not all). */
struct Cuts {
  int wf, wl;
};
__host__ __device__ __forceinline__ Cuts cuts_of(int w, int share, int j, int je, int nt) {
  const int place = (j > 0 ? w * share - j : (w + 1) * share - je) - SETUP; /* the row tile's place among the weights */
  return Cuts{(place + SETUP + SNAP + share - 1) / share, (place + SETUP + nt - SNAP) / share};
}

struct TilesShared {
  int scan[4], found[4], joins;
  Cursor at_first;
};

template <int FMT, int HDP, bool MARK>
__device__ __forceinline__ void tiles_body(const aos_kv_attn_params &p, int few, int slots, int min_share, TilesShared &sh) {
  constexpr int KS = HDP / 16, DB = HDP / 32, STAGE = 4 * TILE * HDP;
  /* What keeps the kernel within a wave's registers (workgroups hand pieces to each other: the build refuses private memory
   * here): fragments read ahead, blocks of 32 dimensions of a piece in flight as it is joined, and, for infinities in wide
   * quantised heads, the queries read again for each tile and 8-bit tiles fetched in their turn (for other caches that
   * would be 204 us for 127: 512 tokens over 8000, 16/2 heads of 256, 8 bits). */
  constexpr int AHEAD = MARK ? 2 : HDP == 256 ? 4 : 8;
  constexpr int FLY = MARK ? 1 : HDP == 256 ? 2 : FMT == AOS_KV_MXFP8 ? DB / 2 : DB;
  constexpr bool AGAIN = MARK && HDP == 256 && FMT != AOS_KV_BF16, LATE = AGAIN && FMT == AOS_KV_MXFP8;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int g = p.nh / p.b.nkv;
  const int G = gridDim.x, w = (int)(blockIdx.x % 8) * (G / 8) + (int)(blockIdx.x / 8);

  /* weights of a key/value head (each thread a run of slots), this workgroup's share, and its two borders */
  const int per = (slots + 255) / 256, first = tid * per, end = first + per < slots ? first + per : slots;
  Cursor own = {}, cur; /* own: where this thread's run begins */
  int sum = 0;
  if (first < end) {
    seek(p.b, g, first, own);
    sum = run_weight(p, g, few, own, first, end);
  }
  const int upto = wave_scan(sum, lane);
  if (lane == 63) sh.scan[wave] = upto;
  if (__syncthreads_or(starts_fall(p.b, tid, 256) ? 1 : 0)) {
    if (tid == 0) note(p.b.faults, AOS_KV_FAULT_BATCH);
    return;
  }
  int before = upto - sum, N = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < wave) before += sh.scan[i];
    N += sh.scan[i];
  }
  const int total = N * p.b.nkv;
  int share = (total + G - 1) / G;
  if (share < min_share) share = min_share;
  if (w * share >= total) return; /* uniform */
  Walk walk;
  walk.h = w * share / N;
  walk.h1 = p.b.nkv;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int border = (w + i) * share;
    if (border >= total) {
      if (tid == 0) sh.found[2] = sh.found[3] = 0;
      break;
    }
    const int hh = border / N, v = border - hh * N - before;
    if (i) walk.h1 = hh;
    if (v >= 0 && v < sum) {
      cur = own;
      run_border(p, g, few, cur, first, end, v, sh.found[2 * i], sh.found[2 * i + 1]);
      if (i == 0) sh.at_first = cur;
    }
  }
  __syncthreads();
  walk.slot = __builtin_amdgcn_readfirstlane(sh.found[0]);
  walk.j = __builtin_amdgcn_readfirstlane(sh.found[1]);
  walk.slot1 = __builtin_amdgcn_readfirstlane(sh.found[2]);
  walk.j1 = __builtin_amdgcn_readfirstlane(sh.found[3]);
  cur = sh.at_first;
  uniform(cur);
  const float cs = fmaxf(fabsf(p.scale) * LOG2E, 1.17549435e-38f);
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u; /* (both as above) */
  /* the table's entries for 64 tiles from pages_t on of a sequence, one a lane; checked only as a tile's turn comes: what no
   * row sees (left of a window) may be no page any more */
  int pages = -1, pages_s = -1, pages_t = 0;
  for (;; ++walk.slot, walk.j = 0) {
    RowTile x;
    if (!next_row_tile(p, g, few, slots, walk, cur, x)) break;
    const int h = walk.h, j = walk.j;
    const int je = h == walk.h1 && walk.slot == walk.slot1 ? walk.j1 : x.nt; /* its tiles j .. je - 1 are this workgroup's */
    const int n = je - j;
    const int p0 = cur.q.len - cur.q.count;

    /* this lane's row, and the wave's rows' positions: first and last, and what they all see */
    const int wr = 32 * wave, nrows = x.rows - wr;
    const int rr = wr + col < x.rows ? wr + col : x.rows - 1, row = x.r0 + rr;
    const int t = row / g, hh = h * g + row - t * g;
    const int hi = p0 + t, lo = p.window > 0 && hi - p.window + 1 > 0 ? hi - p.window + 1 : 0;
    const int wfirst = x.r0 + (wr < x.rows ? wr : x.rows - 1), wlast = x.r0 + (wr + 31 < x.rows ? wr + 31 : x.rows - 1);
    const int hi_min = p0 + wfirst / g, hi_max = p0 + wlast / g;
    const int lo_min = p.window > 0 && hi_min - p.window + 1 > 0 ? hi_min - p.window + 1 : 0;
    const int lo_max = p.window > 0 && hi_max - p.window + 1 > 0 ? hi_max - p.window + 1 : 0;

    const int last_at = p0 + (x.r0 + x.rows - 1) / g; /* what every row of the tile sees: from wg_lo to wg_hi */
    const int wg_hi = p0 + x.r0 / g;
    const int wg_lo = p.window > 0 && last_at - p.window + 1 > 0 ? last_at - p.window + 1 : 0;

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x16{};
    float m = NINF, l = 0.0f; /* l: this lane's half of the row's sum */

    OddMarks<DB * 16> marks;
    marks.clear();
    /* values: step k takes the 8 positions 32 (k / 2) + 16 half + 8 (k % 2) ..+7 */
    auto va = [&](const unsigned char *vt, int k, int d) {
      return *(const u32x4 *)(vt + ((4 * (k >> 1) + 2 * half + (k & 1)) * HDP + 32 * d + col) * 16);
    };
    const int tile0 = x.t0 + j;
    auto page = [&](int i) { /* of tile i; -1 where it cannot be read */
      const int t = tile0 + i;
      if (cur.s != pages_s || (t & ~63) != pages_t) { /* uniform */
        pages_s = cur.s;
        pages_t = t & ~63;
        const int pos = (pages_t + lane) * TILE;
        pages = pos < cur.q.len ? page_entry(p.b, cur.s, pos) : -1;
      }
      const int page = __builtin_amdgcn_readlane(pages, t & 63);
      return t * TILE < cur.q.len ? page_checked(p.b, page) : -1; /* (tile 0 of a sequence without positions) */
    };
    Stage<FMT, HDP> st;
    int pg = page(0);
    st.fetch(tile_ptr<FMT, HDP>(p.b, pg < 0 ? 0 : pg, h, tile0 * TILE), smem, tid);
    u32x4 qf[KS];
    auto load_queries = [&]() {
      const uint16_t *qr = p.q + (long long)(cur.q.row0 + t) * p.q_ld + hh * p.b.hd;
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        const int d = half * (HDP / 2) + 8 * e;
        qf[e] = d < p.b.hd ? aos_gld16(qr + d) : u32x4{};
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[e][i] ^= flip;
      }
    };
    if (!AGAIN) load_queries();
    st.put(smem, tid);
    for (int i = 0; i < n; ++i) {
      const unsigned char *kt = smem + (i & 1) * STAGE, *vt = kt + TILE * HDP * 2;
      unsigned char *other = smem + ((i + 1) & 1) * STAGE;
      aos_mem_wait(); /* tile i */
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); /* and every wave is past tile i - 1 */
      const bool there = pg >= 0;
      if (i + 1 < n) {
        pg = page(i + 1);
        if (!LATE) st.fetch(tile_ptr<FMT, HDP>(p.b, pg < 0 ? 0 : pg, h, (tile0 + i + 1) * TILE), other, tid);
      }
      const int k0 = (tile0 + i) * TILE;
      if (MARK && (k0 < wg_lo || k0 + TILE - 1 > wg_hi)) { /* uniform over the workgroup */
        u32x4 *vw = (u32x4 *)(kt + TILE * HDP * 2);
        bool odd = false;
#pragma unroll
        for (int c = 0; c < TILE * HDP / 8 / 256; ++c) {
          const u32x4 a = vw[tid + 256 * c];
          odd = odd || odd2(a[0]) || odd2(a[1]) || odd2(a[2]) || odd2(a[3]);
        }
        if (__syncthreads_or(odd ? 1 : 0)) {
          if (there)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll 1
              for (int cls = 0; cls < 3; ++cls) {
                f32x16 c = {};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  u32x4 sf;
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int at = k0 + 32 * (k >> 1) + 16 * half + 8 * (k & 1) + 2 * e;
                    sf[e] = (at >= lo && at <= hi ? 0x3f80u : 0u) | (at + 1 >= lo && at + 1 <= hi ? 0x3f800000u : 0u);
                  }
                  aos_compiler_barrier();
                  c = mfma32(odd_part(va(vt, k, d), cls), sf, c);
                }
#pragma unroll
                for (int v = 0; v < 16; ++v) marks.set(cls, d / 2, c[v] > 0.0f ? 1u << (16 * (d % 2) + v) : 0u);
              }
          __syncthreads();
#pragma unroll
          for (int c = 0; c < TILE * HDP / 8 / 256; ++c) vw[tid + 256 * c] = odd_part(vw[tid + 256 * c], -1);
          __syncthreads();
        }
      }
      if (there && k0 <= hi_max && k0 + TILE > lo_min && nrows > 0) { /* uniform: some row of the wave sees some of it */
        if (AGAIN) load_queries();
        const bool edge = k0 < lo_max || k0 + TILE - 1 > hi_min;
        /* LDS reads run AHEAD matrix instructions before their use (the values' first ones before the softmax): left
         * to itself the compiler reads each fragment right before the instruction that waits for it */
        f32x16 sc[2] = {f32x16{}, f32x16{}};
        {
          const int pos = ((col & 4) << 2) | ((col & 16) >> 1) | ((col & 8) >> 1) | (col & 3);
          const unsigned char *kb = kt + (half * KS * TILE + pos) * 16;
          auto ka = [&](int i) { return *(const u32x4 *)(kb + (i >> 1) * TILE * 16 + 512 * (i & 1)); };
          u32x4 kf[AHEAD];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) kf[i] = ka(i);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 2 * KS; ++i) {
            sc[i & 1] = mfma32(kf[i % AHEAD], qf[i >> 1], sc[i & 1]);
            if (i + AHEAD < 2 * KS) kf[i % AHEAD] = ka(i + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        u32x4 vf[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) vf[i] = va(vt, i / DB, i % DB);
        __builtin_amdgcn_sched_barrier(0);
        if (edge) {
          const int at = k0 + 16 * half;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v)
              if (at + 32 * b + v < lo || at + 32 * b + v > hi) sc[b][v] = NINF;
        }
        float mx = NINF;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[b][v]);
        mx = half_max(mx) * cs;
        if (!edge || (lo < k0 + TILE && hi >= k0)) mx = fmaxf(mx, LEAST);
        if (__ballot(mx > m + SLACK)) {
          const float top = fmaxf(m, mx), alpha = ex2(m - safe_max(top));
          l = l * alpha;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[d][v] = o[d][v] * alpha;
          m = top;
        }
        const float ms = safe_max(m);
        u32x4 pf[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int v = 0; v < 16; v += 2) {
            const float e0 = ex2(fmaf(sc[b][v], cs, -ms)), e1 = ex2(fmaf(sc[b][v + 1], cs, -ms));
            l = l + e0;
            l = l + e1;
            pf[2 * b + v / 8][v / 2 % 4] = pack_bf16(e0, e1);
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i) {
          o[i % DB] = mfma32(vf[i % AHEAD], pf[i / DB], o[i % DB]);
          if (i + AHEAD < 4 * DB) vf[i % AHEAD] = va(vt, (i + AHEAD) / DB, (i + AHEAD) % DB);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (LATE && i + 1 < n) st.fetch(tile_ptr<FMT, HDP>(p.b, pg < 0 ? 0 : pg, h, (tile0 + i + 1) * TILE), other, tid);
      if (i + 1 < n) st.put(other, tid);
    }
    if (MARK)
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = marks.apply(16 * d + v, o[d][v]);
    l = half_sum(l);

    uint16_t *orow = p.out + (long long)(cur.q.row0 + t) * p.out_ld + hh * p.b.hd;
    auto put = [&](int d, int q, f32x4 y, float inv) { /* dimensions 32 d + 8 q + 4 half ..+3 */
      const int at = 32 * d + 8 * q + 4 * half;
      if (col < nrows && at < p.b.hd)
        *(u32x2 *)(orow + at) = u32x2{pack_bf16(y[0] * inv, y[1] * inv), pack_bf16(y[2] * inv, y[3] * inv)};
    };
    if (n == x.nt) {
      const float inv = inverse(l, m);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          put(d, q, f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]}, inv);
    } else {
      constexpr int PF = tile_part_floats<HDP>();
      const Cuts cuts = cuts_of(w, share, j, je, x.nt);
      const int wf = cuts.wf, wl = cuts.wl;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)p.part, (short)0, 0x7fffffff, 0x00020000);
      if (nrows > 0) {
        const int at = (2 * w + (j > 0 ? 0 : 1)) * PF;
        if (half == 0) {
          aos_publish(p.part + at + 64 * wave + col, m);
          aos_publish(p.part + at + 64 * wave + 32 + col, l);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 y = {o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rs,
                                                   (at + 256 + (((wave * DB + d) * 4 + q) * 64 + lane) * 4) * 4, 0, SC1);
          }
      }
      aos_mem_wait();
      __syncthreads();
      if (tid == 0) {
        const uint32_t old = aos_arrive(p.counters + wf);
        if (old == (uint32_t)(wl - wf + 1)) aos_reset(p.counters + wf);
        sh.joins = old == (uint32_t)(wl - wf + 1) ? 1 : 0;
      }
      __syncthreads();
      if (sh.joins && nrows > 0) {
        const int np = wl - wf + 2;
        auto part = [&](int k) { return (k == 0 ? 2 * wf - 1 : 2 * (wf + k - 1)) * PF; };
        float top = NINF;
        for (int k = 0; k < np; ++k) top = fmaxf(top, aos_collect(p.part + part(k) + 64 * wave + col));
        const float ms = safe_max(top);
        float all = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = f32x16{};
        for (int k = 0; k < np; ++k) {
          const Weight<MARK> f(aos_collect(p.part + part(k) + 64 * wave + col), ms);
          all = all + f(aos_collect(p.part + part(k) + 64 * wave + 32 + col));
#pragma unroll
          for (int d0 = 0; d0 < DB; d0 += FLY) {
            f32x4 y[FLY][4]; /* (all in flight together) */
#pragma unroll
            for (int d = 0; d < FLY; ++d)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                y[d][q] = __builtin_bit_cast(
                    f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                               rs, (part(k) + 256 + (((wave * DB + d0 + d) * 4 + q) * 64 + lane) * 4) * 4, 0, SC1));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < FLY; ++d)
#pragma unroll
              for (int v = 0; v < 16; ++v) o[d0 + d][v] = o[d0 + d][v] + f(y[d][v >> 2][v & 3]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        const float inv = inverse(all, top);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            put(d, q, f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]}, inv);
      }
    }
    __syncthreads(); /* the stages and `joins` are free again */
  }
}

/* two bodies, as above */
template <int FMT, int HDP>
__global__ void __launch_bounds__(256, tiles_per_cu(HDP)) aos_kv_tiles_kernel(aos_kv_attn_params p, int few, int slots,
                                                                             int min_share) {
  __shared__ TilesShared sh;
  if (*p.b.nonfinite)
    tiles_body<FMT, HDP, true>(p, few, slots, min_share, sh);
  else
    tiles_body<FMT, HDP, false>(p, few, slots, min_share, sh);
}

/* Least weight of a workgroup of the first kernel: a whole row tile where the batch's longest sequence has few position
 * tiles, else one or two tiles a wave (28 heads of 128 over 4, one token: 512 positions 9.0 us whole and 11.5 cut, 1280
 * positions 12.3 and 12.6; 2000 positions 14.3 us in shares of 13 and 12.9 in shares of 6). */
constexpr int rows_share(int nb, int tiles) { return tiles <= 24 / nb ? tiles + ROWS_SETUP : 6; }
constexpr int TILES_SHARE = 6; /* (prompt of 300, 28 heads of 128: 24 us, 29 with 8, 31 with 12) */

/* Workgroups of the first kernel: as many as keep memory busy, which is one a CU where a tile is 16 KB or more (32
 * streams of up to 8191, 8 bits: 69 us with 256, 74 with 512; 64 of up to 16001, 16 bits: 230 and 236) and two where it
 * is less (24 of 32768, 4 bits: 147 and 122). */
template <int FMT, int HDP>
constexpr int rows_wgs() {
  return tile_bytes<FMT, HDP>() >= 16384 ? 256 : 512;
}

template <int FMT, int HDP, int NB>
int launch_rows(const aos_kv_attn_params *p, const aos_launch_ctx *ctx, int few) { /* sequences of up to `few` rows */
  const int tiles = (p->b.max_len + TILE - 1) / TILE, share = rows_share(NB, tiles);
  /* no more workgroups than shares */
  const long long rts = (long long)p->b.n_tokens * (p->nh / p->b.nkv) / (16 * NB) + p->b.n_seqs;
  const long long weights = rts * p->b.nkv * (tiles + 1 + ROWS_SETUP);
  const long long wgs = (weights + share - 1) / share, most = rows_wgs<FMT, HDP>();
  AOS_LAUNCH(ctx, (aos_kv_rows_kernel<FMT, HDP, NB>), dim3(wgs < most ? (int)wgs : (int)most), dim3(256), 0, *p, few,
             share);
  return (int)hipGetLastError();
}

/* Up to so many (16-row block, key/value head, position tile) of a batch, and bytes of cache read for them, every sequence
 * goes to the first kernel in blocks of 16 rows, each reading the cache for itself: small batches gain more from many
 * workgroups than they lose by reading again. Rows of 16, and in blocks that share a tile or in the second kernel: 12
 * streams x 5 tokens of 7 rows over 2000, heads of 64: 14.3 us and 17.4; 8 x 8 x 7 over 1000, heads of 128: 17 and 28; a
 * prompt of 300 x 7: 22 and 24; 4 x 100 x 3 over 600, 4 bits: 25 and 33. Beyond: a prompt of 420 x 7: 29 and 24; 8 x 4 x 7
 * over 8000: 48 and 34; 32 x 8 x 7 over 8000, heads of 64: 81 and 40. */
constexpr long long SMALL_UNITS = 12288, SMALL_BYTES = 160000000;

template <int FMT, int HDP>
int attend(const aos_kv_attn_params *p, const aos_launch_ctx *ctx) {
  const long long g = p->nh / p->b.nkv, rows = p->b.max_new * g;
  const long long slots = (long long)p->b.n_tokens * g / TR + p->b.n_seqs;
  if (!aos_kv_attention_fits(&p->b, p->nh)) return (int)hipErrorInvalidValue;
  const long long units = ((long long)p->b.n_tokens * g / 16 + p->b.n_seqs) * p->b.nkv * ((p->b.max_len + TILE - 1) / TILE);
  if (rows <= 16 || (!p->no_small && units <= SMALL_UNITS && units * tile_bytes<FMT, HDP>() <= SMALL_BYTES))
    return launch_rows<FMT, HDP, 1>(p, ctx, 0x7fffffff);
  if constexpr (HDP <= 128) /* (the registers of wider heads do not hold two blocks) */
    if (rows <= 32) return launch_rows<FMT, HDP, 2>(p, ctx, 32);
  /* among several sequences, those of up to 16 rows (decoding streams among prompts) are the first kernel's. (Both
   * bodies in one launch, half of the workgroups streaming the few rows' cache while the others multiply, spills the
   * tile loop's registers: chunk of 512 over 15872 at 8 bits 319 us for 200, mixed batch of 32 179 for 127.) */
  const int few = p->b.n_seqs == 1 ? 0 : 16;
  AOS_LAUNCH(ctx, (aos_kv_tiles_kernel<FMT, HDP>), dim3(256 * tiles_per_cu(HDP)), dim3(256), 8 * TILE * HDP, *p, few,
             (int)slots, TILES_SHARE);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !few) return (int)e;
  return launch_rows<FMT, HDP, 1>(p, ctx, few);
}

/* what a launch needs of the device beforehand: the second kernel's LDS size allowed */
template <int FMT, int HDP>
int prepare() {
  return (int)hipFuncSetAttribute((const void *)aos_kv_tiles_kernel<FMT, HDP>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                  8 * TILE * HDP);
}

}  // namespace

/* rows of a sequence and weights of a batch are counted in 32 bits */
int aos_kv_attention_fits(const aos_kv_batch *b, int nh) {
  const long long g = nh / b->nkv, slots = (long long)b->n_tokens * g / TR + b->n_seqs;
  const long long per = b->max_len / TILE + 1 + (SETUP > ROWS_SETUP ? SETUP : ROWS_SETUP);
  return b->max_new * g <= (1ll << 30) && slots <= (1ll << 30) && slots * per <= 0x7f000000ll / b->nkv;
}

/* pieces, two for each workgroup of the larger launch */
size_t aos_kv_part_floats(int hdp) {
  const size_t rows = 2 * 512 * 2 * (size_t)(32 + 16 * hdp);
  const size_t tiles = 2 * 256 * (size_t)(hdp == 256 ? 1 : 2) * (256 + TR * hdp);
  return rows > tiles ? rows : tiles;
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

extern "C" int aos_launch_kv_attention(const aos_kv_attn_params *p, const aos_launch_ctx *ctx) {
  return KV_DISPATCH(attend, p->b.format, p->b.hdp, p, ctx);
}

extern "C" int aos_kv_attention_prepare(int format, int hdp) { return KV_DISPATCH(prepare, format, hdp); }

/* Diagnostic, for tests without a device: the pieces of row tiles that the G workgroups of the second kernel take of a
 * batch (starts and lens: host arrays), walked as it walks them: rows of {workgroup, head, sequence, first row, rows, first
 * position tile, position tiles, j, je, wf, wl} (the last two -1 where the row tile is whole). Returns their number (at
 * most cap are written), or -1 where the kernel takes the batch for one that does not fit. */
extern "C" int aoship_internal_kv_tile_pieces(int nh, int nkv, int window, int n_seqs, int n_tokens, int max_new, int max_len,
                                              const int32_t *starts, const int32_t *lens, int few, int G, int min_share,
                                              int (*out)[11], int cap) {
  uint32_t faults = 0;
  aos_kv_attn_params p = {};
  p.b.nkv = nkv;
  p.b.starts = starts;
  p.b.lens = lens;
  p.b.n_seqs = n_seqs;
  p.b.n_tokens = n_tokens;
  p.b.max_new = max_new;
  p.b.max_len = max_len;
  p.b.faults = &faults;
  p.nh = nh;
  p.window = window;
  const int g = nh / nkv, slots = (int)((long long)n_tokens * g / TR) + n_seqs, per = (slots + 255) / 256;
  if (starts_fall(p.b, 0, 1)) return -1;
  Cursor own[256] = {};
  int before[257] = {};
  for (int t = 0; t < 256; ++t) {
    const int first = t * per, end = first + per < slots ? first + per : slots;
    int sum = 0;
    if (first < end) {
      seek(p.b, g, first, own[t]);
      sum = run_weight(p, g, few, own[t], first, end);
    }
    before[t + 1] = before[t] + sum;
  }
  const int N = before[256], total = N * nkv;
  int share = (total + G - 1) / G, n = 0;
  if (share < min_share) share = min_share;
  for (int w = 0; w < G && w * share < total; ++w) {
    Walk walk = {w * share / N, 0, 0, nkv, 0, 0};
    Cursor cur = {};
    for (int i = 0; i < 2 && (w + i) * share < total; ++i) {
      const int hh = (w + i) * share / N, v = (w + i) * share - hh * N;
      int t = 0;
      while (v >= before[t + 1]) ++t;
      const int first = t * per, end = first + per < slots ? first + per : slots;
      Cursor c = own[t];
      run_border(p, g, few, c, first, end, v - before[t], i ? walk.slot1 : walk.slot, i ? walk.j1 : walk.j);
      if (i)
        walk.h1 = hh;
      else
        cur = c;
    }
    RowTile x;
    for (; next_row_tile(p, g, few, slots, walk, cur, x); ++walk.slot, walk.j = 0) {
      const int je = walk.h == walk.h1 && walk.slot == walk.slot1 ? walk.j1 : x.nt;
      Cuts cuts = {-1, -1};
      if (je - walk.j != x.nt) cuts = cuts_of(w, share, walk.j, je, x.nt);
      const int row[11] = {w, walk.h, cur.s, x.r0, x.rows, x.t0, x.nt, walk.j, je, cuts.wf, cuts.wl};
      for (int i = 0; n < cap && i < 11; ++i) out[n][i] = row[i];
      ++n;
    }
  }
  return n;
}
