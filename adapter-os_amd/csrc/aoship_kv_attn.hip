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
 */
#include "aoship_internal.h"
#include "aoship_kv.h"
#include <hip/hip_ext.h>

using namespace kv;

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int SC1 = 16; /* buffer cache policy: device-coherent (sc1) */
constexpr float LOG2E = 1.44269504f;
constexpr float NINF = -__builtin_inff();

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
/* scale byte j of a word as its power of two; 255 gives infinity, which times its zero codes is NaN */
__device__ __forceinline__ float byte_scale(uint32_t w, int j) {
  return __builtin_bit_cast(float, (j == 3 ? w >> 1 : j == 2 ? w << 7 : j == 1 ? w << 15 : w << 23) & 0x7f800000u);
}

/* whether a word of two bfloat16 holds an infinity or a NaN */
__device__ __forceinline__ bool odd2(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
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
__device__ __forceinline__ float odd_value(int cls) {
  return cls == 0 ? __builtin_inff() : cls == 1 ? -__builtin_inff() : __builtin_nanf("");
}

/* ---- sharing the work ------------------------------------------------------------------------ */

/* What of a sequence the attention walks: rows (token, head) in row tiles of R, each over nt tiles from tile t0 on.
 * A sequence with rows but no positions has one tile, in which nothing is visible. */
struct Work {
  Seq q;
  int rows, rts, t0, nt;
};
template <int R>
__device__ __forceinline__ Work work_of(const aos_kv_attn_params &p, const Seq &q) {
  Work w;
  w.q = q;
  w.rows = q.count * (p.nh / p.b.nkv);
  w.rts = (w.rows + R - 1) / R;
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

/* ---- few rows: 16 to a wave, the cache streamed through registers ------------------------------ */

/* A workgroup takes an even share of all (sequence, key/value head, row tile, tile of positions); its four waves
 * take the tiles of a row tile in turn. Scores S^T[position][row] = K . Q^T, output O^T[dimension][row] = V^T . P^T
 * by v_mfma_f32_16x16x32_bf16: the accumulator of block b (of four 16-position blocks) holds rows 4 quad + i, and
 * the row 4 j + i of block b is made position 16 j + 4 b + i, so a lane's scores are the 16 consecutive positions
 * 16 quad ..+15, which is what the value units hold: the probabilities never cross lanes. Probabilities are rounded
 * to bfloat16 for the second product (half a unit of 8 bits each, like the output's own rounding); sums are float32.
 * In the quantised formats the value scales multiply the probabilities (exactly: powers of two). */
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

/* waves per SIMD that the registers of a tile in flight and the accumulators leave room for */
constexpr int rows_waves(int fmt, int hdp) { return hdp == 256 || (fmt == AOS_KV_BF16 && hdp == 128) ? 1 : 2; }

template <int FMT, int HDP, int NB>
__global__ void __launch_bounds__(256, rows_waves(FMT, HDP)) aos_kv_rows_kernel(aos_kv_attn_params p, int min_share) {
  constexpr int R = 16 * NB, DB = HDP / 16, KS = HDP / 32, W8 = bits<FMT>() / 4; /* W8: words of 8 codes */
  __shared__ float red[2][NB * DB * 4][64];
  __shared__ float mls[4][2][NB][64];
  __shared__ uint32_t last_word;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int G = gridDim.x, w = blockIdx.x;
  const int g = p.nh / p.b.nkv;

  /* all units, this workgroup's share [u0, u1) of them, and the sequence that u0 falls in */
  auto units = [&](int s) {
    if (s >= p.b.n_seqs) return 0;
    const Work x = work_of<R>(p, seq_at(p.b, s));
    return p.b.nkv * x.rts * x.nt;
  };
  int total = 0;
  for (int s0 = 0; s0 < p.b.n_seqs; s0 += 64)
    total += __builtin_amdgcn_readlane(wave_scan(units(s0 + lane), lane), 63);
  int share = (total + G - 1) / G;
  if (share < min_share) share = min_share;
  int u = w * share;
  if (u >= total) return;
  const int u1 = u + share < total ? u + share : total;
  int s = 0, base = 0; /* base: units before sequence s */
  for (int s0 = 0, before = 0; s0 < p.b.n_seqs; s0 += 64) {
    const int mine = units(s0 + lane), upto = before + wave_scan(mine, lane);
    const uint64_t past = __ballot(upto > u);
    if (past) {
      const int l = __builtin_ctzll(past);
      s = s0 + l;
      base = __builtin_amdgcn_readlane(upto - mine, l);
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }

  const float cs = p.scale * LOG2E;
  while (u < u1) {
    Work x = work_of<R>(p, seq_at(p.b, s));
    while (x.rts == 0 && s + 1 < p.b.n_seqs) x = work_of<R>(p, seq_at(p.b, ++s));
    if (x.rts == 0) return; /* (never: u < total, so a later sequence has units) */
    const int seg = (u - base) / x.nt, j = u - base - seg * x.nt; /* which (head, row tile), and its tile */
    const int h = seg / x.rts, rt = seg - h * x.rts;
    const int n = x.nt - j < u1 - u ? x.nt - j : u1 - u;
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
      }
    }
    const int t_first = r0 / g, t_last = (r0 + nrows - 1) / g;
    const int hi_min = p0 + t_first;
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

    const int mine = (n - wave + 3) / 4; /* tiles of this wave: j + wave, j + wave + 4, ... */
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
        tl.load_k(t, lane);
        tl.load_v(t, lane);
      }
      for (int i = 0; i < cnt; ++i) {
        const int tb = (x.t0 + j + wave + 4 * (i0 + i)) * TILE;
        const bool there = __builtin_amdgcn_readlane(pg, i) >= 0;
        const unsigned char *next = ptr(i + 1 < cnt ? i + 1 : i);
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
        if (i + 1 < cnt) tl.load_k(next, lane);

        const bool edge = !there || tb < lo_max || tb + TILE - 1 > hi_min; /* uniform */
        uint32_t seen[NB]; /* bit 4 b + i: the row sees position 16 quad + 4 b + i of the tile */
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          seen[b] = 0xffffu;
          if (edge) {
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
          float mx = m[b];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float y = sc[b][k >> 2][k & 3] * cs;
            if (edge && !(seen[b] >> k & 1)) y = NINF;
            sc[b][k >> 2][k & 3] = y;
            mx = fmaxf(mx, y);
          }
          mx = quad_max(mx);
          if (__ballot(mx > m[b])) {
            const float alpha = ex2(m[b] - safe_max(mx));
            l[b] = l[b] * alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int k = 0; k < 4; ++k) o[b][d][k] = o[b][d][k] * alpha;
            m[b] = mx;
          }
          const float ms = safe_max(m[b]);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float e = ex2(sc[b][k >> 2][k & 3] - ms);
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
        bool odd = false;
        if constexpr (FMT == AOS_KV_BF16) {
          if (edge) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int k = 0; k < Tile<FMT, HDP>::VW; ++k) odd = odd || odd2(tl.v[d][k]);
            odd = __ballot(odd) != 0;
          }
        }
        if (!odd) {
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
                      if (edge && !(seen[b] >> (8 * t + k) & 1)) y[k] = 0.0f;
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
        } else if constexpr (FMT == AOS_KV_BF16) {
          /* An infinity or a NaN among the values of a tile that some row sees only in part: its product with a
           * probability of zero would reach rows that do not see it. The finite values go through the product; of
           * the others, each row counts those that it sees. */
          u32x4 sf[NB][2];
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                sf[b][t][k] = (seen[b] >> (8 * t + 2 * k) & 1 ? 0x3f80u : 0u) |
                              (seen[b] >> (8 * t + 2 * k + 1) & 1 ? 0x3f800000u : 0u);
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll 1
            for (int cls = -1; cls < 3; ++cls) {
              f32x4 c[NB];
#pragma unroll
              for (int b = 0; b < NB; ++b) c[b] = cls < 0 ? o[b][d] : f32x4{};
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                u32x4 a;
#pragma unroll
                for (int k = 0; k < 4; ++k) a[k] = odd_part(tl.v[d][4 * t + k], cls);
#pragma unroll
                for (int b = 0; b < NB; ++b) c[b] = mfma16(a, cls < 0 ? pf[b][t] : sf[b][t], c[b]);
              }
#pragma unroll
              for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  o[b][d][k] = cls < 0 ? c[b][k] : c[b][k] > 0.0f ? o[b][d][k] + odd_value(cls) : o[b][d][k];
            }
        }
        if (i + 1 < cnt) tl.load_v(next, lane);
      }
    }

    /* the waves' pieces: one maximum, then their sums two by two */
    const bool many = n > 1;
#pragma unroll
    for (int b = 0; b < NB; ++b) l[b] = quad_sum(l[b]);
    if (many) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        mls[wave][0][b][lane] = m[b];
        mls[wave][1][b][lane] = l[b];
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float top = NINF;
#pragma unroll
        for (int v = 0; v < 4; ++v) top = fmaxf(top, mls[v][0][b][lane]);
        const float ms = safe_max(top);
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; ++v) sum = sum + mls[v][1][b][lane] * ex2(mls[v][0][b][lane] - ms);
        const float f = ex2(m[b] - ms);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[b][d][k] = o[b][d][k] * f;
        m[b] = top;
        l[b] = sum;
      }
      for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int k = 0; k < 4; ++k) red[wave - half][(b * DB + d) * 4 + k][lane] = o[b][d][k];
        __syncthreads();
        if (wave < half)
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int k = 0; k < 4; ++k) o[b][d][k] = o[b][d][k] + red[wave][(b * DB + d) * 4 + k][lane];
        __syncthreads();
      }
    }

    auto put = [&](int b, int d, f32x4 y, float sum) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum; /* a row that sees nothing: zeros */
      const int at = 16 * d + 4 * quad;
      if (16 * b + col < nrows && at < p.b.hd)
        *(u32x2 *)(p.out + orow[b] + at) = u32x2{pack_bf16(y[0] * inv, y[1] * inv), pack_bf16(y[2] * inv, y[3] * inv)};
    };
    if (n == x.nt) {
      if (wave == 0)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int d = 0; d < DB; ++d) put(b, d, o[b][d], l[b]);
    } else {
      /* a cut row tile: its pieces lie in the slots of workgroups w0 .. w1 (2 w: the piece that w begins with, 2 w + 1:
       * the one that it ends with), and the last to arrive joins them in that order */
      constexpr int PF = part_floats<HDP, NB>();
      const int g0 = u - j, w0 = g0 / share, w1 = (g0 + x.nt - 1) / share;
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
          const uint32_t old = aos_arrive(p.counters + w0);
          if (old == (uint32_t)(w1 - w0)) aos_reset(p.counters + w0);
          last_word = old == (uint32_t)(w1 - w0) ? 1u : 0u;
        }
      }
      __syncthreads();
      const bool last = last_word != 0;
      if (last) {
        const int np = w1 - w0 + 1;
        auto slot = [&](int k) { return (k == 0 ? 2 * w0 + 1 : 2 * (w0 + k)) * PF; };
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float top = NINF;
          for (int k = quad; k < np; k += 4) top = fmaxf(top, aos_collect(p.part + slot(k) + 32 * b + col));
          top = quad_max(top);
          const float ms = safe_max(top);
          float sum = 0.0f;
          for (int k = quad; k < np; k += 4)
            sum = sum + aos_collect(p.part + slot(k) + 32 * b + 16 + col) * ex2(aos_collect(p.part + slot(k) + 32 * b + col) - ms);
          sum = quad_sum(sum);
          if (16 * b + col < nrows)
            for (int d = wave; d < DB; d += 4) {
              f32x4 acc = {};
#pragma unroll 4
              for (int k = 0; k < np; ++k) {
                const float f = ex2(aos_collect(p.part + slot(k) + 32 * b + col) - ms);
                const f32x4 y = __builtin_bit_cast(
                    f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (slot(k) + 32 * NB + ((b * DB + d) * 64 + lane) * 4) * 4, 0, SC1));
                acc = acc + y * f;
              }
              put(b, d, acc, sum);
            }
        }
      }
      __syncthreads(); /* last_word and the reduction's memory are free again */
    }
    u += n;
    if (u - base >= p.b.nkv * x.rts * x.nt) {
      base += p.b.nkv * x.rts * x.nt;
      ++s;
    }
  }
}

constexpr int ROWS_WGS = 512;

template <int FMT, int HDP>
int rows(const aos_kv_attn_params *p, const aos_launch_ctx *ctx) {
  AOS_LAUNCH(ctx, (aos_kv_rows_kernel<FMT, HDP, 1>), dim3(ROWS_WGS), dim3(256), 0, *p, 8);
  return (int)hipGetLastError();
}

}  // namespace

size_t aos_kv_part_floats(int hdp) { return (size_t)2 * AOS_KV_MAX_WGS * (32 + 16 * hdp); }

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
  return KV_DISPATCH(rows, p->b.format, p->b.hdp, p, ctx);
}
