/*
 * aoship_kv.hip — writing new rows into the paged key/value cache and reading rows back.
 *
 *   append  y = x + bias; the two halves of a query or key row are rotated, (a, b) -> (a c - b s, a s + b c), with
 *           its position's cosines and sines (or those of the positions that the caller
 *           gives); float32, each operation rounded on its own; the row is rounded to
 *           bfloat16. Queries go out as rows, keys and values into their sequence's pages: as they are, or per 32
 *           dimensions as codes of the smallest power-of-two scale 2^e whose code range holds the block,
 *               max |y| <= 448 2^e (e4m3 codes, e >= -117)      max |y| <= 6 2^e (e2m1 codes, e >= -125),
 *           codes rounded to nearest even (the bounds on e keep every value that a code can stand for a normal
 *           bfloat16; a power of two makes scaling and reading back exact). A block with an infinity or a NaN has no
 *           scale: its byte is 255 and it reads back as NaN.
 *   read    the values, as bfloat16 rows.
 *
 * Both are bound by memory: a workgroup takes one block of 16 positions (the values' unit, so that a prompt writes
 * whole 16-byte units) and a few heads.
 */
#include "aoship_internal.h"
#include "aoship_kv.h"
#include <hip/hip_ext.h>

using namespace kv;

namespace {

typedef short s16x2 __attribute__((ext_vector_type(2)));

constexpr int Q_HEADS = 8; /* query heads of a workgroup */

/* byte of the scale of a block whose largest magnitude has the bits `top` (of a float32 holding a bfloat16) */
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  constexpr int EMAX = FMT == AOS_KV_MXFP8 ? 8 : 2, LOW = FMT == AOS_KV_MXFP8 ? -117 : -125;
  constexpr uint32_t FULL = FMT == AOS_KV_MXFP8 ? 0x600000u : 0x400000u; /* 448 = 1.75 2^8, 6 = 1.5 2^2 */
  if (top >= 0x7f800000u) return 255u;
  const int e = (int)(top >> 23) - 127 - EMAX + ((top & 0x7fffffu) > FULL ? 1 : 0);
  return (uint32_t)((e < LOW ? LOW : e) + 127);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

/* two values (bfloat16 in the halves of a word) as codes, of one scale; byte 255: zeros */
template <int FMT>
__device__ __forceinline__ uint32_t encode2(uint32_t pair, uint32_t byte) {
  if (byte == 255u) return 0u;
  const bf16x2 x = __builtin_bit_cast(bf16x2, pair);
  if constexpr (FMT == AOS_KV_MXFP8)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(s16x2{0, 0}, x, scale_of(byte), false)) & 0xffffu;
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, x, scale_of(byte), 0) & 0xffu;
}

__device__ __forceinline__ f32x4 ld4(const float *p) { return *(const f32x4 *)p; }

/* four rotated pairs: a' = a c - b s, b' = a s + b c */
struct Quad {
  float a[4], b[4];
};
__device__ __forceinline__ Quad rotate4(uint2 xa, uint2 xb, bool bias, f32x4 ba, f32x4 bb, bool rot, f32x4 cs,
                                        f32x4 sn) {
  Quad r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = aos_bf16_to_f32((uint16_t)((i < 2 ? xa.x : xa.y) >> (16 * (i & 1))));
    float b = aos_bf16_to_f32((uint16_t)((i < 2 ? xb.x : xb.y) >> (16 * (i & 1))));
    if (bias) {
      a = a + ba[i];
      b = b + bb[i];
    }
    r.a[i] = rot ? a * cs[i] - b * sn[i] : a;
    r.b[i] = rot ? a * sn[i] + b * cs[i] : b;
  }
  return r;
}
__device__ __forceinline__ uint2 pack4(const float *x) {
  uint2 r;
  r.x = (uint32_t)aos_f32_to_bf16(x[0]) | ((uint32_t)aos_f32_to_bf16(x[1]) << 16);
  r.y = (uint32_t)aos_f32_to_bf16(x[2]) | ((uint32_t)aos_f32_to_bf16(x[3]) << 16);
  return r;
}

/* largest magnitude (as bits) of the 32 bfloat16 at p */
__device__ __forceinline__ uint32_t block_top(const uint16_t *p) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const u32x4 w = *(const u32x4 *)(p + 8 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = (w[i] << 16) & 0x7fffffffu, hi = w[i] & 0x7fff0000u;
      m = m > lo ? m : lo;
      m = m > hi ? m : hi;
    }
  }
  return m;
}

/* The cosines and sines of the pairs d .. d + 3 of a row: those of its position in the sequence, or (AT) of the positions
 * that the caller gives it, one an axis, each pair with its axis's. A quad of pairs mostly has one axis: one load each. */
template <bool AT>
__device__ __forceinline__ void turn_of(const aos_kv_append_params &p, int pos, long long row, int d, f32x4 &cs, f32x4 &sn) {
  const int half = p.b.hd / 2;
  if constexpr (!AT) {
    const long long at = (long long)pos * half + d;
    cs = ld4(p.cosines + at);
    sn = ld4(p.sines + at);
  } else {
    const uint32_t axes = p.axes ? p.axes[d >> 2] : 0u; /* two bits a pair */
    auto place = [&](uint32_t axis) {
      int at = p.at[(long long)axis * p.at_ld + row];
      if ((unsigned)at >= (unsigned)p.rope_positions) {
        note(p.b.faults, AOS_KV_FAULT_POSITION);
        at = 0;
      }
      return (long long)at * half + d;
    };
    if (axes == (axes & 3u) * 0x55u) {
      const long long at = place(axes & 3u);
      cs = ld4(p.cosines + at);
      sn = ld4(p.sines + at);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long at = place(axes >> (2 * i) & 3u) + i;
        cs[i] = p.cosines[at];
        sn[i] = p.sines[at];
      }
    }
  }
}

/* Grid (blocks of 16 positions, groups of query heads then key/value heads). Bound by memory, by latency where there are
 * few rows: 8191 tokens of 40 query and 8 key/value heads of 128 at 16 bits 47 us (235 MB, 5.0 TB/s), 5 prompts of up to
 * 1531 tokens, 28/4 heads, at 4 bits 21 us, one token 3.9 us. With positions given (AT; on three axes in turn, so that each pair
 * is looked up by itself) two prompts of up to 6111 tokens, 24/8 heads, at 8 bits 52 us (171 MB, 3.3 TB/s; 40 where the caches
 * still hold the rows), 48 tokens of 28/4 heads 4.7. */
template <int FMT, int HDP, bool AT>
__global__ void __launch_bounds__(256) aos_kv_append_kernel(aos_kv_append_params p, int qgroups) {
  constexpr int LD = HDP + 8; /* LDS row: 16 bytes of padding keep the column reads of a value unit apart */
  __shared__ __attribute__((aligned(16))) uint16_t ks[16 * LD], vs[16 * LD];
  __shared__ uint32_t vsc[HDP / 32][16];
  const int tid = threadIdx.x, lane = tid & 63;
  Block o;
  if (!block_at(p.b, (int)blockIdx.x, lane, o)) return;
  const int hd = p.b.hd, half = hd / 2, chunks = half / 4;
  const int n = o.hi - o.lo;
  const bool rot = p.cosines != nullptr;

  if ((int)blockIdx.y < qgroups) {
    /* a thread keeps its four cosines and sines for all heads of the group */
    const int h0 = blockIdx.y * Q_HEADS, h1 = h0 + Q_HEADS < p.nh ? h0 + Q_HEADS : p.nh;
    const int per = n * chunks, par = 256 / per > 1 ? 256 / per : 1;
    for (int c0 = 0; c0 < per; c0 += 256) {
      const int c = c0 + (par > 1 ? tid % per : tid), sub = par > 1 ? tid / per : 0;
      if (c >= per || sub >= par) continue;
      const int t = c / chunks, d = 4 * (c % chunks);
      f32x4 cs = {}, sn = {};
      if (rot) turn_of<AT>(p, o.pos + o.lo + t, o.row + t, d, cs, sn);
      const uint16_t *x = p.q + (long long)(o.row + t) * p.q_ld + d;
      uint16_t *y = p.q_out + (long long)(o.row + t) * p.out_ld + d;
      for (int h = h0 + sub; h < h1; h += par) {
        const uint2 xa = *(const uint2 *)(x + h * hd), xb = *(const uint2 *)(x + h * hd + half);
        f32x4 ba = {}, bb = {};
        if (p.qb) {
          ba = ld4(p.qb + h * hd + d);
          bb = ld4(p.qb + h * hd + d + half);
        }
        const Quad r = rotate4(xa, xb, p.qb != nullptr, ba, bb, rot, cs, sn);
        *(uint2 *)(y + h * hd) = pack4(r.a);
        *(uint2 *)(y + h * hd + half) = pack4(r.b);
      }
    }
    return;
  }

  const int h = blockIdx.y - qgroups;
  const int page = page_of(p.b, o.seq, o.pos);
  if (page < 0) return; /* uniform */
  unsigned char *tile = tile_ptr<FMT, HDP>(p.b, page, h, o.pos);
  const int tp = o.pos & 48; /* the block's first position in its tile */

  /* rows of the block into LDS: zeros where no new row is, and past head_dim */
  for (int c = tid; c < 16 * (HDP / 8); c += 256) {
    const int t = c / (HDP / 8), d = 8 * (c % (HDP / 8));
    u32x4 x = {};
    if (t >= o.lo && t < o.hi && d < hd) {
      const long long row = o.row + t - o.lo;
      x = *(const u32x4 *)(p.v + row * p.v_ld + h * hd + d);
      if (p.vb) {
        const f32x4 b0 = ld4(p.vb + h * hd + d), b1 = ld4(p.vb + h * hd + d + 4);
        const float bias[8] = {b0[0], b0[1], b0[2], b0[3], b1[0], b1[1], b1[2], b1[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = (uint32_t)aos_f32_to_bf16(aos_bf16_to_f32((uint16_t)x[i]) + bias[2 * i]) |
                 ((uint32_t)aos_f32_to_bf16(aos_bf16_to_f32((uint16_t)(x[i] >> 16)) + bias[2 * i + 1]) << 16);
      }
    }
    if (FMT == AOS_KV_BF16 && (odd2(x[0]) || odd2(x[1]) || odd2(x[2]) || odd2(x[3]))) *p.b.nonfinite = 1u;
    *(u32x4 *)(vs + t * LD + d) = x;
    if (d >= hd || t < o.lo || t >= o.hi) *(u32x4 *)(ks + t * LD + d) = u32x4{};
  }
  for (int c = tid; c < n * chunks; c += 256) {
    const int t = c / chunks, d = 4 * (c % chunks);
    const uint16_t *x = p.k + (long long)(o.row + t) * p.k_ld + h * hd + d;
    f32x4 cs = {}, sn = {}, ba = {}, bb = {};
    if (rot) turn_of<AT>(p, o.pos + o.lo + t, o.row + t, d, cs, sn);
    if (p.kb) {
      ba = ld4(p.kb + h * hd + d);
      bb = ld4(p.kb + h * hd + d + half);
    }
    const Quad r = rotate4(*(const uint2 *)x, *(const uint2 *)(x + half), p.kb != nullptr, ba, bb, rot, cs, sn);
    *(uint2 *)(ks + (o.lo + t) * LD + d) = pack4(r.a);
    *(uint2 *)(ks + (o.lo + t) * LD + d + half) = pack4(r.b);
  }
  __syncthreads();

  if constexpr (FMT == AOS_KV_BF16) {
    for (int c = tid; c < 16 * (HDP / 8); c += 256) {
      const int t = c & 15, u = c >> 4;
      if (t >= o.lo && t < o.hi) *(u32x4 *)(tile + (u * TILE + tp + t) * 16) = *(const u32x4 *)(ks + t * LD + 8 * u);
    }
  } else {
    /* keys: a thread per position and block of 32 dimensions; value scales: the threads after them */
    for (int c = tid; c < 2 * 16 * (HDP / 32); c += 256) {
      const int t = c & 15, blk = (c >> 4) % (HDP / 32);
      const bool is_v = c >= 16 * (HDP / 32), fresh = t >= o.lo && t < o.hi;
      const uint16_t *x = (is_v ? vs : ks) + t * LD + 32 * blk;
      const uint32_t byte = scale_byte<FMT>(block_top(x));
      if (is_v) {
        vsc[blk][t] = byte;
        /* (also a scale whose largest code stands for 2^128) */
        if (byte >= (FMT == AOS_KV_MXFP8 ? 247u : 253u)) *p.b.nonfinite = 1u;
        if (fresh) tile[vs_off<FMT, HDP>() + blk * TILE + tp + t] = (unsigned char)byte;
        continue;
      }
      if (!fresh) continue;
      tile[ks_off<FMT, HDP>() + blk * TILE + ks_index(tp + t)] = (unsigned char)byte;
      constexpr int UNITS = FMT == AOS_KV_MXFP8 ? 2 : 1, U = 32 / UNITS;
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        u32x4 w = {};
#pragma unroll
        for (int i = 0; i < U / 2; ++i) {
          const uint32_t pair = *(const uint32_t *)(x + U * j + 2 * i);
          if constexpr (FMT == AOS_KV_MXFP8)
            w[i >> 1] |= encode2<FMT>(pair, byte) << (16 * (i & 1));
          else
            w[i >> 2] |= encode2<FMT>(pair, byte) << (8 * (i & 3));
        }
        *(u32x4 *)(tile + ((blk * UNITS + j) * TILE + tp + t) * 16) = w;
      }
    }
    __syncthreads();
  }

  /* values: a thread per dimension packs its 16 positions; those that are not new keep what they hold */
  for (int d = tid; d < HDP; d += 256) {
    if constexpr (FMT == AOS_KV_BF16) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (o.lo >= 8 * j + 8 || o.hi <= 8 * j) continue;
        u32x4 *at = (u32x4 *)(tile + v_off<FMT, HDP>() + ((tp / 8 + j) * HDP + d) * 16);
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = (uint32_t)vs[(8 * j + 2 * i) * LD + d] | ((uint32_t)vs[(8 * j + 2 * i + 1) * LD + d] << 16);
        if (o.lo > 8 * j || o.hi < 8 * j + 8) {
          const u32x4 old = *at;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = 8 * j + 2 * i;
            const uint32_t m = (t >= o.lo && t < o.hi ? 0xffffu : 0u) |
                               (t + 1 >= o.lo && t + 1 < o.hi ? 0xffff0000u : 0u);
            w[i] = (w[i] & m) | (old[i] & ~m);
          }
        }
        *at = w;
      }
    } else {
      constexpr int W = FMT == AOS_KV_MXFP8 ? 4 : 2, PER = 16 / W; /* words of the unit, positions of a word */
      constexpr int B = 32 / PER;
      uint32_t *at = (uint32_t *)(tile + v_off<FMT, HDP>() + ((tp / 16) * HDP + d) * (4 * W));
      uint32_t w[W];
      const bool part = o.lo > 0 || o.hi < 16;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        uint32_t x = 0, m = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int t = PER * i + j;
          x |= (encode2<FMT>(vs[t * LD + d], vsc[d >> 5][t]) & ((1u << B) - 1u)) << (B * j);
          m |= (t >= o.lo && t < o.hi ? (1u << B) - 1u : 0u) << (B * j);
        }
        w[i] = x;
        if (part) w[i] = (w[i] & m) | (at[i] & ~m);
      }
      if constexpr (FMT == AOS_KV_MXFP8)
        *(u32x4 *)at = u32x4{w[0], w[1], w[W - 2], w[W - 1]};
      else
        *(u32x2 *)at = u32x2{w[0], w[1]};
    }
  }
}

/* two codes of the low bits of a word -> packed bfloat16 */
template <int FMT, int SEL>
__device__ __forceinline__ uint32_t decode2(uint32_t w, uint32_t byte) {
  if constexpr (FMT == AOS_KV_MXFP8)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale_of(byte), SEL != 0));
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale_of(byte), SEL));
}

constexpr int READ_HEADS = 4; /* key/value heads of a workgroup */

/* Grid (blocks of 16 positions, groups of key/value heads). Keys: a thread per unit; values: a thread per four
 * dimensions, whose units it holds while it writes them position by position. Bound by memory: 16 sequences of up to 8001
 * positions, 8 heads of 128, at 8 bits 107 us (514 MB read and written, 4.8 TB/s: a large copy's rate). */
template <int FMT, int HDP>
__global__ void __launch_bounds__(256) aos_kv_read_kernel(aos_kv_read_params p) {
  const int tid = threadIdx.x, lane = tid & 63;
  Block o;
  if (!block_at(p.b, (int)blockIdx.x, lane, o)) return;
  const int page = page_of(p.b, o.seq, o.pos);
  const int hd = p.b.hd, tp = o.pos & 48;
  const int h0 = blockIdx.y * READ_HEADS, nheads = p.b.nkv - h0 < READ_HEADS ? p.b.nkv - h0 : READ_HEADS;
  constexpr int U = 128 / bits<FMT>(); /* dimensions of a key unit */
  constexpr int KT = HDP / U * 16, VT = HDP / 4;
  const int row0 = o.row - o.lo;

  for (int c = tid; c < nheads * KT; c += 256) {
    const int h = h0 + c / KT, t = c % 16, u = c % KT / 16;
    if (t < o.lo || t >= o.hi || U * u >= hd) continue;
    uint16_t *y = p.k + (long long)(row0 + t) * p.k_ld + h * hd + U * u;
    uint32_t r[U / 2] = {};
    if (page >= 0) {
      const unsigned char *tile = tile_ptr<FMT, HDP>(p.b, page, h, o.pos);
      const u32x4 w = *(const u32x4 *)(tile + (u * TILE + tp + t) * 16);
      if constexpr (FMT == AOS_KV_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = w[i];
      } else {
        const uint32_t byte = tile[ks_off<FMT, HDP>() + (U * u / 32) * TILE + ks_index(tp + t)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (FMT == AOS_KV_MXFP8) {
            r[2 * i] = decode2<FMT, 0>(w[i], byte);
            r[2 * i + 1] = decode2<FMT, 1>(w[i], byte);
          } else {
            r[(4 * i) % (U / 2)] = decode2<FMT, 0>(w[i], byte);
            r[(4 * i + 1) % (U / 2)] = decode2<FMT, 1>(w[i], byte);
            r[(4 * i + 2) % (U / 2)] = decode2<FMT, 2>(w[i], byte);
            r[(4 * i + 3) % (U / 2)] = decode2<FMT, 3>(w[i], byte);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U / 8; ++i)
      if (U * u + 8 * i < hd) *(u32x4 *)(y + 8 * i) = u32x4{r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]};
  }
  for (int c = tid; c < nheads * VT; c += 256) {
    const int h = h0 + c / VT, d = 4 * (c % VT);
    if (d >= hd) continue;
    uint16_t x[4][16] = {};
    if (page >= 0) {
      const unsigned char *tile = tile_ptr<FMT, HDP>(p.b, page, h, o.pos);
      uint32_t sb[4] = {};
      if constexpr (FMT != AOS_KV_BF16) {
        const u32x4 s = *(const u32x4 *)(tile + vs_off<FMT, HDP>() + (d >> 5) * TILE + tp);
#pragma unroll
        for (int i = 0; i < 4; ++i) sb[i] = s[i];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (FMT == AOS_KV_BF16) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x4 w = *(const u32x4 *)(tile + v_off<FMT, HDP>() + ((tp / 8 + e) * HDP + d + j) * 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][8 * e + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
          }
        } else {
          constexpr int W = FMT == AOS_KV_MXFP8 ? 4 : 2, PER = 16 / W;
          const uint32_t *at = (const uint32_t *)(tile + v_off<FMT, HDP>() + ((tp / 16) * HDP + d + j) * (4 * W));
          uint32_t w[W];
          if constexpr (FMT == AOS_KV_MXFP8) {
            const u32x4 l = *(const u32x4 *)at;
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = l[i];
          } else {
            const u32x2 l = *(const u32x2 *)at;
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = l[i % 2];
          }
#pragma unroll
          for (int t = 0; t < 16; ++t) /* (each position has a scale of its own) */
            x[j][t] = (uint16_t)decode2<FMT, 0>(w[t / PER] >> (32 / PER * (t % PER)), (sb[t >> 2] >> (8 * (t & 3))) & 255u);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      if (t < o.lo || t >= o.hi) continue;
      u32x2 w;
      w.x = (uint32_t)x[0][t] | ((uint32_t)x[1][t] << 16);
      w.y = (uint32_t)x[2][t] | ((uint32_t)x[3][t] << 16);
      *(u32x2 *)(p.v + (long long)(row0 + t) * p.v_ld + h * hd + d) = w;
    }
  }
}

template <int FMT, int HDP>
int append(const aos_kv_append_params *p, const aos_launch_ctx *ctx) {
  const int qg = p->q ? (p->nh + Q_HEADS - 1) / Q_HEADS : 0;
  aos_kv_append_params a = *p;
  const dim3 grid(blocks_of(p->b.max_new, p->b.n_seqs, p->b.n_tokens), qg + p->b.nkv);
  if (p->at)
    AOS_LAUNCH(ctx, (aos_kv_append_kernel<FMT, HDP, true>), grid, dim3(256), 0, a, qg);
  else
    AOS_LAUNCH(ctx, (aos_kv_append_kernel<FMT, HDP, false>), grid, dim3(256), 0, a, qg);
  return (int)hipGetLastError();
}
template <int FMT, int HDP>
int read(const aos_kv_read_params *p, const aos_launch_ctx *ctx) {
  AOS_LAUNCH(ctx, (aos_kv_read_kernel<FMT, HDP>), dim3(blocks_of(p->b.max_new, p->b.n_seqs, p->b.n_tokens), (p->b.nkv + READ_HEADS - 1) / READ_HEADS),
             dim3(256), 0, *p);
  return (int)hipGetLastError();
}

template <int FMT>
size_t tile_of(int hdp) {
  return hdp == 64 ? tile_bytes<FMT, 64>() : hdp == 128 ? tile_bytes<FMT, 128>() : tile_bytes<FMT, 256>();
}

}  // namespace

size_t aos_kv_tile_bytes(int format, int hdp) {
  return format == AOS_KV_BF16 ? tile_of<AOS_KV_BF16>(hdp)
                               : format == AOS_KV_MXFP8 ? tile_of<AOS_KV_MXFP8>(hdp) : tile_of<AOS_KV_MXFP4>(hdp);
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

extern "C" int aos_launch_kv_append(const aos_kv_append_params *p, const aos_launch_ctx *ctx) {
  return KV_DISPATCH(append, p->b.format, p->b.hdp, p, ctx);
}

extern "C" int aos_launch_kv_read(const aos_kv_read_params *p, const aos_launch_ctx *ctx) {
  return KV_DISPATCH(read, p->b.format, p->b.hdp, p, ctx);
}

/* Diagnostic, for tests without a device: the launches' blocks of a batch, and block x of sequence s (its rows row0 ..
 * row0 + count - 1, its length): out = {position, lo, hi, row of position + lo}; 1 where there is such a block. */
extern "C" int aoship_internal_kv_blocks(int max_new, int n_seqs, int n_tokens) {
  return blocks_of(max_new, n_seqs, n_tokens);
}
extern "C" int aoship_internal_kv_block(int max_new, int s, int row0, int count, int len, int x, int *base, int *out) {
  Block o = {};
  *base = block_base(max_new, s, row0);
  if (!block_of(max_new, s, Seq{row0, count, len}, x, o)) return 0;
  out[0] = o.pos;
  out[1] = o.lo;
  out[2] = o.hi;
  out[3] = o.row;
  return 1;
}
