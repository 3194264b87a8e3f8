/*
 * aoship_kv_evict.hip — shortening sequences of the paged cache to the positions that matter.
 *
 * Of each sequence of L positions and each key/value head, n = min(keep, L) stay: the first ones, the last ones, and of those
 * between the ones of greatest weight (a NaN below everything; equal weights: the lower positions), in their order. They
 * are moved to other pages, codes and scales as they are, so that nothing is rounded again.
 *
 *   select  the n-th greatest weight by its bits, two a turn: a workgroup counts the weights that reach each of three bounds, 16
 *           times at most and once more where equal weights part; after eight bits those still in question, if few, are
 *           listed and only they counted. It holds a head's weights itself up to 32768, and reads longer ones again each
 *           turn; then the kept positions' places by counting the kept ones before them.
 *   move    a workgroup gathers a tile of 64 kept positions. Keys are 16-byte units of one position; values, whose units
 *           hold 8 or 16 positions of a dimension, are taken apart and put together element by element.
 */
#include "aoship_internal.h"
#include "aoship_kv.h"
#include <hip/hip_ext.h>

using namespace kv;

namespace {

constexpr int NT = 1024, NW = NT / 64;
constexpr int MOST = 32;     /* weights of a thread at once, at most */
constexpr int LIST = 4 * NT; /* weights that are listed */

/* what stays of a sequence: n positions; n < 0: left out (a fault, noted) */
struct Kept {
  int len, n;
};
__device__ __forceinline__ Kept kept_of(const aos_kv_evict_params &p, int s) {
  Kept k;
  k.len = p.b.lens[s];
  const int keep = p.keep[s];
  k.n = keep < k.len ? keep : k.len;
  const bool ok = k.len >= 0 && k.len <= p.b.max_len && keep >= 0 && k.n <= p.max_keep &&
                  (keep >= k.len || (long long)p.first + p.recent <= keep);
  if (!ok) {
    k.n = -1;
    note(p.b.faults, AOS_KV_FAULT_BATCH);
  }
  return k;
}

/* order of weights as unsigned numbers: a NaN first (0), both zeros alike */
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  return w != w ? 0u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

/* inclusive sums over the wave's lanes */
__device__ __forceinline__ int lane_scan(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = (int)aos_shfl((uint32_t)x, lane - d);
    if (lane >= d) x += y;
  }
  return x;
}

/* Bound by the latency of its turns and by how few workgroups there are: 2 heads of 2047 weights 11 us, 128 of up to 12000 26,
 * 32 of up to 32767 52. The instance of 32 weights a thread (max_len past 16384) is at its 128 registers and keeps 31 of a
 * thread's words in private memory.
 * Grid: sequences times key/value heads. Thread t has the positions t, t + 1024, ... of a span of PER * 1024. */
template <int PER>
__global__ void __launch_bounds__(NT) aos_kv_select_kernel(aos_kv_evict_params p) {
  constexpr int SPAN = NT * PER;
  __shared__ int total[3][3]; /* counts of three bounds, of this turn, the next and the last */
  __shared__ int above[PER * NW], ties[PER * NW]; /* of a wave's 64 positions: kept for sure, and of the bound's weight */
  __shared__ int totals[2], listed;
  __shared__ uint32_t list[LIST];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int sh = (int)(p.wg0 + blockIdx.x), s = sh / p.b.nkv, h = sh - s * p.b.nkv;
  const Kept k = kept_of(p, s);
  if (k.n < 0) return;
  const float *w = p.weights + (long long)s * p.w_seq + (long long)h * p.w_head;
  int32_t *kept = p.kept + (long long)s * p.kept_seq + (long long)h * p.kept_head;
  float *wo = p.w_out ? p.w_out + (long long)s * p.wo_seq + (long long)h * p.wo_head : nullptr;
  if (k.n == k.len) {
    for (int i = tid; i < k.len; i += NT) {
      kept[i] = i;
      if (wo) wo[i] = w[i];
    }
    return;
  }
  const int lo = p.first, hi = k.len - p.recent; /* to choose from: lo .. hi - 1 (there are more than enough) */
  const int m = k.n - p.first - p.recent;

  /* x: a weight's order plus one, 0 for positions that are not to be chosen from (n < len <= 2^30, and the order of
   * the greatest float stays below 2^32 - 1) */
  /* (loads without a condition, all on their way together) */
  auto weight = [&](int pos) { /* (32-bit offsets: 2^30 positions at most) */
    return *(const float *)((const char *)w + (uint32_t)(pos < k.len ? pos : k.len - 1) * 4u);
  };
  auto load = [&](uint32_t (&x)[PER], int base) {
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = weight(base + i * NT + tid);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int pos = base + i * NT + tid;
      x[i] = pos >= lo && pos < hi ? order_of(v[i]) + 1u : 0u;
    }
  };
  const bool once = k.len <= SPAN;
  uint32_t x[PER];
  if (once) load(x, 0);
  auto count_of = [&](auto &&counts) { /* counts(x) of each of a thread's weights, span by span */
    for (int base = 0; base < k.len; base += SPAN) {
      if (!once) load(x, base);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        counts(x[i]);
      }
    }
  };
  /* The greatest bound that at least m reach, two bits a turn; with exactly m there are no ties to part. After eight bits the
   * weights between the bound and the next one are mostly few: listed, a thread has at most four of them to count. */
  uint32_t bound = 0;
  int reach = hi - lo, over = 0; /* how many reach it, and the next bound that the bits so far can make */
  if (m > 0) {
    int turn = 0;
    if (tid < 3) total[0][tid] = 0;
    __syncthreads();
    auto step = [&](int bit, const int (&c)[3], int more) { /* c: this wave's counts; more: what they leave out */
      const uint32_t at = bound | (1u << bit);
      if (lane < 3) atomicAdd(&total[turn][lane], lane == 0 ? c[0] : lane == 1 ? c[1] : c[2]);
      const int next = turn == 2 ? 0 : turn + 1;
      if (tid < 3) total[next][tid] = 0; /* (read last two turns ago) */
      __syncthreads();
      const int all[3] = {total[turn][0], total[turn][1], total[turn][2]};
      turn = next;
#pragma unroll
      for (int j = 2; j >= 0; --j) {
        const int n = __builtin_amdgcn_readfirstlane(all[j]) + more;
        if (n >= m) {
          bound = at + ((uint32_t)j << bit);
          reach = n;
          break;
        }
        over = n;
      }
    };
    auto count_of_one = [&](int bit, uint32_t y, int (&c)[3]) {
#pragma unroll
      for (int j = 0; j < 3; ++j) c[j] += (int)__popcll(__ballot(y >= (bound | (1u << bit)) + ((uint32_t)j << bit)));
    };
    int bit = 30;
    for (; bit >= 24 && reach != m; bit -= 2) { /* (uniform) */
      int c[3] = {};
      count_of([&](uint32_t y) { count_of_one(bit, y, c); });
      step(bit, c, 0);
    }
    if (reach != m && reach - over <= LIST) {
      if (tid == 0) listed = 0;
      __syncthreads();
      count_of([&](uint32_t y) {
        if (y > 0u && y >> 24 == bound >> 24) list[atomicAdd(&listed, 1)] = y; /* reach - over of them */
      });
      __syncthreads();
      const int n = listed, rest = over;
      uint32_t y[LIST / NT];
#pragma unroll
      for (int j = 0; j < LIST / NT; ++j) y[j] = j * NT + tid < n ? list[j * NT + tid] : 0u;
      for (; bit >= 0 && reach != m; bit -= 2) {
        int c[3] = {};
#pragma unroll
        for (int j = 0; j < LIST / NT; ++j)
          if (j * NT < n) count_of_one(bit, y[j], c);
        step(bit, c, rest);
      }
    }
    for (; bit >= 0 && reach != m; bit -= 2) {
      int c[3] = {};
      count_of([&](uint32_t y) { count_of_one(bit, y, c); });
      step(bit, c, 0);
    }
  } else {
    bound = 0xffffffffu; /* (no weight's) */
  }
  const bool exact = m == 0 || reach == m;
  int taken = 0, left = 0; /* places before this span; ties that are still kept */
  if (!exact) {
    /* m less those above the bound */
    int c = 0;
    count_of([&](uint32_t y) { c += (int)__popcll(__ballot(y > bound)); });
    __syncthreads();
    if (tid == 0) total[0][0] = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(&total[0][0], c);
    __syncthreads();
    left = m - total[0][0];
  }

  for (int base = 0; base < k.len; base += SPAN) {
    if (!once) load(x, base);
    auto sure = [&](int i) { /* kept whatever its ties */
      const int pos = base + i * NT + tid;
      return pos < k.len && (pos < lo || pos >= hi || (exact ? x[i] >= bound : x[i] > bound));
    };
    auto tie = [&](int i) { return !exact && x[i] == bound; }; /* (bound > 0) */
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int a = (int)__popcll(__ballot(sure(i))), t = (int)__popcll(__ballot(tie(i)));
      if (lane == 0) {
        above[i * NW + wave] = a;
        ties[i * NW + wave] = t;
      }
    }
    __syncthreads();
    if (wave == 0) {
      /* PER * NW groups of 64 positions in order, EACH a lane: ties before each, then places before each */
      constexpr int EACH = PER * NW / 64;
      int t[EACH], sum = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        t[i] = ties[lane * EACH + i];
        sum += t[i];
      }
      int before = lane_scan(sum, lane) - sum, places = 0;
      const int all_ties = __builtin_amdgcn_readlane(before + sum, 63);
      int a[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int at = lane * EACH + i, room = left - before;
        a[i] = above[at] + (room < 0 ? 0 : room < t[i] ? room : t[i]);
        ties[at] = before;
        before += t[i];
        places += a[i];
      }
      int place = lane_scan(places, lane) - places;
      if (lane == 63) {
        totals[0] = place + places;
        totals[1] = all_ties;
      }
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        above[lane * EACH + i] = place;
        place += a[i];
      }
    }
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1ull;
    constexpr int FLY = PER < 8 ? PER : 8;
#pragma unroll
    for (int i0 = 0; i0 < PER; i0 += FLY) {
      float v[FLY];
#pragma unroll
      for (int i = 0; i < FLY; ++i) v[i] = weight(base + (i0 + i) * NT + tid);
#pragma unroll
      for (int i = 0; i < FLY; ++i) {
        const bool y = sure(i0 + i), t = tie(i0 + i);
        const uint64_t ys = __ballot(y), ts = __ballot(t);
        const int group = (i0 + i) * NW + wave, room = left - ties[group], mine = (int)__popcll(ts & below);
        const uint32_t at = (uint32_t)(taken + above[group] + (int)__popcll(ys & below) + (mine < room ? mine : room > 0 ? room : 0));
        if (y || (t && mine < room)) {
          *(int32_t *)((char *)kept + at * 4u) = base + (i0 + i) * NT + tid;
          if (wo) *(float *)((char *)wo + at * 4u) = v[i];
        }
      }
      aos_compiler_barrier(); /* (no more of them in registers at once) */
    }
    __syncthreads();
    taken += totals[0];
    left -= totals[1] < left ? totals[1] : left;
    __syncthreads(); /* (totals are free again) */
  }
  if (wo)
    for (int i = k.n + tid; i < k.len; i += NT) wo[i] = 0.0f;
}

/* Grid: tiles of 64 kept positions, key/value heads, sequences. Bound by memory at 16 bits: 4 sequences of up to 32767 down to
 * 15000, 8 heads of 128, 126 us (345 MB fetched, 226 written, 4.5 TB/s); by the taking apart of values at 4: 16 of up to
 * 12000 down to 4096, 77 us (141 and 70 MB, 2.7 TB/s). */
template <int FMT, int HDP>
__global__ void __launch_bounds__(256) aos_kv_move_kernel(aos_kv_evict_params p, int tiles) {
  __shared__ const unsigned char *src[TILE]; /* the tiles that the positions are in; NULL: none */
  __shared__ int in[TILE];                   /* their places in them */
  const int tid = threadIdx.x;
  const uint32_t wg = p.wg0 + blockIdx.x;
  const int tile = (int)(wg % (uint32_t)tiles), sh = (int)(wg / (uint32_t)tiles);
  const int s = sh / p.b.nkv, h = sh - s * p.b.nkv, i0 = tile * TILE;
  const Kept k = kept_of(p, s);
  if (i0 >= k.n) return;
  const int n = k.n - i0 < TILE ? k.n - i0 : TILE;
  const int to = page_checked(p.b, p.to[(long long)s * p.to_stride + (i0 >> p.b.page_shift)]);
  if (to < 0) return; /* uniform */
  unsigned char *dst = tile_ptr<FMT, HDP>(p.b, to, h, i0);
  if (tid < TILE) {
    const unsigned char *t = nullptr;
    int pos = 0;
    if (tid < n) {
      pos = p.kept[(long long)s * p.kept_seq + (long long)h * p.kept_head + i0 + tid];
      const int page = (unsigned)pos < (unsigned)k.len ? page_of(p.b, s, pos) : -1;
      if (page >= 0) t = tile_ptr<FMT, HDP>(p.b, page, h, pos);
    }
    src[tid] = t;
    in[tid] = pos & (TILE - 1);
  }
  __syncthreads();

  constexpr int KU = HDP * bits<FMT>() / 128; /* key units of a position */
#pragma unroll 4
  for (int c = tid; c < KU * TILE; c += 256) {
    const int i = c % TILE, u = c / TILE;
    if (i >= n) continue;
    const unsigned char *t = src[i];
    *(u32x4 *)(dst + (u * TILE + i) * 16) = t ? aos_gld16(t + (u * TILE + in[i]) * 16) : u32x4{};
  }
  if constexpr (FMT == AOS_KV_BF16) {
    /* a thread per unit of 8 positions of a dimension. Where its positions come from is the same for all lanes of a
     * wave, so a source unit is loaded once for the run of positions that are in it (127 us where a load for each position
     * took 143; for the quantised formats, whose units are cheaper to load, 81 and 77 the other way) */
    for (int c = tid; c < TILE / 8 * HDP; c += 256) {
      const int u = __builtin_amdgcn_readfirstlane(c / HDP), d = c % HDP;
      if (8 * u >= n) break;
      u32x4 x = {};
      uint32_t y[4] = {};
      const unsigned char *from = nullptr;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint64_t t = (uint64_t)src[8 * u + e];
        const unsigned char *unit = (const unsigned char *)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 32)) << 32) |
                                                            (uint32_t)__builtin_amdgcn_readfirstlane((int)t));
        const int at = __builtin_amdgcn_readfirstlane(in[8 * u + e]);
        if (unit) unit += v_off<FMT, HDP>() + at / 8 * HDP * 16;
        if (e == 0 || unit != from) { /* uniform */
          from = unit;
          x = unit ? aos_gld16(unit + d * 16) : u32x4{};
        }
        uint32_t w = x[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) w = at % 8 / 2 == i ? x[i] : w;
        y[e / 2] |= (w >> (at & 1) * 16 & 0xffffu) << (e % 2 * 16);
      }
      *(u32x4 *)(dst + v_off<FMT, HDP>() + (u * HDP + d) * 16) = u32x4{y[0], y[1], y[2], y[3]};
    }
  } else {
    constexpr int W = FMT == AOS_KV_MXFP8 ? 4 : 2; /* words of a value unit: 16 positions of a dimension */
    for (int c = tid; c < (TILE / 16) * HDP; c += 256) {
      const int d = c % HDP, u = c / HDP;
      if (16 * u >= n) break;
      uint32_t y[W] = {};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const unsigned char *t = src[16 * u + e];
        const int at = in[16 * u + e], byte = FMT == AOS_KV_MXFP8 ? at % 16 : at % 16 / 2;
        uint32_t x = t ? *(const __attribute__((address_space(1))) unsigned char *)(t + v_off<FMT, HDP>() + (at / 16 * HDP + d) * (4 * W) + byte) : 0u;
        if constexpr (FMT == AOS_KV_MXFP8) {
          y[e / 4] |= x << (8 * (e % 4));
        } else {
          x = at & 1 ? x >> 4 : x & 15u;
          y[e / 8] |= x << (4 * (e % 8));
        }
      }
      if constexpr (FMT == AOS_KV_MXFP8)
        *(u32x4 *)(dst + v_off<FMT, HDP>() + (u * HDP + d) * 16) = u32x4{y[0], y[1], y[W - 2], y[W - 1]};
      else
        *(u32x2 *)(dst + v_off<FMT, HDP>() + (u * HDP + d) * 8) = u32x2{y[0], y[1]};
    }
    for (int c = tid; c < 2 * (HDP / 32) * TILE; c += 256) {
      const int i = c % TILE, b = c / TILE % (HDP / 32);
      if (i >= n) continue;
      const bool is_v = c >= (HDP / 32) * TILE;
      const unsigned char *t = src[i];
      const int from = is_v ? vs_off<FMT, HDP>() + b * TILE + in[i] : ks_off<FMT, HDP>() + b * TILE + ks_index(in[i]);
      const int at = is_v ? vs_off<FMT, HDP>() + b * TILE + i : ks_off<FMT, HDP>() + b * TILE + ks_index(i);
      dst[at] = t ? t[from] : 0;
    }
  }
}

template <int FMT, int HDP>
int evict(const aos_kv_evict_params *p, const aos_launch_ctx *ctx) {
  const uint32_t sh = (uint32_t)p->b.n_seqs * (uint32_t)p->b.nkv;
  /* registers for the longest sequence */
  const int len = p->b.max_len;
  aos_kv_evict_params a = *p;
  for (a.wg0 = 0; a.wg0 < sh; a.wg0 += AOS_LAUNCH_PIECE(sh - a.wg0)) {
    const uint32_t n = AOS_LAUNCH_PIECE(sh - a.wg0);
    if (len <= 4 * NT)
      AOS_LAUNCH(ctx, aos_kv_select_kernel<4>, dim3(n), dim3(NT), 0, a);
    else if (len <= 16 * NT)
      AOS_LAUNCH(ctx, aos_kv_select_kernel<16>, dim3(n), dim3(NT), 0, a);
    else
      AOS_LAUNCH(ctx, aos_kv_select_kernel<MOST>, dim3(n), dim3(NT), 0, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  const int tiles = (p->max_keep + TILE - 1) / TILE;
  const uint32_t wgs = sh * (uint32_t)tiles;
  for (a.wg0 = 0; a.wg0 < wgs; a.wg0 += AOS_LAUNCH_PIECE(wgs - a.wg0)) {
    AOS_LAUNCH(ctx, (aos_kv_move_kernel<FMT, HDP>), dim3(AOS_LAUNCH_PIECE(wgs - a.wg0)), dim3(256), 0, a, tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

}  // namespace

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

extern "C" int aos_launch_kv_evict(const aos_kv_evict_params *p, const aos_launch_ctx *ctx) {
  return KV_DISPATCH(evict, p->b.format, p->b.hdp, p, ctx);
}
