/*
 * aoship_logprobs.hip — log probabilities of rows of logits: of a given token, with its rank and the row's entropy,
 * and of the n most probable tokens.
 *
 *   m = max x,  l = sum e^(x_i - m),  s = sum e^(x_i - m) (x_i - m)
 *   log p_t = x_t - m - ln l     H = ln l - s / l     rank = number of x_i > x_t, or x_i = x_t with i < t
 *
 * in one pass with a running m, l and s in float32 (rescaled where a thread's 16 or 32 values bring a new maximum), and
 * the n largest in the order of value, then index (so that the answer is one set and one order, whoever finds it).
 *
 * The n largest without sorting anything long: a thread's 16-byte units of the row (every 256th) are four groups, of
 * each of which it keeps the largest value and the unit it is in. The n largest elements lie in the n groups whose
 * largest come first; these few groups are read again (from the L2), what is not before the last of their largest
 * goes to a list (about n entries), and an entry's place in the answer is the number of entries before it. The n groups
 * are found in the same way: a bound that n of a wave's lanes reach, then a list and places in it.
 *
 * Few rows are cut into slices, whose pieces the row's last workgroup joins.
 *
 * Bound by reading the logits once, and nearly as much by the vector instructions (an exponential and nine others a logit):
 * 4000 rows of 50257 bfloat16 97 us, 4.1 TB/s. Few rows by the latencies of the choice: 1 row of 152064 with 5 tokens 14
 * us, 64 of 128256 with 20 24 us (taking the n one after the other from 64 lanes 72).
 */
#include "aoship_device.h"
#include "aoship_internal.h"
#include <hip/hip_ext.h>

namespace {

constexpr int NT = 256;         /* threads of a workgroup */
constexpr int SEGS = 4;         /* groups of a thread */
constexpr int LIST = 1024;      /* entries of the list */
constexpr float LEAST = -3.40282347e38f;
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;
constexpr uint32_t NONE = 0xffffffffu;

/* order of candidates: by value (both zeros alike), then by index; 0 is no candidate */
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
  const uint32_t o = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~(uint32_t)k; }

/* largest of the wave's values, by data moves within the vector registers (lane 63 ends with all of them); uniform */
__device__ __forceinline__ uint32_t wave_max32(uint32_t x) {
  auto step = [&](uint32_t y) { x = y > x ? y : x; };
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false)); /* row_shr 1, 2, 4, 8 */
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false)); /* row_bcast 15, 31 */
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ uint64_t lane_key(uint64_t k, int lane) {
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(k >> 32), lane);
  return ((uint64_t)hi << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}
/* largest key: the values first, the indices only where several lanes have the value */
__device__ __forceinline__ uint64_t wave_max(uint64_t k) {
  const uint32_t hi = wave_max32((uint32_t)(k >> 32));
  const uint64_t tied = __ballot((uint32_t)(k >> 32) == hi);
  if (tied & (tied - 1)) return ((uint64_t)hi << 32) | wave_max32((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return lane_key(k, __builtin_ctzll(tied));
}

/* Running maximum m, sum l of 2^a and weighted sum s of 2^a a, a = (x - m) log2 e. (A maximum kept times log2 e would make a
 * one fused operation, but overflows for logits past 2.3e38.) */
struct Stat {
  float m, l, s;
  __device__ __forceinline__ void clear() { m = LEAST, l = 0.0f, s = 0.0f; }
  __device__ __forceinline__ void lift(float top) { /* to a maximum that is no less */
    const float d = (m - top) * LOG2E, f = __builtin_amdgcn_exp2f(d);
    s = f * (s + l * fmaxf(d, -200.0f)); /* (below that f is zero: no zero times infinity) */
    l = l * f;
    m = top;
  }
  __device__ __forceinline__ void add(float x) { /* x <= m */
    const float a = (x - m) * LOG2E, e = __builtin_amdgcn_exp2f(a);
    l = l + e;
    s = fmaf(e, fmaxf(a, -200.0f), s);
  }
  __device__ __forceinline__ void join(Stat o) {
    const float top = fmaxf(m, o.m);
    lift(top);
    o.lift(top);
    l = l + o.l;
    s = s + o.s;
  }
};

constexpr int PAD = 32;

struct Shared {
  uint64_t list[LIST + PAD];
  uint64_t wave[4];
  uint64_t top[AOS_LOGPROBS_MAX_TOP];
  float stat[4][3];
  int before[4];
  uint32_t listed;
};

/* The n first of the list's entries, in order, into sh.top (zeros where there are fewer): each counts those before it. */
__device__ __forceinline__ void rank_list(Shared &sh, int n) {
  __syncthreads();
  const int count = (int)sh.listed, tid = threadIdx.x;
  if (tid < n) sh.top[tid] = 0;
  if (tid < PAD) sh.list[count + tid] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < count; i0 += NT / 4) { /* four lanes an entry, each with every fourth of the others */
    const int i = i0 + tid / 4;
    const uint64_t mine = i < count ? sh.list[i] : 0;
    int before = 0;
    for (int j = tid % 4; j < count; j += PAD) /* (eight reads in flight together) */
#pragma unroll
      for (int k = 0; k < PAD; k += 4) before += sh.list[j + k] > mine ? 1 : 0;
    before += __builtin_amdgcn_update_dpp(0, before, 0xb1, 0xf, 0xf, false); /* quad_perm 1 0 3 2 */
    before += __builtin_amdgcn_update_dpp(0, before, 0x4e, 0xf, 0xf, false); /* 2 3 0 1 */
    if (i < count && tid % 4 == 0 && before < n) sh.top[before] = mine;
  }
  __syncthreads();
}
__device__ __forceinline__ void push(Shared &sh, uint64_t k) {
  const uint32_t at = atomicAdd(&sh.listed, 1u);
  if (at < LIST) sh.list[at] = k;
}

/* The n largest of all threads' four keys (distinct, zeros for none), in order, into sh.top. Of a wave's lanes' largest the
 * n-th is no more than the n-th of all keys: those from the largest such bound on are listed, about twice n. */
__device__ __forceinline__ void largest(Shared &sh, const uint64_t (&k)[4], int n) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t a = k[0] > k[1] ? k[0] : k[1], b = k[2] > k[3] ? k[2] : k[3], mine = a > b ? a : b;
  /* a lane counts the lanes before its own (bisecting the bound's bits by ballots, a chain of scalar turns, made 1 row of
   * 152064 19.3 us for 14.5, 64 of 128256 28.3 for 24.4) */
  int before = 0;
#pragma unroll 16
  for (int j = 0; j < 64; ++j) before += lane_key(mine, j) > mine ? 1 : 0;
  const uint64_t nth = __ballot(mine != 0 && before == n - 1); /* (none: fewer than n keys) */
  const uint64_t bound = nth ? lane_key(mine, __builtin_ctzll(nth)) : 0;
  if (lane == 0) sh.wave[wave] = bound;
  if (tid == 0) sh.listed = 0;
  __syncthreads();
  uint64_t from = 1;
#pragma unroll
  for (int w = 0; w < 4; ++w) from = sh.wave[w] > from ? sh.wave[w] : from;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (k[i] >= from) push(sh, k[i]);
  rank_list(sh, n);
  if (tid == 0) sh.listed = 0;
  __syncthreads();
}

template <bool BF16>
struct Unit { /* 16 bytes of a row */
  static constexpr int N = BF16 ? 8 : 4;
  u32x4 w;
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (BF16)
      return __builtin_bit_cast(float, i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    return __builtin_bit_cast(float, (uint32_t)w[i]); /* (of an element as it stands, the compiler takes the first) */
  }
};
template <bool BF16>
__device__ __forceinline__ float element(const void *row, long long i) {
  if constexpr (BF16) return aos_bf16_to_f32(((const uint16_t *)row)[i]);
  return ((const float *)row)[i];
}

/* the next float32 under a finite one or +infinity */
__device__ __forceinline__ float next_under(float x) {
  const int u = (int)__builtin_bit_cast(uint32_t, x + 0.0f); /* (-0 as +0) */
  return __builtin_bit_cast(float, (uint32_t)(u > 0 ? u - 1 : u == 0 ? (int)0x80000001 : u + 1));
}

/* what a workgroup writes of a row: the answer, or its slice's piece of it */
__device__ __forceinline__ void answer(const aos_logprobs_params &p, Shared &sh, int row, Stat st, float xt, bool target,
                                       int before) {
  const int tid = threadIdx.x;
  const float bits = log2f(st.l), nan = __builtin_nanf("");
  const bool ok = st.l > 0.0f; /* neither a NaN nor all minus infinity */
  auto lnp = [&](float x) { return (x - st.m) - bits * LN2; };
  if (tid == 0) {
    if (p.logprob) p.logprob[row] = ok && target ? lnp(xt) : nan;
    if (p.rank) p.rank[row] = ok && target ? before : -1;
    if (p.entropy) p.entropy[row] = ok ? (bits - st.s / st.l) * LN2 : nan;
  }
  if (tid < p.n_top) {
    const uint64_t k = sh.top[tid];
    const long long at = (long long)row * p.n_top + tid;
    if (p.top_ids) p.top_ids[at] = ok ? (int)key_index(k) : -1;
    if (p.top_logprobs) p.top_logprobs[at] = ok ? lnp(key_value(k)) : nan;
  }
}

/* the waves' statistics and counts joined, in order, for every thread */
__device__ __forceinline__ void join_block(Shared &sh, Stat &st, int &before) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    Stat o;
    o.m = aos_shfl_f(st.m, lane ^ d);
    o.l = aos_shfl_f(st.l, lane ^ d);
    o.s = aos_shfl_f(st.s, lane ^ d);
    before += (int)aos_shfl((uint32_t)before, lane ^ d);
    st.join(o);
  }
  if (lane == 0) {
    sh.stat[wave][0] = st.m;
    sh.stat[wave][1] = st.l;
    sh.stat[wave][2] = st.s;
    sh.before[wave] = before;
  }
  __syncthreads();
  before = 0;
  st.clear();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    st.join(Stat{sh.stat[w][0], sh.stat[w][1], sh.stat[w][2]});
    before += sh.before[w];
  }
}

/* A slice's piece of its row, for the row's last workgroup (device-coherent: aoship_device.h). */
__device__ __forceinline__ void publish(uint64_t *p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t collect(const uint64_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, a) | ((uint64_t)__builtin_bit_cast(uint32_t, b) << 32);
}
__device__ __forceinline__ float low(uint64_t v) { return __builtin_bit_cast(float, (uint32_t)v); }
__device__ __forceinline__ float high(uint64_t v) { return __builtin_bit_cast(float, (uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t slice_key(uint64_t k, int slice) {
  return (k & 0xffffffff00000000ull) | (uint32_t)~(uint32_t)slice;
}

/* Grid: rows times slices. A workgroup's slice of its row: elements in front of the first 16-byte border and behind the
 * last, one a thread, and the units between. */
template <bool BF16>
__global__ void __launch_bounds__(NT, 4) aos_logprobs_kernel(aos_logprobs_params p) {
  constexpr int N = Unit<BF16>::N, SIZE = 16 / N;
  constexpr int FLY = 2; /* units of a thread on their way while as many are worked on */
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const uint32_t wg = p.wg0 + blockIdx.x;
  const int row = (int)(wg / (uint32_t)p.slices), slice = (int)(wg - (uint32_t)row * (uint32_t)p.slices);
  const char *x = (const char *)p.logits + (long long)row * p.ld * SIZE;
  const int a0 = slice * p.span, a1 = a0 + p.span < p.vocab ? a0 + p.span : p.vocab;
  const int lead = (int)((16u - (uint32_t)((uintptr_t)(x + (long long)a0 * SIZE) & 15u)) & 15u) / SIZE;
  const int head = lead < a1 - a0 ? lead : a1 - a0; /* elements a0 .. a0 + head - 1 are before the first unit */
  const int u0 = a0 + head, units = (a1 - u0) / N, t0 = u0 + units * N; /* t0 .. a1 - 1 behind the last */
  const char *body = x + (long long)u0 * SIZE;

  const int t = p.targets ? p.targets[row] : -1;
  const bool target = t >= 0 && t < p.vocab;
  const float xt = target ? element<BF16>(x, t) : 0.0f;

  /* An element comes before the target if it is not <= edge: the target's logit, or behind it, where equal ones come first
   * (the target's own unit counts as behind it and is put right below), the next number under it; a NaN under -infinity,
   * so that everything comes before. */
  const float under = xt == -__builtin_inff() ? __builtin_nanf("") : next_under(xt);
  Stat st;
  st.clear();
  int before = 0, counted = 0; /* a lane's own, the wave's */
  const int each = (units + NT - 1) / NT, per = (each + SEGS - 1) / SEGS; /* units of a thread, of a group */
  const int full = units / NT;                                         /* units that every thread has */
  uint64_t key[SEGS];
#pragma unroll 1
  for (int g = 0; g < SEGS; ++g) {
    float best = __builtin_nanf("");
    uint32_t at = NONE;
    auto unit_max = [&](const Unit<BF16> &w, int u) {
      float um = w[0];
#pragma unroll
      for (int e = 1; e < N; ++e) um = fmaxf(um, w[e]);
      if (!(um <= best)) best = um, at = (uint32_t)u;
      return um;
    };
    const int i1 = (g + 1) * per < full ? (g + 1) * per : full;
    int i = g * per;
    Unit<BF16> w[FLY], next[FLY];
    auto fetch = [&](Unit<BF16> (&x)[FLY], int from) {
#pragma unroll
      for (int j = 0; j < FLY; ++j) x[j].w = aos_gld16(body + (long long)((from + j) * NT + tid) * 16);
    };
    if (i + FLY <= i1) fetch(w, i);
    for (; i + FLY <= i1; i += FLY) {
      if (i + 2 * FLY <= i1) fetch(next, i + FLY);
      float top = w[0][0];
#pragma unroll
      for (int j = 0; j < FLY; ++j) top = fmaxf(top, unit_max(w[j], (i + j) * NT + tid));
      st.lift(fmaxf(st.m, top));
#pragma unroll
      for (int j = 0; j < FLY; ++j) {
        const float edge = u0 + ((i + j) * NT + tid) * N + N <= t ? under : xt;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = w[j][e];
          st.add(v);
          counted += (int)__popcll(__ballot(!(v <= edge)));
        }
      }
#pragma unroll
      for (int j = 0; j < FLY; ++j) w[j] = next[j];
    }
    /* the group's last units, one at a time, and one that only some threads have */
    for (; i < (g + 1) * per; ++i) {
      const int u = i * NT + tid;
      if (u >= units) break;
      Unit<BF16> x;
      x.w = aos_gld16(body + (long long)u * 16);
      st.lift(fmaxf(st.m, unit_max(x, u)));
      const float edge = u0 + u * N + N <= t ? under : xt;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = x[e];
        st.add(v);
        before += !(v <= edge) ? 1 : 0;
      }
    }
    const uint64_t k = at == NONE ? 0 : key_of(best, at);
#pragma unroll
    for (int j = 0; j < SEGS; ++j) key[j] = j == g ? k : key[j];
  }
  if ((tid & 63) == 0) before += counted;
  /* elements outside the units: at most 2 (N - 1), thread i has the i-th */
  const int odd = tid < head ? a0 + tid : tid - head < a1 - t0 ? t0 + tid - head : -1;
  uint64_t mine = 0;
  if (odd >= 0) {
    const float v = element<BF16>(x, odd);
    st.lift(fmaxf(st.m, v));
    st.add(v);
    before += (v > xt) || (odd < t && v == xt) ? 1 : 0;
    mine = key_of(v, (uint32_t)odd);
  }
  if (tid == 0 && target && t >= u0 && t < t0)
    for (int i = t - (t - u0) % N; i < t; ++i) before += element<BF16>(x, i) == xt ? 1 : 0;
  join_block(sh, st, before);
  const int n = p.n_top;
  if (n > 0) {
    largest(sh, key, n);
    /* the last of the n groups' largest: nothing behind it (in value, then unit) is among the n */
    const uint64_t last = sh.top[n - 1];
    const float least = last ? key_value(last) : -__builtin_inff();
    int groups = 0;
    while (groups < n && sh.top[groups]) ++groups;
    /* each unit of the groups, 16 lanes a group */
    auto units_of_groups = [&](auto &&take) {
      for (int gi = tid / 16; gi < groups; gi += NT / 16) {
        const int u = (int)key_index(sh.top[gi]), th = u % NT, from = (u / NT) / per * per;
        for (int i = from + tid % 16; i < from + per; i += 16) {
          const int un = i * NT + th;
          if (un >= units) break;
          Unit<BF16> w;
          w.w = aos_gld16(body + (long long)un * 16);
          take(w, un);
        }
      }
    };
    units_of_groups([&](const Unit<BF16> &w, int un) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (w[e] >= least && key_of(w[e], (uint32_t)un) >= last) push(sh, key_of(w[e], (uint32_t)(u0 + un * N + e)));
    });
    if (mine) push(sh, mine);
    __syncthreads();
    if (sh.listed <= LIST) {
      rank_list(sh, n);
    } else {
      /* a list that overflows (groups full of large values): the n largest one after the other, each the largest below
       * the one before */
      uint64_t below = ~0ull, found = 0;
      for (int r = 0; r < n; ++r) {
        uint64_t best = mine < below ? mine : 0;
        units_of_groups([&](const Unit<BF16> &w, int un) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const uint64_t k = key_of(w[e], (uint32_t)(u0 + un * N + e));
            best = k < below && k > best ? k : best;
          }
        });
        best = wave_max(best);
        if ((tid & 63) == 0) sh.wave[tid >> 6] = best;
        __syncthreads();
        below = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) below = sh.wave[w] > below ? sh.wave[w] : below;
        if (tid == r) found = below;
        __syncthreads();
      }
      if (tid < n) sh.top[tid] = found;
      __syncthreads();
    }
  }
  if (p.slices == 1) {
    answer(p, sh, row, st, xt, target, before);
    return;
  }
  uint64_t *part = p.part + (size_t)wg * AOS_LOGPROBS_PART;
  if (tid == 0) {
    publish(part, pair(st.m, st.l));
    publish(part + 1, pair(st.s, __builtin_bit_cast(float, before)));
  }
  if (tid < n) publish(part + 2 + tid, sh.top[tid]);
  aos_mem_wait();
  __syncthreads();
  if (tid == 0) {
    const bool last = aos_arrive(p.counters + row) == (uint32_t)p.slices - 1u;
    if (last) aos_reset(p.counters + row);
    sh.listed = last ? 1u : 0u;
  }
  __syncthreads();
  if (!sh.listed) return;

  /* the row's last workgroup joins the slices' pieces: their n largest lie in the n slices whose largest come first */
  part = p.part + (size_t)row * p.slices * AOS_LOGPROBS_PART;
  st.clear();
  before = 0;
#pragma unroll
  for (int i = 0; i < SEGS; ++i) { /* (at most SEGS NT slices) */
    const int s = i * NT + tid;
    key[i] = 0;
    if (s < p.slices) {
      const uint64_t *q = part + (size_t)s * AOS_LOGPROBS_PART;
      const uint64_t ml = collect(q), sb = collect(q + 1), k = n > 0 ? collect(q + 2) : 0;
      st.join(Stat{low(ml), high(ml), low(sb)});
      before += __builtin_bit_cast(int, high(sb));
      /* a slice's place among slices: its largest's value, then the slice */
      if (k) key[i] = slice_key(k, s);
    }
  }
  __syncthreads(); /* (sh.listed has been read) */
  join_block(sh, st, before);
  if (n > 0) {
    largest(sh, key, n);
    const uint64_t last = sh.top[n - 1];
    for (int i = tid / 32; i < n && sh.top[i]; i += NT / 32) { /* (at most LIST keys) */
      if (tid % 32 >= n) break;
      const int s = (int)key_index(sh.top[i]);
      const uint64_t k = collect(part + (size_t)s * AOS_LOGPROBS_PART + 2 + tid % 32);
      if (k && slice_key(k, s) >= last) push(sh, k);
    }
    rank_list(sh, n);
  }
  answer(p, sh, row, st, xt, target, before);
}

template <bool BF16>
int launch(const aos_logprobs_params *p, const aos_launch_ctx *ctx) {
  const uint32_t wgs = (uint32_t)p->T * (uint32_t)p->slices;
  aos_logprobs_params a = *p;
  for (a.wg0 = 0; a.wg0 < wgs; a.wg0 += AOS_LAUNCH_PIECE(wgs - a.wg0)) {
    AOS_LAUNCH(ctx, (aos_logprobs_kernel<BF16>), dim3(AOS_LAUNCH_PIECE(wgs - a.wg0)), dim3(NT), 0, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

}  // namespace

static_assert(AOS_LOGPROBS_MAX_TOP <= 32 && AOS_LOGPROBS_MAX_TOP * AOS_LOGPROBS_MAX_TOP <= LIST, "lists");
static_assert(AOS_LOGPROBS_MAX_SLICES <= SEGS * NT, "a thread takes SEGS slices");

/* Slices of a row: as many as give the rows 512 workgroups, of at least 2048 elements. A workgroup's choice of candidates
 * costs as much as reading some 10000 elements: 64 rows of 128256 with 20 of them 36 us in 1024 workgroups, 24.5 in 512,
 * 25.4 in 256. */
extern "C" void aos_logprobs_shape(int T, int vocab, int *slices, int *span) {
  long long s = T > 0 ? (512 + T - 1) / T : 1;
  if (s > vocab / 2048) s = vocab / 2048;
  if (s > AOS_LOGPROBS_MAX_SLICES) s = AOS_LOGPROBS_MAX_SLICES;
  if (s < 1) s = 1;
  /* (whole 64-byte lines of either type, so that aligned rows have aligned slices) */
  const long long per = ((vocab + s - 1) / s + 31) / 32 * 32;
  *span = (int)(s == 1 ? vocab : per);
  *slices = (int)(s == 1 ? 1 : (vocab + per - 1) / per);
}

extern "C" int aos_launch_logprobs(const aos_logprobs_params *p, const aos_launch_ctx *ctx) {
  return p->bf16 ? launch<true>(p, ctx) : launch<false>(p, ctx);
}
