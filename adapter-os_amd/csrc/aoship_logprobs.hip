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
 * goes to a list (about n entries), and an entry's place in the answer is the number of entries before it.
 *
 * Bound by reading the logits once.
 */
#include "aoship_device.h"
#include "aoship_internal.h"
#include <hip/hip_ext.h>

namespace {

constexpr int NT = 256;         /* threads of a workgroup */
constexpr int SEGS = 4;         /* groups of a thread */
constexpr int LIST = 1024;      /* entries of the list */
constexpr float LEAST = -3.40282347e38f;
constexpr float LOG2E = 1.44269504f;
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

__device__ __forceinline__ uint64_t wave_max(uint64_t k) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = aos_shfl64(k, (int)(threadIdx.x & 63) ^ d);
    k = o > k ? o : k;
  }
  return k;
}

/* running maximum, sum and weighted sum */
struct Stat {
  float m, l, s;
  __device__ __forceinline__ void clear() { m = LEAST, l = 0.0f, s = 0.0f; }
  __device__ __forceinline__ void lift(float top) { /* to a maximum that is no less */
    const float d = m - top, f = __builtin_amdgcn_exp2f(d * LOG2E);
    s = f * (s + l * fmaxf(d, -200.0f)); /* (below that f is zero: no zero times infinity) */
    l = l * f;
    m = top;
  }
  __device__ __forceinline__ void add(float x) { /* x <= m */
    const float d = x - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
    l = l + e;
    s = s + e * fmaxf(d, -200.0f);
  }
  __device__ __forceinline__ void join(Stat o) {
    const float top = fmaxf(m, o.m);
    lift(top);
    o.lift(top);
    l = l + o.l;
    s = s + o.s;
  }
};

struct Shared {
  uint64_t list[LIST];
  uint64_t wave[4][AOS_LOGPROBS_MAX_TOP];
  uint64_t top[AOS_LOGPROBS_MAX_TOP];
  float stat[4][3];
  int before[4];
  uint32_t listed;
};

/* The n largest of all threads' four keys, in order, into sh.top (zeros where there are fewer). */
__device__ __forceinline__ void largest(Shared &sh, uint64_t (&k)[4], int n) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto order = [](uint64_t &a, uint64_t &b) {
    const uint64_t hi = a > b ? a : b, lo = a > b ? b : a;
    a = hi;
    b = lo;
  };
  order(k[0], k[1]);
  order(k[2], k[3]);
  order(k[0], k[2]);
  order(k[1], k[3]);
  order(k[1], k[2]);
  for (int i = 0; i < n; ++i) {
    const uint64_t best = wave_max(k[0]);
    if (lane == 0) sh.wave[wave][i] = best;
    if (k[0] == best) k[0] = k[1], k[1] = k[2], k[2] = k[3], k[3] = 0; /* (keys are distinct, zeros apart) */
  }
  __syncthreads();
  if (wave == 0) {
    uint64_t a = lane < n ? sh.wave[0][lane] : lane >= 32 && lane - 32 < n ? sh.wave[1][lane - 32] : 0;
    uint64_t b = lane < n ? sh.wave[2][lane] : lane >= 32 && lane - 32 < n ? sh.wave[3][lane - 32] : 0;
    order(a, b);
    for (int i = 0; i < n; ++i) {
      const uint64_t best = wave_max(a);
      if (lane == 0) sh.top[i] = best;
      if (a == best) a = b, b = 0;
    }
  }
  __syncthreads();
}

/* The n first of the list's entries into sh.top: each entry counts those before it. */
__device__ __forceinline__ void rank_list(Shared &sh, int n) {
  const int count = (int)sh.listed;
  if ((int)threadIdx.x < n) sh.top[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += NT) {
    const uint64_t mine = sh.list[i];
    int before = 0;
    for (int j = 0; j < count; ++j) before += sh.list[j] > mine ? 1 : 0;
    if (before < n) sh.top[before] = mine;
  }
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

/* what a workgroup writes of a row: the answer, or its slice's piece of it */
__device__ __forceinline__ void answer(const aos_logprobs_params &p, Shared &sh, int row, Stat st, float xt, bool target,
                                       int before) {
  const int tid = threadIdx.x;
  const float ln = logf(st.l), nan = __builtin_nanf("");
  const bool ok = st.l > 0.0f; /* neither a NaN nor all minus infinity */
  if (tid == 0) {
    if (p.logprob) p.logprob[row] = ok && target ? xt - st.m - ln : nan;
    if (p.rank) p.rank[row] = ok && target ? before : -1;
    if (p.entropy) p.entropy[row] = ok ? ln - st.s / st.l : nan;
  }
  if (tid < p.n_top) {
    const uint64_t k = sh.top[tid];
    const long long at = (long long)row * p.n_top + tid;
    if (p.top_ids) p.top_ids[at] = ok ? (int)key_index(k) : -1;
    if (p.top_logprobs) p.top_logprobs[at] = ok ? key_value(k) - st.m - ln : nan;
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

/* Grid: rows times slices. A workgroup's slice of its row: elements in front of the first 16-byte border and behind the
 * last, one a thread, and the units between. */
template <bool BF16>
__global__ void __launch_bounds__(NT) aos_logprobs_kernel(aos_logprobs_params p) {
  constexpr int N = Unit<BF16>::N, SIZE = 16 / N;
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const int row = (int)(blockIdx.x / (uint32_t)p.slices), slice = (int)(blockIdx.x - (uint32_t)row * (uint32_t)p.slices);
  const char *x = (const char *)p.logits + (long long)row * p.ld * SIZE;
  const int a0 = slice * p.span, a1 = a0 + p.span < p.vocab ? a0 + p.span : p.vocab;
  const int lead = (int)((16u - (uint32_t)((uintptr_t)(x + (long long)a0 * SIZE) & 15u)) & 15u) / SIZE;
  const int head = lead < a1 - a0 ? lead : a1 - a0; /* elements a0 .. a0 + head - 1 are before the first unit */
  const int u0 = a0 + head, units = (a1 - u0) / N, t0 = u0 + units * N; /* t0 .. a1 - 1 behind the last */
  const char *body = x + (long long)u0 * SIZE;

  const int t = p.targets ? p.targets[row] : -1;
  const bool target = t >= 0 && t < p.vocab;
  const float xt = target ? element<BF16>(x, t) : 0.0f;

  Stat st;
  st.clear();
  int before = 0;
  const int each = (units + NT - 1) / NT, per = (each + SEGS - 1) / SEGS; /* units of a thread, of a group */
  uint64_t key[SEGS];
#pragma unroll
  for (int g = 0; g < SEGS; ++g) {
    float best = __builtin_nanf("");
    uint32_t at = NONE;
    for (int i0 = g * per; i0 < (g + 1) * per; i0 += 4) {
      Unit<BF16> w[4];
      int live = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int u = (i0 + j) * NT + tid;
        const bool in = i0 + j < (g + 1) * per && u < units;
        if (in) w[j].w = aos_gld16(body + (long long)u * 16);
        live += in ? 1 : 0; /* (the first so many) */
      }
      float top = st.m;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= live) continue;
        float um = w[j][0];
#pragma unroll
        for (int e = 1; e < N; ++e) um = fmaxf(um, w[j][e]);
        if (!(um <= best)) best = um, at = (uint32_t)((i0 + j) * NT + tid);
        top = fmaxf(top, um);
      }
      st.lift(top);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= live) continue;
        const int i = u0 + ((i0 + j) * NT + tid) * N;
        const bool front = i + N <= t; /* (the unit that holds t: counted as behind it, put right below) */
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = w[j][e];
          st.add(v);
          before += (v > xt) || (front && v == xt) ? 1 : 0;
        }
      }
    }
    key[g] = at == NONE ? 0 : key_of(best, at);
  }
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
    if (tid == 0) sh.listed = 0;
    largest(sh, key, n);
    /* the last of the n groups' largest: nothing behind it (in value, then unit) is among the n */
    const uint64_t last = sh.top[n - 1];
    int groups = 0;
    while (groups < n && sh.top[groups]) ++groups;
    auto wanted = [&](float v, uint32_t unit) { return key_of(v, unit) >= last; };
    auto push = [&](uint64_t k) {
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < LIST) sh.list[at] = k;
    };
    auto unit_of = [&](int q) { /* of the q-th unit of the groups; -1 past the row's end */
      const int gi = q / per, i = q - gi * per;
      const uint32_t u = key_index(sh.top[gi]);
      const int th = (int)(u % NT), g = (int)(u / NT) / per;
      const int un = (g * per + i) * NT + th;
      return un < units ? un : -1;
    };
    for (int q = tid; q < groups * per; q += NT) {
      const int un = unit_of(q);
      if (un < 0) continue;
      Unit<BF16> w;
      w.w = aos_gld16(body + (long long)un * 16);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (wanted(w[e], (uint32_t)un)) push(key_of(w[e], (uint32_t)(u0 + un * N + e)));
    }
    if (mine) push(mine);
    __syncthreads();
    if (sh.listed <= LIST) {
      rank_list(sh, n);
    } else {
      /* a list that overflows (groups full of large values): the n largest one after the other, each the largest below
       * the one before */
      uint64_t below = ~0ull, found = 0;
      for (int r = 0; r < n; ++r) {
        uint64_t best = mine < below ? mine : 0;
        for (int q = tid; q < groups * per; q += NT) {
          const int un = unit_of(q);
          if (un < 0) continue;
          Unit<BF16> w;
          w.w = aos_gld16(body + (long long)un * 16);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const uint64_t k = key_of(w[e], (uint32_t)(u0 + un * N + e));
            best = k < below && k > best ? k : best;
          }
        }
        best = wave_max(best);
        if ((tid & 63) == 0) sh.wave[tid >> 6][0] = best;
        __syncthreads();
        below = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) below = sh.wave[w][0] > below ? sh.wave[w][0] : below;
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
  float *part = p.part + (size_t)blockIdx.x * AOS_LOGPROBS_PART;
  if (tid == 0) {
    part[0] = st.m;
    part[1] = st.l;
    part[2] = st.s;
    ((int *)part)[3] = before;
  }
  if (tid < n) ((uint64_t *)(part + 4))[tid] = sh.top[tid];
}

/* Grid: rows. The slices' pieces joined: their n largest lie in the n slices whose largest come first. */
template <bool BF16>
__global__ void __launch_bounds__(NT) aos_logprobs_join_kernel(aos_logprobs_params p) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, row = blockIdx.x, n = p.n_top;
  const float *part = p.part + (size_t)row * p.slices * AOS_LOGPROBS_PART;
  auto keys = [&](int slice) { return (const uint64_t *)(part + (size_t)slice * AOS_LOGPROBS_PART + 4); };
  Stat st;
  st.clear();
  int before = 0;
  uint64_t key[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { /* (at most 4 NT slices) */
    const int s = i * NT + tid;
    key[i] = 0;
    if (s < p.slices) {
      const float *q = part + (size_t)s * AOS_LOGPROBS_PART;
      st.join(Stat{q[0], q[1], q[2]});
      before += ((const int *)q)[3];
      /* a slice's rank among slices: its largest's value, then the slice */
      if (n > 0 && keys(s)[0]) key[i] = (keys(s)[0] & 0xffffffff00000000ull) | (uint32_t)~(uint32_t)s;
    }
  }
  join_block(sh, st, before);
  if (n > 0) {
    if (tid == 0) sh.listed = 0;
    largest(sh, key, n);
    const uint64_t last = sh.top[n - 1];
    for (int q = tid; q < n * n; q += NT) { /* (at most LIST) */
      if (!sh.top[q / n]) continue;
      const uint32_t s = key_index(sh.top[q / n]);
      const uint64_t k = keys((int)s)[q % n];
      if (k && ((k & 0xffffffff00000000ull) | (uint32_t)~s) >= last) sh.list[atomicAdd(&sh.listed, 1u)] = k;
    }
    __syncthreads();
    rank_list(sh, n);
  }
  const char *x = (const char *)p.logits + (long long)row * p.ld * (BF16 ? 2 : 4);
  const int t = p.targets ? p.targets[row] : -1;
  const bool target = t >= 0 && t < p.vocab;
  answer(p, sh, row, st, target ? element<BF16>(x, t) : 0.0f, target, before);
}

template <bool BF16>
int launch(const aos_logprobs_params *p, const aos_launch_ctx *ctx) {
  AOS_LAUNCH(ctx, (aos_logprobs_kernel<BF16>), dim3((uint32_t)p->T * (uint32_t)p->slices), dim3(NT), 0, *p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p->slices == 1) return (int)e;
  AOS_LAUNCH(ctx, (aos_logprobs_join_kernel<BF16>), dim3(p->T), dim3(NT), 0, *p);
  return (int)hipGetLastError();
}

}  // namespace

static_assert(AOS_LOGPROBS_MAX_TOP <= 32 && AOS_LOGPROBS_MAX_TOP * AOS_LOGPROBS_MAX_TOP <= LIST, "lists");
static_assert(AOS_LOGPROBS_MAX_SLICES <= 4 * NT, "a thread takes four slices");

/* Slices of a row: one where there are rows enough to fill the chip with a workgroup each (eight a CU), else as many as
 * do, of at least 2048 elements. */
extern "C" void aos_logprobs_shape(int T, int vocab, int *slices, int *span) {
  long long s = T > 0 ? AOS_LOGPROBS_WGS / T : 1;
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
