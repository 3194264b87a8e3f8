/*
 * aoship_kv.h — the layout of the paged key/value cache and what its kernels share.
 *
 * Keys and values of one head are kept in tiles of 64 positions, in the order in which the matrix cores take
 * them, so that attention loads its operands as they lie (the contraction runs over dimensions for the keys and
 * over positions for the values):
 *
 *   keys    units of 16 bytes = U consecutive dimensions of one position (U = 8 bfloat16, 16 8-bit or 32 4-bit
 *           codes), [unit of dimensions][64 positions]
 *   values  units of 16 consecutive positions of one dimension (32, 16 or 8 bytes; bfloat16 in two pieces of 8
 *           positions): bfloat16 [8 pieces][dimension][8], quantised [4 units][dimension][16]
 *   scales  (quantised) a byte per position and block of 32 dimensions, 2^(byte - 127), 255 = not a number (its
 *           codes are then zeros): keys [block][swapped position], values [block][position]. The key bytes swap
 *           the two low and the next two bits of the position within 16, so that the four positions 4 apart that a
 *           lane's key rows have (rows 4 j + i of four 16-row blocks) are one word.
 *
 * The dimensions from head_dim to the padded hdp (64, 128 or 256) hold zeros.
 */
#ifndef AOSHIP_KV_H
#define AOSHIP_KV_H

#include "aoship_device.h"

namespace kv {

constexpr int TILE = 64; /* positions of a tile */

template <int FMT>
constexpr int bits() {
  return FMT == AOS_KV_BF16 ? 16 : FMT == AOS_KV_MXFP8 ? 8 : 4;
}
template <int FMT, int HDP>
constexpr int k_bytes() {
  return TILE * HDP * bits<FMT>() / 8;
}
template <int FMT, int HDP>
constexpr int scale_bytes() { /* of the keys or of the values */
  return FMT == AOS_KV_BF16 ? 0 : TILE * HDP / 32;
}
template <int FMT, int HDP>
constexpr int tile_bytes() {
  return 2 * (k_bytes<FMT, HDP>() + scale_bytes<FMT, HDP>());
}
/* offsets in a tile: keys 0, values, key scales, value scales */
template <int FMT, int HDP>
constexpr int v_off() {
  return k_bytes<FMT, HDP>();
}
template <int FMT, int HDP>
constexpr int ks_off() {
  return 2 * k_bytes<FMT, HDP>();
}
template <int FMT, int HDP>
constexpr int vs_off() {
  return ks_off<FMT, HDP>() + scale_bytes<FMT, HDP>();
}

/* whether a word of two bfloat16 holds an infinity or a NaN */
__device__ __forceinline__ bool odd2(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

/* byte of a position's key scale within its block's 64 */
__device__ __forceinline__ int ks_index(int pos) { return (pos & 48) | ((pos & 3) << 2) | ((pos >> 2) & 3); }

template <int FMT, int HDP>
__device__ __forceinline__ unsigned char *tile_ptr(const aos_kv_batch &b, int page, int head, int pos) {
  const int tpp = 1 << (b.page_shift - 6);
  const long long t = ((long long)page * b.nkv + head) * tpp + ((pos & ((1 << b.page_shift) - 1)) >> 6);
  return b.pool + t * tile_bytes<FMT, HDP>();
}

/* A sequence of a batch: its first row, its new rows and its positions (the new ones the last). */
struct Seq {
  int row0, count, len;
};

/* notes a fault in the cache's word (on the host, where tests walk a batch, in an ordinary one) */
__host__ __device__ __forceinline__ void note(uint32_t *faults, uint32_t bits) {
#ifdef __HIP_DEVICE_COMPILE__
  __hip_atomic_fetch_or(faults, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#else
  *faults |= bits;
#endif
}

/* What the caller's device arrays say of sequence s, refused (no rows, the fault noted) where it does not fit the
 * sizes that the launch was made for: nothing below indexes with a value that was not checked here. */
__host__ __device__ __forceinline__ Seq seq_of(const aos_kv_batch &b, int r0, int r1, int len) {
  Seq q;
  q.row0 = r0;
  q.count = r1 - r0;
  q.len = len;
  const bool ok = r0 >= 0 && r1 >= r0 && r1 <= b.n_tokens && r1 - r0 <= b.max_new && len >= 0 && len <= b.max_len;
  if (!ok) {
    q.row0 = q.count = q.len = 0;
    note(b.faults, AOS_KV_FAULT_BATCH);
  }
  return q;
}
__device__ __forceinline__ Seq seq_at(const aos_kv_batch &b, int s) {
  return seq_of(b, b.starts[s], b.starts[s + 1], b.lens[s]);
}

/* What the table says of the page that holds a position (0 <= pos < max_len, which the table covers). */
__device__ __forceinline__ int page_entry(const aos_kv_batch &b, int s, int pos) {
  return b.pages[(long long)s * b.stride + (pos >> b.page_shift)];
}
/* The page of a position that a launch reads or writes, or -1 where the table's entry is none. */
__device__ __forceinline__ int page_checked(const aos_kv_batch &b, int page) {
  if ((unsigned)page < (unsigned)b.num_pages) return page;
  note(b.faults, AOS_KV_FAULT_PAGE);
  return -1;
}
__device__ __forceinline__ int page_of(const aos_kv_batch &b, int s, int pos) {
  return page_checked(b, page_entry(b, s, pos));
}

/* Blocks of 16 positions, aligned in their sequence, that a batch's new rows can touch: sequence s has its blocks
 * from number block_base(s) on (count / 16 + 2 of them at most); one each where every sequence has one row. */
__host__ __device__ __forceinline__ int block_base(int max_new, int s, int start) {
  return max_new == 1 ? s : (start >> 4) + 2 * s;
}
inline int blocks_of(int max_new, int n_seqs, int n_tokens) {
  return max_new == 1 ? n_seqs : n_tokens / 16 + 2 * n_seqs;
}

/* Block number x of a sequence: its first position and the rows of it that are new: positions [lo, hi) of the 16. */
struct Block {
  int seq, pos, lo, hi, row; /* row: the batch row of position pos + lo */
};
__host__ __device__ __forceinline__ bool block_of(int max_new, int s, const Seq &q, int x, Block &o) {
  const int first = q.len - q.count, lo = first > 0 ? first : 0; /* (rows before position 0 are not kept) */
  const int pos = (lo & ~15) + 16 * (x - block_base(max_new, s, q.row0));
  if (q.count == 0 || pos >= q.len || pos + 16 <= lo) return false;
  o.seq = s;
  o.pos = pos;
  o.lo = lo > pos ? lo - pos : 0;
  o.hi = q.len - pos < 16 ? q.len - pos : 16;
  o.row = q.row0 + pos + o.lo - first;
  return true;
}

/* The same for block x of the whole batch, its sequence searched for (by each wave). False where there is none;
 * uniform over the workgroup. */
__device__ __forceinline__ bool block_at(const aos_kv_batch &b, int x, int lane, Block &o) {
  int s = x;
  if (b.max_new != 1) {
    int below = 0; /* sequences whose blocks begin at or before x */
    for (int s0 = 0; s0 < b.n_seqs; s0 += 64) {
      const int i = s0 + lane;
      const bool yes = i < b.n_seqs && block_base(b.max_new, i, b.starts[i]) <= x;
      const int n = (int)__popcll(__ballot(yes));
      below += n;
      if (n < 64) break;
    }
    s = below - 1;
    if (s < 0) return false;
  }
  s = __builtin_amdgcn_readfirstlane(s);
  return block_of(b.max_new, s, seq_at(b, s), x, o);
}

}  // namespace kv

#endif
