#pragma once
// Device-side view of ragged sequences in a paged cache: lengths and page ids are device data and are bounded here, so
// that no value of theirs makes a kernel read or write outside the arrays it was given. What is out of range is recorded
// in the status word (PHANTOM_ATTN_STATUS_PAGE).
#include "paged.h"
#include "sm100_ptx.cuh"

namespace phantom {

// One sequence: its first packed token, new tokens, cached tokens within its row of the page table, and the position of
// its first new token. Token i of the new ones is at off + i, whatever had to be bounded; there may be no place for it.
struct Seq {
  int tok0, n, len, off;
};

__device__ __forceinline__ Seq seq_of(const PagedSeqs& s, int b) {
  const int c0 = s.cu_new[b], c1 = s.cu_new[b + 1], len = s.kv_lens[b];
  const long long room = (long long)s.width << s.page_log2;
  Seq x;
  x.tok0 = min(max(c0, 0), s.total);
  x.n = min(max(c1, x.tok0), s.total) - x.tok0;
  x.len = (int)min((long long)max(len, 0), min(room, 0x7ffff000LL));
  x.off = (int)max((long long)min(len, 0x7fff0000) - ((long long)c1 - x.tok0), -0x7fffffffLL);
  if (x.tok0 != c0 || x.tok0 + x.n != c1 || x.len != len) atomicOr(s.status, PHANTOM_ATTN_STATUS_PAGE);
  return x;
}

// Page id of entry i of sequence b; -1 where there is none.
__device__ __forceinline__ int page_of(const PagedSeqs& s, int b, int i) {
  int id = (unsigned)i < (unsigned)s.width ? s.table[(long long)b * s.table_stride + i] : -1;
  if ((unsigned)id >= (unsigned)s.num_pages) {
    atomicOr(s.status, PHANTOM_ATTN_STATUS_PAGE);
    id = -1;
  }
  return id;
}

// Sequence of packed token `tok` (whole warp, one token): how many sequences end at or before it.
__device__ __forceinline__ int seq_index(const PagedSeqs& s, int tok) {
  const int lane = threadIdx.x & 31;
  int b = 0;
  for (int i0 = 0; i0 < s.batch; i0 += 32) {
    const int i = i0 + lane;
    b += __popc(__ballot_sync(0xffffffffu, i < s.batch && s.cu_new[min(i, s.batch - 1) + 1] <= tok));
  }
  return b;
}

// Zeroes the rows of packed tokens that belong to no sequence: those from cu_new[batch] on (a captured call's unused ones,
// nothing wrong) and those before cu_new[0], which has to be 0. `row`: 16-byte pieces of a token. Worker `me` of `n`.
__device__ __forceinline__ void zero_unowned(const PagedSeqs& s, void* o, int row, long long me, long long n) {
  const int first = min(max(s.cu_new[0], 0), s.total), last = max(min(max(s.cu_new[s.batch], 0), s.total), first);
  if (me == 0 && s.cu_new[0] != 0) atomicOr(s.status, PHANTOM_ATTN_STATUS_PAGE);
  const long long lead = (long long)first * row, skip = (long long)last * row - lead, count = (long long)s.total * row - skip;
  for (long long i = me; i < count; i += n) static_cast<uint4*>(o)[i < lead ? i : i + skip] = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------ even shares of work
// An attention call's work: units (sequence, key head, block of query rows) in a row, each of as many tiles of keys as its
// rows see. CTA c of G takes the tiles [c W / G, (c + 1) W / G) of all W, so a unit may be shared by several CTAs.
// `Blocks` says how the rows are cut: kTile keys to a tile; count(x) blocks; the keys key_end(x, blk) that a block sees;
// head_tiles(x) tiles in all of one head. A unit costs something besides its tiles (its queries, its output, the start of
// its pipeline), as much as kUnit tiles; these are counted before its first one when the shares are cut, and a share that
// ends among them has nothing of the unit. Joining a shared unit costs as much as kJoin tiles, and kPart tiles for each part.

// At least one tile, so that rows without any key are written too (as zeros).
template <typename Blocks>
__device__ __forceinline__ int tiles_of(const Blocks& k, const Seq& x, int blk) {
  return max(1, (k.key_end(x, blk) + Blocks::kTile - 1) / Blocks::kTile);
}
// Tiles of one head, the units' own costs counted.
template <typename Blocks>
__device__ __forceinline__ long long head_work(const Blocks& k, const Seq& x) {
  return k.head_tiles(x) + (long long)k.count(x) * Blocks::kUnit;
}
template <typename Blocks>
__device__ __forceinline__ long long sum_tiles(const Blocks& k, const Seq& x) {
  long long w = 0;
  for (int i = k.count(x) - 1; i >= 0; --i) w += tiles_of(k, x, i);
  return w;
}

// A whole warp walks one CTA's share; every value is uniform over the warp. Positions count tiles and units' own costs.
// Lengths and offsets are read more than once, and a caller may (by mistake) have them change meanwhile: whatever the reads
// give, the walk ends, and its units, blocks and owners are ones that exist.
template <typename Blocks>
struct Walk {
  static constexpr int kUnit = Blocks::kUnit;
  long long share, at, end;  // at: where the unit begins; end: where the share does
  int more, ctas;            // CTA c has share + (c < more); CTAs that have any
  bool by_unit;              // or CTA c has the unit c
  Seq x;
  int b, h, blk, nt;         // the unit, its tiles
  int tile, cnt;             // the first of them here, how many are; 0 at the end of the share

  __device__ static long long scan(long long w, int lane) {
    for (int m = 1; m < 32; m <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, w, m);
      if (lane >= m) w += y;
    }
    return w;
  }
  __device__ static long long quotient(long long a, long long b) {  // 64-bit division is a long call
    return a <= 0x7fffffffLL && b <= 0x7fffffffLL ? (long long)((unsigned)a / (unsigned)b) : a / b;
  }
  __device__ void start(const PagedSeqs& s, const Blocks& k, int cta, int grid) {
    const int lane = threadIdx.x & 31;
    // Whole units, one to a CTA, where that takes no more than kJoin tiles longer than even shares. A head's last block sees
    // the most keys.
    long long w = 0, total = 0;
    unsigned units = 0, units0 = 0;  // (of a lane's sequence among the first 32; kept within 32 bits, the grid is smaller)
    int most = 0;
    for (int i0 = 0; i0 < s.batch; i0 += 32) {
      long long y = 0;
      unsigned u = 0;
      if (i0 + lane < s.batch) {
        const Seq q = seq_of(s, i0 + lane);
        const int c = k.count(q);
        y = (k.head_tiles(q) + (long long)c * kUnit) * s.heads;
        u = (unsigned)min((long long)c * s.heads, 1LL << 20);
        if (c > 0) most = max(most, tiles_of(k, q, c - 1));
      }
      const long long z = scan(y, lane);
      if (i0 == 0) w = z, units0 = u;  // (up to 32 sequences: one scan gives the total and the place)
      total += __shfl_sync(0xffffffffu, z, 31);
      units = min(units + __reduce_add_sync(0xffffffffu, u), 1u << 30);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    // No smaller shares than pay: with s tiles to a share the longest unit takes as long as s tiles and most / s parts to
    // join, kPart tiles each, least where s^2 = kPart most.
    const long long least = max(1LL, (long long)sqrtf(Blocks::kPart * (float)most));
    ctas = (int)min((long long)grid, quotient(total + least - 1, least));
    share = ctas > 0 ? quotient(total, ctas) : 0;
    more = (int)(total - share * ctas);
    by_unit = units <= (unsigned)grid && most + kUnit <= share + Blocks::kJoin;
    if (by_unit) ctas = (int)units;
    cnt = 0;
    if (cta >= ctas) return;
    // the place of the share's beginning, or of the CTA's unit, among all
    const long long pos = by_unit ? cta : first(cta);
    auto seq_part = [&](int i) {
      if (i >= s.batch) return 0LL;
      const Seq q = seq_of(s, i);
      return by_unit ? (long long)k.count(q) * s.heads : head_work(k, q) * s.heads;
    };
    if (by_unit) w = scan(units0, lane);
    long long before = 0;
    for (int i0 = 0;; i0 += 32) {
      if (i0 >= s.batch) return;
      if (i0 > 0) w = scan(seq_part(i0 + lane), lane);
      const unsigned past = __ballot_sync(0xffffffffu, before + w > pos);
      if (past) {
        const int l = __ffs(past) - 1;
        const long long up_to = __shfl_sync(0xffffffffu, w, max(l - 1, 0));
        b = i0 + l;
        before += l > 0 ? up_to : 0;
        break;
      }
      before += __shfl_sync(0xffffffffu, w, 31);
    }
    x = seq_of(s, b);
    const int count = k.count(x);
    if (count == 0) return;
    const long long head = by_unit ? count : head_work(k, x);
    long long r = pos - before;
    if (r >= head * s.heads) return;
    h = (int)quotient(r, head);
    r -= h * head;
    blk = 0;
    if (by_unit) {
      blk = (int)r;
      r = 0;
    }
    for (int i0 = 0; !by_unit && count > 1; i0 += 32) {
      if (i0 >= count) return;
      const int y = i0 + lane < count ? tiles_of(k, x, i0 + lane) + kUnit : 0;
      w = scan(y, lane);
      const unsigned past = __ballot_sync(0xffffffffu, w > r);
      if (past) {
        const int l = __ffs(past) - 1;
        const long long up_to = __shfl_sync(0xffffffffu, w, max(l - 1, 0));
        blk = i0 + l;
        r -= l > 0 ? up_to : 0;
        break;
      }
      r -= __shfl_sync(0xffffffffu, w, 31);
    }
    nt = tiles_of(k, x, blk);
    at = by_unit ? 0 : pos - r;
    end = by_unit ? nt + kUnit : first(cta + 1);
    tile = max(0, (int)r - kUnit);
    cnt = (int)min((long long)nt, end - at - kUnit) - tile;
  }
  // Where a CTA's share begins (even shares).
  __device__ long long first(int cta) const { return cta * share + min(cta, more); }
  // The first and the last CTA that have tiles of the unit, the caller being CTA `cta`.
  __device__ int2 owners(int cta) const {
    return by_unit ? make_int2(cta, cta) : make_int2(owner(at + kUnit), owner(at + kUnit + nt - 1));
  }
  __device__ int owner(long long pos) const {
    const long long big = more * (share + 1);
    return (int)min(pos < big ? quotient(pos, share + 1) : more + quotient(pos - big, share), ctas - 1LL);
  }
  // A unit that several CTAs share: CTA c's part of it lies in the place 2 c + 1 if its first tile is c's, else 2 c.
  __device__ static int place(int cta, bool begins) { return 2 * cta + (begins ? 1 : 0); }
  __device__ void advance(const PagedSeqs& s, const Blocks& k) {
    at += nt + kUnit;
    cnt = 0;
    if (at >= end) return;
    if (++blk == k.count(x)) {
      blk = 0;
      if (++h == s.heads) {
        h = 0;
        do {
          if (++b >= s.batch) return;
          x = seq_of(s, b);
        } while (x.n == 0);
      }
    }
    nt = tiles_of(k, x, blk);
    tile = 0;
    cnt = (int)max(0LL, min((long long)nt, end - at - kUnit));
  }
};

// The parts of a shared unit are joined by the CTA that arrives last. Each unit has a 64-bit word: the call's number (unique
// in the process; its last kCountBits dropped) and how many parts are in memory. It needs no initialisation: what a pool's
// memory held before does not equal the number, and the first to arrive puts the number there. An arrival on the old value
// counts for nothing, so whoever made one starts over once the number is there; each CTA changes the word at most twice
// before that, which bounds the loop. The last one leaves 0, for a call replayed from a graph has the same number each time.
// (A flag for each part, set and then all of them read past a fence.sc, took 3200 cycles.)
constexpr int kCountBits = 12;
__device__ __forceinline__ unsigned long long atom_add64(unsigned long long* word, unsigned long long y) {
  unsigned long long old;
  asm volatile("atom.add.acq_rel.gpu.global.u64 %0, [%1], %2;" : "=l"(old) : "l"(word), "l"(y) : "memory");
  return old;
}
__device__ __forceinline__ unsigned long long atom_cas64(unsigned long long* word, unsigned long long from, unsigned long long to) {
  unsigned long long old;
  asm volatile("atom.cas.acq_rel.gpu.global.b64 %0, [%1], %2, %3;" : "=l"(old) : "l"(word), "l"(from), "l"(to) : "memory");
  return old;
}
// One thread, whose CTA's part is written (and seen by this thread): is it the last of `parts` > 1?
__device__ __forceinline__ bool last_part(unsigned long long* word, unsigned long long call, int parts) {
  const unsigned long long tag = call >> kCountBits;
  unsigned long long old = atom_add64(word, 1);
  if (old >> kCountBits != tag) {
    for (unsigned long long seen = old + 1;;) {
      const unsigned long long y = atom_cas64(word, seen, tag << kCountBits | 1);
      if (y == seen) return false;  // the first
      if (y >> kCountBits == tag) break;
      seen = y;
    }
    old = atom_add64(word, 1);
  }
  const bool last = (int)(old & ((1 << kCountBits) - 1)) + 1 == parts;
  if (last) *word = 0;
  return last;
}

// ------------------------------------------------------------------------------------------------ copies, 8-bit values
// Untiled bulk copy into shared memory (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2, int c3,
                                            int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}
// A value's scale, at least what paged_append writes (log2 and the reciprocal stay in range); a NaN stays one.
__device__ __forceinline__ float least_scale(float x) { return x < 0x1p-100f ? 0x1p-100f : x; }

// Two signed bytes of w (chosen by sel: result bytes [lo, 4, hi, 4], byte 4 = 0x64) as exact fp16 pairs; w already has its
// sign bits flipped, so a byte u = b + 128 gives the fp16 number 1024 + u.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_f16(uint32_t w) {
  const uint32_t r = __byte_perm(w, 0x64646464u, SEL);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&x);
}
// Two signed bytes as exact bf16 pairs (SEL: result bytes [lo, 0, hi, 0]): with sign bit s and low bits u, 128 + u and
// 128 + 128 s are both bf16 numbers, and b is their difference.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_bf16(uint32_t w) {
  const uint32_t r = __byte_perm(w, 0, SEL);
  const uint32_t lo = (r & 0x007F007Fu) | 0x43004300u, hi = (r & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&hi));
  return *reinterpret_cast<const uint32_t*>(&x);
}

}  // namespace phantom
