// Attention of few query rows over a paged cache (decoding; a few new tokens). For sequence b with n new and len cached
// tokens (the new ones among them), key head h, its `group` query heads, and new token i:
//
//   o[i, g] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[i, g] . k_j),   j < len, causal: j <= len - n + i
//
// in one pass over the keys with a running maximum and sum (log2 domain). What it has to do is read the cached keys and
// values once: 2 len d elements for each key head against 2 * 2 len d operations for each query row, so with up to 16 rows
// it is bound by memory, and everything here serves the reads:
//
//   * Queries are the narrow operand. The matrix instruction takes 16 keys by 16 of d from shared memory against 8 query
//     rows (new tokens x query heads of one key head, token-major) held in registers: scores come out as keys x queries,
//     are turned around by movmatrix, and meet V^T the same way. With queries as the 16-high operand a group of 4 or 8
//     heads left half of every instruction and of the softmax unused (812 instructions for 32 keys of a key head, all roles
//     counted, against 610).
//   * Work is cut evenly: all (sequence, head, row block) units in a row, tiles of 64 or 128 keys, and every CTA takes its
//     share (paged_dev.cuh). Ragged lengths then cost nothing, and one long sequence spreads over the GPU. The parts of a
//     unit that several CTAs share (fp32 rows, reference maximum, sum) are joined in the order of the CTAs by the one that
//     finishes last: a call's result does not depend on which does. (It depends on the lengths of the whole batch, on the
//     GPU's SM count and on the choice of kernel and unit in capi.cu.)
//   * Producer warps for keys and for values read the page table and keep a ring of tiles in flight by TMA (a box per page,
//     swizzled, so that pages of 16 tokens land as one conflict-free tile), two tiles to each pair of consumer warps. A
//     third brings the queries.
//   * Six or eight consumer warps work without meeting: two to a tile, half of its keys each, every warp with its own
//     running maximum, sum and output. At the end of a unit they leave these in shared memory and go on to the next, whose
//     queries a producer has brought there; four further warps join and write them. (With the consumers doing this
//     themselves a unit cost them 3.9 us besides its tiles.)
//
// Precision: scores and sums are fp32. 16-bit caches: P enters the second product as hi + lo (two 16-bit numbers), so its
// rounding (which alone would be as large as the output's) is gone; the tensor cores idle here and the second product is
// free. 8-bit caches: keys and values enter as the whole numbers they are, exact in fp16. bf16 queries turn into fp16 with
// a power of two for each row, exact but for what is below 2^-31 of the row's largest: fp16's 10 bits take a byte as it is,
// where bf16 needs a subtraction for each (contexts of 2000 to 16383 tokens, pages of 64: 60.6 us, and 62.7 in bf16). The
// key's scale multiplies the score, and the value's goes into the exponent: p'_j = 2^(s_j + log2 vs_j - m') is p_j vs_j
// normalised to at most 1, whatever the scales, and is rounded to fp16 once; the sum adds p'_j / vs_j. (fp32 spans the scales
// that meet in a row: one 2^126 below what has the largest p'_j loses its weight. A vector of zeros counts as 2^-100, so
// values of 1e10 beside vectors of zeros are the limit.)
#include <cuda.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "launchers.h"
#include "paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace phantom {
namespace rows {

// A unit has 8 NT query rows (NT = 1, 2).
constexpr int kJoiners = 4;
constexpr int kUnitRing = 4;
constexpr int kErrCopyWait = 1, kErrTileWait = 4, kErrJoinWait = 8;

// Warps: eight consumers, in pairs that take the tiles in turn; the joiners; three producers and, completing their warpgroup,
// one that zeroes the rows of no sequence. Registers (setmaxnreg, by warpgroup): 512 threads launch with 128 each;
// 2 * 168 + 104 + 72 = 4 * 128.
constexpr int kConsumers = 8, PRODUCER = kConsumers + kJoiners, kThreads = 32 * (PRODUCER + 4);
constexpr int kRegsConsumer = 168, kRegsJoiner = 104, kRegsProducer = 72;

template <int D, bool INT8, int NT>
struct Cfg {
  static constexpr int BR = 8 * NT;
  static constexpr int ROW = INT8 ? D : 128;              // bytes of a swizzled row (16-bit: 64 columns)
  static constexpr int BLOCKS = INT8 ? 1 : D / 64;        // such blocks across d
  static constexpr bool WIDE = !INT8 && D == 128;
  static_assert(INT8 || NT == 1);
  static constexpr int SLOT = (WIDE ? 32 : 16) * 1024, HALF = SLOT / 2;  // a tile: its keys, its values
  static constexpr int BN = HALF / (D * (INT8 ? 1 : 2));  // keys of a tile: 64 or 128
  static constexpr int MT = BN <= 64 || NT == 1 ? BN / 32 : 2;  // 16 MT keys at a time go through a warp
  static constexpr int SUB = BN / (32 * MT);              // times
  // Two slots to a pair, so that a pair's next tile is on its way while it works on one. A slot's tiles all go to one pair,
  // which so sees every phase of its barriers. (With a slot passed between pairs, a pair could wait for a phase whose
  // predecessor was still open, and parity would let it by.)
  static constexpr int PAIRS = WIDE ? 3 : 4, WARPS = 2 * PAIRS, SLOTS = 2 * PAIRS;
  static constexpr int OFF_MERGE = SLOTS * SLOT;          // [WARPS][BR][D] fp32
  static constexpr int OFF_ML = OFF_MERGE + WARPS * BR * D * 4;
  static constexpr int Q_ROW = 2 * D + 16;                // padded: lanes of 8 rows and 4 words read without conflicts
  static constexpr int OFF_Q = OFF_ML + WARPS * BR * 8;
  static constexpr int OFF_IDS = OFF_Q + kUnitRing * BR * Q_ROW;  // page ids, 64 to each producer
  static constexpr int OFF_UNIT = OFF_IDS + 2 * 64 * 4;
  static constexpr int OFF_BAR = OFF_UNIT + kUnitRing * 48;
  static constexpr int OFF_FLAG = OFF_BAR + (2 * SLOTS + 2 * kUnitRing + 2) * 8;
  static constexpr int SMEM = OFF_FLAG + 16 + 1024;       // + slack to align the base
  static_assert(SMEM <= 227 * 1024, "shared memory plan exceeds 227 KB");
};

// ------------------------------------------------------------------------------------------------ units and tiles
// Units of 8 NT rows; tiles of BN keys.
template <int NT, int BN>
struct RowBlocks {
  int group, causal;
  // Measured (us): kJoin 8 | 5: 4 sequences of 500 tokens 10.7 | 12.0, 8 of 700 12.6 | 15.0, 32 of 200 to 4095 the same.
  // kPart 0.4 | 0.8: one of 4096 14.3 | 15.6, of 1024 11.9 | 12.1; 16 rows, 0.5 | 2: one of 1000 17.3 | 23.3.
  static constexpr int kTile = BN, kUnit = 2, kJoin = 8, BR = 8 * NT;
  static constexpr float kPart = NT == 1 ? 0.4f : 0.5f;
  __device__ int count(const Seq& x) const { return (x.n * group + BR - 1) / BR; }
  __device__ int key_end(const Seq& x, int rb) const {
    if (!causal) return x.len;
    const int last = min(x.n * group - 1, rb * BR + BR - 1) / group;
    return min(max(x.off + last + 1, 0), x.len);
  }
  __device__ long long head_tiles(const Seq& x) const { return sum_tiles(*this, x); }
};

template <int NT, int BN>
struct Params {
  PagedSeqs s;
  const uint16_t* q;
  long long q_token, q_head;
  uint16_t* o;
  const float *ks, *vs;
  Strides3 kss, vss;
  RowBlocks<NT, BN> blocks;
  float scale_log2;  // of the scores' size
  uint32_t flip;     // sign bits to flip in the queries (a negative scale)
  float* part;       // parts of shared units, [place][8 NT] rows of D sums of values
  float2* ml;        // their (reference maximum, sum)
  unsigned long long* words;  // of shared units, at the number of their first CTA
  unsigned long long call;
};

// ------------------------------------------------------------------------------------------------ matrix instructions
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void joiners_meet() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool joiners_all(bool x) {
  uint32_t y;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(y) : "r"((uint32_t)x) : "memory");
  return y != 0;
}
// Transposes the 8 x 8 matrix of 16-bit numbers that a warp holds (lane 4 r + c: row r, columns 2 c and 2 c + 1).
__device__ __forceinline__ uint32_t turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// What the records' producer tells the others of a unit (48 bytes).
struct Unit {
  int cnt, tile0, end, id;    // its tiles here, the first of them; the keys that its rows see; id -1 ends the roles
  int off, n, row0, tok0;     // the sequence: where its new tokens begin, how many; the unit's first row; its packed place
  int h, c0, c1, b;           // key head; the first and the last CTA that have tiles of it; the sequence
};

template <int D, bool BF16, bool INT8, int NT>
__global__ void __launch_bounds__(kThreads, 1)
attn_rows(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params<NT, Cfg<D, INT8, NT>::BN> p) {
  using C = Cfg<D, INT8, NT>;
  using Blocks = RowBlocks<NT, C::BN>;
  constexpr int BR = C::BR, BN = C::BN, MT = C::MT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem), bars = sbase + C::OFF_BAR;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (C::SLOTS + s); };
  auto q_full = [&](int u) { return bars + 8u * (2 * C::SLOTS + u % kUnitRing); };
  auto q_empty = [&](int u) { return bars + 8u * (2 * C::SLOTS + kUnitRing + u % kUnitRing); };
  const uint32_t join_full = bars + 8u * (2 * C::SLOTS + 2 * kUnitRing), join_empty = join_full + 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_FLAG);
  volatile int* joined = reinterpret_cast<volatile int*>(smem + C::OFF_FLAG + 4);
  int4* ring = reinterpret_cast<int4*>(smem + C::OFF_UNIT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.blocks.group, causal = p.blocks.causal;
  int* status = p.s.status;

  if (warp == 0) {
    constexpr int N = 2 * C::SLOTS;  // of full (the two producers arrive) and empty (the consuming pair does)
    static_assert(N + 2 * kUnitRing + 2 <= 32);
    if (lane < N + 2 * kUnitRing + 2)
      mbar_init(bars + 8u * lane, lane < N ? 2 : lane < N + kUnitRing ? 1 : lane < N + 2 * kUnitRing ? C::WARPS + kJoiners :
                                  lane == N + 2 * kUnitRing ? C::WARPS : kJoiners);
    if (lane == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  auto wait = [&](uint32_t bar, int parity, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code)) != 0;
  };
  // A consuming role's next unit (id -1 at the end, or when a wait gave up).
  auto next_unit = [&](int u) {
    Unit x;
    x.id = -1;
    if (wait(q_full(u), (u / kUnitRing) & 1, kErrTileWait)) {
      const int4* r = ring + 3 * (u % kUnitRing);
      const int4 a = r[0], b = r[1], c = r[2];
      x.cnt = a.x, x.tile0 = a.y, x.end = a.z, x.id = a.w;
      x.off = b.x, x.n = b.y, x.row0 = b.z, x.tok0 = b.w;
      x.h = c.x, x.c0 = c.y, x.c1 = c.z, x.b = c.w;
    }
    return x;
  };

  if (warp >= PRODUCER) {
    setmaxnreg_dec<kRegsProducer>();
    const int role = warp - PRODUCER;
    if (role > 2) {
      zero_unowned(p.s, p.o, p.s.heads * group * (D / 8), blockIdx.x * 32 + lane, gridDim.x * 32);
      return;
    }
    // Producers, of the keys, of the values, and of the units' records and queries. Each walks the CTA's share by itself.
    if (role < 2 && elect_one()) tma_prefetch_desc(role ? &tmV : &tmK);
    __syncwarp();
    Walk<Blocks> w;
    w.start(p.s, p.blocks, blockIdx.x, gridDim.x);
    bool ok = true;
    if (role == 2) {
      int nu = 0;
      for (; w.cnt > 0; w.advance(p.s, p.blocks)) {
        if (nu >= kUnitRing && !(ok = wait(q_empty(nu), (nu / kUnitRing - 1) & 1, kErrCopyWait))) break;
        const int row0 = w.blk * BR, rows = min(BR, w.x.n * group - row0);
        if (elect_one()) mbar_expect_tx(q_full(nu), rows * D * 2);
        __syncwarp();
        if (lane < rows) {
          const int tok = (row0 + lane) / group;
          bulk_load(sbase + C::OFF_Q + ((nu % kUnitRing) * BR + lane) * C::Q_ROW,
                    p.q + (w.x.tok0 + tok) * p.q_token + (w.h * group + (row0 + lane - tok * group)) * p.q_head, D * 2, q_full(nu));
        }
        const int2 own = w.owners(blockIdx.x);
        if (elect_one()) {
          int4* r = ring + 3 * (nu % kUnitRing);
          r[0] = make_int4(w.cnt, w.tile, p.blocks.key_end(w.x, w.blk), nu);
          r[1] = make_int4(w.x.off, w.x.n, row0, w.x.tok0);
          r[2] = make_int4(w.h, own.x, own.y, w.b);
          mbar_arrive(q_full(nu));
        }
        __syncwarp();
        ++nu;
      }
      if (ok && nu >= kUnitRing) ok = wait(q_empty(nu), (nu / kUnitRing - 1) & 1, kErrCopyWait);
      if (ok) {
        if (elect_one()) {
          ring[3 * (nu % kUnitRing)] = make_int4(0, 0, 0, -1);
          mbar_arrive(q_full(nu));
        }
        __syncwarp();
        ++nu;
      }
      if (!ok) *abort_flag = 1;
      for (int u = max(0, nu - kUnitRing); u < nu; ++u) mbar_wait_drain(q_full(u), (u / kUnitRing) & 1);
      return;
    }
    // Keys and values: a copy to a page. One elected lane issues the copies, whose issue is what limits pages of 16 tokens,
    // hence a warp for each. Page ids wait in shared memory.
    const CUtensorMap* map = role ? &tmV : &tmK;
    int t = 0;
    const int page_log2 = p.s.page_log2, page = 1 << page_log2, box = min(page, BN);
    const uint32_t bytes = box * D * (INT8 ? 1 : 2);  // of a copy
    const uint32_t dst0 = sbase + role * C::HALF;
    int* ids = reinterpret_cast<int*>(smem + C::OFF_IDS) + role * 64;  // page i's id at i % 64
    while (w.cnt > 0) {
      const int end = p.blocks.key_end(w.x, w.blk), cnt = w.cnt;
      const int pages = (end + page - 1) >> page_log2;    // that the unit sees
      int ahead = ((w.tile * BN) >> page_log2) & ~31;     // ids are there for pages below
      auto ids_more = [&]() {
        ids[(ahead + lane) & 63] = ahead + lane < pages ? page_of(p.s, w.b, ahead + lane) : 0;
        ahead += 32;
      };
      ids_more();
      if (ahead < pages) ids_more();
      __syncwarp();
      for (int i = 0; i < cnt; ++i, ++t) {
        const int s = t % C::SLOTS, round = t / C::SLOTS;
        const int j0 = (w.tile + i) * BN, place = j0 & (page - 1), first = j0 >> page_log2;
        const int boxes = max(0, (min(j0 + BN, end) - j0 + box - 1) / box);  // pages of the tile that hold keys
        if (round > 0 && !(ok = wait(empty(s), (round - 1) & 1, kErrCopyWait))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(full(s), boxes * bytes);
          uint32_t dst = dst0 + s * C::SLOT;
#pragma unroll 1
          for (int pg = 0; pg < boxes; ++pg, dst += bytes) {
            const int from = ids[(first + pg) & 63];  // one that is out of range reads as zeros (the map's bounds)
            tma_load_5d(dst, map, full(s), 0, place, 0, w.h, from);
          }
        }
        __syncwarp();
        // (a tile has at most 8 pages; those below ahead - 32, which the next ones take the place of, are done with)
        if (first >= ahead - 32 && ahead < pages) ids_more();
        __syncwarp();
      }
      if (!ok) break;
      w.advance(p.s, p.blocks);
    }
    if (!ok) *abort_flag = 1;
    // every issued copy lands before this CTA's shared memory is released
    for (int i = max(0, t - C::SLOTS); i < t; ++i) mbar_wait_drain(full(i % C::SLOTS), (i / C::SLOTS) & 1);
    return;
  }

  float* merge = reinterpret_cast<float*>(smem + C::OFF_MERGE);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  if (warp >= kConsumers) {
    setmaxnreg_dec<kRegsJoiner>();
    // Joiners: a unit's rows from the consumers' sums, to the output or to the parts of a shared unit.
    constexpr int PER = BR * D / 128;  // columns of a thread: 16, 8 or 4
    const int tid = threadIdx.x - 32 * kConsumers;
    const int r = tid / (128 / BR), col = (tid % (128 / BR)) * PER;
    int u = 0;
    for (;; ++u) {
      const Unit x = next_unit(u);
      __syncwarp();
      if (x.id >= 0 && lane == 0) mbar_arrive(q_empty(u));
      const int row = x.row0 + r, tok = row / group;
      const bool there = row < x.n * group;
      uint2* dst = reinterpret_cast<uint2*>(
          p.o + ((long long)(x.tok0 + tok) * p.s.heads * group + x.h * group + (row - tok * group)) * D + col);
      // all four warps go on, or none (a wait that gave up ends the roles; no warp may be left at a barrier)
      if (!joiners_all(x.id >= 0 && wait(join_full, u & 1, kErrJoinWait))) break;
      float M = -CUDART_INF_F, L = 0.f, acc[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll
      for (int v = 0; v < C::WARPS; ++v) M = fmaxf(M, ml[v * BR + r].x);
      {
        const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll 2
        for (int v = 0; v < C::WARPS; ++v) {
          const float2 y = ml[v * BR + r];
          if (y.x == -CUDART_INF_F && y.y == 0.f) continue;  // no key seen, and maybe nothing written
          const float wt = ex2(y.x - ref);
          L = fmaf(wt, y.y, L);
          const float* src = merge + (v * BR + r) * D;
#pragma unroll
          for (int i = 0; i < PER; i += 4) {
            const float4 f = *reinterpret_cast<const float4*>(src + ((col + i) ^ (((r >> 1) & 3) * 8)));
            acc[i] = fmaf(wt, f.x, acc[i]);
            acc[i + 1] = fmaf(wt, f.y, acc[i + 1]);
            acc[i + 2] = fmaf(wt, f.z, acc[i + 2]);
            acc[i + 3] = fmaf(wt, f.w, acc[i + 3]);
          }
        }
      }
      bool done = x.c0 == x.c1;
      if (done) {
        __syncwarp();
        if (lane == 0) mbar_arrive(join_empty);
      } else {
        const long long slot = Walk<Blocks>::place(blockIdx.x, (int)blockIdx.x == x.c0);
        if (there) {
          float* to = p.part + (slot * BR + r) * D + col;
#pragma unroll
          for (int i = 0; i < PER; i += 4)
            *reinterpret_cast<float4*>(to + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
          if (col == 0) p.ml[slot * BR + r] = make_float2(M, L);
        }
        joiners_meet();
        const int parts = x.c1 - x.c0 + 1;
        if (threadIdx.x == 32 * kConsumers) *joined = last_part(p.words + x.c0, p.call, parts);
        joiners_meet();
        done = *joined != 0;
        if (done) {
          // Warp v takes every fourth part, four rows of it at once (32 lanes to a row), each with a running maximum; the
          // four warps' sums meet in shared memory as the consumers' did.
          const int rows = min(BR, x.n * group - x.row0);
          const int v = warp - kConsumers;
          constexpr int W = D / 32;  // columns of a lane
          float* sums = merge;       // [warp][BR][D]
          for (int r0 = 0; r0 < rows; r0 += 4) {
            float m4[4], l4[4], a4[4][W];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              m4[k] = -CUDART_INF_F;
              l4[k] = 0.f;
#pragma unroll
              for (int e = 0; e < W; ++e) a4[k][e] = 0.f;
            }
#pragma unroll 1
            for (int c = v; c < parts; c += 2 * kJoiners) {  // two parts' loads at once
              float2 y[2][4];
              float f[2][4][W];
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int part = c + i * kJoiners;
                  const bool in = part < parts && r0 + k < rows;
                  const long long at = Walk<Blocks>::place(x.c0 + part, part == 0) * BR + r0 + k;
                  y[i][k] = in ? __ldcg(p.ml + at) : make_float2(-CUDART_INF_F, 0.f);
                  const float* src = p.part + at * D + lane * W;
                  if constexpr (W == 4) *reinterpret_cast<float4*>(f[i][k]) = in ? __ldcg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
                  else *reinterpret_cast<float2*>(f[i][k]) = in ? __ldcg(reinterpret_cast<const float2*>(src)) : make_float2(0.f, 0.f);
                }
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float y0 = y[0][k].x, y1 = y[1][k].x, top = fmaxf(m4[k], fmaxf(y0, y1)), ref = top == -CUDART_INF_F ? 0.f : top;
                const float wt = ex2(m4[k] - ref), w0 = ex2(y0 - ref), w1 = ex2(y1 - ref);
                m4[k] = top;
                l4[k] = fmaf(l4[k], wt, fmaf(w0, y[0][k].y, w1 * y[1][k].y));
#pragma unroll
                for (int e = 0; e < W; ++e) a4[k][e] = fmaf(a4[k][e], wt, fmaf(w0, f[0][k][e], w1 * f[1][k][e]));
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (r0 + k >= rows) continue;
#pragma unroll
              for (int e = 0; e < W; ++e) sums[(v * BR + r0 + k) * D + lane * W + e] = a4[k][e];
              if (lane == 0) ml[v * BR + r0 + k] = make_float2(m4[k], l4[k]);
            }
          }
          joiners_meet();
          M = -CUDART_INF_F;
          L = 0.f;
#pragma unroll
          for (int i = 0; i < PER; ++i) acc[i] = 0.f;
          if (there) {
#pragma unroll
            for (int u4 = 0; u4 < kJoiners; ++u4) M = fmaxf(M, ml[u4 * BR + r].x);
            const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll 1
            for (int u4 = 0; u4 < kJoiners; ++u4) {
              const float2 y = ml[u4 * BR + r];
              const float wt = ex2(y.x - ref);
              L = fmaf(wt, y.y, L);
#pragma unroll
              for (int i = 0; i < PER; i += 4) {
                const float4 f = *reinterpret_cast<const float4*>(sums + (u4 * BR + r) * D + col + i);
                acc[i] = fmaf(wt, f.x, acc[i]);
                acc[i + 1] = fmaf(wt, f.y, acc[i + 1]);
                acc[i + 2] = fmaf(wt, f.z, acc[i + 2]);
                acc[i + 3] = fmaf(wt, f.w, acc[i + 3]);
              }
            }
          }
          joiners_meet();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(join_empty);
      }
      if (done && there) {
        const float inv = M == -CUDART_INF_F ? 0.f : 1.f / L;
#pragma unroll
        for (int i = 0; i < PER / 4; ++i)
          dst[i] = make_uint2(pack2<BF16>(acc[4 * i] * inv, acc[4 * i + 1] * inv), pack2<BF16>(acc[4 * i + 2] * inv, acc[4 * i + 3] * inv));
      }
    }
    if (*abort_flag && warp == kConsumers) {
      // A wait gave up: this CTA's parts from unit u on will not come, but they are counted, so that the last to be counted
      // leaves 0 in each word. A replay of a graph has the same call's number: it would take a count that was left for its own.
      Walk<Blocks> w;
      w.start(p.s, p.blocks, blockIdx.x, gridDim.x);
      for (int v = 0; w.cnt > 0; w.advance(p.s, p.blocks), ++v) {
        const int2 own = w.owners(blockIdx.x);
        if (v >= u && own.x != own.y && lane == 0) last_part(p.words + own.x, p.call, own.y - own.x + 1);
        __syncwarp();
      }
    }
    return;
  }

  setmaxnreg_inc<kRegsConsumer>();
  if (warp >= C::WARPS) return;
  const int g = lane >> 2, t4 = lane & 3;
  const int pair = warp >> 1;
  constexpr int KEYS = 16 * MT;  // that go through this warp at a time
  const int kr = (warp & 1) * (BN / 2);  // its first key of its pair's tiles
  // Where this lane's rows for ldmatrix lie in a tile: 16 keys from kr + KEYS sub + 16 mt, matrices (keys 0-7, 8-15) x
  // (first, second 16-byte chunk of a pair); V^T of 16-bit values has the two the other way around. Boxes of
  // min(page, BN) tokens, each [64-column block][token][ROW bytes]; a chunk lies at its number ^ the row's swizzle, so
  // stepping over pairs of chunks is an XOR with 32 times the pair's number.
  const int box_log2 = min(p.s.page_log2, BN == 64 ? 6 : 7), blk_stride = C::ROW << box_log2;
  constexpr int AT = C::BLOCKS == 1 ? 1 : MT;  // one column block: 16 rows further on is a constant away
  static_assert(C::SUB == 1 || C::BLOCKS == 1);
  static_assert(!INT8 || (BN / 2 == 32 || BN / 2 == 64) && (C::SUB == 1 || (C::SUB == 2 && KEYS == 32)));
  uint32_t at_k[AT], at_v[AT];
#pragma unroll
  for (int mt = 0; mt < AT; ++mt) {
    auto place_of = [&](int key, int chunk) {
      const int row = C::BLOCKS == 1 ? key : (((key >> box_log2) * C::BLOCKS) << box_log2) + (key & ((1 << box_log2) - 1));
      const int sw = C::ROW == 128 ? key & 7 : (key >> 1) & 3;
      return (uint32_t)(row * C::ROW + ((chunk ^ sw) << 4));
    };
    const int key = kr + mt * 16 + (lane & 7);
    at_k[mt] = place_of(key + ((lane >> 3) & 1) * 8, lane >> 4);
    at_v[mt] = INT8 ? at_k[mt] : place_of(key + (lane >> 4) * 8, (lane >> 3) & 1);
  }
  int t = 0, first = pair;  // tiles before this unit; the first of it that is this pair's
  for (int u = 0;; ++u) {
    const Unit x = next_unit(u);
    if (x.id < 0) break;
    const int R = x.n * group, row0 = x.row0, off = x.off, end = x.end;
    // the queries as B operands: of row 8 nt + g; 8-bit caches: columns in the order that their bytes come in (4 t4 ... + 3
    // of 16). Keys that the rows 8 nt + 2 t4 + e of this lane's scores see. (Rows past the last hold anything; no row's
    // numbers meet another's.)
    uint32_t qb[NT][D / 16][2];
    int lim[NT][2];
    float q_back[NT][2];  // 8-bit caches, bf16: of the rows of this lane's scores, what their queries were divided by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint8_t* src = smem + C::OFF_Q + ((u % kUnitRing) * BR + nt * 8 + g) * C::Q_ROW;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if constexpr (INT8) {
          const uint2 y = *reinterpret_cast<const uint2*>(src + k * 32 + 8 * t4);
          qb[nt][k][0] = y.x;
          qb[nt][k][1] = y.y;
        } else {
          qb[nt][k][0] = *reinterpret_cast<const uint32_t*>(src + k * 32 + 4 * t4) ^ p.flip;
          qb[nt][k][1] = *reinterpret_cast<const uint32_t*>(src + k * 32 + 16 + 4 * t4) ^ p.flip;
        }
      }
      if constexpr (INT8 && BF16) {
        // to fp16, times the power of two that brings the row's largest to [2^14, 2^15)
        uint32_t big = 0;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) big = __vmaxu2(big, __vmaxu2(qb[nt][k][0] & 0x7FFF7FFFu, qb[nt][k][1] & 0x7FFF7FFFu));
        big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int ex = max((int)(max(big & 0xFFFFu, big >> 16) >> 7) - 127, -111);
        const float f = __uint_as_float((uint32_t)(141 - ex) << 23), back = __uint_as_float((uint32_t)(113 + ex) << 23);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t y = qb[nt][k][e];
            qb[nt][k][e] = pack2<false>(__uint_as_float(y << 16) * f, __uint_as_float(y & 0xFFFF0000u) * f);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) q_back[nt][e] = __shfl_sync(0xffffffffu, back, (2 * t4 + e) * 4);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + nt * 8 + 2 * t4 + e;
        lim[nt][e] = row >= R ? 0 : causal ? min(end, off + row / group + 1) : end;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(q_empty(u));
    const int lim_least = causal ? max(0, min(end, off + row0 / group + 1)) : end;  // of the block's rows
    float m[NT][2], l[NT][2], o[D / 16][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -CUDART_INF_F;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) o[c][nt][0] = o[c][nt][1] = o[c][nt][2] = o[c][nt][3] = 0.f;
    }

    bool ok = true;
    // 8-bit: the scales of this warp's keys, a lane each (and a lane's second key 32 further on), are read one tile ahead,
    // their pages' ids while the tile before is waited for and the scales after its first product.
    constexpr int NQ = INT8 ? BN / 64 : 1;
    int ids[NQ];
    float ks[NQ], vs[NQ];
    auto read_ids = [&](int i) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int j = (x.tile0 + i) * BN + kr + 32 * q + lane;
        ids[q] = j < x.end ? page_of(p.s, x.b, j >> p.s.page_log2) : -1;
      }
    };
    auto read_scales = [&](int i) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int place = ((x.tile0 + i) * BN + kr + 32 * q + lane) & ((1 << p.s.page_log2) - 1);
        ks[q] = vs[q] = 0.f;
        if (ids[q] >= 0) {
          ks[q] = p.ks[ids[q] * p.kss.page + x.h * p.kss.head + place];
          vs[q] = p.vs[ids[q] * p.vss.page + x.h * p.vss.head + place];
        }
      }
    };
    if (INT8 && first < x.cnt) {
      read_ids(first);
      read_scales(first);
    }
    for (int i = first; i < x.cnt; i += C::PAIRS) {  // tiles of the whole share go to the pairs in turn
      const int s = (t + i) % C::SLOTS;
      if (!(ok = wait(full(s), ((t + i) / C::SLOTS) & 1, kErrTileWait))) break;
      float ksl[NQ], lvs[NQ], ivs[NQ];  // the key's scale, log2 of the value's, its reciprocal (no effect past the end)
      if constexpr (INT8) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const bool in = (x.tile0 + i) * BN + kr + 32 * q + lane < x.end;
          const float v = least_scale(vs[q]);
          ksl[q] = ks[q] * p.scale_log2;
          lvs[q] = in ? __log2f(v) : 0.f;
          ivs[q] = in && v == v ? __fdividef(1.f, v) : 0.f;  // (NaN: the logarithm alone passes it on, to rows that see it)
        }
        if (i + C::PAIRS < x.cnt) read_ids(i + C::PAIRS);
      }
#pragma unroll 1
      for (int sub_i = 0; sub_i < C::SUB; ++sub_i) {
        const uint32_t kb = sbase + s * C::SLOT + sub_i * KEYS * C::ROW, vb = kb + C::HALF;
        const int j0 = (x.tile0 + i) * BN + kr + sub_i * KEYS;  // the first key
        if (j0 >= end) break;
        // ---- scores: [16 keys][8 rows]: (key g: rows 2 t4, + 1; key g + 8: the same)
        float sc[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[mt][nt][0] = sc[mt][nt][1] = sc[mt][nt][2] = sc[mt][nt][3] = 0.f;
          if constexpr (INT8) {
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
              uint32_t r[4], a[2][4];
              ldsm4(kb + mt * 16 * C::ROW + (at_k[0] ^ (k << 5)), r);
#pragma unroll
              for (int e = 0; e < 4; ++e) {  // r: (keys 0-7, 8-15) of chunk 2 k, then of 2 k + 1
                const uint32_t u = r[e] ^ 0x80808080u;
                a[e >> 1][e & 1] = bytes_f16<0x4140>(u);
                a[e >> 1][2 + (e & 1)] = bytes_f16<0x4342>(u);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(sc[mt][nt], a[0], qb[nt][2 * k][0], qb[nt][2 * k][1]);
                mma16816<false>(sc[mt][nt], a[1], qb[nt][2 * k + 1][0], qb[nt][2 * k + 1][1]);
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              uint32_t r[4];
              ldsm4(kb + (C::BLOCKS == 1 ? mt * 16 * C::ROW : (k >> 2) * blk_stride) + (at_k[C::BLOCKS == 1 ? 0 : mt] ^ ((k & 3) << 5)), r);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<BF16>(sc[mt][nt], r, qb[nt][k][0], qb[nt][k][1]);
            }
          }
        }
        // ---- 8-bit: to the log2 domain, with the values' scales; masks
        float inv_vs[MT][2];
        if constexpr (INT8) {
          if (sub_i == C::SUB - 1 && i + C::PAIRS < x.cnt) read_scales(i + C::PAIRS);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int from = ((mt * 16 + e * 8) & 31) + g;
              auto of_key = [&](const float (&r)[NQ]) {
                return __shfl_sync(0xffffffffu, C::SUB == 1 ? r[mt >> 1] : r[C::SUB > 1 && sub_i > 0 ? NQ - 1 : 0], from);
              };
              const float a = of_key(ksl), lv = of_key(lvs);
              inv_vs[mt][e] = of_key(ivs);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                sc[mt][nt][2 * e] = fmaf(sc[mt][nt][2 * e], BF16 ? a * q_back[nt][0] : a, lv);
                sc[mt][nt][2 * e + 1] = fmaf(sc[mt][nt][2 * e + 1], BF16 ? a * q_back[nt][1] : a, lv);
              }
            }
        }
        if (j0 + KEYS > lim_least) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (j0 + mt * 16 + (e >> 1) * 8 + g >= lim[nt][e & 1]) sc[mt][nt][e] = -CUDART_INF_F;
        }
        // ---- running maximum of each row, over the lanes of one t4
        const float scale = INT8 ? 1.f : p.scale_log2;
        float2 sub[NT], alpha[NT];
        bool grew = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float y = fmaxf(sc[0][nt][e], sc[0][nt][2 + e]);
#pragma unroll
            for (int mt = 1; mt < MT; ++mt) y = fmaxf(y, fmaxf(sc[mt][nt][e], sc[mt][nt][2 + e]));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
            y = fmaxf(y * scale, m[nt][e]);
            const float ref = y == -CUDART_INF_F ? 0.f : y, al = ex2(m[nt][e] - ref);  // 0 while no key was seen
            grew |= y != m[nt][e];
            m[nt][e] = y;
            l[nt][e] *= al;
            if (e == 0) sub[nt].x = -ref, alpha[nt].x = al;
            else sub[nt].y = -ref, alpha[nt].y = al;
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float2 a = mul2(make_float2(o[c][nt][0], o[c][nt][1]), alpha[nt]);
              const float2 b = mul2(make_float2(o[c][nt][2], o[c][nt][3]), alpha[nt]);
              o[c][nt][0] = a.x, o[c][nt][1] = a.y, o[c][nt][2] = b.x, o[c][nt][3] = b.y;
            }
        }
        // ---- probabilities, turned into B operands (16 keys by 8 rows)
        uint32_t hi[MT][NT][2], lo[MT][NT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float2 y = fma2(make_float2(sc[mt][nt][2 * e], sc[mt][nt][2 * e + 1]), make_float2(scale, scale), sub[nt]);
              y.x = ex2(y.x);
              y.y = ex2(y.y);
              if constexpr (INT8) {
                l[nt][0] = fmaf(y.x, inv_vs[mt][e], l[nt][0]);
                l[nt][1] = fmaf(y.y, inv_vs[mt][e], l[nt][1]);
                hi[mt][nt][e] = turn(pack2<false>(y.x, y.y));
              } else {
                l[nt][0] += y.x;
                l[nt][1] += y.y;
                const uint32_t h = pack2<BF16>(y.x, y.y);
                float2 f;
                if constexpr (BF16)
                  f = make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xFFFF0000u));
                else
                  f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                hi[mt][nt][e] = turn(h);
                lo[mt][nt][e] = turn(pack2<BF16>(y.x - f.x, y.y - f.y));
              }
            }
        // ---- values; those of keys past the end are zeroed (what lies in the page there may be anything)
        const bool tail = j0 + KEYS > end;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (tail) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = j0 + mt * 16 + e * 8 + 2 * t4;
              keep[e] = (j < end ? 0xffffu : 0u) | (j + 1 < end ? 0xffff0000u : 0u);
            }
          }
          if constexpr (INT8) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t r[4], a[2][4];
              ldsm4_t(vb + mt * 16 * C::ROW + (at_v[0] ^ (c << 5)), r);
#pragma unroll
              for (int e = 0; e < 4; ++e) {  // r: (keys 0-7, 8-15) of columns 32 c ... + 15, then ... + 31; even and odd columns
                const uint32_t u = (tail ? r[e] & keep[e & 1] : r[e]) ^ 0x80808080u;
                a[e >> 1][2 * (e & 1)] = bytes_f16<0x4240>(u);
                a[e >> 1][2 * (e & 1) + 1] = bytes_f16<0x4341>(u);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(o[2 * c][nt], a[0], hi[mt][nt][0], hi[mt][nt][1]);
                mma16816<false>(o[2 * c + 1][nt], a[1], hi[mt][nt][0], hi[mt][nt][1]);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t r[4];
              ldsm4_t(vb + (C::BLOCKS == 1 ? mt * 16 * C::ROW : (c >> 2) * blk_stride) + (at_v[C::BLOCKS == 1 ? 0 : mt] ^ ((c & 3) << 5)), r);
              if (tail) {
                r[0] &= keep[0];
                r[1] &= keep[0];
                r[2] &= keep[1];
                r[3] &= keep[1];
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<BF16>(o[c][nt], r, hi[mt][nt][0], hi[mt][nt][1]);
                mma16816<BF16>(o[c][nt], r, lo[mt][nt][0], lo[mt][nt][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(s));
    }

    t += x.cnt;
    first = (first - x.cnt) % C::PAIRS;
    if (first < 0) first += C::PAIRS;
    if (!ok) break;

    // ---- for the joiners: rows in shared memory, columns swizzled by 8 floats with the row (no bank conflicts)
    if (u > 0 && !wait(join_empty, (u - 1) & 1, kErrJoinWait)) break;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float y = l[nt][e];
        y += __shfl_xor_sync(0xffffffffu, y, 4);
        y += __shfl_xor_sync(0xffffffffu, y, 8);
        y += __shfl_xor_sync(0xffffffffu, y, 16);
        const int r = nt * 8 + 2 * t4 + e;
        if (g == 0) ml[warp * BR + r] = make_float2(m[nt][e], y);
        float* dst = merge + (warp * BR + r) * D;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          if constexpr (INT8) {
            *reinterpret_cast<float2*>(dst + ((16 * c + 2 * g) ^ (t4 * 8))) = make_float2(o[c][nt][e], o[c][nt][2 + e]);
          } else {
            dst[(16 * c + g) ^ (t4 * 8)] = o[c][nt][e];
            dst[(16 * c + g + 8) ^ (t4 * 8)] = o[c][nt][2 + e];
          }
        }
      }
    __syncwarp();
    if (lane == 0) mbar_arrive(join_full);
  }
}

std::atomic<bool> g_attr[2][2][2][2][64];

template <int D, bool BF16, bool INT8, int NT>
cudaError_t launch(const PagedAttnArgs& a, int dev) {
  using C = Cfg<D, INT8, NT>;
  int ctas = 0;
  cudaError_t e = sm_count(dev, &ctas);
  if (e != cudaSuccess) return e;
  auto kern = attn_rows<D, BF16, INT8, NT>;
  std::atomic<bool>& attr = g_attr[D / 128][BF16][INT8][NT - 1][dev];
  if (!attr.load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
    attr.store(true, std::memory_order_release);
  }
  CUtensorMap mk, mv;
  const int page = 1 << a.s.page_log2, box = std::min(page, C::BN), elem = INT8 ? 1 : 2, cols = INT8 ? D : 64;
  if (!make_paged_map(&mk, a.kc, a.s.num_pages, a.s.heads, page, D, a.kcs, elem, BF16, cols, box, C::BLOCKS, 1) ||
      !make_paged_map(&mv, a.vc, a.s.num_pages, a.s.heads, page, D, a.vcs, elem, BF16, cols, box, C::BLOCKS, 1))
    return cudaErrorInvalidValue;
  const size_t places = (size_t)ctas * 2, part_bytes = places * C::BR * D * sizeof(float), ml_bytes = places * C::BR * sizeof(float2);
  void* block = nullptr;
  if ((e = scratch_alloc(dev, part_bytes + ml_bytes + (size_t)ctas * 8, a.stream, &block)) != cudaSuccess) return e;
  char* base = static_cast<char*>(block);
  constexpr int BN = C::BN;
  Params<NT, BN> p{a.s, static_cast<const uint16_t*>(a.q), a.q_token, a.q_head, static_cast<uint16_t*>(a.o), a.ks, a.vs, a.kss, a.vss,
               RowBlocks<NT, BN>{a.group, a.causal ? 1 : 0},
               (INT8 ? a.scale : fabsf(a.scale)) * 1.4426950408889634f, !INT8 && a.scale < 0.f ? 0x80008000u : 0u,
               reinterpret_cast<float*>(base), reinterpret_cast<float2*>(base + part_bytes),
               reinterpret_cast<unsigned long long*>(base + part_bytes + ml_bytes), next_call()};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  cfg.stream = a.stream;
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  if ((e = cudaLaunchKernelEx(&cfg, kern, mk, mv, p)) == cudaSuccess) {
    note_launch();
    e = cudaGetLastError();
  }
  const cudaError_t ef = cudaFreeAsync(block, a.stream);
  return e != cudaSuccess ? e : ef;
}

template <int D, bool INT8, int NT>
cudaError_t launch_d(const PagedAttnArgs& a, int dev) {
  return a.bf16 ? launch<D, true, INT8, NT>(a, dev) : launch<D, false, INT8, NT>(a, dev);
}

}  // namespace rows

// Units of 8 rows, or (8-bit caches alone, whose conversion then serves twice the rows) of 16.
cudaError_t launch_paged_attn_rows(const PagedAttnArgs& a, int dev, bool wide) {
  using namespace phantom::rows;
  if (!a.int8) return a.d == 64 ? launch_d<64, false, 1>(a, dev) : launch_d<128, false, 1>(a, dev);
  if (a.d == 64) return wide ? launch_d<64, true, 2>(a, dev) : launch_d<64, true, 1>(a, dev);
  return wide ? launch_d<128, true, 2>(a, dev) : launch_d<128, true, 1>(a, dev);
}

}  // namespace phantom
