// Attention of few query rows over a paged cache (decoding; a few new tokens). For sequence b with n new and len cached
// tokens (the new ones among them), key head h, its `group` query heads, and new token i:
//
//   o[i, g] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[i, g] . k_j),   j < len, causal: j <= len - n + i
//
// in one pass over the keys with a running maximum and sum (log2 domain). What it has to do is read the cached keys and
// values once: 2 len d elements for each key head against 2 * 2 len d operations for each query row, so with up to 16 rows
// it is bound by memory, and everything here serves the reads:
//
//   * The rows of one key head (new tokens x its query heads, token-major) are taken 16 at a time, the height of a warp's
//     matrix instruction: the keys are read once for all of them.
//   * Work is cut evenly: all (sequence, head, row block) units in a row, tiles of 64 keys, and CTA c of G takes tiles
//     [c W / G, (c + 1) W / G) of all W. Ragged lengths then cost nothing, and one long sequence spreads over the GPU. A
//     unit that several CTAs share leaves partial results (fp32 rows, reference maximum, sum), which merge_rows joins in
//     the order of the CTAs: the result depends on the lengths and the GPU's SM count alone.
//   * Two producer warps read the page table and keep a ring of tiles in flight by TMA (a box per page, swizzled, so that
//     pages of 16 tokens land as one conflict-free tile); 128 KB in flight for each SM.
//   * Eight consumer warps work without meeting: two to a tile, 32 keys each, every warp with its own running maximum,
//     sum and output; they are joined through shared memory at the end of a unit.
//
// Precision: scores and sums are fp32. 16-bit caches: P enters the second product as hi + lo (two 16-bit numbers), so its
// rounding (which alone would be as large as the output's) is gone; the tensor cores idle here and the second product is
// free. 8-bit caches: keys and values enter as the whole numbers they are (exact in fp16, and in bf16), the key's scale
// multiplies the score, and the value's goes into the exponent: p'_j = 2^(s_j + log2 vs_j - m') is p_j vs_j normalised to
// at most 1, whatever the scales, and is rounded to fp16 once; the sum adds p'_j / vs_j.
#include <cuda.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "launchers.h"
#include "paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace phantom {
namespace rows {

constexpr int BR = 16;        // query rows of a unit
constexpr int BN = 64;        // keys of a tile
constexpr int kConsumers = 8; // warps; pairs of them take the tiles in turn
constexpr int kThreads = 32 * (kConsumers + 2);  // and two producers, of keys and of values
constexpr int kErrCopyWait = 1, kErrTileWait = 4;

template <int D, bool INT8>
struct Cfg {
  static constexpr int ROW = INT8 ? D : 128;              // bytes of a swizzled row (16-bit: 64 columns)
  static constexpr int BLOCKS = INT8 ? 1 : D / 64;        // such blocks across d
  static constexpr int HALF = BN * D * (INT8 ? 1 : 2);    // keys (or values) of a tile
  static constexpr int SLOT = 2 * HALF;
  // A multiple of the four pairs: a slot's tiles then all go to one pair, which sees every phase of its barriers. (With a
  // slot passed between pairs, a pair could wait for a phase whose predecessor was still open, and parity would let it by.)
  static constexpr int SLOTS = INT8 ? (D == 128 ? 8 : 16) : (D == 128 ? 4 : 8);
  static_assert(SLOTS % 4 == 0, "each ring slot belongs to one pair of warps");
  static constexpr int OFF_MERGE = SLOTS * SLOT;          // [kConsumers][BR][D] fp32
  static constexpr int OFF_ML = OFF_MERGE + kConsumers * BR * D * 4;
  static constexpr int OFF_SCALE = OFF_ML + kConsumers * BR * 8;
  static constexpr int OFF_BAR = OFF_SCALE + (INT8 ? SLOTS * 2 * BN * 4 : 0);
  static constexpr int OFF_FLAG = OFF_BAR + 2 * SLOTS * 8;
  static constexpr int SMEM = OFF_FLAG + 16 + 1024;       // + slack to align the base
  static_assert(SMEM <= 227 * 1024, "shared memory plan exceeds 227 KB");
};


// ------------------------------------------------------------------------------------------------ units and tiles
// Units of 16 rows; tiles of 64 keys.
struct RowBlocks {
  int group, causal, heads;
  static constexpr int kTile = BN;
  __device__ int count(const Seq& x) const { return (x.n * group + BR - 1) / BR; }
  __device__ int key_end(const Seq& x, int rb) const {
    if (!causal) return x.len;
    const int last = min(x.n * group - 1, rb * BR + BR - 1) / group;
    return min(max(x.len - x.n + last + 1, 0), x.len);
  }
  __device__ long long head_tiles(const Seq& x) const { return sum_tiles(*this, x); }
};

struct Params {
  PagedSeqs s;
  const uint16_t* q;
  long long q_token, q_head;
  uint16_t* o;
  const float *ks, *vs;
  Strides3 kss, vss;
  RowBlocks blocks;
  float scale_log2;
  float* part;  // partial results, [CTA][2][BR] rows of D sums of values
  float2* ml;   // their (reference maximum, sum)
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

__device__ __forceinline__ void consumers_meet() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D, bool BF16, bool INT8>
__global__ void __launch_bounds__(kThreads, 1)
attn_rows(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params p) {
  using C = Cfg<D, INT8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  auto full = [&](int s) { return sbase + C::OFF_BAR + 8u * s; };
  auto empty = [&](int s) { return sbase + C::OFF_BAR + 8u * (C::SLOTS + s); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_FLAG);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(full(s), 2);   // the producers
      mbar_init(empty(s), 2);  // the consuming pair
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  Walk<RowBlocks> w;
  w.start(p.s, p.blocks, blockIdx.x, gridDim.x);
  const int group = p.blocks.group, causal = p.blocks.causal;
  const long long begin = w.cur;
  // Where token `row` of a tile has its column block `blk`: boxes of min(page, 64) tokens, each [block][token][ROW bytes].
  const int box_log2 = min(p.s.page_log2, 6);
  auto place_of = [&](int row, int blk) {
    return C::BLOCKS == 1 ? row * C::ROW
                          : ((((row >> box_log2) * C::BLOCKS + blk) << box_log2) + (row & ((1 << box_log2) - 1))) * C::ROW;
  };

  if (warp >= kConsumers) {
    // Producers, one of the keys and one of the values: a tile's boxes, one to a page, and an 8-bit cache's scales. One
    // elected lane of warp-uniform code issues the copies; the issue is what limits pages of 16 tokens, hence two warps.
    const bool vals = warp > kConsumers;
    const CUtensorMap* map = vals ? &tmV : &tmK;
    if (lane == 0) tma_prefetch_desc(map);
    int t = 0;
    bool ok = true;
    const int page = 1 << p.s.page_log2, box = min(page, BN);
    const Strides3 st = vals ? p.vss : p.kss;
    const float* scale = vals ? p.vs : p.ks;
    while (ok && w.cur < w.end) {
      const int end = p.blocks.key_end(w.x, w.blk), cnt = w.count();
      for (int i = 0; i < cnt; ++i, ++t) {
        const int s = t % C::SLOTS, round = t / C::SLOTS;
        const int j0 = (w.tile + i) * BN;
        const int boxes = max(0, (min(j0 + BN, end) - j0 + box - 1) / box);  // pages of the tile that hold keys
        int id = 0;
        if (lane < boxes) id = page_of(p.s, w.b, (j0 >> p.s.page_log2) + lane);
        if (round > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(empty(s), (round - 1) & 1, abort_flag, p.s.status, kErrCopyWait))))
          break;
        const int place = j0 & (page - 1);
        const uint32_t dst = sbase + s * C::SLOT + (vals ? C::HALF : 0);
        if (elect_one()) mbar_arrive_expect_tx(full(s), boxes * box * (D * (INT8 ? 1 : 2) + (INT8 ? 4 : 0)));
        for (int pg = 0; pg < boxes; ++pg) {
          const int from = __shfl_sync(0xffffffffu, id, pg);
          if (elect_one()) {
            // an id that is out of range reads as zeros (the map's bounds)
            tma_load_5d(dst + pg * box * C::BLOCKS * C::ROW, map, full(s), 0, place, 0, w.h, from);
            if constexpr (INT8)
              bulk_load(sbase + C::OFF_SCALE + (s * 2 + vals) * BN * 4 + pg * box * 4,
                        scale + max(from, 0) * st.page + w.h * st.head + place, box * 4, full(s));
          }
        }
        __syncwarp();
      }
      w.advance(p.s, p.blocks);
    }
    // every issued copy lands before this CTA's shared memory is released
    for (int i = max(0, t - C::SLOTS); i < t; ++i) mbar_wait_drain(full(i % C::SLOTS), (i / C::SLOTS) & 1);
    return;
  }

  const int g = lane >> 2, t4 = lane & 3;
  const int pair = warp >> 1, kr = (warp & 1) * 32;  // this warp's keys of its pair's tiles
  float* merge = reinterpret_cast<float*>(smem + C::OFF_MERGE);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  int t = 0;
  bool ok = true;
  while (w.cur < w.end) {
    const Seq x = w.x;
    const int cnt = w.count(), R = x.n * group, row0 = w.blk * BR, off = x.len - x.n;
    const int end = p.blocks.key_end(x, w.blk);
    // the A operand of the rows g, g + 8; 8-bit caches: columns in the order that their bytes come in (4 t4 ... + 3 of 16)
    uint32_t qa[D / 16][4];
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + g + 8 * i;
      lim[i] = r >= R ? 0 : causal ? min(x.len, off + r / group + 1) : x.len;
      const uint16_t* src = p.q + (x.tok0 + (r < R ? r / group : 0)) * p.q_token +
                            (w.h * group + (r < R ? r % group : 0)) * p.q_head;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if constexpr (INT8) {
          const uint2 y = *reinterpret_cast<const uint2*>(src + k * 16 + 4 * t4);
          qa[k][i] = r < R ? y.x : 0u;
          qa[k][2 + i] = r < R ? y.y : 0u;
        } else {
          qa[k][i] = r < R ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 2 * t4) : 0u;
          qa[k][2 + i] = r < R ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8 + 2 * t4) : 0u;
        }
      }
    }
    const int lim_least = causal ? max(0, min(x.len, off + row0 / group + 1)) : x.len;  // of the block's rows
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (int i = 0; i < cnt; ++i, ++t) {
      if ((t & 3) != pair) continue;
      const int s = t % C::SLOTS;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(full(s), (t / C::SLOTS) & 1, abort_flag, p.s.status, kErrTileWait));
      if (!ok) continue;
      const uint32_t kb = sbase + s * C::SLOT, vb = kb + C::HALF;
      const int j0 = (w.tile + i) * BN + kr;  // this warp's first key
      if (j0 < end) {
      // ---- scores: [4 groups of 8 keys][row g: keys 2 t4, + 1; row g + 8: the same]
      float sc[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
        const int row = kr + n * 8 + (lane & 7);
        if constexpr (INT8) {
          const int sw = D == 128 ? row & 7 : (row >> 1) & 3;
#pragma unroll
          for (int k = 0; k < D / 64; ++k) {
            uint32_t r[4];
            ldsm4(kb + row * C::ROW + (((k * 4 + (lane >> 3)) ^ sw) << 4), r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (BF16) {
                mma16816<true>(sc[n], qa[k * 4 + e], bytes_bf16<0x4140>(r[e]), bytes_bf16<0x4342>(r[e]));
              } else {
                const uint32_t u = r[e] ^ 0x80808080u;
                mma16816<false>(sc[n], qa[k * 4 + e], bytes_f16<0x4140>(u), bytes_f16<0x4342>(u));
              }
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            uint32_t r[4];
            const int chunk = k * 4 + (lane >> 3);
            ldsm4(kb + place_of(row, chunk >> 3) + (((chunk & 7) ^ (row & 7)) << 4), r);
            mma16816<BF16>(sc[n], qa[2 * k], r[0], r[1]);
            mma16816<BF16>(sc[n], qa[2 * k + 1], r[2], r[3]);
          }
        }
      }
      // ---- to the log2 domain; masks
      float vsc[4][2];  // 8-bit: the values' scales, then their reciprocals
      if constexpr (INT8) {
        const float* scl = reinterpret_cast<const float*>(smem + C::OFF_SCALE + s * 2 * BN * 4) + kr + 2 * t4;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 a = *reinterpret_cast<const float2*>(scl + n * 8), v = *reinterpret_cast<const float2*>(scl + BN + n * 8);
          const float k0 = a.x * p.scale_log2, k1 = a.y * p.scale_log2, l0 = __log2f(v.x), l1 = __log2f(v.y);
          sc[n][0] = fmaf(sc[n][0], k0, l0);
          sc[n][1] = fmaf(sc[n][1], k1, l1);
          sc[n][2] = fmaf(sc[n][2], k0, l0);
          sc[n][3] = fmaf(sc[n][3], k1, l1);
          vsc[n][0] = v.x;
          vsc[n][1] = v.y;
        }
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][e] *= p.scale_log2;
      }
      if (j0 + 32 > lim_least) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j0 + n * 8 + 2 * t4 + (e & 1) >= lim[e >> 1]) sc[n][e] = -CUDART_INF_F;
      }
      // ---- running maximum
      float alpha[2], sub[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y = -CUDART_INF_F;
#pragma unroll
        for (int n = 0; n < 4; ++n) y = fmaxf(y, fmaxf(sc[n][2 * h], sc[n][2 * h + 1]));
        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
        y = fmaxf(y, m[h]);
        sub[h] = y == -CUDART_INF_F ? 0.f : y;
        alpha[h] = ex2(m[h] - sub[h]);  // 0 while no key was seen
        m[h] = y;
        l[h] *= alpha[h];
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][0] *= alpha[0];
          o[n][1] *= alpha[0];
          o[n][2] *= alpha[1];
          o[n][3] *= alpha[1];
        }
      }
      // ---- probabilities
      uint32_t hi[2][4], lo[2][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = ex2(sc[n][2 * h] - sub[h]), c = ex2(sc[n][2 * h + 1] - sub[h]);
          if constexpr (INT8) {
            // masked keys: p' = 0 (their scales may be anything)
            l[h] += (a > 0.f ? __fdividef(a, vsc[n][0]) : a) + (c > 0.f ? __fdividef(c, vsc[n][1]) : c);
            hi[n >> 1][(n & 1) * 2 + h] = pack2<false>(a, c);
          } else {
            l[h] += a + c;
            const uint32_t y = pack2<BF16>(a, c);
            hi[n >> 1][(n & 1) * 2 + h] = y;
            float2 f;
            if constexpr (BF16)
              f = make_float2(__uint_as_float(y << 16), __uint_as_float(y & 0xFFFF0000u));
            else
              f = __half22float2(*reinterpret_cast<const __half2*>(&y));
            lo[n >> 1][(n & 1) * 2 + h] = pack2<BF16>(a - f.x, c - f.y);
          }
        }
      }
      // ---- values; those of keys past the end are zeroed (what lies in the page there may be anything)
      const bool tail = j0 + 32 > end;
      if constexpr (INT8) {
        uint32_t keep[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + e * 8 + 2 * t4;
          keep[e] = tail ? (j < end ? 0xffffu : 0u) | (j + 1 < end ? 0xffff0000u : 0u) : 0xffffffffu;
        }
        const int row = kr + (lane >> 3) * 8 + (lane & 7);
        const int sw = D == 128 ? row & 7 : (row >> 1) & 3;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t r[4];
          ldsm4_t(vb + row * C::ROW + ((c ^ sw) << 4), r);
          uint32_t ev[4], od[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t u = (r[e] & keep[e]) ^ 0x80808080u;
            ev[e] = bytes_f16<0x4240>(u);
            od[e] = bytes_f16<0x4341>(u);
          }
          mma16816<false>(o[2 * c], hi[0], ev[0], ev[1]);
          mma16816<false>(o[2 * c], hi[1], ev[2], ev[3]);
          mma16816<false>(o[2 * c + 1], hi[0], od[0], od[1]);
          mma16816<false>(o[2 * c + 1], hi[1], od[2], od[3]);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (tail) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = j0 + ks * 16 + e * 8 + 2 * t4;
              keep[e] = (j < end ? 0xffffu : 0u) | (j + 1 < end ? 0xffff0000u : 0u);
            }
          }
          const int row = kr + ks * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t r[4];
            const int chunk = 2 * c + (lane >> 4);
            ldsm4_t(vb + place_of(row, chunk >> 3) + (((chunk & 7) ^ (row & 7)) << 4), r);
            if (tail) {
              r[0] &= keep[0];
              r[1] &= keep[1];
              r[2] &= keep[0];
              r[3] &= keep[1];
            }
            mma16816<BF16>(o[2 * c], hi[ks], r[0], r[1]);
            mma16816<BF16>(o[2 * c + 1], hi[ks], r[2], r[3]);
            mma16816<BF16>(o[2 * c], lo[ks], r[0], r[1]);
            mma16816<BF16>(o[2 * c + 1], lo[ks], r[2], r[3]);
          }
        }
      }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(s));
    }

    // ---- join the eight warps: rows in shared memory, columns swizzled by 8 floats with the row (no bank conflicts)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int r = g + 8 * h;
      float* dst = merge + (warp * BR + r) * D;
      if (t4 == 0) ml[warp * BR + r] = make_float2(m[h], l[h]);
      if constexpr (INT8) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          *reinterpret_cast<float4*>(dst + ((16 * c + 4 * t4) ^ ((r & 3) * 8))) =
              make_float4(o[2 * c][2 * h], o[2 * c + 1][2 * h], o[2 * c][2 * h + 1], o[2 * c + 1][2 * h + 1]);
      } else {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(dst + ((8 * n + 2 * t4) ^ ((r & 3) * 8))) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
      }
    }
    consumers_meet();
    {
      constexpr int PER = D / 16;  // columns of a thread: 8 or 4
      const int r = threadIdx.x >> 4, col = (threadIdx.x & 15) * PER, row = row0 + r;
      if (row < R) {
        float M = -CUDART_INF_F, L = 0.f, acc[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll
        for (int v = 0; v < kConsumers; ++v) M = fmaxf(M, ml[v * BR + r].x);
        const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
        for (int v = 0; v < kConsumers; ++v) {
          const float2 y = ml[v * BR + r];
          const float wt = ex2(y.x - ref);
          L = fmaf(wt, y.y, L);
          const float* src = merge + (v * BR + r) * D + (col ^ ((r & 3) * 8));
#pragma unroll
          for (int i = 0; i < PER; i += 4) {
            const float4 f = *reinterpret_cast<const float4*>(src + i);
            acc[i] = fmaf(wt, f.x, acc[i]);
            acc[i + 1] = fmaf(wt, f.y, acc[i + 1]);
            acc[i + 2] = fmaf(wt, f.z, acc[i + 2]);
            acc[i + 3] = fmaf(wt, f.w, acc[i + 3]);
          }
        }
        if (cnt == w.nt) {
          const float inv = M == -CUDART_INF_F ? 0.f : 1.f / L;
          uint32_t out[PER / 2];
#pragma unroll
          for (int i = 0; i < PER / 2; ++i) out[i] = pack2<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
          uint16_t* dst = p.o + ((long long)(x.tok0 + row / group) * p.s.heads * group + w.h * group + row % group) * D + col;
          if constexpr (PER == 8)
            *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
          else
            *reinterpret_cast<uint2*>(dst) = make_uint2(out[0], out[1]);
        } else {
          const long long slot = 2LL * blockIdx.x + (begin > w.cur - w.tile ? 0 : 1);
          float* dst = p.part + (slot * BR + r) * D + col;
#pragma unroll
          for (int i = 0; i < PER; i += 4)
            *reinterpret_cast<float4*>(dst + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
          if (col == 0) p.ml[slot * BR + r] = make_float2(M, L);
        }
      }
    }
    consumers_meet();
    w.advance(p.s, p.blocks);
  }
}

// Joins the parts of the units that several CTAs of attn_rows shared: block (c, four rows) those of the unit that CTA c
// continues, if c is the first to continue it; one thread to a column, the parts in the order of the CTAs. Block (0, 0)
// also zeroes the rows of packed tokens that belong to no sequence.
template <int D, bool BF16>
__global__ void __launch_bounds__(D) merge_rows(const Params p, int grid) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int group = p.blocks.group, c0 = blockIdx.x - 1;
  if (c0 < 0) {
    if (blockIdx.y == 0) {
      const int first = min(max(p.s.cu_new[p.s.batch], 0), p.s.total);
      const long long row = (long long)p.s.heads * group * D;
      for (long long i = first * row + threadIdx.x; i < p.s.total * row; i += D) p.o[i] = 0;
    }
    return;
  }
  Walk<RowBlocks> w;
  w.start(p.s, p.blocks, c0 + 1, grid);
  const long long w0 = w.cur - w.tile;
  if (w.cur >= w.end || w.tile == 0 || w.first(c0) > w0) return;
  const int R = w.x.n * group;
  for (int r = blockIdx.y * 4; r < blockIdx.y * 4 + 4 && w.blk * BR + r < R; ++r) {
    auto slot = [&](int c) { return (2LL * c + (c > c0 ? 0 : 1)) * BR + r; };
    float M = -CUDART_INF_F, L = 0.f, acc = 0.f;
    int c1 = c0;
    for (; c1 < w.ctas && w.first(c1) < w0 + w.nt; ++c1) M = fmaxf(M, p.ml[slot(c1)].x);
    const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll 4
    for (int c = c0; c < c1; ++c) {
      const float2 y = p.ml[slot(c)];
      const float wt = ex2(y.x - ref);
      L = fmaf(wt, y.y, L);
      acc = fmaf(wt, p.part[slot(c) * D + threadIdx.x], acc);
    }
    const int row = w.blk * BR + r;
    const float out = M == -CUDART_INF_F ? 0.f : acc / L;
    p.o[((long long)(w.x.tok0 + row / group) * p.s.heads * group + w.h * group + row % group) * D + threadIdx.x] =
        (uint16_t)pack2<BF16>(out, 0.f);
  }
}

std::atomic<bool> g_attr[2][2][2][64];

template <int D, bool BF16, bool INT8>
cudaError_t launch(const PagedAttnArgs& a, int dev) {
  using C = Cfg<D, INT8>;
  int sms = 0;
  cudaError_t e = sm_count(dev, &sms);
  if (e != cudaSuccess) return e;
  std::atomic<bool>& attr = g_attr[D / 128][BF16][INT8][dev];
  if (!attr.load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(attn_rows<D, BF16, INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess)
      return e;
    attr.store(true, std::memory_order_release);
  }
  CUtensorMap mk, mv;
  const int page = 1 << a.s.page_log2, box = std::min(page, BN), elem = INT8 ? 1 : 2, cols = INT8 ? D : 64;
  if (!make_paged_map(&mk, a.kc, a.s.num_pages, a.s.heads, page, D, a.kcs, elem, BF16, cols, box, C::BLOCKS, 1) ||
      !make_paged_map(&mv, a.vc, a.s.num_pages, a.s.heads, page, D, a.vcs, elem, BF16, cols, box, C::BLOCKS, 1))
    return cudaErrorInvalidValue;
  const int ctas = sms;
  const size_t ml_bytes = (size_t)ctas * 2 * BR * sizeof(float2);
  void* block = nullptr;
  if ((e = scratch_alloc(dev, ml_bytes + (size_t)ctas * 2 * BR * D * sizeof(float), a.stream, &block)) != cudaSuccess) return e;
  Params p{a.s, static_cast<const uint16_t*>(a.q), a.q_token, a.q_head, static_cast<uint16_t*>(a.o), a.ks, a.vs, a.kss, a.vss,
           RowBlocks{a.group, a.causal ? 1 : 0, a.s.heads}, a.scale * 1.4426950408889634f,
           reinterpret_cast<float*>(static_cast<char*>(block) + ml_bytes), static_cast<float2*>(block)};
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
  e = cudaLaunchKernelEx(&cfg, attn_rows<D, BF16, INT8>, mk, mv, p);
  if (e == cudaSuccess) {
    note_launch();
    cfg.gridDim = dim3((unsigned)ctas, BR / 4);
    cfg.blockDim = dim3(D);
    cfg.dynamicSmemBytes = 0;
    if ((e = cudaLaunchKernelEx(&cfg, merge_rows<D, BF16>, p, ctas)) == cudaSuccess) note_launch();
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  const cudaError_t ef = cudaFreeAsync(block, a.stream);
  return e != cudaSuccess ? e : ef;
}

}  // namespace rows

cudaError_t launch_paged_attn_rows(const PagedAttnArgs& a, int dev) {
  using namespace rows;
  if (a.d == 64)
    return a.int8 ? (a.bf16 ? launch<64, true, true>(a, dev) : launch<64, false, true>(a, dev))
                  : (a.bf16 ? launch<64, true, false>(a, dev) : launch<64, false, false>(a, dev));
  return a.int8 ? (a.bf16 ? launch<128, true, true>(a, dev) : launch<128, false, true>(a, dev))
                : (a.bf16 ? launch<128, true, false>(a, dev) : launch<128, false, false>(a, dev));
}

}  // namespace phantom
