// Attention of many query rows over a paged cache (chunks of prompts), on the 5th-generation tensor cores: the operator of
// attn_paged.cu for units of up to 256 query rows, with the pipeline of attn_tc_sm100.cu (TMA, tcgen05.mma, scores and
// outputs in TMEM, a softmax thread per query row). What is different here:
//
//   * A unit is two tiles of 128 / group new tokens with all `group` query heads of one key head (one TMA box each; with
//     a group that does not divide 128 the tile's last rows stay unused), so shared heads cost no more key traffic.
//   * Keys and values come page by page, a TMA box each, into tiles of 128 keys.
//   * Work is cut evenly over the CTAs (paged_dev.cuh): ragged batches and single long prompts leave no partial wave. The
//     units that CTAs share leave partial results for merge_chunk.
//   * Rows of the last tile past the keys that the unit sees may hold anything (the page's stale rest, or what an earlier
//     tile left): their scores are masked by selection, and their values are zeroed, since 0 * NaN is NaN in a product.
//
//   * An 8-bit cache goes through a warpgroup that reads its pages, turns the bytes into 16-bit numbers (the whole numbers
//     themselves, exact: keys in the queries' type, values in fp16) and writes them where TMA would have put them. The
//     scales take no part in the products: the softmax multiplies a key's scale into the score and puts the value's into
//     the exponent, as in attn_paged.cu.
//
// The probabilities are rounded to the 16-bit type of V (fp16 for an 8-bit cache), as tcgen05.mma wants P and V of one type:
// half an ulp of each, which adds to the output an error of the size of its own rounding (sqrt(2) times in all); their sum
// is of the unrounded ones, in fp32. For bf16 that is coarser than fused_tc, which stages V as fp16: here that would be a
// pass over the cache, or P as hi + lo half as many matrix instructions again.
#include <cuda.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "launchers.h"
#include "paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace phantom {
namespace chunk {

constexpr int BM = 128;  // rows of a query tile = TMEM lanes
constexpr int BN = 128;  // keys of a tile
constexpr int MMA_WARP = 8, TMA_WARP = 9, PV_WARP = 10, V_WARP = 11;
constexpr int CONV_WARP = 12;  // and the three after it: 8-bit caches
// Register split (setmaxnreg, by warpgroup). 16-bit: 384 threads launch with 168 each, 2 * 216 + 72 = 3 * 168. 8-bit: 512
// threads with 128 each, 2 * 184 + 72 + 72 = 4 * 128.
constexpr int kRegsProducer = 72;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: rescale O only when the maximum grows by more than 2^8
constexpr int kErrTmaWait = 1, kErrMmaWait = 2, kErrSoftmaxWait = 4, kErrEpilogueWait = 8;
constexpr int kUnitRing = 4;

template <int D, bool INT8>
struct Cfg {
  static constexpr int THREADS = INT8 ? 512 : 384, REGS_SOFTMAX = INT8 ? 184 : 216;
  static constexpr bool SHARED_S = D == 128;       // one S region for both query tiles (d = 128), or one each
  static constexpr int KBLK = D / 64;              // 64-column (128-byte) swizzle blocks across d
  static constexpr int SUB = BN * 128;             // one such block of a tile of 128 rows
  static constexpr int TILE = BN * D * 2;
  static constexpr int STAGES = D == 128 ? 4 : 8;  // ring slots, keys and values in turn
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_OST = OFF_KV + STAGES * TILE;  // output staging: per softmax warp 32 rows of OST_COLS columns
  static constexpr int OST_COLS = INT8 ? 16 : 32, OST_WARP = 32 * 2 * OST_COLS;
  static constexpr int SCALES = INT8 ? 4 : 0;      // tiles' scales in flight: the keys', log2 of the values', 1 / these
  static constexpr int OFF_SCALE = OFF_OST + 8 * OST_WARP;
  static constexpr int OFF_RAW = OFF_SCALE + SCALES * 3 * BN * 4;  // 8-bit: bytes of the item after the one being converted
  static constexpr int OFF_IDS = OFF_RAW + (INT8 ? BN * D : 0);    // 16-bit: page ids, 64 to each of two producers
  static constexpr int OFF_BAR = OFF_IDS + (INT8 ? 0 : 2 * 64 * 4);
  static constexpr int NUM_BARS = 2 * STAGES + 7 * 2 + 3 + kUnitRing + 2 * SCALES;
  static constexpr int OFF_MISC = (OFF_BAR + NUM_BARS * 8 + 15) / 16 * 16;  // TMEM base, abort flag, unit ring
  static constexpr int SMEM = OFF_MISC + 16 + 48 * kUnitRing + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory plan exceeds 227 KB");
  // TMEM columns, as in attn_tc_sm100.cu: P never shares columns with S
  static constexpr uint32_t T_S0 = SHARED_S ? 0 : 2 * D, T_S1 = SHARED_S ? 0 : 2 * D + BN;
  static constexpr uint32_t T_P0 = SHARED_S ? BN : 2 * D + 2 * BN, T_P1 = T_P0 + BN / 2;
  static constexpr uint32_t T_O0 = SHARED_S ? 2 * BN : 0, T_O1 = T_O0 + D;
  static_assert(T_P1 + BN / 2 <= 512 && T_O1 + D <= 512, "TMEM plan exceeds 512 columns");
};

// Units of `per` new tokens; tiles of 128 keys. (Aligned for its place among the parameters: 8-bit chunks 398.3 -> 395.8 us.)
struct alignas(16) TokenBlocks {
  int per, causal;
  static constexpr int kTile = BN, kUnit = 4, kJoin = 5;
  static constexpr float kPart = 0.1f;
  __device__ int count(const Seq& x) const { return (x.n + per - 1) / per; }
  __device__ int key_end(const Seq& x, int blk) const {
    return causal ? min(max(x.off + min(x.n, (blk + 1) * per), 0), x.len) : x.len;
  }
  __device__ long long head_tiles(const Seq& x) const {
    const int c = count(x), off = x.off;
    if (c < 3) return sum_tiles(*this, x);
    if (!causal) return (long long)c * tiles_of(*this, x, 0);
    if (off < 0 || off + x.n > x.len) return sum_tiles(*this, x);
    // sum over the c - 1 whole blocks of ceil((off + i per) / 128), i = 1 ... c - 1, and the last: a sum of
    // floor((a i + r) / m), taken by the Euclidean descent on (a, m)
    long long w = tiles_of(*this, x, c - 1), n = c - 1, a = per, r = off + per + kTile - 1, m = kTile;
    for (;;) {
      w += n * (n - 1) / 2 * (a / m) + n * (r / m);
      a %= m;
      r %= m;
      const long long y = a * n + r;
      if (y < m) break;
      n = y / m;
      r = y % m;
      const long long t = m;
      m = a;
      a = t;
    }
    return w;
  }
};

struct Params {
  PagedSeqs s;
  TokenBlocks blocks;
  int group, tile_tokens;  // query heads of a key head; new tokens of a query tile
  uint16_t* o;
  float scale_log2;        // of the scores' size; their sign is in the instruction (negate)
  int negate;
  const int8_t *kc, *vc;   // 8-bit cache, read by plain loads
  const float *ks, *vs;
  Strides3 kcs, vcs, kss, vss;
  float4* part;            // partial results: [CTA][2][query tile][D / 4][row], fp32
  float2* ml;              // their (reference maximum, sum): [CTA][2][query tile][row]
  int4* starts;            // for merge_chunk, [CTA][2]: the unit that the CTA is the first to continue, or 0 CTAs
};

// What the producer tells the other roles of a unit (48 bytes).
struct Unit {
  int cnt, tile0, end, has_b;  // its tiles here, the first of them; the keys it sees; whether it has a second query tile
  int len, back, tok, tok0;    // the sequence: cached tokens, its new ones begin `back` before; the unit's first; packed place
  int h, slot, n, b;           // key head; place of the partial result (-1: the unit is whole); new tokens, -1 ends the roles
};

// NaN if a score is: the polynomial of softmax64 loses NaNs, so the row's maximum carries them.
template <int N>
__device__ __forceinline__ float row_max(const float (&s)[N]) {
  float a[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) a[k] = max_nan(s[k], s[k + 8]);
#pragma unroll
  for (int i = 16; i < N; i += 16)
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = max3_nan(a[k], s[i + k], s[i + 8 + k]);
  return max_nan(max3_nan(a[0], a[1], a[2]), max3_nan(a[3], a[4], max3_nan(a[5], a[6], a[7])));
}

// p = exp2(s * scale - sub) of 64 scores as packed 16-bit pairs; returns the sum of the unrounded values. Every fourth pair
// by the FMA pipe's polynomial, as in attn_tc_sm100.cu. That one's least value is 2^-125, in fp16 a zero; bf16 would keep it,
// and a key that the row does not see may have a value of 1e38, so bf16 takes the polynomial that ends in an exact zero.
template <bool BF16, int OFF>
__device__ __forceinline__ float softmax64(const float (&s)[BN], float scale_log2, float sub, uint32_t (&p)[32]) {
  const float2 sc = make_float2(scale_log2, scale_log2), nm = make_float2(-sub, -sub);
  float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    float2 x = fma2(make_float2(s[OFF + 2 * c], s[OFF + 2 * c + 1]), sc, nm);
    if ((0x09 >> (c & 7)) & 1) {
      x = BF16 ? exp2_fma2_zero(x) : exp2_fma2(x);
    } else {
      x.x = ex2(x.x);
      x.y = ex2(x.y);
    }
    acc[c & 1] = add2(acc[c & 1], x);
    p[c] = pack2<BF16>(x.x, x.y);
  }
  const float2 t = add2(acc[0], acc[1]);
  return t.x + t.y;
}

// The softmax of an 8-bit cache's tile. Every column has three numbers of its own (the key's scale, log2 of the value's,
// its reciprocal); with a thread to a row, each thread reads all 3 x 128 of them from shared memory, and that, 3000 cycles
// of its bandwidth for two query tiles, was what bound the kernel. So a thread takes 32 columns of four rows: lane 4 g + t
// has columns 8 i + 2 t, + 1 of rows g, g + 8, g + 16, g + 24 of its warp's 32.
struct Rows4 {
  float m[4];   // reference maximum
  float2 l[4];  // this lane's share of the sum
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = -CUDART_INF_F, l[k] = make_float2(0.f, 0.f);
  }
  // Of the row that is this lane's number.
  __device__ __forceinline__ static float of_lane(const float (&x)[4], int lane) {
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float z = __shfl_sync(0xffffffffu, x[k], (lane & 7) * 4);
      y = (lane >> 3) == k ? z : y;
    }
    return y;
  }
};

template <int D, bool BF16, bool INT8>
__global__ void __launch_bounds__(Cfg<D, INT8>::THREADS, 1)
attn_chunk(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
           const __grid_constant__ CUtensorMap tmV, const Params p) {
  using C = Cfg<D, INT8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto kv_full = [&](int s) { return bar0 + 8u * s; };
  auto kv_empty = [&](int s) { return bar0 + 8u * (C::STAGES + s); };
  constexpr int B0 = 2 * C::STAGES;
  // q_full[u & 1]: unit u is published and its queries have landed. unit_read[u & 1]: every role has read unit u's record;
  // the producer waits for that before it publishes unit u + 2, so no role is ever two phases of q_full behind.
  auto q_full = [&](int u) { return bar0 + 8u * (B0 + (u & 1)); };
  auto unit_read = [&](int u) { return bar0 + 8u * (B0 + 2 + (u & 1)); };
  auto s_full = [&](int g) { return bar0 + 8u * (B0 + 4 + g); };
  auto s_free = [&](int g) { return bar0 + 8u * (B0 + 6 + g); };
  auto p_ready = [&](int g) { return bar0 + 8u * (B0 + 8 + g); };
  auto o_done = [&](int g) { return bar0 + 8u * (B0 + 10 + g); };
  auto o_free = [&](int g) { return bar0 + 8u * (B0 + 12 + g); };
  const uint32_t q_free = bar0 + 8u * (B0 + 14), drain_bar = bar0 + 8u * (B0 + 15), drain_pv_bar = bar0 + 8u * (B0 + 16);
  // unit u's record is published (for the roles that work ahead of its queries)
  auto rec_full = [&](int u) { return bar0 + 8u * (B0 + 17 + u % kUnitRing); };
  // 8-bit: the scales of tile j of the share are there, are done with
  auto sc_full = [&](int j) { return bar0 + 8u * (B0 + 17 + kUnitRing + j % 4); };
  auto sc_empty = [&](int j) { return bar0 + 8u * (B0 + 21 + kUnitRing + j % 4); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  int4* ring = reinterpret_cast<int4*>(smem + C::OFF_MISC + 16);  // [kUnitRing][3]
  int* status = p.s.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(kv_full(s), INT8 ? 4 : 1);  // the converting warps, or TMA's issuer
      mbar_init(kv_empty(s), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(q_full(g), 1);
      mbar_init(unit_read(g), INT8 ? 14 : 11);  // eight softmax warps, two MMA warps, the warps that bring the values
      mbar_init(s_full(g), 1);
      mbar_init(s_free(g), 128);
      mbar_init(p_ready(g), 128);
      mbar_init(o_done(g), 1);
      mbar_init(o_free(g), 128);
    }
    for (int u = 0; u < kUnitRing; ++u) mbar_init(rec_full(u), 1);
    if constexpr (INT8)
      for (int j = 0; j < 4; ++j) {
        mbar_init(sc_full(j), 4);
        mbar_init(sc_empty(j), 8);
      }
    mbar_init(q_free, 1);
    mbar_init(drain_bar, 1);
    mbar_init(drain_pv_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  auto publish = [&](int u, const Unit& x) {
    int4* r = ring + 3 * (u % kUnitRing);
    r[0] = make_int4(x.cnt, x.tile0, x.end, x.has_b);
    r[1] = make_int4(x.len, x.back, x.tok, x.tok0);
    r[2] = make_int4(x.h, x.slot, x.n, x.b);
  };
  auto record = [&](int u) {
    const int4* r = ring + 3 * (u % kUnitRing);
    const int4 a = r[0], b = r[1], c = r[2];
    Unit x;
    x.cnt = a.x, x.tile0 = a.y, x.end = a.z, x.has_b = a.w;
    x.len = b.x, x.back = b.y, x.tok = b.z, x.tok0 = b.w;
    x.h = c.x, x.slot = c.y, x.n = c.z, x.b = c.w;
    return x;
  };
  auto wait = [&](uint32_t bar, int parity, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code)) != 0;
  };
  // Next unit of a consuming role (its n is -1 at the end, or when a wait gave up).
  auto next_unit = [&](int u, bool& ok) -> Unit {
    Unit x;
    x.n = -1;
    if ((ok = wait(q_full(u), (u >> 1) & 1, kErrMmaWait))) {
      x = record(u);
      __syncwarp();
      if (lane == 0) mbar_arrive(unit_read(u));
    }
    return x;
  };

  // A role that works ahead: the record of unit u as soon as it is published (n -1 at the end).
  auto take_unit = [&](int u, bool& ok) -> Unit {
    Unit x;
    x.n = -1;
    if ((ok = wait(rec_full(u), (u / kUnitRing) & 1, kErrTmaWait))) {
      x = record(u);
      __syncwarp();
      if (x.n >= 0 && lane == 0) mbar_arrive(unit_read(u));
    }
    return x;
  };

  if (warp == TMA_WARP || warp == V_WARP) {
    setmaxnreg_dec<kRegsProducer>();
    // TMA_WARP walks the CTA's share: each unit's record and queries, and (16-bit) its keys; V_WARP follows the records
    // with the values. Page ids wait in shared memory. The copies' issue is what limits pages of 16 tokens, hence the
    // two warps and, for the values, boxes of all columns (the tensor core takes V 16 keys at a time from anywhere, but K's
    // 128 keys at one stride).
    const int page_log2 = p.s.page_log2, page = 1 << page_log2, box = min(page, BN);
    const bool vals = warp == V_WARP;
    int t = vals;  // copies: keys even, values odd
    bool ok = true;
    int* ids = reinterpret_cast<int*>(smem + C::OFF_IDS) + vals * 64;  // page i's id at i % 64
    int ahead = 0, pages = 0, seq = 0, head = 0;                       // ids are there for pages below `ahead`
    auto ids_more = [&]() {
      ids[(ahead + lane) & 63] = ahead + lane < pages ? page_of(p.s, seq, ahead + lane) : 0;
      ahead += 32;
    };
    auto begin_unit = [&](int b, int h, int tile0, int end) {
      seq = b;
      head = h;
      pages = (end + page - 1) >> page_log2;
      ahead = (tile0 * BN) >> page_log2 & ~31;
      ids_more();
      ids_more();
      __syncwarp();
    };
    auto copy_tile = [&](int j0, int end) {
      const int s = t % C::STAGES, round = t / C::STAGES;
      const int boxes = max(0, (min(j0 + BN, end) - j0 + box - 1) / box);  // pages of the tile that hold keys
      const int first = j0 >> page_log2;
      if (round > 0 && !(ok = wait(kv_empty(s), (round - 1) & 1, kErrTmaWait))) return;
      if (elect_one()) {
        mbar_arrive_expect_tx(kv_full(s), boxes * box * D * 2);
        uint32_t dst = sbase + C::OFF_KV + s * C::TILE;
        const int place = j0 & (page - 1);
        // (left as a loop: the code of all roles shares the instruction cache)
#pragma unroll 1
        for (int pg = 0; pg < boxes; ++pg) {
          const int from = ids[(first + pg) & 63];  // one that is out of range reads as zeros
          if (vals) {
            tma_load_5d(dst, &tmV, kv_full(s), 0, place, 0, head, from);
            dst += box * D * 2;
          } else {
            tma_load_5d(dst, &tmK, kv_full(s), 0, place, 0, head, from);
            if constexpr (C::KBLK == 2) tma_load_5d(dst + C::SUB, &tmK, kv_full(s), 0, place, 1, head, from);
            dst += box * 128;
          }
        }
      }
      __syncwarp();
      // (a tile has at most 8 pages; those below ahead - 32, which the next ones take the place of, are done with)
      if (first >= ahead - 32 && ahead < pages) ids_more();
      __syncwarp();
      t += 2;
    };
    int nq = 0;  // phases of q_full begun
    if (vals) {
      if (!INT8) {
        if (elect_one()) tma_prefetch_desc(&tmV);
        __syncwarp();
        for (int nu = 0;; ++nu) {
          const Unit x = take_unit(nu, ok);
          if (x.n < 0) break;
          begin_unit(x.b, x.h, x.tile0, x.end);
          for (int i = 0; ok && i < x.cnt; ++i) copy_tile((x.tile0 + i) * BN, x.end);
          if (!ok) break;
        }
      }
    } else {
      if (elect_one()) {
        tma_prefetch_desc(&tmQ);
        if (!INT8) tma_prefetch_desc(&tmK);
      }
      __syncwarp();
      Walk<TokenBlocks> w;
      w.start(p.s, p.blocks, blockIdx.x, gridDim.x);
      {
        const int2 own = w.cnt > 0 && w.tile > 0 ? w.owners(blockIdx.x) : make_int2(0, 0);
        const bool first = own.y > own.x && own.x == (int)blockIdx.x - 1;
        if (elect_one()) {
          p.starts[2 * blockIdx.x] = make_int4(first ? own.y - own.x + 1 : 0, w.h, w.blk * p.blocks.per, 0);
          p.starts[2 * blockIdx.x + 1] = make_int4(w.x.tok0, w.x.n, 0, 0);
        }
        __syncwarp();
      }
      int nu = 0;
      for (;; ++nu) {
        if (nu > 1 && !(ok = wait(unit_read(nu), ((nu >> 1) - 1) & 1, kErrTmaWait))) break;
        Unit x = {};
        x.n = w.cnt > 0 ? w.x.n : -1;
        if (x.n >= 0) {
          x.b = w.b;
          x.h = w.h;
          x.cnt = w.cnt;
          x.tile0 = w.tile;
          x.end = p.blocks.key_end(w.x, w.blk);
          x.tok = w.blk * p.blocks.per;
          x.len = w.x.len, x.back = (int)min((long long)w.x.len - w.x.off, 0x7fffffffLL), x.tok0 = w.x.tok0;
          x.has_b = x.tok + p.tile_tokens < x.n;
          x.slot = x.cnt == w.nt ? -1 : w.place(blockIdx.x, w.tile == 0);
        }
        if (elect_one()) {
          publish(nu, x);
          mbar_arrive(rec_full(nu));
          if (x.n < 0) mbar_arrive(q_full(nu));
        }
        __syncwarp();
        if (x.n < 0) {
          ++nq;
          break;
        }
        if (!INT8) {
          begin_unit(x.b, x.h, x.tile0, x.end);
          copy_tile(x.tile0 * BN, x.end);  // before the wait for the last unit's queries to be done with
        }
        if (ok && nu > 0) ok = wait(q_free, (nu - 1) & 1, kErrTmaWait);
        if (!ok) break;
        if (elect_one()) {
          const int tiles = x.has_b ? 2 : 1;
          mbar_arrive_expect_tx(q_full(nu), tiles * C::KBLK * p.tile_tokens * p.group * 128);
          for (int g = 0; g < tiles; ++g)
            for (int c = 0; c < C::KBLK; ++c)
              tma_load_5d(sbase + C::OFF_Q + g * C::TILE + c * C::SUB, &tmQ, q_full(nu), 0, 0, c, x.h,
                          x.tok0 + x.tok + g * p.tile_tokens);
        }
        __syncwarp();
        ++nq;
        for (int i = 1; !INT8 && ok && i < x.cnt; ++i) copy_tile((x.tile0 + i) * BN, x.end);
        if (!ok) break;
        w.advance(p.s, p.blocks);
      }
    }
    if (!ok) *abort_flag = 1;
    // every issued copy lands before this CTA's shared memory can be released
    for (int a = max(0, nq - 2); a < nq; ++a) mbar_wait_drain(q_full(a), (a >> 1) & 1);
    for (int i = max((int)vals, t - C::STAGES); !INT8 && i < t; i += 2) mbar_wait_drain(kv_full(i % C::STAGES), (i / C::STAGES) & 1);
  } else if (INT8 && warp >= CONV_WARP) {
    setmaxnreg_dec<72>();
    // 8-bit pages to 16-bit tiles: keys of tile j, its values, keys of tile j + 1, ... A thread has one 16-byte chunk of a
    // row in every pass over 16 (d = 64: 32) rows; the next item's bytes are on their way into the place that the
    // current one's leave. Eight lanes that store together have four chunks of a column block in two rows: swizzled, these
    // meet no bank twice. Rows past the unit's end turn into whatever the page holds, numbers all (their weights are 0);
    // rows without a page into zeros, of weight like any key's where they are within the length.
    constexpr int STEP = D == 128 ? 16 : 32, N = BN / STEP;  // rows at a time; times
    const int tid = threadIdx.x - 32 * CONV_WARP;
    const int chunk = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;
    const int row_in = D == 128 ? ((lane >> 2) & 1) + 2 * (lane >> 4) + 4 * (warp & 3) : (lane >> 2) + 8 * (warp & 3);
    const int page_log2 = p.s.page_log2, page_mask = (1 << page_log2) - 1;
    // where this thread's chunk goes in pass 0, its halves by the row's swizzle (16 rows further on is 2 KB further)
    const uint32_t at = (chunk >> 2) * C::SUB + row_in * 128, c0 = (chunk & 3) * 2, sw = row_in & 7;
    const uint32_t at_lo = at + ((c0 ^ sw) << 4), at_hi = at + (((c0 + 1) ^ sw) << 4);
    int nu = 0, i = 0, j0 = 0;
    bool ok = true;
    Unit x = take_unit(0, ok);
    // Byte offsets of the tile's 16-row pieces (a page has whole ones), a lane each; -1: no page there, or no keys that the
    // unit sees.
    long long k_off = -1, v_off = -1;
    int id = -1;
    const int8_t *k_base = nullptr, *v_base = nullptr;
    auto begin_tile = [&]() {
      j0 = (x.tile0 + i) * BN;
      const int j = j0 + (lane & 7) * 16;
      id = j < x.end ? page_of(p.s, x.b, j >> page_log2) : -1;
      k_off = id < 0 ? -1 : id * p.kcs.page + (j & page_mask) * p.kcs.token;
      v_off = id < 0 ? -1 : id * p.vcs.page + (j & page_mask) * p.vcs.token;
      k_base = p.kc + x.h * p.kcs.head + (row_in & 15) * p.kcs.token + chunk * 16;
      v_base = p.vc + x.h * p.vcs.head + (row_in & 15) * p.vcs.token + chunk * 16;
    };
    // Pass n's 16 bytes of this thread lie in its own place of shared memory, filled one item ahead by its own asynchronous
    // copies (a copy group to a pass; of no bytes, which fills zeros in, where there is no page), so the roles meet nowhere
    // but at the ring.
    const uint32_t raw = sbase + C::OFF_RAW + tid * 16;
    auto load = [&](int n, const int8_t* base, long long off) {
      const long long o = __shfl_sync(0xffffffffu, off, (n * STEP + row_in) >> 4);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(raw + n * 2048), "l"(base + max(o, 0LL)),
                   "r"(o < 0 ? 0 : 16) : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto take = [&](int n, uint32_t (&in)[4]) {  // the oldest of the N groups in flight
      asm volatile("cp.async.wait_group %0;" ::"n"(N - 1) : "memory");
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(in[0]), "=r"(in[1]), "=r"(in[2]), "=r"(in[3]) : "r"(raw + n * 2048) : "memory");
    };
    float ks = 0.f, vs = 1.f;
    bool past = false;
    auto load_scales = [&]() {
      const int from = __shfl_sync(0xffffffffu, id, (tid >> 4) & 7);
      const int place = (j0 + tid) & page_mask;
      past = j0 + tid >= x.end;
      const bool none = past || from < 0;
      ks = none ? 0.f : p.ks[from * p.kss.page + x.h * p.kss.head + place];
      vs = none ? 0.f : p.vs[from * p.vss.page + x.h * p.vss.head + place];
    };
    if (x.n >= 0) {
      begin_tile();
      for (int n = 0; n < N; ++n) load(n, k_base, k_off);
      load_scales();
    }
    for (int t = 0, j = 0; ok && x.n >= 0; ++j) {
      // -- the tile's scales
      if (j >= 4 && !(ok = wait(sc_empty(j), (j / 4 - 1) & 1, kErrTmaWait))) break;
      float* scl = reinterpret_cast<float*>(smem + C::OFF_SCALE) + (j & 3) * 3 * BN;
      vs = least_scale(vs);
      scl[(tid & ~1) * 2 + (tid & 1)] = ks * p.scale_log2;  // of a pair of keys: two of these, then two of those
      scl[(tid & ~1) * 2 + (tid & 1) + 2] = past ? 0.f : __log2f(vs);
      scl[2 * BN + tid] = past || vs != vs ? 0.f : __fdividef(1.f, vs);  // (NaN: only the logarithm passes it on)
      __syncwarp();
      if (lane == 0) mbar_arrive(sc_full(j));
      // -- keys; the values' bytes take their place
      int s = t % C::STAGES;
      if (t >= C::STAGES && !(ok = wait(kv_empty(s), (t / C::STAGES - 1) & 1, kErrTmaWait))) break;
      uint32_t dst = sbase + C::OFF_KV + s * C::TILE;
#pragma unroll 1
      for (int n = 0; n < N; ++n) {  // (left as loops: the code of all roles shares the instruction cache)
        uint32_t in[4], w[8];
        take(n, in);
        load(n, v_base, v_off);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BF16) {
            w[2 * e] = bytes_bf16<0x4140>(in[e]);
            w[2 * e + 1] = bytes_bf16<0x4342>(in[e]);
          } else {
            in[e] ^= 0x80808080u;
            w[2 * e] = bytes_f16<0x4140>(in[e]);
            w[2 * e + 1] = bytes_f16<0x4342>(in[e]);
          }
        }
        st_shared_v4(dst + at_lo + n * STEP * 128, w[0], w[1], w[2], w[3]);
        st_shared_v4(dst + at_hi + n * STEP * 128, w[4], w[5], w[6], w[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kv_full(s));
      ++t;
      // -- the next tile; values; its keys' bytes take their place
      if (++i == x.cnt) {
        i = 0;
        x = take_unit(++nu, ok);
      }
      k_off = -1;
      if (x.n >= 0) begin_tile();
      s = t % C::STAGES;
      if (!ok || (t >= C::STAGES && !(ok = wait(kv_empty(s), (t / C::STAGES - 1) & 1, kErrTmaWait)))) break;
      dst = sbase + C::OFF_KV + s * C::TILE;
#pragma unroll 1
      for (int n = 0; n < N; ++n) {
        uint32_t in[4], w[8];
        take(n, in);
        load(n, k_base, k_off);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          in[e] ^= 0x80808080u;
          w[2 * e] = bytes_f16<0x4140>(in[e]);
          w[2 * e + 1] = bytes_f16<0x4342>(in[e]);
        }
        st_shared_v4(dst + at_lo + n * STEP * 128, w[0], w[1], w[2], w[3]);
        st_shared_v4(dst + at_hi + n * STEP * 128, w[4], w[5], w[6], w[7]);
      }
      if (x.n >= 0) load_scales();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kv_full(s));
      ++t;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == MMA_WARP || warp == PV_WARP) {
    setmaxnreg_dec<kRegsProducer>();
    const uint64_t dq = smem_desc_sw128(sbase + C::OFF_Q, 16, 1024);
    const uint64_t dk = smem_desc_sw128(sbase + C::OFF_KV, 16, 1024);
    auto kv_wait = [&](int t) { return wait(kv_full(t % C::STAGES), (t / C::STAGES) & 1, kErrMmaWait); };
    if (warp == MMA_WARP) {
      // S_g = Q_g K^T, per key tile for query tile A, then B (see attn_tc_sm100.cu).
      const uint32_t idesc = idesc_f16(BF16, BM, BN, false) | (p.negate ? 1u << 13 : 0u);
      auto issue = [&](int g, int stage) {
        const uint32_t a_off = (uint32_t)(g * C::TILE) >> 4, b_off = (uint32_t)(stage * C::TILE) >> 4;
        const uint32_t d_t = tmem + (g ? C::T_S1 : C::T_S0);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t o = ((kk >> 2) * C::SUB + (kk & 3) * 32) >> 4;
          mma_ss(d_t, dq + (a_off + o), dk + (b_off + o), idesc, kk > 0 ? 1u : 0u);
        }
      };
      int tb = 0, nu = 0, ks = 0;
      int qc[2] = {0, 0};
      bool ok = true;
      for (;;) {
        const Unit x = next_unit(nu, ok);
        if (x.n < 0) break;
        for (int q = 0; ok && q < x.cnt; ++q) {
          const int tk = tb + 2 * q, sk = tk % C::STAGES;
          if (!(ok = kv_wait(tk))) break;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (g == 1 && !x.has_b) continue;
            const int n_prev = C::SHARED_S ? ks : qc[g];
            if (n_prev > 0 && !(ok = wait(s_free(C::SHARED_S ? 0 : g), (n_prev - 1) & 1, kErrMmaWait))) break;
            tc_fence_after();
            if (elect_one()) {
              issue(g, sk);
              mma_commit(s_full(g));
              if (g == x.has_b) mma_commit(kv_empty(sk));
            }
            __syncwarp();
            if (C::SHARED_S) ++ks; else ++qc[g];
          }
        }
        if (!ok) break;
        if (elect_one()) mma_commit(q_free);
        __syncwarp();
        tb += 2 * x.cnt;
        ++nu;
      }
      if (elect_one()) mma_commit(drain_bar);
      __syncwarp();
      mbar_wait_drain(drain_bar, 0);
    } else {
      // O_g += P_g V: P from TMEM, V as an MN-major operand.
      constexpr uint32_t idesc = idesc_f16(BF16 && !INT8, BM, D, true);
      // V lies as boxes of `box` keys, [64-column block][key][128 bytes]
      const int box_log2 = INT8 ? 7 : min(p.s.page_log2, 7), box = 1 << box_log2;
      const uint64_t dv = smem_desc_sw128(sbase + C::OFF_KV, box * 128, 1024);
      auto place_of = [&](int key, int blk) {
        return ((((key >> box_log2) * C::KBLK + blk) << box_log2) + (key & (box - 1))) * 128;
      };
      uint32_t v_off[BN / 16];
#pragma unroll
      for (int kk = 0; kk < BN / 16; ++kk) v_off[kk] = place_of(kk * 16, 0) >> 4;
      auto issue = [&](int g, int stage, bool acc) {
        const uint32_t b_off = (uint32_t)(stage * C::TILE) >> 4;
        const uint32_t d_t = tmem + (g ? C::T_O1 : C::T_O0), p_t = tmem + (g ? C::T_P1 : C::T_P0);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          mma_ts(d_t, p_t + kk * 8, dv + (b_off + v_off[kk]), idesc, (acc || kk > 0) ? 1u : 0u);
      };
      int tb = 0, nu = 0;
      int pc[2] = {0, 0}, uc[2] = {0, 0};
      bool ok = true;
      for (;; ++nu) {
        const Unit x = next_unit(nu, ok);
        if (x.n < 0) break;
        for (int q = 0; ok && q < x.cnt; ++q) {
          const int tv = tb + 2 * q + 1, sv = tv % C::STAGES;
          if (!(ok = kv_wait(tv))) break;
          const int j0 = (x.tile0 + q) * BN;
          if (!INT8 && j0 + BN > x.end) {  // zero the values of keys past the unit's end
            for (int i = max(0, x.end - j0) * 8 + lane; i < BN * 8; i += 32)
              for (int c = 0; c < C::KBLK; ++c)
                st_shared_v4(sbase + C::OFF_KV + sv * C::TILE + place_of(i >> 3, c) + (i & 7) * 16, 0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
          for (int g = 0; g <= x.has_b; ++g) {
            if (q == 0 && uc[g] > 0 && !(ok = wait(o_free(g), (uc[g] - 1) & 1, kErrMmaWait))) break;
            if (!(ok = wait(p_ready(g), pc[g] & 1, kErrMmaWait))) break;
            tc_fence_after();
            if (elect_one()) {
              issue(g, sv, q > 0);
              mma_commit(o_done(g));
              if (g == x.has_b) mma_commit(kv_empty(sv));
            }
            __syncwarp();
            ++pc[g];
          }
        }
        if (!ok) break;
        for (int g = 0; g <= x.has_b; ++g) ++uc[g];
        tb += 2 * x.cnt;
      }
      if (elect_one()) mma_commit(drain_pv_bar);
      __syncwarp();
      mbar_wait_drain(drain_pv_bar, 0);
    }
  } else {
    // Softmax warpgroups: warps 0-3 query tile A, 4-7 tile B; thread = query row = TMEM lane (see attn_tc_sm100.cu).
    setmaxnreg_inc<C::REGS_SOFTMAX>();
    const int g = warp >> 2, r_local = threadIdx.x & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + (g ? C::T_S1 : C::T_S0);
    const uint32_t t_p = tmem + lane_off + (g ? C::T_P1 : C::T_P0);
    const uint32_t t_o = tmem + lane_off + (g ? C::T_O1 : C::T_O0);
    uint8_t* stage = smem + C::OFF_OST + warp * C::OST_WARP;
    const int row_tok = r_local / p.group;  // this row's token within the query tile
    const bool in_use = row_tok < p.tile_tokens;
    // multiplies this lane's row of O
    auto rescale_o = [&](float alpha) {
      const float2 a2 = make_float2(alpha, alpha);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t rr[32];
        tmem_ld32_wait(t_o + c * 32, rr);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 y = mul2(make_float2(__uint_as_float(rr[2 * i]), __uint_as_float(rr[2 * i + 1])), a2);
          rr[2 * i] = __float_as_uint(y.x);
          rr[2 * i + 1] = __float_as_uint(y.y);
        }
        tmem_st32(t_o + c * 32, rr);
      }
    };
    int sc = 0, oc = 0, tiles = 0;
    bool ok = true;
    for (int nu = 0;; ++nu) {
      Unit x = next_unit(nu, ok);
      if (x.n < 0) break;
      const int tb = tiles;  // the share's tiles before this unit
      tiles += x.cnt;
      if (g == 1 && !x.has_b) continue;
      const int tile_tok = x.tok + g * p.tile_tokens;
      const int see = x.len - x.back + tile_tok + 1;  // causal: keys that the tile's first row sees
      const bool causal = p.blocks.causal;
      const int lim = causal ? min(x.len, see + row_tok) : x.len;
      const int lim_least = causal ? min(x.len, see) : x.len;
      const int cnt = x.cnt, jb = x.tile0 * BN;
      float m_used = -CUDART_INF_F, l = 0.f;
      Rows4 r4;
      if constexpr (INT8) r4.start();
      bool s_ready = false;
      for (int j = 0; j < cnt; ++j) {
        if (!s_ready && !(ok = wait(s_full(g), sc & 1, kErrSoftmaxWait))) break;
        ++sc;
        tc_fence_after();
        const int j0 = jb + j * BN;
        float s[BN];
        {
          uint32_t r[BN];
          if constexpr (INT8) tmem_ld_rows4_wait(t_s, r);
          else tmem_ld128_wait(t_s, r);
#pragma unroll
          for (int i = 0; i < BN; ++i) s[i] = __uint_as_float(r[i]);
        }
        tc_fence_before();
        mbar_arrive(s_free(C::SHARED_S ? 0 : g));
        if constexpr (INT8) {
          // (s_full of this tile: the scales are there, since they were written before the keys)
          const float* scl = reinterpret_cast<const float*>(smem + C::OFF_SCALE) + ((tb + j) & 3) * 3 * BN + 4 * (lane & 3);
          if (!(ok = wait(sc_full(tb + j), ((tb + j) >> 2) & 1, kErrSoftmaxWait))) break;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 a = *reinterpret_cast<const float4*>(scl + 16 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = 64 * (k >> 1) + 4 * i + 2 * (k & 1);
              const float2 y = fma2(make_float2(s[e], s[e + 1]), make_float2(a.x, a.y), make_float2(a.z, a.w));
              s[e] = y.x, s[e + 1] = y.y;
            }
          }
          if (j0 + BN > lim_least) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = (warp & 3) * 32 + 8 * k + (lane >> 2);
              const int left = (causal ? min(x.len, see + row / p.group) : x.len) - j0 - 2 * (lane & 3);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int e = 64 * (k >> 1) + 4 * i + 2 * (k & 1);
                s[e] = 8 * i < left ? s[e] : -CUDART_INF_F;
                s[e + 1] = 8 * i + 1 < left ? s[e + 1] : -CUDART_INF_F;
              }
            }
          }
          float alpha[4], sub[4];
          bool need = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int o = 64 * (k >> 1) + 2 * (k & 1);
            float y = fmaxf(s[o], s[o + 1]);
#pragma unroll
            for (int i = 1; i < 16; ++i) y = max3(y, s[o + 4 * i], s[o + 4 * i + 1]);
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
            alpha[k] = 1.f;
            if (j == 0) {
              r4.m[k] = y;
            } else if (y > r4.m[k] + kRescaleThreshold) {
              need = true;
              alpha[k] = ex2(r4.m[k] - y);
              r4.m[k] = y;
              r4.l[k] = mul2(r4.l[k], make_float2(alpha[k], alpha[k]));
            }
            sub[k] = r4.m[k] == -CUDART_INF_F ? 0.f : r4.m[k];
          }
          if (j > 0) {
            if (!(ok = wait(o_done(g), oc & 1, kErrSoftmaxWait))) break;
            ++oc;
            tc_fence_after();
            if (__any_sync(0xffffffffu, need)) rescale_o(Rows4::of_lane(alpha, lane));
          }
          uint32_t pk[2][32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 inv = *reinterpret_cast<const float2*>(scl - 2 * (lane & 3) + 2 * BN + 8 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // (all by ex2: the polynomial's least value, 2^-125, would count in a sum that multiplies it with 1 / vs)
              const int e = 64 * (k >> 1) + 4 * i + 2 * (k & 1);
              float2 x = add2(make_float2(s[e], s[e + 1]), make_float2(-sub[k], -sub[k]));
              x = make_float2(ex2(x.x), ex2(x.y));
              r4.l[k] = fma2(x, inv, r4.l[k]);
              pk[k >> 1][2 * i + (k & 1)] = pack2<false>(x.x, x.y);
            }
          }
          tmem_st_16x128b_x16(t_p, pk[0]);
          tmem_st_16x128b_x16(t_p + (16u << 16), pk[1]);
          bool next_test = false;
          if constexpr (!C::SHARED_S) next_test = j + 1 < cnt && mbar_test(s_full(g), sc & 1);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(p_ready(g));
          __syncwarp();
          if (lane == 0) mbar_arrive(sc_empty(tb + j));
          if (lane == 0 && !x.has_b) mbar_arrive(sc_empty(tb + j));  // in the absent tile's place
          if constexpr (!C::SHARED_S) s_ready = __all_sync(0xffffffffu, next_test);
          continue;
        }
        if (j0 + BN > lim_least) {
          const int left = lim - j0;
#pragma unroll
          for (int c = 0; c < BN; ++c) s[c] = c < left ? s[c] : -CUDART_INF_F;
        }
        const float m_new = row_max<BN>(s) * p.scale_log2;
        float alpha = 1.f;
        bool need = false;
        if (j == 0) {
          m_used = m_new;
        } else {
          need = in_use && !(m_new <= m_used + kRescaleThreshold);  // (a NaN goes on to l and O)
          if (need) {
            alpha = ex2(m_used - m_new);
            m_used = m_new;
          }
          if (!(ok = wait(o_done(g), oc & 1, kErrSoftmaxWait))) break;
          ++oc;
          tc_fence_after();
          if (__any_sync(0xffffffffu, need)) rescale_o(alpha);
        }
        // (infinity less infinity is no weight: all of the row turns NaN, which the sum keeps)
        const float sub = m_used == -CUDART_INF_F ? 0.f : m_used == CUDART_INF_F ? CUDART_NAN_F : m_used;
        uint32_t pk[32];
        float psum = softmax64<BF16, 0>(s, p.scale_log2, sub, pk);
        tmem_st32(t_p, pk);
        bool next_test = false;
        if constexpr (!C::SHARED_S) next_test = j + 1 < cnt && mbar_test(s_full(g), sc & 1);
        psum += softmax64<BF16, 64>(s, p.scale_log2, sub, pk);
        tmem_st32(t_p + 32, pk);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_ready(g));
        if constexpr (!C::SHARED_S) s_ready = __all_sync(0xffffffffu, next_test);
        l = l * alpha + psum;
      }
      if (!ok) break;
      if (!(ok = wait(o_done(g), oc & 1, kErrEpilogueWait))) break;
      ++oc;
      tc_fence_after();
      if constexpr (INT8) {
        float sum[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sum[k] = r4.l[k].x + r4.l[k].y;
          sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
          sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
        }
        m_used = Rows4::of_lane(r4.m, lane);
        l = Rows4::of_lane(sum, lane);
      }
      x = record(nu);  // read again: fewer registers live across the tile loop
      if (x.slot < 0) {
        // O / l, some columns at a time through shared memory (16-byte chunks swizzled by the row: conflict-free) so that a
        // few lanes write consecutive bytes of a row
        constexpr int COLS = C::OST_COLS, NCH = COLS / 8;  // chunks of a row
        const float inv_l = m_used == -CUDART_INF_F ? 0.f : 1.f / l;
        const int rows = min(p.tile_tokens, x.n - (x.tok + g * p.tile_tokens)) * p.group;
        const long long at = (long long)(x.tok0 + x.tok + g * p.tile_tokens) * p.s.heads;
        auto place_of = [](int r, int k) { return r * 2 * COLS + ((k ^ (NCH == 4 ? (r >> 1) & 3 : (r >> 2) & 1)) << 4); };
#pragma unroll 1
        for (int cb = 0; cb < D / COLS; ++cb) {
          uint32_t w[COLS / 2];
          if constexpr (COLS == 32) {
            uint32_t rr[32];
            tmem_ld32_wait(t_o + cb * 32, rr);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              w[i] = pack2<BF16>(__uint_as_float(rr[2 * i]) * inv_l, __uint_as_float(rr[2 * i + 1]) * inv_l);
          } else {
            uint32_t rr[16];
            tmem_ld16_wait(t_o + cb * 16, rr);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[i] = pack2<BF16>(__uint_as_float(rr[2 * i]) * inv_l, __uint_as_float(rr[2 * i + 1]) * inv_l);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < NCH; ++k)
            *reinterpret_cast<uint4*>(stage + place_of(lane, k)) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < NCH; ++i) {
            const int r = (i * 32 + lane) / NCH, k = lane % NCH, row = (warp & 3) * 32 + r;
            if (row < rows) {
              const uint4 v = *reinterpret_cast<const uint4*>(stage + place_of(r, k));
              const int tok = row / p.group;
              *reinterpret_cast<uint4*>(p.o + ((at + (long long)tok * p.s.heads + x.h) * p.group + (row - tok * p.group)) * D +
                                        cb * COLS + k * 8) = v;
            }
          }
        }
      } else {
        float4* po = p.part + ((long long)x.slot * 2 + g) * (D / 4) * BM + r_local;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t rr[32];
          tmem_ld32_wait(t_o + c * 32, rr);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            po[(c * 8 + i) * BM] = make_float4(__uint_as_float(rr[4 * i]), __uint_as_float(rr[4 * i + 1]),
                                               __uint_as_float(rr[4 * i + 2]), __uint_as_float(rr[4 * i + 3]));
        }
        p.ml[((long long)x.slot * 2 + g) * BM + r_local] = make_float2(m_used, l);
      }
      tc_fence_before();
      mbar_arrive(o_free(g));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the units that several CTAs of attn_chunk shared. Block (c, query tile, 32 columns): the unit that CTA c
// is the first to continue; thread = query row and 8 columns; the parts in the order of the CTAs, four on their way at
// once, in one pass with a running maximum. Blocks (0, ...), for which there is no such unit, zero the rows of packed tokens
// that belong to no sequence.
constexpr int kMergeCols = 8, kMergeThreads = 512;
template <int D, bool BF16>
__global__ void __launch_bounds__(kMergeThreads) merge_chunk(const Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int g = blockIdx.y, c0 = blockIdx.x - 1;
  if (c0 < 0) {
    const int block = g * gridDim.z + blockIdx.z;
    zero_unowned(p.s, p.o, p.s.heads * p.group * (D / 8), block * kMergeThreads + threadIdx.x, 2 * gridDim.z * kMergeThreads);
    return;
  }
  const int4 a = p.starts[2 * blockIdx.x], b = p.starts[2 * blockIdx.x + 1];
  const int parts = a.x, h = a.y, tok = a.z + g * p.tile_tokens, tok0 = b.x, n = b.y;
  const int r = threadIdx.x % BM, col = (blockIdx.z * (kMergeThreads / BM) + threadIdx.x / BM) * kMergeCols;
  if (r >= min(p.tile_tokens, n - tok) * p.group) return;
  float M = -CUDART_INF_F, L = 0.f, acc[kMergeCols];
#pragma unroll
  for (int i = 0; i < kMergeCols; ++i) acc[i] = 0.f;
  for (int c = 0; c < parts; c += 4) {
    float2 y[4];
    float4 v[4][kMergeCols / 4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long slot = (long long)(2 * (c0 + c + k) + (c + k == 0)) * 2 + g;
      if (c + k < parts) {
        y[k] = p.ml[slot * BM + r];
#pragma unroll
        for (int i = 0; i < kMergeCols / 4; ++i) v[k][i] = p.part[slot * (D / 4) * BM + (col / 4 + i) * BM + r];
      } else {
        y[k] = make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int i = 0; i < kMergeCols / 4; ++i) v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    const float m = fmaxf(fmaxf(fmaxf(y[0].x, y[1].x), fmaxf(y[2].x, y[3].x)), M);
    const float ref = m == -CUDART_INF_F ? 0.f : m, old = ex2(M - ref);
    M = m;
    L *= old;
#pragma unroll
    for (int i = 0; i < kMergeCols; ++i) acc[i] *= old;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float wt = ex2(y[k].x - ref);
      L = fmaf(wt, y[k].y, L);
#pragma unroll
      for (int i = 0; i < kMergeCols / 4; ++i) {
        acc[4 * i] = fmaf(wt, v[k][i].x, acc[4 * i]);
        acc[4 * i + 1] = fmaf(wt, v[k][i].y, acc[4 * i + 1]);
        acc[4 * i + 2] = fmaf(wt, v[k][i].z, acc[4 * i + 2]);
        acc[4 * i + 3] = fmaf(wt, v[k][i].w, acc[4 * i + 3]);
      }
    }
  }
  if (parts == 0) return;
  const float inv = M == -CUDART_INF_F ? 0.f : 1.f / L;
  const int t = r / p.group;
  uint32_t w[kMergeCols / 2];
#pragma unroll
  for (int i = 0; i < kMergeCols / 2; ++i) w[i] = pack2<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  *reinterpret_cast<uint4*>(p.o + (((long long)(tok0 + tok + t) * p.s.heads + h) * p.group + (r - t * p.group)) * D + col) =
      make_uint4(w[0], w[1], w[2], w[3]);
}

std::atomic<bool> g_attr[2][2][2][64];

template <int D, bool BF16, bool INT8>
cudaError_t launch(const PagedAttnArgs& a, int dev) {
  using C = Cfg<D, INT8>;
  auto kern = attn_chunk<D, BF16, INT8>;
  int ctas = 0;
  cudaError_t e = sm_count(dev, &ctas);
  if (e != cudaSuccess) return e;
  std::atomic<bool>& attr = g_attr[D / 128][BF16][INT8][dev];
  if (!attr.load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess)
      return e;
    attr.store(true, std::memory_order_release);
  }
  const int page = 1 << a.s.page_log2, box = std::min(page, BN), tile_tokens = BM / a.group;
  CUtensorMap mq, mk = {}, mv = {};
  // queries as (packed token, key head, query head of it, d), boxes of one key head's rows of a tile
  const Strides3 qs{a.q_token, a.q_head * a.group, a.q_head};
  if ((!INT8 && !make_paged_map(&mk, a.kc, a.s.num_pages, a.s.heads, page, D, a.kcs, 2, BF16, 64, box, 1, 1)) ||
      (!INT8 && !make_paged_map(&mv, a.vc, a.s.num_pages, a.s.heads, page, D, a.vcs, 2, BF16, 64, box, C::KBLK, 1)) ||
      !make_paged_map(&mq, a.q, a.s.total, a.s.heads, a.group, D, qs, 2, BF16, 64, a.group, 1, tile_tokens))
    return cudaErrorInvalidValue;
  const size_t ml_bytes = (size_t)ctas * 4 * BM * sizeof(float2);
  void* block = nullptr;
  const size_t part_bytes = (size_t)ctas * 4 * BM * D * sizeof(float);
  if ((e = scratch_alloc(dev, ml_bytes + part_bytes + (size_t)ctas * 2 * sizeof(int4), a.stream, &block)) != cudaSuccess) return e;
  Params p{a.s, TokenBlocks{2 * tile_tokens, a.causal ? 1 : 0}, a.group, tile_tokens, static_cast<uint16_t*>(a.o),
           (INT8 ? a.scale : fabsf(a.scale)) * 1.4426950408889634f, !INT8 && a.scale < 0.f ? 1 : 0,
           static_cast<const int8_t*>(a.kc), static_cast<const int8_t*>(a.vc), a.ks, a.vs, a.kcs, a.vcs, a.kss, a.vss,
           reinterpret_cast<float4*>(static_cast<char*>(block) + ml_bytes), static_cast<float2*>(block),
           reinterpret_cast<int4*>(static_cast<char*>(block) + ml_bytes + part_bytes)};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  cfg.stream = a.stream;
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  e = cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, p);
  if (e == cudaSuccess) {
    note_launch();
    cfg.gridDim = dim3((unsigned)ctas, 2, D / (kMergeCols * kMergeThreads / BM));
    cfg.blockDim = dim3(kMergeThreads);
    cfg.dynamicSmemBytes = 0;
    if ((e = cudaLaunchKernelEx(&cfg, merge_chunk<D, BF16>, p)) == cudaSuccess) note_launch();
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  const cudaError_t ef = cudaFreeAsync(block, a.stream);
  return e != cudaSuccess ? e : ef;
}

}  // namespace chunk

cudaError_t launch_paged_attn_chunk(const PagedAttnArgs& a, int dev) {
  using namespace chunk;
  if (a.d == 64)
    return a.int8 ? (a.bf16 ? launch<64, true, true>(a, dev) : launch<64, false, true>(a, dev))
                  : (a.bf16 ? launch<64, true, false>(a, dev) : launch<64, false, false>(a, dev));
  return a.int8 ? (a.bf16 ? launch<128, true, true>(a, dev) : launch<128, false, true>(a, dev))
                : (a.bf16 ? launch<128, true, false>(a, dev) : launch<128, false, false>(a, dev));
}

}  // namespace phantom
