// The cut of an attention call's work (Walk of csrc/paged_dev.cuh) run on the CPU: the lanes of a warp are 32 fibers that
// take turns at its collective operations. Built by tests/test_paged_cut_host.py, which puts blocks.h (the two kernels'
// RowBlocks and TokenBlocks, as they stand in their sources) and an empty sm100_ptx.cuh beside this file's includes.
//
//   paged_cut rows8|rows16|chunk <causal> <group> <heads> <grid> <page> <width> <total> <batch> kv_lens... cu_new...
//             <changes> (<collective> <kv or cu> <index> <value>)...
//
// prints, for each CTA, its units as "cta b h blk tile cnt nt owner owner", and ends with 3 when a walk does not end.
#include <ucontext.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <string>
#include <vector>

#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

struct Index {
  int x;
};
static Index threadIdx;
using std::max;
using std::min;

static int g_lane, g_alive;
static ucontext_t g_main, g_fiber[32];
static bool g_done[32];
static uint64_t g_slot[2][32];
static long long g_collectives;
static long long g_limit = 200000;
static std::vector<std::function<bool(long long)>> g_changes;

static void next_lane() {
  const int me = g_lane;
  for (int i = 1; i <= 32; ++i) {
    const int to = (me + i) % 32;
    if (g_done[to]) continue;
    g_lane = threadIdx.x = to;
    if (to != me) swapcontext(&g_fiber[me], &g_fiber[to]);
    g_lane = threadIdx.x = me;
    return;
  }
}
// Every lane's value of one collective; lanes reach it in turn, so when lane 0 runs again all have written.
static const uint64_t* exchange(uint64_t x) {
  static int parity[32];
  uint64_t* slot = g_slot[parity[g_lane] ^= 1];
  slot[g_lane] = x;
  next_lane();
  if (g_lane == 0) {
    ++g_collectives;
    for (auto& c : g_changes) c(g_collectives);
    if (g_collectives > g_limit) {
      printf("a walk does not end\n");
      exit(3);
    }
  }
  return slot;
}
template <typename T>
T as(uint64_t x) {
  T y;
  __builtin_memcpy(&y, &x, sizeof y);
  return y;
}
template <typename T>
uint64_t bits(T x) {
  uint64_t y = 0;
  __builtin_memcpy(&y, &x, sizeof x);
  return y;
}
template <typename T>
T __shfl_sync(unsigned, T x, int from) { return as<T>(exchange(bits(x))[from & 31]); }
template <typename T>
T __shfl_up_sync(unsigned, T x, int d) {
  const uint64_t* s = exchange(bits(x));
  return g_lane >= d ? as<T>(s[g_lane - d]) : x;
}
inline unsigned __ballot_sync(unsigned, bool p) {
  const uint64_t* s = exchange(p);
  unsigned y = 0;
  for (int i = 0; i < 32; ++i) y |= (unsigned)(s[i] & 1) << i;
  return y;
}
inline unsigned __reduce_add_sync(unsigned, unsigned x) {
  const uint64_t* s = exchange(x);
  unsigned y = 0;
  for (int i = 0; i < 32; ++i) y += (unsigned)s[i];
  return y;
}
inline int __reduce_max_sync(unsigned, int x) {
  const uint64_t* s = exchange((uint32_t)x);
  int y = (int)s[0];
  for (int i = 1; i < 32; ++i) y = max(y, (int)s[i]);
  return y;
}
inline int __popc(unsigned x) { return __builtin_popcount(x); }
inline int __ffs(unsigned x) { return __builtin_ffs((int)x); }
inline int atomicOr(int* p, int x) { return *p |= x, 0; }
inline uint32_t __byte_perm(uint32_t, uint32_t, uint32_t) { return 0; }

#include "paged_dev.cuh"

using namespace phantom;
#include "blocks.h"

static std::vector<int> g_table;

template <typename Blocks>
static void walk(const PagedSeqs& s, const Blocks& k, int grid) {
  for (int cta = 0; cta < grid; ++cta) {
    static std::function<void()> body;
    body = [&]() {
      Walk<Blocks> w;
      w.start(s, k, cta, grid);
      for (; w.cnt > 0; w.advance(s, k)) {
        const int2 own = w.owners(cta);
        if (g_lane == 0) {
          printf("%d %d %d %d %d %d %d %d %d\n", cta, w.b, w.h, w.blk, w.tile, w.cnt, w.nt, own.x, own.y);
          if (++g_collectives > g_limit) {
            printf("a walk does not end\n");
            exit(3);
          }
        }
        __shfl_sync(0xffffffffu, 0, 0);
      }
      g_done[g_lane] = true;
      if (--g_alive == 0) setcontext(&g_main);
      next_lane();
    };
    static std::vector<std::vector<char>> stacks(32, std::vector<char>(256 << 10));
    g_alive = 32;
    g_collectives = 0;
    for (int i = 0; i < 32; ++i) {
      g_done[i] = false;
      getcontext(&g_fiber[i]);
      g_fiber[i].uc_stack.ss_sp = stacks[i].data();
      g_fiber[i].uc_stack.ss_size = stacks[i].size();
      g_fiber[i].uc_link = &g_main;
      makecontext(&g_fiber[i], (void (*)())+[]() { body(); }, 0);
    }
    g_lane = threadIdx.x = 0;
    swapcontext(&g_main, &g_fiber[0]);
  }
}

int main(int argc, char** argv) {
  int at = 1;
  const std::string kind = argv[at++];
  auto number = [&]() { return at < argc ? atoi(argv[at++]) : 0; };
  const int causal = number(), group = number(), heads = number(), grid = number(), page = number(), width = number(), total = number();
  const int batch = number();
  std::vector<int> kv(batch), cu(batch + 1);
  for (int& x : kv) x = number();
  for (int& x : cu) x = number();
  for (int n = number(); n > 0; --n) {
    const long long when = number();
    std::vector<int>& v = number() ? cu : kv;
    const int i = number(), value = number();
    g_changes.push_back([&v, i, value, when](long long c) { return c == when && (v[i] = value, true); });
  }
  int status = 0, page_log2 = 0;
  while ((1 << page_log2) < page) ++page_log2;
  const PagedSeqs s{nullptr, kv.data(), cu.data(), batch, width, width, total, 1, page_log2, heads, &status};
  if (kind == "rows8") walk(s, RowBlocks<1, 64>{group, causal}, grid);
  if (kind == "rows16") walk(s, RowBlocks<2, 128>{group, causal}, grid);
  if (kind == "chunk") walk(s, TokenBlocks{2 * (128 / group), causal}, grid);
  return 0;
}
