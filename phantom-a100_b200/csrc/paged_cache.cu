// The paged key/value cache: new tokens written into their pages (quantised to 8 bits on the way, where the cache is), and
// cached tokens read back packed.
//
//   8-bit cache, for each token and head:  top = max(max|x|, 127 * 2^-100),  q = round(127 x / top),  scale = top / 127
//   read back:                             x' = q * scale, rounded to the output's type
//
// round() takes ties to even, and q is the same whole number as in exact arithmetic: x has at most 11 significant bits, so
// 127 x / top, where it is no tie, is at least 2^-19 of itself away from one, and where it is a tie (x = top / 2 gives
// 63.5, not rare in 16 bits) a correctly rounded fp32 division gives it exactly. The kernel multiplies by 127 / top and
// divides only where the product lies within 1e-4 of a tie. The floor of 2^-100 keeps log2 and the reciprocal of a scale in
// range for the attention kernels. A vector with an infinity or a NaN gets the scale NaN and reads back as NaN throughout.
//
// A memory-bound pass: each vector is read once and written once. One warp takes one token: it finds the token's sequence
// and page once, then moves all heads' keys and values, d / 8 lanes to a vector, kUnroll vectors in flight for each lane.
#include <math_constants.h>

#include <algorithm>

#include "launchers.h"
#include "paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace phantom {
namespace paged {

constexpr int kWarps = 8;
constexpr int kUnroll = 4;

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// Eight values of a vector that LG lanes hold together: their whole numbers (two packed words) and the vector's scale.
template <int LG>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float* scale) {
  float top = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top = fmaxf(top, fabsf(x[i]));
    bad |= !(fabsf(x[i]) < CUDART_INF_F);
  }
  top = bad ? CUDART_INF_F : top;
#pragma unroll
  for (int m = LG / 2; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
  bad = top == CUDART_INF_F;
  top = fmaxf(top, 127.f * 0x1p-100f);
  *scale = bad ? CUDART_NAN_F : __fdiv_rn(top, 127.f);
  const float inv = __fdiv_rn(127.f, top);
  const float down = top > 0x1p64f ? 0x1p-32f : 1.f;  // keeps 127 x in range
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f = x[i] * inv;
    float q = rintf(f);
    if (fabsf(f - q) > 0.4999f) q = rintf(__fdiv_rn(x[i] * down * 127.f, top * down));
    const int n = bad ? 0 : (int)q;
    w[i >> 2] |= (uint32_t)(n & 0xff) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

template <int D, bool BF16, bool INT8>
__global__ void __launch_bounds__(32 * kWarps)
append_pages(const PagedCopyArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int LG = D / 8, PER = 32 / LG;  // lanes to a vector, vectors to a warp
  const int lane = threadIdx.x & 31, sub = lane / LG, c = lane % LG;
  for (int tok = blockIdx.x * kWarps + (threadIdx.x >> 5); tok < a.s.total; tok += gridDim.x * kWarps) {
    const int b = seq_index(a.s, tok);
    if (b >= a.s.batch) continue;
    const Seq x = seq_of(a.s, b);
    const int pos = x.len - (x.tok0 + x.n - tok);
    const int id = pos < 0 || tok < x.tok0 ? -1 : page_of(a.s, b, pos >> a.s.page_log2);
    if (id < 0) {
      if (lane == 0) atomicOr(a.s.status, PHANTOM_ATTN_STATUS_PAGE);
      continue;
    }
    const int place = pos & ((1 << a.s.page_log2) - 1);
    for (int h0 = 0; h0 < a.s.heads; h0 += PER * kUnroll) {
      uint4 w[2][kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int h = h0 + u * PER + sub;
        if (h < a.s.heads) {
          w[0][u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.k) + tok * a.k_token + h * a.k_head + c * 8);
          w[1][u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.v) + tok * a.v_token + h * a.v_head + c * 8);
        } else {
          w[0][u] = w[1][u] = make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        void* cache = t ? a.vc : a.kc;
        const Strides3& st = t ? a.vcs : a.kcs;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int h = h0 + u * PER + sub;
          const long long at = id * st.page + h * st.head + place * st.token + c * 8;
          if constexpr (INT8) {
            float f[8], scale;
            unpack8<BF16>(w[t][u], f);
            const uint2 q = quantise8<LG>(f, &scale);
            if (h < a.s.heads) {
              *reinterpret_cast<uint2*>(static_cast<int8_t*>(cache) + at) = q;
              const Strides3& ss = t ? a.vss : a.kss;
              if (c == 0) (t ? a.vs : a.ks)[id * ss.page + h * ss.head + place * ss.token] = scale;
            }
          } else if (h < a.s.heads) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at) = w[t][u];
          }
        }
      }
    }
  }
}

template <int D, bool BF16, bool INT8>
__global__ void __launch_bounds__(32 * kWarps)
read_pages(const PagedCopyArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int LG = D / 8, PER = 32 / LG;
  const int lane = threadIdx.x & 31, sub = lane / LG, c = lane % LG;
  for (int tok = blockIdx.x * kWarps + (threadIdx.x >> 5); tok < a.s.total; tok += gridDim.x * kWarps) {
    const int b = seq_index(a.s, tok);
    int id = -1, pos = 0;
    if (b < a.s.batch) {
      const Seq x = seq_of(a.s, b);
      pos = x.len - (x.tok0 + x.n - tok);
      id = pos < 0 || tok < x.tok0 ? -1 : page_of(a.s, b, pos >> a.s.page_log2);
      if (id < 0 && lane == 0) atomicOr(a.s.status, PHANTOM_ATTN_STATUS_PAGE);
    }
    const int place = pos & ((1 << a.s.page_log2) - 1);
    for (int h0 = 0; h0 < a.s.heads; h0 += PER * kUnroll) {
      uint4 w[2][kUnroll];
      float scale[2][kUnroll];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Strides3& st = t ? a.vcs : a.kcs;
        const Strides3& ss = t ? a.vss : a.kss;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int h = h0 + u * PER + sub;
          const bool there = id >= 0 && h < a.s.heads;
          const long long at = there ? id * st.page + h * st.head + place * st.token + c * 8 : 0;
          w[t][u] = make_uint4(0, 0, 0, 0);
          scale[t][u] = 0.f;
          if (there) {
            if constexpr (INT8) {
              const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(t ? a.vc : a.kc) + at);
              w[t][u].x = q.x;
              w[t][u].y = q.y;
              scale[t][u] = (t ? a.vs : a.ks)[id * ss.page + h * ss.head + place * ss.token];
            } else {
              w[t][u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t ? a.vc : a.kc) + at);
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int h = h0 + u * PER + sub;
          if (h >= a.s.heads) continue;
          if constexpr (INT8) {
            const uint32_t in[2] = {w[t][u].x, w[t][u].y};
            uint32_t out[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t pair = in[i >> 1] >> (16 * (i & 1));
              out[i] = pack2<BF16>((float)(int8_t)(pair & 0xff) * scale[t][u], (float)(int8_t)((pair >> 8) & 0xff) * scale[t][u]);
            }
            w[t][u] = make_uint4(out[0], out[1], out[2], out[3]);
          }
          const long long at = t ? tok * a.v_token + h * a.v_head : tok * a.k_token + h * a.k_head;
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(t ? a.v : a.k) + at + c * 8) = w[t][u];
        }
      }
    }
  }
}

// One token to a warp, at most kBlocksPerSm blocks to an SM (their warps then loop).
constexpr int kBlocksPerSm = 8;

template <typename Kernel>
cudaError_t launch(Kernel kern, const PagedCopyArgs& a) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = sm_count(dev, &sms);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min((a.s.total + kWarps - 1) / kWarps, sms * kBlocksPerSm));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = a.stream;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, kern, a)) != cudaSuccess) return e;
  note_launch();
  return cudaGetLastError();
}

}  // namespace paged

#define PHANTOM_PAGED_DISPATCH(KERNEL)                                                                              \
  using namespace paged;                                                                                            \
  if (a.d == 64)                                                                                                    \
    return a.int8 ? (a.bf16 ? launch(KERNEL<64, true, true>, a) : launch(KERNEL<64, false, true>, a))               \
                  : (a.bf16 ? launch(KERNEL<64, true, false>, a) : launch(KERNEL<64, false, false>, a));            \
  return a.int8 ? (a.bf16 ? launch(KERNEL<128, true, true>, a) : launch(KERNEL<128, false, true>, a))               \
                : (a.bf16 ? launch(KERNEL<128, true, false>, a) : launch(KERNEL<128, false, false>, a));

cudaError_t launch_paged_append(const PagedCopyArgs& a) { PHANTOM_PAGED_DISPATCH(append_pages) }
cudaError_t launch_paged_read(const PagedCopyArgs& a) { PHANTOM_PAGED_DISPATCH(read_pages) }

#undef PHANTOM_PAGED_DISPATCH

}  // namespace phantom
