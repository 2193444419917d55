// The paged key/value cache: new tokens written into their pages (quantised to 8 bits on the way, where the cache is), and
// cached tokens read back packed.
//
//   8-bit cache, for each token and head:  top = max(max|x|, 127 * 2^-100),  q = round(127 x / top),  scale = top / 127
//   read back:                             x' = q * scale, rounded to the output's type
//
// round() takes ties to even, and q is the same whole number as in exact arithmetic. x has at most 11 significant bits, so
// 127 x is exact in fp32, and 127 x / top, where it is no tie, is at least 2^-19 of itself away from one; ties (x = top / 2
// gives 63.5) are not rare in 16 bits. The quotient is taken as y = 127 x * r, r = 1 / top, and corrected once by its exact
// remainder, y + (127 x - y top) r, which gives every quotient that fp32 holds, the ties among them, exactly, and the others
// to an ulp. The floor of 2^-100 keeps log2 and the reciprocal of a scale in range for the attention kernels. A vector with
// an infinity or a NaN gets the scale NaN and reads back as NaN throughout.
//
// A memory-bound pass: each vector is read once and written once. One warp takes one token: it finds the token's sequence
// and page once, then moves all heads' keys and values, 16 bytes of the cache to a lane, all of a token's loads in flight
// where it has up to 8 heads of 128. What the 8-bit forms compute must fit beside the traffic, about 10 instructions to an
// element at full bandwidth: the largest value is taken on the 16-bit patterns, two at a time, which also finds infinities
// and NaNs; the arithmetic is packed fp32; whole numbers are rounded and read off by adding 1.5 * 2^23. Alone, 22000 tokens
// of 8 heads of 128, 8 bits: written in 28.7 us (4.7 TB/s), read back in 25.6 (5.3); 18500 of 16 heads of 64, 16 bits: 27.0
// and 26.4 (5.6 and 5.7; a copy reaches 6.5).
#include <math_constants.h>

#include "launchers.h"
#include "paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace phantom {
namespace paged {

constexpr int kWarps = 8;
constexpr int kBlocksPerSm = 4;

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

// Sixteen values of a vector that LG lanes hold together: their whole numbers (packed) and the vector's scale.
template <int LG, bool BF16>
__device__ __forceinline__ uint4 quantise16(const uint4 (&in)[2], float* scale) {
  const uint32_t u[8] = {in[0].x, in[0].y, in[0].z, in[0].w, in[1].x, in[1].y, in[1].z, in[1].w};
  uint32_t big = u[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 8; ++i) big = __vmaxu2(big, u[i] & 0x7FFF7FFFu);
#pragma unroll
  for (int m = LG / 2; m > 0; m >>= 1) big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, m));
  big = max(big & 0xFFFFu, big >> 16);  // bits of max |x|
  const bool bad = big >= (BF16 ? 0x7F80u : 0x7C00u);
  float top;
  if constexpr (BF16) top = __uint_as_float(big << 16);
  else top = __half2float(__ushort_as_half((unsigned short)big));
  top = fmaxf(top, 127.f * 0x1p-100f);
  // top / 127, correctly rounded (a remainder step, as below)
  const float part = top * (1.f / 127.f);
  *scale = bad ? CUDART_NAN_F : fmaf(fmaf(-part, 127.f, top), 1.f / 127.f, part);
  float c = 127.f;
  if constexpr (BF16) {  // keeps the products and the reciprocal in range
    const float down = top > 0x1p64f ? 0x1p-64f : 1.f;
    top *= down;
    c *= down;
  }
  const float r = bad ? 0.f : __frcp_rn(top);  // (0: whole numbers of 0)
  const float2 r2 = make_float2(r, r), top2 = make_float2(-top, -top), c127 = make_float2(c, c);
  uint32_t out[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t t[8];
    float x[8];
    unpack8<BF16>(in[h], x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = mul2(make_float2(x[2 * i], x[2 * i + 1]), c127);
      float2 y = mul2(a, r2);
      y = fma2(fma2(y, top2, a), r2, y);
      y = add2(y, make_float2(12582912.f, 12582912.f));  // 1.5 * 2^23: the low byte is the whole number's
      t[2 * i] = __float_as_uint(y.x);
      t[2 * i + 1] = __float_as_uint(y.y);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      out[2 * h + i] = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0040), __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0040), 0x5410);
  }
  return bad ? make_uint4(0, 0, 0, 0) : make_uint4(out[0], out[1], out[2], out[3]);
}

// Four signed bytes (sign bits flipped) times the scale, as two packed 16-bit pairs.
template <bool BF16>
__device__ __forceinline__ uint2 scaled4(uint32_t u, float scale) {
  // 2^23 + (b + 128) has the byte as its lowest
  const float2 off = make_float2(-8388736.f, -8388736.f), s2 = make_float2(scale, scale);
  const float2 a = mul2(add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441))), off), s2);
  const float2 b = mul2(add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443))), off), s2);
  return make_uint2(pack2<BF16>(a.x, a.y), pack2<BF16>(b.x, b.y));
}

// Elements of a lane (16 bytes of the cache), lanes to a vector, vectors to a warp, such rows of vectors in flight.
template <int D, bool INT8>
struct Lanes {
  static constexpr int E = INT8 ? 16 : 8, LG = D / E, PER = 32 / LG, U = INT8 ? 2 : 4;
};

// A packed token's page and place in it; the page is -1 where it has none (said in the status word).
__device__ __forceinline__ int find_page(const PagedSeqs& s, int tok, int* place) {
  const int b = seq_index(s, tok);
  *place = 0;
  if (b >= s.batch) return -1;  // of no sequence: nothing wrong
  const Seq x = seq_of(s, b);
  const int pos = x.off + (tok - x.tok0);
  *place = pos & ((1 << s.page_log2) - 1);
  if (pos >= 0 && pos < x.len && tok >= x.tok0) return page_of(s, b, pos >> s.page_log2);
  if ((threadIdx.x & 31) == 0) atomicOr(s.status, PHANTOM_ATTN_STATUS_PAGE);
  return -1;
}

template <int D, bool BF16, bool INT8>
__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm)
append_pages(const PagedCopyArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  using L = Lanes<D, INT8>;
  constexpr int IN = L::E / 8;  // 16-byte loads of a lane's elements
  const int lane = threadIdx.x & 31, sub = lane / L::LG, c = lane % L::LG;
  const int tok = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tok < a.s.total) {
    int place;
    const int id = find_page(a.s, tok, &place);
    if (id < 0) return;
    const uint4* src[2] = {
        reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.k) + tok * a.k_token + sub * a.k_head + c * L::E),
        reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.v) + tok * a.v_token + sub * a.v_head + c * L::E)};
    const long long src_step[2] = {L::PER * a.k_head / 8, L::PER * a.v_head / 8};  // in 16 bytes
    const int bytes = INT8 ? 1 : 2;
    uint8_t* dst[2] = {static_cast<uint8_t*>(a.kc) + bytes * (id * a.kcs.page + place * a.kcs.token + sub * a.kcs.head + c * L::E),
                       static_cast<uint8_t*>(a.vc) + bytes * (id * a.vcs.page + place * a.vcs.token + sub * a.vcs.head + c * L::E)};
    const long long dst_step[2] = {bytes * L::PER * a.kcs.head, bytes * L::PER * a.vcs.head};
    float* scl[2] = {INT8 ? a.ks + id * a.kss.page + place + sub * a.kss.head : nullptr,
                     INT8 ? a.vs + id * a.vss.page + place + sub * a.vss.head : nullptr};
    for (int h = sub; h - sub < a.s.heads; h += L::PER * L::U) {
      uint4 w[2][L::U][IN];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < L::U; ++u) {
#pragma unroll
          for (int i = 0; i < IN; ++i) w[t][u][i] = h + u * L::PER < a.s.heads ? src[t][i] : make_uint4(0, 0, 0, 0);
          src[t] += src_step[t];
        }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < L::U; ++u) {
          const bool there = h + u * L::PER < a.s.heads;
          if constexpr (INT8) {
            float scale;
            const uint4 q = quantise16<L::LG, BF16>(w[t][u], &scale);
            if (there) *reinterpret_cast<uint4*>(dst[t]) = q;
            if (there && c == 0) *scl[t] = scale;
            scl[t] += L::PER * (t ? a.vss : a.kss).head;
          } else if (there) {
            *reinterpret_cast<uint4*>(dst[t]) = w[t][u][0];
          }
          dst[t] += dst_step[t];
        }
    }
  }
}

template <int D, bool BF16, bool INT8>
__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm)
read_pages(const PagedCopyArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  using L = Lanes<D, INT8>;
  const int lane = threadIdx.x & 31, sub = lane / L::LG, c = lane % L::LG;
  const int tok = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tok < a.s.total) {
    int place;
    const int id = find_page(a.s, tok, &place), page = max(id, 0);  // (nothing is read where there is none)
    const int bytes = INT8 ? 1 : 2;
    const uint8_t* src[2] = {
        static_cast<const uint8_t*>(a.kc) + bytes * (page * a.kcs.page + place * a.kcs.token + sub * a.kcs.head + c * L::E),
        static_cast<const uint8_t*>(a.vc) + bytes * (page * a.vcs.page + place * a.vcs.token + sub * a.vcs.head + c * L::E)};
    const long long src_step[2] = {bytes * L::PER * a.kcs.head, bytes * L::PER * a.vcs.head};
    const float* scl[2] = {INT8 ? a.ks + page * a.kss.page + place + sub * a.kss.head : nullptr,
                           INT8 ? a.vs + page * a.vss.page + place + sub * a.vss.head : nullptr};
    uint16_t* dst[2] = {static_cast<uint16_t*>(a.k) + tok * a.k_token + sub * a.k_head + c * L::E,
                        static_cast<uint16_t*>(a.v) + tok * a.v_token + sub * a.v_head + c * L::E};
    for (int h = sub; h - sub < a.s.heads; h += L::PER * L::U) {
      uint4 w[2][L::U];
      float scale[2][L::U];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < L::U; ++u) {
          const bool there = id >= 0 && h + u * L::PER < a.s.heads;
          w[t][u] = there ? *reinterpret_cast<const uint4*>(src[t]) : make_uint4(0, 0, 0, 0);
          src[t] += src_step[t];
          if constexpr (INT8) {
            scale[t][u] = there ? *scl[t] : 0.f;
            scl[t] += L::PER * (t ? a.vss : a.kss).head;
          }
        }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < L::U; ++u) {
          if (h + u * L::PER < a.s.heads) {
            if constexpr (INT8) {
              const uint32_t in[4] = {w[t][u].x, w[t][u].y, w[t][u].z, w[t][u].w};
              uint32_t o[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint2 y = scaled4<BF16>(in[i] ^ 0x80808080u, scale[t][u]);
                o[2 * i] = y.x;
                o[2 * i + 1] = y.y;
              }
              if (a.wide) {
                st_global_v8(dst[t], o);
              } else {
                reinterpret_cast<uint4*>(dst[t])[0] = make_uint4(o[0], o[1], o[2], o[3]);
                reinterpret_cast<uint4*>(dst[t])[1] = make_uint4(o[4], o[5], o[6], o[7]);
              }
            } else {
              *reinterpret_cast<uint4*>(dst[t]) = w[t][u];
            }
          }
          dst[t] += L::PER * (t ? a.v_head : a.k_head);
        }
    }
  }
}

template <typename Kernel>
cudaError_t launch(Kernel kern, const PagedCopyArgs& a) {
  cudaLaunchConfig_t cfg = {};
  // (a block to every eight tokens: blocks that loop over more, one wave of them, were 8% slower, their last round ragged)
  cfg.gridDim = dim3((unsigned)((a.s.total + kWarps - 1) / kWarps));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = a.stream;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return e;
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
