// AdamW over a list of tensors whose two moments are held in 8 bits.
//
// Blocks of 256 consecutive values of a tensor share one power-of-two scale per moment.  The first moment m is held as
// e4m3 codes, the second as e4m3 codes of its root r = sqrt(v): r spans the range of |gradient|, v would need twice the
// exponents.  One update of an element (every operation rounded to fp32 on its own, so that the result does not depend on
// how the compiler contracts):
//   g = grad * ctrl[0];  m = beta1 m + (1 - beta1) g;  v = beta2 r^2 + (1 - beta2) g^2;  r = sqrt(v)
//   p = p - p * (lr * weight_decay);  p = p - (m / (r + eps)) * step_size
// The parameter moves by the unrounded moments; then m and r are rounded for storage.
//
// Rounding.  A step changes v by a few percent at most and half a step of e4m3 is 3 to 6 %, so rounding to the nearest
// code would leave v where it is for ever.  A value is rounded up with the probability of its remainder instead, drawn from
// a hash of (seed, element number): no bias, no stored state, equal seeds give equal bits.  The scale is a power of
// two (the smallest that brings the block's largest magnitude to at most 448): the grid of codes stays the same when the
// scale does, so a value that does not change is stored without another draw.  A root above zero is never stored as
// zero: next to a live first moment a zero denominator would turn into a step of m / eps.
//
// One warp per block of 256: every lane loads eight values of p, g, m and r, the block's largest magnitudes are found
// with two warp reductions, and everything is written in the same pass: 10 bytes a parameter for 16-bit p and g.
// The tensors' addresses travel in the kernel's parameters: no device table, no copy, nothing kept between calls.
#include <cuda_fp8.h>

#include "sm100_common.cuh"

namespace msq {

constexpr int A8_BLOCK = 256;

struct Adam8Tensor {
  void* p;
  const void* g;
  uint8_t* m;
  float* ms;
  uint8_t* r;
  float* rs;
  long long n;
  int first_tile;   // tiles of the tensors before this one
  int first_block;  // blocks of the tensors before this one (numbers the elements for the draw)
};

template <int COUNT>
struct Adam8Args {
  Adam8Tensor t[COUNT];
  int count;
  int tile_blocks;  // blocks of 256 per CTA
  long long block0;  // blocks of the list before t[0] (long lists take several launches)
  float beta1, omb1, beta2, omb2, eps, decay, step_size;
  uint32_t seed_lo, seed_hi;
  const float* ctrl;
};

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Exponent of the smallest power of two that brings a magnitude with these bits to at most 448 = 1.75 * 2^8.
__device__ __forceinline__ int a8_scale_exp(uint32_t top_bits) {
  const int k = static_cast<int>((top_bits + 0x1FFFFFu) >> 23) - (127 + 8);
  return min(max(k, -110), 110);
}

// e4m3 code of a magnitude in [0, 448], rounded up with the probability of the remainder (16 random bits).
__device__ __forceinline__ uint32_t a8_encode(float mag, uint32_t rnd) {
  const uint32_t u = __float_as_uint(mag);
  const int normal = static_cast<int>((u + (rnd << 4)) >> 20) - (120 << 3);
  const int small = static_cast<int>(__fadd_rn(__fmul_rn(mag, 512.f), __fmul_rn(static_cast<float>(rnd), 1.f / 65536.f)));
  const int code = mag < 0.015625f ? small : normal;
  return u >= 0x7F800000u ? 0x7Fu : static_cast<uint32_t>(min(code, 0x7E));  // not finite: stored as NaN
}

template <int DT>
__device__ __forceinline__ void a8_load8(const void* base, long long i, float (&f)[8]) {
  if constexpr (DT == 2) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    const float4 a = q[0], b = q[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = unpack2<DT == 1>(w[j]);
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ float a8_load1(const void* base, long long i) {
  if constexpr (DT == 0) return __half2float(static_cast<const __half*>(base)[i]);
  else if constexpr (DT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  else return static_cast<const float*>(base)[i];
}

template <int PDT, int GDT, int COUNT>
__global__ void __launch_bounds__(256) adamw8_kernel(const __grid_constant__ Adam8Args<COUNT> a) {
  if (a.ctrl && a.ctrl[1] != 0.f) return;  // overflow: parameters and moments stay as they are
  const float gmul = a.ctrl ? a.ctrl[0] : 1.f;
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first_tile <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
  }
  const Adam8Tensor& t = a.t[lo];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long blocks = (t.n + A8_BLOCK - 1) / A8_BLOCK;
  const long long b0 = static_cast<long long>(static_cast<int>(blockIdx.x) - t.first_tile) * a.tile_blocks;
  const long long b1 = min(b0 + a.tile_blocks, blocks);
  const bool aligned = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) & 15) == 0 &&
                       ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.r)) & 7) == 0;
  for (long long b = b0 + warp; b < b1; b += 8) {
    const long long i0 = b * A8_BLOCK + lane * 8;
    const int live = static_cast<int>(min(8LL, max(0LL, t.n - i0)));
    const bool vec = aligned && live == 8;
    float p[8], g[8], m[8], r[8];
    const float ms = t.ms[b], rs = t.rs[b];
    uint32_t mc[2] = {0u, 0u}, rc[2] = {0u, 0u};
    if (vec) {
      a8_load8<PDT>(t.p, i0, p);
      a8_load8<GDT>(t.g, i0, g);
      const uint2 x = *reinterpret_cast<const uint2*>(t.m + i0), y = *reinterpret_cast<const uint2*>(t.r + i0);
      mc[0] = x.x; mc[1] = x.y; rc[0] = y.x; rc[1] = y.y;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = j < live;
        p[j] = in ? a8_load1<PDT>(t.p, i0 + j) : 0.f;
        g[j] = in ? a8_load1<GDT>(t.g, i0 + j) : 0.f;
        if (in) {
          mc[j >> 2] |= static_cast<uint32_t>(t.m[i0 + j]) << ((j & 3) * 8);
          rc[j >> 2] |= static_cast<uint32_t>(t.r[i0 + j]) << ((j & 3) * 8);
        }
      }
    }
    uint32_t mtop = 0u, rtop = 0u;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 mv = e4m3x2_to_float2(mc[j >> 2] >> ((j & 3) * 8)), rv = e4m3x2_to_float2(rc[j >> 2] >> ((j & 3) * 8));
      m[j] = __fmul_rn(mv.x, ms); m[j + 1] = __fmul_rn(mv.y, ms);
      r[j] = __fmul_rn(rv.x, rs); r[j + 1] = __fmul_rn(rv.y, rs);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gj = __fmul_rn(g[j], gmul);
      m[j] = __fadd_rn(__fmul_rn(m[j], a.beta1), __fmul_rn(gj, a.omb1));
      const float v = __fadd_rn(__fmul_rn(__fmul_rn(r[j], r[j]), a.beta2), __fmul_rn(__fmul_rn(gj, gj), a.omb2));
      r[j] = __fsqrt_rn(v);
      const float q = __fsub_rn(p[j], __fmul_rn(p[j], a.decay));
      p[j] = __fsub_rn(q, __fmul_rn(__fdiv_rn(m[j], __fadd_rn(r[j], a.eps)), a.step_size));
      const uint32_t mu = __float_as_uint(m[j]) & 0x7FFFFFFFu, ru = __float_as_uint(r[j]);
      if (mu < 0x7F800000u) mtop = max(mtop, mu);
      if (ru < 0x7F800000u) rtop = max(rtop, ru);
    }
    mtop = __reduce_max_sync(0xffffffffu, mtop);
    rtop = __reduce_max_sync(0xffffffffu, rtop);
    const int mk = a8_scale_exp(mtop), rk = a8_scale_exp(rtop);
    const float minv = __uint_as_float(static_cast<uint32_t>(127 - mk) << 23), rinv = __uint_as_float(static_cast<uint32_t>(127 - rk) << 23);
    // element number in the list: 256 * block + place in the block
    const unsigned long long e0 = static_cast<unsigned long long>(a.block0 + t.first_block + b) * A8_BLOCK + lane * 8;
    const uint32_t mix = hash32(static_cast<uint32_t>(e0 >> 32) ^ a.seed_hi) ^ a.seed_lo;
    mc[0] = mc[1] = rc[0] = rc[1] = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = hash32((static_cast<uint32_t>(e0) + j) ^ mix);
      const uint32_t cm = a8_encode(__fmul_rn(fabsf(m[j]), minv), bits & 0xFFFFu) | (m[j] < 0.f ? 0x80u : 0u);
      const float rj = __fmul_rn(r[j], rinv);
      uint32_t cr = a8_encode(rj, bits >> 16);
      if (cr == 0u && r[j] > 0.f) cr = 1u;
      mc[j >> 2] |= cm << ((j & 3) * 8);
      rc[j >> 2] |= cr << ((j & 3) * 8);
    }
    if (vec) {
      if constexpr (PDT == 2) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(t.p) + i0);
        q[0] = make_float4(p[0], p[1], p[2], p[3]);
        q[1] = make_float4(p[4], p[5], p[6], p[7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(t.p) + i0) =
            make_uint4(pack2<PDT == 1>(p[0], p[1]), pack2<PDT == 1>(p[2], p[3]), pack2<PDT == 1>(p[4], p[5]), pack2<PDT == 1>(p[6], p[7]));
      }
      *reinterpret_cast<uint2*>(t.m + i0) = make_uint2(mc[0], mc[1]);
      *reinterpret_cast<uint2*>(t.r + i0) = make_uint2(rc[0], rc[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < live) {
          if constexpr (PDT == 0) static_cast<__half*>(t.p)[i0 + j] = __float2half(p[j]);
          else if constexpr (PDT == 1) static_cast<__nv_bfloat16*>(t.p)[i0 + j] = __float2bfloat16(p[j]);
          else static_cast<float*>(t.p)[i0 + j] = p[j];
          t.m[i0 + j] = static_cast<uint8_t>(mc[j >> 2] >> ((j & 3) * 8));
          t.r[i0 + j] = static_cast<uint8_t>(rc[j >> 2] >> ((j & 3) * 8));
        }
      }
    }
    if (lane == 0) {
      t.ms[b] = __uint_as_float(static_cast<uint32_t>(127 + mk) << 23);
      t.rs[b] = __uint_as_float(static_cast<uint32_t>(127 + rk) << 23);
    }
  }
}

struct Adam8Hyper {
  float beta1, omb1, beta2, omb2, eps, decay, step_size;
  unsigned long long seed;
  const float* ctrl;
};

template <int PDT, int GDT, int COUNT>
static int launch_adamw8(const long long* rec, int count, long long block0, int tile_blocks, const Adam8Hyper& h, cudaStream_t stream) {
  Adam8Args<COUNT> a;
  a.count = count;
  a.tile_blocks = tile_blocks;
  a.block0 = block0;
  long long tiles = 0, blocks = 0;
  for (int i = 0; i < count; ++i) {
    const long long* q = rec + 7 * i;
    Adam8Tensor& t = a.t[i];
    t.p = reinterpret_cast<void*>(q[0]);
    t.g = reinterpret_cast<const void*>(q[1]);
    t.m = reinterpret_cast<uint8_t*>(q[2]);
    t.ms = reinterpret_cast<float*>(q[3]);
    t.r = reinterpret_cast<uint8_t*>(q[4]);
    t.rs = reinterpret_cast<float*>(q[5]);
    t.n = q[6];
    t.first_tile = static_cast<int>(tiles);
    t.first_block = static_cast<int>(blocks);
    const long long nb = (t.n + A8_BLOCK - 1) / A8_BLOCK;
    blocks += nb;
    tiles += (nb + tile_blocks - 1) / tile_blocks;
  }
  if (tiles == 0) return 0;
  if (blocks > 0x7fffffffLL || tiles > 0x7fffffffLL) return -4;
  a.beta1 = h.beta1; a.omb1 = h.omb1; a.beta2 = h.beta2; a.omb2 = h.omb2;
  a.eps = h.eps; a.decay = h.decay; a.step_size = h.step_size;
  a.seed_lo = static_cast<uint32_t>(h.seed);
  a.seed_hi = static_cast<uint32_t>(h.seed >> 32);
  a.ctrl = h.ctrl;
  adamw8_kernel<PDT, GDT, COUNT><<<static_cast<unsigned>(tiles), 256, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

}  // namespace msq

// `records`: host memory, seven 64-bit words per tensor: {p, g, codes of m, scales of m, codes of r, scales of r, elements}.
// Scales: one fp32 per block of 256 elements.  Tensors with no elements are allowed.
extern "C" int msq_adamw8_multi(const long long* records, int count, int p_dtype, int g_dtype, float beta1, float omb1,
                                float beta2, float omb2, float eps, float decay, float step_size, unsigned long long seed,
                                const float* ctrl, cudaStream_t stream) {
  using namespace msq;
  constexpr int FEW = 16, MANY = 256;
  const Adam8Hyper h{beta1, omb1, beta2, omb2, eps, decay, step_size, seed, ctrl};
  long long block0 = 0;
  for (int at = 0; at < count;) {
    const int n = count - at < MANY ? count - at : MANY;
    long long blocks = 0;
    for (int i = 0; i < n; ++i) blocks += (records[7 * (at + i) + 6] + A8_BLOCK - 1) / A8_BLOCK;
    const int tile_blocks = blocks >= 148 * 8 * 32 ? 32 : 8;
    int rc = -2;
#define MSQ_A8(PD, GD)                                                                                      \
  rc = n <= FEW ? launch_adamw8<PD, GD, FEW>(records + 7 * at, n, block0, tile_blocks, h, stream)            \
                : launch_adamw8<PD, GD, MANY>(records + 7 * at, n, block0, tile_blocks, h, stream)
    if (p_dtype == 0 && g_dtype == 0) MSQ_A8(0, 0);
    else if (p_dtype == 1 && g_dtype == 1) MSQ_A8(1, 1);
    else if (p_dtype == 2 && g_dtype == 0) MSQ_A8(2, 0);
    else if (p_dtype == 2 && g_dtype == 1) MSQ_A8(2, 1);
    else if (p_dtype == 2 && g_dtype == 2) MSQ_A8(2, 2);
    else if (p_dtype == 0 && g_dtype == 2) MSQ_A8(0, 2);
    else if (p_dtype == 1 && g_dtype == 2) MSQ_A8(1, 2);
#undef MSQ_A8
    if (rc) return rc;
    block0 += blocks;
    at += n;
  }
  return 0;
}
