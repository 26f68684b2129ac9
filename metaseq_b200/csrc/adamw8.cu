// AdamW over a list of tensors whose two moments are held in 8 bits.
//
// Blocks of 256 consecutive values of a tensor share one power-of-two scale per moment.  The first moment m is held as
// e4m3 codes, the second as e4m3 codes of its root r = sqrt(v): r spans the range of |gradient|, v would need twice the
// exponents.  One update of an element (fp32; the operations that make m and v are rounded one by one, so that the scales,
// which come from comparing the largest of them with a power of two, do not depend on contraction; root and quotient use
// the hardware's approximations, 2^-22, except for the root of the largest v that sets the scale):
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
  float beta1, omb1, beta2, omb2, eps, decay, step_size, minus_zero;
  uint32_t seed_lo, seed_hi;
  const float* ctrl;
};

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Exponent of the smallest power of two that brings a finite magnitude with these bits to at most 448 = 1.75 * 2^8.
__device__ __forceinline__ int a8_scale_exp(uint32_t top_bits) {
  return max(static_cast<int>((top_bits + 0x1FFFFFu) >> 23) - (127 + 8), -110);
}

// e4m3 code of a magnitude in [0, 448], rounded up with the probability of the remainder (16 random bits).  Normal codes: the
// bits below the three of the mantissa are the remainder.  Below 2^-6 codes are multiples of 2^-9: mag * 512 + 128 is a
// float whose last bit is 2^-16, so its mantissa is the fixed-point number with 16 fractional bits.
__device__ __forceinline__ uint32_t a8_encode(float mag, uint32_t rnd) {
  const uint32_t normal = ((__float_as_uint(mag) + (rnd << 4)) >> 20) - (120u << 3);
  const uint32_t small = (__float_as_uint(fmaf(mag, 512.f, 128.f)) - 0x43000000u + rnd) >> 16;
  return mag < 0.015625f ? small : normal;
}

struct Adam8Consts {
  float gmul, beta1, omb1, beta2, omb2, eps, decay, step_size, minus_zero;
};

__device__ __forceinline__ float a8_lo(uint64_t v) { float a, b; f2_unpack(v, a, b); return a; }
__device__ __forceinline__ float a8_hi(uint64_t v) { float a, b; f2_unpack(v, a, b); return b; }
__device__ __forceinline__ uint64_t a8_two(float x) { return f2_pack(x, x); }

// A product that is rounded before it is added to something.  A packed product and the packed sum behind it are contracted in
// spite of their rounding modifiers; a fused multiply-add of a -0 that only the caller knows is not.
__device__ __forceinline__ uint64_t a8_mul_rounded(uint64_t a, uint64_t b, float minus_zero) {
  return f2_fma(a, b, f2_pack(minus_zero, minus_zero));
}

// The update of a lane's eight values (pairs of fp32 in 64-bit registers: one instruction works on both).  mc / rc: codes in
// and out, ms / rs: the block's scales in and out.  All lanes of the warp take part (two reductions).
__device__ __forceinline__ void a8_update8(uint64_t (&p)[4], const uint64_t (&grad)[4], uint32_t (&mc)[2], uint32_t (&rc)[2],
                                           float& ms, float& rs, const Adam8Consts& c, uint32_t e0, uint32_t mix) {
  uint64_t m[4], r[4];
  uint32_t mtop = 0u, vtop = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int sh = (j & 1) * 16;
    const float2 mv = e4m3x2_to_float2(mc[j >> 1] >> sh), rv = e4m3x2_to_float2(rc[j >> 1] >> sh);
    const uint64_t g = f2_mul(grad[j], a8_two(c.gmul));
    m[j] = f2_mul(f2_pack(mv.x, mv.y), a8_two(ms));
    r[j] = f2_mul(f2_pack(rv.x, rv.y), a8_two(rs));
    m[j] = f2_add(a8_mul_rounded(m[j], a8_two(c.beta1), c.minus_zero), a8_mul_rounded(g, a8_two(c.omb1), c.minus_zero));
    const uint64_t v = f2_add(a8_mul_rounded(f2_mul(r[j], r[j]), a8_two(c.beta2), c.minus_zero),
                              a8_mul_rounded(f2_mul(g, g), a8_two(c.omb2), c.minus_zero));
    const float v0 = a8_lo(v), v1 = a8_hi(v);
    mtop = max(mtop, max(__float_as_uint(a8_lo(m[j])) & 0x7FFFFFFFu, __float_as_uint(a8_hi(m[j])) & 0x7FFFFFFFu));
    vtop = max(vtop, max(__float_as_uint(v0), __float_as_uint(v1)));
    r[j] = f2_pack(sqrtf(v0), sqrtf(v1));
    const uint64_t d = f2_add(r[j], a8_two(c.eps));
    const uint64_t q = f2_mul(m[j], f2_pack(__fdividef(1.f, a8_lo(d)), __fdividef(1.f, a8_hi(d))));
    p[j] = f2_fma(p[j], a8_two(-c.decay), p[j]);
    p[j] = f2_fma(q, a8_two(-c.step_size), p[j]);
  }
  mtop = __reduce_max_sync(0xffffffffu, mtop);
  vtop = __reduce_max_sync(0xffffffffu, vtop);
  const bool finite = mtop < 0x7F800000u && vtop < 0x7F800000u;
  if (!finite) {  // the scales come from the finite values
    mtop = vtop = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = __float_as_uint(a8_lo(m[j])) & 0x7FFFFFFFu, b = __float_as_uint(a8_hi(m[j])) & 0x7FFFFFFFu;
      if (a < 0x7F800000u) mtop = max(mtop, a);
      if (b < 0x7F800000u) mtop = max(mtop, b);
      const uint32_t x = __float_as_uint(a8_lo(r[j])), y = __float_as_uint(a8_hi(r[j]));
      if (x < 0x7F800000u) vtop = max(vtop, x);
      if (y < 0x7F800000u) vtop = max(vtop, y);
    }
    mtop = __reduce_max_sync(0xffffffffu, mtop);
    vtop = __reduce_max_sync(0xffffffffu, vtop);
  } else {
    vtop = __float_as_uint(__fsqrt_rn(__uint_as_float(vtop)));
  }
  const int mk = a8_scale_exp(mtop), rk = a8_scale_exp(vtop);
  ms = __uint_as_float(static_cast<uint32_t>(127 + mk) << 23);
  rs = __uint_as_float(static_cast<uint32_t>(127 + rk) << 23);
  const uint64_t minv = a8_two(__uint_as_float(static_cast<uint32_t>(127 - mk) << 23));
  const uint64_t rinv = a8_two(__uint_as_float(static_cast<uint32_t>(127 - rk) << 23));
  uint32_t cm[8], cr[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t mm = f2_mul(m[j], minv), rr = f2_mul(r[j], rinv);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = 2 * j + h;
      const uint32_t bits = hash32((e0 + k) ^ mix);
      const float mj = h ? a8_hi(mm) : a8_lo(mm), rj = h ? a8_hi(rr) : a8_lo(rr);
      const uint32_t root = __float_as_uint(h ? a8_hi(r[j]) : a8_lo(r[j]));
      cm[k] = a8_encode(fabsf(mj), bits & 0xFFFFu) | ((__float_as_uint(mj) >> 24) & 0x80u);
      cr[k] = max(a8_encode(rj, bits >> 16), min(root, 1u));  // a root above zero is not stored as zero
    }
  }
  if (!finite) {  // stored as NaN
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint64_t mp = m[k >> 1], rp = r[k >> 1];
      const uint32_t a = __float_as_uint((k & 1) ? a8_hi(mp) : a8_lo(mp)), x = __float_as_uint((k & 1) ? a8_hi(rp) : a8_lo(rp));
      if ((a & 0x7FFFFFFFu) >= 0x7F800000u) cm[k] = 0x7Fu | ((a >> 24) & 0x80u);
      if (x >= 0x7F800000u) cr[k] = 0x7Fu;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mc[h] = __byte_perm(__byte_perm(cm[4 * h], cm[4 * h + 1], 0x0040), __byte_perm(cm[4 * h + 2], cm[4 * h + 3], 0x0040), 0x5410);
    rc[h] = __byte_perm(__byte_perm(cr[4 * h], cr[4 * h + 1], 0x0040), __byte_perm(cr[4 * h + 2], cr[4 * h + 3], 0x0040), 0x5410);
  }
}

// Eight consecutive values as loaded, and as four pairs of fp32.
template <int DT>
struct Raw8 {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* base, long long i) {
    if constexpr (DT == 2) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
      a = q[0];
      b = q[1];
    } else {
      a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    }
  }
  __device__ __forceinline__ void unpack(uint64_t (&f)[4]) const {
    if constexpr (DT == 2) {
      f[0] = f2_pack_bits(a.x, a.y); f[1] = f2_pack_bits(a.z, a.w);
      f[2] = f2_pack_bits(b.x, b.y); f[3] = f2_pack_bits(b.z, b.w);
    } else {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = unpack2<DT == 1>(w[j]);
        f[j] = f2_pack(t.x, t.y);
      }
    }
  }
};
template <int DT>
__device__ __forceinline__ void a8_store8(void* base, long long i, const uint64_t (&f)[4]) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) f2_unpack(f[j], x[2 * j], x[2 * j + 1]);
  if constexpr (DT == 2) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    q[0] = make_float4(x[0], x[1], x[2], x[3]);
    q[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) =
        make_uint4(pack2<DT == 1>(x[0], x[1]), pack2<DT == 1>(x[2], x[3]), pack2<DT == 1>(x[4], x[5]), pack2<DT == 1>(x[6], x[7]));
  }
}
template <int DT>
__device__ __forceinline__ float a8_load1(const void* base, long long i) {
  if constexpr (DT == 0) return __half2float(static_cast<const __half*>(base)[i]);
  else if constexpr (DT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  else return static_cast<const float*>(base)[i];
}
template <int DT>
__device__ __forceinline__ void a8_store1(void* base, long long i, float v) {
  if constexpr (DT == 0) static_cast<__half*>(base)[i] = __float2half(v);
  else if constexpr (DT == 1) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16(v);
  else static_cast<float*>(base)[i] = v;
}

template <int PDT, int GDT, int COUNT>
__global__ void __launch_bounds__(256) adamw8_kernel(const __grid_constant__ Adam8Args<COUNT> a) {
  if (a.ctrl && a.ctrl[1] != 0.f) return;  // overflow: parameters and moments stay as they are
  const Adam8Consts c{a.ctrl ? a.ctrl[0] : 1.f, a.beta1, a.omb1, a.beta2, a.omb2, a.eps, a.decay, a.step_size, a.minus_zero};
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
  // element number in the list: 256 * block + place in the block
  auto number = [&](long long b) { return static_cast<unsigned long long>(a.block0 + t.first_block + b) * A8_BLOCK + lane * 8; };
  auto mix_of = [&](unsigned long long e) { return hash32(static_cast<uint32_t>(e >> 32) ^ a.seed_hi) ^ a.seed_lo; };

  long long b = b0 + warp;
  if (aligned) {
    // whole blocks; the next block's loads are under way while this one is computed
    const long long whole = min(b1, t.n / A8_BLOCK);
    Raw8<PDT> pn;
    Raw8<GDT> gn;
    uint2 mn, rn;
    float msn, rsn;
    auto fetch = [&](long long k) {
      const long long i = k * A8_BLOCK + lane * 8;
      pn.load(t.p, i);
      gn.load(t.g, i);
      mn = *reinterpret_cast<const uint2*>(t.m + i);
      rn = *reinterpret_cast<const uint2*>(t.r + i);
      msn = t.ms[k];
      rsn = t.rs[k];
    };
    if (b < whole) fetch(b);
    for (; b < whole; b += 8) {
      uint64_t p[4], g[4];
      uint32_t mc[2] = {mn.x, mn.y}, rc[2] = {rn.x, rn.y};
      float ms = msn, rs = rsn;
      pn.unpack(p);
      gn.unpack(g);
      if (b + 8 < whole) fetch(b + 8);
      const unsigned long long e = number(b);
      a8_update8(p, g, mc, rc, ms, rs, c, static_cast<uint32_t>(e), mix_of(e));
      const long long i = b * A8_BLOCK + lane * 8;
      a8_store8<PDT>(t.p, i, p);
      *reinterpret_cast<uint2*>(t.m + i) = make_uint2(mc[0], mc[1]);
      *reinterpret_cast<uint2*>(t.r + i) = make_uint2(rc[0], rc[1]);
      if (lane == 0) {
        t.ms[b] = ms;
        t.rs[b] = rs;
      }
    }
  }
  for (; b < b1; b += 8) {  // a tensor's last, shorter block, and tensors that are not aligned
    const long long i0 = b * A8_BLOCK + lane * 8;
    const int live = static_cast<int>(min(8LL, max(0LL, t.n - i0)));
    float pf[8], gf[8];
    uint32_t mc[2] = {0u, 0u}, rc[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = j < live;
      pf[j] = in ? a8_load1<PDT>(t.p, i0 + j) : 0.f;
      gf[j] = in ? a8_load1<GDT>(t.g, i0 + j) : 0.f;
      if (in) {
        mc[j >> 2] |= static_cast<uint32_t>(t.m[i0 + j]) << ((j & 3) * 8);
        rc[j >> 2] |= static_cast<uint32_t>(t.r[i0 + j]) << ((j & 3) * 8);
      }
    }
    uint64_t p[4], g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = f2_pack(pf[2 * j], pf[2 * j + 1]);
      g[j] = f2_pack(gf[2 * j], gf[2 * j + 1]);
    }
    float ms = t.ms[b], rs = t.rs[b];
    const unsigned long long e = number(b);
    a8_update8(p, g, mc, rc, ms, rs, c, static_cast<uint32_t>(e), mix_of(e));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < live) {
        a8_store1<PDT>(t.p, i0 + j, (j & 1) ? a8_hi(p[j >> 1]) : a8_lo(p[j >> 1]));
        t.m[i0 + j] = static_cast<uint8_t>(mc[j >> 2] >> ((j & 3) * 8));
        t.r[i0 + j] = static_cast<uint8_t>(rc[j >> 2] >> ((j & 3) * 8));
      }
    }
    if (lane == 0) {
      t.ms[b] = ms;
      t.rs[b] = rs;
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
  a.eps = h.eps; a.decay = h.decay; a.step_size = h.step_size; a.minus_zero = -0.0f;
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
