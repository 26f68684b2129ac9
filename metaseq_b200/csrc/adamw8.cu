// AdamW over a list of tensors whose two moments are held in 8 bits.
//
// Blocks of 256 consecutive values of a tensor share one power-of-two scale per moment.  The first moment m is held as
// e4m3 codes, the second as e4m3 codes of its root r = sqrt(v): r spans the range of |gradient|, v would need twice the
// exponents.  One update of an element (fp32; the operations that make m and v are rounded one by one, so that the scales,
// which come from comparing the largest of them with a power of two, do not depend on contraction; the quotient uses the
// hardware's reciprocal, 2^-22):
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
// One warp per block of 256: every lane takes eight values of p, g, m and r from a ring of asynchronous copies, the
// block's largest magnitudes are found with two warp reductions, and everything is written in the same pass: 10 bytes a
// parameter for 16-bit p and g.  What bounds it is instruction issue, about 56 per element (403M bf16 parameters: 0.85 to 0.90 ms by GPU,
// 4.5 to 4.7 TB/s; the bytes alone would take 0.63 ms.  The hardware's root alone saves 0.06 ms, but one code in 2^18 is another).
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

// Storage codes.  x * 2^-120 has its e4m3 code in bits 20 .. 26 of the fp32 pattern: the normal codes as they are, and the
// codes below 2^-6, multiples of 2^-9, as fp32 denormals (these products do not flush them).  The bits underneath are the
// remainder; adding 16 random bits on top of them rounds up with its probability, for both kinds alike.  The sum is formed
// four bits higher (multiply-adds: the ALU pipe is what bounds this kernel), so that the code is the top byte.
__device__ __forceinline__ uint32_t a8_code_top(uint32_t bits, uint32_t rnd_256) { return bits * 16u + rnd_256; }
__device__ __forceinline__ uint32_t a8_top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
__device__ __forceinline__ float a8_max3(float a, float b, float c) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float a8_rsqrt(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint64_t a8_add_flush(uint64_t a, uint64_t b) {  // terms below the normal range (2^-150) count as zero
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Roots of two values >= 0: v * y with y = 1/sqrt(v) to 2^-22, and one Newton step on the residual, r - (r^2 - v) y / 2, whose
// fused residual is exact.  That is off by 2^-44 before the last rounding, so the result is the rounded root but for one
// value in a million next to a midpoint: a root off by more would draw other codes now and then.
__device__ __forceinline__ uint64_t a8_root2(uint64_t v) {
  float v0, v1;
  f2_unpack(f2_add(v, f2_pack(1.17549435e-38f, 1.17549435e-38f)), v0, v1);  // keeps 0 * y finite, changes y by nothing above 2^-102
  const uint64_t y = f2_pack(a8_rsqrt(v0), a8_rsqrt(v1));
  const uint64_t r = f2_mul(v, y);
  const uint64_t residual = f2_fma(r, r, f2_mul(v, f2_pack(-1.f, -1.f)));
  return f2_fma(residual, f2_mul(y, f2_pack(-0.5f, -0.5f)), r);
}
__device__ __forceinline__ float a8_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The same exponent for the root of a largest v with these bits: with v = f * 4^e, f in [1, 4), the root is at most
// 1.75 * 2^e exactly where f <= 3.0625 (the next fp32 above 3.0625 has a root that rounds above 1.75).  What is below the
// normal range of fp32 counts as zero.
__device__ __forceinline__ int a8_root_scale_exp(uint32_t top_bits) {
  return top_bits < 0x00800000u ? -110 : (static_cast<int>(top_bits - 0x3F800000u + 0x3BFFFFu) >> 24) - 8;
}

// Gradients and roots are worked on times 2^12, v times 2^24 (exactly: powers of two): second moments down to fp32's smallest
// then lie where the Newton step below has an exact residual (above 2^-103); gradients reach to 2^52.
constexpr float A8_UP = 4096.f;

struct Adam8Consts {
  float gmul_up, beta1, omb1_down, beta2, omb2, eps_up, decay, step_size_up, minus_zero;
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
  uint64_t m[4], r[4], rr[4];
  float mmax = 0.f, vmax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int sh = (j & 1) * 16;
    const float2 mv = e4m3x2_to_float2(mc[j >> 1] >> sh), rv = e4m3x2_to_float2(rc[j >> 1] >> sh);
    const uint64_t g = f2_mul(grad[j], a8_two(c.gmul_up));
    m[j] = f2_mul(f2_pack(mv.x, mv.y), a8_two(ms));
    r[j] = f2_mul(f2_pack(rv.x, rv.y), a8_two(rs * A8_UP));
    m[j] = f2_add(a8_mul_rounded(m[j], a8_two(c.beta1), c.minus_zero), a8_mul_rounded(g, a8_two(c.omb1_down), c.minus_zero));
    const uint64_t v = a8_add_flush(a8_mul_rounded(f2_mul(r[j], r[j]), a8_two(c.beta2), c.minus_zero),
                              a8_mul_rounded(f2_mul(g, g), a8_two(c.omb2), c.minus_zero));
    mmax = a8_max3(mmax, fabsf(a8_lo(m[j])), fabsf(a8_hi(m[j])));
    vmax = a8_max3(vmax, a8_lo(v), a8_hi(v));
    r[j] = a8_root2(v);
    const uint64_t d = f2_add(r[j], a8_two(c.eps_up));
    const uint64_t q = f2_mul(m[j], f2_pack(a8_rcp(a8_lo(d)), a8_rcp(a8_hi(d))));
    p[j] = f2_fma(p[j], a8_two(-c.decay), p[j]);
    p[j] = f2_fma(q, a8_two(-c.step_size_up), p[j]);
  }
  uint32_t mtop = __reduce_max_sync(0xffffffffu, __float_as_uint(mmax));
  uint32_t vtop = __reduce_max_sync(0xffffffffu, __float_as_uint(vmax));
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
  }
  const int mk = a8_scale_exp(mtop), rk = max((finite ? a8_root_scale_exp(vtop) : a8_scale_exp(vtop)) - 12, -110);
  ms = __uint_as_float(static_cast<uint32_t>(127 + mk) << 23);
  rs = __uint_as_float(static_cast<uint32_t>(127 + rk) << 23);
  // Down to where the codes stand: one product with 2^(-k - 120); a scale above 2^6 (2^-6), whose factor fp32 does not have, takes
  // two (the first is exact, so either way there is one rounding).
  if (mk <= 6 && rk <= -6) {
    const uint64_t fm = a8_two(__uint_as_float(static_cast<uint32_t>(7 - mk) << 23)), fr = a8_two(__uint_as_float(static_cast<uint32_t>(7 - 12 - rk) << 23));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = f2_mul(m[j], fm);
      rr[j] = f2_mul(r[j], fr);
    }
  } else {
    const uint64_t fm = a8_two(__uint_as_float(static_cast<uint32_t>(127 - mk) << 23)), fr = a8_two(__uint_as_float(static_cast<uint32_t>(127 - 12 - rk) << 23));
    const uint64_t down = a8_two(__uint_as_float(7u << 23));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = f2_mul(f2_mul(m[j], fm), down);
      rr[j] = f2_mul(f2_mul(r[j], fr), down);
    }
  }
  // hash32((e0 + k) ^ mix) for k = 0 .. 7: e0 is a multiple of eight, so the first step's shift does not depend on k
  const uint32_t seed = e0 ^ mix, start = seed ^ (seed >> 16);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t cm[4], cr[4], sg[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t x = (start ^ static_cast<uint32_t>(4 * h + 2 * j + u)) * 0x7feb352dU;
        x = (x ^ (x >> 15)) * 0x846ca68bU;
        // the last step, x ^ (x >> 16), and its halves times 256: the upper half is left as it is
        const uint32_t high = __byte_perm(x, 0u, 0x4324), low = __byte_perm(x, 0u, 0x4104) ^ high;
        sg[2 * j + u] = __float_as_uint(u ? a8_hi(m[2 * h + j]) : a8_lo(m[2 * h + j]));
        cm[2 * j + u] = a8_code_top(sg[2 * j + u], low);
        cr[2 * j + u] = a8_code_top(__float_as_uint(u ? a8_hi(rr[2 * h + j]) : a8_lo(rr[2 * h + j])), high);
      }
    }
    mc[h] = a8_top_bytes(cm[0], cm[1], cm[2], cm[3]) | (a8_top_bytes(sg[0], sg[1], sg[2], sg[3]) & 0x80808080u);
    rc[h] = a8_top_bytes(cr[0], cr[1], cr[2], cr[3]);
    if (((rc[h] + 0x7F7F7F7Fu) & 0x80808080u) != 0x80808080u) {  // a code of zero: a root above zero is not stored as zero
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float root = (k & 1) ? a8_hi(r[2 * h + (k >> 1)]) : a8_lo(r[2 * h + (k >> 1)]);
        if (((rc[h] >> (8 * k)) & 0xFFu) == 0u && root > 0.f) rc[h] |= 1u << (8 * k);
      }
    }
  }
  if (!finite) {  // stored as NaN
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint64_t mp = m[k >> 1], rp = r[k >> 1];
      const uint32_t a = __float_as_uint((k & 1) ? a8_hi(mp) : a8_lo(mp)), x = __float_as_uint((k & 1) ? a8_hi(rp) : a8_lo(rp));
      const int sh = (k & 3) * 8;
      if ((a & 0x7FFFFFFFu) >= 0x7F800000u) mc[k >> 2] = (mc[k >> 2] & ~(0xFFu << sh)) | ((0x7Fu | ((a >> 24) & 0x80u)) << sh);
      if ((x & 0x7FFFFFFFu) >= 0x7F800000u) rc[k >> 2] = (rc[k >> 2] & ~(0xFFu << sh)) | (0x7Fu << sh);
    }
  }
}

// Asynchronous copies of a lane's own bytes into its slot of shared memory.
template <int BYTES>
__device__ __forceinline__ void a8_copy(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void a8_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void a8_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Eight values of a lane in shared memory (two halves of 16 bytes, 512 bytes apart, for fp32) as four pairs of fp32.
template <int DT>
__device__ __forceinline__ void a8_unpack8(const uint4* q, uint64_t (&f)[4]) {
  const uint4 a = q[0];
  if constexpr (DT == 2) {
    const uint4 b = q[32];
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

// A warp's slot for one block of 256 on its way in.
template <int PDT, int GDT>
struct A8Slot {
  uint4 p[PDT == 2 ? 64 : 32];
  uint4 g[GDT == 2 ? 64 : 32];
  uint2 m[32], r[32];
  float ms, rs, pad[2];
};
// Ring stages of a warp: three where a slot is larger, so that three CTAs fit on an SM.
template <int PDT, int GDT>
__host__ __device__ constexpr int a8_stages() { return PDT == 2 || GDT == 2 ? 3 : 4; }
template <int PDT, int GDT>
constexpr int a8_smem() { return 8 * a8_stages<PDT, GDT>() * static_cast<int>(sizeof(A8Slot<PDT, GDT>)); }

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
__global__ void __launch_bounds__(256, 3) adamw8_kernel(const __grid_constant__ Adam8Args<COUNT> a) {
  extern __shared__ uint4 a8_shared[];
  if (a.ctrl && a.ctrl[1] != 0.f) return;  // overflow: parameters and moments stay as they are
  const Adam8Consts c{(a.ctrl ? a.ctrl[0] : 1.f) * A8_UP, a.beta1, a.omb1 * (1.f / A8_UP), a.beta2, a.omb2, a.eps * A8_UP, a.decay, a.step_size * A8_UP,
                      a.minus_zero};
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
    // Whole blocks: the copies of the next blocks are under way while one is computed (loads into registers one block
    // ahead left the warps waiting for memory).  Every lane copies and reads its own bytes; only the scales are shared.
    const long long whole = min(b1, t.n / A8_BLOCK);
    const int iters = b < whole ? static_cast<int>((whole - b + 7) >> 3) : 0;
    constexpr int STAGES = a8_stages<PDT, GDT>(), PB = PDT == 2 ? 4 : 2, GB = GDT == 2 ? 4 : 2, STEP = 8 * A8_BLOCK;  // elements from one of the warp's blocks to the next
    A8Slot<PDT, GDT>* slots = reinterpret_cast<A8Slot<PDT, GDT>*>(a8_shared) + warp * STAGES;
    const long long i0 = b * A8_BLOCK + lane * 8;
    char* p_at = static_cast<char*>(t.p) + i0 * PB;
    const char* g_at = static_cast<const char*>(t.g) + i0 * GB;
    uint8_t *m_at = t.m + i0, *r_at = t.r + i0;
    float *ms_at = t.ms + b, *rs_at = t.rs + b;
    auto fetch = [&](int ahead, int stage) {  // the block `ahead` steps behind the current one
      A8Slot<PDT, GDT>& s = slots[stage];
      const char *p = p_at + ahead * (STEP * PB), *g = g_at + ahead * (STEP * GB);
      a8_copy<16>(&s.p[lane], p);
      if constexpr (PDT == 2) a8_copy<16>(&s.p[lane + 32], p + 16);
      a8_copy<16>(&s.g[lane], g);
      if constexpr (GDT == 2) a8_copy<16>(&s.g[lane + 32], g + 16);
      a8_copy<8>(&s.m[lane], m_at + ahead * STEP);
      a8_copy<8>(&s.r[lane], r_at + ahead * STEP);
      if (lane < 2) a8_copy<4>(lane ? &s.rs : &s.ms, (lane ? rs_at : ms_at) + ahead * 8);
    };
#pragma unroll
    for (int k = 0; k < STAGES; ++k) {
      if (k < iters) fetch(k, k);
      a8_copy_commit();
    }
    unsigned long long e = number(b);
    uint32_t e_hi = static_cast<uint32_t>(e >> 32), mix = mix_of(e);
    int stage = 0;
    for (int it = 0; it < iters; ++it) {
      a8_copy_wait<STAGES - 1>();
      __syncwarp();
      const A8Slot<PDT, GDT>& s = slots[stage];
      uint64_t p[4], g[4];
      a8_unpack8<PDT>(&s.p[lane], p);
      a8_unpack8<GDT>(&s.g[lane], g);
      uint32_t mc[2] = {s.m[lane].x, s.m[lane].y}, rc[2] = {s.r[lane].x, s.r[lane].y};
      float ms = s.ms, rs = s.rs;
      __syncwarp();  // all lanes have read the scales
      if (it + STAGES < iters) fetch(STAGES, stage);
      a8_copy_commit();
      if (static_cast<uint32_t>(e >> 32) != e_hi) {
        e_hi = static_cast<uint32_t>(e >> 32);
        mix = mix_of(e);
      }
      a8_update8(p, g, mc, rc, ms, rs, c, static_cast<uint32_t>(e), mix);
      a8_store8<PDT>(p_at, 0, p);
      *reinterpret_cast<uint2*>(m_at) = make_uint2(mc[0], mc[1]);
      *reinterpret_cast<uint2*>(r_at) = make_uint2(rc[0], rc[1]);
      if (lane == 0) {
        *ms_at = ms;
        *rs_at = rs;
      }
      p_at += STEP * PB; g_at += STEP * GB; m_at += STEP; r_at += STEP; ms_at += 8; rs_at += 8;
      e += STEP;
      stage = stage + 1 < STAGES ? stage + 1 : 0;
    }
    b += 8LL * iters;
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
static int launch_adamw8(const unsigned long long* ptrs, const long long* sizes, int count, long long block0, int tile_blocks, const Adam8Hyper& h, cudaStream_t stream) {
  Adam8Args<COUNT> a;
  a.count = count;
  a.tile_blocks = tile_blocks;
  a.block0 = block0;
  long long tiles = 0, blocks = 0;
  for (int i = 0; i < count; ++i) {
    const unsigned long long* q = ptrs + 6 * i;
    Adam8Tensor& t = a.t[i];
    t.p = reinterpret_cast<void*>(q[0]);
    t.g = reinterpret_cast<const void*>(q[1]);
    t.m = reinterpret_cast<uint8_t*>(q[2]);
    t.ms = reinterpret_cast<float*>(q[3]);
    t.r = reinterpret_cast<uint8_t*>(q[4]);
    t.rs = reinterpret_cast<float*>(q[5]);
    t.n = sizes[i];
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
  auto kern = adamw8_kernel<PDT, GDT, COUNT>;
  constexpr int smem = a8_smem<PDT, GDT>();
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -10;
  kern<<<static_cast<unsigned>(tiles), 256, smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? 1 : -11;
}

}  // namespace msq

// Host memory: `ptrs` holds six addresses per tensor, {p, g, codes of m, scales of m, codes of r, scales of r}, `sizes` its
// elements.  Scales: one fp32 per block of 256 elements.  Tensors with no elements are allowed.  Returns the number of kernels
// launched, or a negative code.
extern "C" int msq_adamw8_multi(const unsigned long long* ptrs, const long long* sizes, int count, int p_dtype, int g_dtype, float beta1, float omb1,
                                float beta2, float omb2, float eps, float decay, float step_size, unsigned long long seed,
                                const float* ctrl, cudaStream_t stream) {
  using namespace msq;
  constexpr int FEW = 16, MANY = 256;
  const int sms = device_sms();
  if (sms <= 0) return -10;
  const Adam8Hyper h{beta1, omb1, beta2, omb2, eps, decay, step_size, seed, ctrl};
  long long block0 = 0;
  int launched = 0;
  for (int at = 0; at < count;) {
    const int n = count - at < MANY ? count - at : MANY;
    long long blocks = 0;
    for (int i = 0; i < n; ++i) blocks += (sizes[at + i] + A8_BLOCK - 1) / A8_BLOCK;
    // A CTA's tile: long ones save the start-up of the copies (403M elements: 32 blocks 866 us, 128 blocks 831 us), but six
    // tiles an SM keep the last wave short (6.3M fp32 elements: 8 blocks 26.4 us, 24 blocks 20.8 us, 56 blocks 22.6 us).
    const long long tile = blocks / (6 * sms) / 8 * 8;
    const int tile_blocks = static_cast<int>(tile < 8 ? 8 : tile > 128 ? 128 : tile);
    int rc = -2;
#define MSQ_A8(PD, GD)                                                                                      \
  rc = n <= FEW ? launch_adamw8<PD, GD, FEW>(ptrs + 6 * at, sizes + at, n, block0, tile_blocks, h, stream)            \
                : launch_adamw8<PD, GD, MANY>(ptrs + 6 * at, sizes + at, n, block0, tile_blocks, h, stream)
    if (p_dtype == 0 && g_dtype == 0) MSQ_A8(0, 0);
    else if (p_dtype == 1 && g_dtype == 1) MSQ_A8(1, 1);
    else if (p_dtype == 2 && g_dtype == 0) MSQ_A8(2, 0);
    else if (p_dtype == 2 && g_dtype == 1) MSQ_A8(2, 1);
    else if (p_dtype == 2 && g_dtype == 2) MSQ_A8(2, 2);
    else if (p_dtype == 0 && g_dtype == 2) MSQ_A8(0, 2);
    else if (p_dtype == 1 && g_dtype == 2) MSQ_A8(1, 2);
#undef MSQ_A8
    if (rc < 0) return rc;
    launched += rc;
    block0 += blocks;
    at += n;
  }
  return launched;
}
