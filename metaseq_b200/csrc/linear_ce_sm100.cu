// Softmax cross entropy of a linear projection, in pieces of the vocabulary, without keeping the logits:
//   z = x w^T [tokens, V];  lse_n = log sum_v exp(z_nv);  loss_n = lse_n - z_{n, target_n}   (0 where ignored)
//   P_nv = exp(z_nv - lse_n) - [v = target_n];  dx = g P w;  dw = g P^T x                    (g: upstream factor)
//
// The logits exist only as accumulators in tensor memory.  Forward: one product whose epilogue leaves, per 128 columns
// and row, the maximum and the sum of exponentials, and the target's logit.  Backward, per piece of the vocabulary: the
// same product again, whose epilogue turns the accumulators into P (16 bits, the only [tokens, piece] buffer there
// is), then dx += P w_piece (fp32 sums over the pieces) and dw_piece = P^T x.  8 N V D operations where 6 N V D would do
// with the logits kept.
//
// Rows whose target is ignored are left out of every product: a first kernel copies the others to the front of a
// compact matrix, in order, and leaves their number in device memory, where the products read it.  What stands in ignored
// rows (infinities, NaN) therefore reaches nothing.
//
// All products are one kernel, the CTA-pair (cta_group::2) tcgen05 loop of gemm2_sm100.cu with eight epilogue warps:
// 256 x 256 pair tiles, six TMA stages, two accumulators in tensor memory so that the epilogue of a tile runs under the
// product of the next.
//
// What bounds it is the tensor pipe: active 88 to 93 % of the cycles in all four products (8192 x 9472 x 2048 bf16, 1.5 to
// 1.6 PFLOP/s), with the clock lowered by the power limit in long runs.  16384 rows, 50272 columns, width 2048, fp16, loss
// and both gradients: 10.7 to 11.4 ms with 3.7 % of the rows ignored (13.0 TFLOP with the logits computed twice), 11.1 to
// 11.7 ms with all rows kept (13.5 TFLOP); scratch 0.4 GB where the logits alone would take 1.6.  Smaller 16-bit output tiles
// from two staging buffers a warp (64-byte rows) changed nothing.  Few tiles (short pieces, few kept rows) are cut along K
// into fp32 slabs that are added in order (lce_splits): no atomics, equal inputs give equal bits.
#include <atomic>

#include "sm100_pair.cuh"

namespace msq {

int make_tmap_2d(CUtensorMap* out, const void* base, long long rows, long long cols, long long ld, int box_rows,
                 int bf16);  // gemm_sm100.cu

enum : int { LCE_STATS = 0, LCE_PROB = 1, LCE_F32 = 2, LCE_OUT16 = 3 };

constexpr int LC_BM = 128;  // rows per CTA (256 per pair)
constexpr int LC_BN = 256;  // columns per pair; each CTA stages half of the B tile
constexpr int LC_BK = 64;
constexpr int LC_STAGES = 6;
constexpr int LC_EPI_WARPS = 8;
constexpr int LC_THREADS = 64 + 32 * LC_EPI_WARPS;
constexpr uint32_t LC_A_BYTES = LC_BM * LC_BK * 2;
constexpr uint32_t LC_B_BYTES = (LC_BN / 2) * LC_BK * 2;
constexpr uint32_t LC_EPI_BYTES = LC_EPI_WARPS * 4096;  // per warp: 32 rows x 128 bytes on their way out
constexpr uint32_t LC_SMEM = LC_STAGES * (LC_A_BYTES + LC_B_BYTES) + LC_EPI_BYTES + 1024 + 256;
constexpr uint32_t LC_TMEM_COLS = 2 * LC_BN;
constexpr float LC_LOG2E = 1.4426950408889634f;

struct LceParams {
  int M, N, K;
  const int* count;  // kept rows (device memory)
  int count_is;      // 1: the count bounds M, 2: it bounds K
  int pairs;         // CTA pairs of a full grid (LCE_F32: lce_splits)
  int split_k;       // K blocks that the number of parts is chosen for
  int slab_rows;     // rows of the fp32 output; a part has a slab of M rows rounded up to 256
  int accumulate;
  int bf16;
  int* status;
  // LCE_STATS / LCE_PROB
  const int* target;  // [M] column of the target in the whole vocabulary, negative: none
  int v0;             // first vocabulary column of this product
  float* st_max;      // [2 * tiles_n][M]
  float* st_sum;
  float* st_tgt;      // [M] logit of the target
  const float* lse2;  // [M rounded up to the tile] log-sum-exp in units of log 2
  float p_log2;       // log2 of the factor that P is stored with
  // LCE_OUT16
  uint16_t* out;
  long long ldo;
  const float* g;  // upstream factor (device), or null
  float alpha;     // undoes P's factor
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* tmap, const void* smem_src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void tma_reduce_add_2d(const CUtensorMap* tmap, const void* smem_src, int c0, int c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
               : "memory");
}

__device__ __forceinline__ void lce_tile_coords(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int GROUP = 8;  // 8 x 256 rows share the same sweep over column tiles
  const int per_group = GROUP * tiles_n;
  const int g = tile / per_group;
  const int first_m = g * GROUP;
  const int gsize = min(GROUP, tiles_m - first_m);
  const int r = tile - g * per_group;
  tm = first_m + (r % gsize);
  tn = r / gsize;
}

// Parts into which K is cut so that few tiles fill the machine: the number that makes the waves shortest, in units of a
// fifth of one k block of a tile (0.4 us); thirty for the start and end of a wave, one per tile for a further slab's way to
// memory and back.  The kernels find the same number from the rows that are really there.
__host__ __device__ inline int lce_splits(int tiles, int k_blocks, int most, int pairs) {
  int best = 1;
  long long best_cost = 0;
  if (most > 32) most = 32;
  for (int s = 1; s <= most && (s == 1 || s * 4 <= k_blocks); ++s) {
    const long long waves = (tiles * s + pairs - 1) / pairs;
    const long long cost = 5 * waves * ((k_blocks + s - 1) / s + 6) + static_cast<long long>(tiles) * (s - 1);
    if (s == 1 || cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

template <bool A_MN, bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LC_THREADS, 1)
lce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const LceParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + LC_STAGES * LC_A_BYTES;
  uint8_t* sEpi = sB + LC_STAGES * LC_B_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sEpi + LC_EPI_BYTES);
  uint64_t* empty_bar = full_bar + LC_STAGES;
  uint64_t* tfull_bar = empty_bar + LC_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* skip_flag = reinterpret_cast<volatile uint32_t*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0 = leader
  const int pair = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;

  // Everything up to dependents_wait may run while the predecessor drains.
  if (threadIdx.x == 0) {
    for (int s = 0; s < LC_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 2 * LC_EPI_WARPS);
    }
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, LC_TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the barriers of both CTAs are initialised
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  dependents_launch();
  dependents_wait();
  if (threadIdx.x == 0 && rank == 0) {
    // One decision for the pair: skip all work when an earlier launch left a timeout code behind.
    const uint32_t skip = (p.status && *reinterpret_cast<volatile int*>(p.status) != 0) ? 1u : 0u;
    *skip_flag = skip;
    st_shared_cluster_u32(map_to_cta(smem_u32(const_cast<uint32_t*>(skip_flag)), 1), skip);
  }
  __syncthreads();
  cluster_sync_all();

  const bool skip_all = *skip_flag != 0;
  const int count = skip_all ? 0 : *p.count;
  const int M = p.count_is == 1 ? count : p.M;
  const int K = p.count_is == 2 ? count : p.K;
  const int tiles_m = skip_all ? 0 : (M + 2 * LC_BM - 1) / (2 * LC_BM);
  const int tiles_n = (p.N + LC_BN - 1) / LC_BN;
  const int tiles = tiles_m * tiles_n;
  const int m_cap = tiles_m * 2 * LC_BM;
  const int splits = EPI == LCE_F32 && tiles > 0 ? lce_splits(tiles, p.count_is == 2 ? (K + LC_BK - 1) / LC_BK : p.split_k, p.slab_rows / m_cap, p.pairs) : 1;
  const int num_items = tiles * splits;
  const int k_total = (K + LC_BK - 1) / LC_BK;
  const int k_per = (k_total + splits - 1) / splits;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer (both CTAs)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int item = pair; item < num_items && ok; item += num_pairs) {
        const int split = item / tiles;
        int tm, tn;
        lce_tile_coords(item - split * tiles, tiles_m, tiles_n, tm, tn);
        const int m0 = tm * 2 * LC_BM + static_cast<int>(rank) * LC_BM;
        const int n0 = tn * LC_BN + static_cast<int>(rank) * (LC_BN / 2);
        const int kb1 = min((split + 1) * k_per, k_total);
        for (int kb = split * k_per; kb < kb1; ++kb) {
          ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, ST_TIMEOUT_SMEM_EMPTY);
          if (!ok) break;
          if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * (LC_A_BYTES + LC_B_BYTES));
          uint8_t* a_dst = sA + stage * LC_A_BYTES;
          uint8_t* b_dst = sB + stage * LC_B_BYTES;
          const int k0 = kb * LC_BK;
          if constexpr (!A_MN) {
            tma_load_2d_pair(a_dst, &tmA, &full_bar[stage], k0, m0);
          } else {
#pragma unroll
            for (int c = 0; c < LC_BM / 64; ++c)
              tma_load_2d_pair(a_dst + c * (LC_BK * 128), &tmA, &full_bar[stage], m0 + c * 64, k0);
          }
          if constexpr (!B_MN) {
            tma_load_2d_pair(b_dst, &tmB, &full_bar[stage], k0, n0);
          } else {
#pragma unroll
            for (int c = 0; c < (LC_BN / 2) / 64; ++c)
              tma_load_2d_pair(b_dst + c * (LC_BK * 128), &tmB, &full_bar[stage], n0 + c * 64, k0);
          }
          if (++stage == LC_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {  // copies in flight land before the block's shared memory is given up
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) { }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = make_idesc_f16(p.bf16, A_MN ? 1 : 0, B_MN ? 1 : 0, 2 * LC_BM, LC_BN);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int it = 0;
      for (int item = pair; item < num_items && ok; item += num_pairs, ++it) {
        const int buf = it & 1;
        const uint32_t acc = tmem_base + buf * LC_BN;
        ok = mbar_wait(&tempty_bar[buf], ((it >> 1) & 1) ^ 1, abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const int split = item / tiles;
        const int kb0 = split * k_per, kb1 = min(kb0 + k_per, k_total);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, abort_flag, p.status, ST_TIMEOUT_SMEM_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + stage * LC_A_BYTES);
          const uint32_t b_addr = smem_u32(sB + stage * LC_B_BYTES);
#pragma unroll
          for (int kk = 0; kk < LC_BK / 16; ++kk) {
            uint64_t da, db;
            if constexpr (!A_MN) da = make_smem_desc_sw128(a_addr + kk * 32, 16, 1024);
            else da = make_smem_desc_sw128(a_addr + kk * 2048, LC_BK * 128, 1024);
            if constexpr (!B_MN) db = make_smem_desc_sw128(b_addr + kk * 32, 16, 1024);
            else db = make_smem_desc_sw128(b_addr + kk * 2048, LC_BK * 128, 1024);
            tc_mma_f16_pair(acc, da, db, idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
          }
          tc_commit_pair(&empty_bar[stage]);  // frees this stage in both CTAs
          if (++stage == LC_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit_pair(&tfull_bar[buf]);  // accumulator ready in both CTAs
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (both CTAs)
    // Eight warps: a warp may read the quarter of the lanes (rows) that its number names; two warps share a quarter
    // and take 128 columns each.
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    const uint32_t leader_tempty0 = map_to_cta(smem_u32(&tempty_bar[0]), 0);
    const uint32_t leader_tempty1 = map_to_cta(smem_u32(&tempty_bar[1]), 0);
    uint8_t* stage = sEpi + (warp - 2) * 4096;
    uint8_t* my_row = stage + lane * 128;
    const int swz = lane & 7;
    float alpha = p.alpha;
    if constexpr (EPI == LCE_OUT16) {
      if (p.g) alpha *= *p.g;
    }
    bool ok = true;
    int it = 0;
    for (int item = pair; item < num_items && ok; item += num_pairs, ++it) {
      const int split = item / tiles;
      int tm, tn;
      lce_tile_coords(item - split * tiles, tiles_m, tiles_n, tm, tn);
      const bool empty = split * k_per >= k_total;  // no k block in this part: the accumulator was not written
      const int buf = it & 1;
      ok = mbar_wait_warp(&tfull_bar[buf], (it >> 1) & 1, abort_flag, p.status, ST_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      const int row_base = tm * 2 * LC_BM + static_cast<int>(rank) * LC_BM + quarter * 32;
      const int row = row_base + lane;
      const uint32_t taddr = tmem_base + buf * LC_BN + half * 128 + (static_cast<uint32_t>(quarter * 32) << 16);
      const int col_base = tn * LC_BN + half * 128;

      if constexpr (EPI == LCE_STATS) {
        const int tgt = row < M ? p.target[row] - col_base : -1;
        float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int left = p.N - col_base - c * 32;
          if (left <= 0) break;
          uint32_t r[32];
          tmem_ld_32x32(taddr + c * 32, r);
          tmem_ld_wait();
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= left) r[j] = 0xFF800000u;  // -inf
          }
          float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], __uint_as_float(r[j]));
          const float nm = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          const float off = nm == -INFINITY ? 0.f : -nm * LC_LOG2E;  // nothing but -inf so far: sums stay 0
          float s4[4] = {sum == 0.f ? 0.f : sum * exp2f(fmaf(mx, LC_LOG2E, off)), 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 32; ++j) s4[j & 3] += exp2f(fmaf(__uint_as_float(r[j]), LC_LOG2E, off));
          sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
          mx = nm;
          const int d = tgt - c * 32;
          if (static_cast<unsigned>(d) < 32u) {
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) z = j == d ? __uint_as_float(r[j]) : z;
            p.st_tgt[row] = z;
          }
        }
        if (row < M) {
          const long long at = static_cast<long long>(tn * 2 + half) * p.M + row;
          p.st_max[at] = mx;
          p.st_sum[at] = sum;
        }
      } else if constexpr (EPI == LCE_PROB) {
        const int tgt = row < M ? p.target[row] - p.v0 - col_base : -1;
        const float off = p.p_log2 - p.lse2[row];  // rows behind the last kept one: lse is +inf, P is 0
        const float one = exp2f(p.p_log2);
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int left = p.N - col_base - c * 64;
          if (left <= 0) break;
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
            tmem_ld_32x32(taddr + c * 64 + h * 32, r);
            tmem_ld_wait();
            const int d = tgt - c * 64 - h * 32;
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(exp2f(fmaf(__uint_as_float(r[j]), LC_LOG2E, off)));
            if (static_cast<unsigned>(d) < 32u) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j == d) r[j] = __float_as_uint(__uint_as_float(r[j]) - one);
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float a = __uint_as_float(r[v * 8 + 2 * j]), b = __uint_as_float(r[v * 8 + 2 * j + 1]);
                o[j] = p.bf16 ? pack2<true>(a, b) : pack2<false>(a, b);
              }
              *reinterpret_cast<uint4*>(my_row + (((h * 4 + v) ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row_base < p.M) {
            tma_store_2d(&tmC, stage, col_base + c * 64, row_base);  // columns behind the piece are dropped
            bulk_commit_group();
          }
        }
      } else if constexpr (EPI == LCE_F32) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int col0 = col_base + c * 32;
          if (col0 >= p.N || row_base >= M || (empty && p.accumulate)) break;
          uint32_t r[32];
          tmem_ld_32x32(taddr + c * 32, r);
          tmem_ld_wait();
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 8; ++v)
            *reinterpret_cast<uint4*>(my_row + ((v ^ swz) << 4)) =
                empty ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (p.accumulate) tma_reduce_add_2d(&tmC, stage, col0, split * m_cap + row_base);
            else tma_store_2d(&tmC, stage, col0, split * m_cap + row_base);
            bulk_commit_group();
          }
        }
      } else {  // LCE_OUT16: out = alpha * acc (+ out)
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int col0 = col_base + c * 64;
          if (col0 >= p.N || row_base >= M) break;
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
            tmem_ld_32x32(taddr + c * 64 + h * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float f[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] = empty ? 0.f : __uint_as_float(r[v * 8 + j]) * alpha;
              const int col = col0 + h * 32 + v * 8;
              if (p.accumulate && row < M && col < p.N) {
                const uint4 old = *reinterpret_cast<const uint4*>(p.out + static_cast<long long>(row) * p.ldo + col);
                const uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float2 t = p.bf16 ? unpack2<true>(w[j]) : unpack2<false>(w[j]);
                  f[2 * j] += t.x;
                  f[2 * j + 1] += t.y;
                }
              }
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) o[j] = p.bf16 ? pack2<true>(f[2 * j], f[2 * j + 1]) : pack2<false>(f[2 * j], f[2 * j + 1]);
              *reinterpret_cast<uint4*>(my_row + (((h * 4 + v) ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmC, stage, col0, row_base);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(buf ? leader_tempty1 : leader_tempty0);
    }
    if (lane == 0) bulk_wait_all();  // the staging buffers have been read, the stores are done
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer may still signal or read this CTA until it, too, is done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, LC_TMEM_COLS);
  }
}

// Kept rows to the front of `xc`, in order: a CTA counts the kept rows before its 32 and copies its own.  The last CTA
// leaves the count and clears the rows up to the next multiple of 256 (the products read whole tiles).  The counting reads
// n^2 / 8 bytes of targets, from L2: 34 MB at 16384 rows; 137 GB at a million, about half of the 6.3 ms that their loss takes over
// 1024 columns of width 64 (131072 rows: 0.35 ms).
constexpr int LC_COMPACT_ROWS = 32;

struct LceCompact {
  const uint4* x;  // rows of `vecs` 16-byte vectors, ldx vectors apart
  long long ldx;
  uint4* xc;
  int vecs;
  const long long* target;
  long long ignore;
  int n, V;
  int* rows;    // [n] original row of a compact row
  int* tgt;     // [n] its target, -1 where it names no column
  float* st_tgt;
  int* count;
  unsigned* ticket;
  float* loss;  // [n]: set to 0 for ignored rows
};

__global__ void __launch_bounds__(256) lce_compact_kernel(const LceCompact s) {
  __shared__ int red[8];
  __shared__ int place[LC_COMPACT_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  dependents_launch();
  const int r0 = blockIdx.x * LC_COMPACT_ROWS;
  int before = 0;
#pragma unroll 16
  for (int i = tid; i < r0; i += 256) before += s.target[i] != s.ignore;
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) red[warp] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += red[w];
  int end = 0;
  {  // every warp finds the places of the 32 rows; warp 0 writes them down
    const int r = r0 + lane;
    const long long t = r < s.n ? s.target[r] : s.ignore;
    const bool keep = r < s.n && t != s.ignore;
    const unsigned mask = __ballot_sync(0xffffffffu, keep);
    const int at = before + __popc(mask & ((1u << lane) - 1u));
    end = before + __popc(mask);
    if (warp == 0) {
      place[lane] = keep ? at : -1;
      if (keep) {
        s.rows[at] = r;
        s.tgt[at] = t >= 0 && t < s.V ? static_cast<int>(t) : -1;
        s.st_tgt[at] = __uint_as_float(0x7FC00000u);  // stays NaN where the target names no column
      } else if (r < s.n) {
        s.loss[r] = 0.f;
      }
    }
  }
  __syncthreads();
  // A warp's four rows side by side: eight loads a lane in flight.
  const uint4* src[4];
  uint4* dst[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = place[warp * 4 + k];
    src[k] = at < 0 ? nullptr : s.x + static_cast<long long>(r0 + warp * 4 + k) * s.ldx;
    dst[k] = at < 0 ? nullptr : s.xc + static_cast<long long>(at) * s.vecs;
  }
  for (int v = lane; v < s.vecs; v += 64) {
    uint4 t[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (src[k]) t[k][0] = src[k][v];
      if (src[k] && v + 32 < s.vecs) t[k][1] = src[k][v + 32];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (dst[k]) dst[k][v] = t[k][0];
      if (dst[k] && v + 32 < s.vecs) dst[k][v + 32] = t[k][1];
    }
  }
  if (blockIdx.x == gridDim.x - 1) {
    if (tid == 0) {
      *s.count = end;
      *s.ticket = 0u;
    }
    const int stop = min(s.n, (end + 255) & ~255);
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    uint4* tail = s.xc + static_cast<long long>(end) * s.vecs;
    for (long long v = tid; v < static_cast<long long>(stop - end) * s.vecs; v += 256) tail[v] = z;
  }
}

// Per kept row: the pieces of the row folded into its log-sum-exp, the loss to the row's original place; the sum of
// all losses by the CTA that arrives last, over the CTAs' partial sums in order.
struct LceMerge {
  const float* st_max;
  const float* st_sum;
  const float* st_tgt;
  int parts, n;  // n: row capacity (the tables' row length)
  const int* rows;
  const int* count;
  float* lse2;  // [n rounded up to 256]
  float* loss;
  float* partial;  // [CTAs]
  unsigned* ticket;
  float* total;
};

__global__ void __launch_bounds__(1024) lce_merge_kernel(const LceMerge s) {
  __shared__ float sm[32][33], ss[32][33];
  __shared__ float red[32];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  dependents_launch();
  dependents_wait();
  const int count = *s.count;
  const int row = blockIdx.x * 32 + lane;
  auto fold = [](float& mx, float& sum, float m, float e) {  // parts without columns are (-inf, 0)
    const float nm = fmaxf(mx, m);
    sum = (sum == 0.f ? 0.f : sum * exp2f((mx - nm) * LC_LOG2E)) + (e == 0.f ? 0.f : e * exp2f((m - nm) * LC_LOG2E));
    mx = nm;
  };
  float mx = -INFINITY, sum = 0.f;
  if (row < count) {
    for (int i0 = warp; i0 < s.parts; i0 += 128) {  // four parts' loads in flight
      float m[4], e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + 32 * k;
        m[k] = i < s.parts ? s.st_max[static_cast<long long>(i) * s.n + row] : -INFINITY;
        e[k] = i < s.parts ? s.st_sum[static_cast<long long>(i) * s.n + row] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) fold(mx, sum, m[k], e[k]);
    }
  }
  sm[lane][warp] = mx;
  ss[lane][warp] = sum;
  __syncthreads();
  // warp w folds row w of the 32: a butterfly over the warps' parts
  mx = sm[warp][lane];
  sum = ss[warp][lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, mx, o), e = __shfl_xor_sync(0xffffffffu, sum, o);
    fold(mx, sum, m, e);
  }
  const int mine = blockIdx.x * 32 + warp;
  float loss = 0.f;
  if (lane == 0) {
    if (mine < count) {
      // in 64 bits: the loss of a confident token is a small difference, and the hardware's logarithm next to 1 is off by 2^-22
      const double ln = log(static_cast<double>(sum));
      s.lse2[mine] = static_cast<float>((static_cast<double>(mx) + ln) * 1.4426950408889634);
      loss = static_cast<float>(static_cast<double>(mx) - static_cast<double>(s.st_tgt[mine]) + ln);
      s.loss[s.rows[mine]] = loss;
    } else if (mine < ((s.n + 255) & ~255)) {
      s.lse2[mine] = INFINITY;
    }
    red[warp] = loss;
  }
  __syncthreads();
  if (warp == 0) {
    loss = warp_sum(red[lane]);
    if (lane == 0) {
      s.partial[blockIdx.x] = loss;
      __threadfence();
      last = atomicAdd(s.ticket, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!last) return;
  float acc = 0.f;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += 1024) acc += __ldcg(s.partial + i);
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) *s.total = acc;
}

// out[rows[r], :] = alpha * g * sum over the parts of acc[part][r, :] in order; rows[] null: out[r, :] (+ out[r, :]).
// Rows of `out` that no kept row names are cleared by the second half of the grid's y range (zero_target).
struct LceFinish {
  const float* acc;
  int pairs, split_k, slab_rows;  // as for the product that left the parts
  const int* split_count;         // its K is the count (rows null), or null
  int D, M;
  const int* rows;
  const int* count;           // bounds the rows, or null
  const long long* target;    // with rows: [M] targets by original row
  long long ignore;
  uint16_t* out;
  long long ldo;
  const float* g;
  float alpha;
  int accumulate, bf16;
};

__global__ void __launch_bounds__(256) lce_finish_kernel(const LceFinish s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  dependents_launch();
  dependents_wait();
  const int M = s.count ? *s.count : s.M;
  const float alpha = s.g ? s.alpha * *s.g : s.alpha;
  const int m_cap = (M + 2 * LC_BM - 1) / (2 * LC_BM) * (2 * LC_BM);
  const int tiles = m_cap / (2 * LC_BM) * ((s.D + LC_BN - 1) / LC_BN);
  const int parts = tiles > 0 ? lce_splits(tiles, s.split_count ? (*s.split_count + LC_BK - 1) / LC_BK : s.split_k, s.slab_rows / m_cap, s.pairs) : 1;
  const long long slab = static_cast<long long>(m_cap) * s.D;
  for (int r = blockIdx.x * 8 + warp; r < s.M; r += gridDim.x * 8) {
    if (s.rows && s.target[r] == s.ignore) {
      uint16_t* o = s.out + static_cast<long long>(r) * s.ldo;
      for (int c = lane * 8; c < s.D; c += 256) *reinterpret_cast<uint4*>(o + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (r >= M) continue;
    uint16_t* o = s.out + static_cast<long long>(s.rows ? s.rows[r] : r) * s.ldo;
    const float* a = s.acc + static_cast<long long>(r) * s.D;
    for (int c = lane * 8; c < s.D; c += 256) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
#pragma unroll 4
      for (int q = 0; q < parts; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(a + q * slab + c), y = *reinterpret_cast<const float4*>(a + q * slab + c + 4);
        f[0] += x.x; f[1] += x.y; f[2] += x.z; f[3] += x.w;
        f[4] += y.x; f[5] += y.y; f[6] += y.z; f[7] += y.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= alpha;
      if (s.accumulate) {
        const uint4 old = *reinterpret_cast<const uint4*>(o + c);
        const uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 t = s.bf16 ? unpack2<true>(w[j]) : unpack2<false>(w[j]);
          f[2 * j] += t.x;
          f[2 * j + 1] += t.y;
        }
      }
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = s.bf16 ? pack2<true>(f[2 * j], f[2 * j + 1]) : pack2<false>(f[2 * j], f[2 * j + 1]);
      *reinterpret_cast<uint4*>(o + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// Launches inside one call are chained: each may start while its predecessor drains, and waits for it before it touches
// memory.  The first kernel of a call is launched the ordinary way.
template <typename... KArgs, typename... Args>
static int lce_chain(void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, bool chained, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = chained ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? 0 : -11;
}

template <bool A_MN, bool B_MN, int EPI>
static int lce_launch(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmC, const LceParams& p, int sms,
                      cudaStream_t stream, bool chained = true) {
  auto kern = lce_gemm_kernel<A_MN, B_MN, EPI>;
  static std::atomic<unsigned long long> configured{0};  // a bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  if (!(configured.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, LC_SMEM) != cudaSuccess) return -10;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  const long long items = static_cast<long long>((p.M + 2 * LC_BM - 1) / (2 * LC_BM)) * ((p.N + LC_BN - 1) / LC_BN) * (EPI == LCE_F32 ? 32 : 1);
  long long pairs = sms / 2;
  if (pairs > items) pairs = items;
  if (pairs <= 0) return 0;
  return lce_chain(kern, static_cast<unsigned>(2 * pairs), LC_THREADS, LC_SMEM, stream, chained, tmA, tmB, tmC, p);
}

// Tensor map of an output: tiles of 32 rows x 128 bytes.
static int lce_out_map(CUtensorMap* out, const void* base, long long rows, long long cols, long long ld, bool f32, int bf16) {
  const int es = f32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || ((ld * es) & 15)) return -2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * es};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / es), 32u};
  const CUtensorMapDataType dt = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : (bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  return encode_tiled(out, base, 2, dims, strides, box, dt) == CUDA_SUCCESS ? 0 : -3;
}

static long long lce_align(long long b) { return (b + 255) & ~255LL; }

// How the backward pass is cut up.
struct LcePlan {
  int piece;           // columns of the vocabulary per piece
  long long dx_rows;   // rows of dx's fp32 slabs
  long long dw_rows;   // rows of dw's fp32 slabs; 0: one part, written directly
};

// The size of a piece is the one whose three products have the shortest waves (units as in lce_splits, ten for a launch),
// P staying within 256 MB (above 131072 rows within 2 KB a row: four tiles); ignored rows are not known here.  16384 rows, 50272
// columns, width 2048, all kept, one run after the other: pieces of 4096 columns (dw: 128 tiles for 74 pairs) 11.8 ms, of 4608
// (144 tiles) 11.6, of 6912 (216 tiles; the choice) 11.5, of 8192 11.9.
static LcePlan lce_plan(int n, int V, int D, int sms) {
  LcePlan q;
  const int pairs = sms / 2;
  const int tn_d = (D + LC_BN - 1) / LC_BN, tm_n = (n + 2 * LC_BM - 1) / (2 * LC_BM), tv = (V + 255) / 256;
  const int k_d = (D + LC_BK - 1) / LC_BK, k_n = (n + LC_BK - 1) / LC_BK;
  long long most = (256LL << 20) / (512LL * n);
  if (most > tv) most = tv;
  if (most < 4) most = tv < 4 ? tv : 4;
  auto waves = [&](long long tiles) { return (tiles + pairs - 1) / pairs; };
  auto cost = [&](long long t) -> double {  // of a piece of t tiles
    const int s = lce_splits(static_cast<int>(tm_n * tn_d), static_cast<int>(t * 4), 32, pairs);
    const int u = lce_splits(static_cast<int>(t * tn_d), k_n, 32, pairs);
    return 30.0 + waves(tm_n * t) * (k_d + 6) + waves(static_cast<long long>(tm_n) * tn_d * s) * ((t * 4 + s - 1) / s + 6) +
           waves(t * tn_d * u) * ((k_n + u - 1) / u + 6);
  };
  long long piece = most;
  double best = 1e300;
  auto consider = [&](long long t) {
    if (t < 1 || t > most) return;
    const long long whole = tv / t, rest = tv - whole * t;
    const double c = whole * cost(t) + (rest ? cost(rest) : 0.0);
    if (c < best) {
      best = c;
      piece = t;
    }
  };
  const long long fewest = (tv + most - 1) / most;
  for (long long k = fewest; k <= fewest + 6; ++k) consider((tv + k - 1) / k);      // pieces of equal size
  for (long long w = 1; w <= 8; ++w) consider(w * pairs / tn_d);                      // whole waves of dw's tiles
  q.piece = static_cast<int>(piece * 256);
  const int s = lce_splits(tm_n * tn_d, static_cast<int>(piece * 4), 32, pairs);
  const int u = lce_splits(static_cast<int>(piece) * tn_d, k_n, 32, pairs);
  q.dx_rows = static_cast<long long>(s) * tm_n * 256;
  q.dw_rows = u > 1 ? u * piece * 256 : 0;
  return q;
}

// What the forward pass leaves for the backward pass, in one block of memory.
struct LceSaved {
  uint16_t* xc;  // [n][D]
  int* rows;     // [n]
  int* tgt;      // [n]
  float* lse2;   // [n rounded up to 256]
  int* count;
  long long bytes;
};

static LceSaved lce_saved(void* base, int n, int D) {
  LceSaved s;
  char* at = static_cast<char*>(base);
  const char* const from = at;
  s.count = reinterpret_cast<int*>(at);
  at += 256;
  s.xc = reinterpret_cast<uint16_t*>(at);
  at += lce_align(2LL * n * D);
  s.rows = reinterpret_cast<int*>(at);
  at += lce_align(4LL * n);
  s.tgt = reinterpret_cast<int*>(at);
  at += lce_align(4LL * n);
  s.lse2 = reinterpret_cast<float*>(at);
  at += lce_align(4LL * ((n + 255) / 256 * 256));
  s.bytes = at - from;
  return s;
}

static bool lce_sizes_ok(int n, int V, int D) { return n >= 1 && n <= (1 << 24) && V >= 1 && V <= (1 << 24) && D >= 8 && D <= (1 << 20) && D % 8 == 0; }

}  // namespace msq

extern "C" long long msq_lce_saved_bytes(int n, int V, int D) {
  return msq::lce_sizes_ok(n, V, D) ? msq::lce_saved(nullptr, n, D).bytes : -1;
}

// Scratch of the forward pass: the row statistics.
extern "C" long long msq_lce_fwd_bytes(int n, int V, int D) {
  using namespace msq;
  if (!lce_sizes_ok(n, V, D)) return -1;
  const long long parts = 2LL * ((V + LC_BN - 1) / LC_BN);
  return 256 + lce_align(8LL * parts * n) + lce_align(4LL * n) + lce_align(4LL * ((n + 255) / 256 * 8));
}

// Scratch of the backward pass: one piece of P, the fp32 sums of dx, and those of dw where its rows are split.
extern "C" long long msq_lce_bwd_bytes(int n, int V, int D, int need_dx, int need_dw) {
  using namespace msq;
  const int sms = device_sms();
  if (!lce_sizes_ok(n, V, D) || sms < 2) return -1;
  const LcePlan q = lce_plan(n, V, D, sms);
  long long b = lce_align(2LL * n * q.piece);
  if (need_dx) b += lce_align(4LL * q.dx_rows * D);
  if (need_dw) b += lce_align(4LL * q.dw_rows * D);
  return b;
}

// loss[n] (0 for ignored rows) and total[0] = their sum; `saved` (msq_lce_saved_bytes) is what the backward pass reads.
// x [n, D] and w [V, D] are 16-bit, unit inner stride, row strides multiples of eight, 16-byte aligned.  A target that
// is neither `ignore` nor a column makes the loss of its row NaN.  Returns the number of kernels launched, or a negative code.
extern "C" int msq_lce_fwd(const void* x, long long ldx, const void* w, long long ldw, const long long* target, int n, int V,
                           int D, long long ignore, float* loss, float* total, void* saved, void* ws, int bf16, int* status,
                           cudaStream_t stream) {
  using namespace msq;
  if (!lce_sizes_ok(n, V, D) || (ldx & 7) || (ldw & 7) || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(ws)) & 15)) return -4;
  const LceSaved sv = lce_saved(saved, n, D);
  const int tiles_n = (V + LC_BN - 1) / LC_BN, parts = 2 * tiles_n;
  char* at = static_cast<char*>(ws);
  unsigned* ticket = reinterpret_cast<unsigned*>(at);
  at += 256;
  float* st_max = reinterpret_cast<float*>(at);
  float* st_sum = st_max + static_cast<long long>(parts) * n;
  at += lce_align(8LL * parts * n);
  float* st_tgt = reinterpret_cast<float*>(at);
  at += lce_align(4LL * n);
  float* partial = reinterpret_cast<float*>(at);

  LceCompact c;
  c.x = static_cast<const uint4*>(x); c.ldx = ldx / 8; c.xc = reinterpret_cast<uint4*>(sv.xc); c.vecs = D / 8;
  c.target = target; c.ignore = ignore; c.n = n; c.V = V; c.rows = sv.rows; c.tgt = sv.tgt; c.st_tgt = st_tgt;
  c.count = sv.count; c.ticket = ticket; c.loss = loss;
  // (the kernels behind it take their sizes from what it leaves)
  int rc = lce_chain(lce_compact_kernel, (n + LC_COMPACT_ROWS - 1) / LC_COMPACT_ROWS, 256, 0, stream, false, c);
  if (rc) return rc;

  CUtensorMap tmA, tmB;
  rc = make_tmap_2d(&tmA, sv.xc, n, D, D, LC_BM, bf16);
  if (rc) return rc;
  rc = make_tmap_2d(&tmB, w, V, D, ldw, LC_BN / 2, bf16);
  if (rc) return rc;
  LceParams p = {};
  p.M = n; p.N = V; p.K = D;
  p.count = sv.count; p.count_is = 1;
  p.bf16 = bf16; p.status = status;
  p.target = sv.tgt;
  p.st_max = st_max; p.st_sum = st_sum; p.st_tgt = st_tgt;
  rc = lce_launch<false, false, LCE_STATS>(tmA, tmB, tmA, p, device_sms(), stream);
  if (rc) return rc;

  LceMerge m;
  m.st_max = st_max; m.st_sum = st_sum; m.st_tgt = st_tgt; m.parts = parts; m.n = n;
  m.rows = sv.rows; m.count = sv.count; m.lse2 = sv.lse2; m.loss = loss; m.partial = partial; m.ticket = ticket; m.total = total;
  rc = lce_chain(lce_merge_kernel, (n + 255) / 256 * 8, 1024, 0, stream, true, m);
  return rc ? rc : 3;
}

// dx [n, D] (0 in ignored rows) and dw [V, D] (added to what is there when `accumulate`), both times g[0]; either may be
// null.  `saved` from msq_lce_fwd on the same x, w and target.  Returns as msq_lce_fwd does.
extern "C" int msq_lce_bwd(const void* w, long long ldw, const long long* target, int n, int V, int D, long long ignore,
                           const void* saved, const float* g, void* dx, long long lddx, void* dw, long long lddw, int accumulate,
                           void* ws, int bf16, int* status, cudaStream_t stream) {
  using namespace msq;
  if (!lce_sizes_ok(n, V, D) || (ldw & 7) || (lddx & 7) || (lddw & 7)) return -4;
  if ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & 15) return -4;
  if (!dx && !dw) return 0;
  const int sms = device_sms();
  if (sms < 2) return -10;
  const LceSaved sv = lce_saved(const_cast<void*>(saved), n, D);
  const LcePlan q = lce_plan(n, V, D, sms);
  char* at = static_cast<char*>(ws);
  uint16_t* P = reinterpret_cast<uint16_t*>(at);
  at += lce_align(2LL * n * q.piece);
  float* dx32 = reinterpret_cast<float*>(at);
  if (dx) at += lce_align(4LL * q.dx_rows * D);
  float* dw32 = reinterpret_cast<float*>(at);
  // fp16 cannot hold the probabilities of a large vocabulary as they are (2e-5 is below its normal range): P is stored
  // times 2^15 and the factor taken out of the fp32 sums.  |P| <= 1.
  const float p_log2 = bf16 ? 0.f : 15.f, alpha = bf16 ? 1.f : 1.f / 32768.f;

  CUtensorMap tmXk, tmXmn;
  int rc = make_tmap_2d(&tmXk, sv.xc, n, D, D, LC_BM, bf16);
  if (rc) return rc;
  rc = make_tmap_2d(&tmXmn, sv.xc, n, D, D, LC_BK, bf16);
  if (rc) return rc;
  int launched = 0;
  for (int v0 = 0; v0 < V; v0 += q.piece) {
    const int pv = V - v0 < q.piece ? V - v0 : q.piece;
    const uint16_t* wp = static_cast<const uint16_t*>(w) + static_cast<long long>(v0) * ldw;
    CUtensorMap tmW, tmWmn, tmP, tmPk, tmPmn, tmOut;
    LceParams p = {};
    p.count = sv.count; p.bf16 = bf16; p.status = status; p.alpha = alpha; p.pairs = sms / 2;
    // P = (softmax - onehot) of this piece
    if ((rc = make_tmap_2d(&tmW, wp, pv, D, ldw, LC_BN / 2, bf16))) return rc;
    if ((rc = lce_out_map(&tmP, P, n, pv, q.piece, false, bf16))) return rc;
    p.M = n; p.N = pv; p.K = D; p.count_is = 1;
    p.target = sv.tgt; p.v0 = v0; p.lse2 = sv.lse2; p.p_log2 = p_log2;
    if ((rc = lce_launch<false, false, LCE_PROB>(tmXk, tmW, tmP, p, sms, stream, v0 > 0))) return rc;
    ++launched;
    if (dx) {
      if ((rc = make_tmap_2d(&tmPk, P, n, pv, q.piece, LC_BM, bf16))) return rc;
      if ((rc = make_tmap_2d(&tmWmn, wp, pv, D, ldw, LC_BK, bf16))) return rc;
      if ((rc = lce_out_map(&tmOut, dx32, q.dx_rows, D, D, true, bf16))) return rc;
      p.M = n; p.N = D; p.K = pv; p.count_is = 1; p.split_k = q.piece / LC_BK; p.slab_rows = static_cast<int>(q.dx_rows); p.accumulate = v0 > 0;
      if ((rc = lce_launch<false, true, LCE_F32>(tmPk, tmWmn, tmOut, p, sms, stream))) return rc;
      ++launched;
    }
    if (dw) {
      uint16_t* dwp = static_cast<uint16_t*>(dw) + static_cast<long long>(v0) * lddw;
      if ((rc = make_tmap_2d(&tmPmn, P, n, pv, q.piece, LC_BK, bf16))) return rc;
      p.M = pv; p.N = D; p.K = n; p.count_is = 2; p.slab_rows = static_cast<int>(q.dw_rows);
      if (q.dw_rows > 0) {
        if ((rc = lce_out_map(&tmOut, dw32, q.dw_rows, D, D, true, bf16))) return rc;
        p.accumulate = 0;
        if ((rc = lce_launch<true, true, LCE_F32>(tmPmn, tmXmn, tmOut, p, sms, stream))) return rc;
        ++launched;
        LceFinish f = {};
        f.acc = dw32; f.pairs = sms / 2; f.slab_rows = p.slab_rows; f.split_count = sv.count; f.D = D; f.M = pv;
        f.out = dwp; f.ldo = lddw; f.g = g; f.alpha = alpha; f.accumulate = accumulate; f.bf16 = bf16;
        const int blocks = (pv + 7) / 8;
        if ((rc = lce_chain(lce_finish_kernel, blocks < 8 * sms ? blocks : 8 * sms, 256, 0, stream, true, f))) return rc;
        ++launched;
      } else {
        if ((rc = lce_out_map(&tmOut, dwp, pv, D, lddw, false, bf16))) return rc;
        p.accumulate = accumulate; p.out = dwp; p.ldo = lddw; p.g = g;
        if ((rc = lce_launch<true, true, LCE_OUT16>(tmPmn, tmXmn, tmOut, p, sms, stream))) return rc;
        ++launched;
      }
    }
  }
  if (dx) {
    LceFinish f = {};
    f.acc = dx32; f.pairs = sms / 2; f.split_k = q.piece / LC_BK; f.slab_rows = static_cast<int>(q.dx_rows); f.D = D; f.M = n;
    f.rows = sv.rows; f.count = sv.count; f.target = target; f.ignore = ignore;
    f.out = static_cast<uint16_t*>(dx); f.ldo = lddx; f.g = g; f.alpha = alpha; f.bf16 = bf16;
    const int blocks = (n + 7) / 8;
    if ((rc = lce_chain(lce_finish_kernel, blocks < 8 * sms ? blocks : 8 * sms, 256, 0, stream, true, f))) return rc;
    ++launched;
  }
  return launched;
}
