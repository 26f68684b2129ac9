// Embedding gradient by sorted tokens:
//   out[v, :] = (accumulate ? out[v, :] : 0) + scale * sum over rows r with tokens[r] == v of dy[r, :]
// written straight into the 16-bit (or fp32) gradient table, with fp32 sums in a fixed order: equal inputs give equal
// bits.  Tokens equal to pad_idx or outside [vocab_start, vocab_start + table rows) contribute nothing.
//
// What bounds it is memory: every kept row of dy is read once, and either the whole table is written once (new table) or
// the touched rows are read and written (accumulate).  Up to 256 tokens one kernel does everything (after a zero fill of a
// new table): every CTA sorts all tokens in shared memory and sums 256 columns.  Above that, three launches:
//   1. one cluster of eight CTAs sorts (token, row) pairs by a stable radix sort while the other CTAs, when the table is
//      new, fill its first rows with zeros;
//   2. every warp sums the runs of equal tokens in a piece of `chunk` sorted pairs over 256 columns; runs that lie inside
//      the piece are final, the first and last run of a piece that cross its border go to fp32 partial rows.  Further
//      CTAs clear the rest of a new table, leaving out the rows that a token names (found in the sorted pairs);
//   3. runs that cross borders are joined in ascending order.
// The launches are chained (programmatic dependent launch), each starts while its predecessor drains.
// The scatter-add form (embed_ce.cu) needs a zeroed fp32 table, one atomic per element and a pass that folds the table
// into the 16-bit gradient.  16384 x 2048 bf16 into a new table of 50272 rows: 70 us (0.27 GB: 42 us of copying); 8192 x 768
// fp16 added to a table: 23 us, of which the sort takes 9.6 and latencies of the two others most of the rest.
#include "sm100_pair.cuh"

namespace msq {

constexpr int EG_CLUSTER = 8;
constexpr int EG_SORT_THREADS = 1024;
constexpr int EG_SORT_WARPS = EG_SORT_THREADS / 32;
constexpr int EG_MAX_BINS = 512;
// MB of a new table that are cleared beside the sort: what the sort of up to 16384 tokens covers.  16, 40, 64 and 128 MB of a
// bf16 table of 50272 x 2048, us in a graph: 300 tokens 43.9, 42.8, 47.9, 53.6; 8192 55.5, 55.2, 60.1, 66.3; 16384 70.8, 66.7,
// 69.7, 76.3.  The longer radix sort of more tokens would cover more: 32768 109.5, 106.8, 106.2, 96.8; 131072 263, 263, 263, 258.
constexpr long long EG_FILL_FIRST = 40;

__device__ __forceinline__ int eg_ld_remote(const int* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}

struct EmbedGradSort {
  const long long* tokens;
  uint2* buf[2];  // sorted pairs {token - vocab_start or `rows` where nothing is contributed, row}; the result is in buf[passes & 1 ? 0 : 1]
  int n;
  long long vocab_start, pad_idx;
  int rows;      // table rows; the key of pairs that contribute nothing
  int bits;      // digit width of a pass (at most 9)
  int passes;
  uint4* fill;   // table to be zeroed by the other clusters, or null
  long long fill_vecs;
};

// Stable least-significant-digit radix sort of n pairs by one cluster of eight CTAs (256 warps, each owning a contiguous
// part of the input).  Per pass: every warp counts its digits (equal digits of a warp found with match.any, so that
// ranks inside a warp keep the order), the counts are scanned over warps, CTAs (distributed shared memory) and digits,
// and every warp writes its pairs to their places.
__global__ void __cluster_dims__(EG_CLUSTER, 1, 1) __launch_bounds__(EG_SORT_THREADS, 1)
embed_grad_sort_kernel(const EmbedGradSort s) {
  extern __shared__ int eg_smem[];
  int* hist = eg_smem;                              // [warps][bins]
  int* total = hist + EG_SORT_WARPS * EG_MAX_BINS;  // [bins]: this CTA's counts
  int* base = total + EG_MAX_BINS;                  // [bins]: first place of this CTA's pairs of a digit
  int* scan = base + EG_MAX_BINS;                   // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  dependents_launch();
  if (blockIdx.x >= EG_CLUSTER) {  // whole clusters: none of their CTAs meets a cluster barrier
    const long long stride = static_cast<long long>(gridDim.x - EG_CLUSTER) * EG_SORT_THREADS;
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    for (long long i = static_cast<long long>(blockIdx.x - EG_CLUSTER) * EG_SORT_THREADS + tid; i < s.fill_vecs; i += stride)
      s.fill[i] = z;
    return;
  }
  const uint32_t rank = cluster_ctarank();
  const int bins = 1 << s.bits;
  const int parts = EG_CLUSTER * EG_SORT_WARPS;
  const int per = ((s.n + parts - 1) / parts + 31) & ~31;
  const long long lo = static_cast<long long>(rank * EG_SORT_WARPS + warp) * per;
  const int first = static_cast<int>(lo < s.n ? lo : s.n);
  const int last = static_cast<int>(lo + per < s.n ? lo + per : s.n);
  int* wh = hist + warp * EG_MAX_BINS;

  auto load = [&](int pass, int i) -> uint2 {
    if (pass == 0) {
      const long long t = s.tokens[i];
      const bool in = t != s.pad_idx && t >= s.vocab_start && t < s.vocab_start + s.rows;
      return make_uint2(in ? static_cast<uint32_t>(t - s.vocab_start) : static_cast<uint32_t>(s.rows), static_cast<uint32_t>(i));
    }
    return __ldcg(s.buf[(pass - 1) & 1] + i);
  };
  // Four pairs a lane at a time: their loads are in flight together, and where a warp's part is no longer than that (up to
  // 32768 tokens) they stay in registers from the count to the placing.
  const bool stay = per <= 128;
  uint2 kv[4];

  for (int pass = 0; pass < s.passes; ++pass) {
    const int shift = pass * s.bits;
    auto fetch = [&](int i0) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + 32 * q + lane < last) kv[q] = load(pass, i0 + 32 * q + lane);
    };
    for (int b = lane; b < bins; b += 32) wh[b] = 0;
    __syncwarp();
    for (int i0 = first; i0 < last; i0 += 128) {
      fetch(i0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (i0 + 32 * q >= last) break;
        const bool on = i0 + 32 * q + lane < last;
        const uint32_t d = on ? (kv[q].x >> shift) & (bins - 1) : 0xFFFFFFFFu;
        const uint32_t peers = __match_any_sync(0xffffffffu, d);
        if (on && lane == __ffs(peers) - 1) wh[d] += __popc(peers);
        __syncwarp();
      }
    }
    __syncthreads();
    for (int b = tid; b < bins; b += EG_SORT_THREADS) {  // exclusive scan over this CTA's warps
      int run = 0;
#pragma unroll 8
      for (int w = 0; w < EG_SORT_WARPS; ++w) {
        const int t = hist[w * EG_MAX_BINS + b];
        hist[w * EG_MAX_BINS + b] = run;
        run += t;
      }
      total[b] = run;
    }
    __syncthreads();
    cluster_sync_all();
    int before = 0, all = 0;
    if (tid < bins) {
#pragma unroll
      for (uint32_t c = 0; c < EG_CLUSTER; ++c) {
        const int t = eg_ld_remote(total + tid, c);
        if (c < rank) before += t;
        all += t;
      }
    }
    int inc = all;  // inclusive scan over the digits: within warps, then over the warps' sums
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    if (tid < bins) {
      int prev = 0;
      for (int w = 0; w < warp; ++w) prev += scan[w];
      base[tid] = prev + inc - all + before;
    }
    __syncthreads();
    uint2* dst = s.buf[pass & 1];
    for (int i0 = first; i0 < last; i0 += 128) {
      if (!stay) fetch(i0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (i0 + 32 * q >= last) break;
        const bool on = i0 + 32 * q + lane < last;
        const uint32_t d = on ? (kv[q].x >> shift) & (bins - 1) : 0xFFFFFFFFu;
        const uint32_t peers = __match_any_sync(0xffffffffu, d);
        int at = 0;
        if (on) at = base[d] + wh[d] + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (on && lane == __ffs(peers) - 1) wh[d] += __popc(peers);
        __syncwarp();
        if (on) __stcg(dst + at, kv[q]);
      }
    }
    cluster_sync_all();  // (release and acquire at cluster scope) the pairs are in place, and nobody reads `total` of this pass any more
  }
}

// The same result for up to 32768 tokens with one exchange instead of two passes of them: every CTA sorts its contiguous
// part (1024 * E tokens) by itself, a bitonic sort of {token, place in the part} packed into 32 bits, and every pair finds
// its place by binary searches in the seven other parts, copied over distributed shared memory.  8192 tokens: radix sort
// 12.1 us, this 9.6 us; 16384 into a new table 79.0 and 77.0 us as a whole.
template <int E>
__global__ void __cluster_dims__(EG_CLUSTER, 1, 1) __launch_bounds__(EG_SORT_THREADS, 1)
embed_grad_merge_kernel(const EmbedGradSort s) {
  constexpr int L = EG_SORT_THREADS * E;
  extern __shared__ uint4 merge_smem[];
  uint32_t (*list)[L] = reinterpret_cast<uint32_t(*)[L]>(merge_smem);  // [2]: the part while it is sorted
  uint32_t (*all)[L] = list + 2;                                       // [cluster]: every part, sorted
  const int tid = threadIdx.x;
  dependents_launch();
  if (blockIdx.x >= EG_CLUSTER) {  // whole clusters: none of their CTAs meets a cluster barrier
    const long long stride = static_cast<long long>(gridDim.x - EG_CLUSTER) * EG_SORT_THREADS;
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    for (long long i = static_cast<long long>(blockIdx.x - EG_CLUSTER) * EG_SORT_THREADS + tid; i < s.fill_vecs; i += stride)
      s.fill[i] = z;
    return;
  }
  const uint32_t rank = cluster_ctarank();
  // element e of a thread stands at place e * 1024 + tid of the part
  uint32_t v[E];
  long long tok[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = static_cast<int>(rank) * L + e * EG_SORT_THREADS + tid;
    tok[e] = i < s.n ? s.tokens[i] : 0;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int local = e * EG_SORT_THREADS + tid;
    const long long t = tok[e];
    const bool in = t != s.pad_idx && t >= s.vocab_start && t < s.vocab_start + s.rows;
    const uint32_t key = in ? static_cast<uint32_t>(t - s.vocab_start) : static_cast<uint32_t>(s.rows);
    v[e] = static_cast<int>(rank) * L + local < s.n ? key * L + local : 0xFFFFFFFFu;  // nothing stands behind everything
  }
  int buf = 0;
  for (int k = 2; k <= L; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= EG_SORT_THREADS) {  // the partner is another element of this thread
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int o = e ^ (j / EG_SORT_THREADS);
          if (o > e) {
            const bool up = ((e * EG_SORT_THREADS + tid) & k) == 0;
            const uint32_t a = v[e], b = v[o % E];
            v[e] = up ? min(a, b) : max(a, b);
            v[o % E] = up ? max(a, b) : min(a, b);
          }
        }
      } else if (j >= 32) {  // of another warp
#pragma unroll
        for (int e = 0; e < E; ++e) list[buf][e * EG_SORT_THREADS + tid] = v[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = e * EG_SORT_THREADS + tid;
          const uint32_t b = list[buf][i ^ j];
          const bool low = ((i & j) == 0) == ((i & k) == 0);
          v[e] = low ? min(v[e], b) : max(v[e], b);
        }
        buf ^= 1;  // the next exchange goes through the other buffer: one barrier each
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = e * EG_SORT_THREADS + tid;
          const uint32_t b = __shfl_xor_sync(0xffffffffu, v[e], j);
          const bool low = ((i & j) == 0) == ((i & k) == 0);
          v[e] = low ? min(v[e], b) : max(v[e], b);
        }
      }
    }
  }
  // the last exchange through shared memory used buffer buf ^ 1; this one is free
#pragma unroll
  for (int e = 0; e < E; ++e) list[buf][e * EG_SORT_THREADS + tid] = v[e];
  cluster_sync_all();
  // The parts are copied over before they are searched (searched in place, over distributed shared memory, the 12 steps
  // took 17,000 cycles for 8192 tokens).
#pragma unroll
  for (int c = 0; c < EG_CLUSTER; ++c) {
    const uint32_t from = map_to_cta(smem_u32(&list[buf][0]), c);
    if (tid < L / 4) {
      uint4 x;
      asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(from + 16u * tid) : "memory");
      reinterpret_cast<uint4*>(&all[c][0])[tid] = x;
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t key = v[e] / L;
    int at = e * EG_SORT_THREADS + tid;
    int pos[EG_CLUSTER];
#pragma unroll
    for (int c = 0; c < EG_CLUSTER; ++c) pos[c] = 0;
    // how many of part c come first: tokens up to this one in earlier parts, below it in later ones
    for (int step = L / 2; step > 0; step >>= 1) {
#pragma unroll
      for (int c = 0; c < EG_CLUSTER; ++c) {
        const uint32_t bound = (key + (c < static_cast<int>(rank) ? 1u : 0u)) * L;
        if (all[c][pos[c] + step - 1] < bound) pos[c] += step;
      }
    }
#pragma unroll
    for (int c = 0; c < EG_CLUSTER; ++c) {
      const uint32_t bound = (key + (c < static_cast<int>(rank) ? 1u : 0u)) * L;
      if (c != static_cast<int>(rank)) at += pos[c] + (all[c][pos[c]] < bound ? 1 : 0);
    }
    if (v[e] != 0xFFFFFFFFu) s.buf[0][at] = make_uint2(key, rank * L + (v[e] & (L - 1)));
  }
  cluster_sync_all();  // no CTA's list goes away while another one reads it
}

template <int DT>  // 0 fp16, 1 bf16, 2 fp32: eight values of a row
struct Vec8 {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* base, long long elem) {
    if constexpr (DT == 2) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + elem);
      a = __ldcs(p);
      b = __ldcs(p + 1);
    } else {
      a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem));
    }
  }
  __device__ __forceinline__ void add_to(float (&f)[8]) const {
    if constexpr (DT == 2) {
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += __uint_as_float(w[j]);
    } else {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = unpack2<DT == 1>(w[j]);
        f[2 * j] += t.x;
        f[2 * j + 1] += t.y;
      }
    }
  }
};

// out[elem .. elem + 7] = o + scale * f, rounded once; o: what is added to
template <int DT>
__device__ __forceinline__ void store_sum8(void* out, long long elem, const float (&f)[8], float scale, float (&o)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = fmaf(f[j], scale, o[j]);
  if constexpr (DT == 2) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + elem);
    p[0] = make_float4(o[0], o[1], o[2], o[3]);
    p[1] = make_float4(o[4], o[5], o[6], o[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + elem) =
        make_uint4(pack2<DT == 1>(o[0], o[1]), pack2<DT == 1>(o[2], o[3]), pack2<DT == 1>(o[4], o[5]), pack2<DT == 1>(o[6], o[7]));
  }
}
template <int DT>
__device__ __forceinline__ void store_row8(void* out, long long elem, const float (&f)[8], float scale, int accumulate) {
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (accumulate) {
    Vec8<DT> old;
    old.load(out, elem);
    old.add_to(o);
  }
  store_sum8<DT>(out, elem, f, scale, o);
}

// Sums the runs of equal tokens in `count` consecutive sorted pairs; the tokens before and behind them tell which runs
// cross.  Runs inside are written; the first and the last, where they cross, are handed to head(f) and tail(f) by finish().
// Rows are requested a batch at a time, with the old rows that the batch's finished runs are added to (one after the other,
// a read of the table behind every run, 16 runs of one token each took 20 us).
template <int DT, bool ACC>
struct RunWalker {
  static constexpr int BATCH = DT == 2 && !ACC ? 8 : 4;  // 16 bits: eight rows 94 us instead of 74 (16384 x 2048); fp32: four 41 us instead of 26 (6007 x 1000)
  const void* dy;
  long long ldy;
  void* out;
  long long ldo;
  float scale;
  uint32_t none, prev;
  int col;
  bool live;
  float f[8];
  bool first;  // no run has ended yet

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
  }
  template <typename Key, typename Row, typename Head>
  __device__ __forceinline__ void walk(int count, Key key_of, Row row_of, uint32_t behind, Head head) {
    for (int e0 = 0; e0 < count; e0 += BATCH) {
      Vec8<DT> v[BATCH], old[ACC ? BATCH : 1];
      uint32_t key[BATCH + 1];
#pragma unroll
      for (int e = 0; e <= BATCH; ++e) key[e] = e0 + e < count ? key_of(e0 + e) : behind;
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const uint32_t row = row_of(e0 + e);
        if (e0 + e >= count || key[e] == none || !live) continue;
        v[e].load(dy, static_cast<long long>(row) * ldy + col);
        if constexpr (ACC) {
          if (key[e] != key[e + 1]) old[e].load(out, static_cast<long long>(key[e]) * ldo + col);
        }
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        if (e0 + e >= count) break;
        if (key[e] != none && live) v[e].add_to(f);
        if (key[e] != key[e + 1]) {
          if (key[e] != none) {
            if (first && key[e] == prev) {
              head(f);
            } else if (live) {
              float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              if constexpr (ACC) old[e].add_to(o);
              store_sum8<DT>(out, static_cast<long long>(key[e]) * ldo + col, f, scale, o);
            }
          }
          clear();
          first = false;
        }
      }
    }
  }
  // after the last pair, with its token and the one behind it
  template <typename Head, typename Tail>
  __device__ __forceinline__ void finish(uint32_t last, uint32_t behind, Head head, Tail tail) {
    if (last == none || last != behind) return;
    if (first && last == prev) head(f);
    else tail(f);
  }
};

struct EmbedGradSum {
  const uint2* pairs;
  const void* dy;
  long long ldy;
  void* out;
  long long ldo;
  float* head;  // [chunks][D]: sum of a chunk's first run when it began in an earlier chunk
  float* tail;  // [chunks][D]: sum of a chunk's last run when it begins there and goes on in the next one
  int n, rows, D, chunk, chunks, slices, accumulate;
  float scale;
  int fill_blocks;  // the first CTAs clear rows fill_from .. rows - 1 of a new table, the others sum
  int fill_from;
};

// Rows of a new table that no token names, EG_FILL_ROWS rows a warp at a time (few, so that the look-ups of some warps run
// under the stores of others): every lane looks a row up in the sorted pairs.
constexpr int EG_FILL_ROWS = 8;
constexpr int EG_FILL_CTAS = 4;  // per SM (16384 x 2048: one 85.3 us, two 83.3, four 79.0)

template <int DT>
__device__ void embed_grad_fill(const EmbedGradSum& s) {
  constexpr int PER = DT == 2 ? 4 : 8;  // elements of 16 bytes
  const int lane = threadIdx.x & 31, vecs = s.D / PER;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  const long long step = static_cast<long long>(EG_FILL_ROWS) * s.fill_blocks * 8;
  for (long long r0 = s.fill_from + static_cast<long long>(EG_FILL_ROWS) * (blockIdx.x * 8 + (threadIdx.x >> 5)); r0 < s.rows; r0 += step) {
    const long long row = r0 + (lane & (EG_FILL_ROWS - 1));
    bool clear = row < s.rows;
    if (clear) {
      int lo = 0, hi = s.n;  // first pair whose token is not below the row
      while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (s.pairs[mid].x < static_cast<uint32_t>(row)) lo = mid + 1; else hi = mid;
      }
      clear = lo == s.n || s.pairs[lo].x != static_cast<uint32_t>(row);
    }
    const unsigned mask = __ballot_sync(0xffffffffu, clear);
#pragma unroll
    for (int k = 0; k < EG_FILL_ROWS; ++k) {
      if (!((mask >> k) & 1u)) continue;
      uint4* dst = static_cast<uint4*>(s.out) + (r0 + k) * vecs;
      for (int v = lane; v < vecs; v += 32) dst[v] = z;
    }
  }
}

// One warp: `chunk` sorted pairs, 256 columns (eight per lane).
template <int DT, bool ACC>
__global__ void __launch_bounds__(256) embed_grad_sum_kernel(const EmbedGradSum s) {
  dependents_launch();
  dependents_wait();
  if (static_cast<int>(blockIdx.x) < s.fill_blocks) {
    embed_grad_fill<DT>(s);
    return;
  }
  const long long wid = static_cast<long long>(blockIdx.x - s.fill_blocks) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int c = static_cast<int>(wid / s.slices);
  if (c >= s.chunks) return;
  const uint32_t none = static_cast<uint32_t>(s.rows);
  const int p0 = c * s.chunk, p1 = min(p0 + s.chunk, s.n);
  RunWalker<DT, ACC> w;
  w.dy = s.dy; w.ldy = s.ldy; w.out = s.out; w.ldo = s.ldo; w.scale = s.scale;
  w.none = none;
  w.col = static_cast<int>(wid - static_cast<long long>(c) * s.slices) * 256 + lane * 8;
  w.live = w.col < s.D;
  w.prev = p0 > 0 ? s.pairs[p0 - 1].x : none;
  w.first = true;
  w.clear();
  auto keep = [&](float* to, const float (&f)[8]) {
    if (!w.live) return;
    float4* dst = reinterpret_cast<float4*>(to + static_cast<long long>(c) * s.D + w.col);
    dst[0] = make_float4(f[0], f[1], f[2], f[3]);
    dst[1] = make_float4(f[4], f[5], f[6], f[7]);
  };
  auto head = [&](const float (&f)[8]) { keep(s.head, f); };
  uint32_t last = none, behind = none;
  for (int q0 = p0; q0 < p1; q0 += 32) {
    const uint2 mine = q0 + lane < p1 ? s.pairs[q0 + lane] : make_uint2(none, 0u);
    const int cnt = min(32, p1 - q0);
    behind = q0 + cnt < s.n ? s.pairs[q0 + cnt].x : none;
    w.walk(cnt, [&](int i) { return __shfl_sync(0xffffffffu, mine.x, i); }, [&](int i) { return __shfl_sync(0xffffffffu, mine.y, i & 31); }, behind, head);
    last = __shfl_sync(0xffffffffu, mine.x, cnt - 1);
  }
  w.finish(last, behind, head, [&](const float (&f)[8]) { keep(s.tail, f); });
}

// Runs that begin in chunk c and cross its border: tail[c] + head[c + 1] + ... in ascending order, 256 columns per warp.  A
// CTA looks after EG_JOIN chunks (most have nothing to join); runs over more than EG_LONG chunks are summed by all its
// warps, each a contiguous part, and the parts added in order.
constexpr int EG_JOIN = 8;  // 8192 x 768: sixteen 25.4 us, eight 24.9 us, four 25.1 us
constexpr int EG_LONG = 8;  // the same: 64 chunks 28.4 us, sixteen 24.9 us, eight 23.5 us

template <int DT>
__global__ void __launch_bounds__(256) embed_grad_join_kernel(const EmbedGradSum s) {
  __shared__ float part[8][8][32];
  __shared__ int long_runs[EG_JOIN][2];
  __shared__ int long_count;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.y * 256 + lane * 8;
  const bool live = col < s.D;
  const uint32_t none = static_cast<uint32_t>(s.rows);
  if (threadIdx.x == 0) long_count = 0;
  __syncthreads();
  dependents_wait();

  auto add = [&](const float* from, int chunk, float (&f)[8]) {
    const float4* q = reinterpret_cast<const float4*>(from + static_cast<long long>(chunk) * s.D + col);
    const float4 x = q[0], y = q[1];
    f[0] += x.x; f[1] += x.y; f[2] += x.z; f[3] += x.w;
    f[4] += y.x; f[5] += y.y; f[6] += y.z; f[7] += y.w;
  };

  for (int c = blockIdx.x * EG_JOIN + warp; c < min((static_cast<int>(blockIdx.x) + 1) * EG_JOIN, s.chunks - 1); c += 8) {
    const int p0 = c * s.chunk, p1 = p0 + s.chunk;
    const uint32_t before = p0 > 0 ? s.pairs[p0 - 1].x : none, key = s.pairs[p1 - 1].x, after = s.pairs[p1].x;
    if (key == none || after != key || before == key) continue;  // nothing crosses, or it began earlier
    int heads = 0;  // chunks behind c that begin with this token
    while (true) {
      const int q = c + 1 + heads + lane;
      const unsigned same = __ballot_sync(0xffffffffu, q < s.chunks && s.pairs[min(q, s.chunks - 1) * s.chunk].x == key);
      const int run = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
      heads += run;
      if (run < 32) break;
    }
    if (heads > EG_LONG) {
      if (lane == 0) {
        const int k = atomicAdd(&long_count, 1);
        long_runs[k][0] = c;
        long_runs[k][1] = heads;
      }
      continue;
    }
    if (!live) continue;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    add(s.tail, c, f);
#pragma unroll 4
    for (int h = 1; h <= heads; ++h) add(s.head, c + h, f);
    store_row8<DT>(s.out, static_cast<long long>(key) * s.ldo + col, f, s.scale, s.accumulate);
  }
  __syncthreads();
  for (int k = 0; k < long_count; ++k) {
    const int c = long_runs[k][0], heads = long_runs[k][1];
    const int per = (heads + 7) >> 3;
    const int h0 = 1 + warp * per, h1 = min(h0 + per, heads + 1);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    if (live) {
      if (warp == 0) add(s.tail, c, f);
#pragma unroll 4
      for (int h = h0; h < h1; ++h) add(s.head, c + h, f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) part[warp][j][lane] = f[j];
    __syncthreads();
    if (warp == 0 && live) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) f[j] += part[w][j][lane];
      }
      store_row8<DT>(s.out, static_cast<long long>(s.pairs[c * s.chunk + s.chunk - 1].x) * s.ldo + col, f, s.scale, s.accumulate);
    }
    __syncthreads();
  }
}

// Few tokens: a CTA per 256 columns finds every token's place by counting (equal tokens keep their order), its 16 warps sum
// contiguous parts of the sorted list, and runs that cross from one warp to the next are joined through shared memory.
// Tokens up to which this is taken: one kernel against three launches, us in a graph.  Added, 768 columns in 16 bits: 128 tokens 6.3
// (14.3), 256 11.1 (14.5), 320 14.9 (14.7), 400 20.8 (14.9); 256 tokens of 64 columns 11.3 (14.9), of 4096 11.6 (15.0), of 768 in
// fp32 13.0 (14.8).  Wide new tables are behind, since nothing hides their clearing: 2050 rows of 4096, 192 tokens 15.0 (14.5), 256
// 18.0 (14.8).
constexpr int EG_FEW = 256;
constexpr int EG_FEW_THREADS = 512;
constexpr int EG_FEW_WARPS = EG_FEW_THREADS / 32;

struct EmbedGradFew {
  const long long* tokens;
  const void* dy;
  long long ldy;
  void* out;
  long long ldo;
  int n, rows, D, accumulate;
  long long vocab_start, pad_idx;
  float scale;
};

template <int DT, bool ACC>
__global__ void __launch_bounds__(EG_FEW_THREADS, 1) embed_grad_few_kernel(const EmbedGradFew s) {
  __shared__ float head_s[EG_FEW_WARPS][8][32], tail_s[EG_FEW_WARPS][8][32];
  __shared__ __align__(16) uint32_t keys[EG_FEW];  // padded with the largest number
  __shared__ uint32_t skey[EG_FEW], srow[EG_FEW];   // sorted
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t none = static_cast<uint32_t>(s.rows);
  dependents_wait();
  uint32_t mine = 0xFFFFFFFFu;
  if (tid < s.n) {
    const long long t = s.tokens[tid];
    const bool in = t != s.pad_idx && t >= s.vocab_start && t < s.vocab_start + s.rows;
    mine = in ? static_cast<uint32_t>(t - s.vocab_start) : none;
  }
  if (tid < EG_FEW) keys[tid] = mine;
  __syncthreads();
  if (warp * 32 < s.n) {
    int rank = 0;
    const uint4* k4 = reinterpret_cast<const uint4*>(keys);
    for (int i = 0; i < (s.n + 3) / 4; ++i) {  // below, or equal and earlier
      const uint4 k = k4[i];
      rank += (k.x < mine || (k.x == mine && 4 * i < tid)) + (k.y < mine || (k.y == mine && 4 * i + 1 < tid)) +
              (k.z < mine || (k.z == mine && 4 * i + 2 < tid)) + (k.w < mine || (k.w == mine && 4 * i + 3 < tid));
    }
    if (tid < s.n) {
      skey[rank] = mine;
      srow[rank] = static_cast<uint32_t>(tid);
    }
  }
  __syncthreads();
  const int per = (s.n + EG_FEW_WARPS - 1) / EG_FEW_WARPS;
  const int p0 = min(warp * per, s.n), p1 = min(p0 + per, s.n);
  RunWalker<DT, ACC> w;
  w.dy = s.dy; w.ldy = s.ldy; w.out = s.out; w.ldo = s.ldo; w.scale = s.scale;
  w.none = none;
  w.col = blockIdx.x * 256 + lane * 8;
  w.live = w.col < s.D;
  w.prev = p0 > 0 ? skey[p0 - 1] : none;
  w.first = true;
  w.clear();
  auto head = [&](const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) head_s[warp][j][lane] = f[j];
  };
  auto tail = [&](const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) tail_s[warp][j][lane] = f[j];
  };
  const uint32_t last = p1 > p0 ? skey[p1 - 1] : none, behind = p1 < s.n ? skey[p1] : none;
  w.walk(p1 - p0, [&](int i) { return skey[p0 + i]; }, [&](int i) { return srow[min(p0 + i, EG_FEW - 1)]; }, behind, head);
  w.finish(last, behind, head, tail);
  __syncthreads();
  // the warp in whose part a crossing run begins adds the parts that follow
  if (last != none && behind == last && !(skey[p0] == last && w.prev == last)) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = tail_s[warp][j][lane];
    for (int q = warp + 1; q < EG_FEW_WARPS && q * per < s.n && skey[q * per] == last; ++q) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += head_s[q][j][lane];
    }
    if (w.live) store_row8<DT>(s.out, static_cast<long long>(last) * s.ldo + w.col, f, s.scale, ACC);
  }
}

__global__ void __launch_bounds__(512) embed_grad_zero_kernel(uint4* out, long long vecs) {
  dependents_launch();
  const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < vecs; i += stride) out[i] = make_uint4(0u, 0u, 0u, 0u);
}

// A launch that may start while its predecessor in the stream drains (the kernel waits for it itself).
template <typename... KArgs, typename... Args>
static cudaError_t eg_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int DT>
static cudaError_t eg_launch_few(const EmbedGradFew& f, cudaStream_t stream) {
  const dim3 grid((f.D + 255) / 256);
  if (!f.accumulate) return eg_launch(embed_grad_few_kernel<DT, false>, grid, dim3(EG_FEW_THREADS), 0, stream, f);  // behind the fill
  embed_grad_few_kernel<DT, true><<<grid, EG_FEW_THREADS, 0, stream>>>(f);
  return cudaGetLastError();
}

template <int DT>
static cudaError_t eg_launch_sums(const EmbedGradSum& su, unsigned blocks, dim3 join, cudaStream_t stream) {
  const cudaError_t err = eg_launch(su.accumulate ? embed_grad_sum_kernel<DT, true> : embed_grad_sum_kernel<DT, false>, dim3(blocks), dim3(256), 0, stream, su);
  return err != cudaSuccess ? err : eg_launch(embed_grad_join_kernel<DT>, join, dim3(256), 0, stream, su);
}

// Pairs a warp: as few as keep the SMs busy with one wave of warps or so (16384 x 2048: 8 pairs 79.4 us, 16 74.1, 32 72.5).
static int eg_chunk(long long n, int D) {
  const long long slices = (D + 255) / 256;
  int chunk = 8;
  while (chunk < 256 && n * slices > chunk * 4736LL) chunk *= 2;
  return chunk;
}

}  // namespace msq

// Bytes of scratch (16-byte aligned) that msq_embed_grad_sorted needs for n tokens and D columns.
extern "C" long long msq_embed_grad_workspace(int n, int D) {
  if (n <= msq::EG_FEW) return 0;
  const long long chunk = msq::eg_chunk(n, D);
  const long long chunks = (n + chunk - 1) / chunk;
  return ((2LL * n * 8 + 255) & ~255LL) + 2LL * chunks * D * 4;
}

// See the head of this file.  Returns the number of kernels launched, or a negative code.  dtype: 0 fp16, 1 bf16, 2 fp32 (dy
// and out).  D and both row strides are multiples of eight, dy, out and workspace are 16-byte aligned; a new table
// (accumulate == 0) has contiguous rows (ldo == D).
extern "C" int msq_embed_grad_sorted(const long long* tokens, const void* dy, long long ldy, void* out, long long ldo, int n,
                                     int rows, int D, float scale, long long vocab_start, long long pad_idx, int accumulate,
                                     int dtype, void* workspace, cudaStream_t stream) {
  using namespace msq;
  if (n < 0 || n > (1 << 30) || rows <= 0 || D <= 0 || (D & 7) || (ldy & 7) || (ldo & 7) || dtype < 0 || dtype > 2) return -4;
  if ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) return -4;
  if (!accumulate && ldo != D) return -4;
  if (n == 0 && accumulate) return 0;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long vec_per_row = D / (dtype == 2 ? 4 : 8);
  if (n <= EG_FEW) {
    if (!accumulate) {
      const long long vecs = rows * vec_per_row, want = (vecs + 2047) / 2048;
      embed_grad_zero_kernel<<<static_cast<unsigned>(want < 4LL * sms ? want : 4LL * sms), 512, 0, stream>>>(static_cast<uint4*>(out), vecs);
      if (cudaGetLastError() != cudaSuccess) return -11;
      if (n == 0) return 1;
    }
    const EmbedGradFew f{tokens, dy, ldy, out, ldo, n, rows, D, accumulate, vocab_start, pad_idx, scale};
    const cudaError_t err = dtype == 0 ? eg_launch_few<0>(f, stream) : dtype == 1 ? eg_launch_few<1>(f, stream) : eg_launch_few<2>(f, stream);
    return err == cudaSuccess ? (accumulate ? 1 : 2) : -11;
  }
  EmbedGradSort so;
  so.tokens = tokens;
  so.buf[0] = static_cast<uint2*>(workspace);
  so.buf[1] = so.buf[0] + n;
  so.n = n;
  so.vocab_start = vocab_start;
  so.pad_idx = pad_idx;
  so.rows = rows;
  int bits = 1;
  while (bits < 31 && (1LL << bits) <= rows) ++bits;  // keys 0 .. rows
  so.passes = (bits + 8) / 9;
  so.bits = (bits + so.passes - 1) / so.passes;
  long long fill_first = accumulate ? 0 : (EG_FILL_FIRST << 20) / (vec_per_row * 16);
  if (fill_first > rows) fill_first = accumulate ? 0 : rows;
  so.fill = static_cast<uint4*>(out);
  so.fill_vecs = fill_first * vec_per_row;
  const size_t smem = sizeof(int) * (EG_SORT_WARPS * EG_MAX_BINS + 2 * EG_MAX_BINS + 32);
  if (cudaFuncSetAttribute(embed_grad_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) return -10;
  const long long fill_ctas = (so.fill_vecs + EG_SORT_THREADS * 4 - 1) / (EG_SORT_THREADS * 4);
  long long fill_clusters = (fill_ctas + EG_CLUSTER - 1) / EG_CLUSTER;
  if (fill_clusters > sms / EG_CLUSTER - 1) fill_clusters = sms / EG_CLUSTER - 1;
  const unsigned sort_grid = static_cast<unsigned>(EG_CLUSTER * (1 + fill_clusters));
  constexpr int PART = EG_CLUSTER * EG_SORT_THREADS;
  const int parts = n <= PART ? 1 : n <= 2 * PART ? 2 : 4;  // elements a thread of the merging sort
  const bool merge = n <= 4 * PART && (rows + 2LL) * parts * EG_SORT_THREADS <= 1LL << 32;
  if (merge) {
    auto kern = parts == 1 ? embed_grad_merge_kernel<1> : parts == 2 ? embed_grad_merge_kernel<2> : embed_grad_merge_kernel<4>;
    const int bytes = (2 + EG_CLUSTER) * parts * EG_SORT_THREADS * 4;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -10;
    kern<<<sort_grid, EG_SORT_THREADS, bytes, stream>>>(so);
  } else embed_grad_sort_kernel<<<sort_grid, EG_SORT_THREADS, smem, stream>>>(so);
  if (cudaGetLastError() != cudaSuccess) return -11;
  EmbedGradSum su;
  su.pairs = so.buf[merge ? 0 : (so.passes - 1) & 1];
  su.dy = dy; su.ldy = ldy; su.out = out; su.ldo = ldo;
  su.n = n; su.rows = rows; su.D = D;
  su.chunk = eg_chunk(n, D);
  su.chunks = (n + su.chunk - 1) / su.chunk;
  su.slices = (D + 255) / 256;
  su.head = reinterpret_cast<float*>(static_cast<char*>(workspace) + ((2LL * n * 8 + 255) & ~255LL));
  su.tail = su.head + static_cast<long long>(su.chunks) * D;
  su.accumulate = accumulate; su.scale = scale;
  const long long warps = static_cast<long long>(su.chunks) * su.slices;
  su.fill_from = static_cast<int>(fill_first);
  const long long left = accumulate ? 0 : rows - fill_first, want = (left + 8 * EG_FILL_ROWS - 1) / (8 * EG_FILL_ROWS);
  su.fill_blocks = static_cast<int>(want < EG_FILL_CTAS * sms ? want : EG_FILL_CTAS * sms);
  const unsigned blocks = static_cast<unsigned>(su.fill_blocks + (warps + 7) / 8);
  const dim3 join(static_cast<unsigned>((su.chunks + EG_JOIN - 1) / EG_JOIN), static_cast<unsigned>(su.slices));
  const cudaError_t err = dtype == 0 ? eg_launch_sums<0>(su, blocks, join, stream) : dtype == 1 ? eg_launch_sums<1>(su, blocks, join, stream)
                                                                                       : eg_launch_sums<2>(su, blocks, join, stream);
  return err == cudaSuccess ? 3 : -11;
}
