// Scaled embedding lookup and its gradient by sorted ids.
//
//   out_i    = s E[id_i]
//   dE_v     = s sum_{i : id_i = v} g_i
//
// The gradient is the hard-label form of the E-step's mu_acc.  The ids are
// sorted with their positions by a stable radix sort, so the rows of one id
// lie together in the order of i and are summed in fp32 in a fixed order,
// without atomics.  Both directions are bound by DRAM: N D elements read and
// written in the lookup; N D read and V D written in the gradient.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "fgmm_ptx.cuh"
#include "fgmm_vocab.cuh"

namespace fgmm {
namespace {

constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
// Long sorts: blocks of 256 threads x 8 ids.
constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
// Up to 131,072 ids: one cluster of up to 8 blocks, all passes in shared memory.
constexpr int kClusterSortThreads = 1024;
constexpr int kClusterSortBlocks = 8;
constexpr int64_t kClusterSortMax = (int64_t)kClusterSortThreads * 16 * kClusterSortBlocks;
// Sorted positions per block of the gradient.
constexpr int kRun = 32;

// ---------------------------------------------------------------- lookup
// out = scale * table[id].  Each row is read by `lanes` threads (a power of two),
// 16 bytes (VEC elements) each, and a thread has four rows' pieces in flight.
// Bound by DRAM: N D read (distinct rows) and N D written.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
lookup_kernel(const T* __restrict__ table, int64_t tsv, int64_t tsd,
              const int64_t* __restrict__ ids, int64_t ignore, int64_t N, int V, int D, float scale,
              int lanes, T* __restrict__ out) {
  const int rows = 256 / lanes, mine = threadIdx.x / lanes, piece0 = threadIdx.x % lanes;
  const int per_row = D / VEC;
  for (int64_t i0 = blockIdx.x * (4ll * rows) + mine; i0 < N; i0 += gridDim.x * (4ll * rows)) {
    const T* src[4];
    float fill[4];   // of a row that is not read
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + u * rows, id = i < N ? __ldg(ids + i) : ignore;
      const bool skip = id == ignore, bad = !skip && (id < 0 || id >= V);
      src[u] = skip || bad ? nullptr : table + id * tsv;
      fill[u] = bad ? __int_as_float(0x7fffffff) : 0.f;
    }
    for (int c = piece0; c < per_row; c += lanes) {
      Pack<T, VEC> x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (src[u]) x[u].load(src[u] + (int64_t)c * VEC * tsd);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t i = i0 + u * rows;
        if (i >= N) break;
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          x[u].v[k] = from_f32<T>(src[u] ? to_f32(x[u].v[k]) * scale : fill[u]);
        x[u].store(out + i * D + (int64_t)c * VEC);
      }
    }
  }
}

// ---------------------------------------------------------------- sort
// The sort key of an id: ids that contribute nothing go last, as V.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t ignore, int V) {
  return id == ignore || id < 0 || id >= V ? (uint32_t)V : (uint32_t)id;
}

// The lanes of the warp that hold the same digit (one ballot per bit: cheaper here
// than a match instruction, whose time grows with the distinct values).
__device__ __forceinline__ uint32_t same_digit(uint32_t d, int bits) {
  uint32_t same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (d >> b) & 1u;
    const uint32_t m = __ballot_sync(0xffffffffu, one);
    same &= one ? m : ~m;
  }
  return same;
}

__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster2(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}

// Exclusive prefix sum of one value per thread over 1024 threads; *all: the sum.
__device__ __forceinline__ uint32_t block_prefix1024(uint32_t v, uint32_t* warp_sum, uint32_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  if (warp == 0) {
    uint32_t w = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += t;
    }
    warp_sum[lane] = w;
  }
  __syncthreads();
  *all = warp_sum[31];
  return (warp ? warp_sum[warp - 1] : 0u) + s - v;
}

// Stable sort of up to 1024 ITEMS x (blocks of the cluster) ids, all passes in
// shared memory.  A warp owns 32 ITEMS consecutive places; digits are ranked within
// the warp, the warps' counts summed per digit in warp order, the blocks' counts in
// block order (read from each other's shared memory), and each key goes to its place
// in the block that owns it.  Bound by latency: two cluster barriers a pass.
template <int ITEMS>
__global__ void __launch_bounds__(kClusterSortThreads)
cluster_sort_kernel(const int64_t* __restrict__ ids, int64_t ignore, int V, int N, int bits,
                    int digit_bits, uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out,
                    uint32_t* __restrict__ joins) {
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) joins[0] = 0;
  extern __shared__ uint32_t sm[];
  constexpr int kMine = kClusterSortThreads * ITEMS;               // places of a block
  uint2* place = reinterpret_cast<uint2*>(sm);                     // [kMine] (key, pos)
  uint16_t* cnt16 = reinterpret_cast<uint16_t*>(sm + 2 * kMine);   // [32][256]
  __shared__ uint32_t total[kDigits];    // this block's count of each digit
  __shared__ uint32_t offset[kDigits];   // first place of this block's keys of the digit
  __shared__ uint32_t warp_sum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank_c = (int)cluster_rank(), blocks = gridDim.x;      // one cluster
  const int base = warp * 32 * ITEMS;
  uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = rank_c * kMine + base + 32 * r + lane;
    key[r] = i < N ? sort_key(ids[i], ignore, V) : 0xffffffffu;    // behind the last: stays last
    pos[r] = (uint32_t)i;
  }
  const uint32_t mask = (1u << digit_bits) - 1u;
  uint16_t* cnt = cnt16 + warp * kDigits;
  for (int shift = 0; shift < bits; shift += digit_bits) {
    for (int i = threadIdx.x; i < 32 * kDigits / 2; i += kClusterSortThreads)
      reinterpret_cast<uint32_t*>(cnt16)[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const uint32_t d = (key[r] >> shift) & mask;
      const uint32_t same = same_digit(d, digit_bits);
      const uint32_t before = cnt[d];
      __syncwarp();
      rank[r] = before + __popc(same & ((1u << lane) - 1u));
      if (lane == 31 - __clz(same)) cnt[d] = (uint16_t)(rank[r] + 1);
      __syncwarp();
    }
    __syncthreads();
    // four threads per digit, each for 8 warps: the warps' counts become offsets
    {
      const int d = threadIdx.x >> 2, part = threadIdx.x & 3;
      uint32_t c[8], mine = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) { c[w] = cnt16[(part * 8 + w) * kDigits + d]; mine += c[w]; }
      uint32_t run = mine;
      uint32_t t = __shfl_up_sync(0xffffffffu, run, 1, 4);
      if (part >= 1) run += t;
      t = __shfl_up_sync(0xffffffffu, run, 2, 4);
      if (part >= 2) run += t;
      if (part == 3) total[d] = run;
      run -= mine;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        cnt16[(part * 8 + w) * kDigits + d] = (uint16_t)run;
        run += c[w];
      }
    }
    cluster_sync_all();            // every block's totals are there
    uint32_t all_d = 0, below = 0;
    if (threadIdx.x < kDigits) {
      for (int b = 0; b < blocks; ++b) {
        const uint32_t v = ld_cluster(map_to_cta(smem_u32(&total[threadIdx.x]), b));
        all_d += v;
        if (b < rank_c) below += v;
      }
    }
    uint32_t sum;
    const uint32_t first = block_prefix1024(all_d, warp_sum, &sum);
    if (threadIdx.x < kDigits) offset[threadIdx.x] = first + below;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const uint32_t d = (key[r] >> shift) & mask;
      const uint32_t at = offset[d] + cnt[d] + rank[r];
      st_cluster2(map_to_cta(smem_u32(&place[at % kMine]), at / kMine), key[r], pos[r]);
    }
    cluster_sync_all();            // every key is in its place, every total has been read
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const uint2 x = place[base + 32 * r + lane];
      key[r] = x.x;
      pos[r] = x.y;
    }
  }
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = rank_c * kMine + base + 32 * r + lane;
    if (i < N) {
      key_out[i] = key[r];
      pos_out[i] = pos[r];
    }
  }
}

// Long sorts: one pass = count, scan, scatter.  The first pass makes its keys
// from the ids.
struct SortIn {
  const int64_t* ids;   // first pass, else null
  int64_t ignore;
  int V;
  const uint32_t* key;
  const uint32_t* pos;
  __device__ __forceinline__ uint32_t get_key(int64_t i) const {
    return ids ? sort_key(ids[i], ignore, V) : key[i];
  }
  __device__ __forceinline__ uint32_t get_pos(int64_t i) const {
    return ids ? (uint32_t)i : pos[i];
  }
};

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(SortIn in, int64_t N, int shift, uint32_t mask, uint32_t* __restrict__ hist,
                  int nblocks) {
  __shared__ uint32_t h[kDigits];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    if (i < N) atomicAdd(&h[(in.get_key(i) >> shift) & mask], 1u);
  }
  __syncthreads();
  hist[(size_t)threadIdx.x * nblocks + blockIdx.x] = h[threadIdx.x];
}

// Exclusive prefix sum of hist[0, n) by one block.
__global__ void __launch_bounds__(1024)
sort_scan_kernel(uint32_t* __restrict__ hist, int64_t n, uint32_t* __restrict__ joins) {
  if (threadIdx.x == 0) joins[0] = 0;   // (before the next kernel may start)
  __shared__ uint32_t warp_sum[32];
  uint32_t carry = 0;
  for (int64_t base = 0; base < n; base += 8192) {   // 8 consecutive values a thread
    uint32_t v[8], mine = 0, all;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t i = base + threadIdx.x * 8 + k;
      v[k] = i < n ? hist[i] : 0u;
      mine += v[k];
    }
    uint32_t run = carry + block_prefix1024(mine, warp_sum, &all);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t i = base + threadIdx.x * 8 + k;
      if (i < n) hist[i] = run;
      run += v[k];
    }
    carry += all;
  }
}

// Stable scatter: a warp owns 256 consecutive items and ranks 32 at a time.
__global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(SortIn in, int64_t N, int shift, int digit_bits,
                    const uint32_t* __restrict__ offs, int nblocks, uint32_t* __restrict__ key_out,
                    uint32_t* __restrict__ pos_out) {
  const uint32_t mask = (1u << digit_bits) - 1u;
  constexpr int kWarps = kSortThreads / 32;
  __shared__ uint32_t cnt[kWarps][kDigits];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int w = 0; w < kWarps; ++w) cnt[w][threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile + warp * (32 * kSortItems);
  uint32_t key[kSortItems], digit[kSortItems], rank[kSortItems];
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * 32 + lane;
    key[r] = i < N ? in.get_key(i) : 0xffffffffu;   // behind the last: ranked last, not stored
    digit[r] = (key[r] >> shift) & mask;
  }
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const uint32_t same = same_digit(digit[r], digit_bits);
    const uint32_t before = cnt[warp][digit[r]];
    __syncwarp();
    rank[r] = before + __popc(same & ((1u << lane) - 1u));
    if (lane == 31 - __clz(same)) cnt[warp][digit[r]] = rank[r] + 1;
    __syncwarp();
  }
  __syncthreads();
  uint32_t run = offs[(size_t)threadIdx.x * nblocks + blockIdx.x];
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t c = cnt[w][threadIdx.x];
    cnt[w][threadIdx.x] = run;
    run += c;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * 32 + lane;
    if (i < N) {
      const uint32_t at = cnt[warp][digit[r]] + rank[r];
      key_out[at] = key[r];
      pos_out[at] = in.get_pos(i);
    }
  }
}

// ---------------------------------------------------------------- gradient
// A block sums kRun sorted positions of 256 VEC columns.
// Ids whose run of positions lies inside write their row of the table; a run cut by
// the block's ends leaves an fp32 part: parts[2 b] of the one that began before,
// parts[2 b + 1] of the one that began here and goes on.  So a frequent id's rows
// are read by as many blocks as they fill, and every order of sums is fixed.
// The blocks behind the sums (clear_rows) write the rows that no id names: a table
// row is written once, and the two kinds of blocks share the DRAM's time.
constexpr int kClearRows = 32;

// Rows [v0, v0 + 32) of the table: lane = row finds whether an id names it.
template <class T>
__device__ __forceinline__ void clear_rows(const uint32_t* __restrict__ key, int64_t N, int64_t v0,
                                           int V, int D, int vec, T* __restrict__ dtable) {
  __shared__ uint32_t s_empty;
  if (threadIdx.x < 32) {
    const uint32_t v = (uint32_t)v0 + threadIdx.x;
    bool empty = false;
    if (v < (uint32_t)V) {
      int64_t lo = 0, hi = N;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (key[mid] < v) lo = mid + 1; else hi = mid;
      }
      empty = lo == N || key[lo] != v;
    }
    const uint32_t m = __ballot_sync(0xffffffffu, empty);
    if (threadIdx.x == 0) s_empty = m;
  }
  __syncthreads();
  for (uint32_t m = s_empty; m; m &= m - 1) {
    T* row = dtable + (v0 + (__ffs(m) - 1)) * D;
    if (vec) {
      const int n = (int)(D * sizeof(T) / 16);
      for (int i = threadIdx.x; i < n; i += 256) reinterpret_cast<uint4*>(row)[i] = make_uint4(0u, 0u, 0u, 0u);
    } else {
      for (int i = threadIdx.x; i < D; i += 256) row[i] = from_f32<T>(0.f);
    }
  }
}

template <class T, int VEC>
__device__ __forceinline__ void write_row(T* dst, const float (&s)[VEC], float scale,
                                          int accumulate) {
  Pack<T, VEC> x;
  if (accumulate) x.load(dst);
#pragma unroll
  for (int k = 0; k < VEC; ++k)
    x.v[k] = from_f32<T>(fmaf(s[k], scale, accumulate ? to_f32(x.v[k]) : 0.f));
  x.store(dst);
}

template <class T, int VEC>
__global__ void __launch_bounds__(256, 5)
run_sum_kernel(const T* __restrict__ g, int64_t dsn, int64_t dsd, const uint32_t* __restrict__ key,
               const uint32_t* __restrict__ pos, int64_t N, int V, int D, float scale,
               int accumulate, int col_blocks, int64_t sums, T* __restrict__ dtable,
               float* __restrict__ parts, uint32_t* __restrict__ joins) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x >= sums) {
    clear_rows<T>(key, N, (blockIdx.x - sums) * (int64_t)kClearRows, V, D, VEC > 1, dtable);
    return;
  }
  __shared__ uint32_t skey[kRun + 2], spos[kRun];
  const int64_t run = blockIdx.x / col_blocks;
  const int64_t base = run * kRun;
  const int n = (int)min((int64_t)kRun, N - base);
  if (threadIdx.x < kRun + 2) {   // the key before the block's, its keys, and the one behind
    const int64_t i = base + (int)threadIdx.x - 1;
    skey[threadIdx.x] = i >= 0 && i < N ? key[i] : 0xffffffffu;
  }
  if (threadIdx.x < n) spos[threadIdx.x] = pos[base + threadIdx.x];
  __syncthreads();
  const int64_t d0 = ((blockIdx.x - run * col_blocks) * 256ll + threadIdx.x) * VEC;
  // the block's last run began here and goes on: a join for the closing kernel (joins[0]
  // counts them; their order does not matter, each writes its own row)
  if (d0 == 0 && n == kRun && skey[kRun] != (uint32_t)V && skey[kRun + 1] == skey[kRun] &&
      !(skey[1] == skey[kRun] && skey[0] == skey[1]))
    joins[1 + atomicAdd(&joins[0], 1u)] = (uint32_t)run;
  if (d0 >= D) return;
  float s[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[k] = 0.f;
  bool from_before = skey[0] == skey[1];
  for (int j0 = 0; j0 < n; j0 += 4) {
    Pack<T, VEC> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (j0 + u < n && skey[j0 + u + 1] != (uint32_t)V) x[u].load(g + (int64_t)spos[j0 + u] * dsn + d0 * dsd);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + u;
      if (j >= n || skey[j + 1] == (uint32_t)V) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] += to_f32(x[u].v[k]);
      const bool ends = skey[j + 2] != skey[j + 1];
      if (!ends && j + 1 < n) continue;
      if (ends && !from_before) {
        write_row<T, VEC>(dtable + (int64_t)skey[j + 1] * D + d0, s, scale, accumulate);
      } else {
        float* dst = parts + (2 * run + (from_before ? 0 : 1)) * D + d0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) dst[k] = s[k];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] = 0.f;
      from_before = false;
    }
  }
}

// Joins the parts of the runs that blocks cut: the part a run began with, then one
// per block up to its end.  Blocks take (run, 256 columns) in turn; 512 threads = 8
// groups of parts x 64 threads of 4 columns.
template <class T>
__global__ void __launch_bounds__(512)
join_runs_kernel(const uint32_t* __restrict__ key, int64_t N, int V, int D, float scale,
                 int accumulate, T* __restrict__ dtable, const float* __restrict__ parts,
                 const uint32_t* __restrict__ joins) {
  pdl_trigger();
  pdl_wait();
  __shared__ int64_t s_last;
  __shared__ float red[8][64][4];
  const int tiles = (D + 255) / 256;
  const int64_t units = (int64_t)joins[0] * tiles;
  const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const bool vec = D % 4 == 0;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t j = u / tiles, b = joins[1 + j], end = (b + 1) * kRun;
    const uint32_t v = key[end];
    if (threadIdx.x < 32) {   // the block in which the run ends: the last whose first key is v
      int64_t last = b;
      for (;;) {
        const int64_t at = (last + 1 + threadIdx.x) * kRun;
        const int n = __popc(__ballot_sync(0xffffffffu, at < N && key[at] == v));
        last += n;                                      // a prefix of the lanes
        if (n < 32) break;
      }
      if (threadIdx.x == 0) s_last = last;
    }
    __syncthreads();
    const int64_t count = s_last - b + 1;
    const int d0 = (int)(u - j * tiles) * 256 + lane * 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (d0 < D) {
#pragma unroll 4
      for (int64_t i = grp; i < count; i += 8) {
        // part i of the run: i = 0 the beginning, i >= 1 block b + i's first
        const float* src = parts + (i == 0 ? 2 * b + 1 : 2 * (b + i)) * D + d0;
        if (vec) {
          const float4 x = *reinterpret_cast<const float4*>(src);
          s[0] += x.x; s[1] += x.y; s[2] += x.z; s[3] += x.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (d0 + k < D) s[k] += src[k];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) red[grp][lane][k] = s[k];
    __syncthreads();
    if (grp == 0) {
      for (int k = 0; k < 4 && d0 + k < D; ++k) {
        float t = red[0][lane][k];
        for (int q = 1; q < 8; ++q) t += red[q][lane][k];
        T* dst = dtable + (int64_t)v * D + d0 + k;
        *dst = from_f32<T>(fmaf(t, scale, accumulate ? to_f32(*dst) : 0.f));
      }
    }
    __syncthreads();
  }
}

struct EmbedWs {
  uint32_t *key[2], *pos[2], *hist, *joins;
  float* parts;
  size_t bytes;
  EmbedWs(void* p, int64_t N, int D) {
    WsCarve c(p);
    const bool long_sort = N > kClusterSortMax;
    const int64_t nblocks = (N + kSortTile - 1) / kSortTile;
    for (int k = 0; k < 2; ++k) {
      key[k] = c.take<uint32_t>(k == 0 || long_sort ? N : 0);
      pos[k] = c.take<uint32_t>(k == 0 || long_sort ? N : 0);
    }
    hist = c.take<uint32_t>(long_sort ? (size_t)kDigits * nblocks : 0);
    joins = c.take<uint32_t>(1 + (N + kRun - 1) / kRun);
    parts = c.take<float>((size_t)((N + kRun - 1) / kRun) * 2 * D);
    bytes = c.used;
  }
};

template <int ITEMS>
cudaError_t cluster_sort(const int64_t* ids, int64_t ignore, int64_t N, int V, int bits,
                         int digit_bits, const EmbedWs& ws, cudaStream_t stream) {
  const size_t smem = (size_t)kClusterSortThreads * ITEMS * 8 + 32 * kDigits * 2;
  auto* kernel = cluster_sort_kernel<ITEMS>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  int blocks = 1;
  while ((int64_t)blocks * kClusterSortThreads * ITEMS < N) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kClusterSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, kernel, ids, ignore, V, (int)N, bits, digit_bits, ws.key[0],
                            ws.pos[0], ws.joins);
}

// Sorts the ids into ws.key[*at], ws.pos[*at].
cudaError_t sort_ids(const int64_t* ids, int64_t ignore, int64_t N, int V, const EmbedWs& ws,
                     cudaStream_t stream, int* at) {
  int bits = 1;
  while ((int64_t(1) << bits) <= V) ++bits;    // keys 0 .. V
  const int passes = (bits + kDigitBits - 1) / kDigitBits;
  const int digit_bits = (bits + passes - 1) / passes;
  *at = 0;
  if (N <= kClusterSortMax) {
    // few ids a thread: the ranking's rounds are the time of a pass
    auto run = [&](auto items) {
      return cluster_sort<decltype(items)::value>(ids, ignore, N, V, bits, digit_bits, ws, stream);
    };
    constexpr int64_t full = (int64_t)kClusterSortThreads * kClusterSortBlocks;
    if (N <= 2 * full) return run(std::integral_constant<int, 2>{});
    if (N <= 8 * full) return run(std::integral_constant<int, 8>{});
    return run(std::integral_constant<int, 16>{});
  }
  const uint32_t mask = (1u << digit_bits) - 1u;
  const int nblocks = (int)((N + kSortTile - 1) / kSortTile);
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    const SortIn in{pass == 0 ? ids : nullptr, ignore, V, ws.key[*at], ws.pos[*at]};
    const int to = pass == 0 ? 0 : *at ^ 1;
    sort_count_kernel<<<nblocks, kSortThreads, 0, stream>>>(in, N, shift, mask, ws.hist, nblocks);
    sort_scan_kernel<<<1, 1024, 0, stream>>>(ws.hist, (int64_t)kDigits * nblocks, ws.joins);
    sort_scatter_kernel<<<nblocks, kSortThreads, 0, stream>>>(in, N, shift, digit_bits, ws.hist,
                                                             nblocks, ws.key[to], ws.pos[to]);
    count_launches(3);
    *at = to;
  }
  return cudaSuccess;
}

// Rows of `size`-byte elements take 16-byte accesses.
bool rows_vec(const void* p, int64_t s0, int64_t s1, int D, int size) {
  return s1 == 1 && D * (int64_t)size % 16 == 0 && s0 * size % 16 == 0 &&
         (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

}  // namespace
}  // namespace fgmm

extern "C" {

int fgmm_embed_fwd(int type, const void* table, int64_t t_stride_v, int64_t t_stride_d,
                   const int64_t* ids, int64_t ignore_index, int64_t N, int32_t V, int32_t D,
                   float scale, void* out, void* stream) {
  using namespace fgmm;
  static const char* name = "fgmm_embed_fwd";
  return vocab_entry(name, [&]() -> int {
    int rc = vocab_check_shape(name, type, N, V, D);
    if (rc != FGMM_OK) return rc;
    if (N > 0 && (!table || !ids || !out))
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": null pointer argument");
    rc = vocab_check_array(name, "table", table, type_size(type), t_stride_v, t_stride_d);
    if (rc == FGMM_OK) rc = vocab_check_array(name, "out", out, type_size(type), 0, 0);
    if (rc == FGMM_OK) rc = vocab_check_array(name, "ids", ids, 8, 0, 0);
    if (rc != FGMM_OK) return rc;
    std::string why;
    rc = entry_check_device(&why);
    if (rc != FGMM_OK) return entry_fail(rc, std::string(name) + ": " + why);
    if (N == 0) return FGMM_OK;
    with_type(type, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      constexpr int VEC = 16 / sizeof(T);
      const T* t = static_cast<const T*>(table);
      T* o = static_cast<T*>(out);
      cudaStream_t st = (cudaStream_t)stream;
      const bool vec = rows_vec(table, t_stride_v, t_stride_d, D, sizeof(T)) &&
                       rows_vec(out, D, 1, D, sizeof(T));
      int lanes = 1;
      while (lanes < 256 && lanes < (vec ? D / VEC : D)) lanes *= 2;
      const int64_t per_block = 4 * (256 / lanes);
      const int blocks = (int)std::min<int64_t>((N + per_block - 1) / per_block, 1 << 20);
      if (vec)
        lookup_kernel<T, VEC><<<blocks, 256, 0, st>>>(t, t_stride_v, t_stride_d, ids, ignore_index,
                                                      N, V, D, scale, lanes, o);
      else
        lookup_kernel<T, 1><<<blocks, 256, 0, st>>>(t, t_stride_v, t_stride_d, ids, ignore_index, N,
                                                    V, D, scale, lanes, o);
      count_launches(1);
    });
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
      return entry_fail(FGMM_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
    return FGMM_OK;
  });
}

size_t fgmm_embed_workspace_bytes(int64_t N, int32_t V, int32_t D) {
  using namespace fgmm;
  if (N < 0 || V < 1 || D < 1 || N >= kVocabMaxN || V >= kVocabMaxV || D > kVocabMaxD) return 0;
  return EmbedWs(nullptr, N, D).bytes;
}

int fgmm_embed_bwd(int type, const void* dout, int64_t d_stride_n, int64_t d_stride_d,
                   const int64_t* ids, int64_t ignore_index, int64_t N, int32_t V, int32_t D,
                   float scale, void* dtable, void* workspace, size_t workspace_bytes,
                   unsigned flags, void* stream) {
  using namespace fgmm;
  static const char* name = "fgmm_embed_bwd";
  return vocab_entry(name, [&]() -> int {
    int rc = vocab_check_shape(name, type, N, V, D);
    if (rc != FGMM_OK) return rc;
    if (flags & ~FGMM_FLAG_ACCUMULATE)
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": unknown flags");
    if (!dtable || (N > 0 && (!dout || !ids)))
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": null pointer argument");
    rc = vocab_check_array(name, "dout", dout, type_size(type), d_stride_n, d_stride_d);
    if (rc == FGMM_OK) rc = vocab_check_array(name, "dtable", dtable, type_size(type), 0, 0);
    if (rc == FGMM_OK) rc = vocab_check_array(name, "ids", ids, 8, 0, 0);
    const int64_t out_bytes = (int64_t)V * D * type_size(type);
    if (rc == FGMM_OK)
      rc = vocab_check_overlap(name, "dout", dout, N, D, d_stride_n, d_stride_d, type_size(type),
                               "dtable", dtable, out_bytes);
    if (rc == FGMM_OK)
      rc = vocab_check_overlap(name, "ids", ids, N, 1, 1, 1, 8, "dtable", dtable, out_bytes);
    if (rc != FGMM_OK) return rc;
    std::string why;
    rc = entry_check_device(&why);
    if (rc != FGMM_OK) return entry_fail(rc, std::string(name) + ": " + why);
    const EmbedWs ws(workspace, N, D);
    rc = vocab_check_workspace(name, workspace, workspace_bytes, ws.bytes);
    if (rc != FGMM_OK) return rc;
    const int accumulate = (flags & FGMM_FLAG_ACCUMULATE) ? 1 : 0;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = cudaSuccess;
    if (N == 0) {
      if (!accumulate) e = cudaMemsetAsync(dtable, 0, (size_t)V * D * type_size(type), st);
    } else {
      int at = 0;
      e = sort_ids(ids, ignore_index, N, V, ws, st, &at);
      if (e == cudaSuccess) with_type(type, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr int VEC = 16 / sizeof(T);
        const T* g = static_cast<const T*>(dout);
        T* out = static_cast<T*>(dtable);
        const unsigned runs = (unsigned)((N + kRun - 1) / kRun);
        const bool vec = rows_vec(dout, d_stride_n, d_stride_d, D, sizeof(T)) &&
                         rows_vec(dtable, D, 1, D, sizeof(T));
        const int cols = 256 * (vec ? VEC : 1), col_blocks = (D + cols - 1) / cols;
        const int64_t sums = (int64_t)runs * col_blocks;
        const unsigned grid = (unsigned)(sums + (accumulate ? 0 : ((int64_t)V + kClearRows - 1) / kClearRows));
        e = launch(vec ? run_sum_kernel<T, VEC> : run_sum_kernel<T, 1>, grid, 256, 0, st, true, g,
                   d_stride_n, d_stride_d, ws.key[at], ws.pos[at], N, V, D, scale, accumulate,
                   col_blocks, sums, out, ws.parts, ws.joins);
        if (runs > 1 && e == cudaSuccess) {
          const int64_t most = (int64_t)(runs - 1) * ((D + 255) / 256);
          e = launch(join_runs_kernel<T>, std::min<int64_t>(most, 4 * num_sms()), 512, 0, st, true,
                     ws.key[at], N, V, D, scale, accumulate, out, ws.parts, ws.joins);
        }
      });
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess)
      return entry_fail(FGMM_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
    return FGMM_OK;
  });
}

}  // extern "C"
