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

#include "fgmm_vocab.cuh"

namespace fgmm {
namespace {

constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
// Long sorts: blocks of 256 threads x 8 ids.
constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
// Short sorts (up to 16,384 ids): one block, all passes in shared memory.
constexpr int kBlockSortThreads = 1024;
constexpr int64_t kBlockSortMax = 16384;
// Sorted positions per block of the gradient.
constexpr int kRun = 32;

// ---------------------------------------------------------------- lookup
// out = scale * table[id], 16 bytes (VEC elements) a thread; four independent
// rows' pieces in flight each.  Bound by DRAM: N D read (distinct rows) and
// N D written.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
lookup_kernel(const T* __restrict__ table, int64_t tsv, int64_t tsd,
              const int64_t* __restrict__ ids, int64_t ignore, int64_t N, int V, int D, float scale,
              T* __restrict__ out) {
  const int per_row = D / VEC;
  const int64_t total = N * per_row, step = gridDim.x * 256ll;
  for (int64_t e0 = blockIdx.x * 256ll + threadIdx.x; e0 < total; e0 += 4 * step) {
    Pack<T, VEC> x[4];
    int how[4];   // 0 outside, 1 a row, 2 ignored, 3 bad id
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t e = e0 + u * step;
      how[u] = 0;
      if (e < total) {
        const int64_t i = e / per_row;
        const int64_t id = __ldg(ids + i);
        how[u] = id == ignore ? 2 : id < 0 || id >= V ? 3 : 1;
        if (how[u] == 1) {
          const T* src = table + id * tsv + (e - i * per_row) * VEC * tsd;
          x[u].load(src);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (how[u] == 0) continue;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float v = how[u] == 1 ? to_f32(x[u].v[k]) * scale : 0.f;
        if (how[u] == 3) v = __int_as_float(0x7fffffff);
        x[u].v[k] = from_f32<T>(v);
      }
      x[u].store(out + (e0 + u * step) * VEC);
    }
  }
}

// ---------------------------------------------------------------- sort
// The sort key of an id: ids that contribute nothing go last, as V.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t ignore, int V) {
  return id == ignore || id < 0 || id >= V ? (uint32_t)V : (uint32_t)id;
}

// Part of the gradient table that a sorting launch clears: the sort is bound by
// latency and uses few SMs, so the blocks behind its own write the zeros of the
// rows that no id names (and of the others, which the sums overwrite).
struct Fill {
  uint4* ptr;
  int64_t n;   // 16-byte units
  int first;   // first block that fills
  __device__ __forceinline__ bool run() const {
    if ((int)blockIdx.x < first) return false;
    const int64_t step = (int64_t)(gridDim.x - first) * blockDim.x;
    for (int64_t i = (int64_t)(blockIdx.x - first) * blockDim.x + threadIdx.x; i < n; i += step)
      ptr[i] = make_uint4(0u, 0u, 0u, 0u);
    return true;
  }
};

// Rank of each of a warp's ITEMS x 32 consecutive keys among the warp's equal
// digits, in order; cnt (the warp's digit counts, zero before) ends as totals.
template <int ITEMS>
__device__ __forceinline__ void warp_ranks(const uint32_t (&digit)[ITEMS], uint32_t* cnt,
                                           uint32_t (&rank)[ITEMS], int lane) {
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const uint32_t d = digit[r];   // kDigits: none
    const uint32_t same = __match_any_sync(0xffffffffu, d);
    const uint32_t before = d < kDigits ? cnt[d] : 0u;
    __syncwarp();
    rank[r] = before + __popc(same & ((1u << lane) - 1u));
    if (d < kDigits && lane == 31 - __clz(same)) cnt[d] = rank[r] + 1;
    __syncwarp();
  }
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

// Stable sort of up to 1024 ITEMS ids by block 0; the other blocks clear the table.
// A warp owns 32 ITEMS consecutive places; digits are ranked within the warp, the
// warps' counts are summed per digit in warp order, and keys and positions change
// places through shared memory.
template <int ITEMS>
__global__ void __launch_bounds__(kBlockSortThreads)
block_sort_kernel(const int64_t* __restrict__ ids, int64_t ignore, int V, int N, int bits,
                  int digit_bits, uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out,
                  const Fill fill) {
  if (fill.run()) return;
  extern __shared__ uint32_t sm[];
  constexpr int kAll = kBlockSortThreads * ITEMS;
  uint32_t* skey = sm;
  uint32_t* spos = sm + kAll;
  uint16_t* cnt16 = reinterpret_cast<uint16_t*>(sm + 2 * kAll);   // [32][256]
  __shared__ uint32_t warp_sum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = warp * 32 * ITEMS;
  uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = base + 32 * r + lane;
    key[r] = i < N ? sort_key(ids[i], ignore, V) : 0xffffffffu;   // behind the last: stays last
    pos[r] = (uint32_t)i;
  }
  const uint32_t mask = (1u << digit_bits) - 1u;
  for (int shift = 0; shift < bits; shift += digit_bits) {
    for (int i = threadIdx.x; i < 32 * kDigits / 2; i += kBlockSortThreads)
      reinterpret_cast<uint32_t*>(cnt16)[i] = 0u;
    __syncthreads();
    uint16_t* cnt = cnt16 + warp * kDigits;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const uint32_t d = (key[r] >> shift) & mask;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const uint32_t before = cnt[d];
      __syncwarp();
      rank[r] = before + __popc(same & ((1u << lane) - 1u));
      if (lane == 31 - __clz(same)) cnt[d] = (uint16_t)(rank[r] + 1);
      __syncwarp();
    }
    __syncthreads();
    // digit d = thread / 4 of four threads, each for 8 warps: counts -> offsets
    const int d = threadIdx.x >> 2, part = threadIdx.x & 3;
    uint32_t mine = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) mine += cnt16[(part * 8 + w) * kDigits + d];
    uint32_t all;
    uint32_t run = block_prefix1024(mine, warp_sum, &all);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      uint16_t* c = cnt16 + (part * 8 + w) * kDigits + d;
      const uint32_t v = *c;
      *c = (uint16_t)run;
      run += v;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const uint32_t at = cnt[(key[r] >> shift) & mask] + rank[r];
      skey[at] = key[r];
      spos[at] = pos[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      key[r] = skey[base + 32 * r + lane];
      pos[r] = spos[base + 32 * r + lane];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = base + 32 * r + lane;
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
                  int nblocks, const Fill fill) {
  if (fill.run()) return;
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
sort_scan_kernel(uint32_t* __restrict__ hist, int64_t n, const Fill fill) {
  if (fill.run()) return;
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
sort_scatter_kernel(SortIn in, int64_t N, int shift, uint32_t mask,
                    const uint32_t* __restrict__ offs, int nblocks, uint32_t* __restrict__ key_out,
                    uint32_t* __restrict__ pos_out, const Fill fill) {
  if (fill.run()) return;
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
    key[r] = i < N ? in.get_key(i) : 0u;
    digit[r] = i < N ? (key[r] >> shift) & mask : (uint32_t)kDigits;
  }
  warp_ranks<kSortItems>(digit, cnt[warp], rank, lane);
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
// A block sums kRun sorted positions (blockIdx.x) of 256 VEC columns (blockIdx.y).
// Ids whose run of positions lies inside write their row of the table; a run cut by
// the block's ends leaves an fp32 part: parts[2 b] of the one that began before,
// parts[2 b + 1] of the one that began here and goes on.  So a frequent id's rows
// are read by as many blocks as they fill, and every order of sums is fixed.
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
__global__ void __launch_bounds__(256)
run_sum_kernel(const T* __restrict__ g, int64_t dsn, int64_t dsd, const uint32_t* __restrict__ key,
               const uint32_t* __restrict__ pos, int64_t N, int V, int D, float scale,
               int accumulate, T* __restrict__ dtable, float* __restrict__ parts) {
  __shared__ uint32_t skey[kRun + 2], spos[kRun];
  const int64_t base = (int64_t)blockIdx.x * kRun;
  const int n = (int)min((int64_t)kRun, N - base);
  if (threadIdx.x < kRun + 2) {   // the key before the block's, its keys, and the one behind
    const int64_t i = base + (int)threadIdx.x - 1;
    skey[threadIdx.x] = i >= 0 && i < N ? key[i] : 0xffffffffu;
  }
  if (threadIdx.x < n) spos[threadIdx.x] = pos[base + threadIdx.x];
  __syncthreads();
  const int64_t d0 = (blockIdx.y * 256ll + threadIdx.x) * VEC;
  if (d0 >= D) return;
  float s[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[k] = 0.f;
  bool from_before = skey[0] == skey[1];
  for (int j0 = 0; j0 < n; j0 += 8) {
    Pack<T, VEC> x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (j0 + u < n && skey[j0 + u + 1] != (uint32_t)V) x[u].load(g + (int64_t)spos[j0 + u] * dsn + d0 * dsd);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u;
      if (j >= n || skey[j + 1] == (uint32_t)V) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] += to_f32(x[u].v[k]);
      const bool ends = skey[j + 2] != skey[j + 1];
      if (!ends && j + 1 < n) continue;
      if (ends && !from_before) {
        write_row<T, VEC>(dtable + (int64_t)skey[j + 1] * D + d0, s, scale, accumulate);
      } else {
        float* dst = parts + (2 * (int64_t)blockIdx.x + (from_before ? 0 : 1)) * D + d0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) dst[k] = s[k];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] = 0.f;
      from_before = false;
    }
  }
}

// Joins the parts of a run that began in block b and goes on: the part it began
// with, then one per block up to its end.  32 lanes x 4 columns x 8 part groups.
template <class T>
__global__ void __launch_bounds__(256)
join_runs_kernel(const uint32_t* __restrict__ key, int64_t N, int V, int D, float scale,
                 int accumulate, T* __restrict__ dtable, const float* __restrict__ parts) {
  const int64_t b = blockIdx.x, end = (b + 1) * kRun;   // first position behind the block
  if (end >= N) return;
  const uint32_t v = key[end - 1];
  if (v == (uint32_t)V || key[end] != v) return;                // nothing goes on
  const bool whole = key[b * kRun] == v;                        // the block holds nothing else
  if (whole && b > 0 && key[b * kRun - 1] == v) return;         // it began earlier
  __shared__ int64_t s_last;
  if (threadIdx.x == 0) {
    int64_t lo = end, hi = N;                                   // first position with another id
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (key[mid] == v) lo = mid + 1; else hi = mid;
    }
    s_last = (lo - 1) / kRun;
  }
  __shared__ float red[8][32][4];
  __syncthreads();
  const int64_t last = s_last;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int d0 = (blockIdx.y * 32 + lane) * 4;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  // part i of the run: i = 0 the beginning, i >= 1 block b + i's first
  for (int64_t i = grp; i <= last - b; i += 8) {
    const float* src = parts + (i == 0 ? 2 * b + 1 : 2 * (b + i)) * D;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (d0 + k < D) s[k] += src[d0 + k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) red[grp][lane][k] = s[k];
  __syncthreads();
  if (grp == 0) {
    for (int k = 0; k < 4; ++k) {
      if (d0 + k >= D) break;
      float t = red[0][lane][k];
      for (int q = 1; q < 8; ++q) t += red[q][lane][k];
      T* dst = dtable + (int64_t)v * D + d0 + k;
      *dst = from_f32<T>(fmaf(t, scale, accumulate ? to_f32(*dst) : 0.f));
    }
  }
}

struct EmbedWs {
  uint32_t *key[2], *pos[2], *hist;
  float* parts;
  size_t bytes;
  EmbedWs(void* p, int64_t N, int D) {
    WsCarve c(p);
    const bool long_sort = N > kBlockSortMax;
    const int64_t nblocks = (N + kSortTile - 1) / kSortTile;
    for (int k = 0; k < 2; ++k) {
      key[k] = c.take<uint32_t>(k == 0 || long_sort ? N : 0);
      pos[k] = c.take<uint32_t>(k == 0 || long_sort ? N : 0);
    }
    hist = c.take<uint32_t>(long_sort ? (size_t)kDigits * nblocks : 0);
    parts = c.take<float>((size_t)((N + kRun - 1) / kRun) * 2 * D);
    bytes = c.used;
  }
};

// Sorts the ids into ws.key[*at], ws.pos[*at], clearing `bytes` of the table on the way.
cudaError_t sort_ids(const int64_t* ids, int64_t ignore, int64_t N, int V, const EmbedWs& ws,
                     void* table, size_t bytes, cudaStream_t stream, int* at) {
  int bits = 1;
  while ((int64_t(1) << bits) <= V) ++bits;    // keys 0 .. V
  const int passes = (bits + kDigitBits - 1) / kDigitBits;
  const int digit_bits = (bits + passes - 1) / passes;
  const uint32_t mask = (1u << digit_bits) - 1u;
  // 16-byte units of the table between its first and last aligned address, in as many
  // shares as there are launches; the ragged ends (under 16 bytes each) by memset
  char* p0 = static_cast<char*>(table);
  const int launches = N <= kBlockSortMax ? 1 : 3 * passes;
  size_t head = 0, units = 0;
  if (bytes > 0) {
    head = std::min<size_t>(bytes, (16 - (reinterpret_cast<uintptr_t>(p0) & 15)) & 15);
    units = (bytes - head) / 16;
    const size_t tail = bytes - head - 16 * units;
    cudaError_t e = cudaSuccess;
    if (head) e = cudaMemsetAsync(p0, 0, head, stream);
    if (tail && e == cudaSuccess) e = cudaMemsetAsync(p0 + head + 16 * units, 0, tail, stream);
    if (e != cudaSuccess) return e;
  }
  const int64_t share = ((int64_t)units + launches - 1) / launches;
  int64_t filled = 0;
  auto next_fill = [&](int first, int threads) {
    Fill f;
    f.ptr = reinterpret_cast<uint4*>(p0 + head) + filled;
    f.n = std::min<int64_t>(share, (int64_t)units - filled);
    f.first = first;
    filled += f.n;
    const int64_t blocks = std::min<int64_t>((f.n + 4 * threads - 1) / (4 * threads),
                                             (int64_t)num_sms() * (2048 / threads));
    return std::make_pair(f, (unsigned)(first + blocks));
  };
  *at = 0;
  if (N <= kBlockSortMax) {
    auto run = [&](auto items) {
      constexpr int ITEMS = decltype(items)::value;
      const size_t smem = (size_t)kBlockSortThreads * ITEMS * 8 + 32 * kDigits * 2;
      cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(block_sort_kernel<ITEMS>), smem);
      if (e != cudaSuccess) return e;
      const auto f = next_fill(1, kBlockSortThreads);
      block_sort_kernel<ITEMS><<<f.second, kBlockSortThreads, smem, stream>>>(
          ids, ignore, V, (int)N, bits, digit_bits, ws.key[0], ws.pos[0], f.first);
      count_launches(1);
      return cudaSuccess;
    };
    if (N <= 1024) return run(std::integral_constant<int, 1>{});
    if (N <= 4096) return run(std::integral_constant<int, 4>{});
    return run(std::integral_constant<int, 16>{});
  }
  const int nblocks = (int)((N + kSortTile - 1) / kSortTile);
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    const SortIn in{pass == 0 ? ids : nullptr, ignore, V, ws.key[*at], ws.pos[*at]};
    const int to = pass == 0 ? 0 : *at ^ 1;
    auto f = next_fill(nblocks, kSortThreads);
    sort_count_kernel<<<f.second, kSortThreads, 0, stream>>>(in, N, shift, mask, ws.hist, nblocks, f.first);
    f = next_fill(1, 1024);
    sort_scan_kernel<<<f.second, 1024, 0, stream>>>(ws.hist, (int64_t)kDigits * nblocks, f.first);
    f = next_fill(nblocks, kSortThreads);
    sort_scatter_kernel<<<f.second, kSortThreads, 0, stream>>>(in, N, shift, mask, ws.hist, nblocks,
                                                              ws.key[to], ws.pos[to], f.first);
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
      // a block per 256 pieces while they all fit on the SMs at once, then four each
      const int64_t pieces = N * (vec ? D / VEC : D);
      const int blocks = (int)std::max<int64_t>(
          std::min<int64_t>((pieces + 255) / 256, 8 * num_sms()),
          std::min<int64_t>((pieces + 1023) / 1024, 1 << 20));
      if (vec)
        lookup_kernel<T, VEC><<<blocks, 256, 0, st>>>(t, t_stride_v, t_stride_d, ids, ignore_index,
                                                      N, V, D, scale, o);
      else
        lookup_kernel<T, 1><<<blocks, 256, 0, st>>>(t, t_stride_v, t_stride_d, ids, ignore_index, N,
                                                    V, D, scale, o);
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
    if (rc != FGMM_OK) return rc;
    std::string why;
    rc = entry_check_device(&why);
    if (rc != FGMM_OK) return entry_fail(rc, std::string(name) + ": " + why);
    const EmbedWs ws(workspace, N, D);
    rc = vocab_check_workspace(name, workspace, workspace_bytes, ws.bytes);
    if (rc != FGMM_OK) return rc;
    const int accumulate = (flags & FGMM_FLAG_ACCUMULATE) ? 1 : 0;
    cudaStream_t st = (cudaStream_t)stream;
    const size_t bytes = accumulate ? 0 : (size_t)V * D * type_size(type);
    cudaError_t e = cudaSuccess;
    if (N == 0) {
      if (bytes) e = cudaMemsetAsync(dtable, 0, bytes, st);
    } else {
      int at = 0;
      e = sort_ids(ids, ignore_index, N, V, ws, dtable, bytes, st, &at);
      if (e == cudaSuccess) with_type(type, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr int VEC = 16 / sizeof(T);
        const T* g = static_cast<const T*>(dout);
        T* out = static_cast<T*>(dtable);
        const unsigned runs = (unsigned)((N + kRun - 1) / kRun);
        const bool vec = rows_vec(dout, d_stride_n, d_stride_d, D, sizeof(T)) &&
                         rows_vec(dtable, D, 1, D, sizeof(T));
        const unsigned cols = 256 * (vec ? VEC : 1);
        const dim3 grid(runs, (D + cols - 1) / cols);
        if (vec)
          run_sum_kernel<T, VEC><<<grid, 256, 0, st>>>(g, d_stride_n, d_stride_d, ws.key[at], ws.pos[at],
                                                       N, V, D, scale, accumulate, out, ws.parts);
        else
          run_sum_kernel<T, 1><<<grid, 256, 0, st>>>(g, d_stride_n, d_stride_d, ws.key[at], ws.pos[at], N,
                                                     V, D, scale, accumulate, out, ws.parts);
        count_launches(1);
        if (runs > 1) {
          join_runs_kernel<T><<<dim3(runs - 1, (D + 127) / 128), 256, 0, st>>>(
              ws.key[at], N, V, D, scale, accumulate, out, ws.parts);
          count_launches(1);
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
