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

#include "fgmm_vocab.cuh"

namespace fgmm {
namespace {

constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;                            // per thread
constexpr int kSortTile = kSortThreads * kSortItems;     // ids per block
constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;

template <class T>
__global__ void lookup_kernel(const T* __restrict__ table, int64_t tsv, int64_t tsd,
                              const int64_t* __restrict__ ids, int64_t ignore, int64_t N, int V,
                              int D, float scale, T* __restrict__ out) {
  for (int64_t i = blockIdx.x; i < N; i += gridDim.x) {
    const int64_t id = ids[i];
    const bool skip = id == ignore;
    const bool bad = !skip && (id < 0 || id >= V);
    const T* row = table + (skip || bad ? 0 : id) * tsv;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
      float v = skip ? 0.f : bad ? __int_as_float(0x7fffffff) : to_f32(row[d * tsd]) * scale;
      out[i * D + d] = from_f32<T>(v);
    }
  }
}

// The sort key of an id: ids that contribute nothing go last, as V.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t ignore, int V) {
  return id == ignore || id < 0 || id >= V ? (uint32_t)V : (uint32_t)id;
}

// One pass of the radix sort reads (key, pos) from the arrays, or makes them
// from the ids in the first pass.
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
sort_count_kernel(SortIn in, int64_t N, int shift, uint32_t* __restrict__ hist, int nblocks) {
  __shared__ uint32_t h[kDigits];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    if (i < N) atomicAdd(&h[(in.get_key(i) >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  hist[(size_t)threadIdx.x * nblocks + blockIdx.x] = h[threadIdx.x];
}

// Exclusive prefix sum of hist[0, n) by one block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* __restrict__ hist, int n) {
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int base = 0; base < n; base += 1024) {
    const int i = base + threadIdx.x;
    const uint32_t v = i < n ? hist[i] : 0u;
    uint32_t s = v;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    if (warp == 0) {
      uint32_t w = warp_sum[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += t;
      }
      warp_sum[lane] = w;
    }
    __syncthreads();
    const uint32_t before = carry + (warp ? warp_sum[warp - 1] : 0u) + s - v;
    if (i < n) hist[i] = before;
    __syncthreads();
    if (threadIdx.x == 1023) carry = before + v;
    __syncthreads();
  }
}

// Stable scatter: a warp owns 256 consecutive items and ranks 32 at a time.
__global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(SortIn in, int64_t N, int shift, const uint32_t* __restrict__ offs,
                    int nblocks, uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out) {
  constexpr int kWarps = kSortThreads / 32;
  __shared__ uint32_t cnt[kWarps][kDigits];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int w = 0; w < kWarps; ++w) cnt[w][threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile + warp * (32 * kSortItems);
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * 32 + lane;
    const bool in_range = i < N;
    key[r] = in_range ? in.get_key(i) : 0u;
    const uint32_t d = in_range ? (key[r] >> shift) & (kDigits - 1) : (uint32_t)kDigits;
    const uint32_t same = __match_any_sync(0xffffffffu, d);
    uint32_t before = 0;
    if (in_range) before = cnt[warp][d];
    __syncwarp();
    rank[r] = before + __popc(same & ((1u << lane) - 1u));
    if (in_range && lane == 31 - __clz(same)) cnt[warp][d] = rank[r] + 1;
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
      const uint32_t at = cnt[warp][(key[r] >> shift) & (kDigits - 1)] + rank[r];
      key_out[at] = key[r];
      pos_out[at] = in.get_pos(i);
    }
  }
}

__device__ __forceinline__ int64_t lower_bound(const uint32_t* key, int64_t n, uint32_t v) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (key[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// One block per table row at a time.
template <class T>
__global__ void embed_grad_kernel(const T* __restrict__ g, int64_t dsn, int64_t dsd,
                                  const uint32_t* __restrict__ key,
                                  const uint32_t* __restrict__ pos, int64_t N, int V, int D,
                                  float scale, int accumulate, T* __restrict__ dtable) {
  for (int64_t v = blockIdx.x; v < V; v += gridDim.x) {
    const int64_t lo = lower_bound(key, N, (uint32_t)v);
    const int64_t hi = lower_bound(key, N, (uint32_t)v + 1);
    if (accumulate && lo == hi) continue;
    T* row = dtable + v * D;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
      float s = 0.f;
      for (int64_t j = lo; j < hi; ++j) s += to_f32(g[pos[j] * dsn + d * dsd]);
      s *= scale;
      if (accumulate) s += to_f32(row[d]);
      row[d] = from_f32<T>(s);
    }
  }
}

struct EmbedWs {
  uint32_t *key[2], *pos[2], *hist;
  size_t bytes;
  EmbedWs(void* p, int64_t N) {
    WsCarve c(p);
    const int64_t nblocks = (N + kSortTile - 1) / kSortTile;
    for (int k = 0; k < 2; ++k) {
      key[k] = c.take<uint32_t>(N);
      pos[k] = c.take<uint32_t>(N);
    }
    hist = c.take<uint32_t>((size_t)kDigits * nblocks);
    bytes = c.used;
  }
};

// Sorts the ids; returns the index (0 or 1) of the arrays that hold the result.
int sort_ids(const int64_t* ids, int64_t ignore, int64_t N, int V, const EmbedWs& ws,
             cudaStream_t stream) {
  const int nblocks = (int)((N + kSortTile - 1) / kSortTile);
  int bits = 1;
  while ((int64_t(1) << bits) <= V) ++bits;    // keys 0 .. V
  int at = 0;
  for (int shift = 0, pass = 0; shift < bits; shift += kDigitBits, ++pass) {
    const SortIn in{pass == 0 ? ids : nullptr, ignore, V, ws.key[at], ws.pos[at]};
    const int to = pass == 0 ? 0 : at ^ 1;
    sort_count_kernel<<<nblocks, kSortThreads, 0, stream>>>(in, N, shift, ws.hist, nblocks);
    sort_scan_kernel<<<1, 1024, 0, stream>>>(ws.hist, kDigits * nblocks);
    sort_scatter_kernel<<<nblocks, kSortThreads, 0, stream>>>(in, N, shift, ws.hist, nblocks,
                                                             ws.key[to], ws.pos[to]);
    count_launches(3);
    at = to;
  }
  return at;
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
      const int threads = std::min(256, (D + 31) / 32 * 32);
      const int blocks = (int)std::min<int64_t>(N, 16 * num_sms());
      lookup_kernel<T><<<blocks, threads, 0, (cudaStream_t)stream>>>(
          static_cast<const T*>(table), t_stride_v, t_stride_d, ids, ignore_index, N, V, D, scale,
          static_cast<T*>(out));
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
  return EmbedWs(nullptr, N).bytes;
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
    const EmbedWs ws(workspace, N);
    rc = vocab_check_workspace(name, workspace, workspace_bytes, ws.bytes);
    if (rc != FGMM_OK) return rc;
    const int accumulate = (flags & FGMM_FLAG_ACCUMULATE) ? 1 : 0;
    if (N == 0 && accumulate) return FGMM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const int at = N > 0 ? sort_ids(ids, ignore_index, N, V, ws, st) : 0;
    with_type(type, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      const int threads = std::min(256, (D + 31) / 32 * 32);
      const int blocks = (int)std::min<int64_t>(V, 16 * num_sms());
      embed_grad_kernel<T><<<blocks, threads, 0, st>>>(
          static_cast<const T*>(dout), d_stride_n, d_stride_d, ws.key[at], ws.pos[at], N, V, D,
          scale, accumulate, static_cast<T*>(dtable));
      count_launches(1);
    });
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
      return entry_fail(FGMM_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
    return FGMM_OK;
  });
}

}  // extern "C"
