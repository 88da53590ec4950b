// Linear softmax cross entropy over the V rows of a table W, and its gradient,
// without keeping the N x V logits.
//
//   S = X W^T + c,   logZ_n = log sum_v exp S_nv,   loss_n = logZ_n - S_{n,t_n}
//   g_nv = a_n exp(S_nv - logZ_n) - b_n [v = t_n],   a = w + dlogZ,  b = w
//   dX = g W,   dW = g^T X,   dc_v = sum_n g_nv
//
// Rows that are not ignored are gathered into a dense, zero-padded copy of X
// first ("live" rows, in their order): ignored rows cost no products, and what
// they hold never meets a product.  The vocabulary then runs in pieces: each
// piece's logits go to the workspace, and are folded into the rows' running
// (max, sum) (forward) or turned into g and multiplied with W and X (backward).
#include <algorithm>

#include "fgmm_vocab.cuh"

namespace fgmm {
namespace {

constexpr int kRowTile = 256;   // live rows are padded to this
constexpr float kLog2Ef = 1.4426950408889634f;
constexpr float kLn2f = 0.6931471805599453f;

struct XentArgs {
  const char* name;
  int type;
  const void* X;
  int64_t sxn, sxd;
  const void* W;
  int64_t swv, swd;
  const float* bias;
  const int64_t* targets;
  int64_t ignore;
  int64_t N;
  int V, D;
  // forward
  float *loss, *logZ;
  int reduction;
  float *reduced, *count;
  // backward
  const float* logZ_in;
  const float* dloss;
  int64_t dloss_stride;
  const float* count_in;
  const float* dlogZ;
  void *dX, *dW;
  float* dbias;
  void* ws;
  size_t ws_bytes;
  cudaStream_t stream;
};

// What the backward pass knows of a live row.
struct __align__(16) RowGrad {
  float lse;     // logZ
  float a, b;
  int target;
};

constexpr int kRowsPerBlock = 4096;

// Lists the live rows in their order (rows[0, *live)); block b counts the
// live rows before its own 4096 by reading all earlier labels (from L2), so
// one launch does it without a second pass.  Ignored rows get loss = logZ = 0.
// The last block pads the list to a multiple of kRowTile with -1.
__global__ void __launch_bounds__(1024)
rows_kernel(const XentArgs a, int* __restrict__ rows, int* __restrict__ live) {
  __shared__ int wsum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = (int64_t)blockIdx.x * kRowsPerBlock;
  int before = 0;
  for (int64_t i = threadIdx.x; i < base; i += 1024) before += a.targets[i] != a.ignore;
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) wsum[warp] = before;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < 32; ++w) at += wsum[w];
  for (int r = 0; r < kRowsPerBlock; r += 1024) {
    const int64_t i = base + r + threadIdx.x;
    const bool keep = i < a.N && a.targets[i] != a.ignore;
    const unsigned m = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) wsum[warp] = __popc(m);
    __syncthreads();
    int mine = at, all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) mine += wsum[w];
      all += wsum[w];
    }
    if (keep) rows[mine + __popc(m & ((1u << lane) - 1u))] = (int)i;
    else if (i < a.N && a.loss) a.loss[i] = a.logZ[i] = 0.f;
    at += all;
  }
  if (blockIdx.x == gridDim.x - 1) {
    const int64_t padded = (a.N + kRowTile - 1) / kRowTile * kRowTile;
    for (int64_t i = at + threadIdx.x; i < padded; i += 1024) rows[i] = -1;
    if (threadIdx.x == 0) *live = at;
  }
}

// Xp[i] = X[rows[i]], zero behind the last live row of its tile and behind D.
template <class T>
__global__ void pack_rows_kernel(const T* __restrict__ X, int64_t sxn, int64_t sxd, int D, int Dp,
                                 const int* __restrict__ rows, const int* __restrict__ live,
                                 T* __restrict__ Xp) {
  const int64_t nrows = (*live + kRowTile - 1) / kRowTile * kRowTile;
  for (int64_t i = blockIdx.x; i < nrows; i += gridDim.x) {
    const int r = rows[i];
    for (int d = threadIdx.x; d < Dp; d += blockDim.x)
      Xp[i * Dp + d] = r >= 0 && d < D ? X[r * sxn + d * sxd] : from_f32<T>(0.f);
  }
}

__global__ void row_grad_kernel(const XentArgs a, const int* __restrict__ rows,
                                const int* __restrict__ live, RowGrad* __restrict__ rg) {
  const int64_t n = (*live + kRowTile - 1) / kRowTile * kRowTile;
  const float inv = a.count_in ? 1.f / *a.count_in : 1.f;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    RowGrad r{0.f, 0.f, 0.f, -1};
    const int n0 = rows[i];
    if (n0 >= 0) {
      const int64_t t = a.targets[n0];
      r.b = a.dloss ? a.dloss[n0 * a.dloss_stride] * inv : 0.f;
      r.a = r.b + (a.dlogZ ? a.dlogZ[n0] : 0.f);
      r.lse = a.logZ_in[n0];
      if (t >= 0 && t < a.V) r.target = (int)t;
      else r.a = __int_as_float(0x7fffffff);   // a label outside the table: NaN
    }
    rg[i] = r;
  }
}

// C[m, n] (+)= sum_k A(m, k) B(k, n) for m < M, k < K, where M and K are also
// bounded by *live when live_m / live_k is set (rounded up to kRowTile rows).
// 64 x 64 tiles, 256 threads, 4 x 4 outputs a thread.
template <class TA, class TB>
__global__ void __launch_bounds__(256)
gemm_kernel(const TA* __restrict__ A, int64_t sam, int64_t sak, const TB* __restrict__ B,
            int64_t sbk, int64_t sbn, float* __restrict__ C, int64_t ldc, int64_t M, int64_t Nn,
            int64_t K, const int* live_m, const int* live_k, int add) {
  __shared__ float As[16][65], Bs[16][65];
  if (live_m) M = min(M, (int64_t)((*live_m + kRowTile - 1) / kRowTile * kRowTile));
  if (live_k) K = min(K, (int64_t)*live_k);
  const int64_t n0 = (int64_t)blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t m0 = (int64_t)blockIdx.y * 64; m0 < M; m0 += (int64_t)gridDim.y * 64) {
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += 16) {
      for (int e = threadIdx.x; e < 1024; e += 256) {
        int mm = e >> 4, kk = e & 15;
        if (sam == 1) { mm = e & 63; kk = e >> 6; }
        As[kk][mm] = m0 + mm < M && k0 + kk < K ? to_f32(A[(m0 + mm) * sam + (k0 + kk) * sak]) : 0.f;
        int nn = e >> 4;
        kk = e & 15;
        if (sbn == 1) { nn = e & 63; kk = e >> 6; }
        Bs[kk][nn] = n0 + nn < Nn && k0 + kk < K ? to_f32(B[(k0 + kk) * sbk + (n0 + nn) * sbn]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < 16; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += As[kk][ty * 4 + i] * Bs[kk][tx * 4 + j];
      __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
        if (m < M && n < Nn) C[m * ldc + n] = acc[i][j] + (add ? C[m * ldc + n] : 0.f);
      }
  }
}

template <class TA, class TB>
void gemm(cudaStream_t st, const TA* A, int64_t sam, int64_t sak, const TB* B, int64_t sbk,
          int64_t sbn, float* C, int64_t ldc, int64_t M, int64_t Nn, int64_t K, const int* live_m,
          const int* live_k, int add) {
  const dim3 grid((unsigned)((Nn + 63) / 64), (unsigned)std::min<int64_t>((M + 63) / 64, 1024));
  gemm_kernel<TA, TB><<<grid, 256, 0, st>>>(A, sam, sak, B, sbk, sbn, C, ldc, M, Nn, K, live_m,
                                            live_k, add);
  count_launches(1);
}

// Sum of v over the block's 256 threads, in a fixed order.
__device__ __forceinline__ float block_sum256(float v, float* red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < 8; ++w) s += red[w];
  return s;
}

// Folds one piece of logits into the rows' running (max, sum, target logit);
// the last piece writes loss and logZ.  One block per live row.
__global__ void __launch_bounds__(256)
lse_piece_kernel(const XentArgs a, const int* __restrict__ rows, const int* __restrict__ live,
                 const float* __restrict__ S, int64_t ld, int v0, int nv, float* __restrict__ m_run,
                 float* __restrict__ s_run, float* __restrict__ t_run, int last) {
  __shared__ float red[8];
  for (int64_t i = blockIdx.x; i < *live; i += gridDim.x) {
    const float* s = S + i * ld;
    float m = -3.402823466e38f;
    for (int v = threadIdx.x; v < nv; v += 256) m = fmaxf(m, s[v] + (a.bias ? a.bias[v0 + v] : 0.f));
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
    if (v0 > 0) m = fmaxf(m, m_run[i]);
    float sum = 0.f;
    for (int v = threadIdx.x; v < nv; v += 256)
      sum += expf(s[v] + (a.bias ? a.bias[v0 + v] : 0.f) - m);
    sum = block_sum256(sum, red);
    if (threadIdx.x == 0) {
      if (v0 > 0) sum += s_run[i] * expf(m_run[i] - m);
      m_run[i] = m;
      s_run[i] = sum;
      const int r = rows[i];
      const int64_t t = a.targets[r];
      if (t >= v0 && t < (int64_t)v0 + nv) t_run[i] = s[t - v0] + (a.bias ? a.bias[t] : 0.f);
      else if (t < 0 || t >= a.V) t_run[i] = __int_as_float(0x7fffffff);
      if (last) {
        const float lz = m + logf(sum);
        a.logZ[r] = lz;
        a.loss[r] = lz - t_run[i];
      }
    }
    __syncthreads();
  }
}

// Sum or mean of the live rows' losses, one block, in double.
__global__ void __launch_bounds__(1024)
reduce_loss_kernel(const XentArgs a, const int* __restrict__ rows, const int* __restrict__ live) {
  __shared__ double red[1024];
  double s = 0;
  for (int64_t i = threadIdx.x; i < *live; i += 1024) s += a.loss[rows[i]];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 512; o; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *a.count = (float)*live;
    *a.reduced = (float)(a.reduction == FGMM_REDUCE_MEAN ? red[0] / *live : red[0]);
  }
}

// Logits -> g in place, for the padded live rows.
__global__ void __launch_bounds__(256)
grad_piece_kernel(const XentArgs a, const int* __restrict__ live, const RowGrad* __restrict__ rg,
                  float* __restrict__ S, int64_t ld, int v0, int nv) {
  const int64_t n = (*live + kRowTile - 1) / kRowTile * kRowTile;
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const RowGrad r = rg[i];
    for (int v = threadIdx.x; v < nv; v += 256) {
      const float s = S[i * ld + v] + (a.bias ? a.bias[v0 + v] : 0.f);
      float g = r.a == 0.f ? 0.f : r.a * expf(s - r.lse);
      if (v0 + v == r.target) g -= r.b;
      S[i * ld + v] = g;
    }
  }
}

__global__ void col_sum_kernel(const int* __restrict__ live, const float* __restrict__ G,
                               int64_t ld, int nv, float* __restrict__ out) {
  for (int v = blockIdx.x * blockDim.x + threadIdx.x; v < nv; v += gridDim.x * blockDim.x) {
    double s = 0;
    for (int64_t i = 0; i < *live; ++i) s += G[i * ld + v];
    out[v] = (float)s;
  }
}

// out rows of type T from fp32 rows; dX: scattered to the live rows, the
// ignored rows (rows_of == null: every row in place) having been cleared.
template <class T>
__global__ void store_rows_kernel(const float* __restrict__ acc, int D, int64_t n,
                                  const int* __restrict__ rows, const int* __restrict__ live,
                                  T* __restrict__ out) {
  if (live) n = *live;
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t r = rows ? rows[i] : i;
    for (int d = threadIdx.x; d < D; d += blockDim.x) out[r * D + d] = from_f32<T>(acc[i * D + d]);
  }
}

struct XentWs {
  int *live, *rows;
  void* Xp;
  float *m_run, *s_run, *t_run;
  RowGrad* rg;
  float *S, *dXacc, *dWacc;
  int piece;
  int64_t Np;
  int Dp;
  size_t bytes;
  XentWs(void* p, bool backward, int type, int64_t N, int V, int D) {
    WsCarve c(p);
    Np = (N + kRowTile - 1) / kRowTile * kRowTile;
    Dp = (D + 7) / 8 * 8;
    piece = (int)std::min<int64_t>(V, std::max<int64_t>(128, (int64_t(1) << 26) / std::max<int64_t>(Np, 1)));
    live = c.take<int>(1);
    rows = c.take<int>(Np);
    Xp = c.take<char>((size_t)Np * Dp * type_size(type));
    S = c.take<float>((size_t)Np * piece);
    if (backward) {
      rg = c.take<RowGrad>(Np);
      dXacc = c.take<float>((size_t)Np * D);
      dWacc = c.take<float>((size_t)piece * D);
    } else {
      m_run = c.take<float>(Np);
      s_run = c.take<float>(Np);
      t_run = c.take<float>(Np);
    }
    bytes = c.used;
  }
};

int grid_for(int64_t n) { return (int)std::min<int64_t>(std::max<int64_t>(n, 1), 16 * num_sms()); }

template <class T>
void pack_rows(const XentArgs& a, const XentWs& w) {
  rows_kernel<<<(unsigned)((a.N + kRowsPerBlock - 1) / kRowsPerBlock), 1024, 0, a.stream>>>(a, w.rows, w.live);
  pack_rows_kernel<T><<<grid_for(w.Np), 256, 0, a.stream>>>(
      static_cast<const T*>(a.X), a.sxn, a.sxd, a.D, w.Dp, w.rows, w.live, static_cast<T*>(w.Xp));
  count_launches(2);
}

template <class T>
void logits_piece(const XentArgs& a, const XentWs& w, int v0, int nv) {
  const T* W = static_cast<const T*>(a.W);
  gemm<T, T>(a.stream, static_cast<const T*>(w.Xp), w.Dp, 1, W + (int64_t)v0 * a.swv, a.swd, a.swv,
             w.S, w.piece, w.Np, nv, a.D, w.live, nullptr, 0);
}

template <class T>
void xent_forward(const XentArgs& a, const XentWs& w) {
  pack_rows<T>(a, w);
  for (int v0 = 0; v0 < a.V; v0 += w.piece) {
    const int nv = std::min(w.piece, a.V - v0);
    logits_piece<T>(a, w, v0, nv);
    lse_piece_kernel<<<grid_for(a.N), 256, 0, a.stream>>>(a, w.rows, w.live, w.S, w.piece, v0, nv,
                                                         w.m_run, w.s_run, w.t_run,
                                                         v0 + nv == a.V);
    count_launches(1);
  }
  if (a.reduction != FGMM_REDUCE_NONE) {
    reduce_loss_kernel<<<1, 1024, 0, a.stream>>>(a, w.rows, w.live);
    count_launches(1);
  }
}

template <class T>
cudaError_t xent_backward(const XentArgs& a, const XentWs& w) {
  pack_rows<T>(a, w);
  row_grad_kernel<<<grid_for(w.Np / 256), 256, 0, a.stream>>>(a, w.rows, w.live, w.rg);
  count_launches(1);
  const T* W = static_cast<const T*>(a.W);
  const T* Xp = static_cast<const T*>(w.Xp);
  for (int v0 = 0; v0 < a.V; v0 += w.piece) {
    const int nv = std::min(w.piece, a.V - v0);
    logits_piece<T>(a, w, v0, nv);
    grad_piece_kernel<<<grid_for(w.Np), 256, 0, a.stream>>>(a, w.live, w.rg, w.S, w.piece, v0, nv);
    count_launches(1);
    if (a.dbias) {
      col_sum_kernel<<<(nv + 63) / 64, 64, 0, a.stream>>>(w.live, w.S, w.piece, nv, a.dbias + v0);
      count_launches(1);
    }
    if (a.dX)
      gemm<float, T>(a.stream, w.S, w.piece, 1, W + (int64_t)v0 * a.swv, a.swv, a.swd, w.dXacc,
                     a.D, w.Np, a.D, nv, w.live, nullptr, v0 > 0);
    if (a.dW) {
      gemm<float, T>(a.stream, w.S, 1, w.piece, Xp, w.Dp, 1, w.dWacc, a.D, nv, a.D, w.Np, nullptr,
                     w.live, 0);
      store_rows_kernel<T><<<grid_for(nv), 256, 0, a.stream>>>(
          w.dWacc, a.D, nv, nullptr, nullptr, static_cast<T*>(a.dW) + (int64_t)v0 * a.D);
      count_launches(1);
    }
  }
  if (a.dX) {
    cudaError_t e = cudaMemsetAsync(a.dX, 0, (size_t)a.N * a.D * sizeof(T), a.stream);
    if (e != cudaSuccess) return e;
    store_rows_kernel<T><<<grid_for(a.N), 256, 0, a.stream>>>(w.dXacc, a.D, 0, w.rows, w.live,
                                                             static_cast<T*>(a.dX));
    count_launches(1);
  }
  return cudaSuccess;
}

int check_common(const XentArgs& a) {
  int rc = vocab_check_shape(a.name, a.type, a.N, a.V, a.D);
  if (rc != FGMM_OK) return rc;
  if (!a.W || (a.N > 0 && (!a.X || !a.targets)))
    return entry_fail(FGMM_ERR_ARG, std::string(a.name) + ": null pointer argument");
  rc = vocab_check_array(a.name, "X", a.X, type_size(a.type), a.sxn, a.sxd);
  if (rc == FGMM_OK) rc = vocab_check_array(a.name, "W", a.W, type_size(a.type), a.swv, a.swd);
  if (rc == FGMM_OK) rc = vocab_check_array(a.name, "targets", a.targets, 8, 0, 0);
  if (rc == FGMM_OK) rc = vocab_check_array(a.name, "bias", a.bias, 4, 0, 0);
  return rc;
}

int check_device_and_workspace(const XentArgs& a, size_t need) {
  std::string why;
  const int rc = entry_check_device(&why);
  if (rc != FGMM_OK) return entry_fail(rc, std::string(a.name) + ": " + why);
  return vocab_check_workspace(a.name, a.ws, a.ws_bytes, need);
}

int finish(const XentArgs& a, cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess)
    return entry_fail(FGMM_ERR_CUDA, std::string(a.name) + ": " + cudaGetErrorString(e));
  return FGMM_OK;
}

__global__ void empty_reduction_kernel(int mean, float* reduced, float* count) {
  *reduced = mean ? __int_as_float(0x7fffffff) : 0.f;
  *count = 0.f;
}

}  // namespace
}  // namespace fgmm

extern "C" {

size_t fgmm_xent_workspace_bytes(int backward, int type, int64_t N, int32_t V, int32_t D) {
  using namespace fgmm;
  if (type < 0 || type > 2 || N < 0 || V < 1 || D < 1 || N >= kVocabMaxN || V >= kVocabMaxV ||
      D > kVocabMaxD)
    return 0;
  return XentWs(nullptr, backward != 0, type, N, V, D).bytes;
}

int fgmm_xent_fwd(int type, const void* X, int64_t x_stride_n, int64_t x_stride_d, const void* W,
                  int64_t w_stride_v, int64_t w_stride_d, const float* bias,
                  const int64_t* targets, int64_t ignore_index, int64_t N, int32_t V, int32_t D,
                  float* loss, float* logZ, int reduction, float* reduced, float* count,
                  void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fgmm;
  static const char* name = "fgmm_xent_fwd";
  return vocab_entry(name, [&]() -> int {
    XentArgs a{};
    a.name = name; a.type = type;
    a.X = X; a.sxn = x_stride_n; a.sxd = x_stride_d;
    a.W = W; a.swv = w_stride_v; a.swd = w_stride_d;
    a.bias = bias; a.targets = targets; a.ignore = ignore_index;
    a.N = N; a.V = V; a.D = D;
    a.loss = loss; a.logZ = logZ;
    a.reduction = reduction; a.reduced = reduced; a.count = count;
    a.ws = workspace; a.ws_bytes = workspace_bytes; a.stream = (cudaStream_t)stream;
    int rc = check_common(a);
    if (rc != FGMM_OK) return rc;
    if (reduction < FGMM_REDUCE_NONE || reduction > FGMM_REDUCE_MEAN)
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": unknown reduction");
    if ((N > 0 && (!loss || !logZ)) || (reduction != FGMM_REDUCE_NONE && (!reduced || !count)))
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": null pointer argument");
    const XentWs w(workspace, false, type, N, V, D);
    rc = check_device_and_workspace(a, w.bytes);
    if (rc != FGMM_OK) return rc;
    if (N == 0) {
      if (reduction != FGMM_REDUCE_NONE) {
        empty_reduction_kernel<<<1, 1, 0, a.stream>>>(reduction == FGMM_REDUCE_MEAN, reduced, count);
        count_launches(1);
      }
      return finish(a, cudaSuccess);
    }
    with_type(type, [&](auto* tag) { xent_forward<std::remove_pointer_t<decltype(tag)>>(a, w); });
    return finish(a, cudaSuccess);
  });
}

int fgmm_xent_bwd(int type, const void* X, int64_t x_stride_n, int64_t x_stride_d, const void* W,
                  int64_t w_stride_v, int64_t w_stride_d, const float* bias,
                  const int64_t* targets, int64_t ignore_index, int64_t N, int32_t V, int32_t D,
                  const float* logZ, const float* dloss, int64_t dloss_stride, const float* count,
                  const float* dlogZ, void* dX, void* dW, float* dbias, void* workspace,
                  size_t workspace_bytes, void* stream) {
  using namespace fgmm;
  static const char* name = "fgmm_xent_bwd";
  return vocab_entry(name, [&]() -> int {
    XentArgs a{};
    a.name = name; a.type = type;
    a.X = X; a.sxn = x_stride_n; a.sxd = x_stride_d;
    a.W = W; a.swv = w_stride_v; a.swd = w_stride_d;
    a.bias = bias; a.targets = targets; a.ignore = ignore_index;
    a.N = N; a.V = V; a.D = D;
    a.logZ_in = logZ; a.dloss = dloss; a.dloss_stride = dloss_stride; a.count_in = count;
    a.dlogZ = dlogZ; a.dX = dX; a.dW = dW; a.dbias = dbias;
    a.ws = workspace; a.ws_bytes = workspace_bytes; a.stream = (cudaStream_t)stream;
    int rc = check_common(a);
    if (rc != FGMM_OK) return rc;
    if (dloss_stride != 0 && dloss_stride != 1)
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": dloss_stride must be 0 or 1");
    if (N > 0 && !logZ)
      return entry_fail(FGMM_ERR_ARG, std::string(name) + ": null pointer argument");
    rc = vocab_check_array(name, "dX", dX, type_size(type), 0, 0);
    if (rc == FGMM_OK) rc = vocab_check_array(name, "dW", dW, type_size(type), 0, 0);
    if (rc != FGMM_OK) return rc;
    const XentWs w(workspace, true, type, N, V, D);
    rc = check_device_and_workspace(a, w.bytes);
    if (rc != FGMM_OK) return rc;
    cudaError_t e = cudaSuccess;
    if (N == 0) {
      if (dW) e = cudaMemsetAsync(dW, 0, (size_t)V * D * type_size(type), a.stream);
      if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, (size_t)V * 4, a.stream);
      return finish(a, e);
    }
    with_type(type, [&](auto* tag) { e = xent_backward<std::remove_pointer_t<decltype(tag)>>(a, w); });
    return finish(a, e);
  });
}

}  // extern "C"
