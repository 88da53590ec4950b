// Linear softmax cross entropy over the V rows of a table W, and its gradient,
// without keeping the N x V logits.
//
//   S = X W^T + c,   logZ_n = log sum_v exp S_nv,   loss_n = logZ_n - S_{n,t_n}
//   g_nv = a_n exp(S_nv - logZ_n) - b_n [v = t_n],   a = w + dlogZ,  b = w
//   dX = g W,   dW = g^T X,   dc_v = sum_n g_nv
//
// Rows that are not ignored are gathered into a dense, zero-padded copy of X
// first ("live" rows, in their order): ignored rows cost no products, and what
// they hold never meets a product.  Forward, logits stay in TMEM and registers and
// leave as a (max, sum) per row and range of the vocabulary.  Backward, they are
// computed again in pieces of the vocabulary; a piece's g goes to the workspace
// and is multiplied with W and X while the next piece's is made.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fgmm_ptx.cuh"
#include "fgmm_vocab.cuh"

namespace fgmm {
namespace {

constexpr float kLog2Ef = 1.4426950408889634f;

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

#include "fgmm_xent_mma.cuh"

// First words of the workspace.
struct Header {
  int err;        // a wait of the tensor-core kernel gave up
  int amax[3];    // float bits of the largest finite |weight|, |x|, |w|
  int done;       // blocks of the closing forward kernel that have finished
  int live;       // rows that are not ignored
};

constexpr int kRowsPerBlock = 4096;
constexpr int kBadTarget = -2;

struct XentWs {
  Header* hdr;
  int *rows, *inv, *target;
  float* bias;
  void *Xp, *Xp2, *Wp, *Wp2;      // packed operands (SPLIT: hi and lo words)
  float2* part;
  float* tlogit;
  double* loss_part;
  RowGrad* rg;
  void *G[2], *G2[2];
  float *dbias_part, *dx_slots, *dw_slots;

  int64_t Np, Vp;
  int Dp;                          // row length of the packed operands
  bool split, pack_w;
  int vtiles, per_split, splits;
  int bn_d, tiles_d;
  int64_t ldS;
  int row_chunk, piece, n_chunks, n_pieces, ks_x, ks_w;
  bool dw_direct;
  size_t bytes;

  static constexpr int kPairs = 74;                        // SM pairs the plan is made for
  static constexpr int64_t kPieceBytes = int64_t(1) << 28; // one buffer of G
  static constexpr int64_t kSlotBytes = int64_t(1) << 28;

  XentWs(void* p, bool backward, int type, int64_t N, int V, int D, const void* W, int64_t swv,
         int64_t swd, bool want_bias) {
    WsCarve c(p);
    split = type == FGMM_T_F32;
    Np = std::max<int64_t>((N + kPairRows - 1) / kPairRows * kPairRows, kPairRows);
    Vp = ((int64_t)V + 255) / 256 * 256;
    Dp = (D + 7) / 8 * 8;
    // W is read in place when TMA can: unit feature stride, rows of whole 16-byte units
    pack_w = split || swd != 1 || swv < D || swv % 8 != 0 || swv >= (int64_t(1) << 38) ||
             (reinterpret_cast<uintptr_t>(W) & 15) != 0;
    hdr = c.take<Header>(1);
    rows = c.take<int>(Np);
    inv = c.take<int>(Np);
    target = c.take<int>(Np);
    bias = c.take<float>(want_bias ? Vp : 0);
    Xp = c.take<uint16_t>((size_t)Np * Dp);
    Xp2 = c.take<uint16_t>(split ? (size_t)Np * Dp : 0);
    Wp = c.take<uint16_t>(pack_w ? (size_t)V * Dp : 0);
    Wp2 = c.take<uint16_t>(split ? (size_t)V * Dp : 0);
    const int64_t mt = Np / kPairRows;
    if (!backward) {
      // Vocabulary tiles per unit: the fewest rounds of the pairs, counting a quarter
      // of a tile per unit for what starting and ending one costs.
      vtiles = (int)(((int64_t)V + kBN - 1) / kBN);
      double best = 1e300;
      for (int splits_ = 1; splits_ <= std::min(vtiles, 4 * kPairs); ++splits_) {
        const int per = (vtiles + splits_ - 1) / splits_, got = (vtiles + per - 1) / per;
        if (2.0 * got * Np * 8 > double(int64_t(1) << 29) && got > 1) break;
        const double rounds = double((mt * got + kPairs - 1) / kPairs) * (per + 0.25);
        if (rounds < best * 0.999) { best = rounds; per_split = per; splits = got; }
      }
      part = c.take<float2>((size_t)2 * splits * Np);
      tlogit = c.take<float>(Np);
      loss_part = c.take<double>((N + 31) / 32);
    } else {
      const int word = split ? 4 : 2;
      // column tiles of dX and dW: 128 wide where that pads D less
      bn_d = (D + 127) / 128 * 128 < (D + 255) / 256 * 256 ? 128 : 256;
      tiles_d = (D + bn_d - 1) / bn_d;
      ldS = (int64_t)tiles_d * bn_d;
      // G in pieces of at most kPieceBytes: all rows x at least 2048 entries if possible
      const int64_t wide = std::min<int64_t>(Vp, 2048);
      row_chunk = (int)std::max<int64_t>(
          256, std::min<int64_t>(Np, kPieceBytes / (wide * word) / 256 * 256));
      piece = (int)std::max<int64_t>(
          256, std::min<int64_t>(Vp, kPieceBytes / ((int64_t)row_chunk * word) / 256 * 256));
      n_chunks = (int)((Np + row_chunk - 1) / row_chunk);
      n_pieces = (int)((Vp + piece - 1) / piece);
      // Splits of K, where a product's tiles alone cannot occupy the pairs
      const int64_t dx_tiles = (int64_t)(row_chunk / 256) * tiles_d, dx_kb = piece / 64;
      const int64_t dw_tiles = (int64_t)(piece / 256) * tiles_d, dw_kb = row_chunk / 64;
      auto pick = [](int64_t tiles, int64_t kb, int64_t slot_bytes) {
        int64_t ks = 1;
        if (tiles < 2 * kPairs) ks = (3 * kPairs + tiles - 1) / tiles;
        ks = std::min(ks, std::max<int64_t>(1, kb / 8));
        return (int)std::max<int64_t>(1, std::min(ks, kSlotBytes / std::max<int64_t>(slot_bytes, 1)));
      };
      ks_x = pick(dx_tiles, dx_kb, Np * ldS * 4);
      ks_w = pick(dw_tiles, dw_kb, (int64_t)piece * ldS * 4);
      dw_direct = n_chunks == 1 && ks_w == 1;
      rg = c.take<RowGrad>(Np);
      const bool two = n_chunks * n_pieces > 1;
      for (int b = 0; b < 2; ++b) {
        G[b] = c.take<uint16_t>(b == 0 || two ? (size_t)row_chunk * piece : 0);
        G2[b] = c.take<uint16_t>(split && (b == 0 || two) ? (size_t)row_chunk * piece : 0);
      }
      dbias_part = c.take<float>(want_bias ? (size_t)(Np / 128) * Vp : 0);
      dx_slots = c.take<float>((size_t)ks_x * Np * ldS);
      dw_slots = c.take<float>(dw_direct ? 0 : (size_t)ks_w * piece * ldS);
    }
    bytes = c.used;
  }
};

// Lists the live rows in their order, with their targets; block b counts the
// live rows before its own 4096 by reading all earlier labels (from L2), so
// one launch does it without a second pass.  Ignored rows get loss = logZ = 0.
// The last block pads the list to a multiple of kPairRows with -1.
__global__ void __launch_bounds__(1024) rows_kernel(const XentArgs a, const XentWs w) {
  __shared__ int wsum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = (int64_t)blockIdx.x * kRowsPerBlock;
  int before = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < base; i += 1024) before += a.targets[i] != a.ignore;
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) wsum[warp] = before;
  __syncthreads();
  int at = 0;
  for (int k = 0; k < 32; ++k) at += wsum[k];
  for (int r = 0; r < kRowsPerBlock && base + r < a.N; r += 1024) {
    const int64_t i = base + r + threadIdx.x;
    const int64_t t = i < a.N ? a.targets[i] : a.ignore;
    const bool keep = t != a.ignore;
    const unsigned m = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) wsum[warp] = __popc(m);
    __syncthreads();
    int mine = at, all = 0;
    for (int k = 0; k < 32; ++k) {
      if (k < warp) mine += wsum[k];
      all += wsum[k];
    }
    if (keep) {
      mine += __popc(m & ((1u << lane) - 1u));
      w.rows[mine] = (int)i;
      w.target[mine] = t >= 0 && t < a.V ? (int)t : kBadTarget;
      w.inv[i] = mine;
    } else if (i < a.N) {
      w.inv[i] = -1;
      if (a.loss) a.loss[i] = a.logZ[i] = 0.f;
    }
    at += all;
  }
  if (blockIdx.x == gridDim.x - 1) {
    for (int64_t i = at + threadIdx.x; i < w.Np; i += 1024) {
      w.rows[i] = -1;
      w.target[i] = -1;
    }
    if (threadIdx.x == 0) w.hdr->live = at;
  }
}

// Largest finite magnitude of the listed rows (of every row without a list); a
// warp takes four rows at a time, 16 bytes a lane where the layout allows (vec).
__global__ void __launch_bounds__(256)
amax_kernel(const float* __restrict__ A, int64_t s0, int64_t s1, int D, int64_t n,
            const int* __restrict__ rows, const int* __restrict__ live, int vec,
            int* __restrict__ amax) {
  if (live) n = *live;
  const int lane = threadIdx.x & 31;
  float m = 0.f;
  auto see = [&](float x) {
    x = fabsf(x);
    if (x < INFINITY) m = fmaxf(m, x);
  };
  for (int64_t i0 = (blockIdx.x * 8ll + (threadIdx.x >> 5)) * 4; i0 < n; i0 += gridDim.x * 32ll) {
    const float* row[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = min(i0 + u, n - 1);
      row[u] = A + (rows ? rows[i] : i) * s0;
    }
    if (vec) {
      for (int d = lane * 4; d < D; d += 128) {
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const float4*>(row[u] + d);
#pragma unroll
        for (int u = 0; u < 4; ++u) { see(x[u].x); see(x[u].y); see(x[u].z); see(x[u].w); }
      }
    } else {
      for (int d = lane; d < D; d += 32) {
#pragma unroll
        for (int u = 0; u < 4; ++u) see(row[u][d * s1]);
      }
    }
  }
  m = redux_max(m);
  if (lane == 0 && m > 0.f) atomicMax(amax, __float_as_int(m));
}

// Dense copies of X's live rows (rows != null; zero rows up to a multiple of
// kPairRows) or of W, D padded with zeros to Dp; fp32 becomes two fp16 words of
// the value / 2^e.  8 elements a thread, `lanes` threads (a power of two) a row.
template <class T>
__global__ void __launch_bounds__(256)
pack_kernel(const T* __restrict__ A, int64_t s0, int64_t s1, int D, int Dp, int64_t n,
            const int* __restrict__ rows, const int* __restrict__ live, int vec, int lanes,
            const int* __restrict__ amax, uint16_t* __restrict__ out, uint16_t* __restrict__ out2) {
  constexpr bool kSplit = sizeof(T) == 4;
  if (live) n = ((int64_t)*live + kPairRows - 1) / kPairRows * kPairRows;
  const int per_row = Dp / 8, per_block = 256 / lanes;
  const float scale = kSplit ? ldexpf(1.f, -Scales::exponent(*amax, 14)) : 1.f;
  for (int64_t i = blockIdx.x * (int64_t)per_block + threadIdx.x / lanes; i < n;
       i += gridDim.x * (int64_t)per_block) {
    const int64_t r = rows ? rows[i] : i;
    for (int c = threadIdx.x % lanes; c < per_row; c += lanes) {
    const int64_t e = i * per_row + c;
    const int d0 = c * 8;
    uint4 w = make_uint4(0u, 0u, 0u, 0u), w2 = w;
    if (r >= 0) {
      const T* src = A + r * s0 + (int64_t)d0 * s1;
      if (!kSplit && vec && d0 + 8 <= D) {
        w = *reinterpret_cast<const uint4*>(src);
      } else {
        T v[8];
        if (kSplit && vec && d0 + 8 <= D) {
          reinterpret_cast<uint4*>(v)[0] = reinterpret_cast<const uint4*>(src)[0];
          reinterpret_cast<uint4*>(v)[kSplit ? 1 : 0] = reinterpret_cast<const uint4*>(src)[kSplit ? 1 : 0];
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = d0 + k < D ? src[k * s1] : from_f32<T>(0.f);
        }
        uint32_t h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (kSplit) split2(to_f32(v[2 * k]) * scale, to_f32(v[2 * k + 1]) * scale, h[k], l[k]);
          else h[k] = pack2<T>(to_f32(v[2 * k]), to_f32(v[2 * k + 1]));
        }
        w = make_uint4(h[0], h[1], h[2], h[3]);
        if (kSplit) w2 = make_uint4(l[0], l[1], l[2], l[3]);
      }
    }
    reinterpret_cast<uint4*>(out)[e] = w;
    if (kSplit) reinterpret_cast<uint4*>(out2)[e] = w2;
    }
  }
}

__global__ void pad_bias_kernel(const float* __restrict__ bias, int V, int64_t Vp,
                                float* __restrict__ out) {
  for (int64_t v = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; v < Vp;
       v += (int64_t)gridDim.x * blockDim.x)
    out[v] = v < V ? bias[v] : -INFINITY;
}

__global__ void row_grad_kernel(const XentArgs a, const XentWs w) {
  const int64_t n = ((int64_t)w.hdr->live + kPairRows - 1) / kPairRows * kPairRows;
  const float inv = a.count_in ? 1.f / *a.count_in : 1.f;
  float top = 0.f;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    RowGrad r{0.f, 0.f, 0.f, -1};
    const int n0 = w.rows[i];
    if (n0 >= 0) {
      r.b = a.dloss ? a.dloss[n0 * a.dloss_stride] * inv : 0.f;
      r.a = r.b + (a.dlogZ ? a.dlogZ[n0] : 0.f);
      const float x = fabsf(r.a), y = fabsf(r.b);
      if (x < INFINITY) top = fmaxf(top, x);
      if (y < INFINITY) top = fmaxf(top, y);
      r.lse = a.logZ_in[n0];
      r.target = w.target[i];
      if (r.target < 0) r.a = __int_as_float(0x7fffffff);   // a label outside the table: NaN
    }
    w.rg[i] = r;
  }
  top = redux_max(top);
  if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(&w.hdr->amax[0], __float_as_int(top));
}

// Joins a live row's parts (max, sum) into logZ and loss.  A block takes 32
// rows (lane = row), its 8 warps the parts in turn; the last block to finish
// adds the blocks' loss sums in order.
__global__ void __launch_bounds__(256) finish_forward_kernel(const XentArgs a, const XentWs w) {
  __shared__ float sm[8][32], ss[8][32];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = blockIdx.x * 32ll + lane;
  const int live = w.hdr->live;
  const bool on = i < live;
  float m = -3.402823466e38f, s = 0.f;
  if (on)
#pragma unroll 8
    for (int k = warp; k < 2 * w.splits; k += 8) {
      const float2 p = __ldg(&w.part[(int64_t)k * w.Np + i]);
      const float mn = fmaxf(m, p.x);
      s = s * ex2((m - mn) * kLog2Ef) + p.y * ex2((p.x - mn) * kLog2Ef);
      m = mn;
    }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  if (warp == 0) {
    float top = sm[0][lane];
    for (int k = 1; k < 8; ++k) top = fmaxf(top, sm[k][lane]);
    float sum = 0.f;
    for (int k = 0; k < 8; ++k) sum += ss[k][lane] * ex2((sm[k][lane] - top) * kLog2Ef);
    double mine = 0.0;
    if (on) {
      const int r = w.rows[i];
      float lz = top + logf(sum);
      const float nan = __int_as_float(0x7fffffff);
      if (w.hdr->err) lz = nan;
      const float loss = w.target[i] < 0 ? nan : lz - w.tlogit[i];
      a.logZ[r] = lz;
      a.loss[r] = loss;
      mine = loss;
    }
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0 && a.reduction != FGMM_REDUCE_NONE) {
      w.loss_part[blockIdx.x] = mine;
      __threadfence();
      last = atomicAdd(&w.hdr->done, 1) == (int)gridDim.x - 1;
    }
  }
  if (a.reduction == FGMM_REDUCE_NONE) return;
  __syncthreads();
  if (!last) return;
  __threadfence();
  __shared__ double red[256];
  double s64 = 0.0;
  for (int k = threadIdx.x; k < (int)gridDim.x; k += 256) s64 += __ldcg(&w.loss_part[k]);
  red[threadIdx.x] = s64;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *a.count = (float)live;
    *a.reduced = (float)(a.reduction == FGMM_REDUCE_MEAN ? red[0] / live : red[0]);
  }
}

// out[r, :] = scale * sum of the slots' rows, in slot order; rows of dX without
// a live row are zero.  If a wait gave up, every gradient becomes NaN instead.
template <class T>
__global__ void __launch_bounds__(256)
store_slots_kernel(const float* __restrict__ slots, int ks, int64_t slot_rows, int64_t ldS, int D,
                   int64_t n, const int* __restrict__ inv, const Header* __restrict__ hdr,
                   int is_dw, int split, T* __restrict__ out) {
  const int per_row = (D + 3) / 4;
  const Scales sc(hdr->amax, !std::is_same<T, __nv_bfloat16>::value, split);
  const float scale = is_dw ? sc.dw : sc.dx;
  const bool vec = D % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0;
  const bool bad = hdr->err != 0;
  const int64_t total = n * per_row;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < total; e += gridDim.x * 256ll) {
    const int64_t r = e / per_row;
    const int d0 = (int)(e - r * per_row) * 4;
    const int64_t i = inv ? inv[r] : r;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i >= 0) {
      for (int k = 0; k < ks; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(slots + (k * slot_rows + i) * ldS + d0);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      s.x *= scale; s.y *= scale; s.z *= scale; s.w *= scale;
    }
    if (bad) s.x = s.y = s.z = s.w = __int_as_float(0x7fffffff);
    T* dst = out + r * D + d0;
    if (vec) {
      T v[4] = {from_f32<T>(s.x), from_f32<T>(s.y), from_f32<T>(s.z), from_f32<T>(s.w)};
      if (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(v);
      else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(v);
    } else {
      const float f[4] = {s.x, s.y, s.z, s.w};
      for (int k = 0; k < 4; ++k)
        if (d0 + k < D) dst[k] = from_f32<T>(f[k]);
    }
  }
}

// dbias from the 128-row partial sums (NaN if a wait gave up): 32 entries a block,
// 32 warps that take the parts in turn, joined in warp order.
__global__ void __launch_bounds__(1024) store_dbias_kernel(const XentArgs a, const XentWs w) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nparts = (int)(((int64_t)w.hdr->live + kPairRows - 1) / kPairRows) * 2;
  const int64_t v = blockIdx.x * 32ll + lane;      // < Vp
  float s = 0.f;
#pragma unroll 4
  for (int k = warp; k < nparts; k += 32) s += w.dbias_part[(int64_t)k * w.Vp + v];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && v < a.V) {
    s = red[0][lane];
    for (int k = 1; k < 32; ++k) s += red[k][lane];
    const float back = 1.f / Scales(w.hdr->amax, a.type != FGMM_T_BF16, a.type == FGMM_T_F32).g;
    a.dbias[v] = w.hdr->err ? __int_as_float(0x7fffffff) : s * back;
  }
}

// After the last product: dW that was written directly becomes NaN if a wait gave up.
template <class T>
__global__ void poison_kernel(const Header* __restrict__ hdr, T* __restrict__ out, int64_t n) {
  if (hdr->err == 0) return;
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * blockDim.x)
    out[e] = from_f32<T>(__int_as_float(0x7fffffff));
}

int grid_for(int64_t threads) {
  return (int)std::min<int64_t>(std::max<int64_t>((threads + 255) / 256, 1), 16 * num_sms());
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encode_fn(EncodeTiled* out) {
  static std::atomic<void*> cached{nullptr};
  void* f = cached.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000,
                                                     cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (!f || found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    cached.store(f, std::memory_order_release);
  }
  *out = reinterpret_cast<EncodeTiled>(f);
  return cudaSuccess;
}

// 64 x 64 boxes of a row-major (rows, cols) matrix of 16-bit words, 128-byte
// swizzle; elements outside read as zero.
cudaError_t make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld,
                     bool bf16) {
  EncodeTiled encode;
  cudaError_t e = encode_fn(&encode);
  if (e != cudaSuccess) return e;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)std::max<int64_t>(rows, 1)};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, 64}, es[2] = {1, 1};
  const CUresult r = encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            2, const_cast<void*>(base), dims, strides, box, es,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Operand word of each element type, and what dW is stored as.
template <class T> struct Word { using type = T; };
template <> struct Word<float> { using type = __half; };

template <class T>
cudaError_t prepare_operands(const XentArgs& a, const XentWs& w, MmaMaps* maps) {
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value;
  cudaError_t e = cudaMemsetAsync(w.hdr, 0, sizeof(Header), a.stream);
  if (e != cudaSuccess) return e;
  rows_kernel<<<(unsigned)((a.N + kRowsPerBlock - 1) / kRowsPerBlock), 1024, 0, a.stream>>>(a, w);
  const T* X = static_cast<const T*>(a.X);
  const T* W = static_cast<const T*>(a.W);
  const int* live = &w.hdr->live;
  auto vec = [&](const void* p, int64_t s0, int64_t s1, int whole) {
    return s1 == 1 && s0 * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
           a.D % whole == 0;
  };
  if (kSplit) {
    auto blocks = [&](int64_t n) { return (int)std::min<int64_t>((n + 31) / 32, 8 * num_sms()); };
    amax_kernel<<<blocks(a.N), 256, 0, a.stream>>>(
        reinterpret_cast<const float*>(X), a.sxn, a.sxd, a.D, a.N, w.rows, live,
        vec(X, a.sxn, a.sxd, 4), &w.hdr->amax[1]);
    amax_kernel<<<blocks(a.V), 256, 0, a.stream>>>(
        reinterpret_cast<const float*>(W), a.swv, a.swd, a.D, a.V, nullptr, nullptr,
        vec(W, a.swv, a.swd, 4), &w.hdr->amax[2]);
    count_launches(2);
  }
  int lanes = 1;
  while (lanes < 256 && lanes < w.Dp / 8) lanes *= 2;
  pack_kernel<T><<<grid_for(w.Np * lanes), 256, 0, a.stream>>>(
      X, a.sxn, a.sxd, a.D, w.Dp, 0, w.rows, live, vec(X, a.sxn, a.sxd, 1), lanes, &w.hdr->amax[1],
      static_cast<uint16_t*>(w.Xp), static_cast<uint16_t*>(w.Xp2));
  count_launches(2);
  if (w.pack_w) {
    pack_kernel<T><<<grid_for((int64_t)a.V * lanes), 256, 0, a.stream>>>(
        W, a.swv, a.swd, a.D, w.Dp, a.V, nullptr, nullptr, vec(W, a.swv, a.swd, 1), lanes,
        &w.hdr->amax[2], static_cast<uint16_t*>(w.Wp), static_cast<uint16_t*>(w.Wp2));
    count_launches(1);
  }
  if (a.bias) {
    pad_bias_kernel<<<grid_for(w.Vp), 256, 0, a.stream>>>(a.bias, a.V, w.Vp, w.bias);
    count_launches(1);
  }
  e = make_map(&maps->X, w.Xp, w.Np, a.D, w.Dp, kBf);
  if (e == cudaSuccess)
    e = w.pack_w ? make_map(&maps->W, w.Wp, a.V, a.D, w.Dp, kBf)
                 : make_map(&maps->W, a.W, a.V, a.D, a.swv, kBf);
  if (kSplit && e == cudaSuccess) e = make_map(&maps->X2, w.Xp2, w.Np, a.D, w.Dp, kBf);
  if (kSplit && e == cudaSuccess) e = make_map(&maps->W2, w.Wp2, a.V, a.D, w.Dp, kBf);
  return e;
}

MmaParams common_params(const XentArgs& a, const XentWs& w) {
  MmaParams p{};
  p.live = &w.hdr->live;
  p.err = &w.hdr->err;
  p.amax = w.hdr->amax;
  p.N = a.N;
  p.D = a.D;
  p.V = a.V;
  p.kbD = (a.D + 63) / 64;
  p.Np = w.Np;
  p.Vp = w.Vp;
  p.bias = a.bias ? w.bias : nullptr;
  return p;
}

template <bool FWD, class T>
cudaError_t launch_mma(const XentArgs& a, const MmaParams& p, const MmaMaps& maps, int64_t units) {
  constexpr bool kSplit = sizeof(T) == 4;
  auto* kernel = xent_mma_kernel<FWD, kSplit, typename Word<T>::type, T>;
  constexpr size_t smem = MmaCfg<kSplit>::kSmem;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const int pairs = (int)std::min<int64_t>(units, num_sms() / 2);
  kernel<<<2 * pairs, kMmaThreads, smem, a.stream>>>(p, maps);
  count_launches(1);
  return cudaGetLastError();
}

template <class T>
cudaError_t xent_forward(const XentArgs& a, const XentWs& w) {
  MmaMaps maps{};
  cudaError_t e = prepare_operands<T>(a, w, &maps);
  if (e != cudaSuccess) return e;
  MmaParams p = common_params(a, w);
  p.vtiles = w.vtiles;
  p.per_split = w.per_split;
  p.splits = w.splits;
  p.part = w.part;
  p.tlogit = w.tlogit;
  p.target = w.target;
  e = launch_mma<true, T>(a, p, maps, w.Np / kPairRows * w.splits);
  if (e != cudaSuccess) return e;
  finish_forward_kernel<<<(unsigned)((a.N + 31) / 32), 256, 0, a.stream>>>(a, w);
  count_launches(1);
  return cudaSuccess;
}

template <class T>
cudaError_t xent_backward(const XentArgs& a, const XentWs& w) {
  constexpr bool kSplit = sizeof(T) == 4;
  MmaMaps maps{};
  cudaError_t e = prepare_operands<T>(a, w, &maps);
  if (e != cudaSuccess) return e;
  row_grad_kernel<<<grid_for(w.Np), 256, 0, a.stream>>>(a, w);
  count_launches(1);
  CUtensorMap gmap[2], gmap2[2];
  for (int b = 0; b < 2 && e == cudaSuccess; ++b) {
    e = make_map(&gmap[b], w.G[b], w.row_chunk, w.piece, w.piece, std::is_same<T, __nv_bfloat16>::value);
    if (kSplit && e == cudaSuccess) e = make_map(&gmap2[b], w.G2[b], w.row_chunk, w.piece, w.piece, false);
  }
  if (e != cudaSuccess) return e;
  MmaParams p = common_params(a, w);
  p.bn_d = w.bn_d;
  p.tiles_d = w.tiles_d;
  p.rg = w.rg;
  p.ldG = w.piece;
  p.dbias_part = a.dbias ? w.dbias_part : nullptr;
  p.ks_x = w.ks_x;
  p.ks_w = w.ks_w;
  p.dx_slots = w.dx_slots;
  p.dw_slots = w.dw_direct ? nullptr : w.dw_slots;
  p.ldS = w.ldS;
  p.dw_rows = w.piece;
  p.dW = a.dW;
  p.dw_vec = a.D % 8 == 0 && sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(a.dW) & 15) == 0;
  // The vocabulary's pieces, each over the row chunks: launch j makes piece j's g
  // while it multiplies piece j - 1's.
  const int total = w.n_pieces * w.n_chunks;
  auto piece_at = [&](int j) {
    const int vp = j / w.n_chunks, rc = j % w.n_chunks;
    Piece q;
    q.r0 = (int64_t)rc * w.row_chunk;
    q.rows = (int)std::min<int64_t>(w.row_chunk, w.Np - q.r0);
    q.v0 = (int)((int64_t)vp * w.piece);
    q.nv = std::min(w.piece, a.V - q.v0);
    return q;
  };
  for (int j = 0; j <= total; ++j) {
    p.has_grad = j < total;
    p.has_dx = j > 0 && a.dX != nullptr;
    p.has_dw = j > 0 && a.dW != nullptr;
    if (!p.has_grad && !p.has_dx && !p.has_dw) break;
    p.cur = piece_at(std::min(j, total - 1));
    p.prev = piece_at(std::max(j - 1, 0));
    p.dx_add = j - 1 >= w.n_chunks;
    p.dw_add = p.prev.r0 > 0;
    p.G = w.G[j & 1];
    p.G2 = w.G2[j & 1];
    maps.G = gmap[(j & 1) ^ 1];
    maps.G2 = gmap2[(j & 1) ^ 1];
    const int64_t units =
        (p.has_grad ? (int64_t)(p.cur.rows / 256) * ((p.cur.nv + kBN - 1) / kBN) : 0) +
        (p.has_dx ? (int64_t)(p.prev.rows / 256) * w.tiles_d * w.ks_x : 0) +
        (p.has_dw ? (int64_t)((p.prev.nv + 255) / 256) * w.tiles_d * w.ks_w : 0);
    e = launch_mma<false, T>(a, p, maps, units);
    if (e != cudaSuccess) return e;
    if (p.has_dw && !w.dw_direct && j % w.n_chunks == 0) {   // the piece's last row chunk
      store_slots_kernel<T><<<grid_for((int64_t)p.prev.nv * ((a.D + 3) / 4)), 256, 0, a.stream>>>(
          w.dw_slots, w.ks_w, w.piece, w.ldS, a.D, p.prev.nv, nullptr, w.hdr, 1, kSplit,
          static_cast<T*>(a.dW) + (int64_t)p.prev.v0 * a.D);
      count_launches(1);
    }
  }
  if (a.dX) {
    store_slots_kernel<T><<<grid_for(a.N * ((a.D + 3) / 4)), 256, 0, a.stream>>>(
        w.dx_slots, w.ks_x, w.Np, w.ldS, a.D, a.N, w.inv, w.hdr, 0, kSplit, static_cast<T*>(a.dX));
    count_launches(1);
  }
  if (a.dbias) {
    store_dbias_kernel<<<(unsigned)((a.V + 31) / 32), 1024, 0, a.stream>>>(a, w);
    count_launches(1);
  }
  if (a.dW) {
    poison_kernel<T><<<num_sms(), 256, 0, a.stream>>>(w.hdr, static_cast<T*>(a.dW), (int64_t)a.V * a.D);
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

size_t fgmm_xent_workspace_bytes(int backward, int type, int64_t N, int32_t V, int32_t D,
                                 const void* W, int64_t w_stride_v, int64_t w_stride_d,
                                 int has_bias) {
  using namespace fgmm;
  if (type < 0 || type > 2 || N < 0 || V < 1 || D < 1 || N >= kVocabMaxN || V >= kVocabMaxV ||
      D > kVocabMaxD)
    return 0;
  return XentWs(nullptr, backward != 0, type, N, V, D, W, w_stride_v, w_stride_d, has_bias != 0).bytes;
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
    const XentWs w(workspace, false, type, N, V, D, W, w_stride_v, w_stride_d, bias != nullptr);
    rc = check_device_and_workspace(a, w.bytes);
    if (rc != FGMM_OK) return rc;
    if (N == 0) {
      if (reduction != FGMM_REDUCE_NONE) {
        empty_reduction_kernel<<<1, 1, 0, a.stream>>>(reduction == FGMM_REDUCE_MEAN, reduced, count);
        count_launches(1);
      }
      return finish(a, cudaSuccess);
    }
    return finish(a, with_type(type, [&](auto* tag) {
      return xent_forward<std::remove_pointer_t<decltype(tag)>>(a, w);
    }));
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
    const XentWs w(workspace, true, type, N, V, D, W, w_stride_v, w_stride_d, bias != nullptr);
    rc = check_device_and_workspace(a, w.bytes);
    if (rc != FGMM_OK) return rc;
    cudaError_t e = cudaSuccess;
    if (N == 0) {
      if (dW) e = cudaMemsetAsync(dW, 0, (size_t)V * D * type_size(type), a.stream);
      if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, (size_t)V * 4, a.stream);
      return finish(a, e);
    }
    return finish(a, with_type(type, [&](auto* tag) {
      return xent_backward<std::remove_pointer_t<decltype(tag)>>(a, w);
    }));
  });
}

}  // extern "C"
