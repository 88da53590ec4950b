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
// computed again in pieces; a piece's g goes to a small ring of buffers and is
// multiplied with W and X, partly still in the L2, while the next pieces' are made.
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

// First words of the workspace.  Every word is written before it is read: err and
// done by the tensor-core kernel, the others by rows_kernel.
struct Header {
  int err[kErrSlots];   // nonzero: a wait of that block of the tensor-core kernel gave up
  int done;             // blocks of the closing forward kernel that have finished
  int live;             // rows that are not ignored
  int amax;             // backward: float bits of the largest finite |weight|
};

constexpr int kRowsPerBlock = 4096;
constexpr int kBadTarget = -2;

// The launches of fgmm_xent_small.cuh.
constexpr int kSmallRows = 16;             // rows at most
constexpr int kSmallCols = 512;            // columns of a products block: 128 threads x 4
struct SmallPlan {
  int nb;            // rows the kernels are made for: 1, 8 or 16
  int blocks;        // of small_logits_kernel; its parts
  int splits;        // ranges of the vocabulary of the products
  int per_split;     // entries of one
};

SmallPlan small_plan(int64_t N, int V, int D) {
  SmallPlan p;
  p.nb = N <= 1 ? 1 : N <= 8 ? 8 : 16;
  const int rows = p.nb == 16 ? 2 : p.nb == 8 ? 4 : 8;       // of W, per warp
  p.blocks = (int)std::min<int64_t>(((int64_t)V + 8 * rows - 1) / (8 * rows), 4 * 148);
  const int64_t tiles = (D + kSmallCols - 1) / kSmallCols;
  const int64_t want = std::max<int64_t>(1, (6 * 148 + tiles - 1) / tiles);
  p.per_split = (int)std::max<int64_t>(64, (V + want - 1) / want);
  p.splits = (V + p.per_split - 1) / p.per_split;
  return p;
}

struct XentWs {
  Header* hdr;
  int *rows, *inv, *target, *counts;
  float* bias;
  void *Xp[3], *Wp[3];             // packed operands (fp32: hi, mid and lo words)
  float2* part;
  float* tlogit;
  double* loss_part;               // [blocks][2] sum, count
  RowGrad* rg;
  uint32_t* sync;
  void* G[3];
  float *dbias_part, *dx_slots, *dw_slots;
  float *small_g, *small_dx;       // of a few rows: g [V][nb], parts of dX [splits][nb][D]

  int64_t Np, Vp;
  int Dp;                          // row length of the packed operands
  bool split, pack_w, small;
  int vtiles, per_split, splits;
  int bn_d, tiles_d;
  int64_t ldS;
  int row_chunk, piece, n_chunks, n_pieces, ks_x, ks_w, parts;
  int64_t sync_words, units = 0;
  size_t bytes;

  static constexpr int kPairs = 74;                        // SM pairs the plan is made for
  static constexpr int64_t kPieceBytes = int64_t(1) << 25; // one buffer of G, of kRing
  static constexpr int kPiecesWanted = 4;   // of a short batch: products begin while g is made
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
    // fp32 rows of W that do not take 16-byte loads: forward 8 rows at most (12 of 5000 x 4095:
    // 291 us against 169 as words on the tensor cores; of 100000 x 999 393 and 405), with
    // gradients all 16 (12 of 100000 x 999: 735 against 995, of 5000 x 4095 267 and 309).
    const bool w16 = swd == 1 && swv % 4 == 0 && D % 4 == 0 && (reinterpret_cast<uintptr_t>(W) & 15) == 0;
    // One 16-bit row whose W would be copied for TMA: 131072 x 4095 bf16 674 -> 288 us, with
    // gradients 3181 -> 1337, W transposed (100000 x 1000) 655 -> 253; four rows 676 -> 803.
    small = split ? N <= (w16 || backward ? kSmallRows : 8) : pack_w && N <= 1;
    if (small) {
      const SmallPlan sp = small_plan(N, V, D);
      if (!backward) {
        part = c.take<float2>((size_t)sp.blocks * Np);
        tlogit = c.take<float>(Np);
        loss_part = c.take<double>(2);
      } else {
        small_g = c.take<float>((size_t)V * sp.nb);
        small_dx = c.take<float>((size_t)sp.splits * sp.nb * D);
      }
      bytes = c.used;
      return;
    }
    rows = c.take<int>(Np);
    inv = c.take<int>(Np);
    target = c.take<int>(Np);
    counts = c.take<int>((N + kRowsPerBlock - 1) / kRowsPerBlock);
    bias = c.take<float>(want_bias ? Vp : 0);
    const int words = split ? 3 : 1;
    for (int h = 0; h < 3; ++h) {
      Xp[h] = c.take<uint16_t>(h < words ? (size_t)Np * Dp : 0);
      Wp[h] = c.take<uint16_t>(h < words && pack_w ? (size_t)V * Dp : 0);
    }
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
      loss_part = c.take<double>(2 * ((N + 31) / 32));
    } else {
      const int word = 2 * words;
      // column tiles of dX and dW: a 128-wide block takes about 0.7 of a 256-wide one's time
      bn_d = D <= 128 ? 128 : 256;
      tiles_d = (D + bn_d - 1) / bn_d;
      ldS = (int64_t)tiles_d * bn_d;
      // Pieces of G: wide ones, so that dX's slots are added to rarely, and all rows of a
      // short batch.
      piece = (int)std::min<int64_t>(Vp, 4096);
      row_chunk = (int)std::max<int64_t>(
          256, std::min<int64_t>(Np, kPieceBytes / ((int64_t)piece * word) / 256 * 256));
      if (row_chunk == Np)
        piece = (int)std::max<int64_t>(
            piece, std::min<int64_t>((Vp / kPiecesWanted + 255) / 256 * 256,
                                     kPieceBytes / ((int64_t)row_chunk * word) / 256 * 256));
      n_chunks = (int)((Np + row_chunk - 1) / row_chunk);
      n_pieces = (int)((Vp + piece - 1) / piece);
      // Splits of K: products of at most `unit` blocks, shorter where a product's tiles
      // could not occupy the pairs twice; dW's only where its slots hold all of V.  fp32
      // blocks take six times the MMAs: 131072 x 1024 x 128 816 us with 12, 955 with 16,
      // 984 with 24; 2048 x 16384 x 512 595, 607 and 659.
      const int64_t unit = split ? 12 : 64;
      auto pick = [&](int64_t tiles, int64_t kb, int64_t slot_bytes) {
        int64_t ks = std::max<int64_t>((kb + unit - 1) / unit, (2 * kPairs + tiles - 1) / tiles);
        ks = std::min(ks, std::max<int64_t>(1, kb / 8));
        return (int)std::max<int64_t>(1, std::min(ks, kSlotBytes / std::max<int64_t>(slot_bytes, 1)));
      };
      const int64_t steps = (int64_t)n_chunks * n_pieces;
      ks_x = pick((int64_t)(row_chunk / 256) * tiles_d * steps, piece / 64, Np * ldS * 4);
      ks_w = n_pieces > 1 ? 1 : pick((int64_t)(piece / 256) * tiles_d * steps, row_chunk / 64,
                                     (int64_t)piece * ldS * 4);
      // tiles of all kinds, which the product kernel counts in 32 bits
      units = Np / 256 * (Vp / 256) + steps * tiles_d *
              ((int64_t)(row_chunk / 256) * ks_x + (int64_t)(piece / 256) * ks_w);
      rg = c.take<RowGrad>(Np);
      sync_words = 1 + 2 * steps + (Np / kPairRows * ks_x + (int64_t)(piece / 256) * ks_w) * tiles_d;
      sync = c.take<uint32_t>(sync_words);
      for (int h = 0; h < 3; ++h)
        G[h] = c.take<uint16_t>(h < words ? (size_t)kRing * row_chunk * piece : 0);
      // one part per 128 rows of the first kRing chunks, to which the later ones add
      parts = (int)std::min<int64_t>(n_chunks, kRing) * (row_chunk / 128);
      dbias_part = c.take<float>(want_bias ? (size_t)parts * Vp : 0);
      dx_slots = c.take<float>((size_t)ks_x * Np * ldS);
      dw_slots = c.take<float>(n_chunks == 1 && ks_w == 1 ? 0 : (size_t)ks_w * piece * ldS);
    }
    bytes = c.used;
  }
};

#include "fgmm_xent_small.cuh"

// Live rows among each 4096 labels, for long batches (rows_kernel).
__global__ void __launch_bounds__(1024) count_kernel(const XentArgs a, const XentWs w) {
  pdl_trigger();
  __shared__ int wsum[32];
  const int64_t base = (int64_t)blockIdx.x * kRowsPerBlock;
  int n = 0;
#pragma unroll
  for (int r = 0; r < kRowsPerBlock; r += 1024) {
    const int64_t i = base + r + threadIdx.x;
    n += i < a.N && a.targets[i] != a.ignore;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, wsum[threadIdx.x]);
    if (threadIdx.x == 0) w.counts[blockIdx.x] = n;
  }
}

// Lists the live rows in their order, with their targets.  Block b needs the live
// rows before its own 4096: from count_kernel's sums where that ran (`counted`), else
// it reads all earlier labels.  Ignored rows get loss = logZ = 0.
// The last block pads the list to a multiple of kPairRows with -1.
__global__ void __launch_bounds__(1024)
rows_kernel(const XentArgs a, const XentWs w, int counted) {
  pdl_trigger();
  pdl_wait();
  __shared__ int wsum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = (int64_t)blockIdx.x * kRowsPerBlock;
  if (blockIdx.x == 0 && threadIdx.x == 0) w.hdr->amax = 0;
  if (a.logZ_in)   // backward: the product kernel's counts
    for (int64_t i = blockIdx.x * 1024 + threadIdx.x; i < w.sync_words; i += gridDim.x * 1024)
      w.sync[i] = 0;
  int before = 0;
  if (counted) {
    for (int k = threadIdx.x; k < (int)blockIdx.x; k += 1024) before += w.counts[k];
  } else {
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < base; i += 1024) before += a.targets[i] != a.ignore;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) wsum[warp] = before;
  __syncthreads();
  int at = __reduce_add_sync(0xffffffffu, wsum[lane]);
  for (int r = 0; r < kRowsPerBlock && base + r < a.N; r += 1024) {
    const int64_t i = base + r + threadIdx.x;
    const int64_t t = i < a.N ? a.targets[i] : a.ignore;
    const bool keep = t != a.ignore;
    const unsigned m = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) wsum[warp] = __popc(m);
    __syncthreads();
    const int c = wsum[lane];
    const int all = __reduce_add_sync(0xffffffffu, c);
    int mine = at + __reduce_add_sync(0xffffffffu, lane < warp ? c : 0);
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

// A share of a launch: its block number and how many blocks work on it.
struct Share {
  int block, blocks;
};

// Dense copies of X's live rows (rows != null; zero rows up to a multiple of
// kPairRows) or of W, D padded with zeros to Dp; fp32 becomes three bf16 words.
// 8 elements a thread, `lanes` threads (a power of two) a row.
template <class T>
__device__ __forceinline__ void pack_rows(const Share sh, const T* __restrict__ A, int64_t s0,
                                          int64_t s1, int D, int Dp, int64_t n,
                                          const int* __restrict__ rows, int vec, int lanes,
                                          void* const (&out)[3]) {
  constexpr bool kSplit = sizeof(T) == 4;
  const int per_row = Dp / 8, per_block = 256 / lanes;
  for (int64_t i = sh.block * (int64_t)per_block + threadIdx.x / lanes; i < n;
       i += sh.blocks * (int64_t)per_block) {
    const int64_t r = rows ? rows[i] : i;
    for (int c = threadIdx.x % lanes; c < per_row; c += lanes) {
      const int64_t e = i * per_row + c;
      const int d0 = c * 8;
      uint4 w[3];
      w[0] = w[1] = w[2] = make_uint4(0u, 0u, 0u, 0u);
      if (r >= 0) {
        const T* src = A + r * s0 + (int64_t)d0 * s1;
        if (!kSplit && vec && d0 + 8 <= D) {
          w[0] = *reinterpret_cast<const uint4*>(src);
        } else {
          T v[8];
          if (kSplit && vec && d0 + 8 <= D) {
            reinterpret_cast<uint4*>(v)[0] = reinterpret_cast<const uint4*>(src)[0];
            reinterpret_cast<uint4*>(v)[kSplit ? 1 : 0] = reinterpret_cast<const uint4*>(src)[kSplit ? 1 : 0];
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = d0 + k < D ? src[k * s1] : from_f32<T>(0.f);
          }
          uint32_t u[4][3];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (kSplit) split3(to_f32(v[2 * k]), to_f32(v[2 * k + 1]), u[k]);
            else u[k][0] = pack2<T>(to_f32(v[2 * k]), to_f32(v[2 * k + 1]));
          }
#pragma unroll
          for (int h = 0; h < (kSplit ? 3 : 1); ++h)
            w[h] = make_uint4(u[0][h], u[1][h], u[2][h], u[3][h]);
        }
      }
#pragma unroll
      for (int h = 0; h < (kSplit ? 3 : 1); ++h) static_cast<uint4*>(out[h])[e] = w[h];
    }
  }
}

// What the backward pass knows of the (padded) live rows, and the largest weight.
__device__ __forceinline__ void row_weights(const Share sh, const XentArgs& a, const XentWs& w) {
  const int64_t n = ((int64_t)w.hdr->live + kPairRows - 1) / kPairRows * kPairRows;
  const float inv = a.count_in ? 1.f / *a.count_in : 1.f;
  float top = 0.f;
  for (int64_t i = sh.block * 256ll + threadIdx.x; i < n; i += sh.blocks * 256ll) {
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
  if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(&w.hdr->amax, __float_as_int(top));
}

// Blocks of prepare_kernel by what they do, in this order.
struct PrepareShares {
  int x, w, bias, rows;
  int vec_x, vec_w, lanes;
};

// Everything the products need, in one launch: the packed rows of X, W where it
// cannot be read in place, the bias padded with -inf, and the rows' weights.
template <class T>
__global__ void __launch_bounds__(256)
prepare_kernel(const XentArgs a, const XentWs w, const PrepareShares sh) {
  pdl_trigger();
  pdl_wait();
  int b = blockIdx.x;
  if (b < sh.x) {
    const int64_t n = ((int64_t)w.hdr->live + kPairRows - 1) / kPairRows * kPairRows;
    pack_rows<T>(Share{b, sh.x}, static_cast<const T*>(a.X), a.sxn, a.sxd, a.D, w.Dp, n, w.rows,
                 sh.vec_x, sh.lanes, w.Xp);
    return;
  }
  b -= sh.x;
  if (b < sh.w) {
    pack_rows<T>(Share{b, sh.w}, static_cast<const T*>(a.W), a.swv, a.swd, a.D, w.Dp, a.V, nullptr,
                 sh.vec_w, sh.lanes, w.Wp);
    return;
  }
  b -= sh.w;
  if (b < sh.bias) {
    for (int64_t v = b * 256ll + threadIdx.x; v < w.Vp; v += sh.bias * 256ll)
      w.bias[v] = v < a.V ? a.bias[v] : -INFINITY;
    return;
  }
  row_weights(Share{b - sh.bias, sh.rows}, a, w);
}

// Whether a wait of the tensor-core kernel gave up (the same for all threads).
__device__ __forceinline__ bool any_error(const Header* hdr) {
  int e = 0;
  for (int i = threadIdx.x; i < kErrSlots; i += blockDim.x) e |= hdr->err[i];
  return __syncthreads_or(e) != 0;
}

// Joins a live row's parts (max, sum) into logZ and loss.  With many parts a block
// takes 32 rows (lane = row) and its 32 warps the parts in turn; with few (`few`)
// every thread takes a row.  The last block to finish adds the blocks' sums in order.
// `direct`: row i of X is live row i, ignored rows among them.
__global__ void __launch_bounds__(1024)
finish_forward_kernel(const XentArgs a, const XentWs w, int parts, int direct, int few) {
  pdl_trigger();
  pdl_wait();
  __shared__ float sm[32][33], ss[32][33];
  __shared__ double block_sum[32];
  __shared__ int block_count[32];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = few ? blockIdx.x * 1024ll + threadIdx.x : blockIdx.x * 32ll + lane;
  const int64_t live = direct ? a.N : w.hdr->live;
  const bool bad = any_error(w.hdr);
  const bool on = i < live;
  float m = -3.402823466e38f, s = 0.f;
  if (on)
#pragma unroll 4
    for (int k = few ? 0 : warp; k < parts; k += few ? 1 : 32) {
      const float2 p = __ldg(&w.part[(int64_t)k * w.Np + i]);
      const float mn = fmaxf(m, p.x);
      s = s * ex2((m - mn) * kLog2Ef) + p.y * ex2((p.x - mn) * kLog2Ef);
      m = mn;
    }
  if (!few) {
    sm[warp][lane] = m;
    ss[warp][lane] = s;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int k = 1; k < 32; ++k) m = fmaxf(m, sm[k][lane]);
      s = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) s += ss[k][lane] * ex2((sm[k][lane] - m) * kLog2Ef);
    }
  }
  if (few || warp == 0) {
    double mine = 0.0;
    bool counted = false;
    if (on) {
      const int64_t r = direct ? i : w.rows[i], t = a.targets[r];
      counted = t != a.ignore;
      float lz = 0.f, loss = 0.f;
      if (counted) {
        const float nan = __int_as_float(0x7fffffff);
        lz = bad ? nan : m + logf(s);
        loss = t < 0 || t >= a.V ? nan : lz - w.tlogit[i];
        mine = loss;
      }
      a.logZ[r] = lz;
      a.loss[r] = loss;
    }
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    const int n = __popc(__ballot_sync(0xffffffffu, counted));
    if (lane == 0) { block_sum[warp] = mine; block_count[warp] = n; }
  }
  if (a.reduction == FGMM_REDUCE_NONE) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    int n = 0;
    for (int k = 0; k < (few ? 32 : 1); ++k) { total += block_sum[k]; n += block_count[k]; }
    w.loss_part[2 * blockIdx.x] = total;
    w.loss_part[2 * blockIdx.x + 1] = n;
    __threadfence();
    last = atomicAdd(&w.hdr->done, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last || warp != 0) return;
  __threadfence();
  double total = 0.0, n = 0.0;
  for (int k = lane; k < (int)gridDim.x; k += 32) {
    total += __ldcg(&w.loss_part[2 * k]);
    n += __ldcg(&w.loss_part[2 * k + 1]);
  }
  for (int o = 16; o; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (lane == 0) {
    *a.count = (float)n;
    *a.reduced = (float)(a.reduction == FGMM_REDUCE_MEAN ? total / n : total);
  }
}

// out[r, :] = scale * sum of the ks slots' rows, in slot order; rows of dX without
// a live row (inv < 0) are zero.
template <class T>
__device__ __forceinline__ void store_slots(const Share sh, const float* __restrict__ slots, int ks,
                                            int64_t slot_rows, int64_t ldS, int D, int64_t n,
                                            const int* __restrict__ inv, float scale, int lanes,
                                            T* __restrict__ out) {
  const int per_row = (D + 3) / 4, per_block = (int)blockDim.x / lanes;
  const bool vec = D % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0;
  for (int64_t r = sh.block * (int64_t)per_block + threadIdx.x / lanes; r < n;
       r += sh.blocks * (int64_t)per_block) {
    const int64_t i = inv ? inv[r] : r;
    for (int c = threadIdx.x % lanes; c < per_row; c += lanes) {
      const int d0 = c * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i >= 0) {
#pragma unroll 4
        for (int k = 0; k < ks; ++k) {
          const float4 x = *reinterpret_cast<const float4*>(slots + (k * slot_rows + i) * ldS + d0);
          s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
        s.x *= scale; s.y *= scale; s.z *= scale; s.w *= scale;
      }
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
}

// dbias from the 128-row partial sums: 32 entries a block, whose 32 warps take
// the parts in turn and are joined in order.
__device__ __forceinline__ void store_dbias(int block, const XentArgs& a, const XentWs& w) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nparts = min((int)(((int64_t)w.hdr->live + kPairRows - 1) / kPairRows) * 2, w.parts);
  const int64_t v = block * 32ll + lane;      // < Vp
  float s = 0.f;
#pragma unroll 4
  for (int k = warp; k < nparts; k += 32) s += w.dbias_part[(int64_t)k * w.Vp + v];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && v < a.V) {
    s = red[0][lane];
#pragma unroll
    for (int k = 1; k < 32; ++k) s += red[k][lane];
    a.dbias[v] = s / Scales(&w.hdr->amax, a.type == FGMM_T_F16).g;
  }
}

template <class T>
__device__ __forceinline__ void fill_nan(T* out, int64_t n) {
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * blockDim.x)
    out[e] = from_f32<T>(__int_as_float(0x7fffffff));
}

// Blocks of finish_backward_kernel by what they do, in this order.
struct FinishShares {
  int dx, dw, dbias;
  int lanes;
};

// Gradients from their fp32 sums.  If a wait gave up, all of them become NaN instead.
template <class T>
__global__ void __launch_bounds__(1024)
finish_backward_kernel(const XentArgs a, const XentWs w, const FinishShares sh) {
  pdl_trigger();
  pdl_wait();
  if (any_error(w.hdr)) {
    if (a.dX) fill_nan(static_cast<T*>(a.dX), a.N * a.D);
    if (a.dW) fill_nan(static_cast<T*>(a.dW), (int64_t)a.V * a.D);
    if (a.dbias) fill_nan(a.dbias, a.V);
    return;
  }
  const float back = Scales(&w.hdr->amax, std::is_same<T, __half>::value).back;
  int b = blockIdx.x;
  if (b < sh.dx) {
    store_slots<T>(Share{b, sh.dx}, w.dx_slots, w.ks_x, w.Np, w.ldS, a.D, a.N, w.inv, back,
                   sh.lanes, static_cast<T*>(a.dX));
    return;
  }
  b -= sh.dx;
  if (b < sh.dw) {
    store_slots<T>(Share{b, sh.dw}, w.dw_slots, w.ks_w, w.piece, w.ldS, a.D, a.V, nullptr, back,
                   sh.lanes, static_cast<T*>(a.dW));
    return;
  }
  if (b - sh.dw < sh.dbias) store_dbias(b - sh.dw, a, w);
}

// Blocks of 256 threads for that many threads' work: all resident at once at most.
int blocks_for(int64_t threads) {
  return (int)std::min<int64_t>(std::max<int64_t>((threads + 255) / 256, 1), 8 * num_sms());
}
int row_lanes(int64_t pieces, int most) {
  int lanes = 1;
  while (lanes < most && lanes < pieces) lanes *= 2;
  return lanes;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder.  It needs the device's context current on the calling thread,
// which a thread that has made no runtime call yet (autograd's, a new host thread) lacks
// until cudaSetDevice binds it.
cudaError_t encode_fn(EncodeTiled* out) {
  static std::atomic<void*> cached{nullptr};
  int dev = 0;
  cudaError_t bound = cudaGetDevice(&dev);
  if (bound == cudaSuccess) bound = cudaSetDevice(dev);
  if (bound != cudaSuccess) return bound;
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

// Boxes of 128 bytes x box_rows of a row-major (rows, cols) matrix, 128-byte
// swizzle; elements outside read as zero.
cudaError_t make_map(EncodeTiled encode, CUtensorMap* m, CUtensorMapDataType type, const void* base,
                     int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  const int size = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)std::max<int64_t>(rows, 1)};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, es[2] = {1, 1};
  const CUresult r = encode(m, type, 2, const_cast<void*>(base), dims, strides, box, es,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
template <class T>
constexpr CUtensorMapDataType word_type() {
  return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// Operand word of each element type, and what dW is stored as.
template <class T> struct Word { using type = T; };
template <> struct Word<float> { using type = __nv_bfloat16; };
template <class T> constexpr int kWordsOf = sizeof(T) == 4 ? 3 : 1;

template <class T>
cudaError_t make_operand_maps(const XentArgs& a, const XentWs& w, bool direct, MmaMaps* maps) {
  constexpr CUtensorMapDataType type = word_type<T>();
  EncodeTiled enc;
  cudaError_t e = encode_fn(&enc);
  for (int h = 0; h < kWordsOf<T>; ++h) {
    if (e == cudaSuccess)
      e = direct ? make_map(enc, &maps->X[h], type, a.X, a.N, a.D, a.sxn, 64)
                 : make_map(enc, &maps->X[h], type, w.Xp[h], w.Np, a.D, w.Dp, 64);
    if (e == cudaSuccess)
      e = w.pack_w ? make_map(enc, &maps->W[h], type, w.Wp[h], a.V, a.D, w.Dp, 64)
                   : make_map(enc, &maps->W[h], type, a.W, a.V, a.D, a.swv, 64);
  }
  return e;
}

// Maps of G, loaded and stored, and of the fp32 slots.
template <class T>
cudaError_t make_backward_maps(const XentWs& w, MmaMaps* maps) {
  constexpr CUtensorMapDataType type = word_type<T>(), f32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const int64_t rows = (int64_t)kRing * w.row_chunk;
  EncodeTiled enc;
  cudaError_t e = encode_fn(&enc);
  for (int h = 0; h < kWordsOf<T>; ++h) {
    if (e == cudaSuccess) e = make_map(enc, &maps->G[h], type, w.G[h], rows, w.piece, w.piece, 64);
    if (e == cudaSuccess) e = make_map(enc, &maps->Gs[h], type, w.G[h], rows, w.piece, w.piece, 32);
  }
  if (e == cudaSuccess) e = make_map(enc, &maps->dxs, f32, w.dx_slots, w.ks_x * w.Np, w.ldS, w.ldS, 32);
  if (e == cudaSuccess)
    e = make_map(enc, &maps->dws, f32, w.dw_slots, (int64_t)w.ks_w * w.piece, w.ldS, w.ldS, 32);
  return e;
}

// The launches before the first product.  `direct`: X is read in place; *dependent
// tells whether there was a launch.
template <class T>
cudaError_t prepare(const XentArgs& a, const XentWs& w, bool direct, bool backward, bool* dependent) {
  *dependent = false;
  cudaError_t e = cudaSuccess;
  auto vec = [&](const void* p, int64_t s0, int64_t s1) {
    return s1 == 1 && s0 * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  };
  if (!direct) {
    const int64_t blocks = (a.N + kRowsPerBlock - 1) / kRowsPerBlock;
    const bool counted = blocks > 4;
    if (counted) e = launch(count_kernel, blocks, 1024, 0, a.stream, false, a, w);
    if (e == cudaSuccess) e = launch(rows_kernel, blocks, 1024, 0, a.stream, counted, a, w, (int)counted);
    *dependent = true;
  }
  PrepareShares sh{};
  sh.lanes = row_lanes(w.Dp / 8, 256);
  sh.x = direct ? 0 : blocks_for(w.Np * sh.lanes);
  sh.w = w.pack_w ? blocks_for((int64_t)a.V * sh.lanes) : 0;
  sh.bias = a.bias ? blocks_for(w.Vp) : 0;
  sh.rows = backward ? blocks_for(w.Np) : 0;
  sh.vec_x = vec(a.X, a.sxn, a.sxd);
  sh.vec_w = vec(a.W, a.swv, a.swd);
  const int grid = sh.x + sh.w + sh.bias + sh.rows;
  if (e == cudaSuccess && grid > 0) {
    e = launch(prepare_kernel<T>, grid, 256, 0, a.stream, *dependent, a, w, sh);
    *dependent = true;
  }
  return e;
}

MmaParams common_params(const XentArgs& a, const XentWs& w) {
  MmaParams p{};
  p.live = &w.hdr->live;
  p.err = w.hdr->err;
  p.done = &w.hdr->done;
  p.amax = &w.hdr->amax;
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
cudaError_t launch_mma(const XentArgs& a, const MmaParams& p, const MmaMaps& maps, int64_t units,
                       bool dependent) {
  constexpr bool kSplit = sizeof(T) == 4;
  auto* kernel = xent_mma_kernel<FWD, kSplit, typename Word<T>::type, T>;
  constexpr size_t smem = MmaCfg<kSplit>::kSmem;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const int64_t pairs = std::min<int64_t>(units, std::min(num_sms(), kErrSlots) / 2);
  return launch(kernel, 2 * pairs, kMmaThreads, smem, a.stream, dependent, p, maps);
}

// How X, W (and `out`, contiguous rows) can be accessed.
template <class T>
int small_mode(const XentArgs& a, const void* out) {
  auto four = [&](const void* p, int64_t s0) {
    return s0 % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0;
  };
  if (a.sxd != 1 || a.swd != 1) return kAnyStride;
  return a.D % 4 == 0 && four(a.X, a.sxn) && four(a.W, a.swv) && four(out, a.D) ? kVector : kUnitStride;
}
template <class F>
cudaError_t with_mode(int mode, F&& f) {
  if (mode == kVector) return f(std::integral_constant<int, kVector>{});
  if (mode == kUnitStride) return f(std::integral_constant<int, kUnitStride>{});
  return f(std::integral_constant<int, kAnyStride>{});
}

template <class T, bool GRAD>
cudaError_t small_logits(const XentArgs& a, const XentWs& w, const SmallPlan& p) {
  auto run = [&](auto nb, auto r, auto mode) {
    return launch(small_logits_kernel<T, nb, r, mode, GRAD>, p.blocks, 32 * kSmallWarps, 0, a.stream, false,
                  a, w, p);
  };
  return with_mode(small_mode<T>(a, nullptr), [&](auto mode) {
    using std::integral_constant;
    if constexpr (sizeof(T) == 4) {   // 16-bit types come with one row
      if (p.nb == 16) return run(integral_constant<int, 16>{}, integral_constant<int, 2>{}, mode);
      if (p.nb == 8) return run(integral_constant<int, 8>{}, integral_constant<int, 4>{}, mode);
    }
    return run(integral_constant<int, 1>{}, integral_constant<int, 8>{}, mode);
  });
}

template <class T>
cudaError_t small_forward(const XentArgs& a, const XentWs& w) {
  const SmallPlan p = small_plan(a.N, a.V, a.D);
  cudaError_t e = small_logits<T, false>(a, w, p);
  if (e != cudaSuccess) return e;
  return launch(finish_forward_kernel, 1, 1024, 0, a.stream, true, a, w, p.blocks, 1, 0);
}

template <class T>
cudaError_t small_backward(const XentArgs& a, const XentWs& w) {
  const SmallPlan p = small_plan(a.N, a.V, a.D);
  cudaError_t e = small_logits<T, true>(a, w, p);
  if (e != cudaSuccess || (!a.dX && !a.dW)) return e;
  auto run = [&](auto nb, auto mode) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.D + kSmallCols - 1) / kSmallCols), (unsigned)p.splits);
    cfg.blockDim = dim3(128);
    cfg.stream = a.stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    count_launches(1);
    return cudaLaunchKernelEx(&cfg, small_products_kernel<T, nb, mode>, a, w, p);
  };
  e = with_mode(small_mode<T>(a, a.dW), [&](auto mode) {
    using std::integral_constant;
    if constexpr (sizeof(T) == 4) {
      if (p.nb == 16) return run(integral_constant<int, 16>{}, mode);
      if (p.nb == 8) return run(integral_constant<int, 8>{}, mode);
    }
    return run(integral_constant<int, 1>{}, mode);
  });
  if (e != cudaSuccess || !a.dX) return e;
  return launch(small_finish_kernel<T>, (a.N * a.D + 31) / 32, 256, 0, a.stream, true, a, w, p);
}

template <class T>
cudaError_t xent_forward(const XentArgs& a, const XentWs& w) {
  if (w.small) return small_forward<T>(a, w);
  MmaMaps maps{};
  // Up to one tile of rows that TMA can read is used in place: no list, no copy, and
  // the ignored rows among them cost nothing.
  const bool direct = sizeof(T) == 2 && a.N <= kPairRows && a.sxd == 1 && a.sxn >= a.D &&
                      a.sxn % 8 == 0 && a.sxn < (int64_t(1) << 38) &&
                      (reinterpret_cast<uintptr_t>(a.X) & 15) == 0;
  cudaError_t e = make_operand_maps<T>(a, w, direct, &maps);
  bool dependent;
  if (e == cudaSuccess) e = prepare<T>(a, w, direct, false, &dependent);
  if (e != cudaSuccess) return e;
  MmaParams p = common_params(a, w);
  p.vtiles = w.vtiles;
  p.per_split = w.per_split;
  p.splits = w.splits;
  p.part = w.part;
  p.tlogit = w.tlogit;
  p.target = direct ? nullptr : w.target;
  p.targets = a.targets;
  e = launch_mma<true, T>(a, p, maps, w.Np / kPairRows * w.splits, dependent);
  if (e != cudaSuccess) return e;
  const bool few = w.splits <= 8 && a.N > 32;   // up to 16 parts a row
  return launch(finish_forward_kernel, few ? (a.N + 1023) / 1024 : (a.N + 31) / 32, 1024, 0, a.stream,
                true, a, w, 2 * w.splits, (int)direct, (int)few);
}

template <class T>
cudaError_t xent_backward(const XentArgs& a, const XentWs& w) {
  if (w.small) return small_backward<T>(a, w);
  MmaMaps maps{};
  cudaError_t e = make_operand_maps<T>(a, w, false, &maps);
  if (e == cudaSuccess) e = make_backward_maps<T>(w, &maps);
  bool dependent;
  if (e == cudaSuccess) e = prepare<T>(a, w, false, true, &dependent);
  if (e != cudaSuccess) return e;
  MmaParams p = common_params(a, w);
  p.bn_d = w.bn_d;
  p.tiles_d = w.tiles_d;
  p.has_dx = a.dX != nullptr;
  p.has_dw = a.dW != nullptr;
  p.row_chunk = w.row_chunk;
  p.piece = w.piece;
  p.n_chunks = w.n_chunks;
  p.n_pieces = w.n_pieces;
  p.sync = w.sync;
  p.rg = w.rg;
  p.dbias_part = a.dbias ? w.dbias_part : nullptr;
  p.ks_x = w.ks_x;
  p.ks_w = w.ks_w;
  p.dw_slots = w.dw_slots;
  p.ldS = w.ldS;
  p.dW = a.dW;
  p.dw_vec = a.D % 4 == 0 && (reinterpret_cast<uintptr_t>(a.dW) & (4 * sizeof(T) - 1)) == 0;
  const int64_t units = (int64_t)(w.row_chunk / 256) * (w.piece / 256) * w.n_chunks * w.n_pieces;
  e = launch_mma<false, T>(a, p, maps, std::max<int64_t>(units, XentWs::kPairs), true);
  if (e != cudaSuccess) return e;
  FinishShares sh{};
  sh.lanes = row_lanes((a.D + 3) / 4, 1024);
  auto blocks = [&](int64_t rows) {
    return (int)std::min<int64_t>((rows * sh.lanes + 1023) / 1024, 2 * num_sms());
  };
  sh.dx = a.dX ? blocks(a.N) : 0;
  sh.dw = a.dW && w.ks_w > 1 ? blocks(a.V) : 0;
  sh.dbias = a.dbias ? (a.V + 31) / 32 : 0;
  return launch(finish_backward_kernel<T>, std::max(sh.dx + sh.dw + sh.dbias, 1), 1024, 0, a.stream,
                true, a, w, sh);
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

int check_workspace_and_device(const XentArgs& a, size_t need) {
  int rc = vocab_check_workspace(a.name, a.ws, a.ws_bytes, need);
  if (rc != FGMM_OK) return rc;
  std::string why;
  rc = entry_check_device(&why);
  return rc == FGMM_OK ? rc : entry_fail(rc, std::string(a.name) + ": " + why);
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
    rc = check_workspace_and_device(a, w.bytes);
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
    const XentWs w(workspace, true, type, N, V, D, W, w_stride_v, w_stride_d, bias || dbias);
    if (w.units >= (int64_t(1) << 31) - (1 << 16))
      return entry_fail(FGMM_ERR_UNSUPPORTED, std::string(name) + ": N * V exceeds what one call counts; split the rows");
    rc = check_workspace_and_device(a, w.bytes);
    if (rc != FGMM_OK) return rc;
    cudaError_t e = cudaSuccess;
    if (!dX && !dW && !dbias) return FGMM_OK;
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
