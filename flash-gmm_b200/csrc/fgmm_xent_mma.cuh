// The tensor-core kernel of the linear cross entropy (included by fgmm_xent.cu).
//
// One persistent kernel of two-SM pairs serves four products, all as 256-row
// tiles of C = A B^T with K in blocks of 64:
//   kLse   S  = Xp W^T       rows x vocabulary, K = D     -> running (max, sum) per row
//   kGrad  S  = Xp W^T       again, with logZ known       -> g, stored as G (rows x piece)
//   kDx    dX = G W          rows x D, K = the piece      -> fp32 slots
//   kDw    dW = G^T Xp       piece x D, K = the rows      -> dW, or fp32 slots
// Every operand comes from one of three row-major matrices (Xp, W, G) through
// 64 x 64 TMA boxes of 8 KB, 128-byte swizzled: read with K along the row (K-major)
// or across rows (MN-major), so G and W serve two products each untransposed.
//
// A pair's MMA is M = 256 (128 rows per SM) x BN: each SM stages its 128 rows of A
// and its half of B, so a 256 x 256 x 64 block costs each SM 32 KB of staged bytes
// against 512 cycles of MMA; one SM alone would need 48 KB for half the product and
// be bound by the L2.  Two BN-column accumulators in TMEM let eight epilogue warps
// work on one tile while the next is multiplied.
//
// SPLIT (fp32 inputs): operands are pairs of fp16 words hi + lo of the values scaled
// by one power of two per matrix, and a K-block runs lo hi, hi lo and hi hi.
//
// The tensor core cuts its running sum toward zero at each step of 16, about 2^-24 of
// it on average: logits of 63 steps measured 2.3e-6 low.  Logits (and all of SPLIT) are
// therefore emptied into fp32 registers every few K-blocks (group_blocks), where sums
// round to nearest.  Products with G stored in 16 bits are not: their words' rounding
// of 2^-9 or 2^-12 outweighs a chain's 2^-14.
//
// Warps: 0 TMA loads, 1 MMA (the pair's first SM), 2 TMEM, 4-11 epilogue in two
// warpgroups (TMEM lane quadrant = warp & 3) that take a tile's halves, 128 columns of
// a row per thread.  Every wait is bounded; a timeout sets the error word, all roles
// leave, and the closing kernels write NaN.
//
// Measured and not kept: 128-wide tiles that the warpgroups take in turn (so that one's
// exponentials overlap the other's waits): an M = 256, N = 128 step reads shared memory
// at its full rate, 65536 x 8192 x 256 bf16 logits 285 -> 444 us.  Three of eight
// exponentials as a polynomial on the FMA pipe: 303 -> 317 us at D = 64; the epilogue is
// bound by its dependent latencies, not by the special-function unit (50% busy).

constexpr int kPairRows = 256;
constexpr int kErrSlots = 256;    // blocks of this kernel, at most
constexpr int kBoxBytes = 64 * 128;
constexpr int kEpiWarps = 8;
constexpr int kMmaThreads = (4 + kEpiWarps) * 32;
constexpr int kSplitBlocks = 2;   // K-blocks per group: 24 steps
constexpr int kLogitBlocks = 4;   // 16 steps

enum TileKind { kLse = 0, kGrad = 1, kDx = 2, kDw = 3 };

// A rectangle of live rows x vocabulary.
struct Piece {
  int64_t r0;   // first live row (multiple of 256)
  int rows;     // rows at most (multiple of 256); the last live row may end it earlier
  int v0, nv;   // vocabulary [v0, v0 + nv); v0 multiple of 256
};

struct MmaParams {
  const int* live;         // unused where target is null
  int *err, *done;         // Header
  int first;               // first launch of the call: err and done start at 0
  int64_t N;
  int D, V, kbD;           // kbD = ceil(D / 64)
  int bn_d, tiles_d;       // column tiles of dX and dW: width 128 or 256, count
  // forward
  int vtiles, per_split, splits;
  float2* part;            // [2 splits][Np] (max, sum of exp(S - max)), natural units
  float* tlogit;           // [Np] S at the target
  const int* target;       // [Np] the live rows' targets (-1: none); null: X is read in place,
  const int64_t* targets;  // row i's target is targets[i]
  int64_t Np;
  const float* bias;       // padded to 256 with -inf, or null
  const int* amax;         // float bits of the largest |g weight|, |x|, |w| (Scales)
  // backward
  int has_grad, has_dx, has_dw;
  Piece cur, prev;         // of kGrad, and of kDx / kDw
  const RowGrad* rg;
  void *G, *G2;            // written by kGrad (G2: lo words)
  int64_t ldG;
  float* dbias_part;       // [2 Np / 256][Vp], or null
  int64_t Vp;
  int ks_x, ks_w;          // splits of K
  float* dx_slots;         // [ks_x][Np][ldS]
  float* dw_slots;         // [ks_w][piece rows][ldS], or null: written to dW
  int64_t ldS;
  int64_t dw_rows;
  int dx_add, dw_add;      // add to the slots (a later piece / row chunk)
  void* dW;
  int dw_vec;              // dW's rows take 16-byte stores
};

struct MmaMaps {
  CUtensorMap X, W, G, X2, W2, G2;
};

// Scales of the stored words.  G is stored over the largest row weight: with equal
// weights (a sum or a mean) the -1 at the label is then exact, where a weight like
// 1/7372 rounded to bf16 would scale the whole gradient by up to 2^-9.  fp16 words are
// 2^12 times that (at most 2^13, down to p = 2^-27 without losing bits).  SPLIT: X and
// W too, by a power of two each with the largest finite magnitude in [2^13, 2^14), so
// values down to 2^-16 of the largest keep 22 bits and smaller ones an error of 2^-39
// of the largest.
struct Scales {
  float s, g, dx, dw;   // S, stored G, and the products with G
  __device__ static int exponent(int bits, int target) {
    return max(-100, min(100, scale_exp_to(__int_as_float(bits), target)));
  }
  __device__ Scales(const int* amax, bool f16, bool split) {
    if (!amax) { s = g = dx = dw = 1.f; return; }   // 16-bit logits: nothing is scaled
    const float top = __int_as_float(amax[0]);
    const float unit = f16 ? 4096.f : 1.f;
    // weights outside 2^-100 .. 2^100: their reciprocal would leave fp32
    const bool sane = top > 7.9e-31f && top < 1.2e30f;
    g = sane ? unit / top : unit;
    const float back = sane ? top / unit : 1.f / unit;
    const int ex = split ? exponent(amax[1], 14) : 0, ew = split ? exponent(amax[2], 14) : 0;
    s = ldexpf(1.f, ex + ew);
    dx = ldexpf(back, ew);
    dw = ldexpf(back, ex);
  }
};

struct Tile {
  int kind;
  int64_t arow, brow;   // first A / B row (K-major) or column (MN-major) of the pair's tile
  int64_t ak, bk;       // first K of A / B
  int nkb;              // K blocks
  int bn;
  int m, n, ks;         // tile indices
  int last;             // kLse: last tile of the unit
};

// Programmatic dependent launch: let the next kernel of the stream be set up, and wait
// for the end of the one before (no-ops in a launch without the attribute).
__device__ __forceinline__ void pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                              uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 ad, bd;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 ad, {%1, %3};\n\t"
      "mov.b64 bd, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on `bar` of both SMs of the pair once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// What an epilogue warp hands back is TMEM it has read (tcgen05.wait::ld and the
// tcgen05 fence order that): nothing of its memory writes, so no cluster-wide release,
// which cost about 900 cycles a tile.
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// K-blocks that the accumulator takes before it is emptied into registers.
template <bool SPLIT, bool F16>
__device__ __forceinline__ int group_blocks(const MmaParams& p, const Tile& t) {
  if (SPLIT) return kSplitBlocks;
  // bf16's g does not see the cut of its logits; fp16's and a fp32 dbias do
  if (t.kind == kLse || (t.kind == kGrad && (F16 || p.dbias_part))) return kLogitBlocks;
  return t.nkb;
}

// Moves registers between the warpgroups: 4 warps x 72 + 8 x 216 = 12 x 168.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void idle_cycles(long long n) {
  const long long t0 = clock64();
  while (clock64() - t0 < n) {}
}

constexpr int kBN = 256;          // widest tile: the width of logits

template <bool SPLIT>
struct MmaCfg {
  static constexpr int kStages = SPLIT ? 3 : 6;
  static constexpr int kA = 2 * kBoxBytes;                   // 128 rows x 64
  static constexpr int kB = (kBN / 2 / 64) * kBoxBytes;      // this SM's half of B
  static constexpr int kStage = (SPLIT ? 2 : 1) * (kA + kB);
  static constexpr int kStageOut = kEpiWarps * 4096;         // 32 rows x 128 B per warp
  static constexpr int kCtl = 256;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kStageOut + kCtl;
  static_assert(kSmem <= 232448, "shared memory budget");
};

struct MmaCtl {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  volatile int abort_flag;
};
static_assert(sizeof(MmaCtl) <= 256, "control block");

// The pair's tiles in order: the same sequence for every role.
template <bool FWD, bool SPLIT>
struct TileWalk {
  const MmaParams& p;
  int64_t live;
  int unit, step, sub = 0, um = 0, us = 0;
  int mt, mtx, n_dw, n_dx, n_grad, units;
  __device__ TileWalk(const MmaParams& p_, int pair, int npairs) : p(p_), unit(pair), step(npairs) {
    live = FWD && !p.target ? p.N : *p.live;
    if (FWD) {
      mt = (int)((live + kPairRows - 1) / kPairRows);
      units = mt * p.splits;
    } else {
      auto tiles = [&](const Piece& q) {
        const int64_t r = live - q.r0;
        return (int)((max((int64_t)0, min(r, (int64_t)q.rows)) + kPairRows - 1) / kPairRows);
      };
      mtx = tiles(p.prev);
      mt = tiles(p.cur);
      n_dw = p.has_dw ? (p.prev.nv + kPairRows - 1) / kPairRows * p.tiles_d * p.ks_w : 0;
      n_dx = p.has_dx ? mtx * p.tiles_d * p.ks_x : 0;
      n_grad = p.has_grad ? mt * ((p.cur.nv + kBN - 1) / kBN) : 0;
      units = n_dw + n_dx + n_grad;
    }
  }
  __device__ bool next(Tile& t) {
    if (unit >= units) return false;
    if (FWD) {
      if (sub == 0) { us = unit / mt; um = unit - us * mt; }
      const int m = um, s = us;
      const int v = s * p.per_split + sub;
      t.kind = kLse;
      t.m = m; t.n = v; t.ks = s;
      t.arow = (int64_t)m * kPairRows; t.ak = 0;
      t.brow = (int64_t)v * kBN; t.bk = 0;
      t.nkb = p.kbD; t.bn = kBN;
      ++sub;
      t.last = sub == p.per_split || v + 1 == p.vtiles;
      if (t.last) { sub = 0; unit += step; }
      return true;
    }
    int u = unit;
    unit += step;
    t.last = 0;
    if (u < n_dw) {          // column tiles fastest: they share G's columns
      t.kind = kDw;
      t.n = u % p.tiles_d; u /= p.tiles_d;
      t.ks = u % p.ks_w; t.m = u / p.ks_w;
      const int64_t rows = max((int64_t)0, min(live - p.prev.r0, (int64_t)p.prev.rows));
      const int nkb = (int)((rows + 63) / 64), per = (nkb + p.ks_w - 1) / p.ks_w;
      const int k0 = t.ks * per;
      t.nkb = max(0, min(per, nkb - k0));
      t.arow = (int64_t)t.m * kPairRows; t.ak = (int64_t)k0 * 64;            // of G
      t.brow = (int64_t)t.n * p.bn_d; t.bk = p.prev.r0 + (int64_t)k0 * 64;   // of Xp
      t.bn = p.bn_d;
    } else if ((u -= n_dw) < n_dx) {
      t.kind = kDx;
      t.n = u % p.tiles_d; u /= p.tiles_d;
      t.ks = u % p.ks_x; t.m = u / p.ks_x;
      const int nkb = (p.prev.nv + 63) / 64, per = (nkb + p.ks_x - 1) / p.ks_x;
      const int k0 = t.ks * per;
      t.nkb = max(0, min(per, nkb - k0));
      t.arow = (int64_t)t.m * kPairRows; t.ak = (int64_t)k0 * 64;            // of G
      t.brow = (int64_t)t.n * p.bn_d; t.bk = p.prev.v0 + (int64_t)k0 * 64;   // of W
      t.bn = p.bn_d;
    } else {
      u -= n_dx;
      t.kind = kGrad;
      t.m = u % mt; t.n = u / mt; t.ks = 0;
      t.arow = p.cur.r0 + (int64_t)t.m * kPairRows; t.ak = 0;                // of Xp
      t.brow = p.cur.v0 + (int64_t)t.n * kBN; t.bk = 0;                       // of W
      t.nkb = p.kbD; t.bn = kBN;
    }
    return true;
  }
};

// Sums the 32 values of each column over the warp's 32 rows: lane c gets column c.
__device__ __forceinline__ float column_sums(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// Two fp32 values in one register pair: Blackwell's packed add, multiply and FMA take
// one issue slot for both.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack(F2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 exp2_pair(F2 x) {
  float a, b;
  unpack(x, a, b);
  return f2(ex2(a), ex2(b));
}

__device__ __forceinline__ void tmem_ld32f(uint32_t taddr, float (&v)[32]) {
  uint32_t u[32];
  tmem_ld32(taddr, u);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_f16(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<float>(float, float) { return 0; }

// T: the type of the operand words (SPLIT: __half); TO: the type of dW.
template <bool FWD, bool SPLIT, class T, class TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMmaThreads, 1)
xent_mma_kernel(const __grid_constant__ MmaParams p, const __grid_constant__ MmaMaps maps) {
  using Cfg = MmaCfg<SPLIT>;
  constexpr int NS = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* out_stage = smem + NS * Cfg::kStage;
  MmaCtl* ctl = reinterpret_cast<MmaCtl*>(out_stage + Cfg::kStageOut);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&ctl->full[s], 1);    // first SM's arrive.expect_tx + both SMs' bytes
      mbar_init(&ctl->empty[s], 1);   // commit
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl->acc_full[b], 1);                // commit
      mbar_init(&ctl->acc_empty[b], 2 * kEpiWarps);   // both SMs' epilogue warps
    }
    mbar_init(&ctl->drain, 1);
    ctl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&ctl->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the other SM's barriers are ready before anything arrives there
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  // set up; now what the launches before this one write
  pdl_trigger();
  pdl_wait();
  int* err = p.err + blockIdx.x;
  if (p.first) {
    if (threadIdx.x == 0)
      for (int i = blockIdx.x; i < kErrSlots; i += gridDim.x) p.err[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;
    __syncthreads();
  }
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return mbar_wait_flag(bar, parity, &ctl->abort_flag, err, code);
  };

  if (warp < 4) {
    regs_down<72>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ loads
      TileWalk<FWD, SPLIT> walk(p, pair, npairs);
      Tile t;
      uint32_t it = 0;
      bool ok = true;
      while (ok && walk.next(t)) {
        const bool a_mn = t.kind == kDw, b_mn = t.kind >= kDx;
        const CUtensorMap* ma = t.kind <= kGrad ? &maps.X : &maps.G;
        const CUtensorMap* mb = t.kind == kDw ? &maps.X : &maps.W;
        const CUtensorMap* ma2 = t.kind <= kGrad ? &maps.X2 : &maps.G2;
        const CUtensorMap* mb2 = t.kind == kDw ? &maps.X2 : &maps.W2;
        const int bboxes = t.bn / 128;                       // 64-row boxes of B per SM
        const int ar = (int)t.arow + 128 * (int)rank, br = (int)t.brow + t.bn / 2 * (int)rank;
        const uint32_t bytes = (uint32_t)((SPLIT ? 2 : 1) * (2 + bboxes) * kBoxBytes);
        for (int kb = 0; kb < t.nkb; ++kb, ++it) {
          const int s = it % NS;
          if (it >= NS && !wait(&ctl->empty[s], ((it / NS) - 1) & 1, 1)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], 2 * bytes);
          const uint32_t bar = map_to_cta(smem_u32(&ctl->full[s]), 0);
          uint32_t dst = smem_u32(smem + s * Cfg::kStage);
          const int ka = (int)t.ak + kb * 64, kbb = (int)t.bk + kb * 64;
          for (int h = 0; h < (SPLIT ? 2 : 1); ++h) {
            const CUtensorMap* a = h ? ma2 : ma;
            const CUtensorMap* b = h ? mb2 : mb;
            for (int j = 0; j < 2; ++j, dst += kBoxBytes)
              tma_load_pair(dst, a, a_mn ? ar + 64 * j : ka, a_mn ? ka : ar + 64 * j, bar);
            for (int j = 0; j < bboxes; ++j, dst += kBoxBytes)
              tma_load_pair(dst, b, b_mn ? br + 64 * j : kbb, b_mn ? kbb : br + 64 * j, bar);
            if (SPLIT) dst = smem_u32(smem + s * Cfg::kStage) + Cfg::kA + Cfg::kB;
          }
        }
      }
      // every stage handed back; after a timeout, time for the copies in flight to land
      for (uint32_t k = it > NS ? it - NS : 0; ok && k < it; ++k)
        ok = wait(&ctl->empty[k % NS], (k / NS) & 1, 2);
      if (!ok) idle_cycles(4000000);
    } else if (warp == 1 && rank == 0 && lane == 0) {
      // ------------------------------------------------------------ MMA
      TileWalk<FWD, SPLIT> walk(p, pair, npairs);
      Tile t;
      uint32_t it = 0, ac = 0;
      bool ok = true;
      constexpr bool f16 = std::is_same<T, __half>::value;
      while (ok && walk.next(t)) {
        const bool a_mn = t.kind == kDw, b_mn = t.kind >= kDx;
        const uint32_t idesc = (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) |
                               (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
                               ((uint32_t)(t.bn >> 3) << 17) | (16u << 24);
        const int group = group_blocks<SPLIT, f16>(p, t);
        for (int k0 = 0; ok && k0 < t.nkb; k0 += group, ++ac) {
          const uint32_t d = tmem + (uint32_t)kBN * (ac & 1);
          if (ac >= 2 && !wait(&ctl->acc_empty[ac & 1], ((ac >> 1) - 1) & 1, 4)) { ok = false; break; }
          tc_fence_after();
          const int k1 = min(t.nkb, k0 + group);
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int s = it % NS;
            if (!wait(&ctl->full[s], (it / NS) & 1, 8)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a0 = smem_u32(smem + s * Cfg::kStage);
            const uint32_t b0 = a0 + Cfg::kA;
            constexpr uint32_t lo = Cfg::kA + Cfg::kB;
#pragma unroll
            for (int term = SPLIT ? 0 : 2; term < 3; ++term) {   // lo hi, hi lo, hi hi
              const uint32_t a = a0 + (term == 0 ? lo : 0u), b = b0 + (term == 1 ? lo : 0u);
              const uint32_t ad = a_mn ? desc_lo_mnmajor(a, kBoxBytes) : desc_lo_kmajor(a);
              const uint32_t bd = b_mn ? desc_lo_mnmajor(b, kBoxBytes) : desc_lo_kmajor(b);
              const uint32_t as = a_mn ? 2048 >> 4 : 32 >> 4, bs = b_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_pair(d, ad + k * as, bd + k * bs, idesc,
                         (kb > k0 || k > 0 || term > (SPLIT ? 0 : 2)) ? 1u : 0u);
            }
            commit_pair(&ctl->empty[s]);
          }
          if (ok) commit_pair(&ctl->acc_full[ac & 1]);
        }
      }
      // after a timeout: let what was issued finish (bounded) before TMEM is freed
      if (!ok) {
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                smem_u32(&ctl->drain))
            : "memory");
        const long long t0 = clock64();
        while (!mbar_try(smem_u32(&ctl->drain), 0) && clock64() - t0 < 100000000LL) {}
      }
    }
  } else {
    regs_up<216>();
    // -------------------------------------------------------------- epilogue
    TileWalk<FWD, SPLIT> walk(p, pair, npairs);
    Tile t;
    uint32_t ac = 0;
    const int q = warp & 3, wg = (warp - 4) >> 2;
    const int row_in = 128 * (int)rank + 32 * q + lane;     // row of the 256-row tile
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
    uint8_t* stage = out_stage + (warp - 4) * 4096;
    const uint32_t empty0 = map_to_cta(smem_u32(&ctl->acc_empty[0]), 0);
    constexpr bool f16 = std::is_same<T, __half>::value;
    const Scales scales(FWD && !SPLIT ? nullptr : p.amax, f16, SPLIT);
    const float sc_s = scales.s;
    float m_run = -3.402823466e38f, s_run = 0.f;            // kLse, over the unit's tiles
    int target = -1;
    constexpr int kCols = 128;                              // columns per warp
    constexpr int kChunks = kCols / 32;

    auto release = [&](uint32_t a) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(empty0 + 8u * (a & 1));
    };
    auto wg_sync = [&] {   // the warpgroup's 128 threads
      asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
    };
    bool ok = true;
    while (ok && walk.next(t)) {
      const int col0 = wg * (t.bn / 2);                     // this warp's columns of the tile
      const int chunks = t.bn / 2 / 32;
      const int group = group_blocks<SPLIT, f16>(p, t);
      const int64_t row = t.arow + row_in;                  // kLse, kGrad: the live row
      if (FWD && t.n == t.ks * p.per_split) {               // first tile of the unit
        m_run = -3.402823466e38f;
        s_run = 0.f;
        if (p.target) {
          target = p.target[row];
        } else {
          const int64_t x = row < p.N ? p.targets[row] : -1;
          target = x >= 0 && x < p.V ? (int)x : -1;
        }
      }
      RowGrad rg;
      if (!FWD && t.kind == kGrad) rg = p.rg[row];          // in flight while the MMAs run
      // The tile's products of this thread's row, in registers; the accumulator is given
      // back before they are worked on.
      float acc[kChunks][32];
      for (int k0 = 0; ok && k0 < t.nkb; k0 += group, ++ac) {
        if (!__all_sync(0xffffffffu, wait(&ctl->acc_full[ac & 1], (ac >> 1) & 1, 32))) ok = false;
        tc_fence_after();
        const uint32_t at = lanes + (uint32_t)kBN * (ac & 1) + col0;
        if (k0 == 0) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            if (c < chunks) tmem_ld32f(at + 32 * c, acc[c]);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if (c >= chunks) break;
            float v[32];
            tmem_ld32f(at + 32 * c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c][i] += v[i];
          }
        }
        release(ac);
      }
      if (!ok) break;
      if (t.nkb == 0) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
      }

      if (t.kind <= kGrad) {   // products -> logits
        const int v0 = (int)t.brow + col0;
        if (SPLIT) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c][i] *= sc_s;
        }
        if (p.bias) {
          const float4* b = reinterpret_cast<const float4*>(p.bias + v0);
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 x = __ldg(b + 8 * c + i);
              acc[c][4 * i] += x.x; acc[c][4 * i + 1] += x.y;
              acc[c][4 * i + 2] += x.z; acc[c][4 * i + 3] += x.w;
            }
        }
      }

      if (FWD) {
        const int v0 = (int)t.brow + col0;
        if (v0 + kCols > p.V) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (v0 + 32 * c + i >= p.V) acc[c][i] = __int_as_float(0xff800000);
        }
        const int tc = target - v0;
        const bool mine = tc >= 0 && tc < kCols;
        if (__any_sync(0xffffffffu, mine)) {
          float x = 0.f;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) x = tc == 32 * c + i ? acc[c][i] : x;
          if (mine) p.tlogit[row] = x;
        }
        float m8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) m8[k] = acc[0][k];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) m8[i & 7] = fmaxf(m8[i & 7], acc[c][i]);
        const float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                               fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
        const float mn = fmaxf(m_run, mx);
        s_run *= ex2((m_run - mn) * kLog2Ef);
        m_run = mn;
        if (p.bias) {   // differences first, and exact zeros: a bias may be the lowest float
          float s8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) s8[i & 7] += ex2((acc[c][i] - mn) * kLog2Ef);
          s_run += ((s8[0] + s8[1]) + (s8[2] + s8[3])) + ((s8[4] + s8[5]) + (s8[6] + s8[7]));
        } else {
          const float nm = fminf(-mn, 2e38f) * kLog2Ef;   // finite where every entry is masked
          const F2 l2 = f2(kLog2Ef, kLog2Ef), nm2 = f2(nm, nm);
          F2 s4[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              s4[j & 3] = add2(s4[j & 3], exp2_pair(fma2(f2(acc[c][2 * j], acc[c][2 * j + 1]), l2, nm2)));
          float sa, sb;
          unpack(add2(add2(s4[0], s4[1]), add2(s4[2], s4[3])), sa, sb);
          s_run += sa + sb;
        }
        if (t.last) p.part[(int64_t)(2 * t.ks + wg) * p.Np + row] = make_float2(m_run, s_run);
        continue;
      }

      if (t.kind == kGrad) {
        const int v0 = (int)t.brow + col0;
        const int vend = p.cur.v0 + p.cur.nv;
        const float ga = rg.a * scales.g, gb = rg.b * scales.g;
        if (p.bias) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c][i] = ga * ex2((acc[c][i] - rg.lse) * kLog2Ef);
        } else {
          // bf16 and fp16 words hide the rounding of lse log2(e) in the product's FMA
          const F2 l2 = f2(kLog2Ef, kLog2Ef), ga2 = f2(ga, ga);
          const F2 off = SPLIT ? f2(-rg.lse, -rg.lse) : f2(-rg.lse * kLog2Ef, -rg.lse * kLog2Ef);
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const F2 v = f2(acc[c][2 * j], acc[c][2 * j + 1]);
              const F2 x = SPLIT ? mul2(add2(v, off), l2) : fma2(v, l2, off);
              unpack(mul2(exp2_pair(x), ga2), acc[c][2 * j], acc[c][2 * j + 1]);
            }
        }
        const int tc = rg.target - v0;
        if (__any_sync(0xffffffffu, tc >= 0 && tc < kCols)) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (tc == 32 * c + i) acc[c][i] -= gb;
        }
        // rows without a weight (padding) and entries behind the last: exactly zero
        const bool empty = rg.a == 0.f && rg.b == 0.f;
        if (v0 + kCols > vend || __any_sync(0xffffffffu, empty)) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (empty || v0 + 32 * c + i >= vend) acc[c][i] = 0.f;
        }
        // 128-byte staged rows: 64 columns of 16-bit words, or 32 of hi and lo words
        const int64_t grow0 = row - lane - p.cur.r0;        // rows of the G buffer
        const int64_t gcol0 = t.brow - p.cur.v0 + col0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
          for (int h = 0; h < (SPLIT ? 2 : 1); ++h) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float a = acc[c][2 * i], bb = acc[c][2 * i + 1];
              uint32_t hi = pack2<T>(a, bb);
              if (SPLIT && h) hi = pack_f16(a - f16lo_f(hi), bb - f16hi_f(hi));
              w[i] = hi;
            }
            const int g0 = SPLIT ? h * 4 : (c & 1) * 4;       // first 16-byte granule
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((g0 + i) ^ (lane & 7)) << 4)) =
                  make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          }
          if (SPLIT || (c & 1)) {
            __syncwarp();
            const int64_t gcol = gcol0 + 32 * (SPLIT ? c : c - 1);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = 4 * i + (lane >> 3), g = lane & 7;
              const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
              uint16_t* dst;
              if (SPLIT)
                dst = static_cast<uint16_t*>(g < 4 ? p.G : p.G2) + (grow0 + r) * p.ldG + gcol + 8 * (g & 3);
              else
                dst = static_cast<uint16_t*>(p.G) + (grow0 + r) * p.ldG + gcol + 8 * g;
              *reinterpret_cast<uint4*>(dst) = x;
            }
            __syncwarp();
          }
        }
        if (p.dbias_part) {
          // column sums of the unrounded g; the four quadrants' meet in the warpgroup's
          // (now free) stages
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            reinterpret_cast<float*>(stage)[32 * c + lane] = column_sums(acc[c], lane);
          wg_sync();
          const int e = (int)threadIdx.x & 127;
          const float* cs = reinterpret_cast<const float*>(out_stage + wg * 16384) + e;
          const float s = (cs[0] + cs[1024]) + (cs[2048] + cs[3072]);
          p.dbias_part[(2 * (t.arow / kPairRows) + rank) * p.Vp + t.brow + col0 + e] = s;
          wg_sync();
        }
        continue;
      }

      // kDx, kDw: fp32 slots, or dW rows in their type
      const bool dw = t.kind == kDw;
      const bool direct = dw && !p.dw_slots;
      const int64_t row0 = (dw ? t.arow : p.prev.r0 + t.arow) + 128 * (int)rank + 32 * q;
      float* slots = dw ? p.dw_slots + (int64_t)t.ks * p.dw_rows * p.ldS
                        : p.dx_slots + (int64_t)t.ks * p.Np * p.ldS;
      const int add = dw ? p.dw_add : p.dx_add;
      const float so = scales.dw;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (c >= chunks) break;
        const float (&v)[32] = acc[c];
        const int64_t col = t.brow + col0 + 32 * c;
        // 32 fp32 columns = a 128-byte staged row
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
              make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        __syncwarp();
        if (!direct) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3), g = lane & 7;
            float4 x = *reinterpret_cast<const float4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
            float4* dst = reinterpret_cast<float4*>(slots + (row0 + r) * p.ldS + col + 4 * g);
            if (add) {
              const float4 o = *dst;
              x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w;
            }
            *dst = x;
          }
        } else if (p.dw_vec && col + 32 <= p.D) {
          // 16-byte stores: 4 lanes a row, 8 rows at a time
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + (lane >> 2), g = 2 * (lane & 3);
            const float4 x = *reinterpret_cast<const float4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
            const float4 y = *reinterpret_cast<const float4*>(stage + r * 128 + (((g + 1) ^ (r & 7)) << 4));
            const int64_t vrow = row0 + r;
            if (vrow < p.prev.nv) {
              const uint4 w = make_uint4(pack2<TO>(x.x * so, x.y * so), pack2<TO>(x.z * so, x.w * so),
                                         pack2<TO>(y.x * so, y.y * so), pack2<TO>(y.z * so, y.w * so));
              *reinterpret_cast<uint4*>(static_cast<TO*>(p.dW) + (p.prev.v0 + vrow) * p.D + col + 4 * g) = w;
            }
          }
        } else {
          for (int r = 0; r < 32; ++r) {
            const float x = *reinterpret_cast<const float*>(
                stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3));
            const int64_t vrow = row0 + r;
            if (vrow < p.prev.nv && col + lane < p.D)
              static_cast<TO*>(p.dW)[(p.prev.v0 + vrow) * p.D + col + lane] = from_f32<TO>(x * so);
          }
        }
        __syncwarp();
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // nobody frees shared memory or TMEM that the other SM still uses
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}
