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
// A pair's MMA is M = 256 (128 rows per SM) x 256: each SM stages its 128 rows of A
// and its half of B, so a 256 x 256 x 64 block costs each SM 32 KB of staged bytes
// against 512 cycles of MMA; one SM alone would need 48 KB for half the product and
// be bound by the L2.  Two 256-column accumulators in TMEM let eight epilogue warps
// work on one tile while the next is multiplied.
//
// SPLIT (fp32 inputs): operands are three bf16 words hi + mid + lo, each the rounding of
// what the ones before leave (2^-9 of it), so they hold a value to 2^-27 over fp32's whole
// range: no scale per matrix, and small values beside large ones keep their bits.  A
// K-block runs the six products of words above 2^-27, smallest first: lo hi, hi lo, mid mid,
// mid hi, hi mid, hi hi.  (Two fp16 words with three products took about half the time but
// share one exponent range of 2^-39 with the matrix's largest value: a column, a row or a
// row weight 1e8 times the others' lost the others.)
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
constexpr int kSplitBlocks = 1;   // K-blocks per group: 4 steps of hi hi upon small ones
constexpr int kLogitBlocks = 4;   // 16 steps
constexpr int kGradBlocks = 16;   // 64 steps, D = 1024: a cut of 2^-18 of the logit at any D (one
                                  // chain of 4096 steps: p 26% low at D = 65536, logits of 800)

enum TileKind { kLse = 0, kGrad = 1, kDx = 2, kDw = 3 };

struct MmaParams {
  const int* live;         // unused where target is null
  int *err, *done;         // Header
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
  const int* amax;         // backward: float bits of the largest |g weight| (Scales)
  // backward
  int has_dx, has_dw;
  int row_chunk, piece;    // rows x entries of a piece of G (multiples of 256)
  int n_chunks, n_pieces;  // row chunks at most, pieces of the vocabulary
  uint32_t* sync;          // from 0: units claimed, then marks of kGrad and of the products by
                           // piece, then of each tile of dX's and of dW's slots
  const RowGrad* rg;
  float* dbias_part;       // [2 kRing row_chunk / 256][Vp] at most, or null
  int64_t Vp;
  int ks_x, ks_w;          // splits of K
  const float* dw_slots;   // [ks_w][piece][ldS]
  int64_t ldS;
  void* dW;
  int dw_vec;              // dW's rows take stores of four elements
};

struct MmaMaps {
  CUtensorMap X[3], W[3], G[3];   // 64 x 64 boxes of words, loaded (SPLIT: hi, mid, lo)
  CUtensorMap Gs[3];              // 64 x 32 boxes of words, stored
  CUtensorMap dxs, dws;           // 32 x 32 boxes of fp32, stored or added
};

// Scale of the stored g, and what undoes it in the products.  G is stored over the largest
// row weight: with equal weights (a sum or a mean) the -1 at the label is then exact, where
// a weight like 1/7372 rounded to bf16 would scale the whole gradient by up to 2^-9.  bf16
// words (and SPLIT's) keep their bits over fp32's range.  fp16 words are 2^12 times that:
// |g| of 2^-26 of the largest weight and more keeps its 11 bits, smaller ones an error of
// 2^-37 of the largest weight.
struct Scales {
  float g, back;
  __device__ Scales(const int* amax, bool f16) {
    const float top = __int_as_float(*amax);
    const float unit = f16 ? 4096.f : 1.f;
    // weights outside 2^-100 .. 2^100: their reciprocal would leave fp32
    const bool sane = top > 7.9e-31f && top < 1.2e30f;
    g = sane ? unit / top : unit;
    back = sane ? top / unit : 1.f / unit;
  }
};

// One tile, as every role gets it (16 words).
struct __align__(16) Tile {
  int kind;             // TileKind, or -1: no more
  int arow, brow;       // first A / B row (K-major) or column (MN-major) of the pair's tile
  int ak, bk;           // first K of A / B
  int nkb, bn;          // K blocks, columns
  int ks;               // split of K; kLse: the unit's range of the vocabulary
  int flags;            // kLse: 1 last, 2 first tile of its unit; kGrad: 1 add to dbias's part;
                        // products: 1 add, 2 final
  int j;                // backward: the piece
  int x0, x1;           // kGrad: row, column of G; kDx: row of dX; kDw: row of the piece, v0
  uint32_t w0, w1;      // marks to wait for (wait_marks)
  int cell;             // products: their tile of the slots; kGrad: row tile of dbias's parts
  int pad;
};

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                              uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// An epilogue warp's staged 32 rows x 128 bytes, stored to (x, y) or added to it in the
// L2; one bulk group of the issuing thread.
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\t"
      "cp.async.bulk.commit_group;" ::"l"(map),
      "r"(x), "r"(y), "r"(src)
      : "memory");
}
__device__ __forceinline__ void tma_add(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];\n\t"
      "cp.async.bulk.commit_group;" ::"l"(map),
      "r"(x), "r"(y), "r"(src)
      : "memory");
}
// All groups of this thread: their shared memory has been read / their writes are done.
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_done() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
  // bf16's g sees less of its logits' cut; fp16's and a fp32 dbias see as much as logZ does
  if (t.kind == kLse || (t.kind == kGrad && (F16 || p.dbias_part))) return kLogitBlocks;
  if (t.kind == kGrad) return kGradBlocks;
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
constexpr int kFeedMax = 4;       // places of the feed

template <bool SPLIT>
struct MmaCfg {
  static constexpr int kWords = SPLIT ? 3 : 1;
  static constexpr int kStages = SPLIT ? 2 : 6;
  static constexpr int kFeed = SPLIT ? 3 : kFeedMax;         // tiles handed out ahead
  static constexpr int kA = 2 * kBoxBytes;                   // 128 rows x 64
  static constexpr int kB = (kBN / 2 / 64) * kBoxBytes;      // this SM's half of B
  static constexpr int kStage = kWords * (kA + kB);
  static constexpr int kStageOut = kEpiWarps * 4096;         // 32 rows x 128 B per warp
  static constexpr int kCtl = 768;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kStageOut + kCtl;
  static_assert(kSmem <= 232448, "shared memory budget");
};


struct MmaCtl {
  Tile feed[kFeedMax];
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drain;
  uint64_t feed_full[kFeedMax], feed_empty[kFeedMax], unit_done[kFeedMax];
  uint64_t wg_here[2];                // a warpgroup's four warps (wg_sync)
  uint32_t tmem;
  volatile int abort_flag;
};
static_assert(sizeof(MmaCtl) <= 768, "control block");

// The forward tiles of a pair in order: units of per_split vocabulary tiles of a row
// tile, dealt in turn (rows fastest: pairs at work share the vocabulary's tiles).
struct ForwardWalk {
  const MmaParams& p;
  int unit, step, sub = 0, m = 0, s = 0, mt;
  int64_t units;
  __device__ ForwardWalk(const MmaParams& p_, int pair, int npairs) : p(p_), unit(pair), step(npairs) {
    const int64_t live = p.target ? *p.live : p.N;
    mt = (int)((live + kPairRows - 1) / kPairRows);
    units = (int64_t)mt * p.splits;
  }
  __device__ bool next(Tile& t) {
    if (unit >= units) return false;
    if (sub == 0) { s = unit / mt; m = unit - s * mt; }
    const int v = s * p.per_split + sub;
    t.kind = kLse;
    t.ks = s;
    t.arow = m * kPairRows; t.ak = 0;
    t.brow = v * kBN; t.bk = 0;
    t.nkb = p.kbD; t.bn = kBN;
    t.flags = sub == 0 ? 2 : 0;
    ++sub;
    if (sub == p.per_split || v + 1 == p.vtiles) {
      t.flags |= 1;
      sub = 0;
      unit += step;
    }
    return true;
  }
};

// The backward tiles.  G runs through a ring of kRing pieces (row chunk x piece of the
// vocabulary, the chunks of one piece of the vocabulary in a row).  It bounds the workspace
// (kRing buffers of 32 MB, more than the 126 MB L2 holds, so part of G meets the DRAM):
// step j makes piece j's g (kGrad) and multiplies piece j - lag's (kDx, kDw), the two
// kinds mixed, since one is bound by its epilogue and the other by its products.  Pairs
// claim units in this one order, and a unit waits only for units before it in the order,
// so whichever pairs are resident make progress.  What a unit needs of others:
//   kGrad j       the products of piece j - kRing (the ring's buffer is free)
//                 and, where it adds to the parts of dbias, that piece's g: chunk rc uses those
//                 of chunk rc - kRing, which is kRing pieces back, so they do not grow with N
//   products i    all of piece i's g, and the unit before it on the same tile of the slots
// Each is a count of marks, one per SM that has finished its half of a unit (mark role).
constexpr int kRing = 5;
constexpr int kLag = 2;
constexpr uint32_t kMarks = 2;

struct BackwardList {
  const MmaParams& p;
  int live, chunks, pieces, lag;         // row chunks that hold live rows, pieces in all
  int step = 0, base = 0, n_grad = 0, n_prod = 0;
  struct Size { int rows, mt, v0, nv, vt; };
  __device__ explicit BackwardList(const MmaParams& p_) : p(p_) {
    live = *p.live;
    chunks = max(1, (live + p.row_chunk - 1) / p.row_chunk);
    pieces = chunks * p.n_pieces;
    lag = pieces <= kRing ? pieces : kLag;   // few pieces: all of g first
    load();
  }
  __device__ Size size(int j) const {
    const int vp = j / chunks, rc = j - vp * chunks;
    Size s;
    s.rows = min(live - rc * p.row_chunk, p.row_chunk);
    s.mt = (s.rows + kPairRows - 1) / kPairRows;
    s.v0 = vp * p.piece;
    s.nv = min(p.piece, p.V - s.v0);
    s.vt = (s.nv + 255) / 256;
    return s;
  }
  __device__ int grads(int j) const {
    if (j < 0 || j >= pieces) return 0;
    const Size s = size(j);
    return s.mt * s.vt;
  }
  __device__ int products(int j) const {
    if (j < 0 || j >= pieces) return 0;
    const Size s = size(j);
    return (p.has_dx ? s.mt * p.tiles_d * p.ks_x : 0) + (p.has_dw ? s.vt * p.tiles_d * p.ks_w : 0);
  }
  uint64_t share = 0;
  __device__ void load() {
    n_grad = grads(step);
    n_prod = products(step - lag);
    const int n = n_grad + n_prod;
    share = n > 0 ? ((uint64_t)n_prod << 32) / (uint64_t)n : 0;
  }
  // Products among the step's first i of n units, floor(i n_prod / n): in steps of 0 or 1.
  // The multiplication errs by less than n 2^-32 downwards, the quotients below n_prod are
  // at least 1/n off a whole number or exactly one: right for n < 2^15.
  __device__ int upto(int i) const {
    const int n = n_grad + n_prod;
    if (i >= n) return n_prod;
    if (n >= 1 << 15) return (int)((uint64_t)i * n_prod / n);
    return (int)(((uint64_t)(uint32_t)i * share + (1u << 16)) >> 32);
  }
  // Unit u (never smaller than the one before); kind -1 behind the last.
  __device__ void get(int u, Tile& t) {
    while (step < pieces + lag && u >= base + n_grad + n_prod) {
      base += n_grad + n_prod;
      ++step;
      load();
    }
    if (step >= pieces + lag) { t.kind = -1; return; }
    // products spread evenly among the step's units
    const int i = u - base;
    const int prod = upto(i);
    if (upto(i + 1) == prod) {
      const Size s = size(step);
      const int g = i - prod, vt = g / s.mt, m = g - vt * s.mt;
      t.kind = kGrad;
      t.j = step;
      t.arow = (step % chunks) * p.row_chunk + m * kPairRows; t.ak = 0;   // of Xp
      t.brow = s.v0 + vt * kBN; t.bk = 0;                                 // of W
      t.nkb = p.kbD; t.bn = kBN;
      t.ks = 0;
      const int rc = step % chunks;
      t.flags = rc >= kRing ? 1 : 0;
      t.cell = (rc % kRing) * (p.row_chunk / kPairRows) + m;
      t.x0 = (step % kRing) * p.row_chunk + m * kPairRows;
      t.x1 = vt * kBN;
      t.w0 = kMarks * (uint32_t)products(step - kRing);
      t.w1 = kMarks * (uint32_t)grads(step - kRing);
      return;
    }
    const int j = step - lag;
    const Size s = size(j);
    const int rc = j % chunks, g0 = (j % kRing) * p.row_chunk;
    const int n_dx = p.has_dx ? s.mt * p.tiles_d * p.ks_x : 0;
    t.j = j;
    t.bn = p.bn_d;
    t.w0 = kMarks * (uint32_t)(s.mt * s.vt);
    if (prod < n_dx) {
      int u2 = prod;
      const int tn = u2 % p.tiles_d;
      u2 /= p.tiles_d;
      t.ks = u2 % p.ks_x;
      const int m = u2 / p.ks_x;
      const int nkb = (s.nv + 63) / 64, per = (nkb + p.ks_x - 1) / p.ks_x, k0 = t.ks * per;
      t.kind = kDx;
      t.nkb = max(0, min(per, nkb - k0));
      t.arow = g0 + m * kPairRows; t.ak = k0 * 64;                        // of G
      t.brow = tn * p.bn_d; t.bk = s.v0 + k0 * 64;                        // of W
      t.flags = j >= chunks ? 1 : 0;
      t.x0 = rc * p.row_chunk + m * kPairRows;
      t.x1 = 0;
      t.w1 = kMarks * (uint32_t)(j / chunks);
      t.cell = ((t.x0 / kPairRows) * p.ks_x + t.ks) * p.tiles_d + tn;
    } else {
      int u2 = prod - n_dx;
      const int tn = u2 % p.tiles_d;
      u2 /= p.tiles_d;
      t.ks = u2 % p.ks_w;
      const int m = u2 / p.ks_w;
      const int nkb = (s.rows + 63) / 64, per = (nkb + p.ks_w - 1) / p.ks_w, k0 = t.ks * per;
      t.kind = kDw;
      t.nkb = max(0, min(per, nkb - k0));
      t.arow = m * kPairRows; t.ak = g0 + k0 * 64;                        // of G
      t.brow = tn * p.bn_d; t.bk = rc * p.row_chunk + k0 * 64;            // of Xp
      t.flags = (rc > 0 ? 1 : 0) | (rc == chunks - 1 && p.ks_w == 1 ? 2 : 0);
      t.x0 = m * kPairRows;
      t.x1 = s.v0;
      t.w1 = kMarks * (uint32_t)j;
      t.cell = ((int)(p.Np / kPairRows) * p.ks_x + m * p.ks_w + t.ks) * p.tiles_d + tn;
    }
  }
};

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void fence_async_all() {
  asm volatile("fence.proxy.async;" ::: "memory");
}
// One lane's bounded wait until *count reaches `need`.
__device__ __forceinline__ bool wait_marks(const uint32_t* count, uint32_t need,
                                           volatile int* abort_flag, int* err, int code) {
  if (need == 0 || ld_acquire(count) >= need) return true;
  const long long t0 = clock64();
  while (ld_acquire(count) < need) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kTimeoutCycles) {
      *abort_flag = 1;
      atomicOr(err, code);
      return false;
    }
    __nanosleep(32);
  }
  return true;
}
// Writes a tile into the feed of an SM of the pair; its barrier completes when all 64
// bytes are there (no fence: a release at cluster scope took most of the claim's time).
__device__ __forceinline__ void send_tile(uint32_t dst, uint32_t bar, const Tile& t) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar),
               "r"((uint32_t)sizeof(Tile))
               : "memory");
  const uint4* v = reinterpret_cast<const uint4*>(&t);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    asm volatile(
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
            dst + 16u * k),
        "r"(v[k].x), "r"(v[k].y), "r"(v[k].z), "r"(v[k].w), "r"(bar)
        : "memory");
}
static_assert(sizeof(Tile) == 64, "a feed entry");

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

// Two fp32 values in one register pair: Blackwell's packed add and multiply take one
// issue slot for both.
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
// What a pair of bf16 words leaves of (a, b), exact in fp32.
__device__ __forceinline__ void minus_word(float& a, float& b, uint32_t w) {
  a -= __uint_as_float(w << 16);
  b -= __uint_as_float(w & 0xffff0000u);
}
// The three words of a pair of fp32 values.  Values that would round to infinity are cut.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3]) {
  w[0] = pack2<__nv_bfloat16>(a, b);
  if (fmaxf(fabsf(a), fabsf(b)) >= 0x1p127f)
    w[0] = (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u);
  minus_word(a, b, w[0]);
  w[1] = pack2<__nv_bfloat16>(a, b);
  minus_word(a, b, w[1]);
  w[2] = pack2<__nv_bfloat16>(a, b);
}

// T: the type of the operand words (SPLIT: bf16); TO: the type of dW.
template <bool FWD, bool SPLIT, class T, class TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMmaThreads, 1)
xent_mma_kernel(const __grid_constant__ MmaParams p, const __grid_constant__ MmaMaps maps) {
  using Cfg = MmaCfg<SPLIT>;
  constexpr int NS = Cfg::kStages, kFeed = Cfg::kFeed;
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
    for (int b = 0; b < kFeed; ++b) {
      mbar_init(&ctl->feed_full[b], 1);
      mbar_init(&ctl->feed_empty[b], 2 * (kEpiWarps + 2) + 1);   // epilogue, loads, marks; MMA
      mbar_init(&ctl->unit_done[b], kEpiWarps);
    }
    for (int b = 0; b < 2; ++b) mbar_init(&ctl->wg_here[b], 4);
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
  if (threadIdx.x == 0) {
    for (int i = blockIdx.x; i < kErrSlots; i += gridDim.x) p.err[i] = 0;
    if (FWD && blockIdx.x == 0) *p.done = 0;
  }
  __syncthreads();
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return mbar_wait_flag(bar, parity, &ctl->abort_flag, err, code);
  };
  const uint32_t feed_empty0 = map_to_cta(smem_u32(&ctl->feed_empty[0]), 0);
  uint32_t* grad_marks = p.sync + 1;
  uint32_t* prod_marks = grad_marks + p.n_chunks * p.n_pieces;
  uint32_t* cell_marks = prod_marks + p.n_chunks * p.n_pieces;

  if (warp < 4) {
    regs_down<72>();
    // Loads and MMAs: the whole warp runs the loop, so that addresses, descriptors and
    // coordinates are warp-uniform values, and an elected lane issues.  From one lane's
    // branch, a K-block of four MMAs took 690 to 850 cycles against 512 at the full rate.
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
      return (bool)__all_sync(0xffffffffu, wait(bar, parity, code));
    };
    // Backward: tile number n of the feed; false after the last and on abort.
    auto take = [&](uint32_t n, Tile& t) {
      const uint32_t s = n % kFeed;
      if (!wait_all(&ctl->feed_full[s], (n / kFeed) & 1, 64)) return false;
      t = ctl->feed[s];
      __syncwarp();
      if (lane == 0) arrive_cluster(feed_empty0 + 8u * s);
      return t.kind >= 0;
    };
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      ForwardWalk walk(p, pair, npairs);
      Tile t;
      uint32_t it = 0;
      bool ok = true;
      const uint32_t smem0 = smem_u32(smem), full0 = map_to_cta(smem_u32(&ctl->full[0]), 0);
      for (uint32_t n = 0; ok && (FWD ? walk.next(t) : take(n, t)); ++n) {
        if (!FWD && t.kind >= kDx) {   // its G was written by other SMs' bulk stores
          const bool there = wait_marks(grad_marks + t.j, t.w0, &ctl->abort_flag, err, 128);
          if (!__all_sync(0xffffffffu, there)) { ok = false; break; }
          fence_async_all();
        }
        const bool a_mn = t.kind == kDw, b_mn = t.kind >= kDx;
        const CUtensorMap* ma = t.kind <= kGrad ? maps.X : maps.G;
        const CUtensorMap* mb = t.kind == kDw ? maps.X : maps.W;
        const bool wide = t.bn == 256;                       // two 64-row boxes of B per SM
        const int ar = t.arow + 128 * (int)rank, br = t.brow + t.bn / 2 * (int)rank;
        const uint32_t bytes = (uint32_t)(2 * Cfg::kWords * (wide ? 4 : 3) * kBoxBytes);
        // coordinates of the boxes at K-block 0, and what a K-block and a box add to them
        int ax = a_mn ? ar : t.ak, ay = a_mn ? t.ak : ar, bx = b_mn ? br : t.bk, by = b_mn ? t.bk : br;
        const int akx = a_mn ? 0 : 64, aky = 64 - akx, bkx = b_mn ? 0 : 64, bky = 64 - bkx;
        for (int kb = 0; kb < t.nkb; ++kb, ++it) {
          const uint32_t s = it % NS;
          if (it >= NS && !wait_all(&ctl->empty[s], ((it / NS) - 1) & 1, 1)) { ok = false; break; }
          const uint32_t dst = smem0 + s * Cfg::kStage, bar = full0 + 8u * s;
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], bytes);
#pragma unroll
            for (int h = 0; h < Cfg::kWords; ++h) {
              const CUtensorMap *a = ma + h, *b = mb + h;
              const uint32_t d = dst + h * (Cfg::kA + Cfg::kB);
              tma_load_pair(d, a, ax, ay, bar);
              tma_load_pair(d + kBoxBytes, a, ax + aky, ay + akx, bar);
              tma_load_pair(d + 2 * kBoxBytes, b, bx, by, bar);
              if (wide) tma_load_pair(d + 3 * kBoxBytes, b, bx + bky, by + bkx, bar);
            }
          }
          __syncwarp();
          ax += akx; ay += aky; bx += bkx; by += bky;
        }
      }
      // every stage handed back; after a timeout, time for the copies in flight to land
      for (uint32_t k = it > NS ? it - NS : 0; ok && k < it; ++k)
        ok = wait_all(&ctl->empty[k % NS], (k / NS) & 1, 2);
      if (!ok || ctl->abort_flag) idle_cycles(4000000);
    } else if (warp == 1 && rank == 0) {
      // ------------------------------------------------------------ MMA
      ForwardWalk walk(p, pair, npairs);
      Tile t;
      uint32_t it = 0, ac = 0;
      bool ok = true;
      constexpr bool f16 = std::is_same<T, __half>::value;
      const uint32_t smem0 = smem_u32(smem);
      for (uint32_t n = 0; ok && (FWD ? walk.next(t) : take(n, t)); ++n) {
        const bool a_mn = t.kind == kDw, b_mn = t.kind >= kDx;
        const uint32_t idesc = (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) |
                               (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
                               ((uint32_t)(t.bn >> 3) << 17) | (16u << 24);
        // K-major: 16 K are 32 bytes of a row; MN-major: 16 rows of 128 bytes
        const uint32_t as = a_mn ? 2048 >> 4 : 32 >> 4, bs = b_mn ? 2048 >> 4 : 32 >> 4;
        const uint32_t alo = a_mn ? (uint32_t)(kBoxBytes >> 4) << 16 : 1u << 16;
        const uint32_t blo = b_mn ? (uint32_t)(kBoxBytes >> 4) << 16 : 1u << 16;
        const int group = group_blocks<SPLIT, f16>(p, t);
        for (int k0 = 0; ok && k0 < t.nkb; k0 += group, ++ac) {
          const uint32_t d = tmem + (uint32_t)kBN * (ac & 1);
          if (ac >= 2 && !wait_all(&ctl->acc_empty[ac & 1], ((ac >> 1) - 1) & 1, 4)) { ok = false; break; }
          tc_fence_after();
          const int k1 = min(t.nkb, k0 + group);
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int s = it % NS;
            if (!wait_all(&ctl->full[s], (it / NS) & 1, 8)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a0 = (smem0 + (uint32_t)(s * Cfg::kStage)) >> 4;
            const uint32_t ad = a0 | alo, bd = (a0 + (Cfg::kA >> 4)) | blo;
            // the words of each product, from the smallest up
            constexpr uint32_t word = (Cfg::kA + Cfg::kB) >> 4;
            constexpr int kTerms = SPLIT ? 6 : 1;
            constexpr int wa[6] = {SPLIT ? 2 : 0, 0, 1, 1, 0, 0}, wb[6] = {0, 2, 1, 0, 1, 0};
            const uint32_t more = kb > k0 ? 1u : 0u;
            if (elect_one()) {
#pragma unroll
              for (int term = 0; term < kTerms; ++term) {
                const uint32_t at = ad + wa[term] * word, bt = bd + wb[term] * word;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_pair(d, at + k * as, bt + k * bs, idesc, (k > 0 || term > 0) ? 1u : more);
              }
              commit_pair(&ctl->empty[s]);
              if (kb + 1 == k1) commit_pair(&ctl->acc_full[ac & 1]);
            }
            __syncwarp();
          }
        }
      }
      // after a timeout: let what was issued finish (bounded) before TMEM is freed
      if (!ok && lane == 0) {
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                smem_u32(&ctl->drain))
            : "memory");
        const long long t0 = clock64();
        while (!mbar_try(smem_u32(&ctl->drain), 0) && clock64() - t0 < 100000000LL) {}
      }
    } else if (!FWD && warp == 2 && lane == 0) {
      // ------------------------------------------------------------ marks
      // The fence that makes a unit's stores visible to other SMs takes its time here, not
      // in the epilogue.  The feed's place is kept until the unit is done, which bounds how
      // far the epilogue can run ahead of its marks.
      for (uint32_t n = 0;; ++n) {
        const uint32_t s = n % kFeed, parity = (n / kFeed) & 1;
        if (!wait(&ctl->feed_full[s], parity, 64)) break;
        const int kind = ctl->feed[s].kind, j = ctl->feed[s].j, cell = ctl->feed[s].cell;
        if (kind < 0) break;
        if (!wait(&ctl->unit_done[s], parity, 1024)) break;
        arrive_cluster(feed_empty0 + 8u * s);
        __threadfence();
        fence_async_all();
        if (kind == kGrad) {
          atomicAdd(grad_marks + j, 1u);
        } else {
          atomicAdd(prod_marks + j, 1u);
          atomicAdd(cell_marks + cell, 1u);
        }
      }
    } else if (!FWD && warp == 3 && rank == 0 && lane == 0) {
      // ------------------------------------------------------------ claims
      BackwardList list(p);
      uint32_t claim = atomicAdd(p.sync, 1u);
      for (uint32_t n = 0;; ++n) {
        const uint32_t s = n % kFeed;
        if (n >= kFeed && !wait(&ctl->feed_empty[s], (n / kFeed - 1) & 1, 256)) break;
        Tile t = {};
        list.get((int)claim, t);
        if (t.kind >= 0) claim = atomicAdd(p.sync, 1u);   // the next, on its way meanwhile
#pragma unroll
        for (uint32_t c = 0; c < 2; ++c)
          send_tile(map_to_cta(smem_u32(&ctl->feed[s]), c),
                    map_to_cta(smem_u32(&ctl->feed_full[s]), c), t);
        if (t.kind < 0) break;
        // products are long: no others are claimed until the unit before this one is done
        if (!SPLIT && t.kind >= kDx && n > 0 &&
            !wait(&ctl->feed_empty[(n - 1) % kFeed], ((n - 1) / kFeed) & 1, 256))
          break;
      }
    }
  } else {
    regs_up<216>();
    // -------------------------------------------------------------- epilogue
    ForwardWalk walk(p, pair, npairs);
    Tile t;
    uint32_t ac = 0;
    const int q = warp & 3, wg = (warp - 4) >> 2;
    const int row_in = 128 * (int)rank + 32 * q + lane;     // row of the 256-row tile
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
    uint8_t* stage = out_stage + (warp - 4) * 4096;
    const uint32_t empty0 = map_to_cta(smem_u32(&ctl->acc_empty[0]), 0);
    constexpr bool f16 = std::is_same<T, __half>::value;
    float scale_g = 1.f, scale_back = 1.f;
    if (!FWD) {
      const Scales scales(p.amax, f16);
      scale_g = scales.g;
      scale_back = scales.back;
    }
    float m_run = -3.402823466e38f, s_run = 0.f;            // kLse, over the unit's tiles
    int target = -1;
    constexpr int kCols = 128;                              // columns per warp
    constexpr int kChunks = kCols / 32;

    auto release = [&](uint32_t a) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(empty0 + 8u * (a & 1));
    };
    // A unit is reported when its bulk stores are done: not at once, but in the middle of
    // the next unit or before anything is waited for.
    int to_report = -1;
    auto report = [&] {
      __syncwarp();
      if (to_report >= 0 && lane == 0) {
        bulk_wait_done();
        mbar_arrive(&ctl->unit_done[to_report]);
      }
      to_report = -1;
    };
    // The warp's stage is free to be written / holds data for the bulk store to come.
    auto stage_free = [&] {
      if (lane == 0) bulk_wait_read();
      __syncwarp();
    };
    auto stage_full = [&] {
      fence_async_smem();
      __syncwarp();
    };
    const uint32_t stage_at = smem_u32(stage);
    // The warpgroup's four warps.  Bounded like every other wait (a hardware barrier is
    // not): a warp that has left after a timeout does not keep the others.
    uint32_t wg_parity = 0;
    auto wg_sync = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->wg_here[wg]);
      const bool there = wait(&ctl->wg_here[wg], wg_parity, 2048);
      wg_parity ^= 1;
      return (bool)__all_sync(0xffffffffu, there);
    };
    // Marks that other SMs set once their bulk stores were done.  Behind the wait come bulk
    // stores and adds to the same memory (lane 0) and plain loads of it (all lanes): the
    // proxy fence orders the first behind lane 0's acquire, __syncwarp the second (a vote
    // orders no memory).
    auto wait_warp = [&](const uint32_t* count, uint32_t need) {
      bool there = true;
      if (lane == 0) {
        there = wait_marks(count, need, &ctl->abort_flag, err, 512);
        if (need != 0) fence_async_all();
      }
      there = __all_sync(0xffffffffu, there);
      __syncwarp();
      return there;
    };
    auto next = [&](uint32_t n) {
      if (FWD) return walk.next(t);
      const uint32_t s = n % kFeed, parity = (n / kFeed) & 1;
      if (!__all_sync(0xffffffffu, mbar_try(smem_u32(&ctl->feed_full[s]), parity))) report();
      bool there = true;
      if (lane == 0) there = wait(&ctl->feed_full[s], parity, 64);
      if (!__all_sync(0xffffffffu, there)) return false;
      t = ctl->feed[s];
      __syncwarp();
      if (lane == 0) arrive_cluster(feed_empty0 + 8u * s);
      return t.kind >= 0;
    };
    bool ok = true;
    for (uint32_t n = 0; ok && next(n); ++n) {
      const int col0 = wg * (t.bn / 2);                     // this warp's columns of the tile
      const int chunks = t.bn / 2 / 32;
      const int group = group_blocks<SPLIT, f16>(p, t);
      const int64_t row = t.arow + row_in;                  // kLse, kGrad: the live row
      if (FWD && (t.flags & 2)) {                           // first tile of the unit
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
        if (!FWD && to_report >= 0 &&
            !__all_sync(0xffffffffu, mbar_try(smem_u32(&ctl->acc_full[ac & 1]), (ac >> 1) & 1)))
          report();
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
      if (!FWD) {
        report();
        // the ring's buffer is free; the slots' tile holds the sums so far
        ok = t.kind == kGrad ? wait_warp(prod_marks + t.j - kRing, t.w0)
                             : wait_warp(cell_marks + t.cell, t.w1);
        if (!ok) break;
      }
      if (t.nkb == 0) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
      }

      if (t.kind <= kGrad) {   // products -> logits
        const int v0 = (int)t.brow + col0;
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
        // Differences first: the largest logit's term is exactly one, however large it is
        // (an FMA with the rounded m log2 e was 2^60 off at logits of 1e9), and a removed
        // entry's, or a bias of the lowest float's, exactly zero.
        const F2 l2 = f2(kLog2Ef, kLog2Ef), nm2 = f2(-mn, -mn);
        F2 s4[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s4[j & 3] = add2(s4[j & 3], exp2_pair(mul2(
                add2(f2(acc[c][2 * j], acc[c][2 * j + 1]), nm2), l2)));
        float sa, sb;
        unpack(add2(add2(s4[0], s4[1]), add2(s4[2], s4[3])), sa, sb);
        s_run += sa + sb;
        if (t.flags & 1) p.part[(int64_t)(2 * t.ks + wg) * p.Np + row] = make_float2(m_run, s_run);
        continue;
      }

      if (t.kind == kGrad) {
        const int v0 = (int)t.brow + col0;
        const float ga = rg.a * scale_g, gb = rg.b * scale_g;
        // (S - logZ) first, for the same reason: p stays at most one
        const F2 l2 = f2(kLog2Ef, kLog2Ef), ga2 = f2(ga, ga), off = f2(-rg.lse, -rg.lse);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const F2 v = f2(acc[c][2 * j], acc[c][2 * j + 1]);
            unpack(mul2(exp2_pair(mul2(add2(v, off), l2)), ga2), acc[c][2 * j], acc[c][2 * j + 1]);
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
        if (v0 + kCols > p.V || __any_sync(0xffffffffu, empty)) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (empty || v0 + 32 * c + i >= p.V) acc[c][i] = 0.f;
        }
        if (p.dbias_part) {
          // column sums of the unrounded g; the four quadrants' meet in the warpgroup's
          // stages
          if (t.flags && !wait_warp(grad_marks + t.j - kRing, t.w1)) { ok = false; break; }
          stage_free();
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = acc[c][i];
            reinterpret_cast<float*>(stage)[32 * c + lane] = column_sums(v, lane);
          }
          if (!wg_sync()) { ok = false; break; }
          const int e = (int)threadIdx.x & 127;
          const float* cs = reinterpret_cast<const float*>(out_stage + wg * 16384) + e;
          const float s = (cs[0] + cs[1 * 1024]) + (cs[2 * 1024] + cs[3 * 1024]);
          float* part = p.dbias_part + (2 * t.cell + rank) * p.Vp + t.brow + col0 + e;
          *part = t.flags ? __ldcg(part) + s : s;
          if (!wg_sync()) { ok = false; break; }
        }
        // 64 columns of words at a time are a warp's stage (SPLIT: their hi words, then
        // their mid, then their lo words)
        const int gx = t.x1 + col0, gy = t.x0 + 128 * (int)rank + 32 * q;
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
#pragma unroll
          for (int h = 0; h < Cfg::kWords; ++h) {
            stage_free();
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int e = 8 * g + 2 * i;
                float &a = acc[c + e / 32][e % 32], &b = acc[c + e / 32][e % 32 + 1];
                w[i] = pack2<T>(a, b);
                if (h + 1 < Cfg::kWords) minus_word(a, b, w[i]);
              }
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((g ^ (lane & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
            stage_full();
            if (lane == 0) tma_store(&maps.Gs[h], gx + 32 * c, gy, stage_at);
          }
        }
        to_report = (int)(n % kFeed);
        continue;
      }

      // kDx, kDw: into fp32 slots, or (the last sum of a dW tile) dW in its type
      const bool dw = t.kind == kDw, add = t.flags & 1, direct = t.flags & 2;
      const int row0 = t.x0 + 128 * (int)rank + 32 * q;
      const int slot_row = dw ? t.ks * p.piece + row0 : t.ks * (int)p.Np + row0;
      const float so = scale_back;
      const int rows_left = p.V - t.x1 - row0;                // kDw: rows of dW from row0
      const int g = lane & 7;                                 // direct: 8 lanes a row
      // the sums so far of a chunk's rows r = 4 i + lane / 8, written by other SMs: all in
      // flight at once, and the next chunk's while one is worked on
      float4 old[2][8];
      auto fetch = [&](int c, float4 (&o)[8]) {
        const float4* slot = reinterpret_cast<const float4*>(
            p.dw_slots + (int64_t)(slot_row + (lane >> 3)) * p.ldS + t.brow + col0 + 32 * c + 4 * g);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __ldcg(slot + i * p.ldS);   // 4 rows of floats
      };
      if (direct && add) fetch(0, old[0]);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (c >= chunks) break;
        const float (&v)[32] = acc[c];
        const int col = t.brow + col0 + 32 * c;
        // 32 fp32 columns = a 128-byte staged row
        stage_free();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
              make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        if (!direct) {
          stage_full();
          if (lane == 0) {
            if (add) tma_add(dw ? &maps.dws : &maps.dxs, col, slot_row, stage_at);
            else tma_store(dw ? &maps.dws : &maps.dxs, col, slot_row, stage_at);
          }
          continue;
        }
        __syncwarp();
        if (add && c + 1 < chunks) fetch(c + 1, old[(c + 1) & 1]);
        const int at = col + 4 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + (lane >> 3);
          float4 x = *reinterpret_cast<const float4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
          if (add) {
            const float4 o = old[c & 1][i];
            x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w;
          }
          if (!p.dw_vec) {   // rows of dW start anywhere: stored below
            *reinterpret_cast<float4*>(stage + r * 128 + ((g ^ (r & 7)) << 4)) = x;
          } else if (r < rows_left && at < p.D) {
            TO* dst = static_cast<TO*>(p.dW) + (int64_t)(t.x1 + row0 + r) * p.D + at;
            TO y[4] = {from_f32<TO>(x.x * so), from_f32<TO>(x.y * so), from_f32<TO>(x.z * so),
                       from_f32<TO>(x.w * so)};
            if (sizeof(TO) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(y);
            else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(y);
          }
        }
        if (!p.dw_vec) {     // lane = column
          __syncwarp();
          TO* dst = static_cast<TO*>(p.dW) + (int64_t)(t.x1 + row0) * p.D + col + lane;
          if (col + lane < p.D) {
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
              if (r >= rows_left) break;
              const float x = *reinterpret_cast<const float*>(
                  stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3));
              dst[(int64_t)r * p.D] = from_f32<TO>(x * so);
            }
          }
        }
        __syncwarp();
      }
      to_report = (int)(n % kFeed);
    }
    if (!FWD) report();
    if (lane == 0) bulk_wait_done();
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
