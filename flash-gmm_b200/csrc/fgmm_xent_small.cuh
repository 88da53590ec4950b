// The linear cross entropy of a few fp32 rows (included by fgmm_xent.cu): up to 16, as
// when single tokens are scored.  Such a batch is bound by reading W; on the tensor cores
// an fp32 W would first be read for its scale, and read and written as two words.  These
// kernels read it in place, whatever its strides, and multiply in fp32.  So does one 16-bit
// row whose W TMA cannot read.  (Other 16-bit rows keep the tensor-core tile: it reads W
// once, in place, at four rows of 131072 x 4096 in 243 us where these kernels took 618, with
// fewer bytes in flight per thread.)
//
//   small_logits_kernel   S = X W^T: a warp takes R rows of W at a time, its lanes along D,
//                         and keeps R x NB sums; forward they are folded into running
//                         (max, sum) pairs, backward they become g, stored as [V][NB]
//   small_products_kernel dW = g^T X and the parts of dX = g W over ranges of the
//                         vocabulary, in one pass over W
//
// Bytes: W once forward; backward W twice and dW once.

constexpr int kSmallWarps = 8;

// How rows are read: any strides, unit stride, or 16 bytes at a time.
enum SmallMode { kAnyStride = 0, kUnitStride = 1, kVector = 2 };

// A lane's four elements of the 128 from d on: consecutive (kVector, where D is a
// multiple of 4) or 32 apart.
template <class T, int MODE>
__device__ __forceinline__ void small_load(const T* row, int64_t s1, int d, int lane, int D,
                                           float (&v)[4]) {
  if constexpr (MODE == kVector) {
    Pack<T, 4> x;
    if (d + 4 * lane < D) {
      x.load(row + d + 4 * lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f32(x.v[i]);
    } else {
      v[0] = v[1] = v[2] = v[3] = 0.f;
    }
  } else if (MODE == kUnitStride && d + 128 <= D) {
    const T* p = row + d + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f32(p[32 * i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = d + 32 * i + lane;
      v[i] = at < D ? to_f32(row[at * s1]) : 0.f;
    }
  }
}

template <class T, int NB, int R, int MODE, bool GRAD>
__global__ void __launch_bounds__(32 * kSmallWarps, 2)
small_logits_kernel(const XentArgs a, const XentWs w, const SmallPlan plan) {
  pdl_trigger();
  constexpr int kSums = R * NB, kBatches = (kSums + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (!GRAD) {
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < kErrSlots; i += 32 * kSmallWarps) w.hdr->err[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) w.hdr->done = 0;
  }
  const T* X = static_cast<const T*>(a.X);
  const T* W = static_cast<const T*>(a.W);
  // this lane's sums after the reduction: number 32 q + lane = r NB + n
  int my_r[kBatches], my_n[kBatches], target[kBatches];
  float m[kBatches], s[kBatches], wa[kBatches], wb[kBatches], lse[kBatches];
#pragma unroll
  for (int q = 0; q < kBatches; ++q) {
    const int c = 32 * q + lane;
    my_r[q] = c / NB;
    my_n[q] = c % NB;
    m[q] = -3.402823466e38f;
    s[q] = 0.f;
    target[q] = -1;
    wa[q] = wb[q] = lse[q] = 0.f;
    const int64_t n = my_n[q];
    if (n < a.N && a.targets[n] != a.ignore) {
      const int64_t t = a.targets[n];
      target[q] = t >= 0 && t < a.V ? (int)t : kBadTarget;
      if (GRAD) {
        const float inv = a.count_in ? 1.f / *a.count_in : 1.f;
        wb[q] = a.dloss ? a.dloss[n * a.dloss_stride] * inv : 0.f;
        wa[q] = wb[q] + (a.dlogZ ? a.dlogZ[n] : 0.f);
        lse[q] = a.logZ_in[n];
        if (target[q] < 0) wa[q] = __int_as_float(0x7fffffff);
      }
    }
  }
  const int64_t step = (int64_t)gridDim.x * kSmallWarps * R;
  for (int64_t v0 = ((int64_t)blockIdx.x * kSmallWarps + warp) * R; v0 < a.V; v0 += step) {
    float acc[kBatches * 32];
#pragma unroll
    for (int c = 0; c < kBatches * 32; ++c) acc[c] = 0.f;
    // (the next step's loads issued ahead cost more warps than they hid: 131072 x 2048, four
    // rows, 274 -> 395 us)
    for (int d = 0; d < a.D; d += 128) {
      float wv[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r)   // past the last entry: the last again, not used
        small_load<T, MODE>(W + min(v0 + r, (int64_t)a.V - 1) * a.swv, a.swd, d, lane, a.D, wv[r]);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float x[4];   // an ignored row spoils no sums but its own, which nobody reads
        small_load<T, MODE>(X + min((int64_t)n, a.N - 1) * a.sxn, a.sxd, d, lane, a.D, x);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r * NB + n] = fmaf(wv[r][i], x[i], acc[r * NB + n]);
        // at most four rows' loads at once: more spill
        if ((n & 3) == 3) asm volatile("" ::: "memory");
      }
    }
#pragma unroll
    for (int q = 0; q < kBatches; ++q) {
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = acc[32 * q + i];
      float x = column_sums(v, lane);
      const int64_t e = v0 + my_r[q];
      const bool there = 32 * q + lane < kSums && e < a.V;
      if (there && a.bias) x += a.bias[e];
      if (!GRAD) {
        if (there && target[q] != -1) {
          if (e == target[q]) w.tlogit[my_n[q]] = x;
          const float mn = fmaxf(m[q], x);
          s[q] = s[q] * ex2((m[q] - mn) * kLog2Ef) + ex2((x - mn) * kLog2Ef);
          m[q] = mn;
        }
      } else {
        float g = 0.f;
        if (there && target[q] != -1 && !(wa[q] == 0.f && wb[q] == 0.f)) {
          g = wa[q] * ex2((x - lse[q]) * kLog2Ef);
          if (e == target[q]) g -= wb[q];
        }
        if (there) w.small_g[e * NB + my_n[q]] = g;
        if (a.dbias) {
          float sum = g;     // over the NB lanes of the entry
          if constexpr (NB > 1) {
#pragma unroll
            for (int o = NB / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          }
          if (there && my_n[q] == 0) a.dbias[e] = sum;
        }
      }
    }
  }
  if constexpr (!GRAD) {
  // the block's part of each row: the warps' R pairs each, in order
  __shared__ float sm[kSmallWarps][kBatches * 32], ss[kSmallWarps][kBatches * 32];
#pragma unroll
  for (int q = 0; q < kBatches; ++q) {
    sm[warp][32 * q + lane] = m[q];
    ss[warp][32 * q + lane] = s[q];
  }
  __syncthreads();
  if (threadIdx.x < NB) {
    float mm = -3.402823466e38f, sum = 0.f;
    for (int k = 0; k < kSmallWarps * R; ++k) mm = fmaxf(mm, sm[k / R][(k % R) * NB + threadIdx.x]);
    for (int k = 0; k < kSmallWarps * R; ++k)
      sum += ss[k / R][(k % R) * NB + threadIdx.x] *
             ex2((sm[k / R][(k % R) * NB + threadIdx.x] - mm) * kLog2Ef);
    w.part[(int64_t)blockIdx.x * w.Np + threadIdx.x] = make_float2(mm, sum);
  }
  }
}

// Columns of the block (4 a thread) of the vocabulary's range blockIdx.y: x stays in
// registers for dW, the sums of dX leave as one part.
template <class T, int NB, int MODE>
__global__ void __launch_bounds__(128)
small_products_kernel(const XentArgs a, const XentWs w, const SmallPlan plan) {
  pdl_trigger();
  pdl_wait();
  constexpr int kStage = 64;      // entries whose g is staged
  __shared__ __align__(16) float sg[kStage * NB];
  const T* X = static_cast<const T*>(a.X);
  const T* W = static_cast<const T*>(a.W);
  const int col0 = blockIdx.x * kSmallCols;
  constexpr bool VEC = MODE == kVector;
  auto col = [&](int i) { return col0 + (VEC ? 4 * (int)threadIdx.x + i : 128 * i + (int)threadIdx.x); };
  int64_t off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) off[i] = MODE == kAnyStride ? col(i) * a.swd : (int64_t)col(i);
  float x[NB][4], acc[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const bool live = n < a.N && a.targets[n] != a.ignore;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[n][i] = live && col(i) < a.D ? to_f32(X[n * a.sxn + col(i) * a.sxd]) : 0.f;
      acc[n][i] = 0.f;
    }
  }
  const int64_t v_begin = (int64_t)blockIdx.y * plan.per_split;
  const int64_t v_end = min(v_begin + plan.per_split, (int64_t)a.V);
  constexpr int U = 8;            // entries in flight
  for (int64_t v0 = v_begin; v0 < v_end; v0 += kStage) {
    const int count = (int)min((int64_t)kStage, v_end - v0);
    __syncthreads();
    for (int i = threadIdx.x; i < kStage * NB; i += 128)
      sg[i] = i < count * NB ? w.small_g[v0 * NB + i] : 0.f;
    __syncthreads();
    for (int e0 = 0; e0 < count; e0 += U) {
      float wv[U][4];
      if (a.dX) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const T* r = W + min(v0 + e0 + u, v_end - 1) * a.swv;
          if (VEC) {
            if (col(0) < a.D) {
              Pack<T, 4> p;
              p.load(r + col(0));
#pragma unroll
              for (int i = 0; i < 4; ++i) wv[u][i] = to_f32(p.v[i]);
            } else {
              wv[u][0] = wv[u][1] = wv[u][2] = wv[u][3] = 0.f;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) wv[u][i] = col(i) < a.D ? to_f32(r[off[i]]) : 0.f;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (e0 + u >= count) break;
        float out[4] = {0.f, 0.f, 0.f, 0.f}, gs[NB];
        if constexpr (NB % 4 == 0) {
#pragma unroll
          for (int n = 0; n < NB; n += 4)
            *reinterpret_cast<float4*>(gs + n) = *reinterpret_cast<const float4*>(sg + (e0 + u) * NB + n);
        } else {
          gs[0] = sg[e0 + u];
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const float g = gs[n];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            out[i] = fmaf(g, x[n][i], out[i]);
            if (a.dX) acc[n][i] = fmaf(g, wv[u][i], acc[n][i]);
          }
        }
        if (a.dW) {
          T* dst = static_cast<T*>(a.dW) + (v0 + e0 + u) * a.D;
          if (VEC) {
            if (col(0) < a.D) {
              Pack<T, 4> p;
#pragma unroll
              for (int i = 0; i < 4; ++i) p.v[i] = from_f32<T>(out[i]);
              p.store(dst + col(0));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (col(i) < a.D) dst[col(i)] = from_f32<T>(out[i]);
          }
        }
      }
    }
  }
  if (a.dX) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n < a.N && col(i) < a.D)
          w.small_dx[((int64_t)blockIdx.y * NB + n) * a.D + col(i)] = acc[n][i];
  }
}

// dX[n, d] = sum of its parts, in order; ignored rows are zero.  8 warps take the
// parts of 32 elements in turn.
template <class T>
__global__ void __launch_bounds__(256)
small_finish_kernel(const XentArgs a, const XentWs w, const SmallPlan plan) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t e = blockIdx.x * 32ll + lane, total = a.N * a.D;
  float s = 0.f;
  if (e < total)
#pragma unroll 8
    for (int k = warp; k < plan.splits; k += 8) s += w.small_dx[(int64_t)k * plan.nb * a.D + e];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && e < total) {
    s = red[0][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][lane];
    const bool live = a.targets[e / a.D] != a.ignore;
    static_cast<T*>(a.dX)[e] = from_f32<T>(live ? s : 0.f);
  }
}
