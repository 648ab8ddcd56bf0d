// Layer norm over rows, forward and backward.
//
//   mean = sum x / N, rstd = 1 / sqrt(sum (x - mean)^2 / N + eps), h = (x - mean) rstd, y = h w + b
//   g = dy w, dx = rstd (g - sum g / N - h sum(g h) / N), dw = sum over rows of dy h, db = sum over rows of dy
//
// Everything is bound by memory: a row is read once into registers (a warp's or a block's), and all that is done to it
// happens there, the variance as a second pass over the registers.  The backward keeps its columns' sums for dw and db in
// registers from row to row; each block writes them once and a small kernel adds the blocks' sums in their order.  With 768 features
// of 16 bits instruction issue was the bound (82 and 72 %) until two values went through an instruction: 65536 rows forward 35 us = 5.7 TB/s,
// backward 52 us = 5.8 TB/s, 0.9 of what a copy reaches; rows of 768 in fp32 forward 64 us = 6.3 TB/s.
#include "lik_layers.cuh"

namespace lik {
namespace {

struct NormParams {
  const void* x;
  long long x_stride, rows;
  int width;
  const void *w, *b;
  float eps;
  void* y;
  float *mean, *rstd;
  const void* dy;
  void* dx;
  float* partial;  // [blocks][2][width]
};

constexpr int NORM_THREADS = 256;

// Sums of one or two numbers over the threads of a row: a warp, or several, which meet at a barrier of their own.  Of two numbers the lower lanes go on
// with the first and the upper ones with the second after the first exchange: five exchanges, or six with the way back, instead of ten.
struct RowBuf {
  float4 sum[2][2][NORM_THREADS / 128];  // [turn][which sum], a float per warp
};
template <int TPR, bool TWO>
__device__ __forceinline__ float2 row_sum(float a, float b, RowBuf& buf, int& turn) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = threadIdx.x / TPR;
  if constexpr (TWO) {
    const bool up = lane & 16;
    a = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
  } else {
    a += __shfl_xor_sync(0xffffffffu, a, 16);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if constexpr (TPR == 32) {
    if constexpr (!TWO) return make_float2(a, 0.0f);
    b = __shfl_xor_sync(0xffffffffu, a, 16);
    return lane & 16 ? make_float2(b, a) : make_float2(a, b);
  } else {
    static_assert(NORM_THREADS / TPR <= 2, "a barrier per row");
    // two buffers in turn: nobody is more than one barrier ahead of who still reads
    turn ^= 1;
    if (TWO ? lane % 16 == 0 : lane == 0) reinterpret_cast<float*>(buf.sum[turn][lane / 16])[warp] = a;
    if (TPR == NORM_THREADS) __syncthreads();
    else if (group == 0) asm volatile("bar.sync 1, %0;" ::"n"(TPR) : "memory");  // (a number in a register would reserve all sixteen barriers)
    else asm volatile("bar.sync 2, %0;" ::"n"(TPR) : "memory");
    auto add_up = [&](const float4* f) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < TPR / 128; ++w) s = (((s + f[w].x) + f[w].y) + f[w].z) + f[w].w;
      return s;
    };
    return make_float2(add_up(&buf.sum[turn][0][group * (TPR / 128)]), TWO ? add_up(&buf.sum[turn][1][group * (TPR / 128)]) : 0.0f);
  }
}

// a vector of V elements as it came from memory
template <typename T, int V>
struct RawVec {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
    } else {
      unpack2(u.x, f[0], f[1], T());
      unpack2(u.y, f[2], f[3], T());
      unpack2(u.z, f[4], f[5], T());
      unpack2(u.w, f[6], f[7], T());
    }
  }
};
template <typename T>
struct RawVec<T, 1> {
  T e;
  __device__ __forceinline__ void load(const T* p) { e = *p; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f32(e); }
};

// A row's statistics from the sums of the differences' squares and of the differences from its mean.  That mean is rounded - a step of a value far
// from zero may be more than the row's deviation, and 1 / N is rounded too - but the differences are all but exact, so their own mean says by how
// much it is off: a row of one value comes out as zeros, and one around 1e4 as exact as one around 0.  (What is within a rounding of the
// deviation is itself the rounding of these sums, and is left alone.)
struct NormStats {
  float off, rstd;
  __device__ __forceinline__ NormStats(float2 sums, float inv_n, float eps) : off(sums.y * inv_n) {
    float var = fmaf(-off, off, sums.x * inv_n);
    var = (var < 0.0f ? 0.0f : var) + eps;  // (a NaN stays one)
    if (!(off * off > 1.4210854715202004e-14f * var)) off = 0.0f;
    rstd = 1.0f / sqrtf(var);
  }
};

template <typename T, typename P, int V, int NV, int TPR>
__global__ void __launch_bounds__(NORM_THREADS) norm_fwd_kernel(const NormParams p) {
  __shared__ RowBuf buf;
  after_the_kernel_in_front();
  int turn = 0;
  constexpr int PER_BLOCK = NORM_THREADS / TPR;
  const int lane = threadIdx.x % TPR;
  const float inv_n = 1.0f / (float)p.width;
  RawVec<T, V> raw[NV];
  auto fetch = [&](long long r) {  // the next row, while the present one is dealt with
    if (r >= p.rows) return;
    const T* x = (const T*)p.x + r * p.x_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c < p.width) raw[i].load(x + c);
    }
  };
  const long long step = (long long)gridDim.x * PER_BLOCK;
  long long r = (long long)blockIdx.x * PER_BLOCK + threadIdx.x / TPR;
  fetch(r);
  for (; r < p.rows; r += step) {
    float v[NV][V];
    PairSum s, t, q;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * TPR + lane) * V < p.width) {
        raw[i].get(v[i]);
        s.add(v[i]);
      }
    fetch(r + step);
    const float mean = row_sum<TPR, false>(s.sum(), 0.0f, buf, turn).x * inv_n;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * TPR + lane) * V < p.width) {
        vec_add(v[i], -mean);
        t.add(v[i]);
        q.dot(v[i], v[i]);
      }
    const NormStats st(row_sum<TPR, true>(q.sum(), t.sum(), buf, turn), inv_n, p.eps);
    if (lane == 0 && p.mean) {
      p.mean[r] = mean + st.off;
      p.rstd[r] = st.rstd;
    }
    T* y = (T*)p.y + r * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c < p.width) {
        float w[V], b[V];
        vec_fma(v[i], st.rstd, -st.off * st.rstd);
        if (p.w) {
          load_vec<P, V>((const P*)p.w + c, w);
          if (p.b) {
            load_vec<P, V>((const P*)p.b + c, b);
            vec_fma(v[i], w, b);
          } else {
            vec_mul(v[i], w);
          }
        } else if (p.b) {
          load_vec<P, V>((const P*)p.b + c, b);
          vec_add(v[i], b);
        }
        store_vec<T, V>(y + c, v[i]);
      }
    }
  }
}

// (blocks of four warps where a warp has its row to itself: three of them, at up to 168 registers a thread, where eight warps at a time would leave
// an SM one block or spill)
__host__ __device__ constexpr int norm_bwd_threads(int tpr) { return tpr == 32 ? 128 : NORM_THREADS; }
// The next row is fetched while the present one is reduced and written; both stay as they came from memory, since two rows and the columns'
// sums in fp32 would leave an SM one block.
template <typename T, typename P, int V, int NV, int TPR, bool PARAMS>
__global__ void __launch_bounds__(norm_bwd_threads(TPR), TPR == 32 ? 3 : (NV * V <= 24 ? 2 : 1)) norm_bwd_kernel(const NormParams p) {
  __shared__ RowBuf buf;
  after_the_kernel_in_front();
  int turn = 0;
  constexpr int THREADS = norm_bwd_threads(TPR), PER_BLOCK = THREADS / TPR;
  const int lane = threadIdx.x % TPR;
  const float inv_n = 1.0f / (float)p.width;
  float dw[PARAMS ? NV : 1][V], db[PARAMS ? NV : 1][V];
#pragma unroll
  for (int i = 0; i < (PARAMS ? NV : 1); ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
  RawVec<T, V> rx[NV], rg[NV];
  float mean = 0.0f, rstd = 0.0f;
  auto fetch = [&](long long r) {
    if (r >= p.rows) return;
    const T* x = (const T*)p.x + r * p.x_stride;
    const T* dy = (const T*)p.dy + r * p.width;
    mean = p.mean[r];
    rstd = p.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c < p.width) {
        rx[i].load(x + c);
        rg[i].load(dy + c);
      }
    }
  };
  const long long step = (long long)gridDim.x * PER_BLOCK;
  long long r = (long long)blockIdx.x * PER_BLOCK + threadIdx.x / TPR;
  fetch(r);
  for (; r < p.rows; r += step) {
    RawVec<T, V> x[NV], y[NV];
    const float m = mean, s = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = rx[i], y[i] = rg[i];
    fetch(r + step);
    PairSum sg, sgh;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c < p.width) {
        float w[V], h[V], g[V];
        x[i].get(h);
        y[i].get(g);
        vec_add(h, -m);
        vec_mul(h, s);
        if constexpr (PARAMS) {
#pragma unroll
          for (int j = 0; j < V; j += V == 1 ? 1 : 2) {
            if constexpr (V == 1) dw[i][0] = fmaf(g[0], h[0], dw[i][0]);
            else fma2(Pair(g[j], g[j + 1]), Pair(h[j], h[j + 1]), Pair(dw[i][j], dw[i][j + 1])).get(dw[i][j], dw[i][j + 1]);
          }
          vec_add(db[i], g);
        }
        if (p.w) {
          load_vec<P, V>((const P*)p.w + c, w);
          vec_mul(g, w);
        }
        sg.add(g);
        sgh.dot(g, h);
      }
    }
    if (p.dx) {
      const float2 sums = row_sum<TPR, true>(sg.sum(), sgh.sum(), buf, turn);
      // rstd (g - c1 - h c2), h = (x - mean) rstd
      const float c1 = -sums.x * inv_n, c2 = -sums.y * inv_n * s;
      T* dx = (T*)p.dx + r * p.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V;
        if (c < p.width) {
          float w[V], h[V], g[V];
          x[i].get(h);
          y[i].get(g);
          vec_add(h, -m);
          vec_fma(h, c2, c1);
          if (p.w) {
            load_vec<P, V>((const P*)p.w + c, w);
            vec_fma(g, w, h);
          } else {
            vec_add(g, h);
          }
          vec_mul(g, s);
          store_vec<T, V>(dx + c, g);
        }
      }
    }
  }
  if constexpr (PARAMS) {
    float* out = p.partial + (long long)blockIdx.x * 2 * p.width;
    if constexpr (TPR == NORM_THREADS) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V;
        if (c < p.width)
#pragma unroll
          for (int j = 0; j < V; ++j) out[c + j] = dw[i][j], out[p.width + c + j] = db[i][j];
      }
    } else {
      // the block's warps in their order, each adding to what is in shared memory
      extern __shared__ float acc[];  // [2][NV * TPR * V]
      constexpr int COLS = NV * TPR * V;
      for (int w = 0; w < PER_BLOCK; ++w) {
        if (threadIdx.x / TPR == w) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int c = (i * V + j) * TPR + lane;  // (one bank per lane)
              acc[c] = w ? acc[c] + dw[i][j] : dw[i][j];
              acc[COLS + c] = w ? acc[COLS + c] + db[i][j] : db[i][j];
            }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < COLS; c += THREADS) {
        // (i, lane, j) of a column
        const int i = c / (TPR * V), l = c / V % TPR, j = c % V, at = (i * V + j) * TPR + l;
        if (c < p.width) out[c] = acc[at], out[p.width + c] = acc[COLS + at];
      }
    }
  }
}

// Rows that no block holds in registers: a block goes through its row three times, the later ones out of L2.
template <typename T, typename P>
__global__ void __launch_bounds__(NORM_THREADS) norm_fwd_wide_kernel(const NormParams p) {
  __shared__ RowBuf buf;
  after_the_kernel_in_front();
  int turn = 0;
  const float inv_n = 1.0f / (float)p.width;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = (const T*)p.x + r * p.x_stride;
    float s = 0.0f, t = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += NORM_THREADS) s += to_f32(x[c]);
    const float mean = row_sum<NORM_THREADS, false>(s, 0.0f, buf, turn).x * inv_n;
    for (int c = threadIdx.x; c < p.width; c += NORM_THREADS) {
      const float d = to_f32(x[c]) - mean;
      t += d;
      q = fmaf(d, d, q);
    }
    const NormStats st(row_sum<NORM_THREADS, true>(q, t, buf, turn), inv_n, p.eps);
    if (threadIdx.x == 0 && p.mean) p.mean[r] = mean + st.off, p.rstd[r] = st.rstd;
    for (int c = threadIdx.x; c < p.width; c += NORM_THREADS)
      ((T*)p.y)[r * p.width + c] =
          from_f32<T>(fmaf((to_f32(x[c]) - mean - st.off) * st.rstd, p.w ? to_f32(((const P*)p.w)[c]) : 1.0f, p.b ? to_f32(((const P*)p.b)[c]) : 0.0f));
  }
}
template <typename T, typename P>
__global__ void __launch_bounds__(NORM_THREADS) norm_dx_wide_kernel(const NormParams p) {
  __shared__ RowBuf buf;
  after_the_kernel_in_front();
  int turn = 0;
  const float inv_n = 1.0f / (float)p.width;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T *x = (const T*)p.x + r * p.x_stride, *dy = (const T*)p.dy + r * p.width;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float s = 0.0f, t = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += NORM_THREADS) {
      const float g = to_f32(dy[c]) * (p.w ? to_f32(((const P*)p.w)[c]) : 1.0f);
      s += g;
      t = fmaf(g, (to_f32(x[c]) - mean) * rstd, t);
    }
    const float2 m = row_sum<NORM_THREADS, true>(s, t, buf, turn);
    const float c1 = m.x * inv_n, c2 = m.y * inv_n;
    for (int c = threadIdx.x; c < p.width; c += NORM_THREADS) {
      const float g = to_f32(dy[c]) * (p.w ? to_f32(((const P*)p.w)[c]) : 1.0f);
      ((T*)p.dx)[r * p.width + c] = from_f32<T>(rstd * (g - c1 - (to_f32(x[c]) - mean) * rstd * c2));
    }
  }
}
// a thread's column over every gridDim.y-th row
template <typename T>
__global__ void __launch_bounds__(NORM_THREADS) norm_dparam_wide_kernel(const NormParams p) {
  after_the_kernel_in_front();
  const int c = blockIdx.x * NORM_THREADS + threadIdx.x;
  if (c >= p.width) return;
  float dw = 0.0f, db = 0.0f;
  for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
    const float g = to_f32(((const T*)p.dy)[r * p.width + c]);
    dw = fmaf(g, (to_f32(((const T*)p.x)[r * p.x_stride + c]) - p.mean[r]) * p.rstd[r], dw);
    db += g;
  }
  float* out = p.partial + (long long)blockIdx.y * 2 * p.width;
  out[c] = dw;
  out[p.width + c] = db;
}

constexpr int NORM_WIDE_PARTS = 64;

// Which kernel a width goes to: a warp per row, four warps or the block's eight; vectors of 16 bytes where rows and parameters are aligned, else
// single elements (9001 x 1023 fp32: forward 16 us by four warps per row, 20 by a block; backward 23 by a block, 58 by a warp with 32 elements per lane).  The
// forward keeps a row with a warp up to 1024 features (65536 x 768 fp32: 64 us; 110 by a block per row, of which each warp adds the row's sums up
// for itself), the backward, which holds a row twice and its columns' sums, up to three vectors per lane: 65536 x 768 bf16 52 us, 102 with four warps per row, of which the fourth has nothing; 16384 x 1024 36 us with a warp per row, 24 with four.
struct NormPlan {
  bool wide, vec;
  int nv, tpr;
};
NormPlan norm_plan(const lik_norm_args& a, bool bwd) {
  const int item = (int)dtype_size(a.dtype), v = 16 / item;
  NormPlan pl{};
  pl.vec = vec_ok(a.x, a.x_stride, a.width, item) && vec_ok(a.y, a.width, a.width, item) && vec_ok(a.dy, a.width, a.width, item) &&
           vec_ok(a.dx, a.width, a.width, item) && ((uintptr_t)a.weight & 15) == 0 && ((uintptr_t)a.bias & 15) == 0;
  const long long vecs = ceil_div(a.width, pl.vec ? v : 1);
  if (pl.vec) {
    pl.tpr = vecs <= (bwd ? 96 : 1024 / v) ? 32 : (vecs <= 128 ? 128 : 256);
    pl.nv = (int)ceil_div(vecs, pl.tpr);
    if (pl.tpr == 256 && pl.nv == 3) pl.nv = 4;
    if (pl.tpr == 32 && pl.nv > 4) pl.nv = (pl.nv + 1) / 2 * 2;
    pl.wide = pl.tpr == 256 && pl.nv > 4;
  } else {
    pl.tpr = vecs <= 256 ? 32 : (!bwd && vecs <= 1024 ? 128 : 256);
    const long long need = ceil_div(vecs, pl.tpr);
    pl.nv = need == 1 && pl.tpr == 32 ? 1 : (need <= 4 ? 4 : (need <= 8 ? 8 : 16));
    pl.wide = need > 16;
  }
  return pl;
}
int norm_bwd_blocks(const lik_norm_args& a, const NormPlan& pl) {
  if (pl.wide) return (int)(a.rows < NORM_WIDE_PARTS ? (a.rows ? a.rows : 1) : NORM_WIDE_PARTS);
  const long long need = ceil_div(a.rows, norm_bwd_threads(pl.tpr) / pl.tpr), most = (pl.tpr == 32 || (pl.tpr == 256 && pl.nv <= (pl.vec ? 1 : 4)) ? 3ll : 2ll) * sm_count();  // (what an SM holds)
  return (int)(need < most ? (need ? need : 1) : most);
}

template <typename T, typename P, int V, int NV, int TPR>
int run_norm(const NormParams& p, bool bwd, bool params, int blocks, cudaStream_t st) {
  if (!bwd) {
    if constexpr (V == 1 || (TPR != 128 && (TPR != 32 || NV * V <= 32))) return launch_after(norm_fwd_kernel<T, P, V, NV, TPR>, blocks, NORM_THREADS, 0, st, 1, p);
  } else if constexpr (V == 1 ? TPR != 128 : TPR != 32 || NV <= 3) {
    const size_t smem = TPR < NORM_THREADS ? sizeof(float) * 2 * NV * TPR * V : 0;
    return params ? launch_after(norm_bwd_kernel<T, P, V, NV, TPR, true>, blocks, norm_bwd_threads(TPR), smem, st, 1, p)
                  : launch_after(norm_bwd_kernel<T, P, V, NV, TPR, false>, blocks, norm_bwd_threads(TPR), 0, st, 1, p);
  }
  return LIK_ERR_UNSUPPORTED;  // (a shape that the plan does not give)
}
template <typename T, typename P>
int run_norm(const NormPlan& pl, const NormParams& p, bool bwd, bool params, int blocks, cudaStream_t st) {
  constexpr int V = vec_elems<T>();
  if (pl.wide) {
    if (!bwd) return launch_after(norm_fwd_wide_kernel<T, P>, blocks, NORM_THREADS, 0, st, 1, p);
    if (p.dx)
      if (int rc = launch_after(norm_dx_wide_kernel<T, P>, (unsigned)(p.rows < 8ll * sm_count() ? p.rows : 8ll * sm_count()), NORM_THREADS, 0, st, 1, p)) return rc;
    return params ? launch_after(norm_dparam_wide_kernel<T>, dim3((unsigned)ceil_div(p.width, NORM_THREADS), blocks), NORM_THREADS, 0, st, 1, p) : LIK_OK;
  }
#define LIK_NORM_CASE(VV, NN, TT) \
  if ((pl.vec ? V : 1) == VV && pl.nv == NN && pl.tpr == TT) return run_norm<T, P, VV, NN, TT>(p, bwd, params, blocks, st)
  LIK_NORM_CASE(V, 1, 32);
  LIK_NORM_CASE(V, 2, 32);
  LIK_NORM_CASE(V, 3, 32);
  LIK_NORM_CASE(V, 4, 32);
  LIK_NORM_CASE(V, 6, 32);
  LIK_NORM_CASE(V, 8, 32);
  LIK_NORM_CASE(V, 1, 128);
  LIK_NORM_CASE(V, 1, 256);
  LIK_NORM_CASE(V, 2, 256);
  LIK_NORM_CASE(V, 4, 256);
  LIK_NORM_CASE(1, 1, 32);
  LIK_NORM_CASE(1, 4, 32);
  LIK_NORM_CASE(1, 8, 32);
  LIK_NORM_CASE(1, 4, 128);
  LIK_NORM_CASE(1, 8, 128);
  LIK_NORM_CASE(1, 4, 256);
  LIK_NORM_CASE(1, 8, 256);
  LIK_NORM_CASE(1, 16, 256);
#undef LIK_NORM_CASE
  set_error("layer norm: no kernel for width %d", p.width);
  return LIK_ERR_UNSUPPORTED;
}
int run_norm(const lik_norm_args& a, const NormPlan& pl, const NormParams& p, bool bwd, bool params, int blocks, cudaStream_t st) {
  if (a.dtype == LIK_F32) return run_norm<float, float>(pl, p, bwd, params, blocks, st);
  if (a.dtype == LIK_F16)
    return a.param_dtype == LIK_F32 ? run_norm<__half, float>(pl, p, bwd, params, blocks, st) : run_norm<__half, __half>(pl, p, bwd, params, blocks, st);
  return a.param_dtype == LIK_F32 ? run_norm<__nv_bfloat16, float>(pl, p, bwd, params, blocks, st)
                                  : run_norm<__nv_bfloat16, __nv_bfloat16>(pl, p, bwd, params, blocks, st);
}
NormParams norm_params(const lik_norm_args& a) {
  return NormParams{a.x, a.x_stride, a.rows, a.width, a.weight, a.bias, a.eps, a.y, a.mean, a.rstd, a.dy, a.dx, nullptr};
}
int check_norm(const lik_norm_args* a) {
  LIK_REQUIRE(a != nullptr, "args is NULL");
  LIK_REQUIRE(a->dtype == LIK_F32 || a->dtype == LIK_F16 || a->dtype == LIK_BF16, "dtype must be fp32, fp16 or bf16");
  LIK_REQUIRE(a->param_dtype == a->dtype || a->param_dtype == LIK_F32, "param_dtype must be dtype or fp32");
  LIK_REQUIRE(a->rows >= 0 && a->width > 0 && a->width < (1 << 30) && a->x_stride >= a->width, "sizes must be positive, width below 2^30, x_stride at least width");
  LIK_REQUIRE(a->eps >= 0.0f, "eps must not be negative");
  return LIK_OK;
}

}  // namespace
}  // namespace lik

extern "C" int lik_layer_norm_fwd(const lik_norm_args* args, lik_stream_t stream) {
  using namespace lik;
  if (int rc = check_norm(args)) return rc;
  const lik_norm_args& a = *args;
  if (a.rows == 0) return LIK_OK;
  LIK_REQUIRE(a.x && a.y && !a.mean == !a.rstd, "x and y must not be NULL; mean and rstd go together");
  const NormPlan pl = norm_plan(a, false);
  const long long need = ceil_div(a.rows, pl.wide ? 1 : NORM_THREADS / pl.tpr), most = 8ll * sm_count();
  return run_norm(a, pl, norm_params(a), false, false, (int)(need < most ? need : most), (cudaStream_t)stream);
}

extern "C" size_t lik_layer_norm_bwd_workspace(const lik_norm_args* a) {
  using namespace lik;
  if (check_norm(a) || a->rows == 0 || (!a->dweight && !a->dbias)) return 0;
  return (size_t)norm_bwd_blocks(*a, norm_plan(*a, true)) * 2 * a->width * sizeof(float);
}

extern "C" int lik_layer_norm_bwd(const lik_norm_args* args, lik_stream_t stream) {
  using namespace lik;
  if (int rc = check_norm(args)) return rc;
  const lik_norm_args& a = *args;
  cudaStream_t st = (cudaStream_t)stream;
  const bool params = a.dweight || a.dbias;
  if (a.rows == 0) {
    const size_t bytes = (size_t)a.width * dtype_size(a.param_dtype);
    if (a.dweight) LIK_CUDA_OK(cudaMemsetAsync(a.dweight, 0, bytes, st));
    if (a.dbias) LIK_CUDA_OK(cudaMemsetAsync(a.dbias, 0, bytes, st));
    return LIK_OK;
  }
  if (!a.dx && !params) return LIK_OK;
  LIK_REQUIRE(a.x && a.dy && a.mean && a.rstd, "x, dy, mean and rstd must not be NULL");
  if (params && (!a.workspace || a.workspace_bytes < lik_layer_norm_bwd_workspace(args))) {
    set_error("lik_layer_norm_bwd: workspace too small");
    return LIK_ERR_WORKSPACE;
  }
  const NormPlan pl = norm_plan(a, true);
  NormParams p = norm_params(a);
  p.partial = (float*)a.workspace;
  const int blocks = norm_bwd_blocks(a, pl);
  if (int rc = run_norm(a, pl, p, true, params, blocks, st)) return rc;
  if (!params) return LIK_OK;
  const SumOuts outs{{a.dweight, a.dbias, nullptr}, {a.width, 2ll * a.width, 2ll * a.width}, a.param_dtype == LIK_F32};
  return launch_sum_parts(p.partial, blocks, outs, a.dtype, st);
}
