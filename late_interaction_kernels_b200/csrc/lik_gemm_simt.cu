// Matrix products by fp32 multiply-add: c[m, n] = sum over k of a(m, k) b(n, k), any strides, and what the layers do to the
// elements of c (GemmKind) before they are rounded once and written.
//
// A block of 256 threads owns a tile of BM x BN, a thread TM x TN of it in registers; slabs of 16 k go through shared memory as
// fp32, the next one loaded into registers while the present one is multiplied.  Bound by the multiply-adds: TM + TN loads from
// shared memory feed TM * TN of them.  Products with few tiles and a long sum are cut along k: partial sums in the workspace,
// added in their order by a second kernel.
#include "lik_layers.cuh"

namespace lik {
namespace {

constexpr int SIMT_THREADS = 256, SIMT_BK = 16;

struct SimtParams {
  GemmDesc d;
  int tiles_n, splits;
  long long per_split;  // k of a split, a multiple of SIMT_BK
  float* partial;       // [splits][m][n], where splits > 1
};

template <typename T, int BM, int BN, int TM, int TN, bool DUAL>
struct SimtTile {
  float as[SIMT_BK][BM + 4];
  float bs[DUAL ? 2 : 1][SIMT_BK][BN + 4];
};

// element e of a slab of ROWS x SIMT_BK: neighbours are neighbours in memory
template <int ROWS>
__device__ __forceinline__ void slab_at(int e, bool k_major, int& r, int& k) {
  if (k_major) {
    k = e % SIMT_BK;
    r = e / SIMT_BK;
  } else {
    r = e % ROWS;
    k = e / ROWS;
  }
}
template <typename T, int ROWS>
__device__ __forceinline__ void slab_load(const GemmOperand& o, long long row0, long long rows, long long k0, long long k1,
                                          float (&v)[ROWS * SIMT_BK / SIMT_THREADS]) {
#pragma unroll
  for (int i = 0; i < ROWS * SIMT_BK / SIMT_THREADS; ++i) {
    int r, k;
    slab_at<ROWS>(threadIdx.x + i * SIMT_THREADS, o.k == 1, r, k);
    v[i] = row0 + r < rows && k0 + k < k1 ? to_f32(((const T*)o.p)[(row0 + r) * o.row + (k0 + k) * o.k]) : 0.0f;
  }
}
template <int ROWS>
__device__ __forceinline__ void slab_store(const GemmOperand& o, const float (&v)[ROWS * SIMT_BK / SIMT_THREADS], float (&s)[SIMT_BK][ROWS + 4]) {
#pragma unroll
  for (int i = 0; i < ROWS * SIMT_BK / SIMT_THREADS; ++i) {
    int r, k;
    slab_at<ROWS>(threadIdx.x + i * SIMT_THREADS, o.k == 1, r, k);
    s[k][r] = v[i];
  }
}

template <typename T, typename O, int KIND, int BM, int BN, int TM, int TN>
__global__ void __launch_bounds__(SIMT_THREADS) gemm_simt_kernel(const __grid_constant__ SimtParams p) {
  constexpr bool DUAL = KIND == GEMM_GATED;
  constexpr int TX = BN / TN;
  static_assert(TX * (BM / TM) == SIMT_THREADS, "a thread per block of the tile");
  __shared__ SimtTile<T, BM, BN, TM, TN, DUAL> sm;
  const GemmDesc& d = p.d;
  const long long m0 = (long long)(blockIdx.x / p.tiles_n) * BM;
  const int n0 = (int)(blockIdx.x % p.tiles_n) * BN;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  float acc[DUAL ? 2 : 1][TM][TN];
#pragma unroll
  for (int q = 0; q < (DUAL ? 2 : 1); ++q)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[q][i][j] = 0.0f;
  for (int seg = 0; seg < d.n_seg; ++seg) {
    const GemmOperand &a = d.a[seg], &b = d.b[seg];
    const long long k_lo = blockIdx.y * p.per_split, k_hi = p.splits > 1 && k_lo + p.per_split < d.k[seg] ? k_lo + p.per_split : d.k[seg];
    float ra[BM * SIMT_BK / SIMT_THREADS], rb[DUAL ? 2 : 1][BN * SIMT_BK / SIMT_THREADS];
    auto fetch = [&](long long k0) {
      slab_load<T, BM>(a, m0, d.m, k0, k_hi, ra);
      slab_load<T, BN>(b, n0, d.n, k0, k_hi, rb[0]);
      if constexpr (DUAL) slab_load<T, BN>(d.b[1], n0, d.n, k0, k_hi, rb[1]);
    };
    if (k_lo < k_hi) fetch(k_lo);
    for (long long k0 = k_lo; k0 < k_hi; k0 += SIMT_BK) {
      slab_store<BM>(a, ra, sm.as);
      slab_store<BN>(b, rb[0], sm.bs[0]);
      if constexpr (DUAL) slab_store<BN>(d.b[1], rb[1], sm.bs[1]);
      __syncthreads();
      if (k0 + SIMT_BK < k_hi) fetch(k0 + SIMT_BK);
#pragma unroll
      for (int k = 0; k < SIMT_BK; ++k) {
        float va[TM], vb[TN];
#pragma unroll
        for (int i = 0; i < TM; i += 4) *reinterpret_cast<float4*>(va + i) = *reinterpret_cast<const float4*>(&sm.as[k][ty * TM + i]);
#pragma unroll
        for (int q = 0; q < (DUAL ? 2 : 1); ++q) {
#pragma unroll
          for (int j = 0; j < TN; j += 4) *reinterpret_cast<float4*>(vb + j) = *reinterpret_cast<const float4*>(&sm.bs[q][k][tx * TN + j]);
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[q][i][j] = fmaf(va[i], vb[j], acc[q][i][j]);
        }
      }
      __syncthreads();
    }
  }
  if (p.splits > 1) {
    float* out = p.partial + (long long)blockIdx.y * d.m * d.n;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const long long m = m0 + ty * TM + i;
        const int n = n0 + tx * TN + j;
        if (m < d.m && n < d.n) out[m * d.n + n] = acc[0][i][j];
      }
    return;
  }
  with_activation_dev(d.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const long long m = m0 + ty * TM + i;
        const int n = n0 + tx * TN + j;
        if (m < d.m && n < d.n) gemm_element<T, O, KIND, decltype(act)::value>(d, m, n, acc[0][i][j], DUAL ? acc[DUAL ? 1 : 0][i][j] : 0.0f);
      }
  });
}

struct SimtPlan {
  bool large;
  long long tiles;
  int tiles_n, splits;
  long long per_split;
};
SimtPlan simt_plan(const GemmDesc& d) {
  SimtPlan pl{};
  const long long big = ceil_div(d.m, 128) * ceil_div(d.n, 128);
  // tiles of 128 x 128 (8 x 8 per thread) need half as many loads from shared memory per multiply-add as 64 x 64 ones, but fill the
  // machine only with a block for every SM
  pl.large = d.kind != GEMM_GATED && big >= sm_count();
  const int b = pl.large ? 128 : 64;
  pl.tiles_n = (int)ceil_div(d.n, b);
  pl.tiles = ceil_div(d.m, b) * pl.tiles_n;
  pl.splits = 1;
  pl.per_split = 0;
  const bool plain = gemm_plain(d) && d.n_seg == 1 && d.out_stride == d.n;
  if (plain && pl.tiles < sm_count() && d.k[0] >= 512) {
    long long want = ceil_div(2ll * sm_count(), pl.tiles);
    if (want > d.k[0] / 256) want = d.k[0] / 256;
    if (want > 1) {
      pl.per_split = (ceil_div(d.k[0], want) + SIMT_BK - 1) / SIMT_BK * SIMT_BK;
      pl.splits = (int)ceil_div(d.k[0], pl.per_split);
    }
  }
  return pl;
}

template <typename T, typename O, int KIND>
int run_simt(const SimtParams& p, const SimtPlan& pl, cudaStream_t st) {
  const dim3 grid((unsigned)pl.tiles, pl.splits);
  if constexpr (KIND != GEMM_GATED) {
    if (pl.large) {
      gemm_simt_kernel<T, O, KIND, 128, 128, 8, 8><<<grid, SIMT_THREADS, 0, st>>>(p), count_launch();
      LIK_CUDA_OK(cudaGetLastError());
      return LIK_OK;
    }
  }
  gemm_simt_kernel<T, O, KIND, 64, 64, 4, 4><<<grid, SIMT_THREADS, 0, st>>>(p), count_launch();
  LIK_CUDA_OK(cudaGetLastError());
  return LIK_OK;
}
template <typename T>
int run_simt(const SimtParams& p, const SimtPlan& pl, cudaStream_t st) {
  if (p.d.kind == GEMM_GATED) return run_simt<T, T, GEMM_GATED>(p, pl, st);
  if (p.d.kind == GEMM_GATED_BWD) return run_simt<T, T, GEMM_GATED_BWD>(p, pl, st);
  if (p.d.out_dtype == LIK_F32) return run_simt<T, float, GEMM_LINEAR>(p, pl, st);
  return run_simt<T, T, GEMM_LINEAR>(p, pl, st);
}

}  // namespace

size_t gemm_simt_workspace(const GemmDesc& d) {
  const SimtPlan pl = simt_plan(d);
  return pl.splits > 1 ? align_up((size_t)pl.splits * d.m * d.n * sizeof(float), 256) : 0;
}

int launch_gemm_simt(const GemmDesc& d, void* ws, size_t ws_bytes, cudaStream_t st) {
  const SimtPlan pl = simt_plan(d);
  LIK_REQUIRE(pl.tiles < (1ll << 31), "the product has too many tiles");
  SimtParams p{d, pl.tiles_n, pl.splits, pl.per_split, (float*)ws};
  if (pl.splits > 1 && (!ws || ws_bytes < gemm_simt_workspace(d))) {
    set_error("workspace too small");
    return LIK_ERR_WORKSPACE;
  }
  int rc = d.dtype == LIK_F32 ? run_simt<float>(p, pl, st) : (d.dtype == LIK_F16 ? run_simt<__half>(p, pl, st) : run_simt<__nv_bfloat16>(p, pl, st));
  if (rc || pl.splits == 1) return rc;
  return launch_sum_parts((const float*)ws, pl.splits, d.m * d.n, d.m * d.n, d.out_dtype, d.out[0], nullptr, st);
}

}  // namespace lik
