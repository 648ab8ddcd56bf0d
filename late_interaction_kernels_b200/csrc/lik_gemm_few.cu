// Matrix products with few rows of a (a token, or the tokens of a query or four): c[m, n] = sum over k of a[m, k] b[n, k].
//
// What there is to do is to read b once, so the work is cut for loads in flight: a block of eight warps owns 16 rows of b (MMA) or four
// (multiply-add), each warp an eighth of k, and the warps' sums meet in shared memory in a fixed order.  The rows of a come out of L1
// and L2.  One launch.
//   16-bit, rows of whole 16-byte pieces: mma.sync, b's rows as its 16 rows and up to 32 rows of a as its columns, eight at a time.  A sum
//     may be taken in any order of k, so a lane's fragments are 16 consecutive bytes of either operand as they lie in memory: no shared memory
//     and no shuffles before the end.  (tcgen05 would take its operands by way of shared memory, in tiles of 128 rows of b, of which
//     768 features have six for 148 SMs: 7.8 us for one token against 2.4.)
//   otherwise: fp32 multiply-add, lanes along k, 4 x 8 sums per lane that a transposing reduction brings to one per lane.
#include "lik_layers.cuh"

namespace lik {
namespace {

constexpr int FEW_WARPS = 8, FEW_THREADS = 32 * FEW_WARPS;  // of the multiply-add kernel, and of the other one unless k is long

struct FewParams {
  GemmDesc d;
};

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// NT: tiles of eight rows of a
template <typename T, int KIND, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) few_mma_kernel(const __grid_constant__ FewParams p) {
  constexpr int DUAL = KIND == GEMM_GATED ? 2 : 1;
  __shared__ float part[WARPS][DUAL][NT][32][4];
  after_the_kernel_in_front();
  const GemmDesc& d = p.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8 * NT;
  // blocks of 32 k (64 bytes of a row): this warp's share
  const int blocks = (int)((d.k[0] + 31) / 32), per = (blocks + WARPS - 1) / WARPS;
  const int kb_lo = warp * per, kb_hi = min(kb_lo + per, blocks);
  const int k_left = (int)d.k[0];
  float c[DUAL][NT][4];
#pragma unroll
  for (int q = 0; q < DUAL; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[q][i][j] = 0.0f;
  const T* w[DUAL][2];
  bool w_there[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    w_there[r] = n0 + g + 8 * r < d.n;
#pragma unroll
    for (int q = 0; q < DUAL; ++q) w[q][r] = (const T*)d.b[q].p + (long long)(w_there[r] ? n0 + g + 8 * r : 0) * d.b[q].row + t * 8;
  }
  const T* x[NT];
  bool x_there[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    x_there[i] = m0 + i * 8 + g < d.m;
    x[i] = (const T*)d.a[0].p + (x_there[i] ? (m0 + i * 8 + g) * d.a[0].row : 0) + t * 8;
  }
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
  for (int kb = kb_lo; kb < kb_hi; ++kb) {
    const int k = kb * 32;
    const bool there = k + t * 8 < k_left;  // (k is a multiple of eight)
    uint4 a[DUAL][2], b[NT];
#pragma unroll
    for (int q = 0; q < DUAL; ++q)
#pragma unroll
      for (int r = 0; r < 2; ++r) a[q][r] = there && w_there[r] ? __ldg(reinterpret_cast<const uint4*>(w[q][r] + k)) : none;
#pragma unroll
    for (int i = 0; i < NT; ++i) b[i] = there && x_there[i] ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : none;
    // a lane's eight consecutive k are four of one MMA and four of the next: the same ones of either operand
#pragma unroll
    for (int q = 0; q < DUAL; ++q) {
      const uint32_t lo[4] = {a[q][0].x, a[q][1].x, a[q][0].y, a[q][1].y}, hi[4] = {a[q][0].z, a[q][1].z, a[q][0].w, a[q][1].w};
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        mma_16x8x16<T>(c[q][i], lo, b[i].x, b[i].y);
        mma_16x8x16<T>(c[q][i], hi, b[i].z, b[i].w);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < DUAL; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i) *reinterpret_cast<float4*>(part[warp][q][i][lane]) = make_float4(c[q][i][0], c[q][i][1], c[q][i][2], c[q][i][3]);
  __syncthreads();
  with_activation_dev(d.act, [&](auto act) {
    // neighbouring threads: neighbouring rows of b, which are neighbours in the result
    for (int e = threadIdx.x; e < NT * 128; e += 32 * WARPS) {
      const int r = e % 16, in = e / 16, i = in / 8, col = in % 8, m = m0 + in;
      const bool there = m < d.m && n0 + r < d.n;
      float v[2] = {0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < DUAL; ++q)
#pragma unroll
        for (int s = 0; s < WARPS; ++s) v[q] += part[s][q][i][(r % 8) * 4 + col / 2][(r / 8) * 2 + col % 2];
      bool above = true;
      if constexpr (decltype(act)::value == LIK_ACT_RELU) {  // (whole warps come here)
        const float z = there && d.bias[0] ? v[0] + to_f32(((const T*)d.bias[0])[n0 + r]) : v[0];
        above = d.norm_a ? above_zero<T>(d, there ? m : 0, there ? n0 + r : 0, z, there, lane) : z > 0.0f;
      }
      if (there) gemm_element<T, T, KIND, decltype(act)::value>(d, m, n0 + r, v[0], v[1], above);
    }
  });
}

constexpr int FMA_ROWS = 4, FMA_COLS = 8;  // rows of b and of a per block
// V: elements of k per lane and step
template <typename T, int KIND, int V>
__global__ void __launch_bounds__(FEW_THREADS) few_fma_kernel(const __grid_constant__ FewParams p) {
  constexpr int DUAL = KIND == GEMM_GATED ? 2 : 1;
  __shared__ float part[DUAL][FEW_WARPS][32];
  after_the_kernel_in_front();
  const GemmDesc& d = p.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * FMA_ROWS, m0 = blockIdx.y * FMA_COLS;
  const long long K = d.k[0];
#pragma unroll
  for (int q = 0; q < DUAL; ++q) {
    float c[FMA_ROWS][FMA_COLS];
#pragma unroll
    for (int r = 0; r < FMA_ROWS; ++r)
#pragma unroll
      for (int m = 0; m < FMA_COLS; ++m) c[r][m] = 0.0f;
#pragma unroll 2
    for (long long k = (warp * 32 + lane) * V; k < K; k += FEW_THREADS * V) {
      float w[FMA_ROWS][V];
#pragma unroll
      for (int r = 0; r < FMA_ROWS; ++r) load_vec<T, V>((const T*)d.b[q].p + (long long)min(n0 + r, d.n - 1) * d.b[q].row + k, w[r]);
#pragma unroll
      for (int m = 0; m < FMA_COLS; ++m) {
        if (m0 + m < d.m) {
          float x[V];
          load_vec<T, V>((const T*)d.a[0].p + (m0 + m) * d.a[0].row + k, x);
#pragma unroll
          for (int r = 0; r < FMA_ROWS; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) c[r][m] = fmaf(w[r][j], x[j], c[r][m]);
        }
      }
    }
    // 32 sums per lane -> one sum over the lanes per lane: lane l ends up with sum l = r * 8 + m
    float s[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = c[i / FMA_COLS][i % FMA_COLS];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (i < o) {
          const float mine = up ? s[i + o] : s[i], other = up ? s[i] : s[i + o];
          s[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
      }
    }
    part[q][warp][lane] = s[0];
  }
  __syncthreads();
  if (warp == 0) {
    const int m = m0 + lane / FMA_ROWS, r = lane % FMA_ROWS, at = r * FMA_COLS + lane / FMA_ROWS;
    const bool there = m < d.m && n0 + r < d.n;
    float v[2] = {0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < DUAL; ++q)
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) v[q] += part[q][w][at];
    with_activation_dev(d.act, [&](auto act) {
      bool above = true;
      if constexpr (decltype(act)::value == LIK_ACT_RELU) {
        const float z = there && d.bias[0] ? v[0] + to_f32(((const T*)d.bias[0])[n0 + r]) : v[0];
        above = z > 0.0f;
        if constexpr (sizeof(T) == 2) {
          if (d.norm_a) above = above_zero<T>(d, there ? m : 0, there ? n0 + r : 0, z, there, lane);
        }
      }
      if (there) gemm_element<T, T, KIND, decltype(act)::value>(d, m, n0 + r, v[0], v[1], above);
    });
  }
}

bool few_vec(const GemmDesc& d) {
  const int item = (int)dtype_size(d.dtype);
  for (int q = 0; q < (d.kind == GEMM_GATED ? 2 : 1); ++q)
    if (((uintptr_t)d.b[q].p & 15) || (d.n > 1 && d.b[q].row * item % 16)) return false;
  return d.k[0] * item % 16 == 0 && ((uintptr_t)d.a[0].p & 15) == 0 && (d.m == 1 || d.a[0].row * item % 16 == 0);
}
template <typename T, int KIND, int NT>
int run_mma(const FewParams& p, cudaStream_t st) {
  const GemmDesc& d = p.d;
  const dim3 grid((unsigned)ceil_div(d.n, 16), (unsigned)ceil_div(d.m, 8 * NT));
  // a long k: twice the warps, half the loads one after another (32 rows, 2048 x 768: 9.3 us against 6.1)
  if constexpr (KIND == GEMM_LINEAR) {
    if (d.k[0] >= 1024) {
      return launch_after(few_mma_kernel<T, KIND, NT, 2 * FEW_WARPS>, grid, 64 * FEW_WARPS, 0, st, 1, p);
    }
  }
  return launch_after(few_mma_kernel<T, KIND, NT, FEW_WARPS>, grid, FEW_THREADS, 0, st, 1, p);
}
template <typename T, int KIND>
int run_few(const FewParams& p, cudaStream_t st) {
  const GemmDesc& d = p.d;
  const bool vec = few_vec(d);
  if constexpr (sizeof(T) == 2) {
    if (vec) return d.m <= 8 ? run_mma<T, KIND, 1>(p, st) : (d.m <= 16 ? run_mma<T, KIND, 2>(p, st) : run_mma<T, KIND, 4>(p, st));
  }
  const dim3 grid((unsigned)ceil_div(d.n, FMA_ROWS), (unsigned)ceil_div(d.m, FMA_COLS));
  if constexpr (sizeof(T) == 4) {
    if (vec) return launch_after(few_fma_kernel<T, KIND, vec_elems<T>()>, grid, FEW_THREADS, 0, st, 1, p);
  }
  return launch_after(few_fma_kernel<T, KIND, 1>, grid, FEW_THREADS, 0, st, 1, p);
}
template <typename T>
int run_few(const FewParams& p, cudaStream_t st) {
  return p.d.kind == GEMM_GATED ? run_few<T, GEMM_GATED>(p, st) : run_few<T, GEMM_LINEAR>(p, st);
}

}  // namespace

// By the blocks that there are for an SM, and from k = 1024 on, where a block's 512 threads have an SM to themselves, by the k that an SM goes through
// one after another; the tensor-core kernels have a start of their own of 6 us (fp32: 10 with the cuts) and can cut a long k.  Measured on both
// sides of each limit, few rows against tensor cores in us: 16-bit 768 x 768, 256 rows (2.6 blocks) 6.5 / 8.0; 768 x 2048, 128 rows (3.5) 9.8 / 8.0;
// k = 1024, 96 rows of 1024 (two of 1024) 6.4 / 6.8, 192 (three) 9.4 / 7.4; k = 2048, 96 rows of 768 (one) 6.0 / 7.0, 128 (two) 10.5 / 7.4;
// k = 4096, 32 rows (one) 9.1 / 7.7, 16 rows 6.8 / 7.4; k = 8192, 16 rows 11.2 / 8.2, 8 rows 6.8 / 8.3; k = 16384, 8 rows 11.4 / 9.9; fp32 768 x 768, 32 rows
// (5.2 blocks) 9.6 / 11.5, 64 rows (10.4) 16 / 11.3.
bool gemm_few_pays(const GemmDesc& d) {
  if (d.kind == GEMM_GATED_BWD || d.n_seg != 1 || d.a[0].k != 1 || d.b[0].k != 1 || d.out_dtype != d.dtype || d.k[0] >= (1ll << 31) - 4096) return false;
  const long long sms = sm_count(), dual = d.kind == GEMM_GATED ? 2 : 1;
  if (d.dtype != LIK_F32 && few_vec(d)) {
    const long long rows = d.m <= 8 ? 8 : (d.m <= 16 ? 16 : 32);
    const long long blocks = dual * ceil_div(d.n, 16) * ceil_div(d.m, rows);
    if (d.kind == GEMM_LINEAR && d.k[0] >= 1024) {
      const long long in_turn = rows == 8 ? d.k[0] : ceil_div(blocks, sms) * d.k[0];
      if (in_turn > (rows == 8 ? 12000 : (rows == 16 ? 5000 : 2500))) return false;
    }
    return blocks * 5 <= 13 * sms * (32 / rows);
  }
  return dual * ceil_div(d.n, FMA_ROWS) * ceil_div(d.m, FMA_COLS) <= 8 * sms;
}
int launch_gemm_few(const GemmDesc& d, cudaStream_t st) {
  const FewParams p{d};
  return d.dtype == LIK_F32 ? run_few<float>(p, st) : (d.dtype == LIK_F16 ? run_few<__half>(p, st) : run_few<__nv_bfloat16>(p, st));
}

}  // namespace lik
