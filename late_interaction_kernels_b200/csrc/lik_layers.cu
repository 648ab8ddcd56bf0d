// The layers' C entry points: which products and passes a call is made of, and the passes that are not products.
#include "lik_layers.cuh"

namespace lik {
namespace {

// ---------------------------------------------------------------------------------------------
// Sums over parts of partial[part][i], in the order of the parts, to up to SUM_OUTS vectors one behind the other
// ---------------------------------------------------------------------------------------------
constexpr int SUM_COLS = 8;  // a sector of each part; the block's 32 groups of threads take every 32nd part
template <typename T>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* __restrict__ partial, int parts, const __grid_constant__ SumOuts outs) {
  __shared__ float s[8][SUM_COLS];
  after_the_kernel_in_front();
  const int col = threadIdx.x % SUM_COLS, group = threadIdx.x / SUM_COLS, warp = threadIdx.x / 32;
  const long long i = blockIdx.x * (long long)SUM_COLS + col, n = outs.end[SUM_OUTS - 1];
  float v = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int q = group; q < parts; q += 32) v += partial[q * n + i];
  }
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  if (threadIdx.x % 32 < SUM_COLS) s[warp][col] = v;
  __syncthreads();
  if (group == 0 && i < n) {
#pragma unroll
    for (int w = 1; w < 8; ++w) v += s[w][col];
    outs.put<T>(i, v);
  }
}

// ---------------------------------------------------------------------------------------------
// dz = dy * act'(z), rounded to T as the operand of two products, and the sums of its columns before that rounding; or the sums of up to SUM_OUTS matrices' columns.  Memory-bound: each element read once, dz
// written once.  A block takes 32 vectors of columns (a lane's V columns) of a matrix and a share of the rows, eight at a time; with one
// share the sums are done, else sum_parts_kernel adds them up.
// ---------------------------------------------------------------------------------------------
constexpr int SLOPE_LANES = 8;
struct SlopeJob {
  const void *dy, *z;
  long long dy_stride, z_stride;
  int n, blocks;  // blocks of columns
  void* dz;       // or NULL: sums only
  long long dz_stride;
  bool padded;    // what lies between n and the next 16 bytes belongs to the row
};
struct SlopeParams {
  SlopeJob job[SUM_OUTS];
  int n_jobs;
  long long rows, rows_per;
  float* partial;  // [gridDim.y][columns of all jobs]; NULL: straight to outs
  bool sums;
  SumOuts outs;
};
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(32 * SLOPE_LANES, 4) slope_kernel(const __grid_constant__ SlopeParams p) {
  __shared__ float s[SLOPE_LANES][32 * V + 1];
  after_the_kernel_in_front();
  const int lane = threadIdx.x % 32, row = threadIdx.x / 32;
  int q = 0, block = blockIdx.x;
  while (block >= p.job[q].blocks) block -= p.job[q++].blocks;
  const SlopeJob& j = p.job[q];
  const int c = (block * 32 + lane) * V;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  if (c < j.n) {
    const long long r0 = blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.rows ? r0 + p.rows_per : p.rows;
#pragma unroll 2
    for (long long r = r0 + row; r < r1; r += SLOPE_LANES) {
      float g[V], z[V];
      load_vec<T, V>((const T*)j.dy + r * j.dy_stride + c, g);
      if constexpr (ACT != LIK_ACT_NONE) {
        load_vec<T, V>((const T*)j.z + r * j.z_stride + c, z);
        if constexpr (sizeof(T) == 4 || V == 1) {
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] *= act_slope<ACT, sizeof(T) == 4>(z[i], z[i]);
        } else {
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            float sx, sy;
            act_pair<ACT, true>(z[i], z[i + 1], sx, sy);
            mul2(Pair(g[i], g[i + 1]), Pair(sx, sy)).get(g[i], g[i + 1]);
          }
        }
        store_vec<T, V>((T*)j.dz + r * j.dz_stride + c, g);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += g[i];
    }
  }
  if (!p.sums) return;
#pragma unroll
  for (int i = 0; i < V; ++i) s[row][i * 32 + lane] = sum[i];
  __syncthreads();
  const long long first = q ? p.outs.end[q - 1] : 0, total = p.outs.end[SUM_OUTS - 1];
  for (int i = threadIdx.x; i < 32 * V; i += 32 * SLOPE_LANES) {
    float v = 0.0f;
#pragma unroll
    for (int l = 0; l < SLOPE_LANES; ++l) v += s[l][i];
    const int col = (block * 32 + i % 32) * V + i / 32;
    if (col < j.n) {
      if (p.partial) p.partial[blockIdx.y * total + first + col] = v;
      else p.outs.put<T>(first + col, v);
    }
  }
}
// (128 rows: a lane's sixteen, in four trips to memory)
int slope_parts(long long rows, long long cols, int dtype) {
  if (rows <= 128) return 1;
  // four blocks per SM, and none that would wait for one of them to end
  long long want = 4ll * sm_count() / ceil_div(cols, 32 * (16 / (int)dtype_size(dtype)));
  if (want > ceil_div(rows, SLOPE_LANES)) want = ceil_div(rows, SLOPE_LANES);
  if (want > 65535) want = 65535;
  return want < 1 ? 1 : (int)want;
}
size_t slope_workspace(long long rows, long long cols, int dtype) {
  const int parts = slope_parts(rows, cols, dtype);
  return parts == 1 ? 0 : align_up((size_t)parts * cols * sizeof(float), 256);
}
template <typename T>
int run_slope(SlopeParams& p, int act, bool vec, int parts, cudaStream_t st) {
  constexpr int V = vec_elems<T>();
  unsigned blocks = 0;
  for (int i = 0; i < p.n_jobs; ++i) blocks += p.job[i].blocks = (int)ceil_div(p.job[i].n, 32 * (vec ? V : 1));
  int rc = LIK_OK;
  with_activation(act, [&](auto a) {
    rc = vec ? launch_after(slope_kernel<T, V, decltype(a)::value>, dim3(blocks, parts), 32 * SLOPE_LANES, 0, st, 1, p)
             : launch_after(slope_kernel<T, 1, decltype(a)::value>, dim3(blocks, parts), 32 * SLOPE_LANES, 0, st, 1, p);
  });
  return rc;
}
// jobs, rows, partial and the addresses of the sums (of sums_dtype, as the outs say) are filled in
int launch_slope(SlopeParams& p, int act, int dtype, bool sums, cudaStream_t st) {
  const int item = (int)dtype_size(dtype);
  long long cols = 0;
  bool vec = true;
  for (int i = 0; i < SUM_OUTS; ++i) {
    if (i < p.n_jobs) {
      const SlopeJob& j = p.job[i];
      cols += j.n;
      vec = vec && vec_ok(j.dy, j.dy_stride, j.padded ? 0 : j.n, item) && (act == LIK_ACT_NONE || (vec_ok(j.z, j.z_stride, j.n, item) && vec_ok(j.dz, j.dz_stride, j.n, item)));
    }
    p.outs.end[i] = cols;
  }
  const int parts = sums || p.rows > 128 ? slope_parts(p.rows, cols, dtype) : 1;
  p.rows_per = ceil_div(p.rows, parts);
  p.sums = sums;
  if (parts == 1) p.partial = nullptr;
  int rc = dtype == LIK_F32 ? run_slope<float>(p, act, vec, parts, st)
                            : (dtype == LIK_F16 ? run_slope<__half>(p, act, vec, parts, st) : run_slope<__nv_bfloat16>(p, act, vec, parts, st));
  if (rc || !sums || parts == 1) return rc;
  return launch_sum_parts(p.partial, parts, p.outs, dtype, st);
}

// ---------------------------------------------------------------------------------------------
// Lengths of the rows of two matrices (kink_bound), a warp per row.  Bound by memory: each element read once.
// ---------------------------------------------------------------------------------------------
struct KinkNorms {
  const void* p[2];
  long long stride[2], rows[2];
  long long k;
  float* norm[2];
};
template <typename T>
__global__ void __launch_bounds__(256) kink_norms_kernel(const __grid_constant__ KinkNorms p) {
  after_the_kernel_in_front();
  const int lane = threadIdx.x & 31;
  for (long long g = blockIdx.x * 8ll + threadIdx.x / 32; g < p.rows[0] + p.rows[1]; g += gridDim.x * 8ll) {
    const int q = g < p.rows[0] ? 0 : 1;
    const long long r = q ? g - p.rows[0] : g;
    const T* x = (const T*)p.p[q] + r * p.stride[q];
    float s = 0.0f, largest = 0.0f;
    auto take = [&](float v) {
      s = fmaf(v, v, s);
      largest = fmaxf(largest, fabsf(v));
    };
    // (up to the first 16-byte boundary element by element, and behind the last)
    const long long head = min((long long)((16 - ((uintptr_t)x & 15)) % 16 / sizeof(T)), p.k), end = head + ((p.k - head) & ~7ll);
    if (lane < head) take(to_f32(x[lane]));
    if (end + lane < p.k) take(to_f32(x[end + lane]));
#pragma unroll 4
    for (long long i = head + lane * 8; i < end; i += 256) {
      float v[8];
      load_vec<T, 8>(x + i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) take(v[j]);
    }
    s = warp_sum(s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    // (where squares would leave fp32's range: the bound by the largest; a NaN is no bound, and its row's sums have no sign)
    if (lane == 0) p.norm[q][r] = largest < 1e-15f || largest > 1e15f ? (s != s ? s : largest * sqrtf((float)p.k)) : sqrtf(s);
  }
}
bool keeps_side(const GemmDesc& d) { return d.dtype != LIK_F32 && d.act == LIK_ACT_RELU && d.kept[0]; }
int launch_kink_norms(const GemmDesc& d, cudaStream_t st) {
  if (!d.norm_a) return LIK_OK;
  const KinkNorms p{{d.a[0].p, d.b[0].p}, {d.a[0].row, d.b[0].row}, {d.m, d.n}, d.k[0], {(float*)d.norm_a, (float*)d.norm_b}};
  const long long need = ceil_div(d.m + d.n, 8), most = 16ll * sm_count();
  const unsigned grid = (unsigned)(need < most ? need : most);
  return d.dtype == LIK_F16 ? launch_after(kink_norms_kernel<__half>, grid, 256, 0, st, 1, p) : launch_after(kink_norms_kernel<__nv_bfloat16>, grid, 256, 0, st, 1, p);
}

// Which kernel a product goes to.  Several products of a pass are plain ones and go to the tensor cores together.
size_t gemm_workspace(const GemmDesc* d, int n = 1) {
  if (n == 0 || (n == 1 && gemm_few_pays(*d))) return 0;
  return d->dtype == LIK_F32 ? gemm_f32_workspace(d, n) : gemm_tc_workspace(d, n);
}
int launch_gemm(const GemmDesc* d, int n, void* ws, size_t ws_bytes, int* status, cudaStream_t st) {
  if (n == 0) return LIK_OK;
  if (n == 1 && gemm_few_pays(*d)) return launch_gemm_few(*d, st);
  return d->dtype == LIK_F32 ? launch_gemm_f32(d, n, ws, ws_bytes, status, st) : launch_gemm_tc(d, n, ws, ws_bytes, status, st);
}

bool act_known(int a) { return a >= LIK_ACT_NONE && a <= LIK_ACT_SIGMOID; }
bool dtype_known(int d) { return d == LIK_F32 || d == LIK_F16 || d == LIK_BF16; }
// rows of kept and internal matrices start on 16 bytes
long long pad_cols(long long n, int dtype) {
  const long long v = 16 / (long long)dtype_size(dtype);
  return (n + v - 1) / v * v;
}

// Workspace, taken piece by piece.  Without a base only the sizes are added up; the addresses are then made up, but as far apart and as
// aligned as the real ones, since a plan looks at both.
struct Carve {
  char* base;
  size_t off = 0;
  explicit Carve(void* ws) : base(ws ? (char*)ws : (char*)256) {}
  template <typename P = void>
  P* take(size_t bytes) {
    P* p = (P*)(base + off);
    off += align_up(bytes, 256);
    return p;
  }
};

// room for the lengths of the rows that a kept side of relu asks for
void take_norms(GemmDesc& d, Carve& c) {
  if (!keeps_side(d)) return;
  d.norm_a = c.take<float>((size_t)d.m * sizeof(float));
  d.norm_b = c.take<float>((size_t)d.n * sizeof(float));
}

// units of the products are counted in 32 bits, shares of k included
bool tiles_fit(long long m, long long n) { return ceil_div(m, 128) * ceil_div(n, 64) < (1ll << 30); }

int check_linear(const lik_linear_args* a) {
  LIK_REQUIRE(a != nullptr, "args is NULL");
  LIK_REQUIRE(dtype_known(a->dtype), "dtype must be fp32, fp16 or bf16");
  LIK_REQUIRE(a->param_dtype == a->dtype || a->param_dtype == LIK_F32, "param_dtype must be dtype or fp32");
  LIK_REQUIRE(act_known(a->activation), "unknown activation");
  LIK_REQUIRE(a->rows >= 0 && a->rows < (1ll << 31) && a->in > 0 && a->out > 0, "sizes must be positive, rows below 2^31");
  LIK_REQUIRE(tiles_fit(a->rows, a->out) && tiles_fit(a->rows, a->in) && tiles_fit(a->out, a->in), "the matrices are too large");
  LIK_REQUIRE(((uintptr_t)a->workspace & 15) == 0, "the workspace must be 16-byte aligned");
  LIK_REQUIRE(a->x_stride >= a->in && a->w_stride >= a->in, "x_stride and w_stride must be at least in");
  return LIK_OK;
}
GemmDesc linear_fwd_desc(const lik_linear_args& a) {
  GemmDesc d;
  d.act = a.activation;
  d.dtype = d.out_dtype = a.dtype;
  d.m = a.rows;
  d.n = a.out;
  d.k[0] = a.in;
  d.a[0] = {a.x, a.x_stride, 1};
  d.b[0] = {a.w, a.w_stride, 1};
  d.bias[0] = a.bias;
  d.residual = a.residual;
  d.residual_stride = a.residual_stride;
  d.out[0] = a.y;
  d.out_stride = a.out;
  d.kept[0] = a.activation == LIK_ACT_NONE ? nullptr : a.z;
  d.kept_stride = a.z_stride;
  return d;
}
struct LinearFwd {
  GemmDesc d;
  void* gemm;
  size_t gemm_bytes, total;
};
LinearFwd linear_fwd_layout(const lik_linear_args& a, void* ws) {
  LinearFwd l{linear_fwd_desc(a)};
  Carve c(ws);
  take_norms(l.d, c);
  l.gemm_bytes = gemm_workspace(&l.d);
  l.gemm = c.take(l.gemm_bytes);
  l.total = c.off;
  return l;
}
// dx = dz w and dw = dz^T x
GemmDesc grad_x_desc(int dtype, long long rows, int out, int in, const void* dz, long long dz_stride, const void* w, long long w_stride, void* dx) {
  GemmDesc d;
  d.dtype = d.out_dtype = dtype;
  d.m = rows;
  d.n = in;
  d.k[0] = out;
  d.a[0] = {dz, dz_stride, 1};
  d.b[0] = {w, 1, w_stride};
  d.out[0] = dx;
  d.out_stride = in;
  return d;
}
GemmDesc grad_w_desc(int dtype, int param_dtype, long long rows, int out, int in, const void* dz, long long dz_stride, const void* x, long long x_stride,
                     void* dw) {
  GemmDesc d;
  d.dtype = dtype;
  d.out_dtype = param_dtype;
  d.m = out;
  d.n = in;
  d.k[0] = rows;
  d.a[0] = {dz, 1, dz_stride};
  d.b[0] = {x, 1, x_stride};
  d.out[0] = dw;
  d.out_stride = in;
  return d;
}

struct LinearBwd {
  GemmDesc grads[2];  // dx and dw, as far as they are asked for
  int n_grads = 0;
  void* dz;
  long long dz_stride;
  float* partial;
  void* gemm;
  size_t gemm_bytes, total;
};
LinearBwd linear_bwd_layout(const lik_linear_args& a, void* ws) {
  LinearBwd l{};
  Carve c(ws);
  const bool act = a.activation != LIK_ACT_NONE;
  if (act) {
    l.dz_stride = pad_cols(a.out, a.dtype);
    l.dz = c.take((size_t)a.rows * l.dz_stride * dtype_size(a.dtype));
  }
  if (a.dbias) l.partial = c.take<float>(slope_workspace(a.rows, a.out, a.dtype));
  const void* dz = act ? l.dz : a.dy;
  const long long st = act ? l.dz_stride : a.dy_stride;
  if (a.dw) l.grads[l.n_grads++] = grad_w_desc(a.dtype, a.param_dtype, a.rows, a.out, a.in, dz, st, a.x, a.x_stride, a.dw);
  if (a.dx) l.grads[l.n_grads++] = grad_x_desc(a.dtype, a.rows, a.out, a.in, dz, st, a.w, a.w_stride, a.dx);
  l.gemm_bytes = gemm_workspace(l.grads, l.n_grads);
  l.gemm = c.take(l.gemm_bytes);
  l.total = c.off;
  return l;
}
int too_small(const char* what) {
  set_error("%s: workspace too small", what);
  return LIK_ERR_WORKSPACE;
}
int zero(void* p, size_t bytes, cudaStream_t st) {
  if (p) LIK_CUDA_OK(cudaMemsetAsync(p, 0, bytes, st));
  return LIK_OK;
}

int check_gated(const lik_gated_args* a) {
  LIK_REQUIRE(a != nullptr, "args is NULL");
  LIK_REQUIRE(dtype_known(a->dtype), "dtype must be fp32, fp16 or bf16");
  LIK_REQUIRE(a->param_dtype == a->dtype || a->param_dtype == LIK_F32, "param_dtype must be dtype or fp32");
  LIK_REQUIRE(act_known(a->activation), "unknown activation");
  LIK_REQUIRE(a->rows >= 0 && a->rows < (1ll << 31) && a->in > 0 && a->hidden > 0 && a->out > 0, "sizes must be positive, rows below 2^31");
  LIK_REQUIRE(tiles_fit(a->rows, a->hidden) && tiles_fit(a->rows, a->in) && tiles_fit(a->rows, a->out) && tiles_fit(a->hidden, a->in) &&
                  tiles_fit(a->hidden, a->out), "the matrices are too large");
  LIK_REQUIRE(((uintptr_t)a->workspace & 15) == 0, "the workspace must be 16-byte aligned");
  LIK_REQUIRE(a->x_stride >= a->in && a->w_gate_stride >= a->in && a->w_up_stride >= a->in && a->w_down_stride >= a->hidden, "a stride is below its row");
  return LIK_OK;
}
struct GatedFwd {
  GemmDesc up, down;
  void* gemm;
  size_t gemm_bytes, total;
};
GatedFwd gated_fwd_layout(const lik_gated_args& a, void* ws) {
  GatedFwd l{};
  Carve c(ws);
  void* h = a.h;
  long long h_stride = a.kept_stride;
  if (!a.gate_factor) {
    h_stride = pad_cols(a.hidden, a.dtype);
    h = c.take((size_t)a.rows * h_stride * dtype_size(a.dtype));
  }
  GemmDesc& u = l.up;
  u.kind = GEMM_GATED;
  u.act = a.activation;
  u.dtype = u.out_dtype = a.dtype;
  u.m = a.rows;
  u.n = a.hidden;
  u.k[0] = a.in;
  u.a[0] = {a.x, a.x_stride, 1};
  u.b[0] = {a.w_gate, a.w_gate_stride, 1};
  u.b[1] = {a.w_up, a.w_up_stride, 1};
  u.bias[0] = a.b_gate;
  u.bias[1] = a.b_up;
  u.out[0] = h;
  u.out_stride = h_stride;
  u.kept[0] = a.gate_factor;
  u.kept[1] = a.up_factor;
  u.kept_stride = a.kept_stride;
  take_norms(u, c);
  GemmDesc& d = l.down;
  d.dtype = d.out_dtype = a.dtype;
  d.m = a.rows;
  d.n = a.out;
  d.k[0] = a.hidden;
  d.a[0] = {h, h_stride, 1};
  d.b[0] = {a.w_down, a.w_down_stride, 1};
  d.bias[0] = a.b_down;
  d.residual = a.residual;
  d.residual_stride = a.residual_stride;
  d.out[0] = a.y;
  d.out_stride = a.out;
  const size_t b1 = gemm_workspace(&u), b2 = gemm_workspace(&d);
  l.gemm_bytes = b1 > b2 ? b1 : b2;
  l.gemm = c.take(l.gemm_bytes);
  l.total = c.off;
  return l;
}
struct GatedBwd {
  GemmDesc dh, grads[4];  // dh for the gradients behind it; dx and the weights' gradients, as far as they are asked for
  int n_grads = 0;
  void *dg, *du;
  long long stride;
  float* partial;
  void* gemm;
  size_t gemm_bytes, total;
};
GatedBwd gated_bwd_layout(const lik_gated_args& a, void* ws) {
  GatedBwd l{};
  Carve c(ws);
  l.stride = pad_cols(a.hidden, a.dtype);
  const bool inner = a.dx || a.dw_gate || a.dw_up || a.db_gate || a.db_up;
  if (inner) {
    l.dg = c.take((size_t)a.rows * l.stride * dtype_size(a.dtype));
    l.du = c.take((size_t)a.rows * l.stride * dtype_size(a.dtype));
    GemmDesc& h = l.dh;
    h.kind = GEMM_GATED_BWD;
    h.dtype = h.out_dtype = a.dtype;
    h.m = a.rows;
    h.n = a.hidden;
    h.k[0] = a.out;
    h.a[0] = {a.dy, a.dy_stride, 1};
    h.b[0] = {a.w_down, 1, a.w_down_stride};
    h.out[0] = l.dg;
    h.out[1] = l.du;
    h.out_stride = l.stride;
    h.kept[0] = a.gate_factor;
    h.kept[1] = a.up_factor;
    h.kept_stride = a.kept_stride;
  }
  if (a.dw_gate) l.grads[l.n_grads++] = grad_w_desc(a.dtype, a.param_dtype, a.rows, a.hidden, a.in, l.dg, l.stride, a.x, a.x_stride, a.dw_gate);
  if (a.dw_up) l.grads[l.n_grads++] = grad_w_desc(a.dtype, a.param_dtype, a.rows, a.hidden, a.in, l.du, l.stride, a.x, a.x_stride, a.dw_up);
  if (a.dw_down) l.grads[l.n_grads++] = grad_w_desc(a.dtype, a.param_dtype, a.rows, a.out, a.hidden, a.dy, a.dy_stride, a.h, a.kept_stride, a.dw_down);
  if (a.dx) {
    GemmDesc& d = l.grads[l.n_grads++] = grad_x_desc(a.dtype, a.rows, a.hidden, a.in, l.dg, l.stride, a.w_gate, a.w_gate_stride, a.dx);
    d.n_seg = 2;
    d.k[1] = a.hidden;
    d.a[1] = {l.du, l.stride, 1};
    d.b[1] = {a.w_up, 1, a.w_up_stride};
  }
  for (int i = 0; i < l.n_grads; ++i) l.grads[i].several = true;
  l.gemm_bytes = gemm_workspace(l.grads, l.n_grads);
  if (inner) {
    const size_t b = gemm_workspace(&l.dh);
    l.gemm_bytes = b > l.gemm_bytes ? b : l.gemm_bytes;
  }
  const long long sums = (a.db_gate ? a.hidden : 0ll) + (a.db_up ? a.hidden : 0ll) + (a.db_down ? a.out : 0ll);
  if (sums) l.partial = c.take<float>(slope_workspace(a.rows, sums, a.dtype));
  l.gemm = c.take(l.gemm_bytes);
  l.total = c.off;
  return l;
}

}  // namespace

int launch_sum_parts(const float* partial, int parts, const SumOuts& outs, int dtype, cudaStream_t st) {
  const long long grid = ceil_div(outs.end[SUM_OUTS - 1], SUM_COLS);
  LIK_REQUIRE(grid < (1ll << 31), "too many sums");
  return dtype == LIK_F32   ? launch_after(sum_parts_kernel<float>, (unsigned)grid, 256, 0, st, 1, partial, parts, outs)
         : dtype == LIK_F16 ? launch_after(sum_parts_kernel<__half>, (unsigned)grid, 256, 0, st, 1, partial, parts, outs)
                            : launch_after(sum_parts_kernel<__nv_bfloat16>, (unsigned)grid, 256, 0, st, 1, partial, parts, outs);
}

}  // namespace lik

extern "C" size_t lik_linear_fwd_workspace(const lik_linear_args* a) {
  using namespace lik;
  if (check_linear(a) || a->rows == 0) return 0;
  return linear_fwd_layout(*a, nullptr).total;
}
extern "C" int lik_linear_fwd(const lik_linear_args* args, lik_stream_t stream) {
  using namespace lik;
  if (int rc = check_linear(args)) return rc;
  const lik_linear_args& a = *args;
  if (a.rows == 0) return LIK_OK;
  LIK_REQUIRE(a.x && a.w && a.y, "x, w and y must not be NULL");
  LIK_REQUIRE(!a.z || (a.z_stride >= a.out && a.z_stride * dtype_size(a.dtype) % 16 == 0 && ((uintptr_t)a.z & 15) == 0), "z must have 16-byte rows");
  LIK_REQUIRE(!a.residual || a.residual_stride >= a.out, "residual_stride must be at least out");
  const LinearFwd l = linear_fwd_layout(a, a.workspace);
  if (a.workspace_bytes < l.total || (l.total && !a.workspace)) return too_small("lik_linear_fwd");
  if (int rc = launch_kink_norms(l.d, (cudaStream_t)stream)) return rc;
  return launch_gemm(&l.d, 1, l.gemm, l.gemm_bytes, a.status, (cudaStream_t)stream);
}

extern "C" size_t lik_linear_bwd_workspace(const lik_linear_args* a) {
  using namespace lik;
  if (check_linear(a) || a->rows == 0) return 0;
  return linear_bwd_layout(*a, nullptr).total;
}
extern "C" int lik_linear_bwd(const lik_linear_args* args, lik_stream_t stream) {
  using namespace lik;
  if (int rc = check_linear(args)) return rc;
  const lik_linear_args& a = *args;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t pi = dtype_size(a.param_dtype);
  if (a.rows == 0) {
    if (int rc = zero(a.dw, pi * a.out * a.in, st)) return rc;
    return zero(a.dbias, pi * a.out, st);
  }
  if (!a.dx && !a.dw && !a.dbias) return LIK_OK;
  LIK_REQUIRE(a.x && a.w && a.dy && a.dy_stride >= a.out, "x, w and dy must not be NULL, dy_stride at least out");
  const bool act = a.activation != LIK_ACT_NONE;
  LIK_REQUIRE(!act || (a.z && a.z_stride >= a.out && a.z_stride * dtype_size(a.dtype) % 16 == 0 && ((uintptr_t)a.z & 15) == 0),
              "z must be there, with 16-byte rows");
  const LinearBwd l = linear_bwd_layout(a, a.workspace);
  if (a.workspace_bytes < l.total || (l.total && !a.workspace)) return too_small("lik_linear_bwd");
  if (act || a.dbias) {
    SlopeParams p{};
    p.job[0] = {a.dy, a.z, a.dy_stride, a.z_stride, a.out, 0, l.dz, l.dz_stride, false};
    p.n_jobs = 1;
    p.rows = a.rows;
    p.partial = l.partial;
    p.outs.out[0] = a.dbias;
    p.outs.f32 = a.param_dtype == LIK_F32;
    if (int rc = launch_slope(p, a.activation, a.dtype, a.dbias != nullptr, st)) return rc;
  }
  return launch_gemm(l.grads, l.n_grads, l.gemm, l.gemm_bytes, a.status, st);
}

extern "C" size_t lik_gated_fwd_workspace(const lik_gated_args* a) {
  using namespace lik;
  if (check_gated(a) || a->rows == 0) return 0;
  return gated_fwd_layout(*a, nullptr).total;
}
extern "C" int lik_gated_fwd(const lik_gated_args* args, lik_stream_t stream) {
  using namespace lik;
  if (int rc = check_gated(args)) return rc;
  const lik_gated_args& a = *args;
  if (a.rows == 0) return LIK_OK;
  LIK_REQUIRE(a.x && a.w_gate && a.w_up && a.w_down && a.y, "x, the weights and y must not be NULL");
  LIK_REQUIRE(!a.gate_factor == !a.up_factor && !a.gate_factor == !a.h, "gate_factor, up_factor and h are kept together");
  LIK_REQUIRE(!a.gate_factor || (a.kept_stride >= a.hidden && a.kept_stride * dtype_size(a.dtype) % 16 == 0 &&
                          (((uintptr_t)a.gate_factor | (uintptr_t)a.up_factor | (uintptr_t)a.h) & 15) == 0), "gate_factor, up_factor and h must have 16-byte rows");
  LIK_REQUIRE(!a.residual || a.residual_stride >= a.out, "residual_stride must be at least out");
  const GatedFwd l = gated_fwd_layout(a, a.workspace);
  if (a.workspace_bytes < l.total || (l.total && !a.workspace)) return too_small("lik_gated_fwd");
  if (int rc = launch_kink_norms(l.up, (cudaStream_t)stream)) return rc;
  if (int rc = launch_gemm(&l.up, 1, l.gemm, l.gemm_bytes, a.status, (cudaStream_t)stream)) return rc;
  return launch_gemm(&l.down, 1, l.gemm, l.gemm_bytes, a.status, (cudaStream_t)stream);
}

extern "C" size_t lik_gated_bwd_workspace(const lik_gated_args* a) {
  using namespace lik;
  if (check_gated(a) || a->rows == 0) return 0;
  return gated_bwd_layout(*a, nullptr).total;
}
extern "C" int lik_gated_bwd(const lik_gated_args* args, lik_stream_t stream) {
  using namespace lik;
  if (int rc = check_gated(args)) return rc;
  const lik_gated_args& a = *args;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t pi = dtype_size(a.param_dtype);
  if (a.rows == 0) {
    void* const ptrs[] = {a.dw_gate, a.dw_up, a.dw_down, a.db_gate, a.db_up, a.db_down};
    const size_t sizes[] = {pi * a.hidden * a.in, pi * a.hidden * a.in, pi * a.hidden * a.out, pi * a.hidden, pi * a.hidden, pi * a.out};
    for (int i = 0; i < 6; ++i)
      if (int rc = zero(ptrs[i], sizes[i], st)) return rc;
    return LIK_OK;
  }
  LIK_REQUIRE(a.x && a.w_gate && a.w_up && a.w_down && a.dy && a.dy_stride >= a.out, "x, the weights and dy must not be NULL, dy_stride at least out");
  const bool kept = a.dx || a.dw_gate || a.dw_up || a.dw_down || a.db_gate || a.db_up;  // (db_down is made of dy alone)
  LIK_REQUIRE(!kept || (a.gate_factor && a.up_factor && a.h && a.kept_stride >= a.hidden && a.kept_stride * dtype_size(a.dtype) % 16 == 0 &&
                        (((uintptr_t)a.gate_factor | (uintptr_t)a.up_factor | (uintptr_t)a.h) & 15) == 0), "gate_factor, up_factor and h must be there, with 16-byte rows");
  const GatedBwd l = gated_bwd_layout(a, a.workspace);
  if (a.workspace_bytes < l.total || (l.total && !a.workspace)) return too_small("lik_gated_bwd");
  if (l.dg)
    if (int rc = launch_gemm(&l.dh, 1, l.gemm, l.gemm_bytes, a.status, st)) return rc;
  if (int rc = launch_gemm(l.grads, l.n_grads, l.gemm, l.gemm_bytes, a.status, st)) return rc;
  SlopeParams p{};
  auto sum = [&](const void* g, long long stride, int n, void* out, bool padded) {
    if (!out) return;
    p.job[p.n_jobs] = {g, nullptr, stride, 0, n, 0, nullptr, 0, padded};
    p.outs.out[p.n_jobs++] = out;
  };
  // (of dg and du as they were rounded for the products: before that they are in an epilogue that has each column in pieces, and over many rows what
  // the roundings add up to is small beside one rounding of the sum)
  sum(l.dg, l.stride, a.hidden, a.db_gate, true);
  sum(l.du, l.stride, a.hidden, a.db_up, true);
  sum(a.dy, a.dy_stride, a.out, a.db_down, false);
  if (!p.n_jobs) return LIK_OK;
  p.rows = a.rows;
  p.partial = l.partial;
  p.outs.f32 = a.param_dtype == LIK_F32;
  return launch_slope(p, LIK_ACT_NONE, a.dtype, true, st);
}
