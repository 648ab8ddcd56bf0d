// Matrix products of fp32 operands on the tensor cores: c[m, n] = sum over k of a(m, k) b(n, k), with what the layers do to c.
//
// A value is cut into three bf16 parts, a = a0 + a1 + a2 to 2^-26 of itself, in a pass over the operand, and of the nine products of
// parts the six largest are taken (what is left out is at most 2^-25 of |a b|).  The tensor core adds into fp32 but cuts the sum off
// instead of rounding it, a shift of some 0.3 last places towards zero per 16 products; so a0 b0 and the five small products have
// an accumulator each - cutting off the small one's sums is 2^-8 as bad - and after 128 k both are added to sums in registers, which are
// rounded.  What remains is below 2e-7 of a sum of 768 Gaussian products, less than fp32 multiply-adds in a row leave.
// Infinities and NaN come out as fp32 products would have them (cut3).
//
// Roles as in the 16-bit kernel: a persistent CTA per SM, tiles of 128 x 128; a stage is 64 k of three parts of either operand (96 KB,
// 24 MMAs), and there are two.  Bound by shared memory, which the MMAs read at 128 bytes per cycle while TMA writes half as much.
#include "lik_gemm.cuh"

namespace lik {
namespace {

constexpr int GF_EPI = 8, GF_PRODUCER = 8, GF_ISSUER = 9, GF_THREADS = 320;
constexpr int GF_PARTS = 3, GF_STAGES = 2, GF_OPERAND = 2 * GT_BOX_BYTES, GF_STAGE_BYTES = 2 * GF_PARTS * GF_OPERAND;
constexpr int GF_BN = 128, GF_DRAIN = 2;  // slabs of 64 k between two visits to the accumulators
constexpr int GF_SLOT = 32 * 32 * 4;
constexpr size_t GF_CTL_AT = (size_t)GF_STAGES * GF_STAGE_BYTES + GF_EPI * GF_SLOT;

struct GfMaps {
  CUtensorMap m[GT_MATRICES][GF_PARTS];
};
struct GfParams {
  GtProblem q[GT_PROBLEMS];
  int n_prob, units;
  bool raw;  // products only: several of them, or shares of one
  // what follows is for a single problem
  int act;
  const float *bias[2], *residual;
  float *out2, *kept[2];
  long long residual_stride, kept_stride;
  bool residual_vec, keep;
  int* status;
};
struct GfCtl {
  unsigned long long full[GF_STAGES], empty[GF_STAGES], acc_full[2], acc_empty[2];
  uint32_t tmem;
  WaitCtl wait;
};

template <int KIND>
__global__ void __launch_bounds__(GF_THREADS, 1) gemm_f32_kernel(const __grid_constant__ GfMaps maps, const __grid_constant__ GfParams p) {
  constexpr bool DUAL = KIND == GEMM_GATED;
  constexpr int OUT_N = DUAL ? GF_BN / 2 : GF_BN;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* gen = raw + (base - smem_u32(raw));
  GfCtl* ctl = reinterpret_cast<GfCtl*>(gen + GF_CTL_AT);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < GF_STAGES; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&ctl->acc_full[b]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[b]), GF_EPI);
    }
    ctl->wait.init();
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == GF_ISSUER) {
    tmem_alloc(smem_u32(&ctl->tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_the_kernel_in_front();
  const uint32_t tmem = ctl->tmem;  // accumulator pair b: a0 b0 in columns [256 b, 256 b + 128), the small products behind

  if (warp == GF_PRODUCER) {
    int s = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
      const GtUnit t = gt_unit<KIND == GEMM_LINEAR>(p.q, p.n_prob, u);
      const GtProblem& pr = p.q[t.q];
      for (int kb = t.kb_lo; kb < t.kb_hi; ++kb) {
        if (!wait_bar_all(&ctl->empty[s], phase ^ 1, &ctl->wait, p.status)) {
          ok = false;
          break;
        }
        const int seg = kb < pr.kb0 ? 0 : 1, k = (kb - (seg ? pr.kb0 : 0)) * GT_BK;
        if (elect_one()) {
          const uint32_t bar = smem_u32(&ctl->full[s]);
          mbar_arrive_expect_tx(bar, GF_STAGE_BYTES);
          const uint32_t dst = base + s * GF_STAGE_BYTES;
#pragma unroll
          for (int q = 0; q < GF_PARTS; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int ra = t.tm * 128 + h * GT_BOX, rb = t.tn * OUT_N + (DUAL ? 0 : h * GT_BOX);
              tma_load_2d(dst + q * GF_OPERAND + h * GT_BOX_BYTES, &maps.m[pr.a[seg]][q], pr.a_mn ? ra : k, pr.a_mn ? k : ra, bar);
              tma_load_2d(dst + (GF_PARTS + q) * GF_OPERAND + h * GT_BOX_BYTES, &maps.m[pr.b[DUAL ? h : seg]][q], pr.b_mn ? rb : k, pr.b_mn ? k : rb, bar);
            }
        }
        __syncwarp();
        ++issued;
        if (++s == GF_STAGES) s = 0, phase ^= 1;
      }
    }
    // the last stages' releases arrive here: not after this CTA is gone
    for (int i = 0; i < GF_STAGES && i < issued && ok; ++i) {
      const int back = issued - 1 - i;
      ok = wait_bar_all(&ctl->empty[back % GF_STAGES], (back / GF_STAGES) & 1, &ctl->wait, p.status);
    }
    if (!ok) {  // copies in flight land before the shared memory goes away
      const long long t0 = clock64();
      for (int i = 0; i < GF_STAGES && i < issued; ++i) {
        const int back = issued - 1 - i;
        while (!mbar_try_wait(smem_u32(&ctl->full[back % GF_STAGES]), (back / GF_STAGES) & 1) && clock64() - t0 < ctl->wait.limit) {
        }
      }
    }
  } else if (warp == GF_ISSUER) {
    int s = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t hi = (uint32_t)(smem_desc_sw128(0) >> 32);
    for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
      const GtUnit t = gt_unit<KIND == GEMM_LINEAR>(p.q, p.n_prob, u);
      const GtProblem& pr = p.q[t.q];
      const uint32_t a_lbo = (pr.a_mn ? GT_BOX_BYTES >> 4 : 1) << 16, b_lbo = (pr.b_mn ? GT_BOX_BYTES >> 4 : 1) << 16;
      const uint32_t a_step = pr.a_mn ? 128 : 2, b_step = pr.b_mn ? 128 : 2;
      const uint32_t idesc = instr_desc(1, GF_BN) | ((pr.a_mn ? 1u : 0u) << 15) | ((pr.b_mn ? 1u : 0u) << 16);
      for (int kb = t.kb_lo; kb < t.kb_hi && ok; ++it) {
        const int buf = it & 1, end = min(kb + GF_DRAIN, t.kb_hi);
        if (!(ok = wait_bar_all(&ctl->acc_empty[buf], ((it >> 1) & 1) ^ 1, &ctl->wait, p.status))) break;
        tc_fence_after();
        for (int first = kb; kb < end; ++kb) {
          if (!(ok = wait_bar_all(&ctl->full[s], phase, &ctl->wait, p.status))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t at = ((base + s * GF_STAGE_BYTES) & 0x3FFFFu) >> 4;
            const uint32_t a = at | a_lbo, b = (at + (GF_PARTS * GF_OPERAND >> 4)) | b_lbo;
            constexpr uint32_t PART = GF_OPERAND >> 4;
            const uint32_t big = tmem + buf * 256, small = big + 128;
            // (products of parts, the sums of the same accumulator apart from one another)
            constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {0, 0, 1, 2, 0, 1};
#pragma unroll
            for (int k = 0; k < GT_BK / 16; ++k)
#pragma unroll
              for (int q = 0; q < 6; ++q)
                tc_mma<false>(q ? small : big, a + PA[q] * PART + k * a_step, b + PB[q] * PART + k * b_step, hi, idesc, kb > first || k > 0 || q > 1);
            tc_commit(smem_u32(&ctl->empty[s]));
            if (kb + 1 == end) tc_commit(smem_u32(&ctl->acc_full[buf]));
          }
          __syncwarp();
          if (++s == GF_STAGES) s = 0, phase ^= 1;
        }
      }
    }
  } else {
    const int quad = warp & 3, part = warp >> 2;
    uint8_t* const slot = gen + GF_STAGES * GF_STAGE_BYTES + warp * GF_SLOT;
    int it = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
      const GtUnit t = gt_unit<KIND == GEMM_LINEAR>(p.q, p.n_prob, u);
      const GtProblem& pr = p.q[t.q];
      // the warp's 64 columns: two chunks of 32, of the result or (DUAL) one of the gate and the same one of up
      float sum[2][2][16];
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[0][0][j] = sum[0][1][j] = sum[1][0][j] = sum[1][1][j] = 0.0f;
      for (int kb = t.kb_lo; kb < t.kb_hi; kb += GF_DRAIN, ++it) {
        const int buf = it & 1;
        if (!(ok = wait_bar_all(&ctl->acc_full[buf], (it >> 1) & 1, &ctl->wait, p.status))) break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * 256 + ((uint32_t)(quad * 32) << 16);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = DUAL ? c * 64 + part * 32 + h * 16 : part * 64 + c * 32 + h * 16;
            float big[16], small[16];
            tmem_ld16(acc + col, big);
            tmem_ld16(acc + 128 + col, small);
            tmem_wait16(big);
            tmem_wait16(small);
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[c][h][j] += big[j] + small[j];
          }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->acc_empty[buf]));
      }
      if (!ok) break;
      const int row0 = t.tm * 128 + quad * 32, rows = pr.m - row0;
      if (rows <= 0) continue;
      // 32 x 32 of a matrix between memory and the lanes' rows, by way of the slot
      auto in = [&](const float* src, long long stride, int cols, bool vec, float (&f)[2][16]) {
        slot_fetch<float>(slot, lane, src, stride, rows, cols, vec);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        slot_get<float>(slot, lane, 0, f[0]);
        slot_get<float>(slot, lane, 1, f[1]);
        __syncwarp();
      };
      auto out = [&](float* dst, long long stride, int cols, bool vec, const float (&f)[2][16]) {
        slot_put<float>(slot, lane, 0, f[0]);
        slot_put<float>(slot, lane, 1, f[1]);
        __syncwarp();
        slot_store<float>(slot, lane, dst, stride, rows, cols, vec);
        __syncwarp();
      };
#pragma unroll
      for (int c = 0; c < (DUAL ? 1 : 2); ++c) {
        const int col = t.tn * OUT_N + (DUAL ? part * 32 : part * 64 + c * 32), left = pr.n - col;
        if (left <= 0) continue;
        float* const to = (float*)pr.out + t.split * pr.split_stride + row0 * pr.out_stride + col;
        float* const keep0 = p.kept[0] + row0 * p.kept_stride + col;
        float* const keep1 = p.kept[1] + row0 * p.kept_stride + col;
        float(&v)[2][16] = sum[c];
        if constexpr (KIND == GEMM_GATED_BWD) {
          float f[2][16];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            in(q ? keep1 : keep0, p.kept_stride, left, true, f);
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j / 16][j % 16] *= v[j / 16][j % 16];
            out(q ? p.out2 + row0 * pr.out_stride + col : to, pr.out_stride, left, true, f);
          }
        } else {
          if (KIND == GEMM_LINEAR && p.raw) {
            out(to, pr.out_stride, left, pr.out_vec, v);
            continue;
          }
          if (p.bias[0]) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j / 16][j % 16] += j < left ? __ldg(p.bias[0] + col + j) : 0.0f;
          }
          if constexpr (DUAL) {
            float(&w)[2][16] = sum[1];
            if (p.bias[1]) {
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j / 16][j % 16] += j < left ? __ldg(p.bias[1] + col + j) : 0.0f;
            }
            float f[2][16];
            with_activation_dev(p.act, [&](auto act) {
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j / 16][j % 16] = w[j / 16][j % 16] * act_slope<decltype(act)::value, true>(v[j / 16][j % 16], v[j / 16][j % 16]);
            });
            if (p.keep) {
              out(keep0, p.kept_stride, left, true, f);
              out(keep1, p.kept_stride, left, true, v);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j / 16][j % 16] *= w[j / 16][j % 16];
          } else {
            if (p.keep) out(keep0, p.kept_stride, left, true, v);
            if (p.act != LIK_ACT_NONE)
              with_activation_dev(p.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j / 16][j % 16] = act_value<decltype(act)::value, true>(v[j / 16][j % 16]);
              });
            if (p.residual) {
              float f[2][16];
              in(p.residual + row0 * p.residual_stride + col, p.residual_stride, left, p.residual_vec, f);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j / 16][j % 16] += f[j / 16][j % 16];
            }
          }
          out(to, pr.out_stride, left, pr.out_vec, v);
        }
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == GF_ISSUER) tmem_dealloc(tmem, 512);
}

// x = p0 + p1 + p2 in bf16, each the nearest to what the ones before leave.  A value that bf16 would round to infinity is cut off instead.  Of an infinite
// one the last part is infinite, which meets p0 of the other operand alone - in the first place it would meet that one's small parts, of any
// sign, and 0 - and p0 is its sign, for where that one is infinite too.  A NaN has no further parts.
__device__ __forceinline__ void cut3(float x, uint32_t (&p)[3]) {
  if (fabsf(x) <= 3.402823466e38f) {
    __nv_bfloat16 h = fabsf(x) > 3.3895e38f ? __float2bfloat16_rz(x) : __float2bfloat16_rn(x);
    p[0] = __bfloat16_as_ushort(h);
    float r = x - __bfloat162float(h);
    h = __float2bfloat16_rn(r);
    p[1] = __bfloat16_as_ushort(h);
    p[2] = __bfloat16_as_ushort(__float2bfloat16_rn(r - __bfloat162float(h)));
  } else {
    const uint32_t sign = __float_as_uint(x) >> 16 & 0x8000u;
    p[0] = x != x ? 0x7FC0u : sign | 0x3F80u;
    p[1] = 0u;
    p[2] = x != x ? 0u : sign | 0x7F80u;
  }
}
// matrices in their three parts, rows of whole 16-byte pieces (zeros behind the columns).  Bound by memory: 4 bytes in and 6 out per value.
struct CutJobs {
  Stored m[GT_MATRICES];
  void* parts[GT_MATRICES];
  long long end[GT_MATRICES];  // pieces up to and with this matrix
  int n;
};
__global__ void __launch_bounds__(256) cut_kernel(const __grid_constant__ CutJobs p) {
  after_the_kernel_in_front();
  const long long total = p.end[p.n - 1];
  for (long long g = blockIdx.x * 256ll + threadIdx.x; g < total; g += gridDim.x * 256ll) {
    int q = 0;
    while (g >= p.end[q]) ++q;
    const long long i = q ? g - p.end[q - 1] : g;
    const int cols = (int)p.m[q].cols, vecs = (cols + 7) / 8;
    const long long r = i / vecs;
    const int c = (int)(i - r * vecs) * 8;
    const float* s = (const float*)p.m[q].p + r * p.m[q].stride + c;
    float x[8];
    if (((uintptr_t)s & 15) == 0 && c + 8 <= cols) {
      load_vec<float, 8>(s, x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = c + j < cols ? s[j] : 0.0f;
    }
    uint32_t w[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo[3], hi[3];
      cut3(x[2 * j], lo);
      cut3(x[2 * j + 1], hi);
#pragma unroll
      for (int k = 0; k < 3; ++k) w[k][j] = lo[k] | hi[k] << 16;
    }
    uint4* dst = (uint4*)p.parts[q] + i;
    const long long part = p.m[q].rows * vecs;
#pragma unroll
    for (int k = 0; k < 3; ++k) dst[k * part] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
  }
}

GtPlan f32_plan(const GemmDesc* d, int n) {  // (a slab of k takes a CTA 1.5 to 1.9 us)
  return gt_plan(d, n, {6, 12}, 2, 0, [](const GemmDesc&) { return 1; }, [](const Stored& o) { return align_up((size_t)o.rows * o.padded() * 2 * GF_PARTS, 256); },
                 [](const GemmDesc&) { return 1 << 30; });
}
template <int KIND>
int run_f32(const GfMaps& maps, const GfParams& p, cudaStream_t st) {
  LIK_CUDA_OK(allow_smem<gemm_f32_kernel<KIND>>());
  return launch_after(gemm_f32_kernel<KIND>, p.units < sm_count() ? p.units : sm_count(), GF_THREADS, 1024 + GF_CTL_AT + sizeof(GfCtl), st, 1, maps, p);
}

}  // namespace

size_t gemm_f32_workspace(const GemmDesc* d, int n) { return f32_plan(d, n).total; }

int launch_gemm_f32(const GemmDesc* d, int n, void* ws, size_t ws_bytes, int* status, cudaStream_t st) {
  GtPlan pl = f32_plan(d, n);
  if (ws_bytes < pl.total || (pl.total && !ws)) {
    set_error("workspace too small");
    return LIK_ERR_WORKSPACE;
  }
  if (int rc = make_context_current()) return rc;
  GfMaps maps{};
  GfParams p{};
  CutJobs cuts{};
  long long total = 0;
  for (int i = 0; i < pl.n_mat; ++i) {
    const Stored& o = pl.mat[i];
    uint8_t* parts = (uint8_t*)ws + pl.copy[i];
    cuts.m[i] = o;
    cuts.parts[i] = parts;
    cuts.end[i] = total += o.rows * (o.padded() / 8);
    for (int q = 0; q < GF_PARTS; ++q)
      if (int rc = make_tmap_rows(&maps.m[i][q], parts + q * o.rows * o.padded() * 2, LIK_BF16, o.cols, o.rows, o.padded(), GT_BOX)) return rc;
  }
  cuts.n = pl.n_mat;
  const long long blocks = ceil_div(total, 256), most = 16ll * sm_count();
  if (int rc = launch_after(cut_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0, st, 1, cuts)) return rc;
  gt_outputs(pl, d, ws);
  p.act = d->act;
  for (int i = 0; i < 2; ++i) {
    p.bias[i] = (const float*)d->bias[i];
    p.kept[i] = (float*)d->kept[i];
  }
  p.out2 = (float*)d->out[1];
  p.keep = d->kind != GEMM_GATED_BWD && d->kept[0];
  p.kept_stride = d->kept_stride;
  p.residual = (const float*)d->residual;
  p.residual_stride = d->residual_stride;
  p.residual_vec = d->n % 4 == 0 && rows_of_pieces(d->residual, d->residual_stride, LIK_F32);
  p.status = status;
  for (int i = 0, end; i < n; i = end) {
    end = pl.group_end(i);
    p.n_prob = end - i;
    p.units = 0;
    for (int k = i; k < end; ++k) {
      p.q[k - i] = pl.q[k];
      p.q[k - i].unit0 = p.units;
      p.units += pl.units[k];
    }
    p.raw = p.n_prob > 1 || pl.splits[i] > 1;
    const int rc = d->kind == GEMM_GATED ? run_f32<GEMM_GATED>(maps, p, st) : (d->kind == GEMM_GATED_BWD ? run_f32<GEMM_GATED_BWD>(maps, p, st) : run_f32<GEMM_LINEAR>(maps, p, st));
    if (rc) return rc;
  }
  return launch_sum_splits<float>(pl, d, st);
}

}  // namespace lik
