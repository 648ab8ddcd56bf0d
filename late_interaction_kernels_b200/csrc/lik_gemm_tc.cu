// Matrix products on the tensor cores for 16-bit operands: c[m, n] = sum over k of a(m, k) b(n, k), either operand with its rows or
// its k contiguous in memory, and what the layers do to the elements of c (GemmKind) on the way out of tensor memory.
//
// A persistent kernel.  A unit is a tile of 256 x 256 for a pair of CTAs on two SMs (cta_group::2: each holds 128 rows of A, 128 of
// B and 128 rows of the accumulator), or of 128 x 128 for a single CTA where there are too few of the larger ones to fill the
// machine, over all of k or a share of it.  Per CTA:
//   producer warp  TMA boxes of 64 x 64 elements, two of A and two of B per slab of 64 k, into a ring of stages in shared memory.
//                  Where k is contiguous a box is 64 rows of 128 bytes, else 64 k of 128 bytes: the same box, and the MMA's
//                  descriptors say which (K-major or MN-major, 128-byte swizzle).  Rows and k behind the ends arrive as zeros.
//   issuer warp    (of the pair's first CTA) four MMAs of 16 k per slab, one elected lane issuing; two accumulators in tensor memory, so
//                  that the next unit's product runs while this unit's accumulator is read.
//   16 epilogue warps (8 where one needs more registers)  32 rows x a quarter (a half) of the columns each, 32 columns at a time: tensor memory ->
//                  registers, bias, activation, residual in fp32, one rounding, a swizzled slot in shared memory, and plain stores from there,
//                  neighbouring lanes on neighbouring pieces of a row (element by element where rows are not whole 16-byte pieces).
// The gated block's two projections are one unit: half of its columns are the gate's, half are up's.
// Products with few tiles and a long k are cut along k; the shares' fp32 sums go to the workspace and are added in their order.
#include "lik_gemm.cuh"

namespace lik {
namespace {

constexpr int GT_STAGE_BYTES = 4 * GT_BOX_BYTES, GT_STAGES = 5;
constexpr int GT_SLOTS_BYTES = 65536;  // of all epilogue warps: slots of 32 rows x 32 columns on their way in and out
constexpr size_t GT_CTL_AT = (size_t)GT_STAGES * GT_STAGE_BYTES + GT_SLOTS_BYTES;
// Epilogue warps: 16 where the registers of 18 warps (112 per thread) are enough, 8 for the gated product, which needs 120.
template <int KIND, bool F32_OUT>
struct GtWarps {
  static constexpr int EPI = KIND == GEMM_GATED || F32_OUT ? 8 : 16, PRODUCER = EPI, ISSUER = EPI + 1, THREADS = 32 * (EPI + 2);
};

struct GtMaps {
  CUtensorMap m[GT_MATRICES];
};
struct GtParams {
  GtProblem q[GT_PROBLEMS];
  int n_prob, units;
  bool bf16;
  // what follows is for a single problem
  int act;
  const void *bias[2], *residual;
  void *out2, *kept[2];  // kept: written, or read by GEMM_GATED_BWD
  long long residual_stride, kept_stride;
  bool bias_vec, residual_vec, keep;  // *_vec: rows of whole 16-byte pieces
  const void *a, *b;                  // the operands of z as the caller has them, k contiguous, and their rows' lengths
  long long a_stride, b_stride, k;
  const float *norm_a, *norm_b;
  int* status;
};
struct GtCtl {
  unsigned long long full[GT_STAGES], empty[GT_STAGES], acc_full[2], acc_empty[2];
  uint32_t tmem;
  WaitCtl wait;
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// this shared-memory address in the pair's first CTA
__device__ __forceinline__ uint32_t leader_addr(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_remote(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void gt_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 1)
    tma_load_2d(dst, map, x, y, bar);
  else  // (completes on a barrier of the pair's first CTA)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void gt_alloc(uint32_t dst, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(dst, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void gt_dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
template <int CG>
__device__ __forceinline__ void gt_mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    tc_mma<false>(d, a_lo, b_lo, hi, idesc, accumulate);
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the barrier at this address, in both CTAs of a pair, once the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void gt_commit(uint32_t bar) {
  if constexpr (CG == 1)
    tc_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// the chunks of a warp that have anything in them, in the order in which it comes to them
template <int CG, int OUT_N, int WARP_N>
__device__ __forceinline__ bool gt_chunk(const GtParams& p, int u, int c, int rank, int quad, int part, int& col, int& row0) {
  const GtUnit t = gt_unit<false>(p.q, 1, u);
  row0 = t.tm * (128 * CG) + rank * 128 + quad * 32;
  col = t.tn * OUT_N + part * WARP_N + c * 32;
  return row0 < p.q[0].m && col < p.q[0].n;
}

// Which of 16 z, columns of the lane's row, are above 0 (bit i: column col + i): those near relu's kink are taken by the warp's lanes together.
template <typename T>
__device__ __forceinline__ uint32_t above_kink(const GtParams& p, int row0, int col, int lane, const float (&v)[16]) {
  uint32_t above = 0, unsure = 0;
  const float norm = row0 + lane < p.q[0].m ? __ldg(p.norm_a + row0 + lane) : 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i += 4) {  // (there is room for whole vectors behind the lengths)
    const float4 n = __ldg(reinterpret_cast<const float4*>(p.norm_b + col + i));
    const float ns[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      above |= (v[i + j] > 0.0f ? 1u : 0u) << (i + j);
      unsure |= (fabsf(v[i + j]) < kink_bound(norm, ns[j], p.k) && col + i + j < p.q[0].n ? 1u : 0u) << (i + j);
    }
  }
  for (uint32_t lanes = __ballot_sync(0xffffffffu, unsure != 0); lanes; lanes &= lanes - 1) {
    const int l = __ffs(lanes) - 1;
    for (uint32_t cols = __shfl_sync(0xffffffffu, unsure, l); cols; cols &= cols - 1) {
      const int c = __ffs(cols) - 1;
      double z = exact_sum((const T*)p.a + (row0 + l) * p.a_stride, (const T*)p.b + (col + c) * p.b_stride, p.k, lane);
      if (p.bias[0]) z += (double)to_f32(((const T*)p.bias[0])[col + c]);
      if (lane == l) above = z > 0.0 ? above | 1u << c : above & ~(1u << c);
    }
  }
  return above;
}

// RES: with a residual (GEMM_LINEAR).  KINK: relu, for a backward pass.  O fp32: plain products, several of them, in fp32 or T, or shares of one.
template <int CG, int KIND, bool RES, bool KINK, typename T, typename O>
__global__ void __launch_bounds__(GtWarps<KIND, !std::is_same<T, O>::value>::THREADS, 1) gemm_tc_kernel(const __grid_constant__ GtMaps maps,
                                                                                                       const __grid_constant__ GtParams p) {
  using Warps = GtWarps<KIND, !std::is_same<T, O>::value>;
  constexpr int STAGES = GT_STAGES, EPI = Warps::EPI;
  constexpr bool DUAL = KIND == GEMM_GATED, MULTI = !std::is_same<T, O>::value;
  constexpr int BN = CG == 2 ? 256 : 128;          // columns of an accumulator
  constexpr int OUT_N = DUAL ? BN / 2 : BN;        // columns of the result in a unit
  constexpr int WARP_N = OUT_N / (EPI / 4), CHUNKS = WARP_N / 32;  // columns of an epilogue warp, 32 at a time
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* gen = raw + (base - smem_u32(raw));
  GtCtl* ctl = reinterpret_cast<GtCtl*>(gen + GT_CTL_AT);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&ctl->acc_full[b]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[b]), CG * EPI);
    }
    ctl->wait.init();
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == Warps::ISSUER) gt_alloc<CG>(smem_u32(&ctl->tmem), 2 * BN);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
  after_the_kernel_in_front();
  const uint32_t tmem = ctl->tmem;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (warp == Warps::PRODUCER) {
    int s = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = first; u < p.units && ok; u += step) {
      const GtUnit t = gt_unit<MULTI>(p.q, p.n_prob, u);
      const GtProblem& q = p.q[t.q];
      const int row_a = t.tm * (128 * CG) + rank * 128;
      const int row_b = DUAL ? t.tn * OUT_N : t.tn * BN + rank * (BN / CG);
      for (int kb = t.kb_lo; kb < t.kb_hi; ++kb) {
        if (!wait_bar_all(&ctl->empty[s], phase ^ 1, &ctl->wait, p.status)) {
          ok = false;
          break;
        }
        const int seg = kb < q.kb0 ? 0 : 1, k = (kb - (seg ? q.kb0 : 0)) * GT_BK;
        if (elect_one()) {
          const uint32_t local = smem_u32(&ctl->full[s]), bar = CG == 2 ? leader_addr(local) : local;
          if (rank == 0) mbar_arrive_expect_tx(local, CG * GT_STAGE_BYTES);
          const uint32_t dst = base + s * GT_STAGE_BYTES;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_a + i * GT_BOX;
            gt_load<CG>(dst + i * GT_BOX_BYTES, &maps.m[q.a[seg]], q.a_mn ? r : k, q.a_mn ? k : r, bar);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_b + (DUAL && CG == 1 ? 0 : i * GT_BOX);
            const CUtensorMap* map = &maps.m[q.b[DUAL ? (CG == 2 ? rank : i) : seg]];
            gt_load<CG>(dst + (2 + i) * GT_BOX_BYTES, map, q.b_mn ? r : k, q.b_mn ? k : r, bar);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == STAGES) s = 0, phase ^= 1;
      }
    }
    // the last stages' releases arrive here, perhaps from the other CTA: not after this one is gone
    for (int i = 0; i < STAGES && i < issued && ok; ++i) {
      const int back = issued - 1 - i;
      ok = wait_bar_all(&ctl->empty[back % STAGES], (back / STAGES) & 1, &ctl->wait, p.status);
    }
    if (!ok && rank == 0) {  // copies in flight land before the shared memory goes away
      const long long t0 = clock64();
      for (int i = 0; i < STAGES && i < issued; ++i) {
        const int back = issued - 1 - i;
        while (!mbar_try_wait(smem_u32(&ctl->full[back % STAGES]), (back / STAGES) & 1) && clock64() - t0 < ctl->wait.limit) {
        }
      }
    }
  } else if (warp == Warps::ISSUER) {
    if (rank == 0) {
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      // (leading dimension: the next 64 rows of an MN-major operand; k steps of 16: 32 bytes along a row, or 16 rows of 128 bytes)
      const uint32_t hi = (uint32_t)(smem_desc_sw128(0) >> 32);
      for (int u = first; u < p.units && ok; u += step, ++it) {
        const GtUnit t = gt_unit<MULTI>(p.q, p.n_prob, u);
        const GtProblem& q = p.q[t.q];
        const uint32_t a_lbo = (q.a_mn ? GT_BOX_BYTES >> 4 : 1) << 16, b_lbo = (q.b_mn ? GT_BOX_BYTES >> 4 : 1) << 16;
        const uint32_t a_step = q.a_mn ? 128 : 2, b_step = q.b_mn ? 128 : 2;
        const uint32_t idesc = (1u << 4) | ((p.bf16 ? 1u : 0u) << 7) | ((p.bf16 ? 1u : 0u) << 10) | ((q.a_mn ? 1u : 0u) << 15) | ((q.b_mn ? 1u : 0u) << 16) |
                               ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
        const int buf = it & 1;
        if (!wait_bar_all(&ctl->acc_empty[buf], ((it >> 1) & 1) ^ 1, &ctl->wait, p.status)) break;
        tc_fence_after();
        for (int kb = t.kb_lo; kb < t.kb_hi; ++kb) {
          if (!wait_bar_all(&ctl->full[s], phase, &ctl->wait, p.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t at = ((base + s * GT_STAGE_BYTES) & 0x3FFFFu) >> 4, a = at | a_lbo, b = (at + (2 * GT_BOX_BYTES >> 4)) | b_lbo;
#pragma unroll
            for (int k = 0; k < GT_BK / 16; ++k)
              gt_mma<CG>(tmem + buf * BN, a + k * a_step, b + k * b_step, hi, idesc, kb > t.kb_lo || k > 0);
            gt_commit<CG>(smem_u32(&ctl->empty[s]));
            if (kb + 1 == t.kb_hi) gt_commit<CG>(smem_u32(&ctl->acc_full[buf]));
          }
          __syncwarp();
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
    }
  } else {
    const int quad = warp & 3, part = warp >> 2;
    // What a chunk of 32 rows x 32 columns is added to or multiplied with is fetched into the slots that its results will leave from, while
    // the chunk before is dealt with.  Both ways are plain accesses, coalesced through the slot.  (TMA on the way in and out took the same
    // time and a tensor map per matrix on the host; a row's 64 bytes per lane straight from memory cost a wavefront of the load unit
    // per lane, 600 us against 530 in the gated backward of 65536 x 1024 x 4096.)
    constexpr int IN = KIND == GEMM_GATED_BWD ? 2 : (RES ? 1 : 0);
    constexpr int OUT = KIND == GEMM_GATED ? 3 : (KIND == GEMM_GATED_BWD || std::is_same<T, O>::value ? 2 : 1);
    constexpr int SLOT = 32 * 32 * (int)sizeof(O), WARP_BYTES = GT_SLOTS_BYTES / EPI;
    static_assert(OUT * SLOT <= WARP_BYTES, "room for a chunk's results");
    uint8_t* const to = gen + STAGES * GT_STAGE_BYTES + warp * WARP_BYTES;
    int in_unit = first, in_chunk = 0;
    auto fetch = [&] {  // for the next chunk that has anything in it
      int col = 0, row0 = 0;
      bool there = false;
      while (in_unit < p.units && !there) {
        there = gt_chunk<CG, OUT_N, WARP_N>(p, in_unit, in_chunk, rank, quad, part, col, row0);
        if (++in_chunk == CHUNKS) in_chunk = 0, in_unit += step;
      }
      if (!there) return;
      if constexpr (KIND == GEMM_GATED_BWD) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          slot_fetch<T>(to + i * SLOT, lane, (const T*)p.kept[i] + row0 * p.kept_stride + col, p.kept_stride, p.q[0].m - row0, p.q[0].n - col, true);
      } else if constexpr (RES) {
        slot_fetch<T>(to, lane, (const T*)p.residual + row0 * p.residual_stride + col, p.residual_stride, p.q[0].m - row0, p.q[0].n - col, p.residual_vec);
      }
    };
    if constexpr (IN > 0) fetch();
    bool ok = true;
    int it = 0;
    for (int u = first; u < p.units && ok; u += step, ++it) {
      const GtUnit t = gt_unit<MULTI>(p.q, p.n_prob, u);
      const GtProblem& q = p.q[t.q];
      const int buf = it & 1;
      if (!wait_bar_all(&ctl->acc_full[buf], (it >> 1) & 1, &ctl->wait, p.status)) break;
      tc_fence_after();
      const int row0 = t.tm * (128 * CG) + rank * 128 + quad * 32;
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(quad * 32) << 16);
      const uint32_t release = CG == 2 ? leader_addr(smem_u32(&ctl->acc_empty[buf])) : smem_u32(&ctl->acc_empty[buf]);
#pragma unroll 1
      for (int c = 0; c < CHUNKS; ++c) {
        const int in_tile = part * WARP_N + c * 32, col = t.tn * OUT_N + in_tile, left = q.n - col;
        const bool live = row0 < q.m && left > 0;
        if (!live) {
          if (c + 1 == CHUNKS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) CG == 2 ? arrive_remote(release) : mbar_arrive(release);
          }
          continue;
        }
        if constexpr (IN > 0) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[16], w[16];
          Raw16<T> bias[2];
          tmem_ld16(acc + in_tile + 16 * h, v);
          if constexpr (DUAL) tmem_ld16(acc + BN / 2 + in_tile + 16 * h, w);
          if constexpr (KIND != GEMM_GATED_BWD && !MULTI) {
            if (p.bias[0]) bias[0].load((const T*)p.bias[0] + col + 16 * h, left - 16 * h, p.bias_vec);
            if (DUAL && p.bias[1]) bias[1].load((const T*)p.bias[1] + col + 16 * h, left - 16 * h, p.bias_vec);
          }
          tmem_wait16(v);
          if constexpr (DUAL) tmem_wait16(w);
          if (h == 1 && c + 1 == CHUNKS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) CG == 2 ? arrive_remote(release) : mbar_arrive(release);
          }
          if constexpr (KIND == GEMM_GATED_BWD) {  // (rounded to T: they are the operands of the next products, which take 16 bits)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float f[16];
              slot_get<T>(to + j * SLOT, lane, h, f);
#pragma unroll
              for (int i = 0; i < 16; i += 2) mul2(Pair(f[i], f[i + 1]), Pair(v[i], v[i + 1])).get(f[i], f[i + 1]);
              slot_put<O>(to + j * SLOT, lane, h, f);
            }
          } else {
            if constexpr (!MULTI) {
              if (p.bias[0]) bias[0].add_to(v);
            }
            if constexpr (DUAL) {
              if (p.bias[1]) bias[1].add_to(w);
            }
            if constexpr (!MULTI) {
              // what the backward pass reads is rounded to T, as what autograd keeps between two 16-bit layers is: z, or both factors and h (a gradient
              // is off by its own rounding and one of these, of a gated block two; fp32 would be twice the bytes of what is kept, written and read again)
              if constexpr (KINK) {
                const uint32_t above = above_kink<T>(p, row0, col + 16 * h, lane, v);
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const bool up = above >> i & 1u;
                  if constexpr (DUAL) f[i] = up ? w[i] : 0.0f;
                  else f[i] = keep_side<T>(v[i], up);
                }
                slot_put<O>(to + SLOT, lane, h, f);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = act_value<LIK_ACT_RELU, false>(v[i]);
                if constexpr (DUAL) slot_put<O>(to + (OUT - 1) * SLOT, lane, h, v);
              } else if (DUAL && p.keep) {
                float f[16];
                with_activation_dev(p.act, [&](auto act) {
#pragma unroll
                  for (int i = 0; i < 16; i += 2) {
                    act_pair<decltype(act)::value, true>(v[i], v[i + 1], f[i], f[i + 1]);
                    mul2(Pair(w[i], w[i + 1]), Pair(f[i], f[i + 1])).get(f[i], f[i + 1]);
                  }
                });
                slot_put<O>(to + SLOT, lane, h, f);
                slot_put<O>(to + (OUT - 1) * SLOT, lane, h, v);
              } else if (p.act != LIK_ACT_NONE) {
                if (!DUAL && p.keep) slot_put<O>(to + (OUT - 1) * SLOT, lane, h, v);
                with_activation_dev(p.act, [&](auto act) {
#pragma unroll
                  for (int i = 0; i < 16; i += 2) act_pair<decltype(act)::value, false>(v[i], v[i + 1], v[i], v[i + 1]);
                });
              }
            }
            if constexpr (DUAL) {
#pragma unroll
              for (int i = 0; i < 16; i += 2) mul2(Pair(v[i], v[i + 1]), Pair(w[i], w[i + 1])).get(v[i], v[i + 1]);
            } else if constexpr (RES) {
              Raw16<T> r;
              slot_get_raw(to, lane, h, r);
              r.add_to(v);
            }
            slot_put<O>(to, lane, h, v);
          }
        }
        __syncwarp();
        const int rows = q.m - row0;
        const long long at = t.split * q.split_stride + row0 * q.out_stride + col;
        if constexpr (MULTI) {
          if (q.out_f32) slot_store<float>(to, lane, (float*)q.out + at, q.out_stride, rows, left, q.out_vec);
          else slot_store_as<T>(to, lane, (T*)q.out + at, q.out_stride, rows, left, q.out_vec);
        } else {
          slot_store<O>(to, lane, (O*)q.out + at, q.out_stride, rows, left, q.out_vec);
        }
        if constexpr (KIND == GEMM_GATED_BWD) {
          slot_store<O>(to + SLOT, lane, (O*)p.out2 + row0 * q.out_stride + col, q.out_stride, rows, left, true);
        } else if constexpr (OUT > 1) {
          if (p.keep) {
            slot_store<O>(to + SLOT, lane, (O*)p.kept[0] + row0 * p.kept_stride + col, p.kept_stride, rows, left, true);
            if constexpr (DUAL) slot_store<O>(to + 2 * SLOT, lane, (O*)p.kept[1] + row0 * p.kept_stride + col, p.kept_stride, rows, left, true);
          }
        }
        __syncwarp();
        if constexpr (IN > 0) fetch();
      }
    }
    if constexpr (IN > 0) asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncwarp();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // nobody still arrives here, and no MMA of the pair reads this shared memory
  if (warp == Warps::ISSUER) gt_dealloc<CG>(tmem, 2 * BN);
}

// Matrices whose rows TMA cannot address, copied to rows of 16 bytes (the columns behind them are zeros).  A lane reads every 32nd element of
// a row's 512, so that neighbours read neighbours, and the warp puts the pieces together in shared memory.
constexpr int REPACK_COLS = 512;
struct RepackJobs {
  Stored m[GT_MATRICES];
  void* to[GT_MATRICES];
  long long end[GT_MATRICES];  // stretches of 512 columns up to and with this matrix
  int n;
};
__global__ void __launch_bounds__(256) repack_kernel(const __grid_constant__ RepackJobs p) {
  __shared__ __align__(16) uint16_t part[8][REPACK_COLS];
  after_the_kernel_in_front();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (long long g = blockIdx.x * 8ll + warp; g < p.end[p.n - 1]; g += gridDim.x * 8ll) {
    int q = 0;
    while (g >= p.end[q]) ++q;
    const long long i = q ? g - p.end[q - 1] : g;
    const int cols = (int)p.m[q].cols, vecs = (cols + 7) / 8, per_row = (vecs * 8 + REPACK_COLS - 1) / REPACK_COLS;
    const long long r = i / per_row;
    const int c0 = (int)(i - r * per_row) * REPACK_COLS;
    const uint16_t* s = (const uint16_t*)p.m[q].p + r * p.m[q].stride + c0;
    uint4* dst = (uint4*)p.to[q] + r * vecs + c0 / 8;
    uint16_t e[REPACK_COLS / 32];
#pragma unroll
    for (int j = 0; j < REPACK_COLS / 32; ++j) e[j] = c0 + j * 32 + lane < cols ? s[j * 32 + lane] : (uint16_t)0;
#pragma unroll
    for (int j = 0; j < REPACK_COLS / 32; ++j) part[warp][j * 32 + lane] = e[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < REPACK_COLS / 256; ++j) {
      const int v = j * 32 + lane;
      if (c0 / 8 + v < vecs) dst[v] = *reinterpret_cast<const uint4*>(&part[warp][v * 8]);
    }
    __syncwarp();
  }
}

// Pairs of CTAs take tiles of 256 x 256 where there are enough of them, or enough k to cut into shares, for every pair; else single CTAs
// tiles of 128 x 128.  A slab of k takes a CTA that is alone with its tile 0.2 us, so shares pay from 12 slabs spared on: 512 rows, 2048 x 768 (6 of 32
// slabs each) 12.3 us whole, 9.0 cut; 1024 rows, 1024 x 1024 (7 of 16) 9.4 and 10.3.  (Four CTAs of a cluster that add their sums up in shared
// memory, without the pass: 10.4 and 9.9; their start costs what the pass does.)
// An addition of 16 products cuts off some 1.6 steps (2^-23) of the accumulator, one-sided: of 65536 terms of one sign 4e-4 of their sum was missing, of 8192
// it is 2e-5.  So fp32 results, which have no rounding that would hide it, are sums of shares of at most 8192 of k, added with rounding (1024 x 1024
// of 65536 tokens: 1.9e-5, where a library's fp32 product is off by up to 1.7e-5); for 16-bit results one accumulator goes through so much of k that a
// tenth or so of what their own rounding may be off comes of it.
GtPlan tc_plan(const GemmDesc* d, int n) {
  auto cg = [](const GemmDesc& g) {
    const long long tiles = ceil_div(g.m, 256) * ceil_div(g.n, g.kind == GEMM_GATED ? 128 : 256), pairs = sm_count() / 2;
    const bool cuttable = gemm_plain(g) && g.m > 128 && g.n > 128;
    return tiles >= pairs || (cuttable && tiles * ceil_div(g.k[0] + g.k[1], GT_BK) >= 16 * pairs) ? 2 : 1;
  };
  return gt_plan(d, n, {16, 96}, 4, 12, cg, [](const Stored& o) { return o.aligned() ? (size_t)0 : align_up((size_t)o.rows * o.padded() * 2, 256); },
                 [](const GemmDesc& g) { return (g.out_dtype == LIK_F32 ? 8192 : (g.out_dtype == LIK_F16 ? 16384 : 65536)) / GT_BK; });
}

template <int CG, int KIND, bool RES, bool KINK, typename T, typename O>
int run_tc(const GtMaps& maps, const GtParams& p, cudaStream_t st) {
  LIK_CUDA_OK((allow_smem<gemm_tc_kernel<CG, KIND, RES, KINK, T, O>>()));
  const int slots = sm_count() / CG;
  return launch_after(gemm_tc_kernel<CG, KIND, RES, KINK, T, O>, (unsigned)((p.units < slots ? p.units : slots) * CG), GtWarps<KIND, !std::is_same<T, O>::value>::THREADS,
                      1024 + GT_CTL_AT + sizeof(GtCtl), st, CG, maps, p);
}
template <int KIND, bool RES, bool KINK, typename T, typename O>
int run_tc(int cg, const GtMaps& maps, const GtParams& p, cudaStream_t st) {
  return cg == 2 ? run_tc<2, KIND, RES, KINK, T, O>(maps, p, st) : run_tc<1, KIND, RES, KINK, T, O>(maps, p, st);
}
template <typename T>
int run_tc(int kind, bool multi, int cg, const GtMaps& maps, const GtParams& p, cudaStream_t st) {
  const bool kink = p.keep && p.act == LIK_ACT_RELU;
  if (kind == GEMM_GATED_BWD) return run_tc<GEMM_GATED_BWD, false, false, T, T>(cg, maps, p, st);
  if (kind == GEMM_GATED) return kink ? run_tc<GEMM_GATED, false, true, T, T>(cg, maps, p, st) : run_tc<GEMM_GATED, false, false, T, T>(cg, maps, p, st);
  if (multi) return run_tc<GEMM_LINEAR, false, false, T, float>(cg, maps, p, st);
  if (p.residual) return kink ? run_tc<GEMM_LINEAR, true, true, T, T>(cg, maps, p, st) : run_tc<GEMM_LINEAR, true, false, T, T>(cg, maps, p, st);
  return kink ? run_tc<GEMM_LINEAR, false, true, T, T>(cg, maps, p, st) : run_tc<GEMM_LINEAR, false, false, T, T>(cg, maps, p, st);
}

}  // namespace

size_t gemm_tc_workspace(const GemmDesc* d, int n) { return tc_plan(d, n).total; }

int launch_gemm_tc(const GemmDesc* d, int n, void* ws, size_t ws_bytes, int* status, cudaStream_t st) {
  GtPlan pl = tc_plan(d, n);
  if (ws_bytes < pl.total || (pl.total && !ws)) {
    set_error("workspace too small");
    return LIK_ERR_WORKSPACE;
  }
  if (int rc = make_context_current()) return rc;
  GtMaps maps{};
  GtParams p{};
  RepackJobs repack{};
  for (int i = 0; i < pl.n_mat; ++i) {
    Stored o = pl.mat[i];
    if (pl.copied[i]) {
      void* to = (char*)ws + pl.copy[i];
      repack.m[repack.n] = o;
      repack.to[repack.n] = to;
      repack.end[repack.n] = (repack.n ? repack.end[repack.n - 1] : 0) + o.rows * ceil_div(o.padded(), REPACK_COLS);
      ++repack.n;
      o.p = to;
      o.stride = o.padded();
    }
    if (o.rows == 1) o.stride = o.padded();
    if (int rc = make_tmap_rows(&maps.m[i], o.p, d->dtype, o.cols, o.rows, o.stride, GT_BOX)) return rc;
  }
  if (repack.n) {
    const long long blocks = ceil_div(repack.end[repack.n - 1], 8), most = 8ll * sm_count();
    if (int rc = launch_after(repack_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0, st, 1, repack)) return rc;
  }
  gt_outputs(pl, d, ws);
  p.bf16 = d->dtype == LIK_BF16;
  p.act = d->act;
  p.bias_vec = d->n % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    p.bias[i] = d->bias[i];
    p.kept[i] = d->kept[i];
    if (d->bias[i] && ((uintptr_t)d->bias[i] & 15)) p.bias_vec = false;
  }
  p.out2 = d->out[1];
  p.keep = d->kind != GEMM_GATED_BWD && d->kept[0];
  p.a = d->a[0].p;
  p.b = d->b[0].p;
  p.a_stride = d->a[0].row;
  p.b_stride = d->b[0].row;
  p.k = d->k[0];
  p.norm_a = d->norm_a;
  p.norm_b = d->norm_b;
  p.kept_stride = d->kept_stride;
  p.residual = d->residual;
  p.residual_stride = d->residual_stride;
  p.residual_vec = d->n % 8 == 0 && rows_of_pieces(d->residual, d->residual_stride, d->dtype);
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
    const bool multi = p.n_prob > 1 || pl.splits[i] > 1 || d[i].out_dtype == LIK_F32;
    const int rc = d->dtype == LIK_F16 ? run_tc<__half>(d->kind, multi, pl.cg[i], maps, p, st) : run_tc<__nv_bfloat16>(d->kind, multi, pl.cg[i], maps, p, st);
    if (rc) return rc;
  }
  return d->dtype == LIK_F16 ? launch_sum_splits<__half>(pl, d, st) : launch_sum_splits<__nv_bfloat16>(pl, d, st);
}

}  // namespace lik
