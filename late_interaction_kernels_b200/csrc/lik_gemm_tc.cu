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
//   8 epilogue warps  32 rows x half of the columns each, 32 columns at a time: tensor memory -> registers, bias, activation,
//                  residual in fp32, one rounding, a swizzled slot in shared memory, a TMA store (which leaves out what lies behind the
//                  matrix).  Rows that TMA cannot address (not multiples of 16 bytes) are written from the slot by plain stores.
// The gated block's two projections are one unit: half of its columns are the gate's, half are up's.
// Products with few tiles and a long k are cut along k; the shares' fp32 sums go to the workspace and are added in their order.
#include "lik_layers.cuh"
#include "lik_tc.cuh"
#include "lik_tc_ptx.cuh"

namespace lik {
namespace {

constexpr int GT_EPI_WARPS = 8, GT_PRODUCER = 8, GT_ISSUER = 9, GT_THREADS = 320;
constexpr int GT_BK = 64, GT_BOX = 64, GT_BOX_BYTES = GT_BOX * GT_BK * 2;
constexpr int GT_STAGE_BYTES = 4 * GT_BOX_BYTES, GT_MAX_STAGES = 5;
// Shared memory: stages of the operands, and per epilogue warp slots of 32 rows x 32 columns on their way in and out.  Kernels whose
// epilogue reads matrices give a stage for the slots of those.
template <bool READS>
struct GtShape {
  static constexpr int STAGES = READS ? 4 : 5, SLOTS_BYTES = READS ? 12288 : 8192;
  static constexpr size_t SLOTS_AT = (size_t)STAGES * GT_STAGE_BYTES, CTL_AT = SLOTS_AT + GT_EPI_WARPS * SLOTS_BYTES;
};

struct GtMaps {
  CUtensorMap a[2], b[2], out[2], kept[2], residual;
};
struct GtParams {
  int m, n, n_seg;
  int kb0, kb_total, kb_per, tiles, tiles_n, units;
  bool a_mn, b_mn, bf16, bias_vec, residual_tma;
  int act;
  const void *bias[2], *residual;
  long long residual_stride;
  bool keep;      // factors are written
  void* direct;   // not NULL: out is written by plain stores, rows of out_stride
  long long out_stride;
  int* status;
};
struct GtCtl {
  unsigned long long full[GT_MAX_STAGES], empty[GT_MAX_STAGES], acc_full[2], acc_empty[2], in_full[GT_EPI_WARPS][2];
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
__device__ __forceinline__ void gt_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x),
               "r"(y), "r"(0), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void gt_store(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
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

struct GtUnit {
  int tm, tn, split, kb_lo, kb_hi;
};
__device__ __forceinline__ GtUnit gt_unit(const GtParams& p, int u) {
  GtUnit t;
  t.split = u / p.tiles;
  const int i = u - t.split * p.tiles;
  t.tm = i / p.tiles_n;
  t.tn = i - t.tm * p.tiles_n;
  t.kb_lo = t.split * p.kb_per;
  t.kb_hi = min(t.kb_lo + p.kb_per, p.kb_total);
  return t;
}

// 32 lanes x 16 columns of tensor memory; the registers may be read after tmem_wait16
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
                 "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait16(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]),
                 "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}

// 16 consecutive elements, the first n of them there: fetched early, unpacked when they are wanted
template <typename T>
struct Raw16 {
  uint4 u[2];
  __device__ __forceinline__ void load(const T* p, int n, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < 2; ++i) u[i] = 8 * i < n ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = (2 * i < n ? (uint32_t)q[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)q[2 * i + 1] << 16 : 0u);
      u[0] = make_uint4(w[0], w[1], w[2], w[3]);
      u[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  __device__ __forceinline__ void add_to(float (&v)[16]) const {
    float f[16];
    get(f);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += f[i];
  }
  __device__ __forceinline__ void get(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unpack2(u[i].x, f[8 * i + 0], f[8 * i + 1], T());
      unpack2(u[i].y, f[8 * i + 2], f[8 * i + 3], T());
      unpack2(u[i].z, f[8 * i + 4], f[8 * i + 5], T());
      unpack2(u[i].w, f[8 * i + 6], f[8 * i + 7], T());
    }
  }
};

// 16-byte piece c of row r in a slot of 32 rows of ROW bytes: the 64-byte or 128-byte swizzle of the slot's tensor map, which also keeps
// the lanes' accesses, a row each, apart
template <int ROW>
__device__ __forceinline__ int slot_offset(int r, int c) {
  return ROW == 64 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 128 + ((c ^ (r & 7)) << 4);
}
// columns [16 h, 16 h + 16) of the lane's row
template <typename O>
__device__ __forceinline__ void slot_put(uint8_t* s, int lane, int h, const float (&v)[16]) {
  constexpr int ROW = 32 * (int)sizeof(O);
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<float4*>(s + slot_offset<ROW>(lane, h * 4 + c)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  } else {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      *reinterpret_cast<uint4*>(s + slot_offset<ROW>(lane, h * 2 + c)) =
          make_uint4(pack2(v[8 * c], v[8 * c + 1], O()), pack2(v[8 * c + 2], v[8 * c + 3], O()), pack2(v[8 * c + 4], v[8 * c + 5], O()),
                     pack2(v[8 * c + 6], v[8 * c + 7], O()));
  }
}
template <typename T>
__device__ __forceinline__ void slot_get(const uint8_t* s, int lane, int h, float (&f)[16]) {
  Raw16<T> r;
#pragma unroll
  for (int c = 0; c < 2; ++c) r.u[c] = *reinterpret_cast<const uint4*>(s + slot_offset<64>(lane, h * 2 + c));
  r.get(f);
}

// the chunks of a warp that have anything in them, in the order in which it comes to them
template <int CG, int OUT_N>
__device__ __forceinline__ bool gt_chunk(const GtParams& p, int u, int c, int rank, int quad, int half, int& col, int& row0) {
  const GtUnit t = gt_unit(p, u);
  row0 = t.tm * (128 * CG) + rank * 128 + quad * 32;
  col = t.tn * OUT_N + half * (OUT_N / 2) + c * 32;
  return row0 < p.m && col < p.n;
}

// RES: a residual that comes by TMA (GEMM_LINEAR)
template <int CG, int KIND, bool RES, typename T, typename O>
__global__ void __launch_bounds__(GT_THREADS, 1) gemm_tc_kernel(const __grid_constant__ GtMaps maps, const __grid_constant__ GtParams p) {
  using Shape = GtShape<RES || KIND == GEMM_GATED_BWD>;
  constexpr int STAGES = Shape::STAGES;
  constexpr bool DUAL = KIND == GEMM_GATED;
  constexpr int BN = CG == 2 ? 256 : 128;          // columns of an accumulator
  constexpr int OUT_N = DUAL ? BN / 2 : BN;        // columns of the result in a unit
  constexpr int CHUNKS = OUT_N / 64;               // 32-column chunks of an epilogue warp
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* gen = raw + (base - smem_u32(raw));
  GtCtl* ctl = reinterpret_cast<GtCtl*>(gen + Shape::CTL_AT);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&ctl->acc_full[b]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[b]), CG * GT_EPI_WARPS);
      for (int w = 0; w < GT_EPI_WARPS; ++w) mbar_init(smem_u32(&ctl->in_full[w][b]), 1);
    }
    ctl->wait.init();
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == GT_ISSUER) gt_alloc<CG>(smem_u32(&ctl->tmem), 2 * BN);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (warp == GT_PRODUCER) {
    int s = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = first; u < p.units && ok; u += step) {
      const GtUnit t = gt_unit(p, u);
      const int row_a = t.tm * (128 * CG) + rank * 128;
      const int row_b = DUAL ? t.tn * OUT_N : t.tn * BN + rank * (BN / CG);
      for (int kb = t.kb_lo; kb < t.kb_hi; ++kb) {
        if (!wait_bar_all(&ctl->empty[s], phase ^ 1, &ctl->wait, p.status)) {
          ok = false;
          break;
        }
        const int seg = kb < p.kb0 ? 0 : 1, k = (kb - (seg ? p.kb0 : 0)) * GT_BK;
        if (elect_one()) {
          const uint32_t local = smem_u32(&ctl->full[s]), bar = CG == 2 ? leader_addr(local) : local;
          if (rank == 0) mbar_arrive_expect_tx(local, CG * GT_STAGE_BYTES);
          const uint32_t dst = base + s * GT_STAGE_BYTES;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_a + i * GT_BOX;
            gt_load<CG>(dst + i * GT_BOX_BYTES, &maps.a[seg], p.a_mn ? r : k, p.a_mn ? k : r, bar);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_b + (DUAL && CG == 1 ? 0 : i * GT_BOX);
            const CUtensorMap* map = DUAL ? (CG == 2 ? &maps.b[rank] : &maps.b[i]) : &maps.b[seg];
            gt_load<CG>(dst + (2 + i) * GT_BOX_BYTES, map, p.b_mn ? r : k, p.b_mn ? k : r, bar);
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
  } else if (warp == GT_ISSUER) {
    if (rank == 0) {
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      // (leading dimension: the next 64 rows of an MN-major operand; k steps of 16: 32 bytes along a row, or 16 rows of 128 bytes)
      const uint32_t hi = (uint32_t)(smem_desc_sw128(0) >> 32);
      const uint32_t a_lbo = (p.a_mn ? GT_BOX_BYTES >> 4 : 1) << 16, b_lbo = (p.b_mn ? GT_BOX_BYTES >> 4 : 1) << 16;
      const uint32_t a_step = p.a_mn ? 128 : 2, b_step = p.b_mn ? 128 : 2;
      const uint32_t idesc = (1u << 4) | ((p.bf16 ? 1u : 0u) << 7) | ((p.bf16 ? 1u : 0u) << 10) | ((p.a_mn ? 1u : 0u) << 15) | ((p.b_mn ? 1u : 0u) << 16) |
                             ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
      for (int u = first; u < p.units && ok; u += step, ++it) {
        const GtUnit t = gt_unit(p, u);
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
    const int quad = warp & 3, half = warp >> 2;
    // What a chunk of 32 rows x 32 columns is added to or multiplied with comes by TMA, two chunks ahead, and what becomes of it leaves by
    // TMA: IN matrices in and OUT matrices out, a slot each.
    constexpr int IN = KIND == GEMM_GATED_BWD ? 2 : (RES ? 1 : 0);
    constexpr int OUT = KIND == GEMM_GATED ? 3 : (KIND == GEMM_GATED_BWD || std::is_same<T, O>::value ? 2 : 1);
    constexpr int SLOT = 32 * 32 * (int)sizeof(O), OUT_SETS = (Shape::SLOTS_BYTES - 2 * IN * SLOT) / (OUT * SLOT);
    static_assert(OUT_SETS >= 1, "room for a chunk's results");
    const uint32_t in_base = base + STAGES * GT_STAGE_BYTES + warp * Shape::SLOTS_BYTES, out_base = in_base + 2 * IN * SLOT;
    uint8_t* const in_gen = gen + (in_base - base);
    uint8_t* const out_gen = gen + (out_base - base);
    int in_unit = IN ? first : p.units, in_chunk = 0, issued = 0, taken = 0, set = 0;
    // fetches for the next chunk that has anything in it, into the slots that were emptied last
    auto fetch = [&] {
      int col = 0, row0 = 0;
      bool there = false;
      while (in_unit < p.units && !there) {
        there = gt_chunk<CG, OUT_N>(p, in_unit, in_chunk, rank, quad, half, col, row0);
        if (++in_chunk == CHUNKS) in_chunk = 0, in_unit += step;
      }
      if (!there) return;
      const int slot = issued & 1;
      if (lane == 0) {
        const uint32_t bar = smem_u32(&ctl->in_full[warp][slot]);
        mbar_arrive_expect_tx(bar, IN * SLOT);
#pragma unroll
        for (int q = 0; q < IN; ++q) gt_load_3d(in_base + (slot * IN + q) * SLOT, KIND == GEMM_GATED_BWD ? &maps.kept[q] : &maps.residual, col, row0, bar);
      }
      ++issued;
    };
    if constexpr (IN > 0) {
      fetch();
      fetch();
    }
    bool ok = true;
    int it = 0;
    for (int u = first; u < p.units && ok; u += step, ++it) {
      const GtUnit t = gt_unit(p, u);
      const int buf = it & 1;
      if (!wait_bar_all(&ctl->acc_full[buf], (it >> 1) & 1, &ctl->wait, p.status)) break;
      tc_fence_after();
      const int row0 = t.tm * (128 * CG) + rank * 128 + quad * 32, row = row0 + lane;
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(quad * 32) << 16);
      const uint32_t release = CG == 2 ? leader_addr(smem_u32(&ctl->acc_empty[buf])) : smem_u32(&ctl->acc_empty[buf]);
#pragma unroll 1
      for (int c = 0; c < CHUNKS; ++c) {
        const int in_tile = half * (OUT_N / 2) + c * 32, col = t.tn * OUT_N + in_tile, left = p.n - col;
        const bool live = row0 < p.m && left > 0;
        if (!live) {
          if (c + 1 == CHUNKS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) CG == 2 ? arrive_remote(release) : mbar_arrive(release);
          }
          continue;
        }
        uint8_t* const to = out_gen + set * OUT * SLOT;
        const uint8_t* from = in_gen + (taken & 1) * IN * SLOT;
        if (IN > 0 && !(ok = wait_bar_all(&ctl->in_full[warp][taken & 1], (taken >> 1) & 1, &ctl->wait, p.status))) break;
        // (the slots' last stores have been read out of them)
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(OUT_SETS - 1) : "memory");
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[16], w[16];
          Raw16<T> bias[2], res;
          tmem_ld16(acc + in_tile + 16 * h, v);
          if constexpr (DUAL) tmem_ld16(acc + BN / 2 + in_tile + 16 * h, w);
          if constexpr (KIND != GEMM_GATED_BWD) {
            if (p.bias[0]) bias[0].load((const T*)p.bias[0] + col + 16 * h, left - 16 * h, p.bias_vec);
            if (DUAL && p.bias[1]) bias[1].load((const T*)p.bias[1] + col + 16 * h, left - 16 * h, p.bias_vec);
            if (!DUAL && !RES && p.residual)  // rows that TMA cannot address
              res.load((const T*)p.residual + (row < p.m ? row * p.residual_stride + col + 16 * h : 0), row < p.m ? left - 16 * h : 0, false);
          }
          tmem_wait16(v);
          if constexpr (DUAL) tmem_wait16(w);
          if (h == 1 && c + 1 == CHUNKS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) CG == 2 ? arrive_remote(release) : mbar_arrive(release);
          }
          if constexpr (KIND == GEMM_GATED_BWD) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float f[16];
              slot_get<T>(from + q * SLOT, lane, h, f);
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] *= v[i];
              slot_put<O>(to + q * SLOT, lane, h, f);
            }
          } else {
            if (p.bias[0]) bias[0].add_to(v);
            if constexpr (DUAL) {
              if (p.bias[1]) bias[1].add_to(w);
            }
            if constexpr (std::is_same<T, O>::value) {
              if (DUAL && p.keep) {
                float f[16];
                with_activation_dev(p.act, [&](auto act) {
#pragma unroll
                  for (int i = 0; i < 16; ++i) f[i] = w[i] * act_slope<decltype(act)::value, false>(v[i], v[i]);
                });
                slot_put<O>(to + SLOT, lane, h, f);
                slot_put<O>(to + (OUT - 1) * SLOT, lane, h, v);
              } else if (p.act != LIK_ACT_NONE) {
                if (!DUAL && p.keep) slot_put<O>(to + (OUT - 1) * SLOT, lane, h, v);
                with_activation_dev(p.act, [&](auto act) {
#pragma unroll
                  for (int i = 0; i < 16; ++i) v[i] = act_value<decltype(act)::value, false>(v[i]);
                });
              }
            }
            if constexpr (DUAL) {
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] *= w[i];
            } else if constexpr (RES) {
              float f[16];
              slot_get<T>(from, lane, h, f);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] += f[i];
            } else if (p.residual) {
              res.add_to(v);
            }
            slot_put<O>(to, lane, h, v);
          }
        }
        if constexpr (IN > 0) ++taken;
        fence_proxy_async();
        __syncwarp();
        if constexpr (IN > 0) fetch();
        if (lane == 0) {
          const uint32_t src = out_base + set * OUT * SLOT;
          if (KIND == GEMM_GATED_BWD || !p.direct) gt_store(&maps.out[0], src, col, row0, t.split);
          if (KIND == GEMM_GATED_BWD) gt_store(&maps.out[1], src + SLOT, col, row0, 0);
          if (KIND != GEMM_GATED_BWD && OUT > 1 && p.keep) {
            gt_store(&maps.kept[0], src + SLOT, col, row0, 0);
            if (DUAL) gt_store(&maps.kept[1], src + (OUT - 1) * SLOT, col, row0, 0);
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if (KIND == GEMM_LINEAR && p.direct) {
          constexpr int PIECE = 16 / (int)sizeof(O);
          const int rows = min(32, p.m - row0);
          if (lane < left)
            for (int r = 0; r < rows; ++r)
              ((O*)p.direct)[(row0 + r) * p.out_stride + col + lane] =
                  *reinterpret_cast<const O*>(to + slot_offset<32 * (int)sizeof(O)>(r, lane / PIECE) + (lane % PIECE) * sizeof(O));
          __syncwarp();
        }
        set = set + 1 == OUT_SETS ? 0 : set + 1;
      }
    }
    // (after an expired wait: what was fetched and not taken lands before the shared memory goes away)
    const long long t0 = clock64();
    for (; taken < issued; ++taken)
      while (!mbar_try_wait(smem_u32(&ctl->in_full[warp][taken & 1]), (taken >> 1) & 1) && clock64() - t0 < ctl->wait.limit) {
      }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // nobody still arrives here, and no MMA of the pair reads this shared memory
  if (warp == GT_ISSUER) gt_dealloc<CG>(tmem, 2 * BN);
}

// out[i][j] = sum over splits of partial[split][i][j], in their order
template <typename O>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* __restrict__ partial, int splits, long long m, int n, int stride, O* __restrict__ out,
                                                         long long out_stride) {
  const int per_row = (n + 3) / 4;
  const long long total = m * per_row;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * 4;
    const float* src = partial + r * stride + c;
    float4 v = *reinterpret_cast<const float4*>(src);
    for (int s = 1; s < splits; ++s) {
      const float4 w = *reinterpret_cast<const float4*>(src + s * m * stride);
      v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
    O* o = out + r * out_stride + c;
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < n) o[j] = from_f32<O>(f[j]);
  }
}

// rows that TMA cannot address, copied to rows of 16 bytes (the columns behind them are zeros)
__global__ void __launch_bounds__(256) repack_kernel(const uint16_t* __restrict__ src, long long src_stride, long long rows, int cols, uint4* __restrict__ dst,
                                                     int vecs) {
  const long long total = rows * vecs;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / vecs;
    const int c = (int)(i - r * vecs) * 8;
    const uint16_t* s = src + r * src_stride + c;
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = c + j < cols ? s[j] : 0;
    dst[i] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (EncodeFn)p : nullptr;
  }();
  return fn;
}
// [splits][rows][cols] in pieces of 32 x 32, for the way in or out
int store_map(CUtensorMap* map, void* p, int dtype, long long cols, long long rows, long long splits, long long stride) {
  const long long item = (long long)dtype_size(dtype);
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)splits};
  const cuuint64_t strides[2] = {(cuuint64_t)(stride * item), (cuuint64_t)(stride * item * rows)};
  const cuuint32_t box[3] = {32, 32, 1}, step[3] = {1, 1, 1};
  const CUtensorMapDataType dt = dtype == LIK_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : (dtype == LIK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  const CUresult r = encode_fn()(map, dt, 3, p, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, dtype == LIK_F32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                 CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return LIK_ERR_CUDA;
  }
  return LIK_OK;
}

// an operand as it lies in memory
struct Stored {
  const void* p;
  long long rows, cols, stride;
  bool mn;  // rows are k
  bool aligned() const { return ((uintptr_t)p & 15) == 0 && (rows == 1 || stride % 8 == 0); }
  long long padded() const { return (cols + 7) / 8 * 8; }
};
Stored stored(const GemmOperand& o, long long rows, long long k) {
  if (o.k == 1) return {o.p, rows, k, o.row, false};
  return {o.p, k, rows, o.k, true};
}
bool tma_out(const void* p, long long stride, int dtype) { return ((uintptr_t)p & 15) == 0 && stride * (long long)dtype_size(dtype) % 16 == 0; }

struct GtPlan {
  int cg, tiles_m, tiles_n, kb[2], kb_total, kb_per, splits;
  size_t copy[4], partial, total;  // offsets; copies of a[0], a[1], b[0], b[1] where they are needed
  bool copies[4];
  int partial_stride;
};
GtPlan gt_plan(const GemmDesc& d) {
  GtPlan pl{};
  const bool dual = d.kind == GEMM_GATED;
  const int sms = sm_count();
  for (int s = 0; s < d.n_seg; ++s) pl.kb_total += pl.kb[s] = (int)ceil_div(d.k[s], GT_BK);
  auto tiles = [&](int cg) { return ceil_div(d.m, 128 * cg) * ceil_div(d.n, (cg == 2 ? 256 : 128) / (dual ? 2 : 1)); };
  const bool plain = d.kind == GEMM_LINEAR && d.act == LIK_ACT_NONE && !d.bias[0] && !d.residual && !d.kept[0];
  pl.cg = tiles(2) * 2 >= sms || (plain && pl.kb_total >= 64 && d.m > 128 && d.n > 128) ? 2 : 1;
  pl.tiles_m = (int)ceil_div(d.m, 128 * pl.cg);
  pl.tiles_n = (int)ceil_div(d.n, (pl.cg == 2 ? 256 : 128) / (dual ? 2 : 1));
  const long long t = (long long)pl.tiles_m * pl.tiles_n, slots = sms / pl.cg;
  pl.splits = 1;
  if (plain && t < slots && pl.kb_total >= 8) {
    long long want = slots / t;
    if (want > pl.kb_total / 4) want = pl.kb_total / 4;
    if (want > 1) pl.splits = (int)want;
  }
  pl.kb_per = (int)ceil_div(pl.kb_total, pl.splits);
  pl.splits = (int)ceil_div(pl.kb_total, pl.kb_per);
  size_t off = 0;
  for (int i = 0; i < 4; ++i) {
    const bool is_b = i >= 2;
    const int s = i & 1;
    if (is_b ? s >= (dual ? 2 : d.n_seg) : s >= d.n_seg) continue;
    const Stored o = stored(is_b ? d.b[s] : d.a[s], is_b ? d.n : d.m, d.k[dual ? 0 : s]);
    pl.copies[i] = !o.aligned();
    if (pl.copies[i]) {
      pl.copy[i] = off;
      off += align_up((size_t)o.rows * o.padded() * 2, 256);
    }
  }
  if (pl.splits > 1) {
    pl.partial = off;
    pl.partial_stride = (d.n + 3) / 4 * 4;
    off += align_up((size_t)pl.splits * d.m * pl.partial_stride * sizeof(float), 256);
  }
  pl.total = off;
  return pl;
}

template <int CG, int KIND, bool RES, typename T, typename O>
int run_tc(const GtMaps& maps, const GtParams& p, cudaStream_t st) {
  LIK_CUDA_OK((allow_smem<gemm_tc_kernel<CG, KIND, RES, T, O>>()));
  const int slots = sm_count() / CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.units < slots ? p.units : slots) * CG));
  cfg.blockDim = dim3(GT_THREADS);
  cfg.dynamicSmemBytes = 1024 + GtShape<RES || KIND == GEMM_GATED_BWD>::CTL_AT + sizeof(GtCtl);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LIK_CUDA_OK(cudaLaunchKernelEx(&cfg, gemm_tc_kernel<CG, KIND, RES, T, O>, maps, p));
  count_launch();
  return LIK_OK;
}
template <int KIND, bool RES, typename T, typename O>
int run_tc(int cg, const GtMaps& maps, const GtParams& p, cudaStream_t st) {
  return cg == 2 ? run_tc<2, KIND, RES, T, O>(maps, p, st) : run_tc<1, KIND, RES, T, O>(maps, p, st);
}
template <typename T>
int run_tc(int kind, bool f32_out, int cg, const GtMaps& maps, const GtParams& p, cudaStream_t st) {
  if (kind == GEMM_GATED) return run_tc<GEMM_GATED, false, T, T>(cg, maps, p, st);
  if (kind == GEMM_GATED_BWD) return run_tc<GEMM_GATED_BWD, false, T, T>(cg, maps, p, st);
  if (f32_out) return run_tc<GEMM_LINEAR, false, T, float>(cg, maps, p, st);
  return p.residual_tma ? run_tc<GEMM_LINEAR, true, T, T>(cg, maps, p, st) : run_tc<GEMM_LINEAR, false, T, T>(cg, maps, p, st);
}

}  // namespace

bool gemm_tc_supported(const GemmDesc& d) {
  if ((d.dtype != LIK_F16 && d.dtype != LIK_BF16) || !tmap_available() || !encode_fn()) return false;
  if (d.m >= (1ll << 31) || d.k[0] >= (1ll << 31) || d.k[1] >= (1ll << 31)) return false;
  const long long tiles = ceil_div(d.m, 128) * ceil_div(d.n, 64);
  return tiles < (1ll << 30);
}
size_t gemm_tc_workspace(const GemmDesc& d) { return gt_plan(d).total; }

int launch_gemm_tc(const GemmDesc& d, void* ws, size_t ws_bytes, int* status, cudaStream_t st) {
  const GtPlan pl = gt_plan(d);
  if (ws_bytes < pl.total || (pl.total && !ws)) {
    set_error("workspace too small");
    return LIK_ERR_WORKSPACE;
  }
  // tensor maps are made by the driver, which wants the device's context to be current: a thread that has made no call of the runtime's
  // yet (autograd's, on the first backward of a process) has none until it says which device it is on
  int dev = 0;
  LIK_CUDA_OK(cudaGetDevice(&dev));
  LIK_CUDA_OK(cudaSetDevice(dev));
  const bool dual = d.kind == GEMM_GATED;
  GtMaps maps{};
  GtParams p{};
  for (int i = 0; i < 4; ++i) {
    const bool is_b = i >= 2;
    const int s = i & 1;
    if (is_b ? s >= (dual ? 2 : d.n_seg) : s >= d.n_seg) continue;
    Stored o = stored(is_b ? d.b[s] : d.a[s], is_b ? d.n : d.m, d.k[dual ? 0 : s]);
    (is_b ? p.b_mn : p.a_mn) = o.mn;
    if (pl.copies[i]) {
      void* to = (char*)ws + pl.copy[i];
      const long long vecs = o.padded() / 8, blocks = ceil_div(o.rows * vecs, 256), most = 16ll * sm_count();
      repack_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>((const uint16_t*)o.p, o.stride, o.rows, (int)o.cols, (uint4*)to, (int)vecs), count_launch();
      LIK_CUDA_OK(cudaGetLastError());
      o.p = to;
      o.stride = o.padded();
    }
    if (o.rows == 1) o.stride = o.padded();
    if (int rc = make_tmap_rows(is_b ? &maps.b[s] : &maps.a[s], o.p, d.dtype, o.cols, o.rows, o.stride, GT_BOX)) return rc;
  }
  const bool f32_out = pl.splits > 1 || d.out_dtype == LIK_F32;
  if (pl.splits > 1) {
    if (int rc = store_map(&maps.out[0], (char*)ws + pl.partial, LIK_F32, d.n, d.m, pl.splits, pl.partial_stride)) return rc;
  } else {
    for (int i = 0; i < (d.kind == GEMM_GATED_BWD ? 2 : 1); ++i) {
      if (tma_out(d.out[i], d.out_stride, d.out_dtype)) {
        if (int rc = store_map(&maps.out[i], d.out[i], d.out_dtype, d.n, d.m, 1, d.out_stride)) return rc;
      } else {
        p.direct = d.out[i];
      }
    }
  }
  p.keep = d.kind != GEMM_GATED_BWD && d.kept[0];
  for (int i = 0; d.kept[0] && i < (d.kind == GEMM_LINEAR ? 1 : 2); ++i)
    if (int rc = store_map(&maps.kept[i], d.kept[i], d.dtype, d.n, d.m, 1, d.kept_stride)) return rc;
  p.m = (int)d.m;
  p.n = d.n;
  p.n_seg = d.n_seg;
  p.kb0 = pl.kb[0];
  p.kb_total = pl.kb_total;
  p.kb_per = pl.kb_per;
  p.tiles_n = pl.tiles_n;
  p.tiles = pl.tiles_m * pl.tiles_n;
  p.units = p.tiles * pl.splits;
  p.bf16 = d.dtype == LIK_BF16;
  p.act = d.act;
  p.bias_vec = d.n % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    p.bias[i] = d.bias[i];
    if (d.bias[i] && ((uintptr_t)d.bias[i] & 15)) p.bias_vec = false;
  }
  p.residual = d.residual;
  p.residual_stride = d.residual_stride;
  p.residual_tma = d.residual && tma_out(d.residual, d.residual_stride, d.dtype);
  if (p.residual_tma)
    if (int rc = store_map(&maps.residual, const_cast<void*>(d.residual), d.dtype, d.n, d.m, 1, d.residual_stride)) return rc;
  p.out_stride = d.out_stride;
  p.status = status;
  int rc = d.dtype == LIK_F16 ? run_tc<__half>(d.kind, f32_out, pl.cg, maps, p, st) : run_tc<__nv_bfloat16>(d.kind, f32_out, pl.cg, maps, p, st);
  if (rc || pl.splits == 1) return rc;
  const float* partial = (const float*)((char*)ws + pl.partial);
  const long long blocks = ceil_div(d.m * ((d.n + 3) / 4), 256), most = 16ll * sm_count();
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  if (d.out_dtype == LIK_F32) sum_splits_kernel<float><<<grid, 256, 0, st>>>(partial, pl.splits, d.m, d.n, pl.partial_stride, (float*)d.out[0], d.out_stride), count_launch();
  else if (d.out_dtype == LIK_F16) sum_splits_kernel<__half><<<grid, 256, 0, st>>>(partial, pl.splits, d.m, d.n, pl.partial_stride, (__half*)d.out[0], d.out_stride), count_launch();
  else sum_splits_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(partial, pl.splits, d.m, d.n, pl.partial_stride, (__nv_bfloat16*)d.out[0], d.out_stride), count_launch();
  LIK_CUDA_OK(cudaGetLastError());
  return LIK_OK;
}

}  // namespace lik
