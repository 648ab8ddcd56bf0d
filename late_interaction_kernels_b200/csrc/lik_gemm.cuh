// What the tensor-core products share (sm_100a): accumulator loads, slots of 32 x 32 elements on the way between an epilogue warp's
// registers (a lane its row) and memory (neighbouring lanes on neighbouring pieces of a row), operands as they lie in memory, the sum of
// the shares of a product that was cut along k.
#pragma once

#include "lik_layers.cuh"
#include "lik_tc.cuh"
#include "lik_tc_ptx.cuh"

namespace lik {
namespace {

constexpr int GT_BK = 64, GT_BOX = 64, GT_BOX_BYTES = GT_BOX * GT_BK * 2;

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
  // v += these: a multiply-add of 16-bit factors, one of them 1, takes them as they are
  __device__ __forceinline__ void add_to(float (&v)[16]) const {
    const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same<T, __half>::value)
        asm("{\n\t.reg .b16 l, h, one;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 one, 0x3C00;\n\tfma.rn.f32.f16 %0, l, one, %0;\n\tfma.rn.f32.f16 %1, h, one, %1;\n\t}"
            : "+f"(v[2 * i]), "+f"(v[2 * i + 1])
            : "r"(w[i]));
      else
        asm("{\n\t.reg .b16 l, h, one;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 one, 0x3F80;\n\tfma.rn.f32.bf16 %0, l, one, %0;\n\tfma.rn.f32.bf16 %1, h, one, %1;\n\t}"
            : "+f"(v[2 * i]), "+f"(v[2 * i + 1])
            : "r"(w[i]));
    }
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

// 16-byte piece c of row r in a slot of 32 rows of ROW bytes: shuffled within its row so that
// the lanes' accesses, a row each, keep apart
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
__device__ __forceinline__ void slot_get_raw(const uint8_t* s, int lane, int h, Raw16<T>& r) {
#pragma unroll
  for (int c = 0; c < 2; ++c) r.u[c] = *reinterpret_cast<const uint4*>(s + slot_offset<64>(lane, h * 2 + c));
}
template <typename T>
__device__ __forceinline__ void slot_get(const uint8_t* s, int lane, int h, float (&f)[16]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 u = *reinterpret_cast<const float4*>(s + slot_offset<128>(lane, h * 4 + c));
      f[4 * c] = u.x, f[4 * c + 1] = u.y, f[4 * c + 2] = u.z, f[4 * c + 3] = u.w;
    }
  } else {
    Raw16<T> r;
    slot_get_raw(s, lane, h, r);
    r.get(f);
  }
}
// Slot -> 32 rows of 32 columns in memory and back, neighbouring lanes on neighbouring pieces of a row.  vec: rows of whole 16-byte pieces
// (what lies between n and the next multiple of 16 bytes belongs to the row); else element by element.
template <typename O>
__device__ __forceinline__ void slot_store(const uint8_t* s, int lane, O* p, long long stride, int rows, int cols, bool vec) {
  constexpr int ROW = 32 * (int)sizeof(O), PIECES = ROW / 16, PER = 16 / (int)sizeof(O);
  if (vec) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int i = lane + 32 * j, r = i / PIECES, c = i % PIECES;
      const uint4 u = *reinterpret_cast<const uint4*>(s + slot_offset<ROW>(r, c));
      if (r < rows && c * PER < cols) *reinterpret_cast<uint4*>(p + r * stride + c * PER) = u;
    }
  } else if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows) p[r * stride + lane] = *reinterpret_cast<const O*>(s + slot_offset<ROW>(r, lane / PER) + (lane % PER) * sizeof(O));
  }
}
template <typename T>
__device__ __forceinline__ void slot_fetch(uint8_t* s, int lane, const T* p, long long stride, int rows, int cols, bool vec) {
  constexpr int ROW = 32 * (int)sizeof(T), PIECES = ROW / 16, PER = 16 / (int)sizeof(T);
  if (vec) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int i = lane + 32 * j, r = i / PIECES, c = i % PIECES;
      const bool there = r < rows && c * PER < cols;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(s + slot_offset<ROW>(r, c))), "l"(there ? p + r * stride + c * PER : p),
                   "r"(there ? 16 : 0)
                   : "memory");
    }
  } else if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows) *reinterpret_cast<T*>(s + slot_offset<ROW>(r, lane / PER) + (lane % PER) * sizeof(T)) = p[r * stride + lane];
  }
}

// a slot of fp32 written as another type
template <typename T>
__device__ __forceinline__ void slot_store_as(const uint8_t* s, int lane, T* p, long long stride, int rows, int cols, bool vec) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = lane + 32 * j, r = i / 4, c = i % 4;
      const float4 x = *reinterpret_cast<const float4*>(s + slot_offset<128>(r, 2 * c)), y = *reinterpret_cast<const float4*>(s + slot_offset<128>(r, 2 * c + 1));
      if (r < rows && c * 8 < cols)
        *reinterpret_cast<uint4*>(p + r * stride + c * 8) = make_uint4(pack2(x.x, x.y, T()), pack2(x.z, x.w, T()), pack2(y.x, y.y, T()), pack2(y.z, y.w, T()));
    }
  } else if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows) p[r * stride + lane] = from_f32<T>(*reinterpret_cast<const float*>(s + slot_offset<128>(r, lane / 4) + (lane % 4) * 4));
  }
}

// ---------------------------------------------------------------------------------------------
// A product's tiles, each cut along k into `splits` shares, are its units.  One launch computes one product, its units dealt to the CTAs (or
// pairs) in turn, or up to four whose units all run side by side.
// ---------------------------------------------------------------------------------------------
constexpr int GT_PROBLEMS = 4, GT_MATRICES = 8;
struct GtProblem {
  int m, n;
  int kb0, kb_total, kb_per, tiles, tiles_n, unit0;  // slabs of 64 k: of the first segment, of both, of a share
  bool a_mn, b_mn, out_vec, out_f32;
  unsigned char a[2], b[2];                          // which matrices, per segment (GEMM_GATED: b of the gate and of up)
  void* out;
  long long out_stride, split_stride;
};
struct GtUnit {
  int q, tm, tn, split, kb_lo, kb_hi;
};
template <bool MULTI>
__device__ __forceinline__ GtUnit gt_unit(const GtProblem (&q)[GT_PROBLEMS], int n, int u) {
  GtUnit t;
  t.q = 0;
  if constexpr (MULTI)
    while (t.q + 1 < n && u >= q[t.q + 1].unit0) ++t.q;
  const GtProblem& p = q[t.q];
  const int v = u - p.unit0;
  t.split = v / p.tiles;
  const int i = v - t.split * p.tiles;
  t.tm = i / p.tiles_n;
  t.tn = i - t.tm * p.tiles_n;
  t.kb_lo = t.split * p.kb_per;
  t.kb_hi = min(t.kb_lo + p.kb_per, p.kb_total);
  return t;
}

// the shares of products that were cut along k, added in their order and rounded
struct SumJob {
  const float* partial;
  int splits, n, stride;
  long long m, end, out_stride;  // end: pieces of four columns up to and with this job
  void* out;
  bool out_f32;
};
struct SumJobs {
  SumJob q[GT_PROBLEMS];
  int n;
};
__device__ __forceinline__ float4 sum_shares(const SumJob& j, long long r, int c) {
  const float* src = j.partial + r * j.stride + c;
  float4 v = *reinterpret_cast<const float4*>(src);
  for (int s = 1; s < j.splits; ++s) {
    const float4 w = *reinterpret_cast<const float4*>(src + s * j.m * j.stride);
    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
  }
  return v;
}
template <typename T>
__global__ void __launch_bounds__(256) sum_splits_kernel(const __grid_constant__ SumJobs p) {
  after_the_kernel_in_front();
  const long long total = p.q[p.n - 1].end;
  for (long long g = blockIdx.x * 256ll + threadIdx.x; g < total; g += gridDim.x * 256ll) {
    int q = 0;
    while (g >= p.q[q].end) ++q;
    const SumJob& j = p.q[q];
    const long long i = q ? g - p.q[q - 1].end : g;
    const int per_row = (j.n + 3) / 4;
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * 4;
    const float4 v = sum_shares(j, r, c);
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < j.n) {
        if (j.out_f32) ((float*)j.out)[r * j.out_stride + c + k] = f[k];
        else ((T*)j.out)[r * j.out_stride + c + k] = from_f32<T>(f[k]);
      }
  }
}
// ... and what GEMM_LINEAR does to them
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ SumJob j, const __grid_constant__ GemmDesc d) {
  after_the_kernel_in_front();
  const int per_row = (j.n + 3) / 4, lane = threadIdx.x & 31;
  with_activation_dev(d.act, [&](auto act) {
    for (long long first = blockIdx.x * 256ll + threadIdx.x - lane; first < j.end; first += gridDim.x * 256ll) {  // (whole warps)
      const long long i = first + lane < j.end ? first + lane : j.end - 1, r = i / per_row;
      const int c = (int)(i - r * per_row) * 4;
      const float4 v = sum_shares(j, r, c);
      const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool there = first + lane < j.end && c + k < j.n;
        bool above = true;
        if constexpr (decltype(act)::value == LIK_ACT_RELU) {
          const float z = there && d.bias[0] ? f[k] + to_f32(((const T*)d.bias[0])[c + k]) : f[k];
          above = z > 0.0f;
          if constexpr (sizeof(T) == 2) {
            if (d.norm_a) above = above_zero<T>(d, r, there ? c + k : 0, z, there, lane);
          }
        }
        if (there) gemm_element<T, T, GEMM_LINEAR, decltype(act)::value>(d, r, c + k, f[k], 0.0f, above);
      }
    }
  });
}

// an operand as it lies in memory
struct Stored {
  const void* p;
  long long rows, cols, stride;
  // as TMA wants 16-bit rows
  bool aligned() const { return ((uintptr_t)p & 15) == 0 && (rows == 1 || stride % 8 == 0); }
  long long padded() const { return (cols + 7) / 8 * 8; }
};
// mn: its rows are k
inline Stored stored(const GemmOperand& o, long long rows, long long k, bool mn) {
  return mn ? Stored{o.p, k, rows, o.k} : Stored{o.p, rows, k, o.row};
}
// Whether k runs along the rows in memory: one answer for all `n` operands of a side, since a unit's MMAs read them the same way.  Where a matrix is
// a single column wide, both of its steps may be 1, or that of k alone may not be (a column of a wider matrix): across fits either.
inline bool stored_across(const GemmOperand* o, int n) {
  for (int i = 0; i < n; ++i)
    if (o[i].k != 1) return true;
  return false;
}
inline bool rows_of_pieces(const void* p, long long stride, int dtype) { return ((uintptr_t)p & 15) == 0 && stride * (long long)dtype_size(dtype) % 16 == 0; }

// What a call is made of: the problems, the matrices that they read (each brought to its layout once, whoever reads it), the workspace.
struct GtPlan {
  int n, n_mat;
  GtProblem q[GT_PROBLEMS];  // without addresses; unit0 as if alone
  int cg[GT_PROBLEMS], splits[GT_PROBLEMS], units[GT_PROBLEMS];
  Stored mat[GT_MATRICES];
  bool copied[GT_MATRICES];
  size_t copy[GT_MATRICES], partial[GT_PROBLEMS], total;  // offsets
  // problems [i, end) that a launch takes together
  int group_end(int i) const {
    int end = i + 1;
    long long sum = units[i];
    while (end < n && cg[end] == cg[i] && sum + units[end] <= sm_count() / cg[i]) sum += units[end++];
    return end;
  }
};
// cg_of: CTAs that share a tile of (128 CTAs)^2; cut_from: slabs of k from which a product is cut into shares, of at least `share` slabs each, if
// that spares a CTA `spare` of them; copy_bytes: of a matrix that is not read as it lies in memory, 0 otherwise.  cut_from[1] is for one of up to
// four products, which share a launch if they are not cut: a step of 3500 x 768 through a gated block of 2048 took 154 us cut from 40 slabs on, 119
// from 96 on; with the two products of a linear layer it is the other way round, 41 and 45 us.  A problem is planned as if it were alone, so its
// result does not depend on which others are asked for.  slabs_of: slabs that one accumulator may go through, for the accuracy's sake.
template <typename CgOf, typename CopyBytes, typename SlabsOf>
GtPlan gt_plan(const GemmDesc* d, int n, const int (&cut_from)[2], int share, int spare, CgOf&& cg_of, CopyBytes&& copy_bytes, SlabsOf&& slabs_of) {
  GtPlan pl{};
  pl.n = n;
  size_t off = 0;
  for (int i = 0; i < n; ++i) {
    const bool dual = d[i].kind == GEMM_GATED;
    GtProblem& q = pl.q[i];
    const int cg = pl.cg[i] = cg_of(d[i]);
    q.m = (int)d[i].m;
    q.n = d[i].n;
    q.tiles_n = (int)ceil_div(q.n, 128 * cg / (dual ? 2 : 1));
    q.tiles = (int)ceil_div(q.m, 128 * cg) * q.tiles_n;
    for (int s = 0; s < d[i].n_seg; ++s) {
      const int kb = (int)ceil_div(d[i].k[s], GT_BK);
      q.kb_total += kb;
      if (s == 0) q.kb0 = kb;
    }
    q.a_mn = stored_across(d[i].a, d[i].n_seg);
    q.b_mn = stored_across(d[i].b, dual ? 2 : d[i].n_seg);
    for (int s = 0; s < 2; ++s)
      for (int is_b = 0; is_b < 2; ++is_b) {
        if (s >= (is_b && dual ? 2 : d[i].n_seg)) continue;
        const Stored o = is_b ? stored(d[i].b[s], d[i].n, d[i].k[dual ? 0 : s], q.b_mn) : stored(d[i].a[s], d[i].m, d[i].k[s], q.a_mn);
        int at = 0;
        while (at < pl.n_mat && !(pl.mat[at].p == o.p && pl.mat[at].rows == o.rows && pl.mat[at].cols == o.cols && pl.mat[at].stride == o.stride)) ++at;
        if (at == pl.n_mat) pl.mat[pl.n_mat++] = o;
        (is_b ? q.b : q.a)[s] = (unsigned char)at;
      }
    // a share of k for every slot, where the time that this saves is worth the pass that adds the shares up (2.5 us)
    long long ideal = ceil_div((long long)q.tiles * q.kb_total, sm_count() / cg);
    if (ideal < share) ideal = share;
    long long s = d[i].kind == GEMM_LINEAR && q.kb_total >= cut_from[d[i].several] && q.kb_total >= 2 * ideal && q.kb_total - ideal >= spare ? q.kb_total / ideal : 1;
    if (d[i].kind == GEMM_LINEAR) {
      long long least = ceil_div(q.kb_total, slabs_of(d[i]));
      if (least > (1 << 30) / q.tiles) least = (1 << 30) / q.tiles;  // (units are counted in 32 bits)
      if (s < least) s = least;
    }
    q.kb_per = (int)ceil_div(q.kb_total, s);
    pl.splits[i] = (int)ceil_div(q.kb_total, q.kb_per);
    pl.units[i] = q.tiles * pl.splits[i];
    if (pl.splits[i] > 1) {
      pl.partial[i] = off;
      off += align_up((size_t)pl.splits[i] * q.m * ((q.n + 3) / 4 * 4) * sizeof(float), 256);
    }
  }
  for (int i = 0; i < pl.n_mat; ++i) {
    const size_t bytes = copy_bytes(pl.mat[i]);
    pl.copied[i] = bytes > 0;
    pl.copy[i] = off;
    off += bytes;
  }
  pl.total = off;
  return pl;
}
// the addresses: where each problem's sums go
inline void gt_outputs(GtPlan& pl, const GemmDesc* d, void* ws) {
  for (int i = 0; i < pl.n; ++i) {
    GtProblem& q = pl.q[i];
    if (pl.splits[i] > 1) {
      q.out = (char*)ws + pl.partial[i];
      q.out_stride = (q.n + 3) / 4 * 4;
      q.split_stride = q.m * q.out_stride;
      q.out_vec = q.out_f32 = true;
    } else {
      q.out = d[i].out[0];
      q.out_stride = d[i].out_stride;
      q.out_f32 = d[i].out_dtype == LIK_F32;
      q.out_vec = rows_of_pieces(q.out, q.out_stride, d[i].out_dtype);
    }
  }
}
template <typename T>
int launch_sum_splits(const GtPlan& pl, const GemmDesc* d, cudaStream_t st) {
  SumJobs jobs{};
  long long total = 0;
  for (int i = 0; i < pl.n; ++i) {
    if (pl.splits[i] == 1) continue;
    const GtProblem& q = pl.q[i];
    SumJob& j = jobs.q[jobs.n++];
    j.partial = (const float*)q.out;
    j.splits = pl.splits[i];
    j.n = q.n;
    j.stride = (int)q.out_stride;
    j.m = q.m;
    j.end = total += (long long)q.m * ((q.n + 3) / 4);
    j.out_stride = d[i].out_stride;
    j.out = d[i].out[0];
    j.out_f32 = d[i].out_dtype == LIK_F32;
  }
  if (!jobs.n) return LIK_OK;
  const long long blocks = ceil_div(total, 256), most = 16ll * sm_count();
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  return gemm_plain(d[0]) ? launch_after(sum_splits_kernel<T>, grid, 256, 0, st, 1, jobs) : launch_after(finish_kernel<T>, grid, 256, 0, st, 1, jobs.q[0], d[0]);
}
// Tensor maps are made by the driver, which wants the device's context to be current: a thread that has made no call of the runtime's
// yet (autograd's, on the first backward of a process) has none until it says which device it is on.
inline int make_context_current() {
  int dev = 0;
  LIK_CUDA_OK(cudaGetDevice(&dev));
  LIK_CUDA_OK(cudaSetDevice(dev));
  return LIK_OK;
}

}  // namespace
}  // namespace lik
