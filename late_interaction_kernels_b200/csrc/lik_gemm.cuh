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
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 u = *reinterpret_cast<const float4*>(s + slot_offset<128>(lane, h * 4 + c));
      f[4 * c] = u.x, f[4 * c + 1] = u.y, f[4 * c + 2] = u.z, f[4 * c + 3] = u.w;
    }
  } else {
    Raw16<T> r;
#pragma unroll
    for (int c = 0; c < 2; ++c) r.u[c] = *reinterpret_cast<const uint4*>(s + slot_offset<64>(lane, h * 2 + c));
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
    for (int r = 0; r < rows && r < 32; ++r) p[r * stride + lane] = *reinterpret_cast<const O*>(s + slot_offset<ROW>(r, lane / PER) + (lane % PER) * sizeof(O));
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
    for (int r = 0; r < rows && r < 32; ++r) *reinterpret_cast<T*>(s + slot_offset<ROW>(r, lane / PER) + (lane % PER) * sizeof(T)) = p[r * stride + lane];
  }
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

// an operand as it lies in memory
struct Stored {
  const void* p;
  long long rows, cols, stride;
  bool mn;  // rows are k
  const void* parts = nullptr;
  // as TMA wants 16-bit rows
  bool aligned() const { return ((uintptr_t)p & 15) == 0 && (rows == 1 || stride % 8 == 0); }
  long long padded() const { return (cols + 7) / 8 * 8; }
};
Stored stored(const GemmOperand& o, long long rows, long long k) {
  if (o.k == 1) return {o.p, rows, k, o.row, false, o.parts};
  return {o.p, k, rows, o.k, true, o.parts};
}
bool rows_of_pieces(const void* p, long long stride, int dtype) { return ((uintptr_t)p & 15) == 0 && stride * (long long)dtype_size(dtype) % 16 == 0; }

int launch_sum_splits(const float* partial, int splits, const GemmDesc& d, int stride, cudaStream_t st) {
  const long long blocks = ceil_div(d.m * ((d.n + 3) / 4), 256), most = 16ll * sm_count();
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  if (d.out_dtype == LIK_F32) sum_splits_kernel<float><<<grid, 256, 0, st>>>(partial, splits, d.m, d.n, stride, (float*)d.out[0], d.out_stride), count_launch();
  else if (d.out_dtype == LIK_F16) sum_splits_kernel<__half><<<grid, 256, 0, st>>>(partial, splits, d.m, d.n, stride, (__half*)d.out[0], d.out_stride), count_launch();
  else sum_splits_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(partial, splits, d.m, d.n, stride, (__nv_bfloat16*)d.out[0], d.out_stride), count_launch();
  LIK_CUDA_OK(cudaGetLastError());
  return LIK_OK;
}
// Tensor maps are made by the driver, which wants the device's context to be current: a thread that has made no call of the runtime's
// yet (autograd's, on the first backward of a process) has none until it says which device it is on.
int make_context_current() {
  int dev = 0;
  LIK_CUDA_OK(cudaGetDevice(&dev));
  LIK_CUDA_OK(cudaSetDevice(dev));
  return LIK_OK;
}

}  // namespace
}  // namespace lik
