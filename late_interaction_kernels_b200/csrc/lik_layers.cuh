// What the kernels of the layers between an encoder and the document head share: activations with their slopes, the
// description of a matrix product with what is done to its elements, vector loads and stores.
#pragma once

#include "lik_common.cuh"

namespace lik {

// ---------------------------------------------------------------------------------------------
// Activations.  PRECISE (fp32 operands): CUDA's own functions.  Otherwise what is stored has 11 or 8 bits, and the two
// hardware approximations (2^x and the reciprocal, each good to 2^-22) are enough.
// ---------------------------------------------------------------------------------------------
// (the two instructions themselves, without the rescaling that keeps results below 2^-126)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool PRECISE>
__device__ __forceinline__ float sigmoid_f(float z) {
  return PRECISE ? 1.0f / (1.0f + expf(-z)) : fast_rcp(1.0f + fast_exp2(-1.4426950408889634f * z));
}
template <bool PRECISE>
__device__ __forceinline__ float tanh_f(float z) {
  if (PRECISE) return tanhf(z);
  // below 1/8 the difference would cancel: three terms of the series, the first one left out is 17/315 z^7
  const float q = z * z;
  return fabsf(z) < 0.125f ? z * fmaf(q, fmaf(q, 2.0f / 15.0f, -1.0f / 3.0f), 1.0f) : fmaf(2.0f, sigmoid_f<false>(2.0f * z), -1.0f);
}
// Phi(-|z|), the lower tail of the normal distribution, and exp(-z^2 / 2).  With t = 1 / (1 + 0.3 |z|) the ratio
// exp(z^2 / 2) Phi(-|z|) is a smooth function on (0, 1]; six coefficients (least squares, reweighted towards the largest relative
// error; our own fit) give it to 8.5e-6 relative for all |z| <= 14, a fiftieth of half a step of fp16.
__device__ __forceinline__ float normal_tail(float z, float& e) {
  const float a = fabsf(z), t = fast_rcp(fmaf(0.3f, a, 1.0f));
  e = fast_exp2(-0.72134752f * z * z);
  float r = fmaf(-0.0770966218f, t, 0.216034401f);
  r = fmaf(r, t, -0.0169447843f);
  r = fmaf(r, t, 0.144194491f);
  r = fmaf(r, t, 0.113742429f);
  r = fmaf(r, t, 0.120074183f);
  return r * t * e;
}
// gelu from the tail: z - z tail above 0, z tail below.  As a product with 0 or 1 the first term is infinite for z = inf and NaN for z = -inf, as z Phi(z)
// is; the second one's factor stays finite, since a tail of 0 has to make it 0.
__device__ __forceinline__ float above0(float z) {
  float r;
  asm("set.gt.f32.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}
__device__ __forceinline__ float minus_abs(float z) { return fmaxf(-fabsf(z), -1e30f); }
__device__ __forceinline__ float gelu_from(float z, float tail) { return fmaf(minus_abs(z), tail, z * above0(z)); }
// A factor beside one that is exactly 0 once z is far from zero: z itself, which a linear layer keeps in its type (infinite beyond fp16's 65504 although
// the sum was finite), and the polynomial in gelu_tanh's slope, infinite from |z| of 1e13 on.  (The factor that may be 0 keeps a NaN.)
__device__ __forceinline__ float bounded(float w) { return fminf(fmaxf(w, -1e30f), 1e30f); }
constexpr float GELU_C = 1.5957691216057308f;  // 2 sqrt(2 / pi): (1 + tanh(y)) / 2 = sigmoid(2 y)

template <int ACT, bool PRECISE>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == LIK_ACT_RELU) return z < 0.0f ? 0.0f : z;  // (a NaN stays one)
  if constexpr (ACT == LIK_ACT_SILU) return z * sigmoid_f<PRECISE>(z);
  if constexpr (ACT == LIK_ACT_GELU) {
    if constexpr (PRECISE) return 0.5f * z * erfcf(-0.70710678118654752f * z);
    float e;
    const float tail = normal_tail(z, e);
    return gelu_from(z, tail);
  }
  if constexpr (ACT == LIK_ACT_GELU_TANH) return z * sigmoid_f<PRECISE>(GELU_C * fmaf(0.044715f * z * z, z, z));
  if constexpr (ACT == LIK_ACT_TANH) return tanh_f<PRECISE>(z);
  if constexpr (ACT == LIK_ACT_SIGMOID) return sigmoid_f<PRECISE>(z);
  return z;
}
// the value and the derivative
template <int ACT, bool PRECISE>
__device__ __forceinline__ float act_slope(float z, float& value) {
  if constexpr (ACT == LIK_ACT_RELU) {
    value = z < 0.0f ? 0.0f : z;
    return z > 0.0f ? 1.0f : 0.0f;
  }
  if constexpr (ACT == LIK_ACT_SILU) {
    const float s = sigmoid_f<PRECISE>(z);
    value = z * s;
    return s * fmaf(bounded(z), 1.0f - s, 1.0f);
  }
  if constexpr (ACT == LIK_ACT_GELU) {
    float cdf, e;
    if constexpr (PRECISE) {
      cdf = 0.5f * erfcf(-0.70710678118654752f * z);
      e = expf(-0.5f * z * z);
      value = z * cdf;
    } else {
      const float tail = normal_tail(z, e);
      cdf = z < 0.0f ? tail : 1.0f - tail;
      value = gelu_from(z, tail);
    }
    return fmaf(0.3989422804014327f * bounded(z), e, cdf);
  }
  if constexpr (ACT == LIK_ACT_GELU_TANH) {
    const float q = 0.044715f * z * z, s = sigmoid_f<PRECISE>(GELU_C * fmaf(q, z, z));
    value = z * s;
    return s * fmaf(bounded(GELU_C * z * fmaf(3.0f, q, 1.0f)), 1.0f - s, 1.0f);
  }
  if constexpr (ACT == LIK_ACT_TANH) {
    value = tanh_f<PRECISE>(z);
    return fmaf(-value, value, 1.0f);
  }
  if constexpr (ACT == LIK_ACT_SIGMOID) {
    value = sigmoid_f<PRECISE>(z);
    return value * (1.0f - value);
  }
  value = z;
  return 1.0f;
}

// Two values at a time, for epilogues that are bound by the instructions they issue: additions, products and multiply-adds take one for both, with
// the bits of the single ones.
struct Pair {
  unsigned long long u;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(u)); }
};
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.u) : "l"(a.u), "l"(b.u));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.u) : "l"(a.u), "l"(b.u));
  return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return d;
}
__device__ __forceinline__ Pair both(float x) { return Pair(x, x); }
__device__ __forceinline__ Pair exp2_2(Pair p) {
  float a, b;
  p.get(a, b);
  return Pair(fast_exp2(a), fast_exp2(b));
}
__device__ __forceinline__ Pair rcp_2(Pair p) {
  float a, b;
  p.get(a, b);
  return Pair(fast_rcp(a), fast_rcp(b));
}
__device__ __forceinline__ Pair bounded_2(Pair p) {
  float a, b;
  p.get(a, b);
  return Pair(bounded(a), bounded(b));
}
__device__ __forceinline__ Pair sigmoid_2(Pair z) { return rcp_2(add2(exp2_2(mul2(z, both(-1.4426950408889634f))), both(1.0f))); }
// the same on vectors of V elements (one by one where V is 1): v = v * a + b, v = v * a, v = v + a, s += v, s += v * a
template <int V>
__device__ __forceinline__ void vec_fma(float (&v)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) v[0] = fmaf(v[0], a[0], b[0]);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) fma2(Pair(v[i], v[i + 1]), Pair(a[i], a[i + 1]), Pair(b[i], b[i + 1])).get(v[i], v[i + 1]);
}
template <int V>
__device__ __forceinline__ void vec_fma(float (&v)[V], float a, float b) {
  if constexpr (V == 1) v[0] = fmaf(v[0], a, b);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) fma2(Pair(v[i], v[i + 1]), both(a), both(b)).get(v[i], v[i + 1]);
}
template <int V>
__device__ __forceinline__ void vec_mul(float (&v)[V], const float (&a)[V]) {
  if constexpr (V == 1) v[0] *= a[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) mul2(Pair(v[i], v[i + 1]), Pair(a[i], a[i + 1])).get(v[i], v[i + 1]);
}
template <int V>
__device__ __forceinline__ void vec_mul(float (&v)[V], float a) {
  if constexpr (V == 1) v[0] *= a;
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) mul2(Pair(v[i], v[i + 1]), both(a)).get(v[i], v[i + 1]);
}
template <int V>
__device__ __forceinline__ void vec_add(float (&v)[V], const float (&a)[V]) {
  if constexpr (V == 1) v[0] += a[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) add2(Pair(v[i], v[i + 1]), Pair(a[i], a[i + 1])).get(v[i], v[i + 1]);
}
template <int V>
__device__ __forceinline__ void vec_add(float (&v)[V], float a) {
  if constexpr (V == 1) v[0] += a;
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) add2(Pair(v[i], v[i + 1]), both(a)).get(v[i], v[i + 1]);
}
struct PairSum {  // sums of the even and of the odd elements
  float a = 0.0f, b = 0.0f;
  template <int V>
  __device__ __forceinline__ void add(const float (&v)[V]) {
    if constexpr (V == 1) a += v[0];
    else
#pragma unroll
      for (int i = 0; i < V; i += 2) add2(Pair(a, b), Pair(v[i], v[i + 1])).get(a, b);
  }
  template <int V>
  __device__ __forceinline__ void dot(const float (&v)[V], const float (&w)[V]) {
    if constexpr (V == 1) a = fmaf(v[0], w[0], a);
    else
#pragma unroll
      for (int i = 0; i < V; i += 2) fma2(Pair(v[i], v[i + 1]), Pair(w[i], w[i + 1]), Pair(a, b)).get(a, b);
  }
  __device__ __forceinline__ float sum() const { return a + b; }
};
// the activation's value of both and, where SLOPE, its derivative (fast functions; see act_value and act_slope)
template <int ACT, bool SLOPE>
__device__ __forceinline__ void act_pair(float& x, float& y, float& sx, float& sy) {
  const Pair z(x, y);
  if constexpr (ACT == LIK_ACT_SILU || ACT == LIK_ACT_GELU_TANH) {
    Pair s, q;
    if constexpr (ACT == LIK_ACT_SILU) {
      s = sigmoid_2(z);
    } else {
      q = mul2(mul2(z, z), both(0.044715f));
      s = sigmoid_2(mul2(fma2(q, z, z), both(GELU_C)));
    }
    mul2(z, s).get(x, y);
    if constexpr (SLOPE) {
      const Pair w = bounded_2(ACT == LIK_ACT_SILU ? z : mul2(mul2(z, both(GELU_C)), fma2(q, both(3.0f), both(1.0f))));
      mul2(s, fma2(w, fma2(s, both(-1.0f), both(1.0f)), both(1.0f))).get(sx, sy);
    }
  } else if constexpr (ACT == LIK_ACT_GELU) {
    const Pair na(minus_abs(x), minus_abs(y)), t = rcp_2(fma2(na, both(-0.3f), both(1.0f))), e = exp2_2(mul2(mul2(z, z), both(-0.72134752f)));
    Pair r = fma2(t, both(-0.0770966218f), both(0.216034401f));
    r = fma2(r, t, both(-0.0169447843f));
    r = fma2(r, t, both(0.144194491f));
    r = fma2(r, t, both(0.113742429f));
    r = fma2(r, t, both(0.120074183f));
    const Pair tail = mul2(mul2(r, t), e);
    if constexpr (SLOPE) {
      float a, b, c, d;
      tail.get(a, b);
      fma2(tail, both(-1.0f), both(1.0f)).get(c, d);
      fma2(mul2(bounded_2(z), both(0.3989422804014327f)), e, Pair(x < 0.0f ? a : c, y < 0.0f ? b : d)).get(sx, sy);
    }
    fma2(na, tail, mul2(z, Pair(above0(x), above0(y)))).get(x, y);  // (gelu_from)
  } else if constexpr (SLOPE) {
    sx = act_slope<ACT, false>(x, x);
    sy = act_slope<ACT, false>(y, y);
  } else {
    x = act_value<ACT, false>(x);
    y = act_value<ACT, false>(y);
  }
}

// f(ActConst<activation>): the activation as a compile-time constant, on the host (which kernel) and on the device (which epilogue)
template <int V>
struct ActConst {
  static constexpr int value = V;
};
#define LIK_WITH_ACTIVATION(NAME, SPACE)                                             \
  template <typename F>                                                              \
  SPACE inline void NAME(int act, F&& f) {                                           \
    switch (act) {                                                                   \
      case LIK_ACT_RELU: f(ActConst<LIK_ACT_RELU>{}); break;                         \
      case LIK_ACT_SILU: f(ActConst<LIK_ACT_SILU>{}); break;                         \
      case LIK_ACT_GELU: f(ActConst<LIK_ACT_GELU>{}); break;                         \
      case LIK_ACT_GELU_TANH: f(ActConst<LIK_ACT_GELU_TANH>{}); break;               \
      case LIK_ACT_TANH: f(ActConst<LIK_ACT_TANH>{}); break;                         \
      case LIK_ACT_SIGMOID: f(ActConst<LIK_ACT_SIGMOID>{}); break;                   \
      default: f(ActConst<LIK_ACT_NONE>{}); break;                                   \
    }                                                                                \
  }
LIK_WITH_ACTIVATION(with_activation, __host__)
LIK_WITH_ACTIVATION(with_activation_dev, __device__)
#undef LIK_WITH_ACTIVATION

// ---------------------------------------------------------------------------------------------
// Launches.  A pass is a chain of short kernels, so each is launched with programmatic stream serialisation: its blocks come to the SMs as those of
// the kernel in front leave, set themselves up and wait for that kernel's end.  Every kernel here begins with after_the_kernel_in_front(),
// before which it touches no device memory (a step of 1000 x 768 x 768 in a graph: 26.6 us without this, 23.0 with it).
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void after_the_kernel_in_front() {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
}
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, int cluster, const A&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  LIK_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
  count_launch();
  return LIK_OK;
}

// ---------------------------------------------------------------------------------------------
// Vectors of V elements, V * sizeof(T) = 16 bytes or one element, as fp32
// ---------------------------------------------------------------------------------------------
template <typename T>
constexpr int vec_elems() {
  return 16 / (int)sizeof(T);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi, __nv_bfloat16) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 4) {
    static_assert(V % 4 == 0, "whole 16-byte vectors");
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
  } else {
    static_assert(V % 8 == 0, "whole 16-byte vectors");
#pragma unroll
    for (int i = 0; i < V; i += 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + i);
      unpack2(u.x, v[i + 0], v[i + 1], T());
      unpack2(u.y, v[i + 2], v[i + 3], T());
      unpack2(u.z, v[i + 4], v[i + 5], T());
      unpack2(u.w, v[i + 6], v[i + 7], T());
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 8)
      *reinterpret_cast<uint4*>(p + i) = make_uint4(pack2(v[i], v[i + 1], T()), pack2(v[i + 2], v[i + 3], T()), pack2(v[i + 4], v[i + 5], T()),
                                                    pack2(v[i + 6], v[i + 7], T()));
  }
}
inline bool vec_ok(const void* p, long long stride, int width, int item) {
  return ((uintptr_t)p & 15) == 0 && stride * item % 16 == 0 && (long long)width * item % 16 == 0;
}

// ---------------------------------------------------------------------------------------------
// A matrix product and what is done to its elements: c[m, n] = sum over segments and k of a(m, k) b(n, k)
// ---------------------------------------------------------------------------------------------
enum GemmKind {
  GEMM_LINEAR = 0,     // z = c + bias, out = act(z) + residual; kept[0] = z where it is asked for
  GEMM_GATED = 1,      // two products of the same a: g = c0 + bias0, u = c1 + bias1, out = act(g) u; kept = u act'(g), act(g)
  GEMM_GATED_BWD = 2,  // c = gradient of act(g) u: out[i] = c kept[i], the gradients of g and u
};
struct GemmOperand {
  const void* p = nullptr;
  long long row = 0, k = 0;  // elements from one row (m or n) to the next, and from one k to the next; one of the two is 1
};
struct GemmDesc {
  int kind = GEMM_LINEAR, act = LIK_ACT_NONE, dtype = 0;
  bool several = false;       // one of up to four products that may share a launch
  long long m = 0;
  int n = 0;
  int n_seg = 1;              // segments of the sum (GEMM_LINEAR) ...
  long long k[2] = {0, 0};
  GemmOperand a[2], b[2];     // ... GEMM_GATED: a[0] with b[0] and b[1], k[0]
  const void* bias[2] = {nullptr, nullptr};
  const void* residual = nullptr;
  long long residual_stride = 0;
  void* out[2] = {nullptr, nullptr};
  long long out_stride = 0;
  int out_dtype = 0;                   // dtype, or LIK_F32 for products without anything else to them
  void* kept[2] = {nullptr, nullptr};  // the factors of the backward: written, or read by GEMM_GATED_BWD; rows of 16 bytes
  long long kept_stride = 0;
  const float *norm_a = nullptr, *norm_b = nullptr;  // of a's rows and of (the gate's) b's, where relu's side is kept from 16-bit operands
};
// The kink of relu.  Its slope goes by the sign of z, and the tensor core's sums, which cut off what they shift out at every 16 products, have a wrong
// sign for a z that is next to nothing beside what it is a sum of: a few in a million, each a whole gradient off.  An addition of 16 products loses
// up to four steps (2^-23; 1.6 on average) of the largest number in it.  Partial sums of a z near 0 are at most half of |a| |b|, the product of
// the rows' lengths: what comes first is bounded by the lengths of its parts, and so is what comes after and cancels it.  So where z is within
// kink_bound and a backward pass will look at its sign, it is taken again from the operands, in 64 bits, by a warp.  The lengths come from a
// pass over the operands (kink_norms): nothing at hand says as much about a sum that came out small.  (The largest of z's neighbours, asked before, is
// small too where a whole row cancels, and beside a feature that is switched off or dead it made every z look small: 65536 x 768 x 768 went from 105
// us to 4 100 with one feature at -1e9 and to 5 400 with a tenth of the features dead; a zero row has length 0 and z of it is sure.)
// What remains is data whose sums are 0 for their own sake, which are taken again like any other: half of x 0 costs nothing, but where a twentieth of x and a
// tenth of the weights are not 0 (2 % of z are 0) that forward takes 690 us, and 9.9 ms with a hundredth of x (46 %).
__device__ __forceinline__ float kink_bound(float norm_a, float norm_b, long long k) { return norm_a * (2.384185791015625e-7f * (float)(k / 16 + 2)) * norm_b; }
// sum over k of a b by a warp, in all lanes; products of 16-bit values are exact in fp32.  (Not inline: it is rarely called, and its loads, all
// of 1024 k at once, would take the registers of the epilogue around it.)
template <typename T>
__device__ __noinline__ double exact_sum(const T* a, const T* b, long long k, int lane) {
  double s[2] = {0.0, 0.0};
  long long done = 0;
  if ((((uintptr_t)a | (uintptr_t)b) & 15) == 0) {
    done = k & ~7ll;
#pragma unroll 1
    for (long long first = 0; first < done; first += 1024) {
      uint4 u[4], w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long i = first + j * 256 + lane * 8;
        const bool there = i < done;
        u[j] = there ? *reinterpret_cast<const uint4*>(a + i) : make_uint4(0u, 0u, 0u, 0u);
        w[j] = there ? *reinterpret_cast<const uint4*>(b + i) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x[4] = {u[j].x, u[j].y, u[j].z, u[j].w}, y[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float xl, xh, yl, yh;
          unpack2(x[e], xl, xh, T());
          unpack2(y[e], yl, yh, T());
          s[0] += (double)(xl * yl);
          s[1] += (double)(xh * yh);
        }
      }
    }
  }
#pragma unroll 1
  for (long long first = done; first < k; first += 512) {
    T x[16], y[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const long long i = first + j * 32 + lane;
      const bool there = i < k;
      x[j] = there ? a[i] : from_f32<T>(0.0f);
      y[j] = there ? b[i] : from_f32<T>(0.0f);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j & 1] += (double)(to_f32(x[j]) * to_f32(y[j]));
  }
  double sum = s[0] + s[1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// Whether z of element (m, n), a lane's own, is above 0; whole warps come here.
template <typename T>
__device__ __forceinline__ bool above_zero(const GemmDesc& d, long long m, int n, float z, bool there, int lane) {
  bool above = z > 0.0f;
  const bool unsure = there && fabsf(z) < kink_bound(d.norm_a[m], d.norm_b[n], d.k[0]);
  for (uint32_t lanes = __ballot_sync(0xffffffffu, unsure); lanes; lanes &= lanes - 1) {
    const int l = __ffs(lanes) - 1;
    const long long lm = __shfl_sync(0xffffffffu, m, l);
    const int ln = __shfl_sync(0xffffffffu, n, l);
    double e = exact_sum((const T*)d.a[0].p + lm * d.a[0].row, (const T*)d.b[0].p + ln * d.b[0].row, d.k[0], lane);
    if (d.bias[0]) e += (double)to_f32(((const T*)d.bias[0])[ln]);
    if (lane == l) above = e > 0.0;
  }
  return above;
}
// z as it is kept for relu's backward pass, which looks at its sign: above 0 also in its type where it is, and not where it is not
template <typename T>
__device__ __forceinline__ float keep_side(float z, bool above) {
  const float least = std::is_same<T, __half>::value ? 5.9604644775390625e-8f : 1.1754943508222875e-38f;
  return above ? fmaxf(z, least) : (z > 0.0f ? 0.0f : z);
}

// one element of the result, from the sums c0 and (GEMM_GATED) c1; above: whether relu's argument is above 0, as far as it is kept
template <typename T, typename O, int KIND, int ACT>
__device__ __forceinline__ void gemm_element(const GemmDesc& d, long long m, int n, float c0, float c1, bool above) {
  constexpr bool PRECISE = sizeof(T) == 4;
  const long long ki = m * d.kept_stride + n, oi = m * d.out_stride + n;
  if (d.bias[0]) c0 += to_f32(((const T*)d.bias[0])[n]);
  float v;
  if constexpr (KIND == GEMM_GATED) {
    float slope = act_slope<ACT, PRECISE>(c0, v);
    if constexpr (ACT == LIK_ACT_RELU) slope = above ? 1.0f : 0.0f;
    if (d.bias[1]) c1 += to_f32(((const T*)d.bias[1])[n]);
    if (d.kept[0]) {
      ((T*)d.kept[0])[ki] = from_f32<T>(c1 * slope);
      ((T*)d.kept[1])[ki] = from_f32<T>(v);
    }
    v *= c1;
  } else {
    v = act_value<ACT, PRECISE>(c0);
    if (d.kept[0]) ((T*)d.kept[0])[ki] = from_f32<T>(ACT == LIK_ACT_RELU ? keep_side<T>(c0, above) : c0);
    if (d.residual) v += to_f32(((const T*)d.residual)[m * d.residual_stride + n]);
  }
  ((O*)d.out[0])[oi] = from_f32<O>(v);
}

// nothing but the product: its sum may be cut along k
inline bool gemm_plain(const GemmDesc& d) {
  return d.kind == GEMM_LINEAR && d.act == LIK_ACT_NONE && !d.bias[0] && !d.residual && !d.kept[0];
}
// few rows of a (lik_gemm_few.cu): any type, both operands with their k contiguous; whether it is the faster one
bool gemm_few_pays(const GemmDesc& d);
int launch_gemm_few(const GemmDesc& d, cudaStream_t st);
// Tensor cores: 16-bit operands (lik_gemm_tc.cu), and fp32 operands in three bf16 parts (lik_gemm_f32.cu).  One product, or up to four plain
// ones of one type in one launch.
size_t gemm_tc_workspace(const GemmDesc* d, int n);
int launch_gemm_tc(const GemmDesc* d, int n, void* ws, size_t ws_bytes, int* status, cudaStream_t st);
size_t gemm_f32_workspace(const GemmDesc* d, int n);
int launch_gemm_f32(const GemmDesc* d, int n, void* ws, size_t ws_bytes, int* status, cudaStream_t st);

// Vectors of sums: element i of all of them, one behind the other, belongs to the first vector whose end is above i.
constexpr int SUM_OUTS = 3;
struct SumOuts {
  void* out[SUM_OUTS];  // of the kernel's T, or fp32; NULL: not wanted
  long long end[SUM_OUTS];
  bool f32;
  template <typename T>
  __device__ __forceinline__ void put(long long i, float v) const {
    const int q = i < end[0] ? 0 : (i < end[1] ? 1 : 2);
    const long long at = i - (q ? end[q - 1] : 0);
    if (!out[q]) return;
    if (f32) ((float*)out[q])[at] = v;
    else ((T*)out[q])[at] = from_f32<T>(v);
  }
};
int launch_sum_parts(const float* partial, int parts, const SumOuts& outs, int dtype, cudaStream_t st);

}  // namespace lik
