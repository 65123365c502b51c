// What the linear-layer operators share: element types, activations and their slopes, and the state an epilogue carries.
//
//   forward    D = act(z) + beta * C,             z = alpha * op(A) * op(B) + bias
//   gradient   D = (alpha * op(A) * op(B) + beta * C) * act'(Z),   dbias(m) = sum over n of D(m, n)
//
// Everything between the matrix product and the store is computed in 32 bits (in 64 for fp64 matrices) from the unrounded
// accumulator and rounded to the output type once; dbias sums the unrounded values.
#ifndef PLK_EPILOGUE_H
#define PLK_EPILOGUE_H
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paralia_hip.h"

namespace plk {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// The type sums and activations are computed in.
template <typename T> struct Wide { using type = float; };
template <> struct Wide<double> { using type = double; };
template <typename T> using wide_t = typename Wide<T>::type;

// 16 bytes at any multiple of the element size: one vector access, whose alignment the hardware does not ask for.
template <typename T> struct Loose {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec type __attribute__((aligned(sizeof(T))));
};

// (What is read or written once goes past the caches, non-temporal: 16384 x 8192 x 4096 with the gradient 1017 -> 967 us, the
// panels of the product keep the L2 to themselves.)
// N consecutive elements, `valid` of which are inside the matrix (the others read as zero and are not written).
template <typename T, int N, typename W, bool ONCE = false>
__device__ __forceinline__ void load_row(const T* p, W (&v)[N], int valid) {
  constexpr int V = Loose<T>::N;
  static_assert(N % V == 0, "whole vectors");
  if (valid >= N) {
#pragma unroll
    for (int q = 0; q < N / V; ++q) {
      typename Loose<T>::vec x;
      if constexpr (ONCE) x = __builtin_nontemporal_load(reinterpret_cast<const typename Loose<T>::type*>(p + q * V));
      else x = *reinterpret_cast<const typename Loose<T>::type*>(p + q * V);
#pragma unroll
      for (int e = 0; e < V; ++e) v[q * V + e] = (W)x[e];
    }
  } else if (valid > 0) {   // (all loads at once: a branch each would wait for each)
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (W)p[e < valid ? e : valid - 1];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < valid ? v[e] : W(0);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = W(0);
  }
}
template <typename T, int N, typename W>
__device__ __forceinline__ void store_row(T* p, const W (&v)[N], int valid) {
  constexpr int V = Loose<T>::N;
  static_assert(N % V == 0, "whole vectors");
  if (valid >= N) {
#pragma unroll
    for (int q = 0; q < N / V; ++q) {
      typename Loose<T>::vec x;
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = (T)v[q * V + e];
      __builtin_nontemporal_store(x, reinterpret_cast<typename Loose<T>::type*>(p + q * V));
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < valid) p[e] = (T)v[e];
  }
}

// ---- activations ----
// Accuracy classes: FAST for results rounded to 16 bits (relative error below 1e-5, which a rounding to 2^-11 or 2^-8 hides),
// and the full precision of W for results in 32 and 64 bits, those of 16-bit operands among them.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// 1 / (1 + e^-x).  FAST takes x times log2 e, which its callers fold into their constants.
template <typename W, bool FAST> constexpr W IN_EXPONENT = FAST ? W(1.44269504088896341) : W(1);
template <bool FAST> __device__ __forceinline__ float sigmoid(float x) {
  if constexpr (FAST) return fast_rcp(1.0f + __builtin_amdgcn_exp2f(-x));
  return 1.0f / (1.0f + expf(-x));
}
template <bool FAST> __device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

// The normal distribution function, accurate in the lower tail too: Phi(z) = erfc(-z / sqrt 2) / 2.  FAST: for z < 0
// erfcx(|z| / sqrt 2) / 2 as a polynomial of degree 7 in t = 1 / (1 + c |z|) without its constant term, fitted here by
// iteratively reweighted least squares for relative error on [0, 12] (1.2e-6; 4.2e-6 with the single-precision
// evaluation and the exponential), and exp(-z^2 / 2), which the slope needs too.  It takes 14 instructions where erfcf
// takes about 60.
template <bool FAST> __device__ __forceinline__ float normal_cdf(float z, float& gauss) {
  if constexpr (FAST) {
    gauss = fast_exp(-0.5f * z * z);
    const float t = fast_rcp(fmaf(0.3676955262f, fabsf(z), 1.0f));
    float q = 0.0483170813f;
    q = fmaf(q, t, -0.1735949573f);
    q = fmaf(q, t, 0.1554887252f);
    q = fmaf(q, t, 0.0406580207f);
    q = fmaf(q, t, 0.1367959960f);
    q = fmaf(q, t, 0.1455989241f);
    q = fmaf(q, t, 0.1467367770f);
    q = q * t * gauss;
    return z < 0.0f ? q : 1.0f - q;
  }
  gauss = expf(-0.5f * z * z);
  return 0.5f * erfcf(z * -0.707106781186547524f);
}
// 64 bits: erfcx(|z| / sqrt 2) / 2 = t * (Chebyshev series in 2 t - 1), t = 1 / (1 + c |z|), coefficients computed here from
// erfcx at 80 nodes in 40 digits; 3e-15 relative on [0, 37].  A rolled loop over constant memory: the library's erfc holds
// so many constants that, hoisted out of the column loop, they spill the scalar registers.
__device__ __constant__ const double NORMAL_CDF_SERIES[22] = {
    2.41390531530956159e-01, 1.88058934450544474e-01, 5.61536590038537106e-02, 1.24768816180276972e-02,
    1.84580253318977067e-03, 1.02578268994159540e-04, -2.35562952824470120e-05, -5.13536623286454059e-06,
    1.48761246171966915e-07, 1.57395904949404302e-07, 3.21133969801588664e-09, -5.10988785511638481e-09,
    -1.89570343315031835e-10, 1.89760393311438657e-10, 4.59570869378926954e-12, -7.86666431782942532e-12,
    1.25372910163215996e-13, 3.40611099452866603e-13, -2.74990967790584548e-14, -1.40465299025601052e-14,
    2.53067309065790210e-15, 4.65919086594141706e-16};
template <bool FAST> __device__ __forceinline__ double normal_cdf(double z, double& gauss) {
  gauss = exp(-0.5 * z * z);
  const double t = 1.0 / fma(0.24748737341529163, fabs(z), 1.0), s = 2.0 * t - 1.0;
  double b1 = 0.0, b2 = 0.0;
#pragma unroll 1
  for (int i = 21; i > 0; --i) {
    const double b = fma(2.0 * s, b1, NORMAL_CDF_SERIES[i] - b2);
    b2 = b1;
    b1 = b;
  }
  const double q = t * fma(s, b1, NORMAL_CDF_SERIES[0] - b2) * gauss;
  return z < 0.0 ? q : 1.0 - q;
}

template <typename W> constexpr W GELU_U1 = W(1.5957691216057307117);    // 2 sqrt(2 / pi)
template <typename W> constexpr W GELU_U3 = W(0.071354816272600248);     // ... times 0.044715
template <typename W> constexpr W GELU_D3 = W(0.21406444881780074);      // ... times 3 * 0.044715
template <typename W> constexpr W INV_SQRT_2PI = W(0.39894228040143267794);

// v <- act(v).  z * s(2u) with u = sqrt(2 / pi) (z + 0.044715 z^3) is the tanh form of gelu: (1 + tanh u) / 2 = s(2u).
template <typename W, bool FAST, int VEC> __device__ __forceinline__ void activate(W (&v)[VEC], int act) {
  if (act == PL_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = v[e] < W(0) ? W(0) : v[e];   // (NaN stays NaN)
  } else if (act == PL_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) { W g; v[e] *= normal_cdf<FAST>(v[e], g); }
  } else if (act == PL_ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] *= sigmoid<FAST>(v[e] * (GELU_U1<W> * IN_EXPONENT<W, FAST> + GELU_U3<W> * IN_EXPONENT<W, FAST> * (v[e] * v[e])));
  } else if (act == PL_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] *= sigmoid<FAST>(v[e] * IN_EXPONENT<W, FAST>);
  }
}
// v <- v * act'(z).  Where z is so large that z^2 would overflow, the tanh form's s (1 - s) is 0 and would meet an infinity:
// its z^2 stops at 40^2, beyond which the slope is 0 or 1 to the last bit.  (The minimum drops a NaN, the other factors keep it.)
template <typename W, bool FAST, int VEC> __device__ __forceinline__ void times_slope(W (&v)[VEC], const W (&zs)[VEC], int act) {
  if (act == PL_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = zs[e] > W(0) ? v[e] : W(0);   // (not times 0: infinities and NaN stay out too)
  } else if (act == PL_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      W g;
      const W p = normal_cdf<FAST>(zs[e], g);
      v[e] *= fma(zs[e] * g, INV_SQRT_2PI<W>, p);
    }
  } else if (act == PL_ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const W z = zs[e], zz = fmin(z * z, W(1600));
      const W s = sigmoid<FAST>(z * (GELU_U1<W> * IN_EXPONENT<W, FAST> + GELU_U3<W> * IN_EXPONENT<W, FAST> * zz));
      v[e] *= fma(z * s * (W(1) - s), GELU_U1<W> + GELU_D3<W> * zz, s);
    }
  } else if (act == PL_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const W z = zs[e], s = sigmoid<FAST>(z * IN_EXPONENT<W, FAST>);
      v[e] *= fma(z * s, W(1) - s, s);
    }
  }
}

// One epilogue, by value in the kernels' arguments.  Typed pointers are cast where the kernel's types are known.
struct Epilogue {
  double alpha, beta;
  const void* bias;        // forward: M elements or null
  const void* C; long ldc; // read only when beta != 0
  void* D; long ldd;
  void* preact; long ldp;  // forward: where z goes, or null
  const void* Z; long ldz; // gradient: z of the forward pass (not read when act is PL_ACT_NONE)
  void* partial;           // gradient: rows of M partial sums of dbias in the wide type, or null
  int act;
};

// What an epilogue reads for VEC elements of a column: C, and Z of the gradient.  Loaded in one step and used in another, so
// that loads can be ahead of their use; the elements beyond `valid` are zero.
template <typename T, typename TD, bool GRAD, int VEC> struct EpilogueInputs {
  typedef T zvec __attribute__((ext_vector_type(VEC)));
  typedef TD cvec __attribute__((ext_vector_type(VEC)));
  typedef zvec zload __attribute__((aligned(sizeof(T))));
  typedef cvec cload __attribute__((aligned(sizeof(TD))));
  cvec c;
  zvec z;
  template <typename V, typename L, typename E> static __device__ __forceinline__ V get(const E* p, int valid) {
    if (valid >= VEC) return __builtin_nontemporal_load(reinterpret_cast<const L*>(p));
    V v;   // (all loads at once: a branch each would wait for each, 11 us of a tile with a ragged edge)
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = p[e < valid ? e : valid - 1];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = e < valid ? v[e] : E(0);
    return v;
  }
  __device__ __forceinline__ void load(const Epilogue& ep, const TD* pc, const T* pz, int valid) {
    if (valid <= 0) return;
    if (ep.beta != 0.0) c = get<cvec, cload>(pc, valid);
    if (GRAD && ep.act != PL_ACT_NONE) z = get<zvec, zload>(pz, valid);
  }
};

// VEC elements of one column of the product, `valid` of them inside the matrix, through the epilogue and to D and z at pd
// and pp.  sums collects the gradient's column values.
template <typename T, typename TD, bool GRAD, int VEC>
__device__ __forceinline__ void apply_epilogue(const Epilogue& ep, const EpilogueInputs<T, TD, GRAD, VEC>& in, wide_t<T> (&v)[VEC], const wide_t<T> (&bias)[VEC], TD* pd,
                                               T* pp, int valid, wide_t<T> (&sums)[VEC]) {
  using W = wide_t<T>;
  constexpr bool FAST = sizeof(T) == 2 && sizeof(TD) == 2;   // (an fp32 D shows the short forms: gelu near 0 24 against 3 units of 2^-24)
  const W alpha = (W)ep.alpha, beta = (W)ep.beta;
  int act = ep.act;
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+s"(act));   // compared anew each time: the outcomes, kept over a loop, would not fit the scalar registers
#endif
  if constexpr (GRAD) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = alpha * v[e];
    if (beta != W(0)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fma(beta, (W)in.c[e], v[e]);
    }
    if (act != PL_ACT_NONE) {
      W z[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) z[e] = (W)in.z[e];
      times_slope<W, FAST, VEC>(v, z, act);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e < valid) sums[e] += v[e];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = fma(alpha, v[e], bias[e]);
    if (ep.preact) store_row<T, VEC, W>(pp, v, valid);
    activate<W, FAST, VEC>(v, act);
    if (beta != W(0)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fma(beta, (W)in.c[e], v[e]);
    }
  }
  if (ep.D) store_row<TD, VEC, W>(pd, v, valid);
}

}  // namespace plk
#endif
