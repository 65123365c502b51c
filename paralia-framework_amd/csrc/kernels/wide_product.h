// fp32 / fp64 product with its epilogue in one kernel, for gfx950 (MI355X): 64 x 64 tiles of four waves, 32 x 32 each in 16 x 16
// blocks of v_mfma_{f32,f64}_16x16x4, for products too small to fill the device with the tile GEMM's 128 x 128 tiles.
//
// A panel is 128 bytes of k (16 of fp64, 32 of fp32).  Its elements are loaded one by one, so that any alignment and any
// edge runs alike: along k for a K-major operand, along the rows for the other, whole cache lines per wave either way.  Two
// panels are in flight in registers, a third is in LDS being multiplied and a fourth being written.
//
// LDS holds a panel as [k][row], rows of 64 elements 80 apart: an operand's read takes 16 rows of 4 consecutive k (fp64: two
// passes of 2), 128 (64) bytes apart modulo the 256 of the banks.  Element (k, row) sits at row ^ turn(k): the writes of a
// K-major panel, which go along k, then meet every bank once too.
//
// A lone tile takes 0.85 us a panel (fp64; fp32 1.0) for 0.43 (0.43) of matrix instructions: the chain of a panel's store,
// barrier, reads and products; four workgroups on a unit overlap theirs: 54 (90) TFLOP/s over 2048^3,
// 69 % (57 %) of the peak.
#ifndef PLK_WIDE_PRODUCT_H
#define PLK_WIDE_PRODUCT_H
#include "kernels/epilogue.h"
#include "kernels/linear.h"

namespace plk {

template <typename T> struct WideTile {
  static constexpr int BK = 128 / (int)sizeof(T);      // panel depth
  static constexpr int LOADS = 64 * BK / 256;          // elements a thread loads of each operand's panel
  static constexpr int AHEAD = 2;                      // panels in flight (even: two buffers take turns; four are no faster)
  static constexpr int PITCH = 80;
  static constexpr int VEC = 16 / (int)sizeof(T);
  static constexpr int TILE_PITCH = sizeof(T) == 8 ? 80 : 68;   // the product on its way to the epilogue: 16 rows of 4 columns at once
  static constexpr int LDS = 4 * BK * PITCH;           // two panels of two operands, in elements
  static_assert(LDS >= 64 * TILE_PITCH, "the product lies where the panels were");
  static __device__ __forceinline__ int turn(int k) { return (sizeof(T) == 8 ? (k >> 1) & 7 : (k >> 2) & 7) * 2; }
};
typedef double wide_f64x4 __attribute__((ext_vector_type(4)));
typedef float wide_f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ wide_f64x4 wide_mfma(double a, double b, wide_f64x4 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
__device__ __forceinline__ wide_f32x4 wide_mfma(float a, float b, wide_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
template <typename T> struct WideAcc;
template <> struct WideAcc<double> { using type = wide_f64x4; static __device__ __forceinline__ int row(int r, int g) { return 4 * r + g; } };
template <> struct WideAcc<float> { using type = wide_f32x4; static __device__ __forceinline__ int row(int r, int g) { return 4 * g + r; } };

// One operand's share of a thread: where its elements lie in a panel, in memory and in LDS.
template <typename T, bool KMAJOR> struct WideOperand {
  using S = WideTile<T>;
  static constexpr int N = S::LOADS;
  const T* base;          // this thread's row, or its column of the panel's first element
  long ld;
  int k, row, last;       // k of element 0 in the panel; row; the operand's last row from this thread's first
  __device__ __forceinline__ WideOperand(const T* p, long ld_, int first, int extent, int tid) : ld(ld_) {
    k = KMAJOR ? tid % S::BK : tid / 64;
    row = KMAJOR ? tid / S::BK : tid % 64;
    // rows behind the last are read as the last: their products are not stored
    const int r = first + row < extent ? first + row : extent - 1;
    last = extent - 1 - r;
    base = KMAJOR ? p + (long)r * ld : p + r;
  }
  static __device__ __forceinline__ int k_of(int k, int i) { return KMAJOR ? k : k + 4 * i; }
  __device__ __forceinline__ void load(T (&v)[N], int k0, int k_last) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int kk = k0 + k_of(k, i);
      kk = kk < k_last ? kk : k_last;
      int down = i * (256 / S::BK);
      down = down < last ? down : last;
      v[i] = KMAJOR ? base[(long)down * ld + kk] : base[(long)kk * ld];
    }
  }
  // k behind the end counts as zero
  __device__ __forceinline__ void store(const T (&v)[N], T* lds, int k0, int k_last) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int kk = k_of(k, i), r = KMAJOR ? row + i * (256 / S::BK) : row;
      lds[kk * S::PITCH + (r ^ S::turn(kk))] = k0 + kk <= k_last ? v[i] : T(0);
    }
  }
};

// blockIdx.x: tile, blockIdx.y: slice of k.  With slices the epilogue is plain and slice y goes to D + y * M * N.
template <typename T, bool AK, bool BKM, bool GRAD>
__global__ __launch_bounds__(256, 3) void wide_tile_kernel(int M, int N, int K, const T* __restrict__ A, long lda, const T* __restrict__ B, long ldb, int gm, int kchunk,
                                                           Epilogue ep) {
  using S = WideTile<T>;
  using acc_t = typename WideAcc<T>::type;
  constexpr int BK = S::BK, VEC = S::VEC;
  __shared__ __attribute__((aligned(16))) T lds[S::LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bn = (int)(blockIdx.x / (unsigned)gm), bm = (int)(blockIdx.x - (unsigned)bn * (unsigned)gm);
  const int m0 = bm * 64, n0 = bn * 64;
  const int k_first = (int)blockIdx.y * kchunk, k_last = (k_first + kchunk < K ? k_first + kchunk : K) - 1;
  ep.D = (T*)ep.D + (long)blockIdx.y * M * N;
  acc_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
  const WideOperand<T, AK> a(A, lda, m0, M, tid);
  const WideOperand<T, BKM> b(B, ldb, n0, N, tid);
  T ra[S::AHEAD][S::LOADS], rb[S::AHEAD][S::LOADS];
  const int i16 = lane & 15, g = lane >> 4, wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  auto panel = [&](T (&pa)[S::LOADS], T (&pb)[S::LOADS], int k0, int half) {
    T* const la = lds + half * 2 * BK * S::PITCH;
    T* const lb = la + BK * S::PITCH;
    a.store(pa, la, k0, k_last);
    b.store(pb, lb, k0, k_last);
    // (the panel before last was multiplied before the barrier that its successor's writers passed: this half is free)
    __syncthreads();
    a.load(pa, k0 + S::AHEAD * BK, k_last);
    b.load(pb, k0 + S::AHEAD * BK, k_last);
#pragma unroll
    for (int s = 0; s < BK / 4; ++s) {
      const int k = 4 * s + g, at = k * S::PITCH + (i16 ^ S::turn(k));
      T va[2], vb[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) va[q] = la[at + wm + 16 * q], vb[q] = lb[at + wn + 16 * q];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = wide_mfma(vb[j], va[i], acc[i][j]);
    }
  };
  if (k_first <= k_last) {
#pragma unroll
    for (int q = 0; q < S::AHEAD; ++q) a.load(ra[q], k_first + q * BK, k_last), b.load(rb[q], k_first + q * BK, k_last);
    for (int k0 = k_first; k0 <= k_last; k0 += S::AHEAD * BK) {
#pragma unroll
      for (int q = 0; q < S::AHEAD; ++q) {
        if (q > 0 && k0 + q * BK > k_last) break;
        panel(ra[q], rb[q], k0 + q * BK, q & 1);
      }
    }
    __syncthreads();
  }
  // the product to LDS as [n][m], then 16 bytes of a column per lane through the epilogue
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) lds[(wn + 16 * j + WideAcc<T>::row(r, g)) * S::TILE_PITCH + wm + 16 * i + i16] = acc[i][j][r];
  __syncthreads();
  constexpr int LPC = 64 / VEC, CPS = 64 / LPC, STEPS = 16 / CPS;
  const int mv = (lane % LPC) * VEC, m = m0 + mv;
  const int valid = M - m < VEC ? (M - m < 0 ? 0 : M - m) : VEC;
  T bias[VEC], sums[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) bias[e] = sums[e] = T(0);
  if (!GRAD && ep.bias) load_row<T, VEC, T>((const T*)ep.bias + m, bias, valid);
  auto column = [&](int it) { return wave * 16 + it * CPS + lane / LPC; };
  auto product = [&](int n, T (&v)[VEC]) {
    typedef T vec __attribute__((ext_vector_type(VEC)));
    const vec x = *reinterpret_cast<const vec*>(lds + n * S::TILE_PITCH + mv);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = x[e];
  };
  if (!GRAD && ep.act == PL_ACT_NONE) {
    // nothing to compute: every column's C at once
    const T alpha = (T)ep.alpha, beta = (T)ep.beta;
    EpilogueInputs<T, T, false, VEC> in[STEPS];
#pragma unroll
    for (int it = 0; it < STEPS; ++it) {
      const long n = n0 + column(it);
      in[it].load(ep, (const T*)ep.C + n * ep.ldc + m, nullptr, n < N ? valid : 0);
    }
#pragma unroll
    for (int it = 0; it < STEPS; ++it) {
      const long n = n0 + column(it);
      if (n >= N || valid <= 0) continue;
      T v[VEC];
      product(column(it), v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fma(alpha, v[e], bias[e]);
      if (ep.preact) store_row<T, VEC, T>((T*)ep.preact + n * ep.ldp + m, v, valid);
      if (beta != T(0)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = fma(beta, in[it].c[e], v[e]);
      }
      store_row<T, VEC, T>((T*)ep.D + n * ep.ldd + m, v, valid);
    }
    return;
  }
#pragma unroll(sizeof(T) == 8 ? 1 : 2)
  for (int it = 0; it < STEPS; ++it) {
    const long n = n0 + column(it);
    if (n >= N || valid <= 0) continue;
    EpilogueInputs<T, T, GRAD, VEC> in;
    in.load(ep, (const T*)ep.C + n * ep.ldc + m, (const T*)ep.Z + n * ep.ldz + m, valid);
    T v[VEC];
    product(column(it), v);
    apply_epilogue<T, T, GRAD, VEC>(ep, in, v, bias, (T*)ep.D + n * ep.ldd + m, (T*)ep.preact + n * ep.ldp + m, valid, sums);
  }
  if constexpr (GRAD) {
    if (ep.partial) {
      // one row of partial sums per tile column: lanes and then waves that hold the same rows, in a fixed order
#pragma unroll
      for (int e = 0; e < VEC; ++e)
#pragma unroll
        for (int d = LPC; d < 64; d <<= 1) sums[e] += __shfl_xor(sums[e], d);
      __syncthreads();
      if (lane < LPC) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) lds[wave * 64 + mv + e] = sums[e];
      }
      __syncthreads();
      if (tid < 64 && m0 + tid < M) ((T*)ep.partial)[(long)bn * M + m0 + tid] = ((lds[tid] + lds[64 + tid]) + lds[128 + tid]) + lds[192 + tid];
    }
  }
}

template <typename T>
int launch_wide(const WidePlan& plan, bool at, bool bt, bool grad, long M, long N, long K, const void* A, long lda, const void* B, long ldb, const Epilogue& ep, hipStream_t stream) {
  const long gm = (M + 63) / 64, gn = (N + 63) / 64;
#define WIDE(AKF, BKF, GRADF)                                                                                                                          \
  return launch(wide_tile_kernel<T, AKF, BKF, GRADF>, dim3((unsigned)(gm * gn), (unsigned)plan.splits), dim3(256), stream, (int)M, (int)N, (int)K,     \
                (const T*)A, lda, (const T*)B, ldb, (int)gm, plan.splits > 1 ? plan.kchunk : (int)K, ep)
#define WIDE_LAYOUT(GRADF)                  \
  do {                                      \
    if (at && !bt) WIDE(true, true, GRADF); \
    if (at) WIDE(true, false, GRADF);       \
    if (!bt) WIDE(false, true, GRADF);      \
    WIDE(false, false, GRADF);              \
  } while (0)
  if (grad) WIDE_LAYOUT(true);
  WIDE_LAYOUT(false);
#undef WIDE_LAYOUT
#undef WIDE
}

// D, or the slices of a split product and the pass that adds and finishes them
template <typename T> int wide_product(const Call& c, const WidePlan& plan, bool at, bool bt, const Epilogue& ep, void* slices) {
  if (plan.splits == 1) return launch_wide<T>(plan, at, bt, c.grad, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, ep, c.stream);
  Epilogue plain = {};
  plain.alpha = 1.0;
  plain.D = slices;
  plain.ldd = c.M;
  int rc = launch_wide<T>(plan, at, bt, false, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, plain, c.stream);
  int left = plan.splits;
  if (rc == PL_OK && c.grad && sizeof(T) == 8) {   // (that pass takes no slices)
    rc = epilogue_pass(c.type, c.type_d, false, c.M, c.N, slices, c.M, c.M * c.N, left, plain, c.stream);
    left = 1;
  }
  return rc != PL_OK ? rc : epilogue_pass(c.type, c.type_d, c.grad, c.M, c.N, slices, c.M, c.M * c.N, left, ep, c.stream);
}

}  // namespace plk
#endif
