// Matrix product with a fused epilogue for gfx950 (MI355X), column-major:
//   pl_gemm_epilogue        D = act(alpha * op(A) * op(B) + bias) + beta * C         (linear layer, weight gradient)
//   pl_gemm_epilogue_grad   D = (alpha * op(A) * op(B) + beta * C) .* act'(Z), dbias (gradient through an activation)
// 16-bit operands (bf16, fp16) run the kernel of this file; fp32 and fp64 operands the library's tile GEMM
// (gemm_mfma.hip) with the epilogue as one pass over its product.
//
// The 16-bit kernel: one workgroup = 4 waves (2 x 2), v_mfma_f32_32x32x16 on 64-deep panels of A and B in LDS.  A panel is
// kept as it lies in memory, K-major ([row][64 k], 128 bytes a row) or MN-major ([64 k][row]), in 16-byte granules whose
// position is swizzled so that neither operand reads nor loads collide in the banks:
//   * K-major: granule c of row r sits at c ^ (r / 2 mod 8): a lane reads its row's 8 k of an MFMA with one ds_read_b128,
//     and 16 consecutive rows touch all 64 banks once;
//   * MN-major: granule g of k-row k sits at g ^ 4 (k mod 4): ds_read_b64_tr_b16 hands a lane 4 k of its row out of four
//     k-rows, which lie in four different quarters of the banks.
// Both layouts are unpadded, so that 1 KiB requests of global_load_lds_dwordx4 can fill them: lane l's 16 bytes land at
// base + 16 l, and the swizzle is in the global address each lane asks for.  Rows beyond the matrix ask for the last
// valid one again (their products are not stored), so ragged edges run the same loop.
#include "kernels/epilogue.h"
#include "kernels/linear.h"

namespace plk {

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr int H_THREADS = 256;
constexpr int H_BK = 64;

__device__ __forceinline__ floatx16 mfma16(short8_t a, short8_t b, floatx16 c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma16(short8_t a, short8_t b, floatx16 c, f16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A panel of EXT rows of op(A) (columns of op(B)) by H_BK values of k, in 16-byte granules of 8 elements.
template <bool KMAJOR, int EXT> struct HalfPanel {
  static constexpr int ELEMS = EXT * H_BK;
  static constexpr int GRANULES = ELEMS / 8;
  static constexpr int PER_ROW = KMAJOR ? H_BK / 8 : EXT / 8;       // granules along the contiguous dimension
  static constexpr int NV = GRANULES / H_THREADS;                   // granules per thread = requests per wave
  static __device__ __forceinline__ int swizzle(int row) { return KMAJOR ? (row >> 1) & 7 : (row & 3) << 2; }
  // granule v of the panel as it lies in LDS: which row (of the strided dimension) and which granule of that row it holds
  static __device__ __forceinline__ void holds(int v, int& row, int& granule) {
    row = v / PER_ROW;
    granule = (v % PER_ROW) ^ swizzle(row);
  }
};

// Byte offsets, from a panel's first element, of what the lanes of a wave ask for with their NV requests.  rows_left:
// rows (columns) of the operand from the panel's first on; what lies beyond is replaced by the last valid row or granule.
template <typename P, bool KMAJOR>
__device__ __forceinline__ void request_offsets(unsigned (&off)[P::NV], long ld, int rows_left, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < P::NV; ++i) {
    int row, g;
    P::holds((wave + 4 * i) * 64 + lane, row, g);
    if (KMAJOR) row = min(row, rows_left - 1);
    else g = min(g, (rows_left - 1) >> 3);
    off[i] = (unsigned)row * (unsigned)ld * 2u + (unsigned)g * 16u;
  }
}

// A wave-uniform pointer in scalar registers, so that a request is "scalar base + 32-bit lane offset".
__device__ __forceinline__ const char* uniform_base(const void* p) {
  const unsigned long long b = reinterpret_cast<unsigned long long>(p);
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)b), hi = __builtin_amdgcn_readfirstlane((unsigned)(b >> 32));
  return reinterpret_cast<const char*>(((unsigned long long)hi << 32) | lo);
}

// Request i of a wave: 1 KiB into the panel at xs.
template <typename P>
__device__ __forceinline__ void request(const char* base, unsigned off, short* xs, int wave, int i) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const short*>(base + off), xs + (wave + 4 * i) * 512, 16, 0, 0);
#endif
}

// The guarded way: granule v of the panel through registers, elements outside the matrix read as zero.
// contig: valid elements along the contiguous dimension, strided: valid rows of the other.
template <typename P, bool KMAJOR>
__device__ __forceinline__ void fetch_guarded(const short* __restrict__ base, long ld, int contig, int strided, short8_t (&regs)[P::NV], int tid) {
#pragma unroll
  for (int i = 0; i < P::NV; ++i) {
    int row, g;
    P::holds(tid + H_THREADS * i, row, g);
    const int left = row < strided ? contig - g * 8 : 0;
    const short* const p = base + (long)row * ld + g * 8;
    short8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (left >= 8) {
      v = *reinterpret_cast<const Loose<short>::type*>(p);
    } else if (left > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) v[e] = p[e];
    }
    regs[i] = v;
  }
}
template <typename P>
__device__ __forceinline__ void put(short* xs, const short8_t (&regs)[P::NV], int tid) {
#pragma unroll
  for (int i = 0; i < P::NV; ++i) *reinterpret_cast<short8_t*>(xs + (tid + H_THREADS * i) * 8) = regs[i];
}

// Workgroup id -> tile: the hardware deals ids round-robin over the 8 XCDs; each XCD gets a contiguous range of a walk
// in groups of GM tile rows, so that its L2 holds a compact block of panels.
__device__ __forceinline__ void half_block_coords(int bid, int gm, int gn, int& bm, int& bn) {
  constexpr int GM = 8;
  const int nb = gm * gn, xcd = bid & 7, loc = bid >> 3;
  const int q = nb >> 3, r = nb & 7;
  const int pid = (xcd < r) ? xcd * (q + 1) + loc : r * (q + 1) + (xcd - r) * q + loc;
  const int width = GM * gn, group = pid / width, first = group * GM;
  const int rows = min(gm - first, GM), in = pid - group * width;
  bm = __builtin_amdgcn_readfirstlane(first + in % rows);
  bn = __builtin_amdgcn_readfirstlane(in / rows);
}

// Lane pointers into a panel for the operand reads of a wave whose part starts at row `first`.
// K-major: block i (32 rows), k-step s: granule 2 s + lane / 32 of row first + 32 i + lane % 32; the swizzle repeats every
// 16 rows, so the four steps need a pointer each and the blocks a constant.  MN-major: k-row 16 s + 8 (lane / 32) + 4 h
// + lane % 16 / 4; the block sits in the swizzled bits, so the blocks need a pointer each and s and h a constant.
template <bool KMAJOR, int EXT, int NB> struct Reader {
  static constexpr int NP = KMAJOR ? H_BK / 16 : NB;
  int at[NP];
  __device__ __forceinline__ Reader(int first, int lane) {
    using P = HalfPanel<KMAJOR, EXT>;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if (KMAJOR) {
        const int row = first + lane % 32;
        at[p] = row * H_BK + (((2 * p + lane / 32) ^ P::swizzle(row)) << 3);
      } else {
        const int krow = 8 * (lane / 32) + (lane % 16) / 4, mn = first + 32 * p + 16 * ((lane / 16) & 1) + (lane & 3) * 4;
        at[p] = krow * EXT + (((mn >> 3) ^ P::swizzle(krow)) << 3) + (mn & 7);
      }
    }
  }
  __device__ __forceinline__ short8_t read(const short* xs, int i, int s) const {
    if constexpr (KMAJOR) {
      return *reinterpret_cast<const short8_t*>(xs + at[s] + i * 32 * H_BK);
    } else {
      short8_t v = {};
#if defined(__HIP_DEVICE_COMPILE__)
      typedef __attribute__((address_space(3))) short4_t* lds4;
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(xs + at[i] + 16 * s * EXT));
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(xs + at[i] + (16 * s + 4) * EXT));
      v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#endif
      return v;
    }
  }
};

// fast: both operands 16-byte aligned with leading dimensions that the request offsets span.
template <typename T, typename TD, bool AK, bool BKM, int BM, int BN, bool GRAD>
__global__ __launch_bounds__(H_THREADS, (BM * BN <= 128 * 128 ? 2 : 1)) void half_product_kernel(int M, int N, int K, const short* __restrict__ A, long lda,
                                                                                               const short* __restrict__ B, long ldb, int gm, int gn, int fast,
                                                                                               Epilogue ep) {
  using PA = HalfPanel<AK, BM>;
  using PB = HalfPanel<BKM, BN>;
  constexpr int WM = BM / 2, WN = BN / 2, NBM = WM / 32, NBN = WN / 32;
  constexpr int STAGE = PA::ELEMS + PB::ELEMS;
  constexpr int EP_LD = WM + 4;                       // floats per column of the epilogue's staging area
  static_assert(4 * 32 * EP_LD * 4 <= 2 * STAGE * 2, "the epilogue stages in the panels' memory");
  __shared__ __attribute__((aligned(1024))) short smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave & 1) * WM, wn = (wave >> 1) * WN;
  int bm, bn;
  half_block_coords(blockIdx.x, gm, gn, bm, bn);
  const int m0 = bm * BM, n0 = bn * BN;
  const int mrem = min(M - m0, BM), nrem = min(N - n0, BN);
  const short* const Ab = AK ? A + (long)m0 * lda : A + m0;
  const short* const Bb = BKM ? B + (long)n0 * ldb : B + n0;
  const long a_step = AK ? H_BK : (long)H_BK * lda, b_step = BKM ? H_BK : (long)H_BK * ldb;

  floatx16 acc[NBM][NBN];
#pragma unroll
  for (int i = 0; i < NBM; ++i)
#pragma unroll
    for (int j = 0; j < NBN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  const Reader<AK, BM, NBM> ra(wm, lane);
  const Reader<BKM, BN, NBN> rb(wn, lane);
  auto multiply = [&](const short* xs) {
#pragma unroll
    for (int s = 0; s < H_BK / 16; ++s) {
      short8_t a[NBM], b[NBN];
#pragma unroll
      for (int i = 0; i < NBM; ++i) a[i] = ra.read(xs, i, s);
#pragma unroll
      for (int j = 0; j < NBN; ++j) b[j] = rb.read(xs + PA::ELEMS, j, s);
#pragma unroll
      for (int i = 0; i < NBM; ++i)
#pragma unroll
        for (int j = 0; j < NBN; ++j) acc[i][j] = mfma16(a[i], b[j], acc[i][j], T());
    }
  };

  // Whole panels that the requests may load.  The last granule of an MN-major row at the edge of the matrix reaches past
  // it where the extent is not a multiple of 8; behind every k-row but the last that is still the operand's own memory
  // (its leading dimension is a multiple of 8), so the last k-row is left to the guarded step.
  const bool last_row_guarded = (!AK && mrem < BM && (M & 7)) || (!BKM && nrem < BN && (N & 7));
  const int nfull = fast ? (K - (last_row_guarded ? 1 : 0)) / H_BK : 0;
  if (nfull > 0) {
    unsigned oa[PA::NV], ob[PB::NV];
    request_offsets<PA, AK>(oa, lda, mrem, wave, lane);
    request_offsets<PB, BKM>(ob, ldb, nrem, wave, lane);
    auto ask = [&](int kt, short* xs) {
      const char* const ba = uniform_base(Ab + kt * a_step);
      const char* const bb = uniform_base(Bb + kt * b_step);
#pragma unroll
      for (int i = 0; i < PA::NV; ++i) request<PA>(ba, oa[i], xs, wave, i);
#pragma unroll
      for (int i = 0; i < PB::NV; ++i) request<PB>(bb, ob[i], xs + PA::ELEMS, wave, i);
    };
    ask(0, smem);
    for (int kt = 0; kt < nfull; ++kt) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of panel kt is in LDS
      __syncthreads();
      if (kt + 1 < nfull) ask(kt + 1, smem + ((kt + 1) & 1) * STAGE);
      multiply(smem + (kt & 1) * STAGE);
    }
    __syncthreads();
  }
  // The rest of K, and all of it where the operands cannot be requested: through registers, one panel ahead.
  if (nfull * H_BK < K) {
    short8_t fa[PA::NV], fb[PB::NV];
    auto fetch = [&](int kt) {
      const int krem = min(K - kt * H_BK, H_BK);
      fetch_guarded<PA, AK>(Ab + kt * a_step, lda, AK ? krem : mrem, AK ? mrem : krem, fa, tid);
      fetch_guarded<PB, BKM>(Bb + kt * b_step, ldb, BKM ? krem : nrem, BKM ? nrem : krem, fb, tid);
    };
    const int nk = (K + H_BK - 1) / H_BK;
    fetch(nfull);
    for (int kt = nfull; kt < nk; ++kt) {
      short* const xs = smem + (kt & 1) * STAGE;
      put<PA>(xs, fa, tid);
      put<PB>(xs + PA::ELEMS, fb, tid);
      __syncthreads();
      if (kt + 1 < nk) fetch(kt + 1);
      multiply(xs);
    }
    __syncthreads();
  }

  // Epilogue.  An accumulator block holds, per lane, 16 rows of one column; each wave turns 32 columns at a time through
  // its own stretch of LDS, so that a lane gets 8 consecutive rows and 8 or 16 lanes a whole stretch of a column: 16-byte
  // accesses of D, C, Z and z in full cache lines.  (No barrier: a wave reads only what it wrote itself.)
  float* const stage = reinterpret_cast<float*>(smem) + wave * 32 * EP_LD;
  constexpr int LPC = WM / 8, CPI = 64 / LPC;          // lanes per column, columns per step
  const int sub = lane % LPC;
  const long m = m0 + wm + sub * 8;
  const int valid = max(0, min(8, (int)(M - m)));
  float bias[8], sums[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bias[e] = sums[e] = 0.0f;
  if (!GRAD && ep.bias) load_row<T, 8, float>((const T*)ep.bias + m, bias, valid);
#pragma unroll
  for (int j = 0; j < NBN; ++j) {
#pragma unroll
    for (int i = 0; i < NBM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
        *reinterpret_cast<floatx4*>(stage + (lane % 32) * EP_LD + 32 * i + 8 * q + 4 * (lane / 32)) = v;
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int c0 = wn + 32 * j;
#pragma unroll 1
    for (int it = 0; it < 32 / CPI; ++it) {
      const int c = it * CPI + lane / LPC;
      const long n = n0 + c0 + c;
      if (n < N && valid > 0) {
        float v[8];
        const floatx4 lo = *reinterpret_cast<const floatx4*>(stage + c * EP_LD + sub * 8), hi = *reinterpret_cast<const floatx4*>(stage + c * EP_LD + sub * 8 + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
        apply_epilogue<T, TD, GRAD, 8>(ep, v, bias, m, n, valid, sums);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  if constexpr (GRAD) {
    if (ep.partial) {
      // the lanes that hold the same rows, then one row of partial sums per wave column of the grid
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = LPC; o < 64; o <<= 1) sums[e] += __shfl_xor(sums[e], o, 64);
      }
      if (lane < LPC) store_row<float, 8, float>((float*)ep.partial + (long)(bn * 2 + (wave >> 1)) * M + m, sums, valid);
    }
  }
}

struct HalfPlan { int tile, splits, kchunk; };
inline HalfPlan plan_half(bool, bool, long, long, long) { return {128, 1, 0}; }

// rows of partial bias gradients the 16-bit product leaves
inline long half_partial_rows(const HalfPlan& p, int type, long M, long N) {
  return p.splits > 1 ? epilogue_pass_rows(type, M, N) : 2 * ((N + p.tile - 1) / p.tile);
}

template <typename T, typename TD, bool GRAD>
int launch_half(bool at, bool bt, long M, long N, long K, const void* A, long lda, const void* B, long ldb, const Epilogue& ep, hipStream_t stream) {
  const HalfPlan plan = plan_half(at, bt, M, N, K);
  const int gm = (int)((M + plan.tile - 1) / plan.tile), gn = (int)((N + plan.tile - 1) / plan.tile);
  // requests: 16-byte granules, and offsets from a panel's first element in 32 bits (256 rows of a K-major operand, 64
  // k-rows of an MN-major one)
  const int fast = aligned_to(A, 16) && aligned_to(B, 16) && lda % 8 == 0 && ldb % 8 == 0 && lda < (1L << 22) && ldb < (1L << 22);
#define HALF(AKF, BKF, TILE)                                                                                                            \
  hipLaunchKernelGGL((half_product_kernel<T, TD, AKF, BKF, TILE, TILE, GRAD>), dim3(gm * gn), dim3(H_THREADS), 0, stream, (int)M, (int)N, \
                     (int)K, (const short*)A, lda, (const short*)B, ldb, gm, gn, fast, ep)
  if (at && !bt) HALF(true, true, 128);
  else if (at) HALF(true, false, 128);
  else if (!bt) HALF(false, true, 128);
  else HALF(false, false, 128);
#undef HALF
  return hipGetLastError() == hipSuccess ? PL_OK : PL_ERR_LAUNCH;
}

// The workspace of one call, in the order it is laid out: what the product needs, the product itself (fp32 and fp64
// operands), the partial bias gradients.
struct Workspace { long product_ws, product, partial; long bytes() const { return product_ws + product + partial; } };
inline long round16(long b) { return (b + 15) & ~15L; }
inline Workspace workspace_for(int type, bool at, bool bt, long M, long N, long K, bool dbias) {
  Workspace w = {0, 0, 0};
  const long wide = type == PL_TYPE_F64 ? 8 : 4;
  if (type_size(type) == 2) {
    const HalfPlan p = plan_half(at, bt, M, N, K);
    if (p.splits > 1) w.product = round16((long)p.splits * M * N * 4);
    if (dbias) w.partial = round16(half_partial_rows(p, type, M, N) * M * wide);
  } else {
    w.product_ws = round16(pl_gemm_tile_alone_workspace_bytes(at ? 'T' : 'N', bt ? 'T' : 'N', M, N, K, 1, type_size(type)));
    w.product = round16(M * N * wide);
    if (dbias) w.partial = round16(epilogue_pass_rows(type, M, N) * M * wide);
  }
  return w;
}

struct Call {
  const char* who;
  int type, type_d;
  char ta, tb;
  long M, N, K;
  double alpha;
  const void* A; long lda;
  const void* B; long ldb;
  Epilogue ep;
  bool grad;
  void* dbias;
  void* workspace; long workspace_bytes;
  hipStream_t stream;
};

template <typename T> int half_by_output(const Call& c, bool at, bool bt, const Epilogue& ep) {
  if (c.grad) return launch_half<T, T, true>(at, bt, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, ep, c.stream);
  if (c.type_d == PL_TYPE_F32) return launch_half<T, float, false>(at, bt, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, ep, c.stream);
  return launch_half<T, T, false>(at, bt, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, ep, c.stream);
}

int run_product(Call& c) {
  const char* const who = c.who;
  const bool at = c.ta == 'T' || c.ta == 't', an = c.ta == 'N' || c.ta == 'n', bt = c.tb == 'T' || c.tb == 't', bnn = c.tb == 'N' || c.tb == 'n';
  if (!valid_type(c.type)) return refuse(PL_ERR_ARG, who, "unknown element type");
  if (c.type_d != c.type && !(type_size(c.type) == 2 && c.type_d == PL_TYPE_F32)) return refuse(PL_ERR_ARG, who, "type_D is neither the operands' type nor fp32 for 16-bit operands");
  if (!valid_act(c.ep.act)) return refuse(PL_ERR_ARG, who, "unknown activation");
  if (!(at || an) || !(bt || bnn)) return refuse(PL_ERR_TRANS, who, "transpose flag is not N or T");
  const long M = c.M, N = c.N, K = c.K;
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX || ((M + 127) / 128) * ((N + 127) / 128) >= (1L << 24))
    return refuse(PL_ERR_DIM, who, "dimension out of range");
  auto short_ld = [](long ld, long rows) { return ld < (rows > 1 ? rows : 1); };
  Epilogue& ep = c.ep;
  const bool uses_c = ep.beta != 0.0, uses_z = c.grad && ep.act != PL_ACT_NONE;
  if (short_ld(c.lda, an ? M : K) || short_ld(c.ldb, bnn ? K : N) || short_ld(ep.ldd, M) || (uses_c && short_ld(ep.ldc, M)) || (uses_z && short_ld(ep.ldz, M)) ||
      (ep.preact && short_ld(ep.ldp, M)))
    return refuse(PL_ERR_LD, who, "leading dimension too small");
  if (M == 0) return PL_OK;
  if (N == 0) return c.dbias ? bias_fold(c.type, M, 0, nullptr, c.dbias, c.stream) : PL_OK;
  const bool empty = K == 0 || c.alpha == 0.0;   // A and B are not read
  if ((!empty && (!c.A || !c.B)) || !ep.D || (uses_c && !ep.C) || (uses_z && !ep.Z)) return refuse(PL_ERR_NULL, who, "null operand");
  const int es = type_size(c.type), ds = type_size(c.type_d);
  if ((!empty && (!aligned_to(c.A, es) || !aligned_to(c.B, es))) || !aligned_to(ep.D, ds) || (uses_c && !aligned_to(ep.C, ds)) || (uses_z && !aligned_to(ep.Z, es)) ||
      !aligned_to(ep.preact, es) || !aligned_to(ep.bias, es) || !aligned_to(c.dbias, es))
    return refuse(PL_ERR_ARG, who, "operand not aligned to its element size");
  const Range a = {empty ? nullptr : c.A, c.lda, an ? M : K, an ? K : M, es}, b = {empty ? nullptr : c.B, c.ldb, bnn ? K : N, bnn ? N : K, es};
  const Range d = {ep.D, ep.ldd, M, N, ds}, p = {ep.preact, ep.ldp, M, N, es}, rc = {uses_c ? ep.C : nullptr, ep.ldc, M, N, ds};
  const Range z = {uses_z ? ep.Z : nullptr, ep.ldz, M, N, es}, bias = {ep.bias, M, M, 1, es}, db = {c.dbias, M, M, 1, es};
  if (overlap(d, a) || overlap(d, b) || overlap(d, p) || overlap(d, bias) || overlap(d, db) || overlap(p, a) || overlap(p, b) || overlap(p, rc) || overlap(p, bias) ||
      overlap(db, a) || overlap(db, b) || overlap(db, rc) || overlap(db, z))
    return refuse(PL_ERR_ARG, who, "an output overlaps another operand");
  // D may be C, or Z, itself: an element is read before it is written, by the same thread
  if (!same_or_apart(d, rc) || !same_or_apart(d, z)) return refuse(PL_ERR_ARG, who, "D overlaps C or Z without being it");
  const Workspace w = workspace_for(c.type, at, bt, M, N, K, c.dbias != nullptr);
  if (w.bytes() > 0 && (!c.workspace || !aligned_to(c.workspace, 16) || c.workspace_bytes < w.bytes())) return refuse(PL_ERR_ARG, who, "workspace null, too small or not 16-byte aligned");
  char* const ws = (char*)c.workspace;
  ep.alpha = empty ? 0.0 : c.alpha;
  ep.partial = c.dbias ? ws + w.product_ws + w.product : nullptr;
  if (empty) c.K = 0;
  int rc_;
  long rows;
  if (es == 2) {
    const HalfPlan plan = plan_half(at, bt, M, N, K);
    rows = half_partial_rows(plan, c.type, M, N);
    rc_ = c.type == PL_TYPE_F16 ? half_by_output<f16_t>(c, at, bt, ep) : half_by_output<bf16_t>(c, at, bt, ep);
  } else {
    void* const product = ws + w.product_ws;
    rows = epilogue_pass_rows(c.type, M, N);
    if (c.type == PL_TYPE_F64)
      rc_ = pl_dgemm_tile_alone(c.ta, c.tb, M, N, c.K, 1.0, (const double*)c.A, c.lda, (const double*)c.B, c.ldb, 0.0, (double*)product, M, ws, w.product_ws, c.stream);
    else
      rc_ = pl_sgemm_tile_alone(c.ta, c.tb, M, N, c.K, 1.0f, (const float*)c.A, c.lda, (const float*)c.B, c.ldb, 0.0f, (float*)product, M, ws, w.product_ws, c.stream);
    if (rc_ == PL_OK) rc_ = epilogue_pass(c.type, c.type_d, c.grad, M, N, product, M, 0, 1, ep, c.stream);
  }
  if (rc_ != PL_OK || !c.dbias) return rc_;
  return bias_fold(c.type, M, rows, ep.partial, c.dbias, c.stream);
}

}  // namespace plk

extern "C" long pl_gemm_epilogue_workspace_bytes(int type, char transA, char transB, long M, long N, long K, int with_dbias) {
  using namespace plk;
  if (!valid_type(type) || M <= 0 || N <= 0 || K < 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
  const bool at = transA == 'T' || transA == 't', bt = transB == 'T' || transB == 't';
  return workspace_for(type, at, bt, M, N, K, with_dbias != 0).bytes();
}

extern "C" int pl_gemm_epilogue(int type, char transA, char transB, long M, long N, long K, double alpha, const void* A, long lda, const void* B, long ldb,
                                const pl_epilogue* epilogue, double beta, const void* C, long ldc, void* D, long ldd, void* workspace,
                                long workspace_bytes, void* stream) {
  plk::Call c = {};
  c.who = "pl_gemm_epilogue";
  if (!epilogue) return plk::refuse(PL_ERR_NULL, c.who, "null epilogue");
  c.type = type; c.type_d = epilogue->type_D;
  c.ta = transA; c.tb = transB; c.M = M; c.N = N; c.K = K; c.alpha = alpha;
  c.A = A; c.lda = lda; c.B = B; c.ldb = ldb;
  c.ep.beta = beta; c.ep.C = C; c.ep.ldc = ldc; c.ep.D = D; c.ep.ldd = ldd;
  c.ep.bias = epilogue->bias; c.ep.preact = epilogue->preact; c.ep.ldp = epilogue->ld_preact; c.ep.act = epilogue->activation;
  c.workspace = workspace; c.workspace_bytes = workspace_bytes; c.stream = (hipStream_t)stream;
  return plk::run_product(c);
}

extern "C" int pl_gemm_epilogue_grad(int type, char transA, char transB, long M, long N, long K, double alpha, const void* A, long lda, const void* B, long ldb,
                                     int activation, const void* Z, long ldz, double beta, const void* C, long ldc, void* D, long ldd, void* dbias,
                                     void* workspace, long workspace_bytes, void* stream) {
  plk::Call c = {};
  c.who = "pl_gemm_epilogue_grad";
  c.type = c.type_d = type;
  c.ta = transA; c.tb = transB; c.M = M; c.N = N; c.K = K; c.alpha = alpha;
  c.A = A; c.lda = lda; c.B = B; c.ldb = ldb;
  c.ep.beta = beta; c.ep.C = C; c.ep.ldc = ldc; c.ep.D = D; c.ep.ldd = ldd; c.ep.Z = Z; c.ep.ldz = ldz; c.ep.act = activation;
  c.grad = true; c.dbias = dbias;
  c.workspace = workspace; c.workspace_bytes = workspace_bytes; c.stream = (hipStream_t)stream;
  return plk::run_product(c);
}
