// 16-bit (bf16, fp16) matrix product with a fused epilogue for gfx950 (MI355X), column-major; its sources are one per operand
// type and direction, so that they compile side by side.
//
// The 16-bit kernel: one workgroup = 4 waves (2 x 2), v_mfma_f32_32x32x16 on 64-deep panels of A and B in LDS.  A panel is
// kept as it lies in memory, K-major ([row][64 k], 128 bytes a row) or MN-major ([64 k][row]), in 16-byte granules whose
// position is swizzled so that neither operand reads nor loads collide in the banks:
//   * K-major: granule c of row r sits at c ^ (r / 2 mod 8): a lane reads its row's 8 k of an MFMA with one ds_read_b128,
//     and 16 consecutive rows touch all 64 banks once;
//   * MN-major: ds_read_b64_tr_b16 hands a lane 4 k of its row out of four k-rows, which have to lie in four different
//     quarters of the banks.  Each 1 KiB that is loaded together holds k-rows k, k + 4, ... and starts 64 bytes past a
//     multiple of 256 behind the one before it, which holds k + 1, k + 5, ...
// Both are filled by 1 KiB requests of global_load_lds_dwordx4: lane l's 16 bytes land at base + 16 l, and what goes there
// is in the global address each lane asks for.  (MN-major rows swizzled in 64-byte pieces like the K-major ones, without
// the padding, have no bank conflicts either, but the requests then run at a quarter of their rate: NT 411 against 1159
// TFLOP/s at 4096 x 4096 x 8192.)  Rows beyond the matrix ask for the last valid one again (their products are not
// stored), so ragged edges run the same loop.
#ifndef PLK_HALF_PRODUCT_H
#define PLK_HALF_PRODUCT_H
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

__device__ __forceinline__ floatx16 mfma16(short8_t a, short8_t b, floatx16 c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma16(short8_t a, short8_t b, floatx16 c, f16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// s_waitcnt: at most n vector memory operations left, nothing else waited for
constexpr int vm_wait(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }

// A panel of EXT rows of op(A) (columns of op(B)) by H_BK values of k, in 16-byte granules of 8 elements; 64 granules, what
// one request of a wave loads, are a piece.
template <bool KMAJOR, int EXT> struct HalfPanel {
  static constexpr int PER_ROW = KMAJOR ? H_BK / 8 : EXT / 8;       // granules along the contiguous dimension
  static constexpr int PIECES = EXT * H_BK / 512;
  static constexpr int PITCH = KMAJOR ? 512 : 544;                  // elements from piece to piece
  static constexpr int SLOTS = 64 / PER_ROW;                        // rows of a piece
  static constexpr int ELEMS = PIECES * PITCH;
  static constexpr int NV = PIECES / 4;                             // granules per thread = requests per wave
  static __device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }   // K-major
  // granule `lane` of a piece: which row (of the strided dimension: mn, or k) and which granule of that row it holds
  static __device__ __forceinline__ void holds(int piece, int lane, int& row, int& granule) {
    if (KMAJOR) {
      row = piece * 8 + lane / 8;
      granule = (lane % 8) ^ swizzle(row);
    } else {
      row = (piece / 4) * 4 * SLOTS + (lane / PER_ROW) * 4 + piece % 4;
      granule = lane % PER_ROW;
    }
  }
  // where element (k, mn) of an MN-major panel sits
  static __device__ __forceinline__ int at(int k, int mn) { return ((k / (4 * SLOTS)) * 4 + k % 4) * PITCH + ((k / 4) % SLOTS) * EXT + mn; }
};

// Byte offsets, from a panel's first element, of what the lanes of a wave ask for with their NV requests.  rows_left:
// rows (columns) of the operand from the panel's first on; what lies beyond is replaced by the last valid row or granule.
template <typename P, bool KMAJOR>
__device__ __forceinline__ void request_offsets(unsigned (&off)[P::NV], long ld, int rows_left, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < P::NV; ++i) {
    int row, g;
    P::holds(wave + 4 * i, lane, row, g);
    if (KMAJOR) row = min(row, rows_left - 1);
    else g = min(g, (rows_left - 1) >> 3);
    off[i] = (unsigned)row * (unsigned)ld * 2u + (unsigned)g * 16u;
  }
}

// The same for loads through registers, which need no alignment.  MN-major: from the start of the panel's first k-row, of
// which `first` is the tile's first element and `extent` the number of elements (at least 8); the granule that reaches
// past them is read 8 elements short of their end, and its first elements, as many as this returns, are dropped later.
template <typename P, bool KMAJOR>
__device__ __forceinline__ int load_offsets(unsigned (&off)[P::NV], long ld, int first, int extent, int tid) {
  int row, g;
  P::holds(tid / 64, tid % 64, row, g);   // (the same granule for all of a thread's vectors)
  const int start = KMAJOR ? g * 8 : min(first + g * 8, extent - 8);
#pragma unroll
  for (int i = 0; i < P::NV; ++i) {
    int r, unused;
    P::holds(tid / 64 + 4 * i, tid % 64, r, unused);
    if (KMAJOR) r = min(r, extent - first - 1);
    off[i] = (unsigned)r * (unsigned)ld * 2u + (unsigned)start * 2u;
  }
  return KMAJOR ? 0 : min(8, first + g * 8 - start);
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
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const short*>(base + off), xs + (wave + 4 * i) * P::PITCH, 16, 0, 0);
#endif
}

// v without its first d elements, zeros behind (0 <= d <= 8).  Bit masks rather than conditions: a condition per lane is a
// pair of scalar registers, and those run out here.
__device__ __forceinline__ short8_t drop_front(short8_t v, int d) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  u32x4 x = __builtin_bit_cast(u32x4, v);
  const unsigned half = (d & 1) * 16, one = (unsigned)((d << 30) >> 31), two = (unsigned)((d << 29) >> 31), none = ~(unsigned)((d << 28) >> 31);
  x[0] = __builtin_amdgcn_alignbit(x[1], x[0], half);
  x[1] = __builtin_amdgcn_alignbit(x[2], x[1], half);
  x[2] = __builtin_amdgcn_alignbit(x[3], x[2], half);
  x[3] = x[3] >> half;
  x[0] = (x[1] & one) | (x[0] & ~one);
  x[1] = (x[2] & one) | (x[1] & ~one);
  x[2] = (x[3] & one) | (x[2] & ~one);
  x[3] &= ~one;
  x[0] = ((x[2] & two) | (x[0] & ~two)) & none;
  x[1] = ((x[3] & two) | (x[1] & ~two)) & none;
  x[2] &= ~two & none;
  x[3] &= ~two & none;
  return __builtin_bit_cast(short8_t, x);
}

// A panel through registers, whatever the alignment.  strided: valid rows of the strided dimension (mn of a K-major operand,
// k of an MN-major one) from the panel's first on; contig: valid elements along the contiguous one, whose rows have at
// least 8 in all.  All loads are unconditional vector loads inside the matrix, so that they are all in flight
// at once: rows beyond the last repeat it, and the granule that reaches past the end of its row is read 8 elements short
// of that end and shifted into place.  k beyond the matrix becomes zero; rows and columns beyond it may be anything.
template <typename P, bool KMAJOR>
__device__ __forceinline__ void fetch_panel(const short* __restrict__ base, long ld, int strided, int contig, short8_t (&regs)[P::NV], int tid) {
#pragma unroll
  for (int i = 0; i < P::NV; ++i) {
    int row, g;
    P::holds(tid / 64 + 4 * i, tid % 64, row, g);
    regs[i] = *reinterpret_cast<const Loose<short>::type*>(base + (long)min(row, strided - 1) * ld + min(g * 8, contig - 8));
    regs[i] = drop_front(regs[i], min(8, max(0, g * 8 - (contig - 8))));
    if (!KMAJOR) regs[i] &= (short)((row - strided) >> 31);
  }
}
template <typename P>
__device__ __forceinline__ void put(short* xs, const short8_t (&regs)[P::NV], int tid) {
#pragma unroll
  for (int i = 0; i < P::NV; ++i) *reinterpret_cast<short8_t*>(xs + (tid / 64 + 4 * i) * P::PITCH + (tid % 64) * 8) = regs[i];
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

// Operand reads of a wave whose part of a panel starts at row `first`: what lane r = lane % 32, g = lane / 32 feeds an MFMA
// with is row r of block i and k = 16 s + 8 g .. + 7 of step s.  K-major: granule 2 s + g of the row; the swizzle repeats
// every 16 rows, so the steps need an offset each and the blocks a constant.  MN-major: lane % 16 / 4 picks one of four
// k-rows for the transposing read, which hands every lane its own row's four values; one offset, the rest constants.
template <bool KMAJOR, int EXT> struct Reader {
  using P = HalfPanel<KMAJOR, EXT>;
  static constexpr int NP = KMAJOR ? H_BK / 16 : 1;
  int at[NP];
  __device__ __forceinline__ Reader(int first, int lane) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int row = first + lane % 32;
      if (KMAJOR) at[p] = row * H_BK + (((2 * p + lane / 32) ^ P::swizzle(row)) << 3);
      else at[p] = P::at(8 * (lane / 32) + (lane % 16) / 4, first + 16 * ((lane / 16) & 1) + (lane & 3) * 4);
    }
  }
  __device__ __forceinline__ short8_t read(const short* xs, int i, int s) const {
    if constexpr (KMAJOR) {
      return *reinterpret_cast<const short8_t*>(xs + at[s] + i * 32 * H_BK);
    } else {
      short8_t v = {};
#if defined(__HIP_DEVICE_COMPILE__)
      typedef __attribute__((address_space(3))) short4_t* lds4;
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(xs + at[0] + P::at(16 * s, 0) + 32 * i));
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(xs + at[0] + P::at(16 * s, 0) + P::at(4, 0) + 32 * i));
      v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#endif
      return v;
    }
  }
};

// fast: 3: both operands can be requested and their rows read to a multiple of 8 elements, 2: requested, 1: leading dimensions within the offsets' range, 0: neither.  kchunk: split K (0: no).
template <typename T, typename TD, bool AK, bool BKM, int BM, int BN, int STAGES, bool GRAD>
__global__ __launch_bounds__(H_THREADS, (BM * BN * STAGES <= 128 * 128 * 2 ? 2 : 1)) void half_product_kernel(int M, int N, int K, const short* __restrict__ A, long lda,
                                                                                               const short* __restrict__ B, long ldb, int gm, int gn, int fast,
                                                                                               int kchunk, Epilogue ep) {
  using PA = HalfPanel<AK, BM>;
  using PB = HalfPanel<BKM, BN>;
  constexpr int WM = BM / 2, WN = BN / 2, NBM = WM / 32, NBN = WN / 32;
  constexpr int STAGE = PA::ELEMS + PB::ELEMS;
  constexpr int EP_LD = WM + 4;                       // floats per column of the epilogue's staging area
  static_assert(4 * 32 * EP_LD * 4 <= 2 * STAGE * 2, "the epilogue stages in the panels' memory");
  __shared__ __attribute__((aligned(1024))) short smem[STAGES * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave & 1) * WM, wn = (wave >> 1) * WN;
  int bm, bn;
  half_block_coords(blockIdx.x, gm, gn, bm, bn);
  const int m0 = bm * BM, n0 = bn * BN;
  const int mrem = min(M - m0, BM), nrem = min(N - n0, BN);
  if (kchunk > 0) {
    // split K: the workgroups of grid row y multiply k in [y * kchunk, (y + 1) * kchunk) and leave their plain partial
    // product in slice y (M x N, dense) of D; a pass adds the slices in order and applies the epilogue
    const int k0 = blockIdx.y * kchunk;
    A += AK ? (long)k0 : (long)k0 * lda;
    B += BKM ? (long)k0 : (long)k0 * ldb;
    K = min(K - k0, kchunk);
    ep.D = (TD*)ep.D + (long)blockIdx.y * M * N;
  }
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

  const Reader<AK, BM> ra(wm, lane);
  const Reader<BKM, BN> rb(wn, lane);
  auto multiply = [&](const short* xs) {   // the operands of a step are read in front of the MFMAs of the one before it
    constexpr int SETS = BM > 128 ? 1 : 2;   // (the large tile comes here for the rest of K only, and has no registers to spare)
    short8_t a[SETS][NBM], b[SETS][NBN];
    auto read = [&](int s) {
#pragma unroll
      for (int i = 0; i < NBM; ++i) a[s % SETS][i] = ra.read(xs, i, s);
#pragma unroll
      for (int j = 0; j < NBN; ++j) b[s % SETS][j] = rb.read(xs + PA::ELEMS, j, s);
    };
    if (SETS > 1) read(0);
#pragma unroll
    for (int s = 0; s < H_BK / 16; ++s) {
      if (SETS == 1) read(s);
      else if (s + 1 < H_BK / 16) read(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NBM; ++i)
#pragma unroll
        for (int j = 0; j < NBN; ++j) acc[i][j] = mfma16(a[s % SETS][i], b[s % SETS][j], acc[i][j], T());
    }
  };

  // Whole panels that the requests may load.  The last granule of an MN-major row at the edge of the matrix reaches past
  // it where the extent is not a multiple of 8; behind every k-row but the last that is still the operand's own memory
  // (its leading dimension is a multiple of 8), so the last k-row is left to the guarded step.
  const bool last_row_guarded = fast < 3 && ((!AK && mrem < BM && (M & 7)) || (!BKM && nrem < BN && (N & 7)));
  const int nfull = fast >= 2 ? (K - (last_row_guarded ? 1 : 0)) / H_BK : 0;
  if (nfull > 0) {
    unsigned oa[PA::NV], ob[PB::NV];
    request_offsets<PA, AK>(oa, lda, mrem, wave, lane);
    request_offsets<PB, BKM>(ob, ldb, nrem, wave, lane);
    constexpr int NR = PA::NV + PB::NV, EARLY = NR / 2;   // requests per wave and panel; how many of them go out a step early
    // request r of panel kt: A's first
    auto ask = [&](const char* base_a, const char* base_b, short* xs, int r) {
      if (r < PA::NV) request<PA>(base_a, oa[r], xs, wave, r);
      else request<PB>(base_b, ob[r - PA::NV], xs + PA::ELEMS, wave, r - PA::NV);
    };
    short8_t fa[2][NBM], fb[2][NBN];
    auto read = [&](const short* xs, int s, int set, int e) {
      if (e < NBM) fa[set][e] = ra.read(xs, e, s);
      else fb[set][e - NBM] = rb.read(xs + PA::ELEMS, e - NBM, s);
    };
    constexpr int STEPS = H_BK / 16, READS = NBM + NBN, MFMAS = NBM * NBN, SPREAD = MFMAS > 4 ? MFMAS * 3 / 4 : MFMAS / 2;   // (the reads go out early enough to be done when the step ends)
    // One panel.  The operands of a step are read during the step before it, so the panel's barrier sits in front of its
    // last step: from there on every wave has read all of panel kt, panel kt + 1 is complete, and the requests of panel
    // kt + STAGES may fill panel kt's buffer, the first half of them at once, the rest during the next panel's first step.
    // The source is in issue order, an MFMA and then what goes out behind it.  STEADY: all those panels exist.
    // (__restrict__: a transposing read that the compiler cannot tell from the requests' buffer waits for all of them.  With two
    // stages the buffer behind this panel's is also the one before it: it is then reached through nxt alone.)
    const short* next_a = Ab + (STAGES - 1) * a_step;   // the panel that is being asked for
    const short* next_b = Bb + (STAGES - 1) * b_step;
    constexpr int NEWER = (STAGES - 2) * NR;   // requests that may be out when panel kt + 1 has landed
    auto panel = [&]<bool STEADY>(int kt, short* __restrict__ cur, short* __restrict__ nxt, short* __restrict__ prv) __attribute__((always_inline)) {
      short* const fill = STAGES == 2 ? nxt : prv;
      const bool ask1 = STEADY || kt + STAGES - 1 < nfull, ask2 = STEADY || kt + STAGES < nfull, next = STEADY || kt + 1 < nfull;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const bool last = s == STEPS - 1;
        if (last) next_a += a_step, next_b += b_step;
        const char* const pa = uniform_base(next_a);
        const char* const pb = uniform_base(next_b);
        if (last && next) {
          // this wave's part of panel kt + 1 is in LDS (vmcnt), and its last reads of panel kt are done (lgkmcnt)
          if (ask1) __builtin_amdgcn_s_waitcnt(vm_wait(NEWER) & ~0x0F00);
          else __builtin_amdgcn_s_waitcnt(vm_wait(0) & ~0x0F00);
          __builtin_amdgcn_s_barrier();
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int m = 0; m < MFMAS; ++m) {
          const int i = m / NBN, j = m % NBN;
          acc[i][j] = mfma16(fa[s & 1][i], fb[s & 1][j], acc[i][j], T());
          if (!last || next) {
#pragma unroll
            for (int e = 0; e < READS; ++e)
              if (e * SPREAD / READS == m) read(last ? nxt : cur, last ? 0 : s + 1, (s + 1) & 1, e);
          }
          if (s == 0 && ask1) {
#pragma unroll
            for (int r = EARLY; r < NR; ++r)
              if ((r - EARLY) * MFMAS / (NR - EARLY) == m) ask(pa, pb, fill, r);
          }
          if (last && ask2) {
#pragma unroll
            for (int r = 0; r < EARLY; ++r)
              if (r * MFMAS / EARLY == m) ask(pa, pb, cur, r);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
#pragma unroll
    for (int q = 0; q < STAGES; ++q) {
      const char* const a0 = uniform_base(Ab + q * a_step);
      const char* const b0 = uniform_base(Bb + q * b_step);
      if (q < nfull) {
#pragma unroll
        for (int r = 0; r < (q == STAGES - 1 ? EARLY : NR); ++r) ask(a0, b0, smem + q * STAGE, r);
      }
    }
    if (nfull >= STAGES) __builtin_amdgcn_s_waitcnt(vm_wait(NEWER + EARLY));   // panel 0 has landed
    else __builtin_amdgcn_s_waitcnt(vm_wait(0));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    static_assert(NEWER + EARLY < 64, "the wait counter's range");
#pragma unroll
    for (int e = 0; e < READS; ++e) read(smem, 0, 0, e);
    int kt = 0;
    for (; kt + 2 * STAGES - 1 < nfull; kt += STAGES) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u)
        panel.template operator()<true>(kt + u, smem + u * STAGE, smem + (u + 1) % STAGES * STAGE, smem + (u + STAGES - 1) % STAGES * STAGE);
    }
    for (; kt < nfull; kt += STAGES) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u)
        if (kt + u < nfull) panel.template operator()<false>(kt + u, smem + u * STAGE, smem + (u + 1) % STAGES * STAGE, smem + (u + STAGES - 1) % STAGES * STAGE);
    }
    __syncthreads();
  }
  int done = nfull;
  if constexpr (BM == 128 && STAGES == 2) {   // (the launcher gives such operands to this tile)
    // Unaligned operands: whole panels through registers, loaded two panels ahead.  No branch between the loads and their
    // use, which would make every use wait for all loads.
    if (fast == 1 && K >= H_BK) {
      unsigned oa[PA::NV], ob[PB::NV];
      const int drop_a = load_offsets<PA, AK>(oa, lda, m0, M, tid), drop_b = load_offsets<PB, BKM>(ob, ldb, n0, N, tid);
      const short* const base_a = AK ? Ab : A;
      const short* const base_b = BKM ? Bb : B;
      const bool edge_a = !AK && mrem < BM, edge_b = !BKM && nrem < BN;
      done = K / H_BK;
      short8_t va[2][PA::NV], vb[2][PB::NV];
      auto load = [&](int kt, int set) {
        kt = min(kt, done - 1);
        const char* const ba = uniform_base(base_a + kt * a_step);
        const char* const bb = uniform_base(base_b + kt * b_step);
#pragma unroll
        for (int i = 0; i < PA::NV; ++i) va[set][i] = *reinterpret_cast<const Loose<short>::type*>(reinterpret_cast<const short*>(ba + oa[i]));
#pragma unroll
        for (int i = 0; i < PB::NV; ++i) vb[set][i] = *reinterpret_cast<const Loose<short>::type*>(reinterpret_cast<const short*>(bb + ob[i]));
      };
      auto step = [&](int kt, int set) {
        if (edge_a) {
#pragma unroll
          for (int i = 0; i < PA::NV; ++i) va[set][i] = drop_front(va[set][i], drop_a);
        }
        if (edge_b) {
#pragma unroll
          for (int i = 0; i < PB::NV; ++i) vb[set][i] = drop_front(vb[set][i], drop_b);
        }
        short* const xs = smem + set * STAGE;
        put<PA>(xs, va[set], tid);
        put<PB>(xs + PA::ELEMS, vb[set], tid);
        __syncthreads();
        load(kt + 2, set);
        multiply(xs);
      };
      load(0, 0);
      load(1, 1);
      for (int kt = 0;; kt += 2) {
        step(kt, 0);
        if (kt + 1 >= done) break;
        step(kt + 1, 1);
        if (kt + 2 >= done) break;
      }
      __syncthreads();
    }
  }
  // The rest of K, and all of it where leading dimensions leave the offsets' range.
  for (int kt = done; kt * H_BK < K; ++kt) {
    short8_t va[PA::NV], vb[PB::NV];
    const int krem = K - kt * H_BK;
    fetch_panel<PA, AK>(Ab + kt * a_step, lda, AK ? mrem : krem, AK ? krem : M - m0, va, tid);
    fetch_panel<PB, BKM>(Bb + kt * b_step, ldb, BKM ? nrem : krem, BKM ? krem : N - n0, vb, tid);
    put<PA>(smem, va, tid);
    put<PB>(smem + PA::ELEMS, vb, tid);
    __syncthreads();
    multiply(smem);
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
  // What the epilogue reads is loaded 32 columns ahead: without that its latency shows 32 times per tile (C: 19, Z: 23 us
  // of a 256 x 256 tile's round at 16384 x 8192 against 13 for all the rest of its end).
  constexpr int ITS = 32 / CPI;
  EpilogueInputs<T, TD, GRAD, 8> in[ITS];
  // (pointers that move on by CPI columns: a 64-bit product per access costs more than the activation)
  int n_in = n0 + wn + lane / LPC, n = n_in;
  const TD* pc = (const TD*)ep.C + n * ep.ldc + m;
  const T* pz = (const T*)ep.Z + n * ep.ldz + m;
  TD* pd = (TD*)ep.D + n * ep.ldd + m;
  T* pp = (T*)ep.preact + n * ep.ldp + m;
  auto load_inputs = [&](int it) {
    in[it].load(ep, pc, pz, n_in < N ? valid : 0);
    pc += CPI * ep.ldc;
    if (GRAD) pz += CPI * ep.ldz;
    n_in += CPI;
  };
#pragma unroll
  for (int it = 0; it < ITS; ++it) load_inputs(it);
#pragma unroll 1
  for (int j = 0; j < NBN; ++j) {
#pragma unroll
    for (int jj = 0; jj < NBN; ++jj) {
      if (jj != j) continue;   // (a uniform branch: accumulators cannot be indexed)
#pragma unroll
      for (int i = 0; i < NBM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          floatx4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][jj][4 * q + e];
          *reinterpret_cast<floatx4*>(stage + (lane % 32) * EP_LD + 32 * i + 8 * q + 4 * (lane / 32)) = v;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
      const int c = it * CPI + lane / LPC;
      float v[8];
      const floatx4 lo = *reinterpret_cast<const floatx4*>(stage + c * EP_LD + sub * 8), hi = *reinterpret_cast<const floatx4*>(stage + c * EP_LD + sub * 8 + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
      if (n < N && valid > 0) apply_epilogue<T, TD, GRAD, 8>(ep, in[it], v, bias, pd, pp, valid, sums);
      pd += CPI * ep.ldd;
      if (!GRAD) pp += CPI * ep.ldp;
      n += CPI;
      if (j + 1 < NBN) load_inputs(it);
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

// ---- few columns (single tokens and small batches of them) ----
// op(A) K-major, op(B) K-major, at most 32 columns: reading A once bounds it, and its latency.  A workgroup owns 16 RB rows
// of D whole, so there is one launch and no slices: its WAVES waves split K, each with a ring of D panels of its own in LDS
// (16 RB rows of A and 16 NB columns of B, 64 deep) that it fills with requests and waits for by itself, without a
// barrier; 64 KiB of A are in flight per compute unit.  The waves' sums are added in wave order.

__device__ __forceinline__ floatx4 mfma16_small(short8_t a, short8_t b, floatx4 c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma16_small(short8_t a, short8_t b, floatx4 c, f16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename T, typename TD, int RB, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void half_few_columns_kernel(int M, int N, int K, const short* __restrict__ A, long lda, const short* __restrict__ B,
                                                                             long ldb, Epilogue ep) {
  constexpr int PIECES = 2 * (RB + NB), RING = 16 / PIECES, SLOT = PIECES * 512;   // requests per panel, panels in flight, elements per panel
  constexpr int ROWS = 16 * RB, COLS = 16 * NB, EP_LD = ROWS + 4;
  static_assert(COLS * EP_LD * 2 <= RING * SLOT, "a wave's sums go where its ring was");
  __shared__ __attribute__((aligned(1024))) short smem[WAVES * RING * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  short* const mine = smem + wave * RING * SLOT;
  const int m0 = blockIdx.x * ROWS;

  unsigned off[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int r = i * 8 + lane / 8, g = (lane % 8) ^ ((r >> 1) & 7);
    const int row = i < 2 * RB ? min(r, M - 1 - m0) : min(r - ROWS, N - 1);
    off[i] = (unsigned)row * (unsigned)(i < 2 * RB ? lda : ldb) * 2u + (unsigned)g * 16u;
  }
  const int panels = K / H_BK, first = panels * wave / WAVES, last = panels * (wave + 1) / WAVES;
  const short* const Ab = A + (long)m0 * lda;
  auto ask = [&](int p, int slot) {
#if defined(__HIP_DEVICE_COMPILE__)
    const char* const ba = uniform_base(Ab + (long)p * H_BK);
    const char* const bb = uniform_base(B + (long)p * H_BK);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const short*>((i < 2 * RB ? ba : bb) + off[i]), mine + slot * SLOT + i * 512, 16, 0, 0);
#endif
  };
  floatx4 acc[RB][NB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  int at[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) at[s] = (lane % 16) * H_BK + (((4 * s + lane / 16) ^ ((lane % 16) >> 1)) << 3);
#pragma unroll
  for (int d = 0; d < RING; ++d)
    if (first + d < last) ask(first + d, d);
  int slot = 0;
  for (int p = first; p < last; ++p) {
    if (p + RING <= last) __builtin_amdgcn_s_waitcnt(vm_wait((RING - 1) * PIECES));   // panel p has landed, RING - 1 newer ones may be out
    else __builtin_amdgcn_s_waitcnt(vm_wait(0));
    const short* const xs = mine + slot * SLOT;
    short8_t a[2][RB], b[2][NB];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < RB; ++i) a[s][i] = *reinterpret_cast<const short8_t*>(xs + at[s] + i * 16 * H_BK);
#pragma unroll
      for (int j = 0; j < NB; ++j) b[s][j] = *reinterpret_cast<const short8_t*>(xs + at[s] + (RB + j) * 16 * H_BK);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): the panel is in registers, its slot may be filled again
    if (p + RING < last) ask(p + RING, slot);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma16_small(a[s][i], b[s][j], acc[i][j], T());
    slot = slot + 1 == RING ? 0 : slot + 1;
  }
  float* const sums = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) *reinterpret_cast<floatx4*>(sums + (16 * j + lane % 16) * EP_LD + 16 * i + 4 * (lane / 16)) = acc[i][j];
  __syncthreads();
  const int sub = tid % (2 * RB), n = tid / (2 * RB), m = m0 + 8 * sub, valid = max(0, min(8, M - m));
  if (n < N && n < COLS && valid > 0) {
    EpilogueInputs<T, TD, false, 8> in;
    in.load(ep, (const TD*)ep.C + n * ep.ldc + m, nullptr, valid);
    float v[8], bias[8], unused[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = bias[e] = unused[e] = 0.0f;
    if (ep.bias) load_row<T, 8, float>((const T*)ep.bias + m, bias, valid);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float* const q = reinterpret_cast<const float*>(smem + w * RING * SLOT) + n * EP_LD + 8 * sub;
      const floatx4 lo = *reinterpret_cast<const floatx4*>(q), hi = *reinterpret_cast<const floatx4*>(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += lo[e], v[4 + e] += hi[e];
    }
    apply_epilogue<T, TD, false, 8>(ep, in, v, bias, (TD*)ep.D + n * ep.ldd + m, (T*)ep.preact + n * ep.ldp + m, valid, unused);
  }
}

template <typename T, typename TD>
int launch_few_columns(long M, long N, long K, const void* A, long lda, const void* B, long ldb, const Epilogue& ep, hipStream_t stream) {
#define FEW(RB, NB, WAVES)                                                                                                                              \
  return launch(half_few_columns_kernel<T, TD, RB, NB, WAVES>, dim3((unsigned)((M + 16 * RB - 1) / (16 * RB))), dim3(WAVES * 64), stream, (int)M, (int)N, \
                (int)K, (const short*)A, lda, (const short*)B, ldb, ep)
  // One workgroup of eight waves per compute unit up to 256 of them; more come in fours, two to a unit, so that one's first
  // requests and its sums overlap the other's stream; 32 rows each where that still gives every unit two: half the reads of B.
  const long blocks = (M + 15) / 16;
#define FEW_COLUMNS(NB)                    \
  do {                                     \
    if (blocks <= 256) FEW(1, NB, 8);      \
    if (blocks < 1024) FEW(1, NB, 4);      \
    FEW(2, NB, 4);                         \
  } while (0)
  if (N <= 16) FEW_COLUMNS(1);
  FEW_COLUMNS(2);
#undef FEW_COLUMNS
#undef FEW
}

// Rows of fewer than 8 elements (K < 8 of a K-major operand, M or N < 8 of an MN-major one) are no 16-byte vectors: a thread
// per element of the product and slice of k (blockIdx.y), summed in order into the workspace for the pass to finish.  Eight
// k at a time: one 16-byte load of an operand whose k are adjacent, eight strided ones of the other.
// 4096 x 1 x 16384 NT (reading A: 27 us) 38 us, unsplit and element by element 1346; 4096 x 7 x 16384 131 (1316), bound by
// the 2-byte loads of A, which every column repeats out of the caches; 5 x 300 x 70000 NN 189 (6320).  More threads (2^20 -
// 2^22) change none of them.
template <typename T, bool KMAJOR> __device__ __forceinline__ void thin_load(const T* p, long ld, float (&v)[8]) {
  if constexpr (KMAJOR) {
    load_row<T, 8, float>(p, v, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)p[e * ld];
  }
}
template <typename T, bool AK, bool BKM>
__global__ __launch_bounds__(256) void half_thin_kernel(long M, long N, int K, int kchunk, const T* __restrict__ A, long lda, const T* __restrict__ B, long ldb,
                                                       float* __restrict__ product) {
  const long total = M * N, stride = (long)gridDim.x * 256;
  const int k0 = (int)blockIdx.y * kchunk, k1 = K - k0 < kchunk ? K : k0 + kchunk;
  product += (long)blockIdx.y * total;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
    const long n = i / M, m = i - n * M, a_k = AK ? 1 : lda, b_k = BKM ? 1 : ldb;
    const T* a = A + (AK ? m * lda : m) + k0 * a_k;
    const T* b = B + (BKM ? n * ldb : n) + k0 * b_k;
    float s = 0.0f;
    int left = k1 - k0;
#pragma unroll 2
    for (; left >= 8; left -= 8, a += 8 * a_k, b += 8 * b_k) {
      float x[8], y[8];
      thin_load<T, AK>(a, lda, x);
      thin_load<T, BKM>(b, ldb, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
    }
    for (; left > 0; --left, a += a_k, b += b_k) s = fmaf((float)*a, (float)*b, s);
    product[i] = s;
  }
}

template <typename T, typename TD, bool GRAD>
int launch_half(const HalfPlan& plan, bool at, bool bt, bool padded, long M, long N, long K, const void* A, long lda, const void* B, long ldb, const Epilogue& ep, hipStream_t stream) {
  const int gm = (int)((M + plan.tile - 1) / plan.tile), gn = (int)((N + plan.tile - 1) / plan.tile);
  const int fast = padded ? 3 : can_request(A, lda, B, ldb) ? 2 : in_offset_range(lda, ldb) ? 1 : 0;
#define HALF(AKF, BKF, TILE, STAGES)                                                                                                                     \
  return launch(half_product_kernel<T, TD, AKF, BKF, TILE, TILE, STAGES, GRAD>, dim3(gm * gn, plan.splits), dim3(H_THREADS), stream, (int)M, (int)N, (int)K, \
                (const short*)A, lda, (const short*)B, ldb, gm, gn, fast, plan.kchunk, ep)
#define HALF_TILE(TILE, STAGES)                    \
  do {                                             \
    if (at && !bt) HALF(true, true, TILE, STAGES); \
    if (at) HALF(true, false, TILE, STAGES);       \
    if (!bt) HALF(false, true, TILE, STAGES);      \
    HALF(false, false, TILE, STAGES);              \
  } while (0)
  if (plan.tile == 256) HALF_TILE(256, 2);
  if (fast >= 2 && (long)gm * gn * plan.splits <= 256) HALF_TILE(128, 4);
  HALF_TILE(128, 2);
#undef HALF_TILE
#undef HALF
}

template <typename T, typename TD, bool GRAD>
int half_direct(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep) {
  if constexpr (!GRAD) {
    if (few_columns(c, at, bt)) return launch_few_columns<T, TD>(c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, ep, c.stream);
  }
  return launch_half<T, TD, GRAD>(plan, at, bt, c.padded, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, ep, c.stream);
}

// The product alone, as fp32 slices for the pass to add and finish.
template <typename T> int half_slices(const Call& c, const HalfPlan& plan, bool at, bool bt, void* slices) {
  if (plan.tile == 0) {
    const long blocks = (c.M * c.N + 255) / 256;
    const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192), (unsigned)plan.splits);
#define THIN(AKF, BKF)                                                                                                                          \
  return launch(half_thin_kernel<T, AKF, BKF>, grid, dim3(256), c.stream, c.M, c.N, (int)c.K, plan.splits > 1 ? plan.kchunk : (int)c.K, (const T*)c.A, \
                c.lda, (const T*)c.B, c.ldb, (float*)slices)
    if (at && !bt) THIN(true, true);
    if (at) THIN(true, false);
    if (!bt) THIN(false, true);
    THIN(false, false);
#undef THIN
  }
  Epilogue plain = {};
  plain.alpha = 1.0;
  plain.D = slices;
  plain.ldd = c.M;
  return launch_half<T, float, false>(plan, at, bt, c.padded, c.M, c.N, c.K, c.A, c.lda, c.B, c.ldb, plain, c.stream);
}

}  // namespace plk
#endif
