// Host side shared by the linear-layer operators: argument checks and the launchers that one source file calls in another.
#ifndef PLK_LINEAR_H
#define PLK_LINEAR_H
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <cmath>
#include <type_traits>

#include "backend/pl_internal.h"
#include "kernels/epilogue.h"
#include "paralia_hip.h"

namespace plk {

inline bool valid_type(int t) { return t >= PL_TYPE_F64 && t <= PL_TYPE_BF16; }
inline bool valid_act(int a) { return a >= PL_ACT_NONE && a <= PL_ACT_SILU; }
inline int type_size(int t) { return t == PL_TYPE_F64 ? 8 : t == PL_TYPE_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

inline int refuse(int code, const char* who, const char* why) {
  char text[200];
  snprintf(text, sizeof(text), "%s: %s", who, why);
  return pl_fail_msg(code, text);
}

// A launch without the triple-chevron's detour, arguments by reference: 128 tensors are 3.6 KB of them.
template <typename... P>
int launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, const std::type_identity_t<P>&... args) {
  void* list[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, list, 0, stream);
  if (e == hipSuccess) return PL_OK;
  (void)hipGetLastError();   // (reported here, not by the caller's next call)
  return refuse(PL_ERR_LAUNCH, "kernel launch", hipGetErrorString(e));
}

// A column-major operand's memory.
struct Range {
  const void* p;
  long ld, rows, cols;
  int size;
  uintptr_t first() const { return reinterpret_cast<uintptr_t>(p); }
  uintptr_t last() const { return first() + ((uintptr_t)(cols - 1) * (uintptr_t)ld + (uintptr_t)rows) * (uintptr_t)size; }
};
inline bool overlap(const Range& a, const Range& b) {
  if (!a.p || !b.p || a.rows <= 0 || a.cols <= 0 || b.rows <= 0 || b.cols <= 0) return false;
  if (a.first() >= b.last() || b.first() >= a.last()) return false;
  if (a.ld == b.ld && a.size == b.size) {
    // two row ranges of one larger matrix: b's columns start `r` rows below a's, and both end before the column does
    const Range& lo = a.first() <= b.first() ? a : b;
    const Range& hi = a.first() <= b.first() ? b : a;
    const uintptr_t d = hi.first() - lo.first();
    const uintptr_t r = d / (uintptr_t)a.size % (uintptr_t)a.ld;
    if (d % (uintptr_t)a.size == 0 && r >= (uintptr_t)lo.rows && r + (uintptr_t)hi.rows <= (uintptr_t)a.ld) return false;
  }
  return true;
}
inline Range bytes_at(const void* p, long bytes) { return Range{p, bytes, bytes, 1, 1}; }
// the same matrix, element for element, or no byte in common
inline bool same_or_apart(const Range& a, const Range& b) {
  return (a.p == b.p && (a.ld == b.ld || a.cols == 1) && a.size == b.size) || !overlap(a, b);
}

// gemm_mfma.hip: the fp32 / fp64 product alone on the device, all under the tile GEMM's built-in constants, so that neither a
// database that is loaded later nor the environment changes a plan.  Its predicted time and the slices it needs, its operands
// readable to m_read rows and n_read columns,
double product_alone_us(int elem_size, char ta, char tb, long M, long N, long K, long m_read, long n_read, long ws_bytes);
long product_alone_slices_bytes(int elem_size, char ta, char tb, long M, long N, long K, long m_read, long n_read);
// the product itself,
int product_alone_f32(char ta, char tb, long M, long N, long K, float alpha, const void* A, long lda, const void* B, long ldb, float beta, void* C, long ldc, void* ws,
                      long ws_bytes, long m_read, long n_read, hipStream_t stream);
int product_alone_f64(char ta, char tb, long M, long N, long K, double alpha, const void* A, long lda, const void* B, long ldb, double beta, void* C, long ldc, void* ws,
                      long ws_bytes, long m_read, long n_read, hipStream_t stream);
// or its slices that are still to be added.
int product_slices_f32(char ta, char tb, long M, long N, long K, const void* A, long lda, const void* B, long ldb, void* ws, long ws_bytes, long m_read, long n_read, bool add,
                       int* slices, hipStream_t stream);
int product_slices_f64(char ta, char tb, long M, long N, long K, const void* A, long lda, const void* B, long ldb, void* ws, long ws_bytes, long m_read, long n_read, bool add,
                       int* slices, hipStream_t stream);

// epilogue.hip
int bias_fold(int type, long M, long rows, const void* partial, void* dbias, hipStream_t stream);
long epilogue_pass_rows(int type, long M, long N);
int epilogue_pass(int type, int type_d, bool grad, long M, long N, const void* P, long ldP, long slice, int slices, const Epilogue& ep, hipStream_t stream);

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
  bool padded;           // 16-bit operands with whole panels of k, whose rows may be read to a multiple of 64 elements
  void* dbias;
  void* workspace; long workspace_bytes;
  hipStream_t stream;
};

inline long whole(long n, long unit) { return (n + unit - 1) / unit * unit; }

constexpr int H_BK = 64;   // panel depth of the 16-bit product

// How a 16-bit product is launched: macro tile, and how many ways K is split so that few tiles still fill the chip.  A
// function of the shape alone (the workspace is sized with it).  The times (microseconds) are fits to products of 256, 512
// and more workgroups at K = 512 .. 8192: a round of 256 x 256 tiles, one per compute unit, 10 + 0.0222 K (1511 TFLOP/s
// but for its ends); of 128 x 128 tiles, two per unit, 5 + 0.0136 K, or with one per unit 3.5 + 0.0069 K; a call 4.  Slices go
// out in 32 bits and come back through a pass at about 4 TB/s, a launch of its own.
struct HalfPlan { int tile, splits, kchunk; };   // tile 0: rows of fewer than 8 elements
// Those: a thread per element of the product, so a long K is split until the threads fill the device; a slice of kc costs
// its thread a wait per eight k, and the pass one per four slices, which are least together at kc near sqrt(2 K).
inline HalfPlan plan_thin(long M, long N, long K) {
  const long threads = 1L << 19, most = threads / (M * N > 0 ? M * N : 1);
  long kc = (long)std::sqrt(2.0 * (double)K);
  if (kc < 64) kc = 64;
  if (most > 0 && kc < K / most) kc = K / most;
  kc = whole(kc, 8);
  const long s = (K + kc - 1) / kc;
  return most < 2 || s < 2 ? HalfPlan{0, 1, 0} : HalfPlan{0, (int)s, (int)kc};
}
inline double half_rounds_us(int tile, long blocks, double k) {
  if (tile == 256) return (double)((blocks + 255) / 256) * (10.0 + 0.0222 * k);
  const long rem = blocks % 512;
  return (double)(blocks / 512) * (5.0 + 0.0136 * k) + (rem == 0 ? 0.0 : rem <= 256 ? 3.5 + 0.0069 * k : 5.0 + 0.0136 * k);
}
inline HalfPlan plan_half(bool at, bool bt, long M, long N, long K) {
  if ((at ? K : M) < 8 || (bt ? N : K) < 8) return plan_thin(M, N, K);
  HalfPlan best = {128, 1, 0};
  double best_us = 1e30;
  const unsigned k = (unsigned)K;
  const double cells = (double)M * (double)N;
  for (const int tile : {128, 256}) {
    const long tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
    for (const unsigned s : {1u, 2u, 3u, 4u, 5u, 6u, 8u, 10u, 12u, 16u, 20u, 24u, 32u}) {
      unsigned kc = k;
      if (s > 1) {
        kc = ((k + s - 1) / s + H_BK - 1) / H_BK * H_BK;
        if (kc < 2 * H_BK || 4.0 * s * cells > (double)(256L << 20) || tiles * s > 2048) break;
        if ((k + kc - 1) / kc != s) continue;
      }
      double us = 4.0 + half_rounds_us(tile, tiles * s, (double)kc);
      if (s > 1) us += 4.0 + (4.0 * s + 4.0) * cells / 4e6;
      if (us < best_us * (s > 1 ? 0.95 : 1.0)) best_us = us, best = {tile, (int)s, s > 1 ? (int)kc : 0};
    }
  }
  return best;
}

// rows of partial bias gradients the 16-bit product leaves: two per tile column, or those of the pass
inline long half_partial_rows(const HalfPlan& p, int type, long M, long N) {
  return p.splits > 1 || p.tile == 0 ? epilogue_pass_rows(type, M, N) : 2 * ((N + p.tile - 1) / p.tile);
}

// Space of the aligned copies of both operands, and their leading dimensions.
struct Copies { long ld_a, bytes_a, ld_b, bytes_b; long bytes() const { return bytes_a + bytes_b; } };

// fp32 and fp64 operands that are unaligned or ragged are multiplied from copies where that pays: their tile GEMM takes
// panels straight into LDS only from 16-byte aligned vectors and only in whole tiles and panels.  From aligned copies with k
// filled up by zeros to whole panels and rows to whole tiles of 256, an unaligned product runs at nearly the full rate
// (3878 x 1869 x 4113 with odd strides, fp32 TN / NN / NT / TT: 970 / 900 / 781 / 900 -> 512 - 552 / 510 / 509 / 508 us, fp64
// 1092 - 1190 -> 1030), and one of aligned operands with ragged edges loses less (3880 x 1872 x 4112: fp32 551 - 598 -> 504,
// fp64 1076 - 1130 -> 1000 - 1010).  Products that fill less of the device lose less; below the copies' own time there are
// none.  The space is set aside for whole extents too: their rows may be those of a wider matrix.
constexpr long WIDE_ROWS = 256, WIDE_K = 32;
inline bool wide_aligned(int es, const void* A, long lda, const void* B, long ldb) {
  return aligned_to(A, 16) && aligned_to(B, 16) && lda % (16 / es) == 0 && ldb % (16 / es) == 0;
}
inline double wide_copy_us(int es, long kw, long mw, long nw) { return 10.0 + (double)es * (double)kw * (double)(2 * mw + 2 * nw) / 3e6; }
inline Copies wide_copies(int es, bool aligned, bool at, bool bt, long M, long N, long K) {
  Copies c = {0, 0, 0, 0};
  if (K <= 0 || M > (1L << 28) || N > (1L << 28) || K > (1L << 28)) return c;
  const bool ragged = M % 128 != 0 || N % 128 != 0 || K % WIDE_K != 0;
  const double product_us = 2.0 * (double)M * (double)N * (double)K / (es == 4 ? 138e6 : 72e6);
  const double gain = !aligned ? (es == 4 ? 0.6 : 0.25) : ragged ? (es == 4 ? 0.15 : 0.1) : 0.0;
  const long kw = whole(K, WIDE_K), mw = whole(M, WIDE_ROWS), nw = whole(N, WIDE_ROWS);
  if (gain * product_us < wide_copy_us(es, kw, mw, nw)) return c;
  c.ld_a = at ? kw : mw;
  c.ld_b = bt ? nw : kw;
  c.bytes_a = (at ? mw : kw) * c.ld_a * es;
  c.bytes_b = (bt ? kw : nw) * c.ld_b * es;
  return c;
}

// How an fp32 or fp64 product is launched: in the tile GEMM's tiles with the epilogue as a pass (splits 0), or in 64 x 64 tiles
// with the epilogue inside, K split `splits` ways where it is long.  A function of the shape and the type alone.  Times in
// microseconds, fitted to 216 products of 64 x 64 x 64 to 8192 x 2048 x 2048: a 64 x 64 tile alone on its unit takes 0.053
// (fp32 0.032) per k, several on one 0.039 (0.0245) each, and 1 (0.5) for its epilogue; a pass over slices 3, and for each
// slice 0.8 and its bytes at 5.7 TB/s (the memory-side cache holds them).  The rule's choices are 1 % from the best of all
// measured ones, the tile GEMM's 24 %.  The tile GEMM is priced as the call would run it: from copies, where it makes them
// (priced by its rate on unaligned operands, large fp32 products of odd extents went to 64 x 64 tiles, up to 1.5 x behind;
// over 187 odd and ragged shapes both ways the choices are now 0.7 % from the better one, at worst 1.16 x).
// Both sides, fp64 / fp32, tile GEMM -> 64 x 64: 605 x 195 x 174 38 / 30 -> 16 / 11, 9472 x 192 x 3 21 / 17 -> 11 / 8,
// 10474 x 17 x 2943 170 / 105 -> 99 / 66; 2048 x 2048 x 512 79 / 44 -> 87 / 54, 2048^3 256 / 133 -> 318 / 192.
// Odd extents, copies / 64 x 64, fp32: 3878 x 1869 x 4113 506 - 552 / 699 - 776, 829 x 10936 x 2184 NT 378 / 502,
// 2253 x 1029 x 2616 132 / 180; 1501 x 1301 x 2003 103 / 99, 320 x 2293 x 1536 46 / 41.
struct WidePlan { int splits, kchunk; };
inline WidePlan plan_wide(int es, bool at, bool bt, long M, long N, long K) {
  if (M > (1L << 27) || N > (1L << 27) || K > (1L << 30)) return {0, 0};
  const double cells_us = (double)M * (double)N * es / 4e6, lone = es == 8 ? 0.053 : 0.032, shared = es == 8 ? 0.039 : 0.0245;
  const long tiles = ((M + 63) / 64) * ((N + 63) / 64);
  const int k = (int)K, gran = 128 / es;
  WidePlan best = {1, 0};
  double best_us = 1e30;
  for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    int kc = k;
    if (s > 1) {
      kc = ((k + s - 1) / s + gran - 1) / gran * gran;
      if (kc < 2 * gran || s * cells_us > 64.0) break;
      if ((k + kc - 1) / kc != s) continue;
    }
    const double per_unit = (double)((tiles * s + 255) / 256);
    double us = 5.5 + (lone > per_unit * shared ? lone : per_unit * shared) * kc + per_unit * (0.125 * es) + 0.5 * cells_us;
    if (s > 1) us += 3.0 + (0.8 + 0.7 * cells_us) * s;
    if (us < best_us) best_us = us, best = {s, s > 1 ? kc : 0};
  }
  if (best_us < 10.0 || K == 0) return best;   // (less than the tile GEMM's two launches ever take)
  // the tile GEMM as the call would run it: from copies, which are readable to the tiles' edges, where it makes them
  const char ta = at ? 'T' : 'N', tb = bt ? 'T' : 'N';
  const long per = 16 / es;
  const bool unaligned = (at ? K : M) % per != 0 || (bt ? N : K) % per != 0, ragged = M % 128 != 0 || N % 128 != 0 || K % 32 != 0;
  const long kw = whole(K, WIDE_K), mw = whole(M, WIDE_ROWS), nw = whole(N, WIDE_ROWS);
  const double gemm = wide_copies(es, !unaligned, at, bt, M, N, K).bytes() > 0
                          ? product_alone_us(es, ta, tb, M, N, kw, mw, nw, 1L << 28) + wide_copy_us(es, kw, mw, nw)
                          : product_alone_us(es, ta, tb, M, N, K, M, N, 1L << 28) * (unaligned ? (es == 4 ? 1.6 : 1.25) : ragged ? 1.1 : 1.0);
  return best_us < 0.95 * (2.0 + gemm + 2.0 * cells_us) ? best : WidePlan{0, 0};
}
int wide_product_f32(const Call& c, const WidePlan& plan, bool at, bool bt, const Epilogue& ep, void* slices);
int wide_product_f64(const Call& c, const WidePlan& plan, bool at, bool bt, const Epilogue& ep, void* slices);

// requests: 16-byte granules, and offsets from a panel's first element in 32 bits (256 rows of a K-major operand, 64 k-rows
// of an MN-major one)
inline bool in_offset_range(long lda, long ldb) { return lda < (1L << 22) && ldb < (1L << 22); }
inline bool can_request(const void* A, long lda, const void* B, long ldb) {
  return aligned_to(A, 16) && aligned_to(B, 16) && lda % 8 == 0 && ldb % 8 == 0 && in_offset_range(lda, ldb);
}

// Operands that cannot be requested are multiplied from aligned copies where that pays: a panel of unaligned 16-byte loads
// takes a compute unit 0.7 - 1.1 us longer than a requested one (misaligned lanes are served one by one), each operand's
// panels are loaded by every tile in its row or column, and the copies cost one launch and one pass over the operands
// (4100 x 1023 x 2052, rows of an odd number of elements: 70 -> 47 us).  The space is set aside by the shape alone: where a
// contiguous extent is no multiple of 8, so that dense operands could not be aligned.
inline Copies half_copies(bool at, bool bt, long M, long N, long K) {
  const long ext_a = at ? K : M, rows_a = at ? M : K, ext_b = bt ? N : K, rows_b = bt ? K : N;
  Copies c = {0, 0, 0, 0};
  if ((ext_a % 8 == 0 && ext_b % 8 == 0) || ext_a < 8 || ext_b < 8 || K > (1L << 30)) return c;
  const double tiles = (double)((M + 127) / 128) * (double)((N + 127) / 128);
  const double slow_us = 0.8 * (double)(K / H_BK) * (tiles > 256.0 ? tiles / 256.0 : 1.0), copy_us = 6.0 + 4.0 * (double)K * (double)(M + N) / 3e6;
  if (slow_us < copy_us) return c;
  // rows in whole cache lines, and k filled up with zeros to whole panels in either layout
  c.ld_a = whole(ext_a, H_BK);
  c.ld_b = whole(ext_b, H_BK);
  c.bytes_a = (at ? rows_a : whole(rows_a, H_BK)) * c.ld_a * 2;
  c.bytes_b = (bt ? whole(rows_b, H_BK) : rows_b) * c.ld_b * 2;
  return c;
}

int copy_operands(int es, const void* A, long lda, void* copy_a, const void* B, long ldb, void* copy_b, const Call& c, bool at, bool bt, const Copies& to);

// few columns of two K-major operands that can be requested, in whole panels of k: a kernel of their own
constexpr int FEW_MAX_N = 32;
inline bool few_columns(const Call& c, bool at, bool bt) {
  return at && !bt && !c.grad && c.N <= FEW_MAX_N && c.K > 0 && c.K % H_BK == 0 && can_request(c.A, c.lda, c.B, c.ldb);
}

// The 16-bit product, one source per operand type and kind: D of the operands' type, D in fp32 (and the fp32 slices of a
// split or thin product), the gradient.
#define PLK_HALF(T)                                                                                              \
  int half_forward_##T(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep);               \
  int half_wide_##T(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep);                  \
  int half_slices_##T(const Call& c, const HalfPlan& plan, bool at, bool bt, void* slices);                      \
  int half_gradient_##T(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep);
PLK_HALF(bf16)
PLK_HALF(f16)
#undef PLK_HALF

}  // namespace plk
#endif
