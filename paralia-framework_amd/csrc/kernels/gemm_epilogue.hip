// Matrix product with a fused epilogue for gfx950 (MI355X), column-major:
//   pl_gemm_epilogue        D = act(alpha * op(A) * op(B) + bias) + beta * C         (linear layer, weight gradient)
//   pl_gemm_epilogue_grad   D = (alpha * op(A) * op(B) + beta * C) .* act'(Z), dbias (gradient through an activation)
// 16-bit operands (bf16, fp16) run the kernels of half_product.h; fp32 and fp64 operands the library's tile GEMM
// (gemm_mfma.hip) with the epilogue as one pass over its product, small ones the kernel of wide_product.h.
#include "kernels/epilogue.h"
#include "kernels/linear.h"

namespace plk {

// The workspace of one call, in the order it is laid out: the product or its slices, the partial bias gradients, aligned copies of the operands.
struct Workspace { long product, partial, copies; long bytes() const { return product + partial + copies; } };
inline long round16(long b) { return (b + 15) & ~15L; }
inline Workspace workspace_for(int type, const HalfPlan& p, const WidePlan& wp, const Copies& copies, bool at, bool bt, long M, long N, long K, bool dbias) {
  Workspace w = {0, 0, 0};
  const long wide = type == PL_TYPE_F64 ? 8 : 4;
  if (type_size(type) == 2) {
    if (p.splits > 1 || p.tile == 0) w.product = round16((long)p.splits * M * N * 4);
    if (dbias) {
      // the small tile's, which unaligned operands are given to, or the pass's: the larger, because a product that turns
      // out to be empty (alpha = 0) is not split
      const long tile_rows = half_partial_rows({128, 1, 0}, type, M, N), pass_rows = half_partial_rows({0, 1, 0}, type, M, N);
      w.partial = round16((tile_rows > pass_rows ? tile_rows : pass_rows) * M * wide);
    }
  } else if (wp.splits > 0) {
    if (wp.splits > 1) w.product = round16((long)wp.splits * M * N * wide);
    const long tile_rows = (N + 63) / 64, pass_rows = epilogue_pass_rows(type, M, N);   // (the larger, as above)
    if (dbias) w.partial = round16((tile_rows > pass_rows ? tile_rows : pass_rows) * M * wide);
  } else {
    // the slices of a product alone on the device, or the product and behind it the slices of its tail; of the operands and
    // of their copies, whichever the call will be given
    const char ta = at ? 'T' : 'N', tb = bt ? 'T' : 'N';
    long slices = product_alone_slices_bytes((int)wide, ta, tb, M, N, K, M, N);
    if (copies.bytes() > 0) {
      const long padded = product_alone_slices_bytes((int)wide, ta, tb, M, N, whole(K, WIDE_K), whole(M, WIDE_ROWS), whole(N, WIDE_ROWS));
      if (padded > slices) slices = padded;
    }
    w.product = round16(M * N * wide) + round16(slices);
    if (dbias) w.partial = round16(epilogue_pass_rows(type, M, N) * M * wide);
  }
  w.copies = copies.bytes();
  return w;
}

// blockIdx.y: which operand.  `rows` rows of `extent` pairs of bytes into `rows_to` rows of ld_to, zeros behind them.
struct CopyJob { const short* from; short* to; long ld, ld_to, rows, rows_to; int extent; };
__global__ __launch_bounds__(256) void copy_kernel(CopyJob a, CopyJob b) {
  const CopyJob j = blockIdx.y == 0 ? a : b;
  const long per_row = j.ld_to / 8, total = per_row * j.rows_to;
  typedef Loose<short>::vec vec;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = i / per_row;
    const int at = (int)(i - row * per_row) * 8, left = row < j.rows ? j.extent - at : 0;
    const short* const p = j.from + row * j.ld + at;
    vec v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (left >= 8) {
      v = *reinterpret_cast<const Loose<short>::type*>(p);
    } else if (left > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[e < left ? e : left - 1];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? v[e] : (short)0;
    }
    *reinterpret_cast<vec*>(j.to + row * j.ld_to + at) = v;
  }
}
int copy_operands(int es, const void* A, long lda, void* copy_a, const void* B, long ldb, void* copy_b, const Call& c, bool at, bool bt, const Copies& to) {
  const long u = es / 2;
  const CopyJob a = {(const short*)A, (short*)copy_a, lda * u, to.ld_a * u, at ? c.M : c.K, to.bytes_a / (es * to.ld_a), (int)((at ? c.K : c.M) * u)};
  const CopyJob b = {(const short*)B, (short*)copy_b, ldb * u, to.ld_b * u, bt ? c.K : c.N, to.bytes_b / (es * to.ld_b), (int)((bt ? c.N : c.K) * u)};
  const long most = (to.bytes_a > to.bytes_b ? to.bytes_a : to.bytes_b) / 16;
  const long blocks = (most + 255) / 256;
  return launch(copy_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096), 2), dim3(256), c.stream, a, b);
}

bool plain_product(const Call& c) {
  return !c.grad && c.ep.act == PL_ACT_NONE && !c.ep.bias && !c.ep.preact && (c.ep.beta == 0.0 || c.ep.C == c.ep.D);
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
  if (c.dbias && M > (1L << 27)) return refuse(PL_ERR_DIM, who, "more than 2^27 rows with a bias gradient");
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
  const bool few = es == 2 && !empty && few_columns(c, at, bt);   // (a kernel that needs no workspace, and no plan)
  HalfPlan plan = {0, 1, 0};
  WidePlan tiles = {0, 0};
  Copies copies = {0, 0, 0, 0};
  Workspace w = {0, 0, 0};
  if (!few) {
    if (es == 2) plan = plan_half(at, bt, M, N, K), copies = half_copies(at, bt, M, N, K);
    else if (tiles = plan_wide(es, at, bt, M, N, K); tiles.splits == 0) copies = wide_copies(es, false, at, bt, M, N, K);
    w = workspace_for(c.type, plan, tiles, copies, at, bt, M, N, K, c.dbias != nullptr);
  }
  if (w.bytes() > 0 && (!c.workspace || !aligned_to(c.workspace, 16) || c.workspace_bytes < w.bytes())) return refuse(PL_ERR_ARG, who, "workspace null, too small or not 16-byte aligned");
  const Range work = bytes_at(w.bytes() > 0 ? c.workspace : nullptr, w.bytes());
  for (const Range& r : {a, b, d, p, rc, z, bias, db})
    if (overlap(work, r)) return refuse(PL_ERR_ARG, who, "the workspace overlaps an operand");
  char* const ws = (char*)c.workspace;
  ep.alpha = empty ? 0.0 : c.alpha;
  ep.partial = c.dbias ? ws + w.product : nullptr;
  if (empty) c.K = 0;
  int rc_;
  long rows, m_read = M, n_read = N;
  const bool copied = es == 2 ? !can_request(c.A, c.lda, c.B, c.ldb) && in_offset_range(copies.ld_a, copies.ld_b)
                              : wide_copies(es, wide_aligned(es, c.A, c.lda, c.B, c.ldb), at, bt, M, N, K).bytes() > 0;
  if (!empty && copies.bytes() > 0 && copied) {
    char* const copy_a = ws + w.product + w.partial;
    rc_ = copy_operands(es, c.A, c.lda, copy_a, c.B, c.ldb, copy_a + copies.bytes_a, c, at, bt, copies);
    if (rc_ != PL_OK) return rc_;
    c.A = copy_a, c.lda = copies.ld_a;
    c.B = copy_a + copies.bytes_a, c.ldb = copies.ld_b;
    c.K = whole(K, es == 2 ? H_BK : WIDE_K);
    c.padded = true;
    m_read = whole(M, WIDE_ROWS), n_read = whole(N, WIDE_ROWS);
  }
  if (es == 2) {
    if (empty) plan.splits = 1, plan.kchunk = 0;
    if (plan.tile == 256 && !can_request(c.A, c.lda, c.B, c.ldb)) plan.tile = 128;
    rows = few ? 0 : half_partial_rows(plan, c.type, M, N);
    // (copies can be requested: few columns of them too, 4263 x 2 x 1387 19 -> 13 us)
    const bool f16 = c.type == PL_TYPE_F16, sliced = !few && (plan.tile == 0 || plan.splits > 1) && !(c.padded && few_columns(c, at, bt));
    if (sliced) {
      rc_ = f16 ? half_slices_f16(c, plan, at, bt, ws) : half_slices_bf16(c, plan, at, bt, ws);
      if (rc_ == PL_OK) rc_ = epilogue_pass(c.type, c.type_d, c.grad, M, N, ws, M, M * N, plan.splits, ep, c.stream);
    } else if (c.grad) {
      rc_ = f16 ? half_gradient_f16(c, plan, at, bt, ep) : half_gradient_bf16(c, plan, at, bt, ep);
    } else if (c.type_d == PL_TYPE_F32) {
      rc_ = f16 ? half_wide_f16(c, plan, at, bt, ep) : half_wide_bf16(c, plan, at, bt, ep);
    } else {
      rc_ = f16 ? half_forward_f16(c, plan, at, bt, ep) : half_forward_bf16(c, plan, at, bt, ep);
    }
  } else if (tiles.splits > 0) {
    if (empty) tiles.splits = 1;
    rows = tiles.splits > 1 ? epilogue_pass_rows(c.type, M, N) : (N + 63) / 64;
    rc_ = (es == 8 ? wide_product_f64 : wide_product_f32)(c, tiles, at, bt, ep, ws);
  } else {
    rows = epilogue_pass_rows(c.type, M, N);
    const bool f64 = c.type == PL_TYPE_F64;
    if (plain_product(c)) {
      // nothing but the product (and C where D is): the tile GEMM's own epilogue
      rc_ = f64 ? product_alone_f64(c.ta, c.tb, M, N, c.K, ep.alpha, c.A, c.lda, c.B, c.ldb, ep.beta, ep.D, ep.ldd, ws, w.product, m_read, n_read, c.stream)
                : product_alone_f32(c.ta, c.tb, M, N, c.K, (float)ep.alpha, c.A, c.lda, c.B, c.ldb, (float)ep.beta, ep.D, ep.ldd, ws, w.product, m_read, n_read, c.stream);
      return rc_ == PL_ERR_LAUNCH ? refuse(rc_, who, "kernel launch failed") : rc_;
    }
    int slices = 1;
    rc_ = (f64 ? product_slices_f64 : product_slices_f32)(c.ta, c.tb, M, N, c.K, c.A, c.lda, c.B, c.ldb, ws, w.product, m_read, n_read, f64 && c.grad, &slices, c.stream);
    if (rc_ == PL_ERR_LAUNCH) return refuse(rc_, who, "kernel launch failed");
    if (rc_ == PL_OK) rc_ = epilogue_pass(c.type, c.type_d, c.grad, M, N, ws, M, M * N, slices, ep, c.stream);
  }
  if (rc_ != PL_OK || !c.dbias) return rc_;
  return bias_fold(c.type, M, rows, ep.partial, c.dbias, c.stream);
}

}  // namespace plk

extern "C" long pl_gemm_epilogue_workspace_bytes(int type, char transA, char transB, long M, long N, long K, int with_dbias) {
  using namespace plk;
  if (!valid_type(type) || M <= 0 || N <= 0 || K < 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
  const bool at = transA == 'T' || transA == 't', bt = transB == 'T' || transB == 't';
  const int es = type_size(type);
  const HalfPlan plan = es == 2 ? plan_half(at, bt, M, N, K) : HalfPlan{0, 1, 0};
  const WidePlan tiles = es == 2 ? WidePlan{0, 0} : plan_wide(es, at, bt, M, N, K);
  const Copies copies = es == 2 ? half_copies(at, bt, M, N, K) : tiles.splits > 0 ? Copies{0, 0, 0, 0} : wide_copies(es, false, at, bt, M, N, K);
  return workspace_for(type, plan, tiles, copies, at, bt, M, N, K, with_dbias != 0).bytes();
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
