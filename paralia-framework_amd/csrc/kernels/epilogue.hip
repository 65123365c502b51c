// Streaming side of the linear-layer operators for gfx950 (MI355X): the epilogue as a pass over a product that is already
// in memory (the fp64 / fp32 products of the tile GEMM, and the split-K slices of the 16-bit GEMM), the gradient of bias
// and activation where the incoming gradient is an operand, and the fold of the partial bias gradients.
//
// Every element is read once and written once, so HBM bounds all of them.  64 lanes take 64 * VEC consecutive rows of a
// column (16 bytes a lane), the four waves of a workgroup take every fourth column of a range: whole cache lines per wave,
// several columns in flight, and the sums over the columns stay in registers until the end.
#include "kernels/epilogue.h"
#include "kernels/linear.h"

namespace plk {

constexpr int PASS_THREADS = 256;

// v(m, n) <- sum over slices of P(m, n), through the epilogue.  blockIdx.x: 64 * VEC rows, blockIdx.y: a range of `per`
// columns.  GRAD with ep.partial: row blockIdx.y of the partial sums.  (P is not __restrict__: it may be D, as C and Z may.)
template <typename TP, typename T, typename TD, bool GRAD, bool SLICES, int VEC>
__global__ __launch_bounds__(PASS_THREADS) void epilogue_pass_kernel(long M, long N, long per, const TP* P, long ldP, long slice, int slices,
                                                                    Epilogue ep) {
  using W = wide_t<T>;
  __shared__ W fold[GRAD ? 4 * 64 * VEC : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long m = ((long)blockIdx.x * 64 + lane) * VEC;
  const int valid = (int)(M - m < VEC ? (M - m < 0 ? 0 : M - m) : VEC);
  const long n0 = (long)blockIdx.y * per, n1 = n0 + per < N ? n0 + per : N;
  W bias[VEC], sums[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) bias[e] = sums[e] = W(0);
  if (valid > 0) {
    if (!GRAD && ep.bias) load_row<T, VEC, W>((const T*)ep.bias + m, bias, valid);
#pragma unroll(sizeof(T) == 8 ? 1 : 2)
    for (long n = n0 + wave; n < n1; n += 4) {
      EpilogueInputs<T, TD, GRAD, VEC> in;
      in.load(ep, (const TD*)ep.C + n * ep.ldc + m, (const T*)ep.Z + n * ep.ldz + m, valid);
      W v[VEC];
      load_row<TP, VEC, W>(P + n * ldP + m, v, valid);
      if constexpr (SLICES) {
#pragma unroll 4
        for (int s = 1; s < slices; ++s) {
          W x[VEC];
          load_row<TP, VEC, W>(P + s * slice + n * ldP + m, x, valid);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] += x[e];
        }
      }
      apply_epilogue<T, TD, GRAD, VEC>(ep, in, v, bias, (TD*)ep.D + n * ep.ldd + m, (T*)ep.preact + n * ep.ldp + m, valid, sums);
    }
  }
  if constexpr (GRAD) {
    if (ep.partial) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) fold[(wave * VEC + e) * 64 + lane] = sums[e];
      __syncthreads();
      if (wave == 0 && valid > 0) {
        W* const out = (W*)ep.partial + (long)blockIdx.y * M + m;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          W s = fold[e * 64 + lane];
          for (int w = 1; w < 4; ++w) s += fold[(w * VEC + e) * 64 + lane];
          if (e < valid) out[e] = s;
        }
      }
    }
  }
}

// dbias(m) <- sum of `rows` partial rows in their order; no rows: zero.  16 rows of 16 threads: thread (x, y) adds rows
// y, y + 16, ... of element x, then the 16 sums in order.
template <typename T>
__global__ __launch_bounds__(256) void bias_fold_kernel(long M, long rows, const wide_t<T>* __restrict__ partial, T* __restrict__ dbias) {
  using W = wide_t<T>;
  __shared__ W part[16][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  const long m = (long)blockIdx.x * 16 + x;
  W s = W(0);
  if (m < M)
    for (long r = y; r < rows; r += 16) s += partial[r * M + m];
  part[y][x] = s;
  __syncthreads();
  if (y == 0 && m < M) {
    for (int i = 1; i < 16; ++i) s += part[i][x];
    dbias[m] = (T)s;
  }
}

// rows of M handled per workgroup, by element type: 64 lanes of 16 bytes
template <typename T> constexpr int pass_vec() { return 16 / (int)sizeof(T); }

// How many column ranges the pass is cut into: enough workgroups to cover the 256 compute units eight times, at least
// eight columns (two per wave) in each.  A function of the shape alone: the order of the sums does not depend on anything else.
template <typename T> long pass_ranges(long M, long N) {
  const long rows = 64 * pass_vec<T>();
  const long gx = (M + rows - 1) / rows;
  long want = (2048 + gx - 1) / gx;
  const long most = (N + 7) / 8;
  if (want > most) want = most;
  if (want > 65535) want = 65535;
  return want < 1 ? 1 : want;
}

template <typename TP, typename T, typename TD, bool GRAD>
int launch_epilogue_pass(long M, long N, const TP* P, long ldP, long slice, int slices, const Epilogue& ep, hipStream_t stream) {
  constexpr int VEC = pass_vec<T>();
  const long ranges = pass_ranges<T>(M, N), per = (N + ranges - 1) / ranges;
  const dim3 grid((unsigned)((M + 64 * VEC - 1) / (64 * VEC)), (unsigned)((N + per - 1) / per));
#define LAUNCH(SLICES) \
  return launch(epilogue_pass_kernel<TP, T, TD, GRAD, SLICES, VEC>, grid, dim3(PASS_THREADS), stream, M, N, per, P, ldP, slice, slices, ep)
  // (a 16-bit operand is no slice of a product; the fp64 gradient has no scalar registers left for slices)
  if constexpr (sizeof(TP) == sizeof(wide_t<T>) && !(GRAD && sizeof(T) == 8)) {
    if (slices > 1) LAUNCH(true);
  }
  LAUNCH(false);
#undef LAUNCH
}

template <typename T> long pass_partial_rows(long M, long N) {
  const long ranges = pass_ranges<T>(M, N), per = (N + ranges - 1) / ranges;
  return (N + per - 1) / per;
}

template <typename T> int launch_bias_fold(long M, long rows, const void* partial, void* dbias, hipStream_t stream) {
  return launch(bias_fold_kernel<T>, dim3((unsigned)((M + 15) / 16)), dim3(256), stream, M, rows, (const wide_t<T>*)partial, (T*)dbias);
}

int bias_fold(int type, long M, long rows, const void* partial, void* dbias, hipStream_t stream) {
  switch (type) {
    case PL_TYPE_F64: return launch_bias_fold<double>(M, rows, partial, dbias, stream);
    case PL_TYPE_F32: return launch_bias_fold<float>(M, rows, partial, dbias, stream);
    case PL_TYPE_F16: return launch_bias_fold<f16_t>(M, rows, partial, dbias, stream);
    default: return launch_bias_fold<bf16_t>(M, rows, partial, dbias, stream);
  }
}

long epilogue_pass_rows(int type, long M, long N) {
  return type == PL_TYPE_F64 ? pass_partial_rows<double>(M, N) : type == PL_TYPE_F32 ? pass_partial_rows<float>(M, N) : pass_partial_rows<f16_t>(M, N);
}

// The product's own type is the wide type of the operands: fp64 and fp32 products, fp32 slices of 16-bit ones.
int epilogue_pass(int type, int type_d, bool grad, long M, long N, const void* P, long ldP, long slice, int slices, const Epilogue& ep, hipStream_t stream) {
#define PASS(TP, T, TD) \
  return grad ? launch_epilogue_pass<TP, T, TD, true>(M, N, (const TP*)P, ldP, slice, slices, ep, stream) \
              : launch_epilogue_pass<TP, T, TD, false>(M, N, (const TP*)P, ldP, slice, slices, ep, stream)
  if (type == PL_TYPE_F64) PASS(double, double, double);
  if (type == PL_TYPE_F32) PASS(float, float, float);
  if (type == PL_TYPE_F16) { if (type_d == PL_TYPE_F32) PASS(float, f16_t, float); PASS(float, f16_t, f16_t); }
  if (type_d == PL_TYPE_F32) PASS(float, bf16_t, float);
  PASS(float, bf16_t, bf16_t);
#undef PASS
}

template <typename T>
int launch_act_grad(int type, int act, long M, long N, const void* dY, long lddy, const void* Z, long ldz, void* dZ, long lddz, void* dbias,
                    void* workspace, hipStream_t stream) {
  Epilogue ep = {};
  ep.alpha = 1.0;
  ep.act = act;
  ep.Z = Z; ep.ldz = ldz;
  ep.D = dZ; ep.ldd = lddz;
  ep.partial = dbias ? workspace : nullptr;
  const int rc = launch_epilogue_pass<T, T, T, true>(M, N, (const T*)dY, lddy, 0, 1, ep, stream);
  if (rc != PL_OK || !dbias) return rc;
  return bias_fold(type, M, pass_partial_rows<T>(M, N), workspace, dbias, stream);
}

}  // namespace plk

extern "C" long pl_bias_act_grad_workspace_bytes(int type, long M, long N) {
  if (!plk::valid_type(type) || M <= 0 || N <= 0 || M > (1L << 27) || N > INT32_MAX) return 0;
  return plk::epilogue_pass_rows(type, M, N) * M * (type == PL_TYPE_F64 ? 8 : 4);
}

extern "C" int pl_bias_act_grad(int type, int activation, long M, long N, const void* dY, long lddy, const void* Z, long ldz, void* dZ, long lddz,
                                void* dbias, void* workspace, long workspace_bytes, void* stream) {
  using namespace plk;
  const char* const who = "pl_bias_act_grad";
  if (!valid_type(type)) return refuse(PL_ERR_ARG, who, "unknown element type");
  if (!valid_act(activation)) return refuse(PL_ERR_ARG, who, "unknown activation");
  if (M < 0 || N < 0 || M > (1L << 27) || N > INT32_MAX) return refuse(PL_ERR_DIM, who, "dimension out of range");
  const bool need_z = activation != PL_ACT_NONE;
  if (lddy < (M > 1 ? M : 1) || (need_z && ldz < (M > 1 ? M : 1)) || (dZ && lddz < (M > 1 ? M : 1))) return refuse(PL_ERR_LD, who, "leading dimension below M");
  if (M == 0) return PL_OK;
  hipStream_t s = (hipStream_t)stream;
  if (N == 0) return dbias ? bias_fold(type, M, 0, nullptr, dbias, s) : PL_OK;
  if (!dY || (need_z && !Z) || (!dZ && !dbias)) return refuse(PL_ERR_NULL, who, "null operand");
  const int es = type_size(type);
  if (!aligned_to(dY, es) || !aligned_to(Z, es) || !aligned_to(dZ, es) || !aligned_to(dbias, es)) return refuse(PL_ERR_ARG, who, "operand not aligned to its element size");
  if (dbias) {
    if (!workspace) return refuse(PL_ERR_NULL, who, "the bias gradient needs a workspace");
    if (!aligned_to(workspace, 16) || workspace_bytes < pl_bias_act_grad_workspace_bytes(type, M, N)) return refuse(PL_ERR_ARG, who, "workspace too small or not 16-byte aligned");
  }
  // dZ may be dY or Z itself (an element is read before it is written, by the same thread), but not a shifted view of them
  const Range dz = {dZ, lddz, M, N, es};
  if (dZ) {
    if (!same_or_apart(dz, Range{dY, lddy, M, N, es}) || (need_z && !same_or_apart(dz, Range{Z, ldz, M, N, es}))) return refuse(PL_ERR_ARG, who, "dZ overlaps an operand it is not");
    if (dbias && overlap(dz, Range{dbias, M, M, 1, es})) return refuse(PL_ERR_ARG, who, "dZ overlaps dbias");
  }
  if (dbias) {
    const Range dy = {dY, lddy, M, N, es}, z = {need_z ? Z : nullptr, ldz, M, N, es}, db = {dbias, M, M, 1, es}, work = bytes_at(workspace, pl_bias_act_grad_workspace_bytes(type, M, N));
    if (overlap(db, dy) || overlap(db, z)) return refuse(PL_ERR_ARG, who, "dbias overlaps an operand");
    if (overlap(work, dy) || overlap(work, z) || overlap(work, dz) || overlap(work, db)) return refuse(PL_ERR_ARG, who, "the workspace overlaps an operand");
  }
  switch (type) {
    case PL_TYPE_F64: return launch_act_grad<double>(type, activation, M, N, dY, lddy, Z, ldz, dZ, lddz, dbias, workspace, s);
    case PL_TYPE_F32: return launch_act_grad<float>(type, activation, M, N, dY, lddy, Z, ldz, dZ, lddz, dbias, workspace, s);
    case PL_TYPE_F16: return launch_act_grad<f16_t>(type, activation, M, N, dY, lddy, Z, ldz, dZ, lddz, dbias, workspace, s);
    default: return launch_act_grad<bf16_t>(type, activation, M, N, dY, lddy, Z, ldz, dZ, lddz, dbias, workspace, s);
  }
}
