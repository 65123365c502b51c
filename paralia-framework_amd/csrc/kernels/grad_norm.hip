// Global gradient norm and clipping over a list of tensors for gfx950 (MI355X):
//   norm = sqrt(sum over all tensors and elements of g^2),   out = g * min(1, max_norm / (norm + eps)).
//
// HBM bounds both passes: the norm reads every element once, the scaling reads and writes it once.  The tensors are cut
// into chunks of CHUNK elements that never span two tensors, and a fixed number of workgroups walks all chunks of up to
// LIST_MAX tensors in one launch, so that many small tensors cost two launches for each 128 of them and a large one is
// spread over the chip.  Pointers and counts travel in the kernel's arguments: no table in device memory to keep, to copy
// or to go stale, and a captured launch holds its own.
//
// Squares are formed and added in 64 bits (a 32-bit square of a 32-bit gradient below 1e-23 or above 1e19 is lost; the
// conversion and the 64-bit fma run at several times the rate at which memory delivers elements).  The order of the sum
// is a function of the list's sizes alone: each workgroup's chunks in order, lanes by a shuffle tree, then the workgroups'
// partial sums in order.
#include "kernels/epilogue.h"
#include "kernels/linear.h"

#include <algorithm>
#include <new>
#include <vector>

namespace plk {

constexpr int NORM_THREADS = 256;
constexpr int CHUNK = 8192;          // elements: 16 - 64 KiB, four steps of eight elements a thread
constexpr int LIST_MAX = 128;        // tensors per launch: two per lane, 28 bytes each in the kernel's arguments
constexpr int NORM_BLOCKS = 2048;    // workgroups of one launch at most (eight per compute unit), and its partial sums

struct TensorList {
  const void* src[LIST_MAX];
  void* dst[LIST_MAX];
  long long count_type[LIST_MAX];    // element count * 4 + type
  unsigned first[LIST_MAX + 1];      // the list's chunk at which each tensor starts; then the number of chunks
  int n;
};
static_assert(sizeof(TensorList) <= 4096 - 64, "the list and what goes with it are kernel arguments");

// The list in registers: lane l holds tensors l and l + 64, fetched all at once (a search through the kernel's arguments is
// seven dependent fetches, 3 us of a small call).  The tensor of a chunk is the number of tensors that start at or before
// it; what the list says of it then comes out of that lane.
struct ListLanes {
  unsigned long long src[2], dst[2], count_type[2];
  unsigned first[2];
  __device__ __forceinline__ explicit ListLanes(const TensorList& list, bool with_dst) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = (int)(threadIdx.x & 63) + 64 * h, j = i < list.n ? i : list.n - 1;
      first[h] = i < list.n ? list.first[j] : 0xffffffffu;
      src[h] = (unsigned long long)list.src[j];
      dst[h] = with_dst ? (unsigned long long)list.dst[j] : 0;
      count_type[h] = (unsigned long long)list.count_type[j];
    }
  }
  static __device__ __forceinline__ unsigned pick(unsigned v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
  static __device__ __forceinline__ unsigned long long pick(unsigned long long v, int lane) {
    return ((unsigned long long)pick((unsigned)(v >> 32), lane) << 32) | pick((unsigned)v, lane);
  }
  struct Chunk { const void* src; void* dst; long long at; int count, type; };
  __device__ __forceinline__ Chunk chunk(unsigned c) const {
    const int t = __popcll(__ballot(first[0] <= c)) + __popcll(__ballot(first[1] <= c)) - 1;
    const int h = t >> 6, lane = t & 63;
    const unsigned long long ct = pick(h ? count_type[1] : count_type[0], lane);
    const long long at = (long long)(c - pick(h ? first[1] : first[0], lane)) * CHUNK, left = (long long)(ct >> 2) - at;
    return {(const void*)pick(h ? src[1] : src[0], lane), (void*)pick(h ? dst[1] : dst[0], lane), at, left < CHUNK ? (int)left : CHUNK, (int)(ct & 3)};
  }
};

__device__ __forceinline__ double sum_block(double v) {
  __shared__ double part[NORM_THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < NORM_THREADS / 64; ++w) s += part[w];
  return s;                          // on every thread
}

template <typename T> __device__ __forceinline__ double chunk_squares(const T* __restrict__ p, int count) {
  double acc[2] = {0.0, 0.0};
#pragma unroll
  for (int i = 0; i < CHUNK / (8 * NORM_THREADS); ++i) {
    const int at = (i * NORM_THREADS + (int)threadIdx.x) * 8;
    const int valid = count - at;
    if (valid > 0) {
      wide_t<T> v[8];
      load_row<T, 8, wide_t<T>>(p + at, v, valid);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e & 1] = fma((double)v[e], (double)v[e], acc[e & 1]);
    }
  }
  return acc[0] + acc[1];
}

__global__ __launch_bounds__(NORM_THREADS) void grad_squares_kernel(TensorList list, double* __restrict__ partial) {
  const unsigned chunks = list.first[list.n];
  const ListLanes lanes(list, false);
  double acc = 0.0;
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const ListLanes::Chunk k = lanes.chunk(c);
    switch (k.type) {
      case PL_TYPE_F64: acc += chunk_squares((const double*)k.src + k.at, k.count); break;
      case PL_TYPE_F32: acc += chunk_squares((const float*)k.src + k.at, k.count); break;
      case PL_TYPE_F16: acc += chunk_squares((const f16_t*)k.src + k.at, k.count); break;
      default: acc += chunk_squares((const bf16_t*)k.src + k.at, k.count); break;
    }
  }
  acc = sum_block(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__device__ __forceinline__ double fold_norm(const double* __restrict__ partial, int partials) {
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < partials; i += NORM_THREADS) s += partial[i];
  return sqrt(sum_block(s));
}

__global__ __launch_bounds__(NORM_THREADS) void grad_norm_kernel(const double* __restrict__ partial, int partials, double* __restrict__ norm) {
  const double r = fold_norm(partial, partials);
  if (threadIdx.x == 0) *norm = r;
}

// The factor is rounded to 32 bits for elements of 32 and 16 (half a unit of 2^-24 that the element's own rounding joins),
// but where it is below their normal numbers, and would lose bits or vanish, the product is formed in 64.
template <typename T> __device__ __forceinline__ void chunk_scale(const T* p, T* q, int count, double scale) {
  const wide_t<T> f = (wide_t<T>)scale;
  const bool tiny = sizeof(wide_t<T>) == 4 && scale < 0x1p-126;
#pragma unroll
  for (int i = 0; i < CHUNK / (8 * NORM_THREADS); ++i) {
    const int at = (i * NORM_THREADS + (int)threadIdx.x) * 8;
    const int valid = count - at;
    if (valid > 0) {
      wide_t<T> v[8];
      load_row<T, 8, wide_t<T>, true>(p + at, v, valid);
      if (tiny) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (wide_t<T>)((double)v[e] * scale);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= f;
      }
      store_row<T, 8, wide_t<T>>(q + at, v, valid);
    }
  }
}

// partials > 0: every workgroup folds the partial sums of the norm's launches itself, in the same order (at most 16 KiB out
// of the L2, against a launch of its own), and workgroup 0 of the first launch stores the norm.  partials == 0: *norm is
// given, or folded already: with more partial sums than one launch leaves, every workgroup of every launch would read all
// of them again, work that grows with the square of the list (bf16 tensors of 100 k elements, folded everywhere / once: 1000
// of them 240 / 162 us, 5000 2719 / 858; 300 of 70 k 52 / 51).
// A factor of exactly 1 leaves tensors that are scaled in place as they are.
__global__ __launch_bounds__(NORM_THREADS) void grad_scale_kernel(TensorList list, const double* __restrict__ partial, int partials, int store, double max_norm,
                                                                 double eps, double* norm) {
  const ListLanes lanes(list, true);
  const unsigned chunks = list.first[list.n];
  const double total = partials > 0 ? fold_norm(partial, partials) : *norm;
  if (partials > 0 && store && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const double ratio = max_norm / (total + eps);
  const double scale = ratio > 1.0 ? 1.0 : ratio;   // (a NaN stays a NaN)
  // last chunk first: what the norm read last is what the caches still hold
  for (unsigned r = blockIdx.x; r < chunks; r += gridDim.x) {
    const ListLanes::Chunk k = lanes.chunk(chunks - 1 - r);
    if (scale == 1.0 && k.src == k.dst) continue;
    switch (k.type) {
      case PL_TYPE_F64: chunk_scale((const double*)k.src + k.at, (double*)k.dst + k.at, k.count, scale); break;
      case PL_TYPE_F32: chunk_scale((const float*)k.src + k.at, (float*)k.dst + k.at, k.count, scale); break;
      case PL_TYPE_F16: chunk_scale((const f16_t*)k.src + k.at, (f16_t*)k.dst + k.at, k.count, scale); break;
      default: chunk_scale((const bf16_t*)k.src + k.at, (bf16_t*)k.dst + k.at, k.count, scale); break;
    }
  }
}

struct Span { uintptr_t first, last; };
inline Span span_of(const void* p, long long count, int type) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return {a, a + (uintptr_t)count * (uintptr_t)type_size(type)};
}

// Refuses what the kernels cannot take: they would scale a tensor that is listed twice twice, or read one tensor's
// gradients after writing another's.
int check_list(const char* who, long n, const void* const* src, const long long* counts, const int* types, void* const* dst, const double* norm, const void* workspace,
               long workspace_bytes) {
  if (n < 0 || n > (1L << 20)) return refuse(PL_ERR_DIM, who, "tensor count out of range");
  if (n == 0) return PL_OK;
  if (!src || !counts || !types) return refuse(PL_ERR_NULL, who, "null list");
  for (long i = 0; i < n; ++i) {
    if (!valid_type(types[i])) return refuse(PL_ERR_ARG, who, "unknown element type");
    if (counts[i] < 0 || counts[i] > (1LL << 37)) return refuse(PL_ERR_DIM, who, "element count out of range");
    if (counts[i] == 0) continue;
    if (!src[i] || (dst && !dst[i])) return refuse(PL_ERR_NULL, who, "null tensor");
    if (!aligned_to(src[i], type_size(types[i])) || (dst && !aligned_to(dst[i], type_size(types[i])))) return refuse(PL_ERR_ARG, who, "tensor not aligned to its element size");
    for (const void* p : {src[i], dst ? (const void*)dst[i] : nullptr}) {
      if (!p) continue;
      const Range t = bytes_at(p, (long)counts[i] * type_size(types[i]));
      if (overlap(t, bytes_at(norm, 8)) || overlap(t, bytes_at(workspace, workspace_bytes))) return refuse(PL_ERR_ARG, who, "norm or workspace overlaps a tensor");
    }
  }
  if (!dst) return PL_OK;
  // (lists of up to 256 tensors on the stack: two allocations are a microsecond of a small call)
  Span few_out[256], few_in[256];
  std::vector<Span> many;
  Span* out = few_out;
  Span* in = few_in;
  if (n > 256) many.resize(2 * n), out = many.data(), in = out + n;
  long outs = 0, ins = 0;
  for (long i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    out[outs++] = span_of(dst[i], counts[i], types[i]);
    if (src[i] != dst[i]) in[ins++] = span_of(src[i], counts[i], types[i]);
  }
  auto by_first = [](const Span& a, const Span& b) { return a.first < b.first; };
  if (!std::is_sorted(out, out + outs, by_first)) std::sort(out, out + outs, by_first);
  for (long i = 1; i < outs; ++i)
    if (out[i].first < out[i - 1].last) return refuse(PL_ERR_ARG, who, "two tensors of the list are written to the same memory");
  // outputs are disjoint and in order: an input that is not its own output must lie between two of them
  for (long i = 0; i < ins; ++i) {
    const Span& s = in[i];
    const Span* const it = std::upper_bound(out, out + outs, s, by_first);
    if ((it != out + outs && it->first < s.last) || (it != out && (it - 1)->last > s.first)) return refuse(PL_ERR_ARG, who, "a tensor is written over another one of the list");
  }
  return PL_OK;
}

// Calls launch(list, blocks) for the list in pieces of LIST_MAX tensors (whose chunks, at most 2^24 of a tensor, are numbered
// in 32 bits).  Empty tensors are left out.
template <typename F> int for_each_piece(long n, const void* const* src, const long long* counts, const int* types, void* const* dst, F&& launch) {
  TensorList list;
  list.n = 0;
  list.first[0] = 0;
  auto flush = [&]() -> int {
    if (list.n == 0) return PL_OK;
    const unsigned chunks = list.first[list.n];
    const int rc = launch(list, (int)(chunks < NORM_BLOCKS ? chunks : NORM_BLOCKS));
    list.n = 0;
    return rc;
  };
  for (long i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    const long long chunks = (counts[i] + CHUNK - 1) / CHUNK;
    if (list.n == LIST_MAX) {
      const int rc = flush();
      if (rc != PL_OK) return rc;
    }
    list.src[list.n] = src[i];
    list.dst[list.n] = dst ? dst[i] : nullptr;
    list.count_type[list.n] = counts[i] * 4 + types[i];
    list.first[list.n + 1] = list.first[list.n] + (unsigned)chunks;
    ++list.n;
  }
  return flush();
}

// the norm's launches: partial sums into the workspace, *partials of them
int launch_squares(long n, const void* const* src, const long long* counts, const int* types, double* workspace, int* partials, hipStream_t stream) {
  int used = 0;
  const int rc = for_each_piece(n, src, counts, types, nullptr, [&](const TensorList& list, int blocks) {
    double* const to = workspace + used;
    used += blocks;
    return launch(grad_squares_kernel, dim3(blocks), dim3(NORM_THREADS), stream, list, to);
  });
  *partials = used;
  return rc;
}

int launch_scale(long n, const void* const* src, const long long* counts, const int* types, void* const* dst, double max_norm, double eps,
                 const double* workspace, int partials, double* norm, hipStream_t stream) {
  int first = 1;
  return for_each_piece(n, src, counts, types, dst, [&](const TensorList& list, int blocks) {
    const int store = first;
    first = 0;
    return launch(grad_scale_kernel, dim3(blocks), dim3(NORM_THREADS), stream, list, workspace, partials, store, max_norm, eps, norm);
  });
}

int check_norm_args(const char* who, long n, const double* norm, const void* workspace, long workspace_bytes) {
  if (!norm) return refuse(PL_ERR_NULL, who, "null norm");
  if (!aligned_to(norm, 8)) return refuse(PL_ERR_ARG, who, "norm not 8-byte aligned");
  if (n > 0 && (!workspace || !aligned_to(workspace, 16) || workspace_bytes < pl_grad_norm_workspace_bytes(n))) return refuse(PL_ERR_ARG, who, "workspace null, too small or not 16-byte aligned");
  // the first workgroup of the scaling stores the norm while others still read the partial sums
  if (n > 0 && overlap(bytes_at(norm, 8), bytes_at(workspace, pl_grad_norm_workspace_bytes(n)))) return refuse(PL_ERR_ARG, who, "norm overlaps the workspace");
  return PL_OK;
}
bool valid_limit(double max_norm, double eps) { return max_norm >= 0.0 && eps >= 0.0 && eps < 1e300; }

int grad_norm_only(long n, const void* const* src, const long long* counts, const int* types, double* norm, double* workspace, hipStream_t s) {
  int partials = 0;
  const int rc = launch_squares(n, src, counts, types, workspace, &partials, s);
  if (rc != PL_OK) return rc;
  return launch(grad_norm_kernel, dim3(1), dim3(NORM_THREADS), s, workspace, partials, norm);
}

// no exception leaves a C entry: the checks' lists are the only thing that allocates
template <typename F> int without_exceptions(const char* who, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return refuse(PL_ERR_NOMEM, who, "out of host memory");
  } catch (...) {
    return refuse(PL_ERR_ARG, who, "unexpected exception");
  }
}

}  // namespace plk

extern "C" long pl_grad_norm_workspace_bytes(long n) {
  if (n <= 0 || n > (1L << 20)) return 0;
  return n * (long)plk::NORM_BLOCKS * 8 / plk::LIST_MAX + 2 * (long)plk::NORM_BLOCKS * 8;
}

extern "C" int pl_grad_norm(long n, const void* const* grads, const long long* counts, const int* types, double* norm, void* workspace, long workspace_bytes,
                            void* stream) {
  using namespace plk;
  const char* const who = "pl_grad_norm";
  return without_exceptions(who, [&]() -> int {
    int rc = check_list(who, n, grads, counts, types, nullptr, norm, workspace, pl_grad_norm_workspace_bytes(n));
    if (rc == PL_OK) rc = check_norm_args(who, n, norm, workspace, workspace_bytes);
    return rc != PL_OK ? rc : grad_norm_only(n, grads, counts, types, norm, (double*)workspace, (hipStream_t)stream);
  });
}

extern "C" int pl_grad_clip(long n, const void* const* grads, const long long* counts, const int* types, void* const* outs, double max_norm, double eps,
                            const double* norm, void* stream) {
  using namespace plk;
  const char* const who = "pl_grad_clip";
  return without_exceptions(who, [&]() -> int {
    if (n > 0 && !outs) return refuse(PL_ERR_NULL, who, "null list");
    const int rc = check_list(who, n, grads, counts, types, outs, norm, nullptr, 0);
    if (rc != PL_OK) return rc;
    if (!norm) return refuse(PL_ERR_NULL, who, "null norm");
    if (!aligned_to(norm, 8) || !valid_limit(max_norm, eps)) return refuse(PL_ERR_ARG, who, "max_norm or eps negative or NaN, or norm not 8-byte aligned");
    return launch_scale(n, grads, counts, types, outs, max_norm, eps, nullptr, 0, const_cast<double*>(norm), (hipStream_t)stream);
  });
}

extern "C" int pl_grad_norm_clip(long n, const void* const* grads, const long long* counts, const int* types, void* const* outs, double max_norm, double eps,
                                 double* norm, void* workspace, long workspace_bytes, void* stream) {
  using namespace plk;
  const char* const who = "pl_grad_norm_clip";
  return without_exceptions(who, [&]() -> int {
    if (n > 0 && !outs) return refuse(PL_ERR_NULL, who, "null list");
    int rc = check_list(who, n, grads, counts, types, outs, norm, workspace, pl_grad_norm_workspace_bytes(n));
    if (rc == PL_OK) rc = check_norm_args(who, n, norm, workspace, workspace_bytes);
    if (rc != PL_OK) return rc;
    if (!valid_limit(max_norm, eps)) return refuse(PL_ERR_ARG, who, "max_norm or eps negative or NaN");
    hipStream_t s = (hipStream_t)stream;
    int partials = 0;
    rc = launch_squares(n, grads, counts, types, (double*)workspace, &partials, s);
    if (rc != PL_OK) return rc;
    if (partials == 0) return grad_norm_only(0, grads, counts, types, norm, (double*)workspace, s);   // nothing to scale: a norm of zero
    if (partials > NORM_BLOCKS) {
      rc = launch(grad_norm_kernel, dim3(1), dim3(NORM_THREADS), s, (const double*)workspace, partials, norm);
      if (rc != PL_OK) return rc;
      partials = 0;
    }
    return launch_scale(n, grads, counts, types, outs, max_norm, eps, (const double*)workspace, partials, norm, s);
  });
}
