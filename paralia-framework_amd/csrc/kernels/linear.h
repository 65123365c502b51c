// Host side shared by the linear-layer operators: argument checks and the launchers that one source file calls in another.
#ifndef PLK_LINEAR_H
#define PLK_LINEAR_H
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

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
// the same matrix, element for element, or no byte in common
inline bool same_or_apart(const Range& a, const Range& b) {
  return (a.p == b.p && (a.ld == b.ld || a.cols == 1) && a.size == b.size) || !overlap(a, b);
}

// epilogue.hip
int bias_fold(int type, long M, long rows, const void* partial, void* dbias, hipStream_t stream);
long epilogue_pass_rows(int type, long M, long N);
int epilogue_pass(int type, int type_d, bool grad, long M, long N, const void* P, long ldP, long slice, int slices, const Epilogue& ep, hipStream_t stream);

}  // namespace plk
#endif
