// The 16-bit product (half_product.h) on f16 operands, result in fp32.
#include "kernels/half_product.h"

namespace plk {
int half_wide_f16(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep) { return half_direct<f16_t, float, false>(c, plan, at, bt, ep); }
int half_slices_f16(const Call& c, const HalfPlan& plan, bool at, bool bt, void* slices) { return half_slices<f16_t>(c, plan, at, bt, slices); }
}  // namespace plk
