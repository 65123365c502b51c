// The 16-bit product (half_product.h) on bf16 operands, result in fp32.
#include "kernels/half_product.h"

namespace plk {
int half_wide_bf16(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep) { return half_direct<bf16_t, float, false>(c, plan, at, bt, ep); }
int half_slices_bf16(const Call& c, const HalfPlan& plan, bool at, bool bt, void* slices) { return half_slices<bf16_t>(c, plan, at, bt, slices); }
}  // namespace plk
