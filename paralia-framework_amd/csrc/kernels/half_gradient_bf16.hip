// The 16-bit product (half_product.h) on bf16 operands, gradient through an activation.
#include "kernels/half_product.h"

namespace plk {
int half_gradient_bf16(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep) { return half_direct<bf16_t, bf16_t, true>(c, plan, at, bt, ep); }
}  // namespace plk
