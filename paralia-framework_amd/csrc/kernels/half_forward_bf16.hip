// The 16-bit product (half_product.h) on bf16 operands, result of the same type.
#include "kernels/half_product.h"

namespace plk {
int half_forward_bf16(const Call& c, const HalfPlan& plan, bool at, bool bt, const Epilogue& ep) { return half_direct<bf16_t, bf16_t, false>(c, plan, at, bt, ep); }
}  // namespace plk
