// The fp32 product in 64 x 64 tiles (wide_product.h).
#include "kernels/wide_product.h"

namespace plk {
int wide_product_f32(const Call& c, const WidePlan& plan, bool at, bool bt, const Epilogue& ep, void* slices) { return wide_product<float>(c, plan, at, bt, ep, slices); }
}  // namespace plk
