// The kernels of mor_mx_matmul for A in E2M1.
#include "mor_mxmatmul.h"

namespace mor {
int launch_product_e2m1(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st) { return launch_product<FMT_E2M1>(args, b_fmt, q, st); }
}  // namespace mor
