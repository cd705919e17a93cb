// The kernels of mor_mx_matmul for A in E5M2.
#include "mor_mxmatmul.h"

namespace mor {
int launch_product_e5m2(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st) { return launch_product<FMT_E5M2>(args, b_fmt, q, st); }
}  // namespace mor
