// The kernels of mor_mx_matmul for A in E4M3.
#include "mor_mxmatmul.h"

namespace mor {
int launch_product_e4m3(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st) { return launch_product<FMT_E4M3>(args, b_fmt, q, st); }
}  // namespace mor
