// The row kernels of residual_rows.cuh for __nv_bfloat16.
#include "residual_rows.cuh"

namespace p3d {
namespace rows {
P3D_ROW_KERNELS(__nv_bfloat16)
}  // namespace rows
}  // namespace p3d
