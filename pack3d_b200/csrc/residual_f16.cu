// The row kernels of residual_rows.cuh for __half.
#include "residual_rows.cuh"

namespace p3d {
namespace rows {
P3D_ROW_KERNELS(__half)
}  // namespace rows
}  // namespace p3d
