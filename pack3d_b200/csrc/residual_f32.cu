// The row kernels of residual_rows.cuh for float.
#include "residual_rows.cuh"

namespace p3d {
namespace rows {
P3D_ROW_KERNELS(float)
}  // namespace rows
}  // namespace p3d
