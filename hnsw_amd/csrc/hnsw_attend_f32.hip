// The attention for f32 queries and outputs.
#include "hnsw_attend_kernels.h"

namespace hnsw_amd {
template void launch_attend<float>(const AttendArgs&, const Cut&, uint32_t, float*, hipStream_t);
}
