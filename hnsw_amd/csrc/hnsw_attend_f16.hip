// The attention for f16 queries and outputs.
#include "hnsw_attend_kernels.h"

namespace hnsw_amd {
template void launch_attend<_Float16>(const AttendArgs&, const Cut&, uint32_t, float*, hipStream_t);
}
