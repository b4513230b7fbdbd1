// The chunked pass of linear attention on fp32 rows.
#include "linear_attn_kernel.h"

namespace mogt {
template void la_launch_passes<float>(const LaArgs&, int, bool, hipStream_t);
}
