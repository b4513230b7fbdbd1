// The chunked pass of linear attention on bf16 rows.
#include "linear_attn_kernel.h"

namespace mogt {
template void la_launch_passes<bf16_t>(const LaArgs&, int, bool, hipStream_t);
}
