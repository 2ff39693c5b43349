// Linear attention over sequences: the chunk kernels for _Float16.
#include "linear_attn_chunk.h"

namespace atk {
template int la_launch_out<_Float16>(const LaArgs&, hipStream_t);
template int la_launch_grads<_Float16>(const LaArgs&, bool, hipStream_t);
template int la_launch_states<_Float16>(const LaArgs&, int, float* const*, float*, hipStream_t);
}  // namespace atk
