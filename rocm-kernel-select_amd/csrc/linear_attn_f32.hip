// Linear attention over sequences: the chunk kernels for float.
#include "linear_attn_chunk.h"

namespace atk {
template int la_launch_out<float>(const LaArgs&, hipStream_t);
template int la_launch_grads<float>(const LaArgs&, bool, hipStream_t);
template int la_launch_states<float>(const LaArgs&, int, float* const*, float*, hipStream_t);
}  // namespace atk
