// Linear attention over sequences: the chunk kernels for __bf16.
#include "linear_attn_chunk.h"

namespace atk {
template int la_launch_out<__bf16>(const LaArgs&, hipStream_t);
template int la_launch_grads<__bf16>(const LaArgs&, bool, hipStream_t);
template int la_launch_states<__bf16>(const LaArgs&, int, float* const*, float*, hipStream_t);
}  // namespace atk
