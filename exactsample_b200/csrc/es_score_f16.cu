// The row operators for f16 logits.
#include "es_top.cuh"

namespace es {
namespace score {
template cudaError_t launch_loss<ES_F16>(const LossParams&, int, cudaStream_t);
template cudaError_t launch_top<ES_F16>(const TopParams&, cudaStream_t);
}  // namespace score
}  // namespace es
