// The row operators for f32 logits.
#include "es_top.cuh"

namespace es {
namespace score {
template cudaError_t launch_loss<ES_F32>(const LossParams&, int, cudaStream_t);
template cudaError_t launch_top<ES_F32>(const TopParams&, cudaStream_t);
}  // namespace score
}  // namespace es
