#include "km_decay.cuh"
namespace km {
int launch_decay_tc(const km_decay_problem &, const DecayArgs &, bool, cudaStream_t) { return KM_ERR_UNSUPPORTED; }
}  // namespace km
