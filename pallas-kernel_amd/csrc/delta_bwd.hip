#include "delta.hpp"
namespace tops {
hipError_t run_delta_bwd(const DeltaParams&, hipStream_t) { return hipErrorNotSupported; }
}
