#include "pa_common.cuh"
namespace pa {
bool prefix_wide_supported(int, int, int) { return false; }
cudaError_t launch_prefix_wide(const SharedParams&, const KvMaps&, int, int, cudaStream_t) { return cudaErrorNotSupported; }
}  // namespace pa
