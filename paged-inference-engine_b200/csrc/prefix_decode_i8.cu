#include "prefix_decode.cuh"

namespace pa {
template int prefix_decode_plan_kv<KV_I8>(int, int, int, int, bool, DecodeLaunch*);
template cudaError_t prefix_decode_launch_kv<KV_I8>(const SharedParams&, const KvMaps&, int, int, bool, const DecodeLaunch&,
                                                    cudaStream_t);
}  // namespace pa
