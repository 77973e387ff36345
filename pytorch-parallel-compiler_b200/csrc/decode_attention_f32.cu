// Single-token attention over a paged cache: the f32 instantiations.
#include "decode_attention.cuh"

namespace widek {
template int launch_decode<DK_F32, false>(const DecodeArgs&, cudaStream_t);
}  // namespace widek
