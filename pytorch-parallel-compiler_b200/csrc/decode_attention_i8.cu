// Single-token attention over a paged cache: the i8 instantiations.
#include "decode_attention.cuh"

namespace widek {
template int launch_decode<DK_I8, false>(const DecodeArgs&, cudaStream_t);
}  // namespace widek
