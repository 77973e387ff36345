// Single-token attention over a paged cache: the e4m3 instantiations.
#include "decode_attention.cuh"

namespace widek {
template int launch_decode<DK_E4M3, false>(const DecodeArgs&, cudaStream_t);
}  // namespace widek
