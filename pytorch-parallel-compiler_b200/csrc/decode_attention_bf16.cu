// Single-token attention over a paged cache: the bf16 instantiations.
#include "decode_attention.cuh"

namespace widek {
template int launch_decode<DK_BF16, false>(const DecodeArgs&, cudaStream_t);
}  // namespace widek
