"""The block-boundary operators at the edges of their sizes, and the 8-bit linear
layer's kernels beside one another."""
import pytest
import torch

from gpu_util import no_device_error
from wide_compiler import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def int8_case(n, m, k, o, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ints = lambda *s: torch.randint(-127, 128, s, generator=gen, dtype=torch.int8).to(DEV)
    return ints(n, m, k), torch.rand(n, m, generator=gen).to(DEV), ints(n, o, k), torch.rand(n, o, generator=gen).to(DEV)


def test_parts_of_k_beside_wide_tiles():
    """Few tokens with K over a cluster (8, 4 and 2 parts) on one stream, 256 x 256 tiles of block pairs on
    another: the results of each alone."""
    few = [int8_case(1, 1, 8192, 512), int8_case(1, 33, 4096, 1024), int8_case(2, 100, 2048, 512)]
    many = [int8_case(4, 1024, 512, 1024), int8_case(1, 4096, 1024, 2048)]
    want = [[ops.linear_int8(*a, dtype=BF16) for a in side] for side in (few, many)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for i in range(30):
        for side, (cases, stream) in enumerate(zip((few, many), streams)):
            with torch.cuda.stream(stream):
                outs[side] += [ops.linear_int8(*a, dtype=BF16) for a in cases]
    torch.cuda.synchronize()
    for side, out in enumerate(outs):
        assert all(torch.equal(y, want[side][i % len(want[side])]) for i, y in enumerate(out))
    no_device_error()
