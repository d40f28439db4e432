"""Every tile of the gated product's kernels against float64, at sizes that end inside a tile, a stage and a piece of 16 bytes.

Which tile a product takes goes by its size (gated.hip); `tiles` is that rule, and each case names the tiles that it is there
for, so that a change of the rule that would leave one without a case shows here.
"""
import pytest
import torch

from test_gpu_encoder import TYPES
from test_gpu_gated import check, operands

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def up(a, b):
    return (a + b - 1) // b


def tile(M, N, K, results, parts, share, rows, size):
    """Rows of the tile of a product with results [M, N] and sums of `parts` times K, or "shared"."""
    few = up(M, 64) * up(N, 64) * results
    stages = up(K, (128 if rows else 64) // size) * parts
    length = stages * (1 if size == 2 else 4 if rows else 2)
    if 1 <= few <= 192 and length >= 32 and min(512 // few, length // 12, stages, 16) > 1:
        return "shared"
    if size == 2:
        large = up(M, 256) * up(N, 256 // share) * results
        if large * 4 >= up(large, 256) * 256 * 3:
            return 256
    return 128 if up(M, 128) * up(N, 128 // share) * results >= 256 else 64


def tiles(M, N, K, dtype):
    size = 4 if dtype is torch.float32 else 2
    return {"h": tile(M, N, K, 1, 1, 2, True, size), "dx": tile(M, K, N, 1, 2, 1, False, size),
            "dw": tile(N, K, M, 2, 1, 1, False, size)}


CASES = [("h", 256, HALVES, [(2999, 2035, 133), (2817, 1921, 40)]),
         ("h", 128, TYPES, [(1499, 1397, 133), (1409, 1400, 72)]),
         ("h", 64, TYPES, [(131, 67, 37), (1000, 130, 8)]),
         ("dx", 256, HALVES, [(2999, 77, 4091), (2817, 40, 3848)]),
         ("dx", 128, TYPES, [(1999, 75, 2037), (1930, 33, 1928)]),
         ("dx", 64, TYPES, [(131, 67, 37), (1000, 24, 1100)]),
         ("dw", 256, HALVES, [(91, 1997, 2991), (40, 1793, 2824)]),
         ("dw", 128, TYPES, [(91, 1397, 1491), (37, 1400, 1416)]),
         ("dw", 64, TYPES, [(131, 67, 37), (100, 1100, 900)])]


@pytest.mark.parametrize("what,rows,dtype,size", [(w, r, d, s) for w, r, types, sizes in CASES for d in types for s in sizes],
                         ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
def test_tiles(dev, what, rows, dtype, size):
    assert tiles(*size, dtype)[what] == rows, tiles(*size, dtype)
    x, wg, wu, grad = operands(sum(size), dtype, *size)
    check(x, wg, wu, ("silu", "gelu", "gelu_tanh")[sum(size) % 3], grad)
