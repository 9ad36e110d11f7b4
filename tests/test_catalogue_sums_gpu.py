"""The 8-bit product's sums are float32 whatever the output's type, rounded once.

Every number here is an integer and every partial sum of a row, in any order, stays below 2^24 (at most 16 pairs
of 448 * 448 a block, and the small products), so float32 sums are exact and the comparison needs no tolerance:
a 16-bit output is the exact sum rounded to its type."""

import numpy as np
import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C

BF, HF, F = "bfloat16", "float16", "float32"


def cancelling(m, n, k, seed):
    """e4m3 operands of small integers; in every 8 neighbours a pair of 448 in a stands against 448, -448 in b."""
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-2, 3, (m, k), generator=g).float()
    b = torch.randint(-2, 3, (n, k), generator=g).float()
    for at in range(0, k - 1, 8):
        i, j = (at + torch.randperm(min(8, k - at), generator=g)[:2]).tolist()
        a[:, i] = a[:, j] = 448.0
        b[:, i], b[:, j] = 448.0, -448.0
    return a, b


def as_e4m3(x, pitch):
    q = torch.empty(x.shape[0], pitch, dtype=torch.float8_e4m3fn, device="cuda")[:, :x.shape[1]]
    q.copy_(x.cuda().to(torch.float8_e4m3fn))
    return q


# a tile a wave, 2 x 2 and 4 x 4 of them (rows that are no multiple of 16 bytes), rows of one block, large tiles
SHAPES = [(1, 40, 64, 64), (9, 333, 300, 304), (40, 200, 128, 128), (2100, 2117, 200, 200), (4100, 4099, 24, 32),
          (4100, 4099, 64, 64), (4100, 4099, 100, 112), (4096, 4096, 128, 128), (3000, 2900, 129, 144),
          (2304, 2304, 384, 384)]


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", [F, BF, HF])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sums_that_cancel(shape, dtype, tile):
    m, n, k, pitch = shape
    a, b = cancelling(m, n, k, seed=k)
    kb = (k + 127) // 128
    one = torch.ones(m, kb, device="cuda"), torch.ones((n + 127) // 128 if tile else n, kb, device="cuda")
    y = C.matmul_blocks(as_e4m3(a, pitch), one[0], as_e4m3(b, pitch), one[1], out_dtype=getattr(torch, dtype))
    want = torch.from_numpy(a.double().numpy() @ b.double().numpy().T).to(getattr(torch, dtype))
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sixteen_bit_outputs_are_the_float32_ones_rounded(shape):
    m, n, k, _ = shape
    g = torch.Generator().manual_seed(k + 1)
    ops = [C.quantize_blocks(torch.randn(r, k, generator=g).cuda()) for r in (m, n)]
    bias = torch.randn(n, generator=g).cuda()
    y = C.matmul_blocks(*ops[0], *ops[1], bias=bias)
    # The last product and addition are one operation, which may be rounded to 16 bits with no float32 between (fp16
    # has such an instruction): the exact v lies within half a float32 step of y, and rounding is monotone, so what v
    # rounds to lies between what y's two neighbours round to.  That is what y rounds to unless y stands at the middle
    # of two 16-bit numbers.
    far = torch.full_like(y, float("inf"))
    for dtype in (torch.bfloat16, torch.float16):
        half = C.matmul_blocks(*ops[0], *ops[1], bias=bias, out_dtype=dtype)
        assert torch.all((torch.nextafter(y, -far).to(dtype) <= half) & (half <= torch.nextafter(y, far).to(dtype)))
        assert (half != y.to(dtype)).sum() <= 2.0 ** -12 * y.numel() + 1     # (one in 2^13 of fp16's roundings)
