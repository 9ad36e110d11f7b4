"""Block-scaled 8-bit quantiser and product against the definition in 64 bits.

Tolerances.  Quantiser: the scale is one correctly rounded quotient and a value one more, then one
rounding to e4m3, all restated below step by step, so both are equal bit for bit.  Product: the 8-bit
products are exact in float32, so with S = |bias| + sum of |a_scale b_scale a b| an output is off by at
most (k + ceil(k / 128) + 3) half steps of float32 of S: one addition per value inside a block, then per
block the scales' product, its product with the block's sum and the addition, then the bias; MFMA
accumulates in float32 with at worst a truncation (a whole step) for each addition, hence the factor
two.  Then one rounding to the output's type (half a step of it).  For 16-bit outputs the block's sum is
taken by the 8-bit MFMA, which aligns 8 products to the largest and drops, from each, less than 2^-13
times the power of two below that largest product: at most 8 * 2^-13 = 2^-10 of the largest of every 8,
so at most 2^-10 of S."""

import numpy as np
import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C

BF, HF, F = "bfloat16", "float16", "float32"


def quantized(x, tile):
    """The definition in numpy: (values, scale) of x (rows x cols, float64)."""
    rows, cols = x.shape
    kb = (cols + 127) // 128
    with np.errstate(all="ignore"):
        mag = np.stack([np.abs(x[:, 128 * j:128 * j + 128]).max(1) for j in range(kb)], 1)   # NaN stays
        if tile:
            mag = np.stack([mag[i:i + 128].max(0) for i in range(0, rows, 128)])
        scale = (mag / 448.0).astype(np.float32)
        scale = np.where(scale < np.float32(2.0 ** -126), np.float32(2.0 ** -126), scale)
        full = scale[np.arange(rows) // 128 if tile else np.arange(rows)][:, np.arange(cols) // 128]
        v = (x / full.astype(np.float64)).astype(np.float32).astype(np.float64)
        _, e = np.frexp(np.where(np.isfinite(v), v, 0))
        step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
        return np.where(np.isfinite(v), np.rint(v / step) * step, np.nan), scale


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", [F, BF, HF])
@pytest.mark.parametrize("shape", [(1, 1), (3, 8), (5, 127), (130, 129), (257, 100), (64, 384), (1000, 64), (33, 515)])
def test_quantize_equals_the_definition(shape, dtype, tile):
    g = torch.Generator().manual_seed(shape[0] * 1000 + shape[1])
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[0], 1, generator=g))
    x[0, 0] = 0
    x = x.to(getattr(torch, dtype))
    q, s = C.quantize_blocks(x.cuda(), tile=tile)
    v, scale = quantized(x.double().numpy(), tile)
    np.testing.assert_array_equal(s.cpu().numpy(), scale)
    np.testing.assert_array_equal(q.float().cpu().numpy(), v)


def test_quantize_edges():
    x = torch.zeros(6, 260)
    x[1, 3] = float("nan")          # the whole block is NaN, its neighbours are not
    x[2, 5], x[2, 6] = float("inf"), 1.0
    x[3, :] = 1e-44                  # a scale below the smallest normal number
    x[4, 259] = 3e38
    x[5, :] = torch.linspace(-448, 448, 260)
    q, s = C.quantize_blocks(x.cuda())
    v, scale = quantized(x.double().numpy(), False)
    np.testing.assert_array_equal(s.cpu().numpy(), scale)
    np.testing.assert_array_equal(q.float().cpu().numpy(), v)


def test_quantize_strided_rows_and_every_alignment():
    base = torch.randn(9, 400, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    for at in range(8):
        x = base[::2, at:at + 131]
        q, s = C.quantize_blocks(x)
        q2, s2 = C.quantize_blocks(x.contiguous())
        assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2)
    x = base[:1, :200].expand(5, 200)   # one row, five times
    q, s = C.quantize_blocks(x)
    assert torch.equal(q.float(), C.quantize_blocks(x.contiguous())[0].float())


def operands(m, n, k, tile, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(m, k, generator=g) * (0.2 + torch.rand(m, 1, generator=g))
    b = torch.randn(n, k, generator=g) * (0.2 + torch.rand(n, 1, generator=g))
    qa, sa = C.quantize_blocks(a.cuda())
    qb, sb = C.quantize_blocks(b.cuda(), tile=tile)
    return qa, sa, qb, sb, (torch.randn(n, generator=g).cuda() if bias else None)


def check_product(qa, sa, qb, sb, bias, dtype, tile):
    y = C.matmul_blocks(qa, sa, qb, sb, bias=bias, out_dtype=getattr(torch, dtype))
    m, k = qa.shape
    n = qb.shape[0]
    col = np.arange(k) // 128
    a = qa.float().double().cpu().numpy() * sa.double().cpu().numpy()[:, col]
    w = sb.double().cpu().numpy()
    if tile:
        w = w[np.arange(n) // 128]
    b = qb.float().double().cpu().numpy() * w[:, col]
    bv = np.zeros(n) if bias is None else bias.double().cpu().numpy()
    ref, mag = a @ b.T + bv, np.abs(a) @ np.abs(b).T + np.abs(bv)
    tol = 2 * (k + (k + 127) // 128 + 3) * 2.0 ** -24 * mag
    if dtype != F:
        fi = torch.finfo(getattr(torch, dtype))
        tol = tol + 2.0 ** -10 * mag
        tol = tol + np.maximum((np.abs(ref) + tol) * fi.eps / 2, fi.smallest_normal * fi.eps)
    assert y.shape == (m, n) and y.dtype == getattr(torch, dtype)
    err = np.abs(y.double().cpu().numpy() - ref)
    assert np.all(err <= tol), (err - tol).max()


SHAPES = [(1, 1, 1), (1, 17, 8), (1, 1000, 64), (2, 300, 200), (16, 257, 128), (17, 129, 100), (64, 64, 256),
          (65, 130, 127), (200, 333, 515), (130, 700, 64), (257, 515, 640), (33, 2000, 384), (300, 260, 1027)]


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product_fp32(shape, tile):
    check_product(*operands(*shape, tile, seed=sum(shape)), F, tile)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape", [(1, 333, 64), (40, 200, 128), (129, 257, 300), (512, 384, 512)], ids=str)
def test_product_half_outputs(shape, dtype):
    check_product(*operands(*shape, False, seed=5, bias=False), dtype, False)
    check_product(*operands(*shape, True, seed=6), dtype, True)


LARGE = [(2819, 2999, 259), (33000, 130, 384), (200, 33000, 144), (3000, 2900, 129)]


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large_products(shape, tile):
    ops = operands(*shape, tile, seed=9)
    check_product(*ops, F, tile)
    check_product(*ops, BF, tile)
    check_product(*ops, HF, tile)


@pytest.mark.parametrize("shape", [(5000, 3000, 64), (4100, 4099, 128), (3000, 5000, 100), (20000, 700, 8),
                                   (17, 70000, 31)], ids=str)
def test_many_outputs_of_short_rows(shape):
    for tile in (False, True):
        check_product(*operands(*shape, tile, seed=10), F, tile)
    check_product(*operands(*shape, False, seed=11, bias=False), BF, False)


@pytest.mark.parametrize("at", [0, 1, 4, 13])
@pytest.mark.parametrize("shape", [(1, 65, 70), (3, 65, 300), (130, 257, 300), (260, 300, 1024)], ids=str)
def test_product_any_alignment_and_row_distance(shape, at):
    """Operands that start at any byte, rows further apart than they are long."""
    m, n, k = shape
    qa, sa, qb, sb, bias = operands(m, n, k, False, seed=at)
    want = C.matmul_blocks(qa, sa, qb, sb, bias=bias)

    def moved(q):
        big = torch.full((q.shape[0], k + 37), 0x7f, dtype=torch.uint8, device="cuda")   # NaN around
        big[:, at:at + k] = q.view(torch.uint8) if q.is_contiguous() else q.contiguous().view(torch.uint8)
        return big.view(torch.float8_e4m3fn)[:, at:at + k]

    got = C.matmul_blocks(moved(qa), sa, moved(qb), sb, bias=bias)
    assert torch.equal(got, want)


def test_product_nan_stays_in_its_row_and_column():
    qa, sa, qb, sb, bias = operands(20, 40, 200, False)
    sa, sb = sa.clone(), sb.clone()
    sa[3, 1] = float("nan")
    sb[7, 0] = float("inf")
    y = C.matmul_blocks(qa, sa, qb, sb, bias=bias).cpu()
    bad = ~torch.isfinite(y)
    want = torch.zeros(20, 40, dtype=torch.bool)
    want[3, :] = True
    want[:, 7] = True
    assert torch.equal(bad, want)


def test_product_one_shared_row_and_empty():
    qa, sa, qb, sb, bias = operands(4, 50, 64, False)
    one = C.matmul_blocks(qa[:1], sa[:1], qb, sb, bias=bias)
    many = C.matmul_blocks(qa[:1].expand(40, 64), sa[:1].expand(40, 1).contiguous(), qb, sb, bias=bias)
    assert torch.equal(many, one.expand(40, 50))
    assert C.matmul_blocks(qa[:0], sa[:0], qb, sb).shape == (0, 50)
    assert C.matmul_blocks(qa, sa, qb[:0], sb[:0]).shape == (4, 0)
    q, s = C.quantize_blocks(torch.empty(0, 64, device="cuda"))
    assert q.shape == (0, 64) and s.shape == (0, 1)


def test_product_on_another_stream_and_in_a_graph():
    qa, sa, qb, sb, bias = operands(100, 300, 128, False)
    x = torch.randn(100, 128, device="cuda")
    want = C.matmul_blocks(*C.quantize_blocks(x), qb, sb, bias=bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = C.matmul_blocks(*C.quantize_blocks(x), qb, sb, bias=bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = C.matmul_blocks(*C.quantize_blocks(x), qb, sb, bias=bias)
    for seed in range(3):
        x.copy_(torch.randn(100, 128, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, C.matmul_blocks(*C.quantize_blocks(x), qb, sb, bias=bias))


def test_refusals():
    qa, sa, qb, sb, bias = operands(4, 50, 64, False)
    bad = [lambda: C.quantize_blocks(torch.zeros(2, 4, dtype=torch.float64, device="cuda")),
           lambda: C.quantize_blocks(torch.zeros(8, device="cuda")),
           lambda: C.quantize_blocks(torch.zeros(2, 0, device="cuda")),
           lambda: C.quantize_blocks(torch.zeros(8, 8, device="cuda").t()[:, ::2]),
           lambda: C.quantize_blocks(torch.zeros(2, 4)),
           lambda: C.matmul_blocks(qa, sa, qb[:, :32], sb),
           lambda: C.matmul_blocks(qa, sa[:3], qb, sb),
           lambda: C.matmul_blocks(qa, sa, qb, sb[:49]),
           lambda: C.matmul_blocks(qa, sa.double(), qb, sb),
           lambda: C.matmul_blocks(qa, sa, qb, sb, bias=bias[:49]),
           lambda: C.matmul_blocks(qa.float(), sa, qb, sb),
           lambda: C.matmul_blocks(qa, sa, qb.cpu(), sb),
           lambda: C.matmul_blocks(qa, sa, qb, sb, out_dtype=torch.float64)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", [F, BF, HF])
@pytest.mark.parametrize("shape", [(4096, 3200, 64), (2080, 6144, 32), (4001, 3201, 96), (130, 40003, 128)], ids=str)
def test_short_rows_on_and_off_their_lines(shape, dtype):
    """Rows of outputs that are whole lines of 128 bytes, and rows that start anywhere in one."""
    check_product(*operands(*shape, False, seed=12), dtype, False)
