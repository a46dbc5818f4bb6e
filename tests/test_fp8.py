"""8-bit matrices with a power-of-two scale for each block of 128: quantisation and product against plain statements in 64 bits.

The quantisation has no freedom (scales are whole exponents, values are rounded to nearest even), so its results are compared bit
for bit.  A product of K terms is summed in fp32: each addition is off by at most 2^-23 of the sum of the terms' sizes, the result is
rounded once to its type."""
import pytest
import torch

from kareus_b200 import kernels as K
from kareus_b200.kernels import ref
from kareus_b200.kernels.cuda import KernelError, lib
from kareus_b200.kernels.fp8 import Fp8Matrix

gpu = pytest.mark.gpu
MAX = {"e4m3": 448.0, "e5m2": 57344.0}
DTYPE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def definition(x, fmt, square=False):
    """(values of the format, exponents) by search, in 64 bits."""
    x = x.double().cpu()
    rows, cols = x.shape
    e = torch.empty(rows, -(-cols // 128), dtype=torch.int64)
    q = torch.empty_like(x)
    limits = torch.tensor([MAX[fmt] * 2.0 ** k for k in range(-127, 130)], dtype=torch.float64)
    step = 128 if square else 1
    for c in range(e.shape[1]):
        for r in range(0, rows, step):
            piece = x[r:r + step, c * 128:(c + 1) * 128]
            if not torch.isfinite(piece).all():
                e[r:r + step, c] = 128
                q[r:r + step, c * 128:(c + 1) * 128] = float("nan")
                continue
            k = int(torch.searchsorted(limits, piece.abs().max())) - 127
            e[r:r + step, c] = k
            q[r:r + step, c * 128:(c + 1) * 128] = (piece * 2.0 ** -k).float().to(DTYPE[fmt]).double()
    return q, e


def check_quantized(m, x, fmt, square=False):
    q, e = definition(x, fmt, square)
    assert m.data.dtype == DTYPE[fmt] and m.fmt == fmt and tuple(m.shape) == tuple(x.shape)
    torch.testing.assert_close(m.data.double().cpu(), q, rtol=0, atol=0, equal_nan=True)
    rows, cols = x.shape
    assert torch.equal(m.scales.cpu(), ref.fp8_pack_scales((e + 127).to(torch.uint8)))
    back = m.dequantize(torch.float64).cpu()
    scale = torch.where(e == 128, float("nan"), 2.0 ** e.clamp(max=127).double()).repeat_interleave(128, 1)[:, :cols]
    torch.testing.assert_close(back, q * scale, rtol=0, atol=0, equal_nan=True)


def sample(rows, cols, device, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * std * torch.exp2(torch.randint(-12, 12, (1, cols), generator=g).float())
    return x.bfloat16().to(device)


def edge_values(device):
    """Pieces at the borders of the definition, a row each."""
    x = torch.zeros(16, 200)
    x[1, 0] = 448.0                                        # fits as it is
    x[2, 0] = 452.0                                        # the next bf16: does not
    x[3, 5], x[3, 6] = 57344.0, -57344.0
    x[4, 5] = 57600.0
    x[5, :128] = torch.arange(128) / 7.0 - 9               # ties and small values
    x[6, 3], x[6, 4] = 3.3e38, 1e-30                       # largest exponents, values that vanish beside them
    x[7, 3] = 2.0 ** -130                                  # subnormal bf16
    x[8, 3], x[8, 130] = float("inf"), 1.0                 # one piece of the row is NaN, the other is not
    x[9, 3], x[9, 130] = 1.0, float("nan")
    x[10, 3] = -float("inf")
    x[11] = -0.0
    x[12, :2] = torch.tensor([1.75, -1.7578125])
    x[13, 0], x[13, 1] = 2.0 ** -126, 2.0 ** -133
    x[14, 0], x[14, 1:40] = 448.0, torch.linspace(-0.02, 0.02, 39)   # subnormal values of the format
    return x.bfloat16().to(device)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 8), (7, 40), (128, 128), (129, 136), (300, 1000), (17, 513), (520, 24)])
@pytest.mark.parametrize("square", [False, True])
def test_quantize(device, fmt, shape, square):
    x = sample(*shape, device)
    r, c = K.fp8_quantize(x, rows=True, cols=True, square=square, fmt=fmt)
    check_quantized(r, x, fmt, square)
    check_quantized(c, x.t(), fmt, square)
    only_r, none = K.fp8_quantize(x, square=square, fmt=fmt)
    assert none is None and torch.equal(only_r.data.view(torch.uint8), r.data.view(torch.uint8)) and torch.equal(only_r.scales, r.scales)
    none, only_c = K.fp8_quantize(x, rows=False, cols=True, square=square, fmt=fmt)
    assert none is None and torch.equal(only_c.data.view(torch.uint8), c.data.view(torch.uint8)) and torch.equal(only_c.scales, c.scales)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_edges(device, fmt):
    x = edge_values(device)
    r, c = K.fp8_quantize(x, cols=True, fmt=fmt)
    check_quantized(r, x, fmt)
    check_quantized(c, x.t(), fmt)
    s, t = K.fp8_quantize(x[:8], cols=True, square=True, fmt=fmt)
    check_quantized(s, x[:8], fmt, True)
    check_quantized(t, x[:8].t(), fmt, True)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_square_blocks_that_are_not_finite(device):
    x = sample(300, 300, device)
    x[5, 7], x[200, 290], x[299, 0] = float("inf"), float("nan"), -float("inf")
    for kw in ({"cols": True}, {}, {"rows": False, "cols": True}):
        r, c = K.fp8_quantize(x, square=True, **kw)
        if r is not None:
            check_quantized(r, x, "e4m3", True)
            assert torch.isnan(r.dequantize()[:128, :128]).all() and not torch.isnan(r.dequantize()[:128, 128:]).any()
        if c is not None:
            check_quantized(c, x.t(), "e4m3", True)


@gpu
def test_offsets_beyond_32_bits():
    """Rows more than 2^30 elements apart, in and out."""
    step = 1_200_000_000
    buf = torch.zeros(2 * step + 512, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, 512), (step, 1))
    x.copy_(sample(3, 512, "cuda", 20))
    r, c = K.fp8_quantize(x, cols=True)
    check_quantized(r, x, "e4m3")
    check_quantized(c, x.t(), "e4m3")
    out = buf.as_strided((3, 200), (step, 1), 256)
    b, _ = K.fp8_quantize(sample(200, 512, "cuda", 21))
    check_product(K.fp8_gemm(r, b, out=out), r, b)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_quantize_views(device):
    """Rows of a wider buffer, an odd offset, a transposed matrix, every second row."""
    base = sample(200, 400, device)
    for x in (base[:, 16:216], base[3:, 1:258], base.t(), base[::2], base[:1, 5:90], base[:, 7:8], base[4].expand(9, 400)):
        r, c = K.fp8_quantize(x, cols=True)
        check_quantized(r, x, "e4m3")
        check_quantized(c, x.t(), "e4m3")


def product(a, b):
    """(product in 64 bits, sum of the terms' sizes)."""
    A, B = a.dequantize(torch.float64), b.dequantize(torch.float64)
    return A @ B.t(), A.abs() @ B.abs().t()


def check_product(y, a, b, before=None):
    want, size = product(a, b)
    if before is not None:
        want, size = want + before.double(), size + before.double().abs()
    half = 2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24
    tol = half * want.abs() + (a.shape[1] + 1) * 2.0 ** -23 * size
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(y), nan)
    off = torch.where(nan, 0.0, (y.double() - want).abs() - tol)
    assert off.max().item() <= 0, (off.max().item(), want[~nan].abs().max().item())


SHAPES = [(1, 8, 16), (5, 64, 8), (128, 128, 128), (256, 256, 512), (130, 200, 264), (300, 776, 1032), (17, 640, 4096), (512, 72, 1500),
          (700, 1000, 513), (257, 2048, 640)]


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("fmts", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
def test_gemm(shape, fmts):
    M, N, Kd = shape
    a, _ = K.fp8_quantize(sample(M, Kd, "cuda", 1), fmt=fmts[0])
    b, _ = K.fp8_quantize(sample(N, Kd, "cuda", 2), fmt=fmts[1])
    check_product(K.fp8_gemm(a, b), a, b)
    check_product(K.fp8_gemm(a, b, out_dtype=torch.float32), a, b)
    acc = torch.randn(M, N, device="cuda")
    before = acc.clone()
    assert K.fp8_gemm(a, b, accumulate=acc) is acc
    check_product(acc, a, b, before)


@gpu
@pytest.mark.parametrize("width", [64, 128, 192, 256])
def test_gemm_tile_widths(width):
    """Every tile width, several tiles a pair (both accumulators and what they share), scales that start inside a block of 128."""
    M, Kd = 148 * 256 // 2 + 40, 1100
    for N in (width, 3 * width - 24):
        a, _ = K.fp8_quantize(sample(M, Kd, "cuda", 3))
        b, _ = K.fp8_quantize(sample(N, Kd, "cuda", 4))
        check_product(K.fp8_gemm(a, b), a, b)
        check_product(K.fp8_gemm(a, b, out_dtype=torch.float32), a, b)


@gpu
@pytest.mark.parametrize("M", [1, 7, 8, 9, 64, 100, 120, 121, 127, 128, 129, 255, 257])
def test_gemm_few_rows(M):
    """Rows of A that are loaded: all there are, in groups of 8, below 128."""
    a, _ = K.fp8_quantize(sample(M, 700, "cuda", 3))
    for N in (40, 300, 9000):
        b, _ = K.fp8_quantize(sample(N, 700, "cuda", 4))
        check_product(K.fp8_gemm(a, b), a, b)
        check_product(K.fp8_gemm(b, a, out_dtype=torch.float32), b, a)


@gpu
def test_gemm_many_tiles():
    a, _ = K.fp8_quantize(sample(4000, 700, "cuda", 3))
    b, _ = K.fp8_quantize(sample(9000, 700, "cuda", 4))
    y = K.fp8_gemm(a, b)
    check_product(y, a, b)
    assert torch.equal(y, K.fp8_gemm(a, b))                       # the same bits every time
    acc = torch.zeros(4000, 9000, device="cuda")
    K.fp8_gemm(a, b, accumulate=acc)
    assert torch.equal(acc, K.fp8_gemm(a, b, out_dtype=torch.float32))


@gpu
def test_gemm_destinations():
    """A destination inside a wider buffer leaves what lies beside it as it was; rows that start anywhere."""
    a, _ = K.fp8_quantize(sample(70, 256, "cuda", 5))
    b, _ = K.fp8_quantize(sample(90, 256, "cuda", 6))
    for dtype in (torch.bfloat16, torch.float32):
        for lead in (0, 1, 8):
            buf = torch.full((72, 120), 7.0, dtype=dtype, device="cuda")
            out = buf[1:71, lead:lead + 90]
            assert K.fp8_gemm(a, b, out=out) is out
            check_product(out, a, b)
            buf[1:71, lead:lead + 90] = 7.0
            assert bool((buf == 7.0).all())
    acc = torch.ones(70, 93, device="cuda")[:, 2:92]
    K.fp8_gemm(a, b, accumulate=acc)
    check_product(acc, a, b, torch.ones(70, 90, device="cuda"))


@gpu
def test_gemm_not_finite_blocks():
    x = sample(40, 400, "cuda", 7)
    x[3, 200] = float("inf")
    x[9, 399] = float("nan")
    a, _ = K.fp8_quantize(x)
    b, _ = K.fp8_quantize(sample(50, 400, "cuda", 8))
    y = K.fp8_gemm(a, b)
    check_product(y, a, b)
    assert torch.isnan(y[3]).all() and torch.isnan(y[9]).all() and torch.isnan(y).sum() == 100


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_linear_layer_gradients(device):
    """Forward, input gradient and weight gradient from the two layouts of each matrix."""
    g = torch.Generator().manual_seed(5)
    x, w, dy = (torch.randn(s, generator=g).bfloat16().to(device) for s in ((200, 264), (136, 264), (200, 136)))
    xr, xc = K.fp8_quantize(x, cols=True)
    wr, wc = K.fp8_quantize(w, cols=True, square=True)
    dr, dc = K.fp8_quantize(dy, cols=True, fmt="e5m2")
    assert torch.equal(wr.dequantize().t(), wc.dequantize())       # one set of values serves both directions
    y, dx, dw = K.fp8_gemm(xr, wr), K.fp8_gemm(dr, wc), torch.zeros(136, 264, device=device)
    K.fp8_gemm(dc, xc, accumulate=dw)
    for got, a, b in ((y, xr, wr), (dx, dr, wc), (dw, dc, xc)):
        check_product(got, a, b)
    # a value of 3 (2) bits of mantissa is off by at most 2^-4 (2^-3) of itself, or by half the smallest step of its piece
    exact = dy.double().t() @ x.double()
    err = (dw.double() - exact).norm() / exact.norm()
    assert err < 2.0 ** -4 + 2.0 ** -3


@gpu
def test_two_streams_and_capture():
    """Calls on two streams at once, and a captured sequence whose inputs change between replays."""
    a0, b0 = sample(300, 512, "cuda", 9), sample(400, 512, "cuda", 10)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2):
        with torch.cuda.stream(s):
            outs.append([K.fp8_gemm(K.fp8_quantize(a0)[0], K.fp8_quantize(b0)[0]) for _ in range(4)])
    torch.cuda.synchronize()
    a, b = K.fp8_quantize(a0)[0], K.fp8_quantize(b0)[0]
    want = K.fp8_gemm(a, b)
    assert all(torch.equal(o, want) for o in outs[0] + outs[1])
    x = a0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = K.fp8_gemm(K.fp8_quantize(x)[0], b)
    for seed in (11, 12):
        x.copy_(sample(300, 512, "cuda", seed))
        graph.replay()
        assert torch.equal(y, K.fp8_gemm(K.fp8_quantize(x)[0], b))


@gpu
def test_empty():
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    r, c = K.fp8_quantize(x, cols=True)
    assert tuple(r.shape) == (0, 64) and tuple(c.shape) == (64, 0)
    w, wt = K.fp8_quantize(sample(24, 64, "cuda"), cols=True)
    assert tuple(K.fp8_gemm(r, w).shape) == (0, 24)
    acc = torch.ones(64, 64, device="cuda")
    K.fp8_gemm(c, c, accumulate=acc)                               # nothing to add
    assert bool((acc == 1).all())
    assert bool((K.fp8_gemm(c, c) == 0).all())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    x = sample(32, 64, device)
    a, _ = K.fp8_quantize(x)
    b, _ = K.fp8_quantize(x[:, :48])
    with pytest.raises(KernelError, match="format"):
        K.fp8_quantize(x, fmt="e3m4")
    with pytest.raises(KernelError, match="matrix"):
        K.fp8_quantize(x[None])
    with pytest.raises(KernelError, match="matrix"):
        K.fp8_quantize(x.to(torch.int32))
    with pytest.raises(KernelError, match="neither"):
        K.fp8_quantize(x, rows=False)
    with pytest.raises(ValueError, match="K=64 vs 48"):
        K.fp8_gemm(a, b)
    with pytest.raises(KernelError, match="Fp8Matrix"):
        K.fp8_gemm(a, x)
    with pytest.raises(KernelError, match="scales"):
        K.fp8_gemm(a, Fp8Matrix(a.data, a.scales[:, :0], "e4m3"))
    with pytest.raises(KernelError, match="format"):
        K.fp8_gemm(a, Fp8Matrix(a.data, a.scales, "e5m2"))
    with pytest.raises(KernelError, match="destination"):
        K.fp8_gemm(a, a, out=torch.zeros(32, 31, device=device))
    with pytest.raises(KernelError, match="accumulate"):
        K.fp8_gemm(a, a, out_dtype=torch.float32, accumulate=torch.zeros(32, 32, device=device))


@gpu
def test_gpu_refusals():
    x = sample(32, 64, "cuda")
    a, _ = K.fp8_quantize(x)
    with pytest.raises(KernelError, match="fp32"):
        K.fp8_gemm(a, a, accumulate=torch.zeros(32, 32, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(KernelError, match="bf16 or fp32"):
        K.fp8_gemm(a, a, out_dtype=torch.float16)
    with pytest.raises(KernelError, match="devices"):
        K.fp8_gemm(a, Fp8Matrix(a.data.cpu(), a.scales.cpu()))
    with pytest.raises(KernelError, match="16 bytes"):
        K.fp8_gemm(Fp8Matrix(a.data[:, 1:], a.scales), Fp8Matrix(a.data[:, 1:], a.scales))
    with pytest.raises(KernelError, match="contiguous"):
        K.fp8_gemm(a, a, out=torch.zeros(32, 32, device="cuda").t()[:, :32].t().t())


def test_largest_sizes():
    """Row and column numbers are ints in the kernels, those of tiles that cross the edge too: sizes near 2^31 are refused."""
    one = torch.zeros(1, 1, dtype=torch.bfloat16)
    for shape in ((2 ** 31 - 511, 1), (1, 2 ** 31 - 1), (2 ** 31, 1)):
        with pytest.raises(KernelError, match="too large"):
            K.fp8_quantize(one.expand(shape))
    L = lib()
    for rows, cols in ((2 ** 31 - 511, 8), (8, 2 ** 31 - 1)):      # refused by the entry itself, before anything is launched
        assert L.kb_fp8_quantize(16, rows, cols, cols, 16, 2 ** 31, 16, 16, 2 ** 31, 16, 0, 0, 0) == 7
    for m, n, k in ((2 ** 31 - 511, 8, 16), (8, 2 ** 31 - 1, 16), (8, 8, 2 ** 31 - 511)):
        assert L.kb_gemm_fp8(16, 16, 0, 2 ** 31, 16, 16, 0, 2 ** 31, 16, 2 ** 31, m, n, k, 0, 0, 0, 0) == 7


@gpu
def test_results_as_tensors():
    """What the native call returns behaves like any tensor: views, inference mode, autograd's saving, storage of its own."""
    x = sample(200, 136, "cuda")
    K.fp8_quantize(x)                                              # the native call takes over from here
    (r, c), (want, _) = K.fp8_quantize(x, cols=True), K.fp8_quantize(x.cpu())
    assert r.data.storage_offset() == 0 and r.data.untyped_storage().data_ptr() != c.data.untyped_storage().data_ptr()
    assert r.scales.is_contiguous() and not r.data.requires_grad and r.data.device == x.device
    assert torch.equal(r.data.cpu().view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(r.scales.clone().cpu(), want.scales)
    with torch.inference_mode():
        y, (inside, _) = x + 0, K.fp8_quantize(x)
        assert inside.data.is_inference() and torch.equal(inside.scales, r.scales)
    outside, _ = K.fp8_quantize(y)                                 # an inference tensor as input, its result is none
    assert not outside.data.is_inference()

    class Keep(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            ctx.save_for_backward(outside.data, outside.scales)
            return t * 2

        @staticmethod
        def backward(ctx, d):
            data, scales = ctx.saved_tensors
            return d * Fp8Matrix(data, scales).dequantize().sum()

    t = torch.ones(1, device="cuda", requires_grad=True)
    Keep.apply(t).backward()
    assert torch.equal(t.grad[0], outside.dequantize().sum())


#: width of the tiles -> rows and columns of a product that takes it with several tiles a pair of SMs, 74 pairs or a few fewer
WIDTHS = {64: (60000, 64), 128: (60000, 120), 192: (18984, 552), 256: (18984, 744)}


def _columns(M, N, Kd, sms):
    import ctypes
    from kareus_b200.kernels import build
    if not build.LIB.exists():
        pytest.skip("native library not built")
    f = ctypes.CDLL(str(build.LIB)).kb_gemm_fp8_columns
    f.argtypes = [ctypes.c_int] * 4
    return f(M, N, Kd, sms)


@pytest.mark.parametrize("sms", [132, 140, 148])
def test_sizes_take_every_tile_width(sms):
    """What the tests of the widths run, and the two borders of the choice: few tiles take narrow ones, many wide ones."""
    assert all(_columns(*size, 1100, sms) == width for width, size in WIDTHS.items())
    assert {_columns(148 * 256 // 2 + 40, n, 1100, 148) for w in WIDTHS for n in (w, 3 * w - 24)} == set(WIDTHS)
    assert _columns(1, 9000, 700, sms) in WIDTHS and _columns(17, 64, 1100, sms) == 64 and _columns(8192, 28672, 4096, sms) == 256


@gpu
@pytest.mark.parametrize("width", sorted(WIDTHS))
def test_gemm_several_tiles_of_every_width(width):
    (M, N), Kd = WIDTHS[width], 1100
    assert _columns(M, N, Kd, torch.cuda.get_device_properties(0).multi_processor_count) == width
    a, _ = K.fp8_quantize(sample(M, Kd, "cuda", 3))
    b, _ = K.fp8_quantize(sample(N, Kd, "cuda", 4))
    y = K.fp8_gemm(a, b)
    check_product(y, a, b)
    assert torch.equal(y, K.fp8_gemm(a, b))
    acc = torch.ones(M, N, device="cuda")
    K.fp8_gemm(a, b, accumulate=acc)
    check_product(acc, a, b, torch.ones(M, N, device="cuda"))
