"""Newton-Schulz orthogonalisation and the Muon step against plain statements in 64 bits.

How far the kernel may be off: it holds X, G and P (without its diagonal) in fp16.  `rounded` is the same iteration in 64 bits with
every stored matrix, diagonal included, rounded so; the kernel may be twice as far from the exact result as that (roundings of
another order), plus the rounding of its result to bf16 (2^-8 of each entry) and 1e-6 for sums in fp32."""
import pytest
import torch

from kareus_b200 import kernels as K
from kareus_b200.kernels.cuda import KernelError
from kareus_b200.kernels.muon import COEFFICIENTS, fp16_scales

gpu = pytest.mark.gpu


def iterate(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7, rnd=lambda t: t):
    a, b, c = coefficients
    x = x.double()
    x = rnd(x / (torch.linalg.matrix_norm(x, keepdim=True) + eps))
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            g = rnd(x @ x.mT)
            x = rnd(a * x + rnd(b * g + c * (g @ g)) @ x)
        else:
            g = rnd(x.mT @ x)
            x = rnd(a * x + x @ rnd(b * g + c * (g @ g)))
    return x


def check(o, x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    scale, _ = fp16_scales(steps, coefficients)
    exact = iterate(x, steps, coefficients, eps)
    rounded = iterate(x, steps, coefficients, eps, lambda t: (t * scale).half().double() / scale)
    assert o.shape == x.shape and o.dtype == torch.bfloat16
    norm = torch.linalg.matrix_norm
    err, own = norm(o.double() - exact), norm(rounded - exact)
    limit = 2 * own + (2.0 ** -8 + 1e-6) * norm(exact)
    assert bool((err <= limit).all()), (err / norm(exact)).max().item()
    # and no entry is far off: an entry's error is spread by the products
    rms = norm(exact) / (x.shape[-1] * x.shape[-2]) ** 0.5
    assert bool(((o.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 0.05 * rms[..., None, None] + 12 * (own / norm(exact).clamp(min=1e-30)
                 )[..., None, None] * rms[..., None, None]).all())


def matrices(batch, m, n, device="cuda", seed=0, std=1e-3):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(batch, m, n, generator=g) * std).to(device)


SIZES = [(1, 1, 1), (1, 1, 7), (1, 9, 1), (1, 5, 3), (2, 16, 16), (1, 64, 200), (3, 130, 70), (3, 333, 1000), (1, 1000, 333), (2, 512, 512),
         (1, 2048, 512), (40, 24, 40), (1, 300, 1504), (1, 1100, 2600), (1, 1500, 900), (1, 257, 256), (1, 256, 321), (2, 1030, 1800), (1, 1700, 1024),
         (1, 24, 9000), (1, 7001, 40), (2, 300, 6000), (1, 5003, 130)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("size", [(1, 5, 3), (2, 16, 16), (3, 30, 70)])
def test_small(device, size):
    x = matrices(*size, device)
    check(K.orthogonalize(x), x)
    check(K.orthogonalize(x[0]), x[0])
    check(K.orthogonalize(x[None]), x[None])


@gpu
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize(size, dtype):
    x = matrices(*size).to(dtype)
    o = K.orthogonalize(x)
    check(o, x)
    assert torch.equal(o, K.orthogonalize(x))                      # the same bits every time


@gpu
@pytest.mark.parametrize("size", [(390, 11850), (11464, 314), (469, 8717), (44, 44), (1024, 1600), (64, 4000)])
def test_as_exact_as_its_result_type(size):
    """The iteration adds little to what rounding the result to bf16 costs (1.66e-3 in the 2-norm): diagonals are kept in fp32, so that
    even nearly orthogonal matrices, whose diagonals' roundings would add up, stay within 1.5 times that."""
    x = matrices(1, *size, seed=14)
    exact = iterate(x)
    norm = torch.linalg.matrix_norm
    assert bool((norm(K.orthogonalize(x).double() - exact) < 1.5 * norm(exact.bfloat16().double() - exact)).all())


@gpu
@pytest.mark.parametrize("steps, coefficients", [(1, COEFFICIENTS), (2, COEFFICIENTS), (3, COEFFICIENTS), (4, COEFFICIENTS),
                                                 (8, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375))])
def test_other_coefficients(steps, coefficients):
    for size in ((1, 200, 456), (2, 321, 130), (1, 1600, 1040)):
        x = matrices(*size, seed=3)
        check(K.orthogonalize(x, steps, coefficients), x, steps, coefficients)


@gpu
def test_singular_values_and_vectors():
    """A matrix with known factors: the vectors stay, the values go where the polynomial takes them."""
    g = torch.Generator().manual_seed(1)
    u, _ = torch.linalg.qr(torch.randn(192, 96, generator=g, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(320, 96, generator=g, dtype=torch.float64))
    s = torch.linspace(1.0, 0.05, 96, dtype=torch.float64)
    x = (u * s) @ v.t()
    a, b, c = COEFFICIENTS
    t = s / s.norm()
    sizes = []
    for _ in range(5):
        sizes.append(t.norm())
        t = a * t + b * t ** 3 + c * t ** 5
    o = K.orthogonalize(x.float().cuda()).double().cpu()
    # Half of the directions are empty, and what rounding puts there grows: rounding X_k to fp16 is off by at most 2^-11 of its norm,
    # and a step multiplies a difference by at most the largest |p'| (3.9 at s = 1.2, 3.4 at 0).  The first step's rounding alone may
    # so be 2^-11 * 3.9^5 / |t| = 5 % of the result; 1.1 % was measured.
    r = torch.linspace(0, 1.2, 1001, dtype=torch.float64)
    grow = (a + 3 * b * r ** 2 + 5 * c * r ** 4).abs().max()
    limit = sum(2.0 ** -11 * n * grow ** (5 - k) for k, n in enumerate(sizes)) + 2.0 ** -8 * t.norm()
    assert (o - (u * t) @ v.t()).norm() < limit
    check(o.bfloat16().cuda(), x.float().cuda())
    kept = torch.linalg.svdvals(o)
    assert kept[:96].min() > 0.6 and kept[0] < 1.25


@gpu
def test_scales_and_special_values():
    x = matrices(4, 48, 80, seed=5)
    x[1] = 0.0
    x[2, 7, 9] = float("inf")
    x[3, 1, 1] = float("nan")
    o = K.orthogonalize(x)
    check(o[:1], x[:1])
    assert bool((o[1] == 0).all()) and bool(torch.isnan(o[2]).all()) and bool(torch.isnan(o[3]).all())
    for f in (1e12, 1e-3):
        check(K.orthogonalize(x[:1] * f), x[:1] * f)
    tiny = torch.zeros(1, 40, 60, device="cuda")
    tiny[0, 3, 5] = 1.0                                            # all of the norm in one entry
    check(K.orthogonalize(tiny), tiny)
    assert bool(torch.isnan(K.orthogonalize(x[:1] * 1e30)).all())  # squares beyond fp32 are not answered with zeros


@gpu
def test_views_and_empty():
    base = matrices(1, 150, 260, seed=6)[0]
    for x in (base.t(), base[3:, 5:200], base[::2], base[:, 1:2]):
        check(K.orthogonalize(x), x)
    flat = torch.zeros(40 * 56 + 3, device="cuda")
    x = flat[3:].view(40, 56)                                      # starts on no 16-byte boundary
    x.copy_(base[:40, :56])
    check(K.orthogonalize(x), x)
    assert K.orthogonalize(base[:0]).shape == (0, 260)


def muon_exact(p, g, m, master, lr, momentum, wd, scale, nesterov, gs):
    g, m, master = (t.double() for t in (g, m, master))
    mm = momentum * m + gs * g
    return mm, (gs * g + momentum * mm if nesterov else mm), master * (1 - lr * wd)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("size", [(1, 3), (40, 56), (130, 67), (67, 131), (512, 384), (300, 1000), (600, 136)])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("clip", [None, 0.37])
def test_muon_step(device, size, nesterov, clip):
    g, m, master = matrices(3, *size, device, seed=7).unbind(0)
    g, m, master = g.clone(), m.clone(), (20 * master).clone()
    p = master.bfloat16()
    lr, beta, wd, scale = 2e-2, 0.9, 0.1, 1.7
    gst = None if clip is None else torch.tensor([clip], device=device)
    gs = 1.0 if clip is None else gst.double().item()
    want_m, u, kept = muon_exact(p, g, m, master, lr, beta, wd, scale, nesterov, gs)
    g0 = g.clone()
    o = K.muon_step(p, g, m, master, lr, beta, wd, scale, nesterov, grad_scale_tensor=gst)
    assert torch.equal(g, g0)
    check(o, u)
    step = 2.0 ** -24
    assert bool(((m.double() - want_m).abs() <= 4 * step * ((beta * want_m).abs() + (gs * g).abs().double() + 1e-12)).all())
    want = kept - lr * scale * o.double()
    assert bool(((master.double() - want).abs() <= 6 * step * (kept.abs() + (lr * scale * o.double()).abs() + 1e-12)).all())
    assert torch.equal(p, master.bfloat16())


@gpu
@pytest.mark.parametrize("size", [(1300, 2600), (2600, 1304), (130, 9000)])
def test_large_muon_step(size):
    """Updates in the last product's epilogue, over several tiles and both forms of the iteration; weights that are views."""
    g, m = matrices(2, *size, seed=12).unbind(0)
    g, m = g.clone(), m.clone()
    for offset in (0, 4, 3):                                       # 3: no 16-byte boundary, a kernel of its own
        flat = torch.full((size[0] * size[1] + 8,), 5.0, device="cuda")
        master = flat[offset:offset + size[0] * size[1]].view(size)
        master.copy_(matrices(1, *size, seed=13, std=0.02)[0])
        before = master.double()
        p = torch.zeros(size, dtype=torch.bfloat16, device="cuda")
        mm = m.clone()
        o = K.muon_step(p, g, mm, master, 1e-2, 0.9, 0.1, 1.5)
        check(o, g.double() + 0.9 * (0.9 * m.double() + g.double()))
        want = before * (1 - 1e-3) - 1.5e-2 * o.double()
        assert bool(((master.double() - want).abs() <= 6 * 2.0 ** -24 * (before.abs() + (1.5e-2 * o.double()).abs() + 1e-12)).all())
        assert torch.equal(p, master.bfloat16())
        assert bool((flat[:offset] == 5).all()) and bool((flat[offset + size[0] * size[1]:] == 5).all())


@gpu
def test_default_scale_and_many_steps():
    g = matrices(1, 96, 160, seed=8)[0]
    m, master = torch.zeros_like(g), matrices(1, 96, 160, seed=9, std=0.02)[0].clone()
    p = master.bfloat16()
    before = master.clone()
    o = K.muon_step(p, g, m, master, lr=1e-2)
    rms = (master - before).square().mean().sqrt().item()
    assert abs(rms - 1e-2 * 0.2 * 160 ** 0.5 * o.float().square().mean().sqrt().item()) < 1e-5 * rms + 1e-6
    for _ in range(3):
        K.muon_step(p, g, m, master, lr=1e-2, weight_decay=0.1)
    assert torch.isfinite(master).all() and torch.equal(p, master.bfloat16())


@gpu
def test_streams_and_capture():
    x = matrices(2, 300, 200, seed=10)
    want = K.orthogonalize(x)
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            outs += [K.orthogonalize(x) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    y = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = K.orthogonalize(y)
    for seed in (11, 12):
        y.copy_(matrices(2, 300, 200, seed=seed))
        graph.replay()
        assert torch.equal(o, K.orthogonalize(y))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    x = matrices(1, 8, 12, device)
    with pytest.raises(KernelError, match="matrices"):
        K.orthogonalize(x[0, 0])
    with pytest.raises(KernelError, match="matrices"):
        K.orthogonalize(x.int())
    with pytest.raises(KernelError, match="one step"):
        K.orthogonalize(x, steps=0)
    with pytest.raises(KernelError, match="coefficients"):
        K.orthogonalize(x, coefficients=(1.0, float("nan"), 0.0))
    with pytest.raises(KernelError, match="eps"):
        K.orthogonalize(x, eps=-1.0)
    g = x[0].clone()
    with pytest.raises(KernelError, match="one shape"):
        K.muon_step(g.bfloat16(), g, g[:4].clone(), g.clone(), lr=1e-3)
    with pytest.raises(KernelError, match="one matrix"):
        K.muon_step(x.bfloat16(), x, x.clone(), x.clone(), lr=1e-3)


def test_scale_of_the_iterates():
    assert fp16_scales(5, COEFFICIENTS) == (2.0 ** 14, 2.0 ** 10)          # three first steps: up to 3.4445^3 = 41
    assert fp16_scales(1, (6.0, -4.0, 2.0))[0] == 2.0 ** 13
    with pytest.raises(KernelError, match="without bound"):
        fp16_scales(5, (5.0, 4.0, 3.0))


@gpu
def test_gpu_refusals():
    g = matrices(1, 8, 12)[0].clone()
    with pytest.raises(KernelError, match="without bound"):
        K.orthogonalize(g, coefficients=(5.0, 4.0, 3.0))
    with pytest.raises(KernelError, match="fp32"):
        K.muon_step(g.bfloat16(), g, g.bfloat16(), g.clone(), lr=1e-3)
    with pytest.raises(KernelError, match="contiguous"):
        K.muon_step(g.bfloat16(), g, torch.zeros(12, 8, device="cuda").t(), g.clone(), lr=1e-3)
    with pytest.raises(KernelError, match="factor"):
        K.muon_step(g.bfloat16(), g, g.clone(), g.clone(), lr=1e-3, grad_scale_tensor=torch.ones(2, device="cuda"))
    with pytest.raises(KernelError, match="devices"):
        K.muon_step(g.bfloat16(), g, g.cpu(), g.clone(), lr=1e-3)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_smallest_eps(device):
    """Squares of entries below 1e-19 are no fp32 numbers, so the norm of a matrix of them reads 0: it must not count beside eps."""
    x = matrices(1, 24, 40, device, seed=15)
    for eps in (0.0, 1e-30, float("inf"), float("nan")):
        with pytest.raises(KernelError, match="eps"):
            K.orthogonalize(x, eps=eps)
    # Entries of 1e-21 leave X at 1e-9 and, times 2^14, among fp16's subnormal numbers: off by 2^-25 of 5e-5 for the largest, a third
    # of that again in each step that takes X to 3.4 times itself, 1e-3 in all; 2^-8 is the result's rounding.  Together below 2^-7.
    for f in (1e-18, 1e-9):
        y = (x * f).float()
        o = K.orthogonalize(y, eps=1e-12)
        exact = iterate(y, eps=1e-12)
        assert torch.isfinite(o).all() and bool((o.double() - exact).abs().max() <= 2.0 ** -7 * exact.abs().max())


@gpu
def test_gradient_type():
    """A bf16 weight on the GPU has an fp32 gradient; no other one is taken through plain PyTorch instead."""
    g = matrices(1, 8, 12)[0].clone()
    for t in (torch.bfloat16, torch.float64):
        with pytest.raises(KernelError, match="fp32"):
            K.muon_step(g.bfloat16(), g.to(t), g.clone(), g.clone(), lr=1e-3)


def test_scales_under_another_default_device():
    want = fp16_scales(5, COEFFICIENTS)
    fp16_scales.cache_clear()
    with torch.device("meta"):
        assert fp16_scales(5, COEFFICIENTS) == want
