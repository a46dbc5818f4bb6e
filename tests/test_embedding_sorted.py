"""Embedding lookup with a scale and its gradient by sorted tokens, against plain statements in 64 bits.

A looked-up value is one product in fp32 (2^-24) rounded to bf16 (2^-8).  The gradient of a row is a sum of n rows in fp32, each
addition off by at most 2^-24 of the sum of their sizes, times the scale, plus the addition to what was there."""
import pytest
import torch

from kareus_b200 import kernels as K
from kareus_b200.kernels.cuda import KernelError, lib

gpu = pytest.mark.gpu


def reference(tokens, weight, dout, grad, start, scale):
    """(out, grad, number of tokens of each row, sum of the sizes) in 64 bits."""
    v, H = weight.shape
    ids = (tokens.reshape(-1) - start)
    keep = torch.nonzero((ids >= 0) & (ids < v)).flatten()
    out = torch.zeros(ids.numel(), H, dtype=torch.float64, device=weight.device)
    out[keep] = weight.double()[ids[keep]] * scale
    d = dout.reshape(-1, H).double()[keep] * scale
    g, size = grad.double(), grad.double().abs()
    g.index_put_((ids[keep],), d, accumulate=True)
    size.index_put_((ids[keep],), d.abs(), accumulate=True)
    n = torch.bincount(ids[keep], minlength=v)
    return out.view(tuple(tokens.shape) + (H,)), g, n, size


def check(tokens, weight, start, scale, seed=1):
    gen = torch.Generator().manual_seed(seed)
    H = weight.shape[1]
    dout = torch.randn(tuple(tokens.shape) + (H,), generator=gen).bfloat16().to(weight.device)
    grad = torch.randn(weight.shape, generator=gen).to(weight.device)
    out, want, n, size = reference(tokens, weight, dout, grad, start, scale)
    got = K.embedding_fwd(tokens, weight, start, scale=scale)
    assert got.dtype == weight.dtype and bool(((got.double() - out).abs() <= 2.0 ** -8 * 1.0001 * out.abs()).all())
    runs = []
    for _ in range(2):
        g = grad.clone()
        assert K.embedding_bwd(dout, tokens, g, start, scale=scale, order="sorted") is g
        runs.append(g)
    assert torch.equal(*runs)                                      # the same bits every time
    limit = 2.0 ** -24 * (n[:, None].double() + 3) * size
    off = ((runs[0].double() - want).abs() - limit).max().item()
    assert off <= 0, off
    assert torch.equal(runs[0][n == 0], grad[n == 0])              # rows without tokens as they were


def table(v, H, device="cuda", seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(v, H, generator=g).bfloat16().to(device)


def draw(n, total, skew=1.0, seed=2, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return ((torch.rand(n, generator=g, dtype=torch.float64) ** skew) * total).long().to(device)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("n, v, H", [(1, 1, 8), (1, 5, 1), (7, 3, 24), (64, 10, 136), (33, 100, 64)])
@pytest.mark.parametrize("scale", [1.0, 64.0, 1.3])
def test_small(device, n, v, H, scale):
    check(draw(n, v, device=device), table(v, H, device), 0, scale)
    check(draw(n, 3 * v, device=device).view(1, n, 1), table(v, H, device), v, scale)      # middle one of three shards


@gpu
@pytest.mark.parametrize("n", [2, 31, 32, 33, 255, 257, 1000, 2047, 2048, 2049, 4097, 8192, 30001, 65536, 65537, 150000])
def test_lengths(n):
    check(draw(n, 500, 2), table(500, 16), 0, 1.0)


@gpu
@pytest.mark.parametrize("v", [1, 2, 255, 256, 257, 511, 65535, 65536, 128256])
def test_vocabularies(v):
    """Every number of digits of the sort, each with keys at both ends."""
    for n in (3000, 900):
        t = draw(n, v, 3)
        t[5], t[6], t[-1] = v - 1, 0, v - 1
        check(t, table(v, 8), 0, 2.0)


@gpu
@pytest.mark.parametrize("H", [1, 7, 8, 72, 520, 1020, 1024, 1032, 2048, 4096])
def test_widths(H):
    check(draw(700, 90), table(90, H), 0, 1.0)
    check(draw(700, 90, seed=4).view(100, 7), table(30, H), 30, 0.5)


@gpu
@pytest.mark.parametrize("n", [63, 64, 65, 128, 700, 5000, 20000])
@pytest.mark.parametrize("share", [0.5, 0.97, 1.0])
def test_one_token_many_times(n, share):
    """Padding: runs that cross windows, fill them, end at their borders."""
    t = draw(n, 40)
    t[: int(n * share)] = 17
    t = t[torch.randperm(n, generator=torch.Generator().manual_seed(3)).to(t.device)]
    check(t, table(40, 264), 0, 1.0)
    check(torch.full((n,), 39, device="cuda"), table(40, 264), 0, 3.0)


@gpu
@pytest.mark.parametrize("H", [7, 24, 136, 520])
def test_long_runs_beside_short_ones(H):
    """Several tokens that fill many windows, one after the other, with tokens of a few rows between them."""
    runs = torch.tensor([3, 900, 1, 70, 2000, 5, 130, 64, 64, 1, 700, 12, 20, 300, 63, 65])
    t = torch.repeat_interleave(torch.arange(16), runs).cuda()
    check(t[torch.randperm(t.numel(), generator=torch.Generator().manual_seed(1)).cuda()], table(16, H), 0, 1.0)


@gpu
def test_runs_of_every_length():
    """Sorted tokens whose runs start and end at every place of a window."""
    runs = torch.arange(1, 200)
    t = torch.repeat_interleave(torch.arange(199), runs).cuda()
    check(t, table(199, 2048), 0, 1.0)
    check(t.flip(0), table(199, 24), 0, 1.0)


@gpu
def test_tokens_of_no_row():
    w = table(50, 64)
    for t in (torch.full((300,), 50), torch.full((300,), -1), torch.tensor([-2 ** 62, 2 ** 62, 49, 0, 2 ** 32 + 3])):
        check(t.cuda(), w, 0, 1.0)
    check(draw(100, 50), w, 2 ** 40, 1.0)


@gpu
def test_offsets_beyond_32_bits():
    """A gradient of more than 2^32 bytes: the last rows of a large table."""
    v, H = 300000, 4096
    t = torch.tensor([v - 1, 5, v - 1, v - 2, 262144], device="cuda")
    dout = torch.randn(5, H, device="cuda").bfloat16()
    grad = torch.zeros(v, H, device="cuda")
    K.embedding_bwd(dout, t, grad, 0, order="sorted")
    d = dout.float()
    for row, want in ((v - 1, d[0] + d[2]), (5, d[1]), (v - 2, d[3]), (262144, d[4])):
        assert torch.equal(grad[row], want)
        grad[row] = 0
    assert not bool(grad.any())


@gpu
def test_views_and_streams():
    base = torch.randn(300, 1, 80, device="cuda").bfloat16()
    t = draw(300, 20).view(300, 1)
    w = table(20, 64)
    g0 = torch.zeros(20, 64, device="cuda")
    K.embedding_bwd(base[..., 8:72].contiguous(), t, g0, 0, order="sorted")
    g1 = torch.zeros(20, 64, device="cuda")
    K.embedding_bwd(base[..., 8:72], t, g1, 0, order="sorted")     # a strided gradient
    assert torch.equal(g0, g1)
    flat = torch.zeros(20 * 64 + 1, device="cuda")
    g2 = flat[1:].view(20, 64)                                     # a gradient that starts on no 16-byte boundary
    K.embedding_bwd(base[..., 8:72], t, g2, 0, order="sorted")
    assert torch.equal(g0, g2) and flat[0].item() == 0
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            g = torch.zeros(20, 64, device="cuda")
            K.embedding_bwd(base[..., 8:72].contiguous(), t, g, 0, order="sorted")
            outs.append(g)
    torch.cuda.synchronize()
    assert all(torch.equal(g, g0) for g in outs)
    grad, d, tok = torch.zeros(20, 64, device="cuda"), base[..., 8:72].contiguous(), t.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.embedding_bwd(d, tok, grad, 0, order="sorted")
    for seed in (5, 6):
        tok.copy_(draw(300, 20, seed=seed).view(300, 1))
        grad.zero_()
        graph.replay()
        want = torch.zeros(20, 64, device="cuda")
        K.embedding_bwd(d, tok, want, 0, order="sorted")
        assert torch.equal(grad, want)


@gpu
def test_not_finite():
    t = torch.tensor([3, 4, 3, 9], device="cuda")
    d = torch.ones(4, 16, device="cuda").bfloat16()
    d[2, 5], d[1, 0], d[3, 2] = float("inf"), float("nan"), float("nan")
    g = torch.zeros(9, 16, device="cuda")
    K.embedding_bwd(d, t, g, 0, order="sorted")                    # the last token belongs to another shard
    assert g[3, 5].isinf() and g[4, 0].isnan() and torch.isfinite(g).sum() == 9 * 16 - 2


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_gradient_is_that_of_the_lookup(device):
    """<dout, lookup(W + E) - lookup(W)> = <gradient, E>: the lookup is linear in its table."""
    t = draw(200, 30, device=device)
    dout, e = table(200, 24, device, 3), table(20, 24, device, 4)
    g = torch.zeros(20, 24, device=device)
    K.embedding_bwd(dout, t, g, 5, scale=2.0, order="sorted")
    left = (dout.double() * K.embedding_fwd(t, e, 5, scale=2.0).double()).sum()        # times 2 is exact in bf16
    assert (left - (g.double() * e.double()).sum()).abs() < 1e-5 * left.abs() + 1e-3


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_empty_and_refusals(device):
    w, g = table(10, 16, device), torch.zeros(10, 16, device=device)
    none = torch.empty(0, dtype=torch.int64, device=device)
    assert tuple(K.embedding_fwd(none, w, 0, scale=2.0).shape) == (0, 16)
    K.embedding_bwd(torch.empty(0, 16, dtype=torch.bfloat16, device=device), none, g, 0, order="sorted")
    assert not bool(g.any())
    with pytest.raises((KernelError, ValueError), match="order"):
        K.embedding_bwd(w[:3].contiguous(), torch.zeros(3, dtype=torch.int64, device=device), g, 0, order="random")


@gpu
def test_gpu_refusals():
    w, g = table(10, 16), torch.zeros(10, 16, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(KernelError, match="int64"):
        K.embedding_fwd(t.int(), w, 0, scale=2.0)
    with pytest.raises(KernelError, match="gradient of shape"):
        K.embedding_bwd(w[:2].contiguous(), t, g, 0, order="sorted")
    with pytest.raises(KernelError, match="contiguous"):
        K.embedding_bwd(w[:3].contiguous(), t, torch.zeros(16, 10, device="cuda").t(), 0, order="sorted")
    with pytest.raises(KernelError, match="current device"):
        K.embedding_fwd(t.cpu(), w, 0, scale=2.0)


def test_widest_table():
    """A table whose columns the last kernel's grid does not reach is refused before the first one has added to it."""
    assert lib().kb_embedding_bwd_sorted(16, 16, 16, 4, 65535 * 128 + 1, 0, 4, 1.0, 256, 0) == 7


@gpu
@pytest.mark.parametrize("n", [1, 2, 3, 127, 128, 129, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 65535, 65537])
@pytest.mark.parametrize("v", [1, 40, 100000])
def test_borders_of_the_sorts(n, v):
    """Batches at the sizes where the way of sorting, or of counting, changes; few tokens and many, half of them another shard's."""
    check(draw(n, v, seed=6), table(v, 24), 0, 1.0)
    check(draw(n, 2 * v, seed=7), table(v, 24), v, 1.0)


@gpu
@pytest.mark.parametrize("H", [1000, 4104, 8191, 20000])
@pytest.mark.parametrize("n", [5, 9, 300, 1024])
def test_few_tokens_of_wide_rows(n, H):
    """Short runs and long ones, whose columns are spread over the blocks of their tokens."""
    t = draw(n, 60, seed=8)
    t[: n // 2] = 7
    t = t[torch.randperm(n, generator=torch.Generator().manual_seed(4)).to(t.device)]
    check(t, table(40, H), 0, 1.0)
    check(torch.full((n,), 3, device="cuda"), table(9, H), 2, 0.5)


@gpu
def test_launches_are_counted():
    from kareus_b200.kernels import launch_count
    g = torch.zeros(9, 16, device="cuda")
    for n, launches in ((1024, 1), (1025, 3), (65536, 3), (65537, 4)):
        d, t = torch.zeros(n, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda")
        for _ in range(2):                                         # the first call goes through the Python statements
            before = launch_count()
            K.embedding_bwd(d, t, g, 0, order="sorted")
            assert launch_count() - before == launches


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_statements_repeat_bit_for_bit(device, dtype):
    """Also where PyTorch computes it: on the CPU, and fp32 gradients on the GPU.  Enough elements for several threads."""
    t, d = draw(4000, 3, device=device), table(4000, 64, device).to(dtype)
    runs = []
    for _ in range(8):
        g = torch.zeros(3, 64, device=device)
        K.embedding_bwd(d, t, g, 0, scale=1.3, order="sorted")
        runs.append(g)
    assert all(torch.equal(r, runs[0]) for r in runs)


#: one length for each way a batch is taken: in one kernel, sorted by counting, by the radix sort, in two chunks
PATHS = [300, 3000, 5000, 70000]


@gpu
@pytest.mark.parametrize("n", [1100, 4096, 4097, 20000])
@pytest.mark.parametrize("v", [1, 2, 3, 511, 512, 513, 2 ** 17, 2 ** 18 - 1, 2 ** 18, 2 ** 18 + 1])
def test_digits_of_the_radix_sort(n, v):
    """Tables at the borders of one, two and three digits, with keys at both ends, beyond 4096 tokens and below."""
    t = draw(n, v, 3)
    t[5], t[6], t[-1] = v - 1, 0, v - 1
    check(t, table(v, 8), 0, 2.0)
    check(t + v // 2, table(v, 8), 0, 1.0)                         # half of the keys are another shard's


@gpu
def test_four_digits():
    """More than 2^27 rows.  Whole numbers whose sums fp32 holds."""
    v, n = 2 ** 27 + 3, 6000
    t = draw(n, v)
    t[:50], t[50:99] = v - 1, 2 ** 27 - 1
    d = torch.randint(-8, 9, (n, 1), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    grad = torch.zeros(v, 1, device="cuda")
    K.embedding_bwd(d, t, grad, 0, order="sorted")
    rows, inverse = torch.unique(t, return_inverse=True)
    want = torch.zeros(rows.numel(), 1, device="cuda").index_add_(0, inverse, d.float())
    assert torch.equal(grad[rows], want)
    grad[rows] = 0
    assert not bool(grad.any())


@gpu
@pytest.mark.parametrize("n", PATHS[:3])
@pytest.mark.parametrize("H", [1, 7, 136, 1020, 1024, 1032, 2056, 4096])
def test_widths_of_every_path(n, H):
    """One block of columns in the sums and the join, several, a last one of few columns; rows that start on 16 bytes and not."""
    check(draw(n, 90, 2), table(90, H), 0, 1.0)
    check(draw(n, 90, seed=4).view(n // 100, 100), table(30, H), 30, 0.5)


@gpu
@pytest.mark.parametrize("n", PATHS)
def test_tokens_of_no_row_in_every_path(n):
    w = table(50, 64)
    far = draw(n, 50)
    far[::2] += torch.tensor(2 ** 32)
    far[1::4] = -2 ** 62
    far[3::8] = 2 ** 62
    for t in (torch.full((n,), 50), torch.full((n,), -1), far):
        check(t.cuda(), w, 0, 1.0)
    check(draw(n, 50), w, 2 ** 40, 1.0)


@gpu
@pytest.mark.parametrize("n", PATHS)
def test_not_finite_in_every_path(n):
    t, d = draw(n, 9), torch.ones(n, 24, device="cuda").bfloat16()
    t[0], t[-1], t[n // 2] = 3, 4, 9
    d[0, 5], d[-1, 0], d[n // 2, 2] = float("inf"), float("nan"), float("nan")
    g = torch.zeros(9, 24, device="cuda")
    K.embedding_bwd(d, t, g, 0, order="sorted")                    # token 9 belongs to another shard
    assert g[3, 5].isinf() and g[4, 0].isnan() and torch.isfinite(g).sum() == 9 * 24 - 2
    count = torch.bincount(t, minlength=10)[:9].float()
    assert torch.equal(g[:, 8], count)                             # sums of ones, 2^24 at most


@gpu
@pytest.mark.parametrize("n", PATHS)
def test_views_streams_and_graphs_of_every_path(n):
    """Strided and unaligned gradients, two streams at once (each call has a workspace of its own), two captured graphs that share a
    pool and take new tokens: the bits of a plain call.  Sums are of whole numbers, which fp32 holds in any order."""
    H = 72
    whole = torch.randint(-4, 5, (n, H + 16), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    d, t = whole[:, 8:8 + H].contiguous(), draw(n, 40, 3)

    def want(t):
        return torch.zeros(40, H, device="cuda", dtype=torch.float64).index_add_(0, t, d.double()).float()

    zeros = lambda: torch.zeros(40, H, device="cuda")
    g = zeros()
    K.embedding_bwd(whole[:, 8:8 + H], t, g, 0, order="sorted")
    assert torch.equal(g, want(t))
    flat = torch.zeros(40 * H + 2, device="cuda")
    K.embedding_bwd(d, t, flat[1:-1].view(40, H), 0, order="sorted")
    assert torch.equal(flat[1:-1].view(40, H), want(t)) and flat[0].item() == flat[-1].item() == 0
    tokens = [draw(n, 40, 3, seed=s) for s in (5, 6)]
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [zeros(), zeros()]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, tok, out in zip(streams, tokens, outs):
            with torch.cuda.stream(s):
                out.zero_()
                K.embedding_bwd(d, tok, out, 0, order="sorted")
    torch.cuda.synchronize()
    assert all(torch.equal(out, want(tok)) for tok, out in zip(tokens, outs))
    graphs, pool = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], None
    for graph, tok, out in zip(graphs, tokens, outs):
        with torch.cuda.graph(graph, pool=pool):
            out.zero_()
            K.embedding_bwd(d, tok, out, 0, order="sorted")
        pool = graph.pool()
    for seed in (7, 8):
        for i, tok in enumerate(tokens):
            tok.copy_(draw(n, 40, 3, seed=seed + 10 * i))
        for graph in (graphs[1], graphs[0], graphs[1]):
            graph.replay()
        assert all(torch.equal(out, want(tok)) for tok, out in zip(tokens, outs))


@gpu
@pytest.mark.parametrize("n", PATHS[1:3])
def test_rows_beyond_32_bits_of_every_path(n):
    """The last rows of a gradient of more than 2^32 bytes, one token on many of them."""
    v, H = 300000, 4096
    t = v - 1 - draw(n, 200, 2)
    t[::7] = v - 1
    d = torch.randint(-4, 5, (n, H), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    grad = torch.zeros(v, H, device="cuda")
    K.embedding_bwd(d, t, grad, 0, order="sorted")
    want = torch.zeros(200, H, device="cuda", dtype=torch.float64).index_add_(0, t - (v - 200), d.double())
    assert torch.equal(grad[v - 200:], want.float())
    assert not bool(grad[:v - 200].any())
    w = torch.zeros(v, H, dtype=torch.bfloat16, device="cuda")
    w[v - 200:] = d[:200]
    assert torch.equal(K.embedding_fwd(t, w, 0), d[t - (v - 200)])


@gpu
def test_batches_beyond_32_bits():
    """Output and gradient of more than 2^32 bytes, chunk after chunk."""
    n, H = 2 ** 19 + 20000, 4096
    t = draw(n, 3000)
    d = torch.zeros(n, H, dtype=torch.bfloat16, device="cuda")
    d[-30000:] = torch.randint(-4, 5, (30000, H), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    grad = torch.zeros(2000, H, device="cuda")
    K.embedding_bwd(d, t, grad, 1000, order="sorted")              # a shard of the middle
    want = torch.zeros(3000, H, device="cuda", dtype=torch.float64).index_add_(0, t[-30000:], d[-30000:].double())
    assert torch.equal(grad, want[1000:].float())
    w = table(2000, H)
    out = K.embedding_fwd(t, w, 1000)
    at = t[-30000:] - 1000
    inside = (at >= 0) & (at < 2000)
    assert torch.equal(out[-30000:], w[at.clamp(0, 1999)] * inside[:, None])
