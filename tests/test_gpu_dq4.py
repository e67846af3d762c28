"""GPU tests of the linear with 4-bit weights (ltxb_dq4_gemm) against float64.

Tolerances. Few rows: exact products, f32 sums, one output rounding: at most
2^-8 |want|, plus f32 accumulation, far below 2^-16 of sum |x w|. More than 16
rows: the weights are rounded to bf16 first, 2^-8 each, so the sum is off by at most
2^-8 sum |x w| more; where the roundings are independent that is a root mean
square of 2^-8 |x| |w| (2-norms), and six of those bound every element here."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [(1, 32, 128), (1, 4096, 4096), (2, 96, 1280), (7, 160, 128), (8, 64, 2176), (9, 288, 640), (16, 1024, 4096),
         (17, 32, 384), (33, 512, 1024), (64, 96, 512), (65, 96, 512), (130, 1056, 896), (300, 512, 4096)]


def weights(n, k, group, scale_dtype, seed, device):
    import ltxb
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(n, k, generator=g) * 0.02 * torch.exp(torch.randn(n, 1, generator=g))
    return ltxb.quantize_g4(w.to(device), group, scale_dtype)


def exact(a, wq, scales, bias=None):
    """(result, sum |x w|, 2-norm of x w) in f64"""
    code = torch.stack((wq & 15, wq >> 4), -1).flatten(-2).double().cpu() - 8
    w = code * scales.double().cpu().repeat_interleave(code.shape[1] // scales.shape[1], 1)
    x = a.double().cpu()
    y = x @ w.T + (0 if bias is None else bias.double().cpu())
    return y, x.abs() @ w.abs().T, (x ** 2 @ (w ** 2).T).sqrt()


def check(got, a, wq, scales, bias=None):
    want, total, norm = exact(a, wq, scales, bias)
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -16 * total
    if a.shape[0] > 16:
        bound += 6 * 2.0 ** -8 * norm
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("group,scale_dtype", [(128, torch.bfloat16), (64, torch.float32), (32, torch.bfloat16)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_dq4_gemm(cuda, M, N, K, group, scale_dtype):
    import ltxb
    wq, s = weights(N, K, group, scale_dtype, M + N, cuda)
    g = torch.Generator().manual_seed(M)
    a = torch.randn(M, K, generator=g).to(torch.bfloat16).to(cuda)
    bias = torch.randn(N, generator=g).to(torch.bfloat16).to(cuda)
    check(ltxb.dq4_gemm(a, wq, s), a, wq, s)
    check(ltxb.dq4_gemm(a, wq, s, bias=bias), a, wq, s, bias)
    assert ltxb.device_status() == ltxb.OK


# Each side of the borders between the three ways: rows in one and several
# chunks, weight rows and columns with a remainder, K split over a cluster.
BORDERS = [(16, 160, 640), (17, 160, 640), (48, 4096, 8320), (255, 32, 2176), (256, 384, 1152), (257, 160, 128),
           (700, 288, 16512), (1024, 96, 512), (1025, 96, 512)]


@pytest.mark.parametrize("group,scale_dtype", [(128, torch.float32), (64, torch.bfloat16), (32, torch.float32),
                                               (32, torch.bfloat16)])
@pytest.mark.parametrize("M,N,K", BORDERS)
def test_borders_between_the_kernels(cuda, M, N, K, group, scale_dtype):
    import ltxb
    wq, s = weights(N, K, group, scale_dtype, M, cuda)
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(cuda)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(N)).to(torch.bfloat16).to(cuda)
    guard = torch.full((M + 2, N), 7.0, dtype=torch.bfloat16, device=cuda)
    out = ltxb.dq4_gemm(a, wq, s, bias=bias, out=guard[1:M + 1])
    check(out, a, wq, s, bias)
    assert bool((guard[0] == 7).all()) and bool((guard[M + 1] == 7).all())
    assert torch.equal(out, ltxb.dq4_gemm(a, wq, s, bias=bias))
    assert ltxb.device_status() == ltxb.OK


def test_all_codes_and_an_offset_input(cuda):
    """Every code in every place of a word, and rows of A with a large common offset (the part the accumulator starts from)."""
    import ltxb
    N, K = 32, 256
    n, k = torch.meshgrid(torch.arange(N), torch.arange(K), indexing="ij")
    code = ((n * 7 + k * 5 + k // 16) % 16).to(torch.uint8)
    wq = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous().to(cuda)
    for group in (32, 64, 128):
        s = (torch.rand(N, K // group, generator=torch.Generator().manual_seed(group)) + 0.5).to(cuda)
        for m in (1, 5, 100):
            a = (torch.randn(m, K, generator=torch.Generator().manual_seed(m)) + 30).to(torch.bfloat16).to(cuda)
            check(ltxb.dq4_gemm(a, wq, s), a, wq, s)


def test_rows_do_not_depend_on_their_neighbours(cuda):
    """NaN and infinity in one row of A stay in that row; a NaN scale stays in its output column."""
    import ltxb
    wq, s = weights(64, 512, 64, torch.float32, 1, cuda)
    a = torch.randn(12, 512, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(cuda)
    clean = ltxb.dq4_gemm(a, wq, s)
    b = a.clone()
    b[3, 100] = float("nan")
    b[5, 7] = float("inf")
    t = s.clone()
    t[20, 2] = float("nan")
    many = ltxb.dq4_gemm(b.repeat(3, 1), wq, t)  # 36 rows: the tcgen05 kernel
    plain = ltxb.dq4_gemm(a.repeat(3, 1), wq, s)
    out = ltxb.dq4_gemm(b, wq, t)
    rows = [r for r in range(12) if r not in (3, 5)]
    cols = [c for c in range(64) if c != 20]
    assert torch.equal(out[rows][:, cols], clean[rows][:, cols])
    keep = [r for r in range(36) if r % 12 not in (3, 5)]
    assert torch.equal(many[keep][:, cols], plain[keep][:, cols]) and bool(many[:, 20].isnan().all())
    assert bool(many[3].isnan().all()) and not bool(many[5].isfinite().any())
    assert bool(out[3].isnan().all()) and not bool(out[5].isfinite().any()) and bool(out[:, 20].isnan().all())


def test_quantize_g4(cuda):
    import ltxb
    w = torch.randn(64, 256, generator=torch.Generator().manual_seed(0)).to(cuda)
    w[3, :32] = 0
    for group in (32, 64, 128):
        wq, s = ltxb.quantize_g4(w, group, torch.float32)
        code = torch.stack((wq & 15, wq >> 4), -1).flatten(-2).float() - 8
        back = code * s.repeat_interleave(group, 1)
        # half a step, and the f32 rounding of the quotient
        assert bool(((back - w).abs() <= s.repeat_interleave(group, 1) * 0.5001).all())
    with pytest.raises(ltxb.LtxbError):
        ltxb.quantize_g4(w, 48)


def test_refusals(cuda):
    import ltxb
    wq, s = weights(64, 256, 64, torch.float32, 1, cuda)
    a = torch.zeros(2, 256, dtype=torch.bfloat16, device=cuda)
    n0 = ltxb.launch_count()
    for f in (lambda: ltxb.dq4_gemm(a.float(), wq, s), lambda: ltxb.dq4_gemm(a, wq.to(torch.int8), s),
              lambda: ltxb.dq4_gemm(a, wq[:, :64], s), lambda: ltxb.dq4_gemm(a, wq, s[:32]),
              lambda: ltxb.dq4_gemm(a, wq, s[:, :3].contiguous()), lambda: ltxb.dq4_gemm(a, wq, s[:, :1].contiguous()),
              lambda: ltxb.dq4_gemm(a, wq[:48], s[:48]), lambda: ltxb.dq4_gemm(a, wq, s, bias=s[:, 0]),
              lambda: ltxb.dq4_gemm(a, wq.cpu(), s), lambda: ltxb.dq4_gemm(a, wq, s, out=a),
              lambda: ltxb.dq4_gemm(a.repeat(8, 1), wq, s, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))):
        with pytest.raises(ltxb.LtxbError):
            f()
    assert ltxb.launch_count() == n0
    assert ltxb.dq4_gemm(a[:0], wq, s).shape == (0, 64)


def test_captured_and_replayed(cuda):
    import ltxb
    wq, s = weights(256, 512, 32, torch.bfloat16, 1, cuda)
    for m in (3, 80):
        a = torch.zeros(m, 512, dtype=torch.bfloat16, device=cuda)
        out = torch.empty(m, 256, dtype=torch.bfloat16, device=cuda)
        ltxb.dq4_gemm(a, wq, s, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ltxb.dq4_gemm(a, wq, s, out=out)
        a.copy_(torch.randn(m, 512, generator=torch.Generator().manual_seed(m)).to(torch.bfloat16))
        graph.replay()
        check(out, a, wq, s)


@pytest.mark.parametrize("M,N,K", [(1, 64, 65536), (2, 37024, 256), (12, 224, 8320), (64, 32, 32768), (3, 128, 128)])
def test_long_and_short_columns(cuda, M, N, K):
    """Rows that the kernel puts in order itself and rows that it does not; K split over a cluster with a remainder."""
    import ltxb
    wq, s = weights(N, K, 64, torch.bfloat16, 5, cuda)
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(cuda)
    out = ltxb.dq4_gemm(a, wq, s)
    check(out, a, wq, s)
    assert torch.equal(out, ltxb.dq4_gemm(a, wq, s))


def test_rows_of_unequal_size(cuda):
    """Rows and columns of A over many powers of two, up to bf16's ends."""
    import ltxb
    wq, s = weights(64, 1024, 32, torch.float32, 1, cuda)
    a = torch.randn(9, 1024, generator=torch.Generator().manual_seed(0))
    a *= torch.exp2(torch.linspace(-100, 100, 9))[:, None]
    a[4] *= torch.exp2(torch.linspace(-30, 30, 1024))
    a = a.to(torch.bfloat16).to(cuda)
    check(ltxb.dq4_gemm(a, wq, s), a, wq, s)
    check(ltxb.dq4_gemm(a[:1], wq, s), a[:1], wq, s)
    check(ltxb.dq4_gemm(a[8:], wq, s), a[8:], wq, s)


def test_captured_with_its_operand_kernel(cuda):
    """12 rows: two kernels, the second starting under the first; replayed on new rows, two streams at once."""
    import ltxb
    wq, s = weights(512, 4096, 128, torch.bfloat16, 1, cuda)
    a = torch.zeros(12, 4096, dtype=torch.bfloat16, device=cuda)
    out = torch.empty(12, 512, dtype=torch.bfloat16, device=cuda)
    ltxb.dq4_gemm(a, wq, s, out=out)
    graphs, outs = [], []
    for _ in range(2):
        o = torch.empty_like(out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ltxb.dq4_gemm(a, wq, s, out=o)
        graphs.append(graph)
        outs.append(o)
    st = torch.cuda.Stream()
    for i in range(4):
        a.copy_(torch.randn(12, 4096, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        check(outs[0], a, wq, s)
        assert torch.equal(outs[0], outs[1])


def test_two_streams_at_once(cuda):
    """Calls of the tcgen05 kernel side by side, with K split over clusters and without."""
    import ltxb
    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs, alone = [], []
    for i, (m, n, k) in enumerate(((40, 2048, 8192), (200, 20480, 1024))):
        wq, s = weights(n, k, 64, torch.bfloat16, i, cuda)
        a = torch.randn(m, k, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(cuda)
        jobs.append((a, wq, s))
        alone.append(ltxb.dq4_gemm(a, wq, s))
        check(alone[i], a, wq, s)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            got[i].append(ltxb.dq4_gemm(*jobs[i], stream=st))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in got[i])
    assert ltxb.device_status() == ltxb.OK
