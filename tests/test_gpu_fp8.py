"""Block-scaled 8-bit linear layers (indextts/utils/fp8.py) against their definition in 64 bits."""
import pytest
import torch

from eightbit_util import codes64, quant64

pytestmark = pytest.mark.gpu


def values(rows, seed=0):
    """rows whose blocks span the whole exponent range, with zeros, denormals and what is not finite among them"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, 512, generator=g)
    x *= torch.exp2(torch.randint(-140, 118, (rows, 4), generator=g).float()).repeat_interleave(128, 1)
    x[0, :128] = 0
    x[1, 5], x[1, 200], x[1, 300] = float("nan"), float("inf"), -float("inf")
    x[2, 128:256] = float("inf")
    x[3, 0] = 3.4028234663852886e38
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [1, 7, 128, 129, 500, 512])
def test_quant_rows_is_exact(dtype, K):
    from indextts.utils.fp8 import quant_rows
    x = values(37)[:, :K].to(dtype)
    q, s = quant_rows(x.cuda())
    kp = -(-K // 128) * 128
    assert q.shape == (37, kp) and s.shape == (37, -(-(kp // 128) // 4) * 4)
    want, e = quant64(torch.nn.functional.pad(x.double(), (0, kp - K)).view(37, -1, 128))
    assert torch.equal(s.cpu()[:, : kp // 128].double() - 127, e)
    assert (s[:, kp // 128:] == 127).all() and (q[:, K:] == 0).all()
    got = codes64(q.cpu().view(37, -1, 128), s.cpu()[:, : kp // 128])
    assert torch.equal(torch.nan_to_num(got, nan=7e77), torch.nan_to_num(want, nan=7e77))


def test_quant_rows_strided():
    from indextts.utils.fp8 import quant_rows
    base = values(9).cuda()
    for x in (base[:, 1:200], base[::2, 3:400], base[:, ::2], base.bfloat16()[:, 8:300], base[1:2, 5:77]):
        q, s = quant_rows(x)
        q2, s2 = quant_rows(x.contiguous().clone())
        assert torch.equal(q, q2) and torch.equal(s, s2)


def oracle(x, w, bias, act, residual, fast):
    """(y, bound on what the accumulation may be off): 64-bit product of the quantised operands"""
    xq, wq = (quant64(torch.nn.functional.pad(t.double(), (0, -t.shape[1] % 128)).view(t.shape[0], -1, 128))[0] for t in (x, w))
    xmax, wmax = xq.abs().amax(-1), wq.abs().amax(-1)
    xq, wq = xq.view(x.shape[0], -1), wq.view(w.shape[0], -1)
    y = xq @ wq.t()
    # every partial sum is within the sum of magnitudes and is rounded, by at most a step (the matrix unit may cut instead of
    # round to nearest), at most once per product
    tol = (xq.abs() @ wq.abs().t()) * (xq.shape[1] + 2) * 2.0 ** -23
    if fast:
        # the 8-bit unit cuts each of a block's 128 products at 2^-13 of the block's largest, by as much and either way: a
        # standard deviation of at most 2^-13 sqrt(128 / 3) of it per block; six of them over all blocks
        tol = tol + 6 * 2.0 ** -13 * (128 / 3) ** 0.5 * (xmax.square() @ wmax.square().t()).sqrt()
    if bias is not None:
        y = y + bias.double()
    tol = tol + y.abs() * 2.0 ** -23
    if act == 1:
        y = torch.nn.functional.gelu(y, approximate="tanh")
    elif act == 2:
        y = torch.nn.functional.silu(y)
    if act:
        tol = tol * 1.2 + 2.0 ** -20 * (y.abs() + 1e-3)  # slopes are at most 1.13; a few f32 steps of tanh / exp
    if residual is not None:
        y = y + residual.double()
        tol = tol + y.abs() * 2.0 ** -24
    return y, tol


def check(got, y, tol):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.to(y.device).double() - y).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol + half * (y.abs() + tol) + 1e-30).all()), float((err / (tol + half * y.abs() + 1e-30)).max())


SIZES = [(1, 1, 1), (1, 64, 32), (1, 1024, 4096), (3, 129, 65), (5, 1000, 130), (16, 128, 64), (17, 300, 100), (33, 4096, 96),
         (64, 512, 256), (96, 1024, 1030), (129, 257, 515), (200, 640, 384), (300, 1024, 512), (515, 384, 777), (1030, 256, 1100)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("form", ["plain", "gelu", "silu", "residual", "bf16"])
def test_linear(M, K, N, form):
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(M * 7 + K + N)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-3, 4, (1, K), generator=g).float())
    x = x.bfloat16() if form in ("bf16", "gelu") else x
    w = torch.randn(N, K, generator=g) / K ** 0.5
    bias = None if form == "silu" else torch.randn(N, generator=g) * 0.3
    res = torch.randn(M, N, generator=g) if form == "residual" else None
    act = {"gelu": 1, "silu": 2}.get(form, 0)
    layer = Fp8Linear.from_weight(w.cuda(), None if bias is None else bias.cuda())
    got = layer(x.cuda(), act=act, residual=None if res is None else res.cuda(), bf16_out=form in ("bf16", "gelu"))
    assert got.shape == (M, N)
    check(got, *oracle(x, w, bias, act, res, got.dtype == torch.bfloat16))


@pytest.mark.parametrize("M,K,N", [(1, 512, 256), (40, 512, 256), (600, 512, 512)])
def test_linear_scales_far_apart(M, K, N):
    """blocks of one row whose scales differ by many powers of two: the exponents reach the products"""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(5)
    ex = torch.exp2(torch.randint(-20, 20, (M, K // 128), generator=g).float()).repeat_interleave(128, 1)
    ew = torch.exp2(torch.randint(-20, 20, (N, K // 128), generator=g).float()).repeat_interleave(128, 1)
    x, w = torch.randn(M, K, generator=g) * ex, torch.randn(N, K, generator=g) * ew
    layer = Fp8Linear.from_weight(w.cuda())
    for fast in (False, True):
        check(layer(x.cuda(), bf16_out=fast), *oracle(x, w, None, 0, None, fast))


def test_linear_shapes_strides_and_streams():
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(1)
    w, b = torch.randn(200, 300, generator=g).cuda(), torch.randn(200, generator=g).cuda()
    layer = Fp8Linear.from_weight(w, b)
    x = torch.randn(6, 5, 300, generator=g).cuda()
    y = layer(x)
    assert y.shape == (6, 5, 200)
    flat = layer(x.reshape(30, 300))
    assert torch.equal(y.reshape(30, 200), flat)
    wide = torch.randn(30, 700, device="cuda")
    wide[:, 33:333] = x.reshape(30, 300)
    assert torch.equal(layer(wide[:, 33:333]), flat)  # rows not 16-B aligned
    assert torch.equal(layer(x.reshape(30, 300).t().contiguous().t()), flat)  # another order
    assert layer(x[:0]).shape == (0, 5, 200)
    assert torch.equal(layer(x[0, 0]), flat[0])
    y0 = torch.randn(30, 200, generator=g).cuda()
    want = layer(x.reshape(30, 300), residual=y0)
    out = y0.clone()
    assert layer(x.reshape(30, 300), residual=out, out=out) is out and torch.equal(out, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = layer(x.reshape(30, 300))
    s.synchronize()
    assert torch.equal(other, flat)
    for bad in (dict(residual=y0[:29]), dict(residual=y0.bfloat16()), dict(out=y0.bfloat16()), dict(out=y0[:29]),
                dict(residual=y0.t().contiguous().t())):
        with pytest.raises(ValueError):
            layer(x.reshape(30, 300), **bad)
    for bad in (x[..., :299], x.half(), x.cpu()):
        with pytest.raises(ValueError):
            layer(bad)


def test_linear_not_finite():
    """a NaN or infinity of x reaches its own row only; one of w its own column"""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(70, 256, generator=g), torch.randn(90, 256, generator=g)
    x[3, 7], x[40, 200], w[11, 3] = float("nan"), float("inf"), float("nan")
    bad = torch.zeros(70, 90, dtype=torch.bool)
    bad[3], bad[40], bad[:, 11] = True, True, True
    for fast in (False, True):
        y = Fp8Linear.from_weight(w.cuda())(x.cuda(), bf16_out=fast).cpu()
        assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("M", [1, 50, 700])
def test_linear_captured(M):
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(3)
    layer = Fp8Linear.from_weight(torch.randn(512, 1024, generator=g).cuda(), torch.randn(512, generator=g).cuda())
    x = torch.randn(M, 1024, generator=g).cuda()
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, act=1)
    for i in range(4):
        x.copy_(torch.randn(M, 1024, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, layer(x, act=1)), i


# more rows x columns than 32 x 16 outputs of a workgroup can take in three turns: 128 x 128 tiles; sides and reductions that
# end inside a tile, one to 65 blocks of k (the scales of 64 are held at once)
TILES = [(51300, 129, 16), (9, 1100, 51300), (1000, 1, 400), (2100, 130, 200), (3333, 300, 144), (1537, 512, 1000), (700, 8200, 640)]
# from 160 tiles of 256 x 256 on, bf16 results: those
LARGE = [(3500, 100, 3600), (3500, 256, 3601), (3585, 300, 3600), (3499, 640, 3700), (51300, 129, 200), (151, 1100, 51300),
         (3500, 8192, 3600)]


BF16_FORMS = ["gelu", "bf16", "bf16 residual"]


@pytest.mark.parametrize("M,K,N,form", [(*s, f) for s in TILES + LARGE for f in BF16_FORMS] +
                         [(*s, f) for s in TILES for f in ("plain", "silu", "residual")])
def test_linear_tiles(M, K, N, form):
    from indextts.utils.fp8 import Fp8Linear
    fast = form in BF16_FORMS
    g = torch.Generator(device="cuda").manual_seed(M * 7 + K + N)
    x = torch.randn(M, K, generator=g, device="cuda") * torch.exp2(torch.randint(-3, 4, (1, K), generator=g, device="cuda").float())
    x = x.bfloat16() if fast else x
    w = torch.randn(N, K, generator=g, device="cuda") / K ** 0.5
    bias = None if form == "silu" else torch.randn(N, generator=g, device="cuda") * 0.3
    res = torch.randn(M, N, generator=g, device="cuda") if "residual" in form else None
    act = {"gelu": 1, "silu": 2}.get(form, 0)
    got = Fp8Linear.from_weight(w, bias)(x, act=act, residual=res, bf16_out=fast)
    check(got, *oracle(x, w, bias, act, res, fast))


@pytest.mark.parametrize("M,K,N,fast", [(1100, 512, 1024, False), (1100, 512, 1024, True), (3500, 512, 3600, True)])
def test_tiles_scales_far_apart_and_not_finite(M, K, N, fast):
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator(device="cuda").manual_seed(6)

    def spread(rows):
        e = torch.exp2(torch.randint(-20, 20, (rows, K // 128), generator=g, device="cuda").float())
        return torch.randn(rows, K, generator=g, device="cuda") * e.repeat_interleave(128, 1)
    x, w = spread(M), spread(N)
    check(Fp8Linear.from_weight(w)(x, bf16_out=fast), *oracle(x, w, None, 0, None, fast))
    x[3, 7], x[M - 1, 200], w[11, 3] = float("nan"), float("inf"), float("nan")
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[3], bad[M - 1], bad[:, 11] = True, True, True
    assert torch.equal(torch.isnan(Fp8Linear.from_weight(w)(x, bf16_out=fast)), bad)


def test_many_rows_of_a_narrow_layer():
    """more rows than 65535 workgroups of 32"""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator(device="cuda").manual_seed(8)
    w = torch.randn(8, 16, generator=g, device="cuda")
    layer = Fp8Linear.from_weight(w, torch.randn(8, generator=g, device="cuda"))
    x = torch.randn(2200001, 16, generator=g, device="cuda")
    y = layer(x)
    for at in (slice(0, 9), slice(2097144, 2097160), slice(2199990, 2200001)):
        check(y[at], *oracle(x[at], w, layer.bias, 0, None, False))


@pytest.mark.parametrize("M,N,fast", [(1100, 1024, False), (1100, 1024, True), (3500, 3600, True)])
def test_tiles_captured(M, N, fast):
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator(device="cuda").manual_seed(9)
    layer = Fp8Linear.from_weight(torch.randn(N, 300, generator=g, device="cuda"))
    x = torch.randn(M, 300, generator=g, device="cuda")
    layer(x, bf16_out=fast)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, act=2, bf16_out=fast)
    for i in range(4):
        x.copy_(torch.randn(M, 300, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer(x, act=2, bf16_out=fast))


def test_out_over_x_is_refused():
    from indextts.utils.fp8 import Fp8Linear
    layer = Fp8Linear.from_weight(torch.randn(128, 128, device="cuda"))
    x = torch.randn(40, 128, device="cuda")
    for out in (x, x[3:13]):
        with pytest.raises(ValueError):
            layer(x[:out.shape[0]] if out is not x else x, out=out)
    both = torch.randn(80, 128, device="cuda")
    want = layer(both[:40])
    assert torch.equal(layer(both[:40], out=both[40:]), want) and torch.equal(both[40:], want)
