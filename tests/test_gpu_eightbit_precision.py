"""The 8-bit operators' f32 forms are told from the cheaper forms beside them: by root mean squares, and by inputs whose result
lies in the bits that a cheaper form drops.  Each test also plants the cheaper form in the 64-bit oracle and sees it fail."""
import pytest
import torch

from eightbit_util import codes64, quant64
from test_gpu_fp8 import check, oracle
from test_gpu_kv8 import filled, i32

pytestmark = pytest.mark.gpu

ROUTES = [(1, 512, 64), (16, 1024, 200), (32, 512, 96), (96, 1024, 130), (300, 512, 512), (1100, 512, 1024), (1537, 640, 1000)]


def rms(x):
    return float(x.double().square().mean().sqrt())


def blocks(t):
    return quant64(t.view(t.shape[0], -1, 128))[0]


@pytest.mark.parametrize("M,K,N", ROUTES)
def test_linear_f32_by_rms(M, K, N):
    """K / 32 additions to a sum whose rms after k of n is sqrt(k / n) of the result's, each off by at most a step of it: 2 n / 3
    steps in all, and two for the waves' parts and the bias.  The 8-bit unit's cut is 1.5e-5 of the result's rms."""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(M + N)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    y = blocks(x).view(M, K) @ blocks(w).view(N, K).t()
    bound = (2 * (K / 32) / 3 + 2) * 2.0 ** -23
    assert bound < 1e-5
    got = Fp8Linear.from_weight(w.cuda())(x.cuda()).cpu()
    assert rms(got - y) <= bound * rms(y), rms(got - y) / rms(y)


@pytest.mark.parametrize("M,N", [(m, n) for m, _, n in ROUTES])
def test_linear_f32_keeps_small_products_beside_large_ones(M, N):
    """two large products of the first block cancel; its others are some 2^-13 of them"""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(M + N)
    x, w = torch.randn(M, 256, generator=g) * 2, torch.randn(N, 256, generator=g) * 2
    x[:, 0], x[:, 1], w[:, 0], w[:, 1] = 256.0, 256.0, 256.0, -256.0
    y, tol = oracle(x, w, None, 0, None, False)
    # the 8-bit unit, as the operators' notes have it: products cut at 2^-13 of the block's largest
    p = blocks(x[:8])[:, None] * blocks(w[:8])[None]
    step = p.abs().amax(-1, keepdim=True) * 2.0 ** -13
    planted = (torch.trunc(p / step) * step).sum((-1, -2))
    assert float(((planted - y[:8, :8]).abs() > tol[:8, :8]).double().mean()) > 0.5
    check(Fp8Linear.from_weight(w.cuda())(x.cuda()).cpu(), y, tol)


def attention(q, k, v, scale):
    """q [B, H, G, hd], k / v [B, H, S, hd] -> (out, sqrt(sum of (w (v - out))^2): what independent errors of the weights come to)"""
    w = torch.softmax(torch.matmul(q.double(), k.transpose(2, 3)) * scale, -1)
    out = torch.matmul(w, v)
    return out, (w.square()[..., None] * (v[:, :, None] - out[..., None, :]).square()).sum(-2).sqrt()


def bound(spread, out, hd, parts, running):
    """rms of the error, twice what follows from: hd * parts additions to a score, each off by at most a step of the running sum,
    independent of each other; 2^-20 for the exponential with its argument's rounding; two steps of the result"""
    return 2 * (((hd * parts) ** 0.5 * 2.0 ** -23 * running + 2.0 ** -20) * rms(spread) + 2.0 ** -22 * rms(out))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("apart", [False, True])
def test_decode_f32_weights(hd, q_dtype, apart):
    """few keys, so that the rounding of a single weight shows: one f16 part of P (11 bits) or one bf16 part (8) would"""
    c, k, v = filled(64, 2, 3, hd, seed=hd, spread=0)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(64, 4, hd, generator=g).to(q_dtype).cuda()
    if apart:  # the third key, which a row never sees the weight of, sends the wave through bf16
        c.v_scale[:, :, 2] -= 20
        v = codes64(c.v, c.v_scale)
    lens = i32([3] * 64)
    qh = q.view(64, 2, 2, hd)
    ref, spread = attention(qh, k, v, hd ** -0.5)
    running = rms(torch.matmul(qh.double().abs(), k.abs().transpose(2, 3))) * hd ** -0.5
    most = bound(spread, ref, hd, 3 if q_dtype == torch.float32 else 1, running)
    s = torch.matmul(qh.double(), k.transpose(2, 3)) * hd ** -0.5
    p = torch.exp(s - s.amax(-1, keepdim=True)).to(torch.bfloat16 if apart else torch.float16).double()
    assert rms(torch.matmul(p, v) / p.sum(-1, keepdim=True) - ref) > 3 * most
    got = c.decode(q, lens, dtype=torch.float32).view(64, 2, 2, hd)
    assert rms(got - ref) <= most, rms(got - ref) / most


@pytest.mark.parametrize("hd", [64, 128])
def test_scores_of_an_f32_q(hd):
    """q in pairs that nearly cancel over K's pairs of +-64: the scores lie in q's low bits, which two bf16 parts (16 bits) lose;
    running sums are one or two products"""
    from indextts.gpt.kv8 import Kv8Cache
    g = torch.Generator().manual_seed(hd)
    B, S = 64, 3
    sign = torch.where(torch.rand(B, 1, S, hd // 2, generator=g) < 0.5, -64.0, 64.0)
    k = torch.stack([sign, -sign], -1).view(B, 1, S, hd).cuda()
    v = torch.randn(B, 1, S, hd, generator=g).cuda() * 8
    half = 1 + torch.rand(B, 1, 1, hd // 2, generator=g)
    q = torch.stack([half, half + torch.randn(half.shape, generator=g) * 2.0 ** -7], -1).view(B, 1, 1, hd).cuda()
    c = Kv8Cache.empty(B, 1, S + 1, hd)  # room for a drafted token
    at = torch.arange(B * S, device="cuda").int()
    c.write(k.view(-1, 1, hd), v.view(-1, 1, hd), at // S, at % S)
    k, v = codes64(c.k, c.k_scale)[:, :, :S], codes64(c.v, c.v_scale)[:, :, :S]
    ref, spread = attention(q, k, v, hd ** -0.5)
    most = bound(spread, ref, hd, 3, 2 * 64 * 2.0 * hd ** -0.5)
    two = q.bfloat16().float()
    two = two + (q - two).bfloat16().float()
    assert rms(attention(two, k, v, hd ** -0.5)[0] - ref) > 1.5 * most
    for got in (c.decode(q[:, 0], i32([S] * B), dtype=torch.float32),
                c.tree(q, i32([S] * B), torch.zeros(1, dtype=torch.int64, device="cuda"), dtype=torch.float32)):
        assert rms(got.view(ref.shape) - ref) <= most, rms(got.view(ref.shape) - ref) / most
