"""8-bit operators on the GPU: layouts, ranges of values and aliasing at the edges of what the calls take."""
import pytest
import torch

from eightbit_util import attend64, attn_tol, codes64, seen_keys
from test_gpu_fp8 import check as check_linear, oracle as linear_oracle
from test_gpu_kv8 import check_rows, filled, i32, pieces, tree_case

pytestmark = pytest.mark.gpu


def test_one_lineage_table_expanded_over_the_rows():
    R, B, S = 5, 6, 130
    c, _, _ = filled(R, 2, S, 64, seed=3)
    g = torch.Generator().manual_seed(4)
    table = torch.randint(R, (1, S + 3), generator=g).int().cuda().expand(B, -1)
    lens = i32([130, 1, 64, 0, 33, 99])
    q = torch.randn(B, 4, 64, generator=g).cuda()
    for longest in (None, 1300):
        got = c.decode(q, lens, kv_rows=table, max_len=longest)
        assert torch.equal(got, c.decode(q, lens, kv_rows=table.contiguous(), max_len=longest))
    mask = torch.tensor([1, 3], device="cuda")
    lens, q = lens.clamp(max=100), torch.randn(B, 2, 4, 64, generator=g).cuda()
    assert torch.equal(c.tree(q, lens, mask, kv_rows=table), c.tree(q, lens, mask, kv_rows=table.contiguous()))
    with pytest.raises(ValueError):
        c.decode(q[:, 0], lens, kv_rows=torch.zeros(400, dtype=torch.int32, device="cuda").as_strided((B, S), (50, 1)))


@pytest.mark.parametrize("N", [3585, 3602])
def test_last_tile_of_few_columns(N):
    """256 x 256 tiles whose last holds one column or 18 of w, at the end of its buffer"""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randn(3500, 1000, generator=g, device="cuda")
    w = torch.randn(N, 1000, generator=g, device="cuda")
    got = Fp8Linear.from_weight(w)(x, bf16_out=True)
    check_linear(got, *linear_oracle(x, w, None, 0, None, True))


@pytest.mark.parametrize("T,lens", [(3, [40, 0, 33]), (40, [40, 64, 7]), (2, [2000, 5, 700])])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
def test_tree_large_finite_values_in_a_bf16_cache(T, lens, q_dtype):
    """the largest sum of weights (relative to the largest) times |V| lies within [2^126, 2^127): finite in f32"""
    from indextts.gpt.kv8 import Kv16Cache
    c, k, v, q, mask = tree_case(3, T, 2, 1, 64, lens, 91, False, q_dtype)
    see = seen_keys(3, T, k.shape[2], i32(lens), None, mask)
    s = torch.matmul(q.double().cpu().transpose(1, 2), k.cpu().transpose(2, 3)) * 0.125
    s = s.masked_fill(~see[:, None], -torch.inf)
    most = torch.matmul(torch.exp(s - s.amax(-1, keepdim=True)), v.cpu().abs()).max()
    big = (v * torch.exp2(126 - torch.floor(torch.log2(most))).cuda()).bfloat16()
    got = Kv16Cache(c.k, big).tree(q, i32(lens), mask)
    check_rows(got, q, k, big.double(), see, 0.125, pieces(q_dtype, torch.bfloat16, False), torch.bfloat16)


# ---- scales of V far apart in an 8-bit cache: every value within f32's range counts where it is seen, and only there ----

OUT = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32)]


def raised(c, places, by):
    """c's V times 2^by at places (an index of [rows, heads, max_kv]); the values it then stands for"""
    c.v_scale[places] += by
    return codes64(c.v, c.v_scale)


def identity(B, S):
    return torch.arange(B, device="cuda", dtype=torch.int32)[:, None].repeat(1, S)


@pytest.mark.parametrize("q_dtype,out_dtype", OUT)
@pytest.mark.parametrize("hd,heads,group", [(64, 2, 1), (128, 1, 3)])
@pytest.mark.parametrize("T", [4, 20])
@pytest.mark.parametrize("by", [25, 40, 100])
def test_a_drafted_token_with_a_large_v_reaches_only_its_own(q_dtype, out_dtype, hd, heads, group, T, by):
    lens = [0, 30, 64, 1500]
    c, k, v, q, mask = tree_case(4, T, heads, group, hd, lens, by, True, q_dtype)
    for b, n in enumerate(lens):
        v = raised(c, (b, slice(None), n + 2), by)
    see = seen_keys(4, T, k.shape[2], i32(lens), None, mask)
    for rows in (None, identity(4, k.shape[2])):
        got = c.tree(q, i32(lens), mask, kv_rows=rows, dtype=out_dtype)
        check_rows(got, q, k, v, see, hd ** -0.5, pieces(q_dtype, out_dtype), out_dtype)


@pytest.mark.parametrize("q_dtype,out_dtype", OUT)
@pytest.mark.parametrize("by", [20, 60, 80, 110])
def test_waves_whose_scales_are_far_apart(q_dtype, out_dtype, by):
    """two drafted tokens in a tile of their own, both with a large V, of which the second sees neither"""
    lens = [32, 64, 96, 2048]
    c, k, v, q, _ = tree_case(4, 2, 2, 2, 64, lens, by, True, q_dtype)
    mask = torch.tensor([1, 0], device="cuda")
    for b, n in enumerate(lens):
        v = raised(c, (b, slice(None), slice(n, n + 2)), by)
    got = c.tree(q, i32(lens), mask, dtype=out_dtype)
    check_rows(got, q, k, v, seen_keys(4, 2, k.shape[2], i32(lens), None, mask), 0.125, pieces(q_dtype, out_dtype), out_dtype)


@pytest.mark.parametrize("q_dtype,out_dtype", OUT)
@pytest.mark.parametrize("hd,heads,group", [(64, 2, 1), (128, 1, 20)])
def test_keys_whose_scales_are_far_apart(q_dtype, out_dtype, hd, heads, group):
    """large V with next to no weight beside small V with all of it, and V of every scale"""
    lens = i32([1, 50, 300, 1999])
    c, k, v = filled(4, heads, 2000, hd, seed=5)
    g = torch.Generator().manual_seed(6)
    q = (torch.randn(4, heads * group, hd, generator=g) * 2).to(q_dtype).cuda()
    see = seen_keys(4, 1, 2000, lens)
    c.k_scale[:, :, 7] += 3  # wide scores: some keys have weights of 2^-40 and less
    c.k_scale[:, :, 100::9] += 3
    k = codes64(c.k, c.k_scale)
    v = raised(c, (slice(None), slice(None), slice(7, None, 31)), 30)
    for _ in range(2):
        got = c.decode(q, lens, dtype=out_dtype)
        check_rows(got[:, None], q[:, None], k, v, see, hd ** -0.5, pieces(q_dtype, out_dtype), out_dtype)
        c.v_scale.copy_(torch.randint(30, 230, c.v_scale.shape, generator=g, dtype=torch.uint8))
        v = codes64(c.v, c.v_scale)


@pytest.mark.parametrize("q_dtype,out_dtype", OUT)
def test_loud_dims(q_dtype, out_dtype):
    """some keys hold one dim 2^30 above the others (whose codes are 0): the other keys' values still make the other dims"""
    from indextts.gpt.kv8 import Kv8Cache
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 100, 2, 64, generator=g)
    y = x.clone()
    y[:, 5::20, :, 9] = 2.0 ** 30
    c = Kv8Cache.empty(2, 2, 100, 64)
    row, pos = torch.arange(2).repeat_interleave(100).int().cuda(), torch.arange(100).repeat(2).int().cuda()
    c.write(x.view(-1, 2, 64).cuda(), y.view(-1, 2, 64).cuda(), row, pos)
    q = torch.randn(2, 2, 64, generator=g).to(q_dtype).cuda()
    k, v = codes64(c.k, c.k_scale), codes64(c.v, c.v_scale)
    got = c.decode(q, i32([100, 61]), dtype=out_dtype)
    check_rows(got[:, None], q[:, None], k, v, seen_keys(2, 1, 100, i32([100, 61])), 0.125, pieces(q_dtype, out_dtype), out_dtype)


@pytest.mark.parametrize("q_dtype,out_dtype", OUT)
@pytest.mark.parametrize("by", [-100, -60, 60, 105])
def test_v_at_the_ends_of_the_range(q_dtype, out_dtype, by):
    """all V times 2^by: the results times 2^by"""
    lens = i32([3, 40, 1400])
    c, k, v = filled(3, 2, 1400, 64, seed=12)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(13)).to(q_dtype).cuda()
    v = raised(c, (slice(None),) * 3, by % 256)
    got = c.decode(q, lens, dtype=out_dtype).double() * 2.0 ** -by
    ref, mag, top = attend64(q[:, None].double(), k, v * 2.0 ** -by, seen_keys(3, 1, 1400, lens), 0.125)
    tol = attn_tol(ref, mag, top, 1400, 64, pieces(q_dtype, out_dtype), out_dtype)
    assert bool(((got[:, None] - ref).abs() <= tol).all())


def test_captured_with_scales_far_apart():
    c, k, v = filled(3, 2, 700, 64, seed=15)
    raised(c, (slice(None), 0, 5), 50)
    q, lens = torch.randn(3, 4, 64, device="cuda"), i32([700, 3, 90])
    c.decode(q, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = c.decode(q, lens, dtype=torch.float32)
    for i in range(4):
        q.copy_(torch.randn(3, 4, 64))
        c.v_scale[1, :, 1 + i] ^= 64  # some keys 2^64 larger or smaller than before
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, c.decode(q, lens, dtype=torch.float32)) and torch.isfinite(y).all(), i


def test_a_residual_that_overlaps_out_is_refused():
    from indextts.utils.fp8 import Fp8Linear
    layer = Fp8Linear.from_weight(torch.randn(64, 128, device="cuda"))
    x, both = torch.randn(40, 128, device="cuda"), torch.randn(81, 64, device="cuda")
    for res, out in ((both[:40], both[1:41]), (both[1:41], both[:40]), (both[39:79], both[:40])):
        with pytest.raises(ValueError):
            layer(x, residual=res, out=out)
    with pytest.raises(ValueError):
        layer(x, residual=both[:40], out=both[:20].view(torch.bfloat16).view(40, 64), bf16_out=True)
    want = layer(x, residual=both[41:])
    assert torch.equal(layer(x, residual=both[41:], out=both[:40]), want)
    assert torch.equal(layer(x, residual=both[41:], out=both[41:]), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("longest", [60, 3000])
def test_out_may_be_q(dtype, longest):
    """in one part and split over the keys; more columns than one workgroup takes; also out between q's rows"""
    c, _, _ = filled(3, 2, 3000, 64, seed=21)
    g = torch.Generator().manual_seed(22)
    lens = i32([60, 0, 33]) if longest == 60 else i32([2900, 7, 1100])
    qkv = torch.randn(3, 3, 2 * 20, 64, generator=g).to(dtype).cuda()
    q = qkv[:, 0]
    want = c.decode(q, lens, max_len=longest, dtype=dtype)
    assert torch.equal(c.decode(q, lens, max_len=longest, out=qkv[:, 1]), want)
    assert c.decode(q, lens, max_len=longest, out=q) is q and torch.equal(q, want)
    q = torch.randn(3, 33, 4, 64, generator=g).to(dtype).cuda()
    mask = torch.arange(1, 34, device="cuda")
    want = c.tree(q, lens, mask, max_len=longest, dtype=dtype)
    assert torch.equal(c.tree(q, lens, mask, max_len=longest, out=q), want)
    for out in (qkv[:, 0, :, :].as_strided((3, 40, 64), qkv[:, 0].stride(), 64), c.k.view(-1)[:3 * 40 * 64 * 4].view(torch.float32).view(3, 40, 64),
                qkv[:, 0, :1].expand(3, 40, 64)):
        with pytest.raises(ValueError):
            c.decode(qkv[:, 0], lens, out=out)


@pytest.mark.parametrize("scale", [-0.125, 0.0])
@pytest.mark.parametrize("e4m3", [True, False])
def test_scales_that_are_not_positive(scale, e4m3):
    lens = [0, 5, 200]
    c, k, v, q, mask = tree_case(3, 6, 2, 2, 64, lens, 33, e4m3, torch.float32)
    got = c.tree(q, i32(lens), mask, scale=scale)
    ref = q * (0.0 if scale == 0 else -1.0)  # the same scores at a positive scale
    check_rows(got, ref, k, v, seen_keys(3, 6, k.shape[2], i32(lens), None, mask), 0.125, pieces(None, torch.bfloat16, e4m3), torch.bfloat16)


@pytest.mark.parametrize("apart", [0, 30])
@pytest.mark.parametrize("longest", [64, 2000])
def test_stale_slots_and_nan_beside_scales_far_apart(apart, longest):
    """what is not seen does not reach a result: slots behind the row and before its padding with any byte as scale, and a drafted NaN"""
    lens = [20, 64]
    c, k, v, q, mask = tree_case(2, 6, 2, 1, 64, lens, 35, True, torch.float32, smax=90)
    raised(c, (slice(None), slice(None), 9), apart)
    pad = i32([3, 40])
    want = c.tree(q, i32(lens), mask, pad=pad, max_len=longest, dtype=torch.float32)
    for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        t[0, :, 26:], t[1, :, 70:], t[0, :, :3] = 0x7F, 0xFF, 0x7E
        s[0, :, 26:], s[1, :, 70:], s[0, :, :3] = 255, 0, 254
    assert torch.equal(c.tree(q, i32(lens), mask, pad=pad, max_len=longest, dtype=torch.float32), want)
    c.v[0, 0, 22, 3], c.v[1, 1, 69, 0] = 0x7F, 0xFF
    got = c.tree(q, i32(lens), mask, pad=pad, max_len=longest, dtype=torch.float32)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :, 0, 3], bad[1, :, 1, 0] = (mask[0] >> 2 & 1).bool(), (mask[1] >> 5 & 1).bool()
    assert torch.equal(torch.isnan(got), bad) and torch.equal(torch.where(bad, 0, got), torch.where(bad, 0, want))


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_many_small_weights_of_larger_v(out_dtype):
    """one key has a weight of 1, each of 131072 others e^-24 (2^-34.6) and a V 2^12 larger: together two per cent of the result.
    In f16 a weight is off by at most 2^-38 of the largest in its wave (half of f16's least step at the scale that weights are held
    at), and the large key's wave takes a fourth of the keys where they are not split."""
    from indextts.gpt.kv8 import Kv8Cache
    S, g = 131073, torch.Generator().manual_seed(17)
    k = torch.zeros(S, 1, 64)
    k[0, 0, 0] = 24.0
    v = 0.5 + torch.rand(1, 1, 64, generator=g).repeat(S, 1, 1)
    v[1:] *= 2.0 ** 12
    c = Kv8Cache.empty(1, 1, S, 64)
    c.write(k.cuda(), v.cuda(), torch.zeros(S, dtype=torch.int32, device="cuda"), torch.arange(S, device="cuda").int())
    k, v = codes64(c.k, c.k_scale), codes64(c.v, c.v_scale)
    q = torch.zeros(1, 1, 64, device="cuda")
    q[..., 0] = 1.0
    ref, mag, top = attend64(q[:, None].double(), k, v, seen_keys(1, 1, S, i32([S])), 1.0)
    tol = attn_tol(ref, mag, top, 0, 64, pieces(None, out_dtype), out_dtype) + S / 4 * 2.0 ** -38 * v[0, 0].amax(0)
    small = ref[0, 0, 0] - v[0, 0, 0] / (1 + (S - 1) * torch.exp(torch.tensor(-24.0, dtype=torch.float64)))
    assert out_dtype == torch.bfloat16 or bool((small / 4 > 4 * tol[0, 0, 0]).all())  # a fourth of that lost would be seen
    got = c.decode(q, i32([S]), scale=1.0, max_len=1, dtype=out_dtype)
    assert bool(((got[:, None].double() - ref).abs() <= tol).all()), float(((got[:, None].double() - ref).abs() / tol).max())
