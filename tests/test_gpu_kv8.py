"""The 8-bit KV cache and the attention over a cache (indextts/gpt/kv8.py) against their definitions in 64 bits."""
import pytest
import torch

from eightbit_util import attend64, attn_tol, codes64, quant64, seen_keys

pytestmark = pytest.mark.gpu

F16_P, F16_P2, BF16_P2 = 2.0 ** -11, 2.0 ** -22, 2.0 ** -16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def filled(rows, heads, smax, hd, seed=0, spread=3):
    """(cache, k, v): an e4m3 cache with every slot written, and the values it stands for (float64, GPU)"""
    from indextts.gpt.kv8 import Kv8Cache
    g = torch.Generator().manual_seed(seed)
    c = Kv8Cache.empty(rows, heads, smax, hd)
    at = torch.arange(rows * smax)
    x = [torch.randn(rows * smax, heads, hd, generator=g) *
         torch.exp2(torch.randint(-spread, spread + 1, (rows * smax, heads, 1), generator=g).float()) for _ in range(2)]
    c.write(x[0].cuda(), x[1].cuda(), (at // smax).int().cuda(), (at % smax).int().cuda())
    return c, codes64(c.k, c.k_scale), codes64(c.v, c.v_scale)


# ---- writing and reading back --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("M", [1, 2, 33, 200])
def test_write_and_read(dtype, hd, M):
    from indextts.gpt.kv8 import Kv8Cache
    g = torch.Generator().manual_seed(M + hd)
    rows, heads, smax = 5, 3, 41
    x = (torch.randn(M, 3, heads, hd, generator=g) * torch.exp2(torch.randint(-140, 118, (M, 3, heads, 1), generator=g).float())).to(dtype)
    x[0, 1, 0, 3], x[0, 2, 1, 0] = float("nan"), float("inf")
    x[-1, 2, 2] = 0
    slot = torch.randperm(rows * smax, generator=g)[:M]
    row, pos = (slot // smax).int(), (slot % smax).int()
    c = Kv8Cache.empty(rows, heads, smax, hd)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        t.fill_(0x55)
    xg = x.cuda()
    c.write(xg[:, 1], xg[:, 2], row.cuda(), pos.cuda())
    free = torch.ones(rows, smax, dtype=torch.bool)
    free[row.long(), pos.long()] = False
    for codes, scale, src in ((c.k, c.k_scale, x[:, 1]), (c.v, c.v_scale, x[:, 2])):
        want, e = quant64(src)
        codes, scale = codes.cpu(), scale.cpu()
        assert torch.equal(scale[row.long(), :, pos.long()].double() - 127, e)
        got = codes64(codes[row.long(), :, pos.long()], scale[row.long(), :, pos.long()])
        assert torch.equal(torch.nan_to_num(got, nan=7e77), torch.nan_to_num(want, nan=7e77))
        keep = free[:, None].expand(rows, heads, smax)  # slots not named keep what they held
        assert (codes[keep] == 0x55).all() and (scale[keep] == 0x55).all()
    for out in (torch.float32, torch.bfloat16):
        for got, src in zip(c.read(row.cuda(), pos.cuda(), dtype=out), (x[:, 1], x[:, 2])):
            want = quant64(src)[0].to(out)  # 4 significant bits: exact in both types but for f32 / bf16 denormals
            assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=7e77), torch.nan_to_num(want.double(), nan=7e77))


def test_write_skips_and_read_zeros_outside():
    from indextts.gpt.kv8 import Kv8Cache
    c = Kv8Cache.empty(2, 2, 10, 64)
    x = torch.randn(6, 2, 64, device="cuda")
    row, pos = i32([0, -1, 1, 2, 1, 0]), i32([9, 3, 10, 0, -1, 0])
    c.write(x, x, row, pos)
    held = torch.zeros(2, 10, dtype=torch.bool)
    held[0, 9] = held[0, 0] = True
    assert torch.equal((c.k_scale[:, 0] != 0).cpu(), held) and torch.equal((c.v_scale[:, 1] != 0).cpu(), held)
    k, v = c.read(row, pos, dtype=torch.float32)
    want = quant64(x.cpu())[0].float()
    want[1:5] = 0
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
    c.write(x[:0], x[:0], row[:0], pos[:0])
    assert c.read(row[:0], pos[:0])[0].shape == (0, 2, 64)


def test_write_strides():
    """views of a fused projection, misaligned ones and ones with the heads in another order"""
    from indextts.gpt.kv8 import Kv8Cache
    row, pos = i32([0, 1, 1]), i32([4, 0, 7])
    for dt in (torch.float32, torch.bfloat16):
        base = torch.randn(3, 4 * 64 * 3 + 5, device="cuda").to(dt)
        views = [base[:, 5 + 256 * i: 5 + 256 * (i + 1)].view(3, 4, 64) for i in range(3)]
        views += [v.transpose(0, 1).contiguous().transpose(0, 1) for v in views]
        got = []
        for i in (0, 3):
            c = Kv8Cache.empty(2, 4, 9, 64)
            c.write(views[i + 1], views[i + 2], row, pos)
            got.append(c)
        assert torch.equal(got[0].k, got[1].k) and torch.equal(got[0].v, got[1].v) and got[0].k.any()
        assert torch.equal(got[0].k_scale, got[1].k_scale) and torch.equal(got[0].v_scale, got[1].v_scale)


def test_reading_and_writing_again_loses_nothing():
    c, k, v = filled(2, 3, 20, 64, spread=60)
    rk, rv = c.read(i32([0] * 20), i32(list(range(20))))
    c.write(rk, rv, i32([1] * 20), i32(list(range(20))))
    assert torch.equal(codes64(c.k, c.k_scale)[1], k[0]) and torch.equal(codes64(c.v, c.v_scale)[1], v[0])


# ---- single-token attention ------------------------------------------------------------------------


def check_rows(got, q, k, v, see, scale, p_step, out_dtype):
    """got [B, T, Hq, hd] against the 64-bit form at the tokens it has"""
    ref, mag, top = attend64(q.double(), k, v, see, scale)
    tol = attn_tol(ref, mag, top, see.shape[2], q.shape[3], p_step, out_dtype)
    assert got.dtype == out_dtype
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), float((err / tol).max())


def pieces(q_dtype, out_dtype, e4m3=True):
    return BF16_P2 if not e4m3 else F16_P2 if out_dtype == torch.float32 else F16_P


LENS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 3), (1, 17), (1, 40)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                               (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_decode_lengths(hd, heads, group, q_dtype, out_dtype):
    c, k, v = filled(len(LENS), heads, 301, hd, seed=hd + group)
    g = torch.Generator().manual_seed(9)
    q = (torch.randn(len(LENS), heads * group, hd, generator=g) * 2).to(q_dtype).cuda()
    pad = i32([[0, 5, 40, 300][i % 4] for i in range(len(LENS))])  # past the end: an empty row
    for pd in (None, pad):
        for longest in (None, 300, 7):  # the expected length changes the split, not the result
            got = c.decode(q, i32(LENS), pad=pd, max_len=longest, dtype=out_dtype)
            see = seen_keys(len(LENS), 1, 301, i32(LENS), pd)
            check_rows(got[:, None], q[:, None], k, v, see, hd ** -0.5, pieces(q_dtype, out_dtype), out_dtype)
            assert (got[0] == 0).all() and (pd is None or (got[3] == 0).all())


def test_decode_long():
    c, k, v = filled(3, 2, 5000, 64, seed=3)
    q = torch.randn(3, 4, 64, device="cuda") * 3
    lens = i32([4999, 1, 3001])
    for out_dtype in (torch.bfloat16, torch.float32):
        got = c.decode(q, lens, dtype=out_dtype)
        check_rows(got[:, None], q[:, None], k, v, seen_keys(3, 1, 5000, lens), 0.125, pieces(torch.float32, out_dtype), out_dtype)


def test_decode_many_rows_one_key():
    c, k, v = filled(200, 1, 4, 64, seed=4)
    q = torch.randn(200, 1, 64, device="cuda").bfloat16()
    got = c.decode(q, i32([1] * 200))
    assert torch.equal(got[:, 0], v[:, 0, 0].bfloat16())


def test_decode_peaked_and_flat_scores():
    """scores far apart (one key has all the weight) and all alike; large and tiny scales of K"""
    c, k, v = filled(4, 1, 200, 64, seed=6, spread=8)
    for f in (0.0, 1e-3, 30.0):
        q = torch.randn(4, 2, 64, device="cuda") * f
        for dt in (torch.float32, torch.bfloat16):
            got = c.decode(q, i32([200, 199, 65, 3]), dtype=dt)
            check_rows(got[:, None], q[:, None], k, v, seen_keys(4, 1, 200, i32([200, 199, 65, 3])), 0.125,
                       pieces(torch.float32, dt), dt)


def test_decode_scale_argument():
    c, k, v = filled(1, 2, 50, 64)
    q = torch.randn(1, 2, 64, device="cuda")
    got = c.decode(q, i32([50]), scale=0.3, dtype=torch.float32)
    check_rows(got[:, None], q[:, None], k, v, seen_keys(1, 1, 50, i32([50])), 0.3, F16_P2, torch.float32)


def test_decode_not_finite():
    """what a row may not see does not reach it (stale NaN behind the end and before the padding); a NaN that it sees does"""
    c, k, v = filled(4, 2, 70, 64, seed=8)
    q = torch.randn(4, 2, 64, device="cuda")
    lens, pad = i32([40, 70, 33, 64]), i32([0, 35, 1, 0])
    want = c.decode(q, lens, pad=pad, dtype=torch.float32)
    for t in (c.k, c.v):
        t[0, :, 40:], t[1, :, :35], t[2, :, 33:], t[2, :, 0] = 0x7F, 0xFF, 0x7F, 0x7F
    for t in (c.k_scale, c.v_scale):
        t[0, :, 40:], t[1, :, :35] = 247, 255
    assert torch.equal(c.decode(q, lens, pad=pad, dtype=torch.float32), want)
    c.v[3, 0, 10, 5] = 0x7F
    c.k[3, 1, 10, 5] = 0x7F
    got = c.decode(q, lens, pad=pad, dtype=torch.float32)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[3, 0, 5] = True
    bad[3, 1] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[:3], want[:3])
    q[1, 0, 3] = float("nan")
    got = c.decode(q, lens, pad=pad, dtype=torch.float32)
    assert torch.isnan(got[1, 0]).all() and torch.equal(got[1, 1], want[1, 1])


def test_decode_refuses_rows_it_cannot_read():
    c, _, _ = filled(3, 2, 30, 64)
    q = torch.randn(3, 2, 64, device="cuda")
    good = c.decode(q, i32([30, 30, 30]))
    got = c.decode(q, i32([-1, 31, 30]))
    assert torch.isnan(got[:2]).all() and torch.equal(got[2], good[2])
    got = c.decode(q, i32([30, 30, 30]), pad=i32([-5, 0, 0]))
    assert torch.equal(got, good)
    assert c.decode(q[:0], i32([])).shape == (0, 2, 64)


@pytest.mark.parametrize("longest", [None, 40])
def test_decode_lineage(longest):
    R, B, S = 7, 6, 290
    c, k, v = filled(R, 2, S, 64, seed=11)
    g = torch.Generator().manual_seed(12)
    kv_rows = torch.randint(R, (B, S + 3), generator=g).int().cuda()
    lens, pad = i32([290, 1, 64, 0, 33, 200]), i32([3, 0, 0, 0, 40, 199])
    q = torch.randn(B, 4, 64, generator=g).cuda()
    at = kv_rows[:, :S].long()[:, None], torch.arange(2, device="cuda")[None, :, None], torch.arange(S, device="cuda")[None, None]
    for dt in (torch.bfloat16, torch.float32):
        got = c.decode(q, lens, pad=pad, kv_rows=kv_rows, max_len=longest, dtype=dt)
        check_rows(got[:, None], q[:, None], k[at], v[at], seen_keys(B, 1, S, lens, pad), 0.125, pieces(torch.float32, dt), dt)
    # entries outside the cache: seen ones give NaN, others do not matter
    want = c.decode(q, lens, pad=pad, kv_rows=kv_rows, max_len=longest)
    kv_rows[0, 2], kv_rows[2, 64:], kv_rows[4, 39] = -1, 1 << 30, R
    assert torch.equal(c.decode(q, lens, pad=pad, kv_rows=kv_rows, max_len=longest), want)
    kv_rows[0, 289], kv_rows[5, 199] = R, -7
    got = c.decode(q, lens, pad=pad, kv_rows=kv_rows, max_len=longest)
    assert torch.isnan(got[0]).all() and torch.isnan(got[5]).all() and torch.equal(got[1:5], want[1:5])


def test_decode_strides():
    """q a view of a fused projection, out a view, codes in a larger buffer"""
    from indextts.gpt.kv8 import Kv8Cache
    c, k, v = filled(3, 2, 33, 64)
    big = [torch.zeros(4, 3, 40, 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
    sc = [torch.zeros(4, 3, 41, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for t, s in zip(big, (c.k, c.v)):
        t[:3, 1:, :33] = s
    for t, s in zip(sc, (c.k_scale, c.v_scale)):
        t[:3, 1:, 1:34] = s
    d = Kv8Cache(big[0][:3, 1:, :33], big[1][:3, 1:, :33], sc[0][:3, 1:, 1:34], sc[1][:3, 1:, 1:34])
    qkv = torch.randn(3, 6 * 64 + 3, device="cuda")
    q = qkv[:, 3:131].view(3, 2, 64)
    out = torch.full((3, 3, 70), 9.0, device="cuda")
    lens = i32([33, 20, 1])
    want = c.decode(q.contiguous(), lens, dtype=torch.float32)
    assert d.decode(q, lens, out=out[:, 1:, 3:67]) .data_ptr() == out[:, 1:, 3:67].data_ptr()
    assert torch.equal(out[:, 1:, 3:67], want)
    out[:, 1:, 3:67] = 9.0
    assert (out == 9.0).all()


def test_decode_offsets_beyond_32_bits():
    from indextts.gpt.kv8 import Kv8Cache
    rows, heads, smax = 300, 16, 16384  # 5 GB of codes each
    c = Kv8Cache.empty(rows, heads, smax, 64)
    at = torch.arange(smax - 50, smax)
    x = torch.randn(50, heads, 64, device="cuda")
    y = torch.randn(50, heads, 64, device="cuda")
    c.write(x, y, i32([299] * 50), at.int().cuda())
    small, k, v = Kv8Cache.empty(1, heads, 50, 64), None, None
    small.write(x, y, i32([0] * 50), i32(list(range(50))))
    q = torch.randn(1, heads, 64, device="cuda")
    kv_rows = torch.full((1, smax), 299, dtype=torch.int32, device="cuda")
    got = c.decode(q, i32([smax]), pad=i32([smax - 50]), kv_rows=kv_rows, dtype=torch.float32)
    k, v = codes64(small.k, small.k_scale), codes64(small.v, small.v_scale)
    check_rows(got[:, None], q[:, None], k, v, seen_keys(1, 1, 50, i32([50])), 0.125, F16_P2, torch.float32)
    rk, _ = c.read(i32([299]), i32([smax - 1]))
    assert torch.equal(rk, small.read(i32([0]), i32([49]))[0])


# ---- drafted tokens --------------------------------------------------------------------------------


def tree_case(B, T, heads, group, hd, lens, seed, e4m3, q_dtype, smax=None):
    from indextts.gpt.kv8 import Kv16Cache, tree_mask
    smax = smax or max(lens) + T
    g = torch.Generator().manual_seed(seed)
    if e4m3:
        c, k, v = filled(B, heads, smax, hd, seed)
    else:
        k, v = (torch.randn(B, heads, smax, hd, generator=g).bfloat16().cuda() for _ in range(2))
        c = Kv16Cache(k, v)
        k, v = k.double(), v.double()
    q = (torch.randn(B, T, heads * group, hd, generator=g) * 2).to(q_dtype).cuda()
    parents = torch.stack([torch.stack([torch.randint(-1, t, (1,), generator=g)[0] if t else torch.tensor(-1) for t in range(T)])
                           for _ in range(B)])
    return c, k, v, q, tree_mask(parents).cuda()


TYPES = [(True, torch.bfloat16, torch.bfloat16), (True, torch.float32, torch.bfloat16), (True, torch.float32, torch.float32),
         (True, torch.bfloat16, torch.float32), (False, torch.bfloat16, torch.bfloat16), (False, torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,heads,group", [(1, 2, 1), (3, 1, 5), (16, 2, 1), (17, 1, 1), (33, 1, 2), (64, 1, 1), (64, 1, 3)])
@pytest.mark.parametrize("e4m3,q_dtype,out_dtype", TYPES)
def test_tree(hd, T, heads, group, e4m3, q_dtype, out_dtype):
    lens = [0, 1, 30, 32, 64, 131]
    B = len(lens)
    c, k, v, q, mask = tree_case(B, T, heads, group, hd, lens, T + hd, e4m3, q_dtype)
    pad, n = i32([0, 5, 7, 0, 64, 131]), i32([T, max(1, T // 2), 0, T, T, max(1, T - 1)])
    for pd, nn, longest in ((None, None, None), (pad, n, 131), (pad, n, 3)):
        out = torch.full(q.shape, 5.0, dtype=out_dtype, device="cuda")
        got = c.tree(q, i32(lens), mask, n_tokens=nn, pad=pd, max_len=longest, out=out)
        see = seen_keys(B, T, k.shape[2], i32(lens), pd, mask, nn)
        live = torch.ones(B, T, dtype=torch.bool) if nn is None else torch.arange(T)[None] < nn.cpu()[:, None]
        assert (got[~live.cuda()] == 5.0).all()
        see &= live[:, :, None]
        ref = got * live.cuda()[:, :, None, None]
        check_rows(ref, q, k, v, see, hd ** -0.5, pieces(q_dtype, out_dtype, e4m3), out_dtype)


@pytest.mark.parametrize("e4m3", [True, False])
def test_tree_any_mask(e4m3):
    """masks that are no trees: none, all, only later tokens; one mask for all rows"""
    lens = [0, 40, 31]
    c, k, v, q, _ = tree_case(3, 5, 2, 1, 64, lens, 21, e4m3, torch.bfloat16)
    for mask in (torch.zeros(5, dtype=torch.int64), torch.full((5,), -1, dtype=torch.int64), torch.tensor([30, 1, 8, 0, 4])):
        for pad in (None, i32([0, 40, 100])):
            got = c.tree(q, i32(lens), mask.cuda(), pad=pad)
            see = seen_keys(3, 5, k.shape[2], i32(lens), pad, mask)
            check_rows(got, q, k, v, see, 0.125, pieces(None, torch.bfloat16, e4m3), torch.bfloat16)
            assert (got[~see.any(-1).cuda()] == 0).all()


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("T,hd", [(6, 64), (40, 128)])
def test_tree_not_finite(e4m3, T, hd):
    """a drafted token that is not finite reaches the tokens that see it and no others"""
    lens = [20, 64]
    c, k, v, q, mask = tree_case(2, T, 2, 1, hd, lens, 31, e4m3, torch.bfloat16, smax=64 + T + 9)
    want = c.tree(q, i32(lens), mask)
    nan = [0x7F, 0xFF] if e4m3 else [float("nan"), float("-inf")]
    c.k[0, :, 20 + T:], c.v[0, :, 20 + T:] = nan[0], nan[1]  # stale
    assert torch.equal(c.tree(q, i32(lens), mask), want)
    c.v[0, 0, 22, 3] = nan[0]
    c.v[1, 1, 64 + T - 1, 0] = nan[1]
    c.k[0, 1, 21] = nan[0]
    got = c.tree(q, i32(lens), mask)
    bits = lambda j: (mask >> j & 1).bool()  # noqa: E731
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :, 0, 3] = bits(2)[0]
    bad[1, :, 1, 0] = bits(T - 1)[1]
    bad[0, :, 1] = bits(1)[0][:, None]
    assert torch.equal(~torch.isfinite(got), bad)
    assert torch.equal(torch.where(bad, 0, got), torch.where(bad, 0, want))
    if not e4m3:
        assert (got[1, :, 1, 0][bits(T - 1)[1]] == float("-inf")).all()


def test_tree_refuses_rows_it_cannot_read():
    c, k, v, q, mask = tree_case(5, 4, 1, 1, 64, [10] * 5, 41, True, torch.bfloat16)
    good = c.tree(q, i32([10] * 5), mask)
    got = c.tree(q, i32([-1, 11, 10, 10, 10]), mask, n_tokens=i32([4, 4, 5, -1, 4]))
    assert torch.isnan(got[:4]).all() and torch.equal(got[4], good[4])
    kv_rows = torch.arange(5, device="cuda", dtype=torch.int32)[:, None].repeat(1, 14)
    assert torch.equal(c.tree(q, i32([10] * 5), mask, kv_rows=kv_rows), good)
    kv_rows[2, 3], kv_rows[1, 12] = 77, -1
    got = c.tree(q, i32([10] * 5), mask, kv_rows=kv_rows)
    assert torch.isnan(got[2]).all() and torch.equal(got[[0, 3, 4]], good[[0, 3, 4]])
    see = (mask[1] >> 2 & 1).bool()
    assert torch.isnan(got[1][see]).all() and torch.equal(got[1][~see], good[1][~see])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,heads,group", [(5, 2, 1), (33, 1, 2)])
@pytest.mark.parametrize("e4m3,q_dtype,out_dtype", TYPES)
@pytest.mark.parametrize("longest", [200, 1300])
def test_tree_lineage(hd, T, heads, group, e4m3, q_dtype, out_dtype, longest):
    """keys, drafted ones too, from rows that a table names; in one part and split over the keys"""
    lens = [0, 3, 190, 64, 129]
    c, k, v, q, mask = tree_case(5, T, heads, group, hd, lens, 51, e4m3, q_dtype)
    g = torch.Generator().manual_seed(52)
    S = k.shape[2]
    kv_rows = torch.randint(5, (5, S + 2), generator=g).int().cuda()
    pad, n = i32([0, 0, 66, 64, 1]), i32([T, 2, T, 1, T - 1])
    out = torch.zeros(q.shape, dtype=out_dtype, device="cuda")
    got = c.tree(q, i32(lens), mask, n_tokens=n, pad=pad, kv_rows=kv_rows, max_len=longest, out=out)
    at = kv_rows[:, :S].long()[:, None], torch.arange(heads, device="cuda")[None, :, None], torch.arange(S, device="cuda")[None, None]
    see = seen_keys(5, T, S, i32(lens), pad, mask, n) & (torch.arange(T)[None] < n.cpu()[:, None])[:, :, None]
    check_rows(got, q, k[at], v[at], see, hd ** -0.5, pieces(q_dtype, out_dtype, e4m3), out_dtype)


@pytest.mark.parametrize("e4m3,q_dtype,out_dtype", TYPES)
@pytest.mark.parametrize("hd,T,heads,group", [(64, 3, 2, 1), (64, 40, 1, 1), (128, 3, 1, 4), (128, 12, 1, 4)])
def test_tree_long(e4m3, q_dtype, out_dtype, hd, T, heads, group):
    """split over the keys, with short rows beside a long one; a drafted value that is not finite in the last part"""
    lens = [2490, 3, 700, 0]
    c, k, v, q, mask = tree_case(4, T, heads, group, hd, lens, 61, e4m3, q_dtype)
    got = c.tree(q, i32(lens), mask, dtype=out_dtype)
    check_rows(got, q, k, v, seen_keys(4, T, k.shape[2], i32(lens), None, mask), hd ** -0.5, pieces(q_dtype, out_dtype, e4m3), out_dtype)
    c.v[0, 0, 2491, 3] = 0x7F if e4m3 else float("nan")
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :, :group, 3] = (mask[0] >> 1 & 1).bool()[:, None]
    again = c.tree(q, i32(lens), mask, dtype=out_dtype)
    assert torch.equal(torch.isnan(again), bad) and torch.equal(torch.where(bad, 0, again), torch.where(bad, 0, got))


@pytest.mark.parametrize("longest", [70, 1300])
def test_tree_infinite_scores(longest):
    """a key whose score is -inf has no weight; where a token sees no other key the result is NaN, where it sees none 0"""
    from indextts.gpt.kv8 import Kv16Cache
    g = torch.Generator().manual_seed(71)
    k, v = (torch.randn(4, 1, 80, 64, generator=g).bfloat16().cuda() for _ in range(2))
    k[:, :, :, 0] = 0
    q = torch.randn(4, 2, 1, 64, generator=g).cuda()
    q[..., 0] = 1.0
    k[0, 0, 5, 0] = float("-inf")
    k[1, 0, :60, 0] = float("-inf")
    k[2, 0, 7, 0] = float("inf")
    got = Kv16Cache(k, v).tree(q, i32([60, 60, 60, 0]), torch.tensor([0, 2], device="cuda"), max_len=longest)
    assert torch.isnan(got[1, 0]).all() and torch.isnan(got[2]).all() and (got[3, 0] == 0).all()
    see = seen_keys(4, 2, 80, i32([60, 60, 60, 0]), None, torch.tensor([0, 2]))
    see[0, :, 5], see[1, :, :60], see[2] = False, False, False
    check_rows(torch.where(torch.isnan(got), 0, got), q, torch.nan_to_num(k.double(), posinf=0, neginf=0), v.double(), see, 0.125,
               BF16_P2, torch.bfloat16)


def test_tree_of_one_token_is_decode():
    c, k, v = filled(4, 2, 90, 64)
    q = torch.randn(4, 6, 64, device="cuda")
    one = c.tree(q[:, None], i32([0, 10, 64, 89]), torch.ones(1, dtype=torch.int64, device="cuda"), dtype=torch.float32)
    two = c.decode(q, i32([1, 11, 65, 90]), dtype=torch.float32)
    assert float((one[:, 0] - two).abs().max()) <= 1e-5 * float(v.abs().max())


# ---- together ---------------------------------------------------------------------------------------


def test_refusals():
    from indextts.gpt.kv8 import Kv8Cache
    c, _, _ = filled(2, 2, 8, 64)
    q = torch.zeros(2, 2, 64, device="cuda")
    one = i32([1, 1])
    for kw in (dict(q=q[:, :1]), dict(q=q.half()), dict(q=q[..., :32]), dict(q=q[0]), dict(kv_len=one.long()), dict(kv_len=one[:1]),
               dict(pad=one.cpu()), dict(kv_rows=one[:, None]), dict(out=q[:1]), dict(out=q.half()), dict(dtype=torch.float16),
               dict(q=torch.zeros(3, 2, 64, device="cuda"), kv_len=i32([1, 1, 1]))):
        with pytest.raises((ValueError, KeyError)):
            c.decode(**{"q": q, "kv_len": one, **kw})
    mask = torch.ones(2, 1, dtype=torch.int64, device="cuda")
    for kw in (dict(q=q), dict(mask=mask.int()), dict(mask=mask[:1]), dict(n_tokens=one.long()), dict(out=q[:, None].half())):
        with pytest.raises(ValueError):
            c.tree(**{"q": q[:, None], "kv_len": one, "mask": mask, **kw})
    with pytest.raises(ValueError):
        c.tree(torch.zeros(1, 65, 2, 64, device="cuda"), i32([0]), torch.zeros(65, dtype=torch.int64, device="cuda"))
    for k, v, r, p in ((q, q[:1], one, one), (q, q.bfloat16(), one, one), (q[:, :1], q[:, :1], one, one), (q, q, one[:1], one),
                       (q, q, one, one.long())):
        with pytest.raises(ValueError):
            c.write(k, v, r, p)
    with pytest.raises(ValueError):
        c.read(one, one[:1])
    with pytest.raises(ValueError):
        Kv8Cache(c.k, c.v[:, :1], c.k_scale, c.v_scale)
    with pytest.raises(ValueError):
        Kv8Cache(c.k, c.v, c.k_scale[..., :7], c.v_scale)
    with pytest.raises(ValueError):
        Kv8Cache(c.k.transpose(1, 2).contiguous().transpose(1, 2), c.v, c.k_scale, c.v_scale)


def block(D=256, H=4, seed=0):
    """one decoder block's attention half in 8 bits: c_attn, the cache, attn.c_proj into the residual stream"""
    from indextts.utils.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(seed)
    attn = Fp8Linear.from_weight((torch.randn(3 * D, D, generator=g) / D ** 0.5).cuda(), (torch.randn(3 * D, generator=g) * 0.1).cuda())
    proj = Fp8Linear.from_weight((torch.randn(D, D, generator=g) / D ** 0.5).cuda(), (torch.randn(D, generator=g) * 0.1).cuda())
    return attn, proj, H, D


def test_block_step_by_step_equals_tree():
    """prompt written, then tokens one by one through linear -> write -> decode -> linear; the same tokens drafted at once
    as a chain beside a wrong branch, then the chain accepted by reading its slots and writing them where they belong"""
    from indextts.gpt.kv8 import Kv8Cache, tree_mask
    attn, proj, H, D = block()
    B, S, T = 3, 37, 4
    g = torch.Generator().manual_seed(77)
    lens = [37, 20, 5]
    prompt, x = torch.randn(B, S, D, generator=g).cuda(), torch.randn(B, T, D, generator=g).cuda()
    row = torch.arange(B, device="cuda").repeat_interleave(S).int()
    pos = torch.arange(S, device="cuda").repeat(B).int()
    row = torch.where(pos < i32(lens).repeat_interleave(S), row, -1)
    step, draft = (Kv8Cache.empty(B, H, 64, D // H) for _ in range(2))
    for c in (step, draft):
        kv = attn(prompt.reshape(-1, D)).view(-1, 3, H, 64)
        c.write(kv[:, 1], kv[:, 2], row, pos)
    b = torch.arange(B, device="cuda").int()
    one = []
    for t in range(T):
        qkv = attn(x[:, t]).view(B, 3, H, 64)
        step.write(qkv[:, 1], qkv[:, 2], b, i32(lens) + t)
        o = step.decode(qkv[:, 0], i32(lens) + t + 1, dtype=torch.float32)
        one.append(proj(o.view(B, D), residual=x[:, t].contiguous()))
    one = torch.stack(one, 1)
    # drafted: 0, a wrong sibling 1, then the chain 2, 3, 4
    tokens = torch.stack([x[:, 0], -x[:, 1], x[:, 1], x[:, 2], x[:, 3]], 1)
    mask = tree_mask(torch.tensor([-1, 0, 0, 2, 3], device="cuda"))
    qkv = attn(tokens).view(B, 5, 3, H, 64)
    draft.write(qkv[:, :, 1].reshape(-1, H, 64), qkv[:, :, 2].reshape(-1, H, 64), b.repeat_interleave(5),
                (i32(lens)[:, None] + torch.arange(5, device="cuda").int()).reshape(-1))
    o = draft.tree(qkv[:, :, 0], i32(lens), mask, dtype=torch.float32)
    path = torch.tensor([0, 2, 3, 4], device="cuda")
    many = proj(o.reshape(B, 5, D), residual=tokens)[:, path]
    # attention differs by f32 rounding alone; where that crosses a rounding border of the next quantiser (half a step of
    # e4m3 is 2^-4 of a value), the output moves by that step times the weight: a few of D terms of size 1/sqrt(D)
    rms = float((one.double() - many.double()).square().mean().sqrt())
    assert rms <= 2.0 ** -4 * float((one - x).square().mean().sqrt()) * 0.25, rms
    at = (i32(lens)[:, None] + path.int()).reshape(-1)
    k, v = draft.read(b.repeat_interleave(4), at, dtype=torch.float32)
    draft.write(k, v, b.repeat_interleave(4), (i32(lens)[:, None] + torch.arange(4, device="cuda").int()).reshape(-1))
    for i in range(B):
        end = lens[i] + 4
        assert torch.equal(codes64(step.k, step.k_scale)[i, :, :end], codes64(draft.k, draft.k_scale)[i, :, :end])
        assert torch.equal(codes64(step.v, step.v_scale)[i, :, :end], codes64(draft.v, draft.v_scale)[i, :, :end])


def test_captured_steps():
    """the step captured once, replayed with the position advancing on the device, against eager steps on another cache"""
    from indextts.gpt.kv8 import Kv8Cache
    attn, proj, H, D = block(seed=3)
    B = 5
    x = torch.randn(B, D, device="cuda")
    lens = i32([0, 3, 31, 32, 60])
    b = torch.arange(B, device="cuda").int()
    caches = []
    for _ in range(2):
        c = Kv8Cache.empty(B, H, 100, 64)
        g = torch.Generator().manual_seed(4)
        c.write(torch.randn(B * 60, H, 64, generator=g).cuda(), torch.randn(B * 60, H, 64, generator=g).cuda(), b.repeat(60),
                torch.arange(60, device="cuda").repeat_interleave(B).int())
        caches.append(c)

    def step(c, ln):
        qkv = attn(x).view(B, 3, H, 64)
        c.write(qkv[:, 1], qkv[:, 2], b, ln)
        ln.add_(1)
        return proj(c.decode(qkv[:, 0], ln).view(B, D), residual=x)

    cap = lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(Kv8Cache.empty(B, H, 100, 64), lens.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(caches[0], cap)
    eager = lens.clone()
    for i in range(6):
        x.copy_(torch.randn(B, D))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step(caches[1], eager)), i
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(cap, eager)


def test_two_streams_at_once():
    c, k, v = filled(8, 4, 700, 64)
    q = [torch.randn(8, 8, 64, device="cuda") for _ in range(2)]
    lens = i32([700, 650, 600, 1, 333, 64, 65, 0])
    want = [c.decode(t, lens, dtype=torch.float32) for t in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.decode(q[i], lens, dtype=torch.float32))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])
