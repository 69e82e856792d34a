"""8-bit operators on the GPU: layouts, ranges of values and aliasing at the edges of what the calls take."""
import pytest
import torch

from eightbit_util import seen_keys
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
