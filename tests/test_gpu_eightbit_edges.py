"""8-bit operators on the GPU: layouts, ranges of values and aliasing at the edges of what the calls take."""
import pytest
import torch

from test_gpu_fp8 import check as check_linear, oracle as linear_oracle
from test_gpu_kv8 import filled, i32

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
