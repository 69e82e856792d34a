"""The 8-bit operators' argument checks (before any HIP call, so without a GPU) and the tree masks."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from indextts import _build, _hip
    _build.build(verbose=False)
    return _hip.load()


def cache(**kw):
    from indextts import _hip
    d = dict(k=4096, v=8192, k_scale=1, v_scale=1, bs=4 * 32 * 64, hs=32 * 64, sbs=128, shs=32, rows=2, heads=4, max_kv=32,
             head_dim=64, dtype=_hip.E4M3)
    d.update(kw)
    return _hip.KvCache(**d)


BAD_CACHES = [dict(head_dim=80), dict(rows=0), dict(heads=0), dict(max_kv=0), dict(max_kv=(1 << 20) + 1), dict(k=None),
              dict(k=4097), dict(hs=32 * 64 - 16), dict(bs=8), dict(hs=32 * 64 + 8), dict(k_scale=None), dict(shs=31),
              dict(sbs=16), dict(dtype=0), dict(dtype=2)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_refused(lib, bad):
    c = ctypes.byref(cache(**bad))
    assert lib.itts_kv8_write(c, 16, 256, 64, 16, 256, 64, 0, 4, 4, 1, None) != 0
    assert b"itts_kv8_write" in lib.itts_last_error()
    assert lib.itts_kv8_read(c, 4, 4, 1, 16, 256, 64, 16, 256, 64, 0, None) != 0
    assert lib.itts_attn_decode_kv8(c, 16, 256, 64, 0, 1, 1, 4, None, None, 0, 1.0, 32, 16, 256, 64, 0, 16, None) != 0
    assert lib.itts_attn_tree(c, 16, 256, 256, 64, 0, 1, 1, 1, 4, None, None, 8, 1, None, 0, 1.0, 32, 16, 256, 256, 64, 0, 16,
                              None) != 0
    assert lib.itts_attn_cached_workspace_bytes(c, 1, 1, 1, 32, 0) == -1


def test_kv8_calls_refuse(lib):
    c = ctypes.byref(cache())
    assert lib.itts_kv8_write(None, 16, 256, 64, 16, 256, 64, 0, 4, 4, 1, None) != 0
    assert lib.itts_kv8_write(c, 16, 256, 64, 16, 256, 64, 2, 4, 4, 1, None) != 0  # f16
    assert lib.itts_kv8_write(c, None, 256, 64, 16, 256, 64, 0, 4, 4, 1, None) != 0
    assert lib.itts_kv8_write(c, 16, 256, 64, 16, 256, 64, 0, None, 4, 1, None) != 0
    assert lib.itts_kv8_write(c, 16, 256, 64, 16, 256, 64, 0, 4, 4, -1, None) != 0
    assert lib.itts_kv8_write(c, None, 256, 64, None, 256, 64, 0, None, None, 0, None) == 0  # nothing to do
    bf = ctypes.byref(cache(dtype=1, k_scale=None, v_scale=None))
    assert lib.itts_kv8_write(bf, 16, 256, 64, 16, 256, 64, 0, 4, 4, 1, None) != 0
    assert lib.itts_attn_decode_kv8(bf, 16, 256, 64, 0, 1, 1, 4, None, None, 0, 1.0, 32, 16, 256, 64, 1, 16, None) != 0


def test_attention_calls_refuse(lib):
    c = ctypes.byref(cache())

    def decode(q=16, q_dtype=0, B=1, group=1, kv_len=4, rows=None, ld=0, max_len=32, out=16, out_dtype=0):
        return lib.itts_attn_decode_kv8(c, q, 256, 64, q_dtype, B, group, kv_len, None, rows, ld, 1.0, max_len, out, 256,
                                        64, out_dtype, 16, None)

    for kw in (dict(q=None), dict(q_dtype=2), dict(B=-1), dict(B=3), dict(group=0), dict(group=4097), dict(kv_len=None),
               dict(rows=4, ld=31, B=2), dict(max_len=-1), dict(out=None), dict(out_dtype=2), dict(B=1 << 24, rows=4, ld=32)):
        assert decode(**kw) != 0, kw
        assert b"itts_attn_decode_kv8" in lib.itts_last_error()
    assert decode(B=0) == 0

    def tree(c=c, T=2, mask=8, out_dtype=0, B=1):
        return lib.itts_attn_tree(c, 16, 512, 256, 64, 0, B, T, 1, 4, None, None, mask, T, None, 0, 1.0, 32, 16, 512, 256, 64,
                                  out_dtype, 16, None)

    assert tree(T=0) != 0 and tree(T=65) != 0 and tree(mask=None) != 0 and tree(B=3) != 0
    bf = ctypes.byref(cache(dtype=1, k_scale=None, v_scale=None))
    assert tree(c=bf, out_dtype=0) != 0  # f32 outputs over a bf16 cache
    assert tree(B=0) == 0
    assert lib.itts_attn_cached_workspace_bytes(c, 1, 65, 1, 32, 0) == -1
    assert lib.itts_attn_cached_workspace_bytes(c, 1, 1, 1, 32, 2) == -1
    assert lib.itts_attn_cached_workspace_bytes(c, 1, 1, 1, 32, 0) >= 0


def test_linear_calls_refuse(lib):
    def quant(x=16, ldx=200, dtype=0, M=2, K=200, q=16, ldq=256, s=4, lds=4):
        return lib.itts_fp8_quant_rows(x, ldx, dtype, M, K, q, ldq, s, lds, None)

    for kw in (dict(x=None), dict(ldx=199), dict(dtype=2), dict(M=-1), dict(K=0), dict(ldq=240), dict(ldq=264), dict(q=8),
               dict(s=2), dict(lds=2), dict(lds=6)):
        assert quant(**kw) != 0, kw
    assert quant(M=0, x=None) == 0

    def linear(x=16, ldx=200, xd=0, M=2, K=200, w=16, ldw=256, ws=4, lds=4, N=8, act=0, res=None, ldr=8, y=16, ldy=8, od=0,
               wk=16):
        return lib.itts_fp8_linear(x, ldx, xd, M, K, w, ldw, ws, lds, N, None, act, res, ldr, y, ldy, od, wk, None)

    for kw in (dict(x=None), dict(ldx=199), dict(xd=2), dict(M=-1), dict(K=0), dict(N=0), dict(w=8), dict(ldw=128),
               dict(ldw=260), dict(ws=None), dict(lds=3), dict(act=3), dict(act=-1), dict(res=16, ldr=7), dict(y=None),
               dict(ldy=7), dict(od=2), dict(wk=8), dict(M=1 << 40), dict(M=4096, N=4096, ldy=4096, wk=None)):
        assert linear(**kw) != 0, kw
        assert b"itts_fp8_linear" in lib.itts_last_error()
    assert linear(M=0, x=None, y=None, wk=None) == 0
    assert lib.itts_fp8_linear_workspace_bytes(-1, 8, 8) == -1
    assert lib.itts_fp8_linear_workspace_bytes(3, 8, 200) == 0
    assert lib.itts_fp8_linear_workspace_bytes(5000, 4096, 200) >= 5000 * (256 + 4)


def test_python_refusals_without_gpu():
    from indextts.gpt.kv8 import Kv8Cache, Kv16Cache
    from indextts.utils.fp8 import Fp8Linear, quant_rows
    with pytest.raises(ValueError):
        quant_rows(torch.zeros(2, 8))
    with pytest.raises(ValueError):
        Fp8Linear(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 100)
    with pytest.raises(ValueError):
        Fp8Linear(torch.zeros(4, 100, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 100)
    with pytest.raises(ValueError):
        Kv8Cache.empty(1, 2, 8, 64, device="cpu")
    with pytest.raises(ValueError):
        Kv16Cache(torch.zeros(1, 2, 8, 96, dtype=torch.bfloat16), torch.zeros(1, 2, 8, 96, dtype=torch.bfloat16))


def test_tree_mask():
    from indextts.gpt.kv8 import tree_mask
    par = torch.tensor([[-1, 0, 0, 1, 3], [-1, -1, 1, 2, 9]])
    want = [[1, 3, 5, 11, 27], [1, 2, 6, 14, 16]]  # a parent that is no earlier token counts as none
    assert tree_mask(par).tolist() == want
    chain = tree_mask(torch.arange(-1, 63))
    assert [int(m) & ((1 << 64) - 1) for m in chain] == [(1 << t + 1) - 1 for t in range(64)]
    with pytest.raises(ValueError):
        tree_mask(torch.zeros(65, dtype=torch.int64))


def test_scale_rule_of_the_plain_form():
    """The definition that the GPU tests hold the kernels to: 448 fits a scale of one, the next value does not."""
    from eightbit_util import quant64
    x = torch.zeros(5, 128, dtype=torch.float64)
    x[0, 3], x[1, 3], x[2, 3], x[3, 3] = 448.0, torch.nextafter(torch.tensor(448.0), torch.tensor(1e9)).double(), 2.0 ** -149, \
        3.4028234663852886e38
    _, e = quant64(x)
    assert e.tolist() == [0, 1, -126, 120, 0]
