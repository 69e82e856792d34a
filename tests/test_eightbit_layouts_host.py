"""8-bit operators without a GPU: layouts of the arguments that the calls derive pitches and offsets from."""
import ctypes

import pytest
import torch


def test_lineage_table_rows_are_read_where_they_are():
    """one table expanded over the rows has row stride 0: no pitch may be made up for it"""
    from indextts.gpt.kv8 import _Cache
    c = object.__new__(_Cache)
    c.rows, c.max_kv, c.index, c.dev = 4, 40, -1, torch.device("cpu")  # get_device() of a CPU tensor is -1
    table = torch.zeros(3, 45, dtype=torch.int32)
    assert c._lineage(table, 3) == (table.data_ptr(), 45)
    assert c._lineage(table[:1].expand(3, -1), 3) == (table.data_ptr(), 0)
    assert c._lineage(table[1:2, 2:], 1) == (table[1, 2:].data_ptr(), 40)
    assert c._lineage(table[:1].expand(1, -1), 1)[1] == 40
    with pytest.raises(ValueError):
        c._lineage(torch.zeros(100, dtype=torch.int32).as_strided((3, 40), (20, 1)), 3)


def test_one_lineage_table_for_all_rows():
    from indextts import _build, _hip
    _build.build(verbose=False)
    lib = _hip.load()
    c = ctypes.byref(_hip.KvCache(k=4096, v=8192, k_scale=1, v_scale=1, bs=4 * 32 * 64, hs=32 * 64, sbs=128, shs=32, rows=2,
                                  heads=4, max_kv=32, head_dim=64, dtype=_hip.E4M3))

    def decode(ld):  # no rows: nothing is launched
        return lib.itts_attn_decode_kv8(c, 16, 256, 64, 0, 0, 1, 4, None, 4, ld, 1.0, 32, 16, 256, 64, 0, 16, None)

    assert decode(0) == 0 and decode(32) == 0 and decode(31) != 0 and decode(-32) != 0


def test_rows_fetched_for_a_tile_of_weights_lie_within_them(tmp_path):
    """csrc/fp8_rows.h as a host program: which row of w is fetched for each of a tile's 256 (or 128) LDS rows"""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "index-tts-dubbing_amd", "csrc")
    src = tmp_path / "rows.cpp"
    src.write_text('#include <cstdio>\n#include "fp8_rows.h"\nint main() { for (int last = 0; last < 256; ++last)'
                   ' for (int i = 0; i < 256; ++i) std::printf("%d ", itts::fetched_row(i, last)); }\n')
    subprocess.run(["g++", "-std=c++17", "-I", csrc, str(src), "-o", str(tmp_path / "rows")], check=True)
    out = subprocess.run([str(tmp_path / "rows")], check=True, capture_output=True, text=True).stdout
    rows = torch.tensor([int(v) for v in out.split()]).view(256, 256)
    assert sorted(rows[255].tolist()) == list(range(256))
    for i in range(256):  # lane r of fragment j: column 16 (r / 4) + 4 j + r % 4 of its wave's 64
        j, r = i >> 4 & 3, i & 15
        assert rows[255, i] == (i & 192) + 16 * (r // 4) + 4 * j + r % 4
    assert torch.equal(rows, torch.minimum(rows[255][None], torch.arange(256)[:, None]))  # never behind the last


def test_where_an_output_may_lie():
    """out beside, over and between q and the cache: exact to the element, also for layouts that interleave"""
    from indextts.gpt.kv8 import _Cache, _distinct, _extent, _meet
    base = torch.zeros(1 << 16, dtype=torch.uint8)

    def places(layout, at):
        el = [0]
        for n, s in zip(layout[0], layout[1]):
            el = [e + i * s for e in el for i in range(n)]
        return [at + e * layout[2] + b for e in el for b in range(layout[2])]

    g = torch.Generator().manual_seed(0)
    for _ in range(300):
        def one():
            shape = tuple(int(v) for v in torch.randint(1, 4, (3,), generator=g)) + (4,)
            return shape, tuple(int(v) for v in torch.randint(0, 40, (3,), generator=g)) + (1,), 2 + 2 * int(torch.randint(2, (1,), generator=g))
        a, b, off = one(), one(), 2 * int(torch.randint(-100, 100, (1,), generator=g))
        pa, pb = places(a, 0), places(b, off)
        assert _meet(a, b, off) == bool(set(pa) & set(pb))
        assert _distinct(*a) == (len(set(pa)) == len(pa))
        assert _extent(*a) == max(pa) + 1

    c = object.__new__(_Cache)
    c.index, c.dev = -1, torch.device("cpu")
    cache = base[8192:8192 + 2 * 2 * 16 * 64].view(2, 2, 16, 64)
    layout = ((2, 2, 16 * 64), (2 * 16 * 64, 16 * 64, 1), 1)
    c._first, c._end = cache.data_ptr(), cache.data_ptr() + cache.numel()
    c._held = [(c._first, c._end, layout)]
    qkv = base[16384:16384 + 3 * 3 * 2 * 64 * 4].view(torch.float32).view(3, 3, 2, 64)
    q = qkv[:, 0]
    for out in (q, qkv[:, 1], qkv[:, 2], q.view(3, 1, 2, 64).squeeze(1), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, dtype=torch.bfloat16),
                base[:768].view(torch.bfloat16).view(3, 2, 64)):
        c._check_out(out, q, out.stride(), q.stride())
    c._check_out(q[:0], q[:0], q.stride(), q.stride())
    flat = qkv.view(-1)
    for out in (flat.as_strided((3, 2, 64), (384, 64, 1), q.storage_offset() + 1),
                flat.as_strided((3, 2, 64), (128, 64, 1), q.storage_offset()),  # rows 1, 2 over q's row 0 .. k
                q.view(torch.bfloat16)[..., :64], q[:1].expand(3, 2, 64), q[:, :1].expand(3, 2, 64),
                cache.view(-1)[64:64 + 768].view(torch.bfloat16).view(3, 2, 64)):
        with pytest.raises(ValueError):
            c._check_out(out, q, out.stride(), q.stride())


def test_the_check_of_the_assembly_products():
    """what _build looks for in the assembly of the products written by hand, on a loop of two of them"""
    from indextts._build import check_products
    good = """_Z5largev:
	v_mov_b32_e32 v40, v41
	s_nop 7
.LBB0_1:                                ; =>This Inner Loop Header: Depth=1
	ds_read_b128 v[8:11], v50
	s_waitcnt lgkmcnt(0)
	v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:7], v[8:15], a[0:3], v40, v42 op_sel_hi:[0,0,0]
	v_add_u32_e32 v60, v61, v62
	v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[16:23], v[8:15], a[4:7], v40, v42 op_sel_hi:[0,0,0]
	s_add_i32 s4, s4, 1
	s_cbranch_scc1 .LBB0_1
	v_accvgpr_read_b32 v0, a0
	s_endpgm
.Lfunc_end0:
"""
    assert check_products(good, "large") == 2 and check_products(good, "other") == 0
    for old, new in (("	v_add_u32_e32 v60, v61, v62", "	v_add_u32_e32 v60, v61, v62\n	v_mov_b32_e32 v17, v62"),
                     ("	s_nop 7\n", ""),
                     ("	s_nop 7\n", "	s_nop 0\n"),
                     ("	s_add_i32 s4, s4, 1", "	v_mov_b32_e32 v42, v43"),  # reaches the first product over the jump
                     ("	v_add_u32_e32 v60, v61, v62", "	v_accvgpr_mov_b32 a9, a0"),
                     ("	v_add_u32_e32 v60, v61, v62", "	v_accvgpr_read_b32 v60, a2"),
                     ("	s_waitcnt lgkmcnt(0)", "	v_lshlrev_b32_e32 v12, 8, v13")):
        bad = good.replace(old, new)
        assert bad != good
        with pytest.raises(RuntimeError):
            check_products(bad, "large")
    assert check_products(good.replace("	s_add_i32 s4, s4, 1", "	v_mov_b32_e32 v42, v43\n	s_nop 3"), "large") == 2
