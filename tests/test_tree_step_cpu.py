"""CPU checks of a speculative step's entry points: the ctypes mirrors' layouts and every refusal,
each before any device work."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest

INC = Path(__file__).resolve().parent.parent / "include"


@pytest.fixture(scope="module")
def vr():
    import vspec_rocm

    vspec_rocm.lib()
    return vspec_rocm


def test_layouts_match_c(vr, tmp_path):
    types = [vr.VspecTreeAttnDesc, vr.VspecRopeRows, vr.VspecRopeDesc]
    lines = []
    for t in types:
        lines.append(f'printf("%zu\\n", sizeof({t.__name__}));')
        lines += [f'printf("%zu\\n", offsetof({t.__name__}, {n.rstrip("_")}));' for n, _ in t._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vspec_rocm.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-std=gnu11", f"-I{INC}", str(src), "-o", str(tmp_path / "p")], check=True)
    out = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for t in types:
        want += [C.sizeof(t)] + [getattr(t, n).offset for n, _ in t._fields_]
    assert out == want


def _kv(vr, dtype=1, **kw):
    kv = vr.VspecPagedKV()
    kv.dtype, kv.num_blocks, kv.block_tokens, kv.num_kv_heads, kv.head_dim = dtype, 64, 16, 2, 128
    kv.k_data, kv.v_data = 1 << 20, 1 << 21
    if dtype == 2:
        kv.k_scales, kv.v_scales = 1 << 22, 1 << 23
    for n, x in kw.items():
        setattr(kv, n, x)
    return kv


def _tree(vr, **kw):
    d = vr.VspecTreeAttnDesc()
    d.kv = _kv(vr)
    d.batch, d.num_q_heads, d.num_nodes, d.max_blocks_per_seq = 2, 8, 8, 16
    d.block_tables = d.start_pos = d.q = d.out = 1 << 20
    d.io_dtype = vr.KV_F16
    for n, x in kw.items():
        if "." in n:
            setattr(d.kv, n[3:], x)
        else:
            setattr(d, n, x)
    return d


@pytest.mark.parametrize("change,word", [
    ({"kv.head_dim": 96}, "head_dim must be 64 or 128"),
    ({"kv.block_tokens": 24}, "multiple of 16"),
    ({"kv.dtype": 3}, "bad dtype"),
    ({"kv.dtype": 2}, "without scales"),
    ({"kv.k_data": None}, "null pool data"),
    ({"kv.num_blocks": 0}, "empty pool"),
    ({"num_nodes": 0}, "1..64"),
    ({"num_nodes": 65}, "1..64"),
    ({"num_q_heads": 0}, "positive multiple"),
    ({"num_q_heads": 7}, "positive multiple"),
    ({"io_dtype": 2}, "io_dtype"),
    ({"numerics": 2}, "numerics"),
    ({"batch": 65536}, "65535"),
    ({"max_blocks_per_seq": 1 << 28}, "2^31"),
    ({"max_start_pos": 257}, "max_start_pos"),
    ({"max_blocks_per_seq": 0}, "null argument"),
    ({"block_tables": None}, "null argument"),
    ({"start_pos": None}, "null argument"),
    ({"q": None}, "null argument"),
    ({"out": None}, "null argument"),
    ({"q": (1 << 20) + 8}, "16-byte"),
    ({"out": (1 << 20) + 4}, "16-byte"),
])
def test_tree_attention_refusals(vr, change, word):
    d = _tree(vr, **change)
    assert vr.lib().vspec_rocm_paged_tree_attention(C.byref(d)) == 0
    assert word in vr.last_error(), vr.last_error()


def test_tree_attention_null_and_empty(vr):
    assert vr.lib().vspec_rocm_paged_tree_attention(None) == 0 and "null" in vr.last_error()
    assert vr.lib().vspec_rocm_paged_tree_attention_workspace_bytes(None) == 0
    d = _tree(vr, batch=0, q=None, out=None, block_tables=None, start_pos=None)
    assert vr.lib().vspec_rocm_paged_tree_attention(C.byref(d)) == 1


@pytest.mark.parametrize("change,word", [
    ({"kvs": []}, "no pools"),
    ({"kvs": [{}, {"dtype": 0}]}, "differs"),
    ({"kvs": [{}, {"num_blocks": 65}]}, "differs"),
    ({"kvs": [{}, {"head_dim": 64}]}, "differs"),
    ({"kvs": [{}, {}]}, "the same"),
    ({"kvs": [{"k_data": (1 << 20) + 8}]}, "16-byte"),
    ({"kvs": [{"block_tokens": 24}]}, "multiple of 16"),
    ({"nodes": 0}, "1..64"),
    ({"nodes": 65}, "1..64"),
    ({"width": 65}, "at most 64"),
    ({"batch": 65536}, "65535"),
    ({"tables": None}, "null argument"),
    ({"start": None}, "null argument"),
    ({"path": None}, "null argument"),
    ({"blocks": 0}, "null argument"),
])
def test_accept_refusals(vr, change, word):
    a = dict(kvs=[{}], batch=2, tables=1 << 20, blocks=16, start=1 << 20, path=1 << 20, width=4, nodes=8)
    a.update(change)
    kvs = (vr.VspecPagedKV * len(a["kvs"]))(*[_kv(vr, **k) for k in a["kvs"]]) if a["kvs"] else None
    assert vr.lib().vspec_rocm_kv_accept(kvs, len(a["kvs"]), a["batch"], a["tables"], a["blocks"], a["start"], a["path"],
                                         a["width"], a["nodes"], None, None) == 0
    assert word in vr.last_error(), vr.last_error()


def test_accept_empty(vr):
    kvs = (vr.VspecPagedKV * 1)(_kv(vr))
    assert vr.lib().vspec_rocm_kv_accept(kvs, 1, 0, None, 0, None, None, 0, 8, None, None) == 1
    assert vr.lib().vspec_rocm_kv_accept(None, 1, 1, None, 0, None, None, 0, 8, None, None) == 0


def _rope(vr, **kw):
    d = vr.VspecRopeDesc()
    d.num_tokens, d.head_dim, d.rope_dim, d.dtype = 4, 128, 128, vr.KV_F16
    d.base, d.factor, d.low, d.high, d.trained_len = 1e4, 4.0, 1.0, 4.0, 4096
    d.positions = 1 << 20
    d.q.in_ = d.q.out = 1 << 20
    d.q.num_heads = 8
    for n, x in kw.items():
        if n[:2] == "q_":
            setattr(d.q, n[2:], x)
        elif n[:2] == "k_":
            setattr(d.k, n[2:], x)
        else:
            setattr(d, n, x)
    return d


@pytest.mark.parametrize("change,word", [
    ({"dtype": 2}, "dtype"),
    ({"layout": 2}, "layout"),
    ({"rope_dim": 0}, "rope_dim"),
    ({"rope_dim": 7}, "rope_dim"),
    ({"rope_dim": 130}, "rope_dim"),
    ({"head_dim": 258, "rope_dim": 2}, "head_dim"),
    ({"base": 1.0}, "base"),
    ({"base": math.nan}, "base"),
    ({"base": math.inf}, "base"),
    ({"scaling": 5}, "scaling"),
    ({"scaling": -1}, "scaling"),
    ({"scaling": 1, "factor": 0.5}, "factor"),
    ({"scaling": 2, "factor": math.nan}, "factor"),
    ({"scaling": 3, "low": 0.0}, "low < high"),
    ({"scaling": 4, "high": 1.0}, "low < high"),
    ({"scaling": 4, "high": math.inf}, "low < high"),
    ({"scaling": 3, "trained_len": 0}, "trained_len"),
    ({"q_out": None}, "q needs"),
    ({"q_in_": None}, "q needs"),
    ({"q_num_heads": 0}, "q needs"),
    ({"k_in_": 1 << 20}, "k needs"),
    ({"q_in_": (1 << 20) + 1}, "aligned"),
    ({"q_in_token_stride": 2048}, "in place"),
    ({"q_num_heads": 65537}, "65536"),
    ({"num_tokens": 1 << 31}, "2^31"),
    ({"positions": None}, "positions"),
])
def test_rope_refusals(vr, change, word):
    d = _rope(vr, **change)
    assert vr.lib().vspec_rocm_rope(C.byref(d)) == 0
    assert word in vr.last_error(), vr.last_error()


def test_rope_null_and_empty(vr):
    assert vr.lib().vspec_rocm_rope(None) == 0 and "null" in vr.last_error()
    assert vr.lib().vspec_rocm_rope(C.byref(_rope(vr, num_tokens=0, positions=None))) == 1
    assert vr.lib().vspec_rocm_rope(C.byref(_rope(vr, q_in_=None, q_out=None, q_num_heads=0, positions=None))) == 1


def test_binding_refusals(vr):
    """The binding refuses data that is not on the current GPU, and pools that their tensors do not fill."""
    import torch

    pool = vr.PagedPool(vr.KV_F16, 4, 16, 1, 64, device="cpu")
    tab, one = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 2, 2, 64))
    for call in (lambda: vr.paged_tree_attention(pool, tab, one, q, max_start_pos=0),
                 lambda: vr.kv_accept([pool], tab, one, torch.zeros((1, 2), dtype=torch.int32), 2),
                 lambda: vr.kv_accept([], tab, one, torch.zeros((1, 2), dtype=torch.int32), 2),
                 lambda: vr.rope(one, q[0]), lambda: vr.rope(one)):
        with pytest.raises(vr.VspecRocmError):
            call()
    k = torch.zeros((4, 1, 16, 64), dtype=torch.float16)
    again = vr.PagedPool.over(vr.KV_F16, 16, 1, 64, k, k.clone())
    assert again.num_blocks == 4 and again.desc().num_blocks == 4
    for args in ((vr.KV_F16, 16, 1, 64, k, k[:2]), (vr.KV_F16, 16, 1, 64, k, None), (vr.KV_F16, 16, 1, 64, k.transpose(0, 2), k),
                 (vr.KV_INT4, 16, 1, 64, k, k)):
        with pytest.raises(vr.VspecRocmError):
            vr.PagedPool.over(*args)
    with pytest.raises(ValueError):
        vr.PagedPool.over(7, 16, 1, 64, k, k)


def test_rope_no_tokens_no_addresses(vr):
    """Empty tensors have no address: nothing to do, not an error."""
    assert vr.lib().vspec_rocm_rope(C.byref(_rope(vr, num_tokens=0, positions=None, q_in_=None, q_out=None))) == 1
