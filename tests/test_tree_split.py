"""GPU checks of how the attention of a drafted tree is split over ragged batches, of its
workspace, and of shapes at the limits of the speculative step's operators."""
import ctypes as C

import pytest

from test_tree_step import DTYPES, F16, F32, INT4, Cache, _attend, _check, _int, _near, _raw, _rotated, _sees, _speeds, _tolerance, vr  # noqa: F401

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("batch", [64, 65, 130, 256, 257])
def test_batches_past_a_wave(vr, dtype, batch):
    """Lengths are dealt out 64 sequences at a time, and past 256 sequences not at all."""
    starts = [(53 * b + 7) % 90 for b in range(batch)]
    starts[batch // 2], starts[-1] = 1500, 777
    c = Cache(vr, dtype, starts, 3, 1, 64, 16, seed=batch)
    _check(vr, c, 3, 2, "f32", "ragged", False, seed=batch)


@DTYPES
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("N", [5, 20, 40])
def test_one_long_sequence_of_many(vr, dtype, io, N):
    """More (sequence, head) pairs than the card holds workgroups: only the long sequence is cut."""
    starts = [(31 * b) % 60 for b in range(70)]
    starts[13] = 5000
    c = Cache(vr, dtype, starts, N, 8, 64, 16, seed=N)
    _check(vr, c, N, 32, io, "tree", True, seed=N)


@DTYPES
@pytest.mark.parametrize("N,Hq", [(4, 4), (9, 8), (64, 8)])
def test_one_kv_head(vr, dtype, N, Hq):
    """One (sequence, head) pair for the whole card: as many parts as there can be."""
    c = Cache(vr, dtype, [9001], N, 1, 128, 16, seed=N)
    _check(vr, c, N, Hq, "f32", "tree", False, seed=N)


@pytest.mark.parametrize("dtype", [F16, INT4], ids=["f16", "int4"])
def test_more_columns_than_a_workgroup_holds(vr, dtype):
    """64 nodes of 8 query heads: two groups of column tiles."""
    c = Cache(vr, dtype, [2100, 33], 64, 2, 128, 16, seed=71)
    _check(vr, c, 64, 16, "f16", "ragged", True, seed=71)


@DTYPES
@pytest.mark.parametrize("N", [5, 24])
def test_lengths_change_between_replays(vr, dtype, N):
    """A captured call follows the lengths that the device holds: cut another way, or not at all."""
    import torch

    cap = [4000, 2500, 700]
    c = Cache(vr, dtype, cap, N, 2, 64, 16, seed=81)
    q = torch.randn((3, N, 8, 64), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    start = c.start.clone()
    args = dict(max_start_pos=max(cap))
    vr.paged_tree_attention(c.pool, c.tables, start, q, **args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = vr.paged_tree_attention(c.pool, c.tables, start, q, **args)
    kv = [c.stored(b) for b in range(3)]
    for turn, starts in enumerate(([4000, 2500, 700], [3, 0, 650], [0, 0, 0], [17, 2499, 1], [3999, 1, 1])):
        start.copy_(_int(starts))
        g.replay()
        torch.cuda.synchronize()
        for b, s in enumerate(starts):
            k, v = (x[:s + N] for x in kv[b])
            want = _attend(k, v, q[b], _sees(s, N, N, [(2 << i) - 1 for i in range(N)]))
            assert float((out[b].double() - want).abs().max()) <= _tolerance("f32", max(1.0, float(v.abs().max()))), (turn, b)
        assert torch.equal(out, vr.paged_tree_attention(c.pool, c.tables, start, q, **args)), turn


def _desc(vr, c, q, out, max_start, workspace=None, size=0):
    return vr.VspecTreeAttnDesc(c.pool.desc(), q.shape[0], q.shape[2], q.shape[1], c.tables.data_ptr(), c.tables.shape[1], c.start.data_ptr(), max_start,
                                None, None, q.data_ptr(), out.data_ptr(), vr.KV_F32, 0.0, vr.NUMERICS_PLAIN, 0.0, workspace, size,
                                vr._stream(None), None)


@DTYPES
@pytest.mark.parametrize("N", [6, 30])
def test_workspace(vr, dtype, N):
    """What it holds before is not read, what lies behind it is not written, one too small or off its
    alignment is refused, and without one the library brings its own: all the same bits."""
    import torch

    c = Cache(vr, dtype, [3000, 100], N, 2, 128, 16, seed=91)
    q = torch.randn((2, N, 8, 128), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    want = vr.paged_tree_attention(c.pool, c.tables, c.start, q)
    out = torch.empty_like(q)
    need = vr.lib().vspec_rocm_paged_tree_attention_workspace_bytes(C.byref(_desc(vr, c, q, out, 3000)))
    assert need > 0
    buf = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    call = lambda *ws: vr.lib().vspec_rocm_paged_tree_attention(C.byref(_desc(vr, c, q, out, 3000, *ws)))
    assert call(buf.data_ptr(), need) == 1
    torch.cuda.synchronize()
    assert torch.equal(out, want) and bool((buf[need:] == 0xFF).all())
    out.zero_()
    assert call() == 1
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    for ws in ((buf.data_ptr(), need - 1), (buf.data_ptr() + 8, need)):
        assert call(*ws) == 0 and "workspace" in vr.last_error()
    torch.cuda.synchronize()
    assert bool((out == 0).all())


def test_two_streams_at_once(vr):
    """Calls on two streams, each with a workspace of its own."""
    import torch

    c = Cache(vr, F16, [6000, 50], 8, 2, 128, 16, seed=95)
    g = torch.Generator(device="cuda").manual_seed(2)
    qs = [torch.randn((2, 8, 8, 128), generator=g, device="cuda") for _ in range(2)]
    want = [vr.paged_tree_attention(c.pool, c.tables, c.start, q, max_start_pos=6000) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(vr.paged_tree_attention(c.pool, c.tables, c.start, q, max_start_pos=6000))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2]), i


@pytest.mark.parametrize("dtype,D,P", [(INT4, 160, 16), (INT4, 256, 32), (INT4, 32, 16), (F32, 24, 10), (F32, 128, 7), (F16, 8, 16), (F16, 264, 48)])
def test_accept_head_sizes(vr, dtype, D, P):
    """Rows of any length that pools have, more than one pass of them too, and many layers to a workgroup."""
    import torch

    N, starts = 64, [0, 13, 50]
    paths = [list(range(1, 64)) + [-1], [63, 0, 62, 1, 61] + [-1] * 59, list(range(63, -1, -1))]
    need = max(-(-(s + N) // P) for s in starts)
    g = torch.Generator(device="cuda").manual_seed(D)
    tables = torch.randperm(3 * need, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(3, need).cuda()
    pools = []
    for _ in range(2):
        pool = vr.PagedPool(dtype, 3 * need + 1, P, 2, D)
        for t in (pool.k, pool.v):
            t.view(torch.uint8).random_(0, 256, generator=g)
        if dtype == INT4:
            for t, top in ((pool.ks, 1 << 14), (pool.vs, 1 << 14), (pool.kf, 1 << 16)):
                t.random_(0, top, generator=g)
        pools.append(pool)
    before = [_raw(vr, p) for p in pools]
    lens = vr.kv_accept(pools, tables, _int(starts), _int(paths), N)
    assert lens.tolist() == [63, 18, 114]
    slot = lambda b, pos: int(tables[b, pos // P]) * P + pos % P
    for pool, old in zip(pools, before):
        want = [x.clone() for x in old]
        for b, (s, p) in enumerate(zip(starts, paths)):
            for i, node in enumerate(p):
                if node < 0:
                    break
                for w, o in zip(want, old):
                    w[slot(b, s + i)] = o[slot(b, s + node)]
        for w, got in zip(want, _raw(vr, pool)):
            assert torch.equal(w, got)


def test_accept_layers_share_a_workgroup(vr):
    """A batch large enough that a workgroup takes several layers."""
    import torch

    B, N, layers = 200, 8, 5
    starts = [(7 * b) % 40 for b in range(B)]
    caches = [Cache(vr, F16, [0] * B, 48, 8, 64, 16, seed=i) for i in range(layers)]
    tables = caches[0].tables
    for i, c in enumerate(caches):
        for t in (c.pool.k, c.pool.v):
            t.copy_(torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda"))
    before = [_raw(vr, c.pool) for c in caches]
    path = torch.stack([torch.randperm(N, generator=torch.Generator().manual_seed(b)) for b in range(B)]).to(torch.int32).cuda()
    lens = vr.kv_accept([c.pool for c in caches], tables, _int(starts), path, N)
    assert lens.tolist() == [s + N for s in starts]
    at = torch.tensor(starts, device="cuda")[:, None]
    slots = lambda pos: torch.gather(tables.long(), 1, pos // 16) * 16 + pos % 16
    to, source = slots(at + torch.arange(N, device="cuda")), slots(at + path.long())
    for c, old in zip(caches, before):
        for w, o, got in zip([x.clone() for x in old], old, _raw(vr, c.pool)):
            w[to.flatten()] = o[source.flatten()]
            assert torch.equal(w, got)


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("T,Hq,Hk,D,R", [(4099, 2, 1, 64, 48), (2050, 1, 0, 16, 16), (3, 8190, 2, 8, 8), (3, 8190, 3, 8, 8), (9000, 3, 0, 128, 128)])
def test_rope_sizes(vr, io, layout, T, Hq, Hk, D, R):
    """Tokens that share a workgroup, a last one that is not full, and as many heads as chunks are counted for."""
    import torch

    t = torch.float32 if io == "f32" else torch.float16
    g = torch.Generator(device="cuda").manual_seed(T)
    pos = torch.randint(0, 1 << 17, (T,), generator=g, device="cuda", dtype=torch.int32)
    q, k = (torch.randn((T, h, D), generator=g, device="cuda").to(t) if h else None for h in (Hq, Hk))
    speeds, m = _speeds(R, 1e4, 0, 1.0, 0, 1, 4)
    a, b = vr.rope(pos, q, k, rope_dim=R, layout=layout)
    for x, y in ((q, a), (k, b)):
        if x is None:
            assert y is None
            continue
        _near(y, _rotated(x, pos, R, layout, speeds, m, False))
        assert torch.equal(y[..., R:], x[..., R:])


@DTYPES
def test_nothing_to_do(vr, dtype):
    """No tokens, no sequences, a path without entries."""
    import torch

    for t in (torch.float32, torch.float16):
        q, k = (torch.empty((0, h, 64), dtype=t, device="cuda") for h in (4, 1))
        a, b = vr.rope(_int([]), q, k)
        assert a.shape == q.shape and b.shape == k.shape
    c = Cache(vr, dtype, [20], 4, 1, 64, 16, seed=97)
    before = _raw(vr, c.pool)
    none = torch.empty((0, c.tables.shape[1]), dtype=torch.int32, device="cuda")
    out = vr.paged_tree_attention(c.pool, none, _int([]), torch.empty((0, 4, 4, 64), device="cuda"))
    assert out.shape == (0, 4, 4, 64)
    assert vr.kv_accept([c.pool], none, _int([]), torch.empty((0, 4), dtype=torch.int32, device="cuda"), 4).numel() == 0
    assert vr.kv_accept([c.pool], c.tables, c.start, torch.empty((1, 0), dtype=torch.int32, device="cuda"), 4).tolist() == [20]
    for a, b in zip(before, _raw(vr, c.pool)):
        assert torch.equal(a, b)
