"""GPU checks of a speculative step over the paged cache: rotary positions per token
(vspec_rocm_rope), attention of a drafted tree (vspec_rocm_paged_tree_attention) and the accepted
path kept (vspec_rocm_kv_accept), against plain 64-bit computations."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, INT4 = 0, 1, 2
DTYPES = pytest.mark.parametrize("dtype", [F32, F16, INT4], ids=["f32", "f16", "int4"])


@pytest.fixture(scope="module")
def vr():
    import torch
    import vspec_rocm

    if not torch.cuda.is_available():
        pytest.fail("no GPU visible for a gpu-marked test")
    vspec_rocm.lib()
    return vspec_rocm


def _int(x, **kw):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda", **kw)


class Cache:
    """A pool whose unused memory holds NaN patterns, and the sequences' rows in it."""

    def __init__(self, vr, dtype, starts, nodes, Hkv, D, P=16, seed=0, spare=3, scale=1.0, outliers=0.0, num_blocks=None):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vr, self.dtype, self.starts, self.nodes = vr, dtype, list(starts), nodes
        need = [max(1, -(-(n + nodes) // P)) for n in starts]
        num_blocks = num_blocks or sum(need) + spare
        self.pool = vr.PagedPool(dtype, num_blocks, P, Hkv, D)
        for t in (self.pool.k, self.pool.v):
            t.view(torch.uint8).fill_(0xFF)
        if dtype == INT4:
            self.pool.ks.fill_(0x7E00)
            self.pool.vs.fill_(0x7E00)
        perm = torch.randperm(min(num_blocks, sum(need) + spare), generator=torch.Generator().manual_seed(seed))
        perm = num_blocks - 1 - perm  # the blocks at the far end of a large pool
        tables = torch.full((len(starts), max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = perm[at:at + n]
            at += n
        self.tables = tables.cuda()
        src = torch.float32 if dtype == F32 else torch.float16
        self.rows = []
        for b, n in enumerate(starts):
            k, v = (torch.randn((1, n + nodes, Hkv, D), generator=g, device="cuda") * scale for _ in range(2))
            if outliers:
                k = torch.where(torch.rand(k.shape, generator=g, device="cuda") < outliers, k * 40, k)
            if n + nodes:
                vr.kv_append(self.pool, self.tables[b:b + 1], _int([0]), k.to(src), v.to(src))
        self.start = _int(self.starts)

    def stored(self, b):
        """K and V [n][Hkv][D] in 64 bits, as the pool holds them."""
        n = self.starts[b] + self.nodes
        k, v, _, _ = self.vr.kv_gather(self.pool, self.tables[b:b + 1], _int([n]), out_mode=self.vr.GATHER_F32)
        return k.double(), v.double()


def _clip(x, three, alpha=4.5):
    import torch

    th = (alpha * x.var(-1, correction=0, keepdim=True).sqrt()).clamp(min=1e-6)
    if three:
        th = th.clamp(max=16.0)
    return torch.minimum(torch.maximum(x, -th), th)


def _attend(k, v, q, sees, three=False, scale=None, alpha=4.5):
    """q [N][Hq][D], k and v [T][Hkv][D], sees [N][T]: 64-bit attention; rows that see nothing: 0."""
    import torch

    N, Hq, D = q.shape
    group = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    q, k = _clip(q.double(), three, alpha), _clip(k, three, alpha)
    out = torch.zeros((N, Hq, D), dtype=torch.float64, device=q.device)
    for h in range(Hq):
        s = (q[:, h] @ k[:, h // group].t().contiguous()) * scale
        if three:
            s = s.clamp(-24, 24)
        s = s.masked_fill(~sees, -math.inf)
        p = torch.softmax(s, -1)
        live = sees.any(-1)
        out[live, h] = p[live] @ torch.where(sees.any(0)[:, None], v[:, h // group], 0.0)
    return out


def _trees(batch, nodes, seed, kind):
    """Node counts and ancestor bits; kind "empty" leaves rows without a visible node."""
    r = np.random.RandomState(seed)
    lens, masks = [], []
    for b in range(batch):
        m = int(r.randint(0, nodes + 1)) if kind in ("ragged", "empty") else nodes
        bits = []
        for i in range(nodes):
            own = 0 if kind == "empty" and r.rand() < 0.5 else 1 << i
            bits.append(own | (bits[r.randint(0, i)] if i else 0))
        if kind == "ragged":  # bits of nodes that are not there say nothing
            bits = [x | ((1 << 64) - (1 << nodes)) | 1 << (nodes - 1) for x in bits]
        lens.append(m)
        masks.append(bits)
    return lens, masks


def _signed(x):
    return x - (1 << 64) if x >> 63 else x


def _sees(start, nodes, m, bits):
    import torch

    out = torch.zeros((nodes, start + nodes), dtype=torch.bool)
    for i in range(m):
        out[i, :start] = True
        for j in range(m):
            out[i, start + j] = bool(bits[i] >> j & 1)
    return out.cuda()


def _tolerance(io, vmax):
    """f32 rows: queries, keys' products and weights keep 22 bits, the sums are f32: a score of at most
    ~11 (log2 units, Cauchy-Schwarz on rows of deviation 1, D = 128) moves by 11 * 2^-21, each weight by that
    times ln 2 and 2^-22 of itself, so an output by 2 * (11 * 2^-21 * 0.7 + 2^-22) < 9e-6 of max |v|.
    f16 rows: half a step, 2^-11 of max |v|, for each of the output, the weights, an int4 pool's values
    and a clipped query."""
    return 9e-6 * vmax if io == "f32" else 4 * 2.0 ** -11 * vmax


def _check(vr, c, N, Hq, io, kind, three, seed=0, qscale=1.0, **kw):
    import torch

    D = c.pool.head_dim
    B = len(c.starts)
    g = torch.Generator(device="cuda").manual_seed(seed + 77)
    q = (torch.randn((B, N, Hq, D), generator=g, device="cuda") * qscale).to(torch.float32 if io == "f32" else torch.float16)
    if kind == "chain":
        lens, masks = [N] * B, [[(2 << i) - 1 for i in range(N)]] * B
        tl = tm = None
    else:
        lens, masks = _trees(B, N, seed, kind)
        tl = _int(lens) if kind != "tree" else None
        tm = torch.tensor([[_signed(x) for x in m] for m in masks], device="cuda")
    out = torch.full_like(q, 7.0)
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q, tree_mask=tm, tree_lens=tl, out=out,
                                  numerics=vr.NUMERICS_3BIT if three else vr.NUMERICS_PLAIN, **kw)
    assert got is out
    for b in range(B):
        k, v = c.stored(b)
        want = _attend(k, v, q[b], _sees(c.starts[b], N, lens[b], masks[b]), three)
        tol = _tolerance(io, max(1.0, float(v.abs().max())))
        err = float((got[b].double() - want).abs().max())
        assert err <= tol, (b, err, tol)  # (also false for NaN)
    return got


SHAPES = [  # Hq, Hkv, D, P
    (8, 2, 128, 16), (4, 4, 64, 16), (12, 4, 128, 32), (6, 1, 64, 64), (16, 2, 128, 48), (33, 3, 128, 16),
]


@DTYPES
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind,N,three", [("chain", 1, True), ("tree", 7, False), ("ragged", 16, True), ("empty", 33, False), ("ragged", 64, True)])
def test_tree_attention(vr, dtype, io, shape, kind, N, three):
    Hq, Hkv, D, P = shape
    starts = [0, 1, 15, 16, 31, 70, 257, 0, 700]
    c = Cache(vr, dtype, starts, N, Hkv, D, P, seed=N)
    _check(vr, c, N, Hq, io, kind, three, seed=N + Hq)


@DTYPES
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_tree_attention_long(vr, dtype, io):
    """Few sequences with long prefixes: parts of a prefix are joined."""
    c = Cache(vr, dtype, [20011, 3, 4096], 19, 2, 128, 16, seed=5)
    _check(vr, c, 19, 8, io, "ragged", True, seed=5)


@DTYPES
@pytest.mark.parametrize("N,batch", [(1, 1), (64, 1), (5, 70)])
def test_tree_attention_batches(vr, dtype, N, batch):
    c = Cache(vr, dtype, [(37 * b + 11) % 400 for b in range(batch)], N, 2, 64, 16, seed=9)
    _check(vr, c, N, 8, "f32", "tree" if N > 1 else "chain", False, seed=9)


@DTYPES
@pytest.mark.parametrize("three", [False, True])
def test_tree_attention_outlier_keys(vr, dtype, three):
    """Keys with outliers reach the clip to 4.5 deviations in most tiles."""
    c = Cache(vr, dtype, [300, 45], 16, 2, 128, 16, seed=21, outliers=0.01)
    _check(vr, c, 16, 8, "f32", "tree", three, seed=3)


@DTYPES
@pytest.mark.parametrize("kscale,qscale", [(1e-3, 1e3), (200.0, 5e-3), (1e-3, 1.0)])
def test_tree_attention_ranges(vr, dtype, kscale, qscale):
    c = Cache(vr, dtype, [130], 9, 2, 128, 16, seed=22, scale=kscale)
    import torch

    q = torch.randn((1, 9, 8, 128), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") * qscale
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q)
    k, v = c.stored(0)
    want = _attend(k, v, q[0], _sees(130, 9, 9, [(2 << i) - 1 for i in range(9)]))
    assert float((got[0].double() - want).abs().max()) <= 9e-6 * float(v.abs().max())


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_tree_attention_int4_large_scales(vr, io):
    """int4 values beyond what one f16 holds: code * scale reaches 8 * 65504."""
    import torch

    c = Cache(vr, INT4, [100], 8, 1, 128, 16, seed=23)
    big = torch.randint(0, 2, c.pool.vs.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    live = (c.pool.vs & 0x7C00) != 0x7C00
    c.pool.vs.copy_(torch.where(live & (big == 1), torch.full_like(c.pool.vs, 0x7BFF), c.pool.vs))
    q = torch.randn((1, 8, 4, 128), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    q = q if io == "f32" else q.half()
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q)
    k, v = c.stored(0)
    want = _attend(k, v, q[0], _sees(100, 8, 8, [(2 << i) - 1 for i in range(8)]))
    if io == "f32":
        assert float((got[0].double() - want).abs().max()) <= 9e-6 * float(v.abs().max())
    else:
        # past the largest f16 an output is infinite, as its rounding is; within half the largest it is held to
        # the weights' and values' steps relative to max |v|
        fits = want.abs() < 60000
        tol = 4 * 2.0 ** -11 * float(v.abs().max())
        assert bool(((got[0].double() - want).abs()[fits] <= tol).all() or not fits.any())
        assert bool(torch.isinf(got[0][want.abs() > 65520 + tol]).all())


@DTYPES
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 6e4])
def test_tree_attention_hidden_nodes_stay_hidden(vr, dtype, io, bad):
    """A node with non-finite keys and values reaches only the rows that see it."""
    import torch

    N, start = 20, 37
    c = Cache(vr, dtype, [start], N, 2, 128, 16, seed=31)
    q = torch.randn((1, N, 8, 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    q = q if io == "f32" else q.half()
    bits = [1 | 1 << i for i in range(N)]  # a root with leaves
    hidden = [3, 11, 12]
    tm = torch.tensor([bits], device="cuda")
    want = vr.paged_tree_attention(c.pool, c.tables, c.start, q, tree_mask=tm)
    for j in hidden:
        pos = start + j
        slot, blk = pos % 16, int(c.tables[0, pos // 16])
        if dtype == INT4:
            s16 = int(torch.tensor(bad, dtype=torch.float16).view(torch.int16))
            c.pool.ks.view(-1, 2, 4, 16)[blk, :, :, slot] = s16  # group-major
            c.pool.vs.view(-1, 2, 16, 4)[blk, :, slot] = s16
        else:
            c.pool.k.view(-1, 2, 16, 128)[blk, :, slot] = bad
            if dtype == F32:
                c.pool.v.view(-1, 2, 16, 128)[blk, :, slot] = bad
            else:
                c.pool.v.view(-1, 2, 4, 128, 4)[blk, :, slot // 4, :, slot % 4] = bad
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q, tree_mask=tm)
    rows = [i for i in range(N) if i not in hidden]
    assert torch.equal(got[0, rows], want[0, rows])
    if not math.isfinite(bad) and dtype != INT4:
        assert bool((~torch.isfinite(got[0, hidden])).any(-1).all())


@DTYPES
def test_tree_attention_table_limits(vr, dtype):
    """Entries that name no block hide their tokens; slots behind the table are not there."""
    import torch

    N, P = 24, 16
    c = Cache(vr, dtype, [70, 200, 500, 90], N, 2, 128, P, seed=41)
    keep = c.tables.clone()
    T = c.tables.shape[1] * P  # every slot of the tables, those that were never written too
    kv = [[x.double() for x in vr.kv_gather(c.pool, c.tables[b:b + 1], _int([T]), out_mode=vr.GATHER_F32)[:2]] for b in range(4)]
    t = c.tables.clone()
    t[0, 2] = -1                       # inside the prefix
    t[1, 5] = c.pool.num_blocks        # a block that is not there
    t[1, 12] = -7                      # first nodes
    q = torch.randn((4, N, 8, 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    start = _int([70, 200, 70000, -5])  # behind the table; a negative start is 0
    got = vr.paged_tree_attention(c.pool, t, start, q, max_start_pos=t.shape[1] * P)
    assert torch.equal(c.tables, keep)
    for b, s in enumerate([70, 200, T, 0]):
        k, v = kv[b]
        sees = _sees(s, N, N, [(2 << i) - 1 for i in range(N)])[:, :T]
        for e in range(t.shape[1]):
            if not 0 <= int(t[b, e]) < c.pool.num_blocks:
                sees[:, e * P:(e + 1) * P] = False
        k, v = k[:sees.shape[1]], v[:sees.shape[1]]
        want = _attend(k, v, q[b], sees)
        if s == T:  # its prefix holds the slots that were never written: NaN is what they say
            assert bool(want.isnan().all()) and bool(got[b].isnan().all())
        else:
            seen = v[sees.any(0)]
            assert float((got[b].double() - want).abs().max()) <= 9e-6 * float(seen.abs().max()), b


@DTYPES
def test_tree_attention_short_bound(vr, dtype):
    """max_start_pos plans the split only: a longer prefix is still read whole."""
    import torch

    c = Cache(vr, dtype, [900, 3], 5, 2, 64, 16, seed=42)
    q = torch.randn((2, 5, 4, 64), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q, max_start_pos=17)
    for b in range(2):
        k, v = c.stored(b)
        want = _attend(k, v, q[b], _sees(c.starts[b], 5, 5, [(2 << i) - 1 for i in range(5)]))
        assert float((got[b].double() - want).abs().max()) <= 9e-6 * float(v.abs().max())


@DTYPES
def test_tree_attention_partly_filled_blocks(vr, dtype):
    """block_used: slots at or above their block's count are skipped."""
    import torch

    P, N = 16, 6
    c = Cache(vr, dtype, [80, 32], N, 2, 128, P, seed=43)
    used = torch.full_like(c.tables, P)
    used[0, 1], used[0, 3], used[0, 5] = 5, 1, N
    used[1, 0], used[1, 2] = 0, N
    q = torch.randn((2, N, 8, 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q, block_used=used)
    for b in range(2):
        k, v = c.stored(b)
        sees = _sees(c.starts[b], N, N, [(2 << i) - 1 for i in range(N)])
        slot = torch.arange(sees.shape[1], device="cuda")
        sees &= (slot % P < used[b].long()[slot // P])[None]
        assert float((got[b].double() - _attend(k, v, q[b], sees)).abs().max()) <= 9e-6 * float(v.abs().max())


@DTYPES
def test_tree_attention_is_the_decode_for_one_node(vr, dtype):
    """One node in slot ctx - 1: the decode's own result, at its tolerances."""
    import torch

    ctx = [1, 17, 300, 1025]
    c = Cache(vr, dtype, [n - 1 for n in ctx], 1, 2, 128, 16, seed=44)
    q = torch.randn((4, 8, 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    for mode in (vr.NUMERICS_PLAIN, vr.NUMERICS_3BIT):
        a = vr.paged_decode(c.pool, c.tables, _int(ctx), q, numerics=mode)
        b = vr.paged_tree_attention(c.pool, c.tables, c.start, q[:, None].contiguous(), numerics=mode)[:, 0]
        vmax = max(float(c.stored(i)[1].abs().max()) for i in range(4))
        assert float((a - b).abs().max()) <= (2.5e-4 * vmax + 4e-5 if dtype == INT4 else 4e-5)


@DTYPES
def test_tree_attention_repeats_and_graphs(vr, dtype):
    """The same bits every time: eager, on another stream, and replayed from a graph with eager work between."""
    import torch

    c = Cache(vr, dtype, [1500, 77, 0], 12, 2, 128, 16, seed=45)
    q = torch.randn((3, 12, 8, 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").half()
    q2 = torch.randn((3, 12, 8, 128), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").half()
    args = dict(max_start_pos=1500)
    want, want2 = (vr.paged_tree_attention(c.pool, c.tables, c.start, x, **args) for x in (q, q2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = vr.paged_tree_attention(c.pool, c.tables, c.start, q, stream=side, **args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs of one library, replayed in turn
    x, y = torch.empty_like(q), torch.empty_like(q)
    graphs = []
    for buf in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = vr.paged_tree_attention(c.pool, c.tables, c.start, buf, **args)
        graphs.append((g, out))
    for turn in range(4):
        a, b = (q, q2) if turn % 2 == 0 else (q2, q)
        x.copy_(a)
        y.copy_(b)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        wa, wb = (want, want2) if turn % 2 == 0 else (want2, want)
        assert torch.equal(graphs[0][1], wa) and torch.equal(graphs[1][1], wb), turn
        assert torch.equal(vr.paged_tree_attention(c.pool, c.tables, c.start, a, **args), wa)


@pytest.mark.parametrize("dtype", [F16, INT4], ids=["f16", "int4"])
def test_tree_attention_far_blocks(vr, dtype):
    """Blocks whose offsets pass 32 bits."""
    P, Hkv, D = 16, 8, 128
    num = ((1 << 32) // (Hkv * P * D * 2) if dtype == F16 else (1 << 32) // (Hkv * P * D // 2)) + 200
    c = Cache(vr, dtype, [500, 20], 9, Hkv, D, P, seed=46, num_blocks=num)
    assert int(c.tables.max()) > num - 100
    _check(vr, c, 9, 16, "f32", "tree", False, seed=6)


# ---- accepted paths ---------------------------------------------------------------------------


def _raw(vr, pool):
    """Every slot of every block, in the raw format: [block][slot] rows."""
    import torch

    tables = torch.arange(pool.num_blocks, dtype=torch.int32, device="cuda")[None]
    n = pool.num_blocks * pool.block_tokens
    got = [x for x in vr.kv_gather(pool, tables, _int([n]), out_mode=vr.GATHER_RAW) if x is not None]
    got = [x.view(torch.int32) if x.dtype == torch.float32 else x.view(torch.int16) if x.dtype == torch.float16 else x for x in got]
    if pool.kf is not None:
        words = pool.kf.view(pool.num_blocks, pool.num_kv_heads, -1)
        bits = (words[..., None] >> torch.arange(16, device="cuda")) & 1
        got.append(bits.flatten(2).permute(0, 2, 1).reshape(n, pool.num_kv_heads, 1).int().contiguous())
    return [x.clone() for x in got]


@DTYPES
@pytest.mark.parametrize("Hkv,D,P", [(2, 128, 16), (3, 64, 32), (1, 96, 48)])
@pytest.mark.parametrize("N", [1, 9, 64])
def test_accept(vr, dtype, Hkv, D, P, N):
    import torch

    r = np.random.RandomState(N + D)
    starts = [0, 5, 16, 47, 130, 131, 15]
    paths = [list(range(0, N, 2)), list(r.permutation(N)), [N - 1], [], [int(x) for x in r.randint(0, N, min(N, 12))],
             [0, N - 1, N, 0], [0, -1, 0]]
    width = max(len(p) for p in paths)
    counts = [len(p) for p in paths[:5]] + [2, 1]
    layers = 3
    caches = [Cache(vr, dtype, starts, N, Hkv, D, P, seed=50 + i) for i in range(layers)]
    tables = caches[0].tables
    for c in caches:
        c.pool.k.view(torch.uint8).random_(0, 256)
        c.pool.v.view(torch.uint8).random_(0, 256)
        if dtype == INT4:
            c.pool.ks.random_(0, 1 << 14)
            c.pool.vs.random_(0, 1 << 14)
            c.pool.kf.random_(0, 1 << 16)
    before = [_raw(vr, c.pool) for c in caches]
    pad = _int([p + [-1] * (width - len(p)) for p in paths])
    lens = vr.kv_accept([c.pool for c in caches], tables, caches[0].start, pad, N)
    assert lens.tolist() == [s + n for s, n in zip(starts, counts)]
    slot = lambda b, pos: int(tables[b, pos // P]) * P + pos % P
    for c, old in zip(caches, before):
        want = [x.clone() for x in old]
        for b, (s, p, n) in enumerate(zip(starts, paths, counts)):
            for i in range(n):
                for w, o in zip(want, old):
                    w[slot(b, s + i)] = o[slot(b, s + int(p[i]))]
        for w, g in zip(want, _raw(vr, c.pool)):
            assert torch.equal(w, g)


def test_accept_many_layers_and_bad_entries(vr):
    """More pools than one launch holds; slots without a block are neither read nor written."""
    import torch

    N, P = 8, 16
    caches = [Cache(vr, F16, [12, 40], N, 2, 64, P, seed=60) for _ in range(37)]
    for i, c in enumerate(caches):
        c.pool.k.copy_(torch.randn(c.pool.k.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda"))
    t = caches[0].tables.clone()
    t[0, 1] = -1                      # slots 16.. of the first sequence: nodes 4.. have no block
    before = [_raw(vr, c.pool) for c in caches]
    arr = vr.pool_array([c.pool for c in caches])
    lens = vr.kv_accept(arr, t, _int([12, 40]), _int([[1, 5, 3], [7, 2, -1]]), N)
    assert lens.tolist() == [15, 42]
    at = lambda b, pos: int(t[b, pos // P]) * P + pos % P
    for c, old in zip(caches, before):
        for w, o, g in zip([x.clone() for x in old], old, _raw(vr, c.pool)):
            w[at(0, 12)], w[at(0, 14)] = o[at(0, 13)], o[at(0, 15)]  # node 5 lies in the missing block
            w[at(1, 40)], w[at(1, 41)] = o[at(1, 47)], o[at(1, 42)]
            assert torch.equal(w, g)


def test_accept_in_a_graph(vr):
    """Replays move what is there at the time."""
    import torch

    c = Cache(vr, F16, [20], 8, 2, 64, 16, seed=61)
    ref = Cache(vr, F16, [20], 8, 2, 64, 16, seed=61)
    path = _int([[0, 2, 5, -1]])
    arr, arr2 = vr.pool_array([c.pool]), vr.pool_array([ref.pool])
    g = torch.cuda.CUDAGraph()
    vr.kv_accept(arr, c.tables, c.start, _int([[-1]]), 8)
    with torch.cuda.graph(g):
        lens = vr.kv_accept(arr, c.tables, c.start, path, 8)
    for turn, p in enumerate(([0, 2, 5, -1], [3, 1, 0, 7], [7, 7, 7, 7], [-1] * 4)):
        path.copy_(_int([p]))
        g.replay()
        torch.cuda.synchronize()
        want = vr.kv_accept(arr2, ref.tables, ref.start, _int([p]), 8)
        assert torch.equal(lens, want), turn
        assert torch.equal(c.pool.k.view(torch.int16), ref.pool.k.view(torch.int16))
        assert torch.equal(c.pool.v.view(torch.int16), ref.pool.v.view(torch.int16))


# ---- rotary positions -------------------------------------------------------------------------


def _speeds(R, base, scaling, factor, L, low, high):
    """Radians a position in 64 bits, and the factor on cos and sin."""
    out, m = [], 1.0
    if scaling == 2 and R > 2:
        base = base * factor ** (R / (R - 2))
    for i in range(R // 2):
        f = base ** (-2.0 * i / R)
        keep = 1.0
        if scaling == 1:
            keep = 0.0
        elif scaling == 3:
            keep = min(1.0, max(0.0, (L * f / (2 * math.pi) - low) / (high - low)))
        elif scaling == 4:
            where = lambda n: R * math.log(L / (2 * math.pi * n)) / (2 * math.log(base))
            a, z = max(0, math.floor(where(high))), min(R - 1, math.ceil(where(low)))
            keep = 1.0 - min(1.0, max(0.0, (i - a) / max(z - a, 0.001)))
            m = 0.1 * math.log(factor) + 1.0
        out.append(keep * f + (1 - keep) * f / factor)
    return np.array(out), m


def _rotated(x, pos, R, layout, speeds, m, inverse):
    import torch

    a = pos.double()[:, None] * torch.tensor(speeds, device=x.device)
    c, s = m * a.cos()[:, None], m * a.sin()[:, None] * (-1 if inverse else 1)
    y = x.double().clone()
    i = torch.arange(R // 2, device=x.device)
    e1, e2 = (i, i + R // 2) if layout == 0 else (2 * i, 2 * i + 1)
    x1, x2 = y[..., e1], y[..., e2]
    y[..., e1], y[..., e2] = x1 * c - x2 * s, x1 * s + x2 * c
    return y


def _near(got, want, m=1.0):
    """Half a step of the output's type, plus f32 work: sine and cosine are within 4 * 2^-24 of the angle's
    (2 units of the functions, the fraction's rounding times pi), each product and sum 2^-24 of at most
    |x1| + |x2| and the f16 rounding follows, so 2^-21 m max |x| bounds it for rows below 2^1 deviations."""
    import torch

    step = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[got.dtype]
    top = float(want.abs().max())
    tol = step * want.abs() + 2.0 ** -21 * top + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert bool(((got.double() - want).abs() <= tol).all()), float((got.double() - want).abs().max())


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 64), (128, 64), (128, 118), (80, 32), (2, 2), (256, 256), (24, 6), (100, 60)])
@pytest.mark.parametrize("T,Hq,Hk", [(1, 4, 1), (37, 5, 2), (1030, 2, 2)])
def test_rope(vr, io, layout, D, R, T, Hq, Hk):
    import torch

    g = torch.Generator(device="cuda").manual_seed(D + R + T)
    t = torch.float32 if io == "f32" else torch.float16
    pos = torch.randint(-5, 1 << 20, (T,), generator=g, device="cuda", dtype=torch.int32)
    q, k = (torch.randn((T, h, D), generator=g, device="cuda").to(t) for h in (Hq, Hk))
    speeds, m = _speeds(R, 5e5, 0, 1.0, 0, 1, 4)
    inverse = T == 37
    a, b = vr.rope(pos, q, k, rope_dim=R, base=5e5, layout=layout, inverse=inverse)
    for x, y in ((q, a), (k, b)):
        want = _rotated(x, pos, R, layout, speeds, m, inverse)
        _near(y, want)
        assert torch.equal(y[..., R:], x[..., R:])


@pytest.mark.parametrize("scaling,factor,low,high", [(0, 1.0, 1, 4), (1, 4.0, 1, 4), (2, 8.0, 1, 4), (3, 8.0, 1, 4), (4, 4.0, 1, 32), (4, 40.0, 1, 32), (3, 1.0, 0.5, 3)])
@pytest.mark.parametrize("R,base", [(128, 1e4), (64, 1e6), (2, 1e4), (8, 500.0)])
def test_rope_scalings(vr, scaling, factor, low, high, R, base):
    import torch

    pos = _int([0, 1, 4095, 8192, 131071, 1 << 20, (1 << 31) - 1, -(1 << 31)])
    q = torch.randn((8, 3, 128), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    speeds, m = _speeds(R, base, scaling, factor, 4096, low, high)
    got, none = vr.rope(pos, q, rope_dim=R, base=base, scaling=scaling, factor=factor, trained_len=4096, low=low, high=high)
    assert none is None
    want = _rotated(q, pos, R, 0, speeds, m, False)
    # at 2^31 positions the 64-bit angles themselves differ by a few 2^-53 * 2^31 radians
    _near(got[:6], want[:6])
    assert float((got[6:].double() - want[6:]).abs().max()) <= 2.0 ** -18 * float(q.abs().max()) + 2.0 ** -21 * m * 8
    again = vr.rope(pos, q, rope_dim=R, base=base, scaling=scaling, factor=factor, trained_len=4096, low=low, high=high, magnitude=0.5)[0]
    _near(again[:6], _rotated(q, pos, R, 0, speeds, 0.5, False)[:6])


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("layout", [0, 1])
def test_rope_strides_and_in_place(vr, io, layout):
    """Slices of a packed projection, transposed heads, rows off a 16-byte boundary, and in place: the
    dense call's bits, and nothing else written."""
    import torch

    T, D, R = 61, 64, 48
    t = torch.float32 if io == "f32" else torch.float16
    g = torch.Generator(device="cuda").manual_seed(2)
    pos = torch.randint(0, 9000, (T,), generator=g, device="cuda", dtype=torch.int32)
    for offset in (0, 1):
        buf = torch.randn(T * (6 + 2 + 2) * D + 8, generator=g, device="cuda").to(t)
        x = buf[offset:offset + T * 10 * D].view(T, 10, D)
        q, k = x[:, :6], x[:, 6:8]
        a, b = vr.rope(pos, q.contiguous(), k.contiguous(), rope_dim=R, layout=layout)
        c, d = vr.rope(pos, q, k, rope_dim=R, layout=layout)
        assert torch.equal(a, c) and torch.equal(b, d)
        heads_first = torch.empty((6, T, D), dtype=t, device="cuda").transpose(0, 1)
        e, _ = vr.rope(pos, q, rope_dim=R, layout=layout, q_out=heads_first)
        assert e is heads_first and torch.equal(e, a)
        keep = buf.clone()
        vr.rope(pos, q, k, rope_dim=R, layout=layout, q_out=q, k_out=k)
        assert torch.equal(q, a) and torch.equal(k, b)
        back = buf.clone()
        back[offset:offset + T * 10 * D].view(T, 10, D)[:, :8] = keep[offset:offset + T * 10 * D].view(T, 10, D)[:, :8]
        assert torch.equal(back, keep)


@pytest.mark.parametrize("layout", [0, 1])
def test_rope_gradient(vr, layout):
    """The inverse call is the gradient: against the formula's transpose and against differences."""
    import torch

    T, H, D, R = 9, 2, 32, 20
    g = torch.Generator(device="cuda").manual_seed(5)
    pos = _int([0, 1, 2, 77, 500, 4096, 9000, 12345, 99999])
    x, w, e = (torch.randn((T, H, D), generator=g, device="cuda") for _ in range(3))
    kw = dict(rope_dim=R, layout=layout, scaling=4, factor=4.0, trained_len=4096, low=1.0, high=32.0)
    grad, _ = vr.rope(pos, w, inverse=True, **kw)
    y = x.double().requires_grad_()
    speeds, m = _speeds(R, 1e4, 4, 4.0, 4096, 1.0, 32.0)
    a = pos.double()[:, None] * torch.tensor(speeds, device="cuda")
    c, s = m * a.cos()[:, None], m * a.sin()[:, None]
    i = torch.arange(R // 2, device="cuda")
    e1, e2 = (i, i + R // 2) if layout == 0 else (2 * i, 2 * i + 1)
    loss = ((y[..., e1] * c - y[..., e2] * s) * w.double()[..., e1]).sum() + ((y[..., e1] * s + y[..., e2] * c) * w.double()[..., e2]).sum()
    loss = loss + (y[..., R:] * w.double()[..., R:]).sum()
    loss.backward()
    _near(grad, y.grad)
    # the map is linear: a difference along e is exact but for f32 rounding, 2^-21 of the sums' terms
    up, down = (vr.rope(pos, x + sign * e, **kw)[0].double() for sign in (1, -1))
    slope = float((((up - down) / 2) * w.double()).sum())
    terms = float((e.double().abs() * grad.double().abs()).sum()) + float((x.double().abs() * w.double().abs()).sum())
    assert abs(slope - float((e.double() * grad.double()).sum())) <= 2.0 ** -20 * terms


def test_rope_in_a_graph(vr):
    import torch

    pos = _int(list(range(50)))
    q = torch.randn((50, 4, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    g = torch.cuda.CUDAGraph()
    vr.rope(pos, q)
    with torch.cuda.graph(g):
        out, _ = vr.rope(pos, q)
    for turn in range(3):
        pos.add_(1000)
        q.mul_(1.5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, vr.rope(pos, q)[0]), turn


# ---- together ---------------------------------------------------------------------------------


@DTYPES
def test_speculative_step(vr, dtype):
    """rope -> append -> tree attention -> accept: the cache afterwards is the one into which the
    accepted tokens alone were appended, byte for byte, each node's output is the one that a decode
    along its own path gives, and a second step goes on from there."""
    import torch

    Hq, Hkv, D, P, N = 8, 2, 64, 16, 7
    starts = [0, 33, 250]
    src = torch.float32 if dtype == F32 else torch.float16
    c = Cache(vr, dtype, starts, 2 * N, Hkv, D, P, seed=70)
    plain = Cache(vr, dtype, starts, 2 * N, Hkv, D, P, seed=70)
    parent = [-1, 0, 0, 1, 1, 2, 4]
    depth, bits = [], []
    for i, a in enumerate(parent):
        depth.append(0 if a < 0 else depth[a] + 1)
        bits.append((bits[a] if a >= 0 else 0) | 1 << i)
    mask = torch.tensor([bits] * 3, device="cuda")
    paths = [[0, 1, 4, 6], [0], [0, 2, 5]]
    path = _int([p + [-1] * (4 - len(p)) for p in paths])
    g = torch.Generator(device="cuda").manual_seed(71)
    start = c.start
    host = list(starts)
    for step in range(2):
        q, k, v = (torch.randn((3, N, h, D), generator=g, device="cuda").to(src) for h in (Hq, Hkv, Hkv))
        pos = (start[:, None] + _int(depth)).flatten()
        qr, kr = vr.rope(pos, q.flatten(0, 1), k.flatten(0, 1))
        qr, kr = qr.view(3, N, Hq, D), kr.view(3, N, Hkv, D)
        vr.kv_append(c.pool, c.tables, start, kr, v)
        out = vr.paged_tree_attention(c.pool, c.tables, start, qr, tree_mask=mask, max_start_pos=max(host))
        lens = vr.kv_accept([c.pool], c.tables, start, path, N)
        for i in range(max(len(p) for p in paths)):
            rows = [b for b in range(3) if i < len(paths[b])]
            pick = torch.tensor([paths[b][i] for b in rows], device="cuda")
            at = torch.tensor(rows, device="cuda")
            pos_i = _int([host[b] + i for b in rows])
            vr.kv_append(plain.pool, plain.tables[at].contiguous(), pos_i, kr[at, pick][:, None].contiguous(), v[at, pick][:, None].contiguous())
            one = vr.paged_decode(plain.pool, plain.tables[at].contiguous(), pos_i + 1, qr[at, pick].float().contiguous())
            vmax = max(float(plain.stored(b)[1].abs().max()) for b in rows)
            # both sides' own tolerances: the decode's, and this one's for its type
            tol = (2.5e-4 * vmax + 2e-5 if dtype == INT4 else 2e-5) + _tolerance("f32" if dtype == F32 else "f16", vmax)
            assert float((one.double() - out[at, pick].double()).abs().max()) <= tol
        host = [h + len(p) for h, p in zip(host, paths)]
        assert lens.tolist() == host
        for b in range(3):
            x = vr.kv_gather(c.pool, c.tables[b:b + 1], lens[b:b + 1])
            y = vr.kv_gather(plain.pool, plain.tables[b:b + 1], lens[b:b + 1])
            assert all(s is None and t is None or torch.equal(s, t) for s, t in zip(x, y))
        if dtype == INT4:  # clamp flags of the kept slots
            for b in range(3):
                for pos_b in range(host[b]):
                    w = [(x.pool.kf.view(-1, Hkv, P // 16)[int(x.tables[b, pos_b // P]), :, pos_b % P // 16] >> pos_b % 16) & 1 for x in (c, plain)]
                    assert torch.equal(*w)
        start = lens
