"""Cases of the operators of a speculative step over the paged KV-cache, with their plain forms.

A step drafts a tree of tokens for every sequence, rotates their queries and keys by depth, writes
them behind the cached prefix, attends each node to the prefix and to its ancestors, and keeps the
path that the model agrees with.  Kinds:

  tree    attention of the drafted nodes over an f32, f16 or int4 pool (vspec_rocm.paged_tree_attention)
  accept  the accepted nodes' rows moved behind the prefix, in the pools of all layers (vspec_rocm.kv_accept)
  rope    rotary positions of queries and keys, given for each token (vspec_rocm.rope)

Lengths, trees and paths come from the case and its "mix" number; data, tables and the order of the
blocks from the seed.  Pools are laid out as include/vspec_rocm.h says.
"""
import math
import os
import random
import sys
from types import SimpleNamespace

import torch

own = False

GQA = dict(q_heads=32, kv_heads=8, head_dim=128, block=16)  # the KV shape of bench.py


def listed():
    return [
        # one interactive user, a drafted chain behind a short chat: latency is all there is
        dict(name="tree-f16-b1-chain5", kind="tree", kv="f16", io="f16", batch=1, start_lo=700, start_hi=700, nodes=5, tree="chain", numerics="3bit", mix=0, **GQA),
        # the smallest cache of the tests in the reference cache's own type: 8 heads of 64, no grouping
        dict(name="tree-f32-b1-257", kind="tree", kv="f32", io="f32", batch=1, start_lo=257, start_hi=257, nodes=8, tree="tree", numerics="plain", mix=1,
             q_heads=8, kv_heads=8, head_dim=64, block=16),
        # a small server batch, f32 rows in and out as in the decode step
        dict(name="tree-f16-b16-2k-n16", kind="tree", kv="f16", io="f32", batch=16, start_lo=2049, start_hi=2049, nodes=16, tree="tree", numerics="3bit", mix=2, **GQA),
        # continuous batching: contexts and trees of all sizes, an odd batch and an odd tree
        dict(name="tree-f16-b13-ragged-n27", kind="tree", kv="f16", io="f32", batch=13, start_lo=0, start_hi=8192, nodes=27, tree="ragged", numerics="plain", mix=3, **GQA),
        # a full batch with the largest trees: the most arithmetic a byte of cache
        dict(name="tree-f16-b64-4k-n64", kind="tree", kv="f16", io="f16", batch=64, start_lo=4097, start_hi=4097, nodes=64, tree="tree", numerics="3bit", mix=4, **GQA),
        # the quantised cache: the small batch, and a full ragged one
        dict(name="tree-int4-b16-2k-n16", kind="tree", kv="int4", io="f32", batch=16, start_lo=2049, start_hi=2049, nodes=16, tree="tree", numerics="3bit", mix=5, **GQA),
        dict(name="tree-int4-b64-ragged-n8", kind="tree", kv="int4", io="f16", batch=64, start_lo=128, start_hi=8192, nodes=8, tree="ragged", numerics="3bit", mix=6, **GQA),
        # one user's accepted path in the caches of all layers
        dict(name="accept-f16-b1-n8-l36", kind="accept", kv="f16", batch=1, start_lo=700, start_hi=700, nodes=8, path=5, layers=36, mix=7, **GQA),
        # a full batch with long paths through large trees, quantised caches
        dict(name="accept-int4-b64-n64-l16", kind="accept", kv="int4", batch=64, start_lo=100, start_hi=500, nodes=64, path=24, layers=16, mix=8, **GQA),
        # queries and keys of a step's drafted nodes, far into a long context whose slow pairs are stretched
        dict(name="rope-f16-256-bands", kind="rope", io="f16", tokens=256, pos_lo=100000, pos_hi=131072, rope_dim=128, layout="half", scaling="bands", factor=8.0,
             inverse=False, packed=False, base=5e5, mix=9, **GQA),
        # a prompt's chunk inside its packed projection, interleaved pairs of half of each head
        dict(name="rope-f16-16k-interleaved", kind="rope", io="f16", tokens=16384, pos_lo=0, pos_hi=65536, rope_dim=64, layout="interleaved", scaling="yarn", factor=4.0,
             inverse=False, packed=True, base=1e4, mix=10, **GQA),
        # the gradient's direction, f32
        dict(name="rope-f32-4k-inverse", kind="rope", io="f32", tokens=4099, pos_lo=0, pos_hi=8192, rope_dim=128, layout="half", scaling="none", factor=1.0,
             inverse=True, packed=False, base=1e6, mix=11, **GQA),
    ]


def draw(rng):
    def spread(lo, hi):  # whole numbers, even over their logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    kind = rng.choices(["tree", "accept", "rope"], [4, 1, 2])[0]
    q_heads, kv_heads, head_dim = rng.choice([(32, 8, 128)] * 4 + [(16, 4, 128), (32, 4, 128), (8, 8, 64), (16, 4, 64), (12, 4, 128)])
    c = dict(kind=kind, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, block=rng.choice([16, 16, 16, 32, 64]), mix=rng.randrange(1 << 20))
    if kind == "tree":
        c["kv"], c["io"] = rng.choice(["f16", "f16", "int4", "int4", "f32"]), rng.choice(["f32", "f16"])
        c["nodes"] = spread(1, 64)
        c["tree"] = rng.choice(["chain", "tree", "ragged"])
        c["numerics"] = rng.choice(["3bit", "3bit", "plain"])
        c["batch"] = spread(1, 64)
        row = 2 * kv_heads * head_dim * {"f32": 4, "f16": 2, "int4": 1}[c["kv"]]
        most = min(0.6e9 / row, 3e9 / (c["nodes"] * q_heads * head_dim * (4 if c["kv"] == "f32" else 1)) * 16) / c["batch"]
        c["start_hi"] = spread(1, max(1, min(16384, int(most))))
        c["start_lo"] = c["start_hi"] if rng.random() < 0.4 else c["start_hi"] // rng.choice([2, 8, 64])
    elif kind == "accept":
        c["kv"] = rng.choice(["f16", "int4", "f32"])
        c["batch"], c["layers"] = spread(1, 64), spread(1, 40)
        c["nodes"] = spread(1, 64)
        c["path"] = rng.randint(1, max(1, c["nodes"] // 2))
        c["start_hi"] = spread(1, max(1, min(600, 400000 // (c["batch"] * c["layers"]))))
        c["start_lo"] = c["start_hi"] // 4
    else:
        c["io"] = rng.choice(["f16", "f16", "f32"])
        c["tokens"] = spread(1, 16384)
        c["pos_lo"], c["pos_hi"] = 0, spread(64, 1 << 20)
        c["rope_dim"] = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, head_dim - 10])
        c["layout"] = rng.choice(["half", "interleaved"])
        c["scaling"] = rng.choice(["none", "linear", "base", "bands", "yarn"])
        c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0, 3.5])
        c["inverse"], c["packed"] = rng.random() < 0.3, rng.random() < 0.5
        c["base"] = rng.choice([1e4, 5e5, 1e6])
    return c


# ---- what prepare() and exact() share: lengths, trees and inputs -----------------------------


def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + what)


def _starts(case):
    r = random.Random(case["mix"])
    return [r.randint(case["start_lo"], case["start_hi"]) for _ in range(case["batch"])]


def _trees(case):
    """(nodes, ancestor bits of each node) of every sequence.  Node 0 is the root, the token that
    the last step kept; every other node hangs below an earlier one."""
    r, n = random.Random(case["mix"] + 1), case["nodes"]
    trees = []
    for _ in range(case["batch"]):
        m = r.randint(0, n) if case["tree"] == "ragged" else n
        bits = []
        for i in range(n):
            above = bits[i - 1 if case["tree"] == "chain" or r.random() < 0.4 else r.randrange(i)] if i else 0
            bits.append(above | 1 << i if i < m else 0)
        trees.append((m, bits))
    return trees


def _signed(x):
    return x - (1 << 64) if x >> 63 else x


def _token_type(case):
    return torch.float32 if case["kv"] == "f32" else torch.float16


def _cached(case, seed, b, n):
    """Key and value rows [n][heads][D] of sequence b, drafted nodes included."""
    g = _gen(seed, 16 + b)
    return [torch.randn((n, case["kv_heads"], case["head_dim"]), generator=g, device="cuda").to(_token_type(case)) for _ in range(2)]


def _queries(case, seed):
    shape = (case["batch"], case["nodes"], case["q_heads"], case["head_dim"])
    return torch.randn(shape, generator=_gen(seed, 1), device="cuda").to(torch.float16 if case["io"] == "f16" else torch.float32)


def _quantised(x):
    """int4 codes and fp16 scales of rows: groups of 32, an eighth of the second largest magnitude."""
    x = x.float().unflatten(-1, (-1, 32))
    rep = x.abs().topk(2, dim=-1).values[..., 1:]
    scale = torch.where(rep > 0, rep / 8, torch.ones_like(rep)).clamp(min=1e-6, max=65504.0).half()
    return (x / scale.float()).round().clamp(-8, 7), scale[..., 0]


def _tables(case, seed, lens):
    """Blocks scattered over a pool with a fifth of them free."""
    p = case["block"]
    need = [max(1, -(-n // p)) for n in lens]
    blocks = int(math.ceil(1.2 * sum(need)))
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(int(seed) + 1)).to(torch.int32)
    tables = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = perm[at:at + n]
        at += n
    return blocks, tables.cuda()


def _v_tile(d):
    """Byte and half (0 low, 1 high) of (token, element) in a 16-token tile of int4 V codes."""
    t, e = torch.arange(16, device="cuda")[:, None], torch.arange(d, device="cuda")[None]
    byte = (16 * (t // 4) + e % 16) * (d // 8) + 4 * (e // 32) + 2 * (t % 2) + t % 4 // 2
    return byte, (e // 16 % 2).int().expand(16, d)


def _empty_pool(case, blocks, lead=()):
    h, p, d = case["kv_heads"], case["block"], case["head_dim"]
    z = lambda *s, t: torch.zeros(lead + (blocks, h) + s, dtype=t, device="cuda")  # noqa: E731
    if case["kv"] == "int4":
        return {"k": z(p, d // 2, t=torch.uint8), "v": z(p, d // 2, t=torch.uint8), "ks": z(d // 32, p, t=torch.int16), "vs": z(p, d // 32, t=torch.int16),
                "kf": z(p // 16, t=torch.int32)}
    t = _token_type(case)
    return {"k": z(p, d, t=t), "v": z(p, d, t=t)}


def _write(case, pool, row, k, v):
    """A sequence's rows [n][H][D] into its blocks, whole blocks at a time."""
    h, p, d = case["kv_heads"], case["block"], case["head_dim"]
    nb = -(-k.shape[0] // p)
    row = row[:nb].long()
    rows = lambda x: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 1) + (0, nb * p - x.shape[0])).unflatten(0, (nb, p)).transpose(1, 2)  # noqa: E731
    if case["kv"] == "f32":
        pool["k"][row], pool["v"][row] = rows(k), rows(v)
    elif case["kv"] == "f16":  # V: groups of 4 tokens, element-major inside a group
        pool["k"][row] = rows(k)
        pool["v"][row] = rows(v).unflatten(2, (p // 4, 4)).transpose(3, 4).reshape(nb, h, p, d)
    else:
        kc, ks = _quantised(k)
        vc, vs = _quantised(v)
        kc, vc = (rows(x.flatten(-2)).to(torch.int32) & 15 for x in (kc, vc))
        pool["k"][row] = (kc[..., ::2] | kc[..., 1::2] << 4).to(torch.uint8)
        pool["ks"][row] = rows(ks).transpose(2, 3).contiguous().view(torch.int16)
        pool["vs"][row] = rows(vs).contiguous().view(torch.int16)
        byte, high = _v_tile(d)
        tile = torch.zeros((nb, h, p // 16, 8 * d), dtype=torch.int32, device="cuda")
        tile.scatter_add_(3, byte.flatten().expand(nb, h, p // 16, -1), (vc.unflatten(2, (p // 16, 16)) << 4 * high).flatten(-2))
        pool["v"][row] = tile.to(torch.uint8).reshape(nb, h, p, d // 2)
        # the flag word of a 16-token tile marks the keys that the clip to 4.5 deviations may reach
        x = rows((_quantised(k)[0] * ks.float()[..., None]).flatten(-2))
        near = x.abs().amax(-1) >= 4.4 * x.std(-1, correction=0)
        pool["kf"][row] = (near.unflatten(2, (p // 16, 16)).int() << torch.arange(16, device="cuda").int()).sum(-1, dtype=torch.int32)


def _int(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def _path(r, n, most):
    """A path through a tree of n nodes: from the root down, each node below the one before."""
    m = r.randint(1, most)
    return [0] + sorted(r.sample(range(1, n), min(m, n) - 1))


def _rope_inputs(case, seed):
    """Positions and the query and key rows, in one packed projection or in tensors of their own."""
    n, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    g = _gen(seed, 1)
    t = torch.float16 if case["io"] == "f16" else torch.float32
    pos = torch.randint(case["pos_lo"], case["pos_hi"], (n,), generator=g, device="cuda", dtype=torch.int32)
    if case["packed"]:
        x = torch.randn((n, hq + 2 * hk, d), generator=g, device="cuda").to(t)
        return pos, x[:, :hq], x[:, hq:hq + hk]
    return pos, torch.randn((n, hq, d), generator=g, device="cuda").to(t), torch.randn((n, hk, d), generator=g, device="cuda").to(t)


LOW, HIGH, LENGTH = {"bands": 1.0, "yarn": 1.0}, {"bands": 4.0, "yarn": 32.0}, 8192  # trained length, and the turns over it between which pairs are stretched in part


def prepare(case, seed):
    if case["kind"] == "rope":
        pos, q, k = _rope_inputs(case, seed)
        return SimpleNamespace(case=case, pos=pos, q=q, k=k)
    starts = _starts(case)
    s = SimpleNamespace(case=case, start=_int(starts), max_start=max(starts))
    blocks, s.tables = _tables(case, seed, [n + case["nodes"] for n in starts])
    if case["kind"] == "accept":
        s.pool = _empty_pool(case, blocks, (case["layers"],))
        g = _gen(seed, 2)
        for name, x in s.pool.items():
            if name == "kf":
                x.random_(0, 1 << 16, generator=g)
            else:
                x.view(torch.uint8).random_(0, 256, generator=g)
        r = random.Random(case["mix"] + 2)
        paths = [_path(r, case["nodes"], case["path"]) for _ in starts]
        s.path = _int([p + [-1] * (case["path"] - len(p)) for p in paths])
        if own:  # the handles of the layers' pools, which an engine keeps
            vr = _vr()
            s.layers = vr.pool_array([_pool_of(vr, case, {n: x[i] for n, x in s.pool.items()}) for i in range(case["layers"])])
        return s
    s.pool = _empty_pool(case, blocks)
    s.q = _queries(case, seed)
    if own:
        s.handle = _pool_of(_vr(), case, s.pool)
    for b, n in enumerate(starts):
        _write(case, s.pool, s.tables[b], *_cached(case, seed, b, n + case["nodes"]))
    trees = _trees(case)
    s.lens = _int([m for m, _ in trees]) if case["tree"] == "ragged" else None
    s.mask = None if case["tree"] == "chain" else torch.tensor([[_signed(x) for x in bits] for _, bits in trees], device="cuda")
    return s


# ---- plain forms -----------------------------------------------------------------------------


def _clip(x, three_bit):
    th = (4.5 * x.var(-1, correction=0, keepdim=True).sqrt()).clamp(min=1e-6)
    return x.clamp(-th, th).clamp(-16, 16) if three_bit else x.clamp(-th, th)


def _halves(x):
    return x.view(torch.float16).float()


def _read(case, pool, tables):
    """The blocks of every sequence as f32 rows [B][H][T][D]."""
    p, d = case["block"], case["head_dim"]
    at = tables.clamp(min=0).long()
    k, v = pool["k"][at], pool["v"][at]  # [B][blocks][H][P][..]
    if case["kv"] == "f16":
        v = v.unflatten(-2, (p // 4, 4)).flatten(-2).unflatten(-1, (d, 4)).transpose(-1, -2).flatten(-3, -2)
    elif case["kv"] == "int4":
        signed = lambda c: ((c ^ 8) - 8).float()  # noqa: E731
        k = k.to(torch.int8)
        k = signed(torch.stack([k & 15, k >> 4 & 15], -1).flatten(-2)) * _halves(pool["ks"][at]).transpose(-1, -2).repeat_interleave(32, -1)
        byte, high = _v_tile(d)
        v = v.unflatten(-2, (p // 16, 16)).flatten(-2)[..., byte]
        v = signed((v >> (4 * high).to(torch.uint8) & 15).to(torch.int8)).flatten(-3, -2) * _halves(pool["vs"][at]).repeat_interleave(32, -1)
    return [x.float().transpose(1, 2).flatten(2, 3) for x in (k, v)]


def _plain_tree(s):
    c = s.case
    n, heads, three = c["nodes"], c["kv_heads"], c["numerics"] == "3bit"
    group, d = c["q_heads"] // heads, c["head_dim"]
    k, v = _read(c, s.pool, s.tables)
    t = torch.arange(k.shape[2], device="cuda")
    j = t[None] - s.start[:, None]  # the node that a slot holds
    bit = torch.arange(n, device="cuda")
    sees = bit[:, None] >= bit[None] if s.mask is None else (s.mask[..., None] >> bit & 1).bool()  # [B][node][node]
    inside = (j >= 0) & (j < (n if s.lens is None else s.lens[:, None]))
    node = torch.gather(sees.expand(len(j), n, n), 2, j.clamp(0, n - 1)[:, None].expand(-1, n, -1))
    row = bit[None] < (n if s.lens is None else s.lens[:, None])
    visible = ((j < 0)[:, None] | (inside[:, None] & node)) & row[..., None]  # [B][node][slot]
    live = ((j < 0) | inside)[:, None, :, None]
    k, v = _clip(torch.where(live, k, 0.0), three), torch.where(live, v, 0.0)
    q = _clip(s.q.float(), three).unflatten(2, (heads, group)).permute(0, 2, 1, 3, 4).reshape(-1, n * group, d)
    score = torch.bmm(q, k.flatten(0, 1).transpose(1, 2).contiguous()) / math.sqrt(d)
    score = (score.clamp(-24, 24) if three else score).view(len(j), heads, n, group, -1)
    score = score.masked_fill(~visible[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = torch.bmm(weight.flatten(2, 3).flatten(0, 1), v.flatten(0, 1)).view(len(j), heads, n, group, d) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous().to(s.q.dtype)


def _plain_accept(s):
    c, pool = s.case, s.pool
    p, d = c["block"], c["head_dim"]
    step = torch.arange(s.path.shape[1], device="cuda")
    count = ((s.path >= 0) & (s.path < c["nodes"])).int().cumprod(1).sum(1)
    to = s.start[:, None] + step
    fro = torch.where(step < count[:, None], s.start[:, None] + s.path, to)  # what is not kept goes to its own place
    place = lambda x: (torch.gather(s.tables.long(), 1, (x // p).long()).flatten(), (x % p).long().flatten())  # noqa: E731
    (b1, s1), (b0, s0) = place(to), place(fro)
    k = pool["k"].view(torch.uint8)
    k[:, b1, :, s1] = k[:, b0, :, s0]
    v = pool["v"].view(torch.uint8)
    if c["kv"] == "f32":
        v[:, b1, :, s1] = v[:, b0, :, s0]
    elif c["kv"] == "f16":
        v = pool["v"].view(torch.int16).unflatten(-2, (p // 4, 4)).flatten(-2).unflatten(-1, (d, 4))
        v[:, b1, :, s1 // 4, :, s1 % 4] = v[:, b0, :, s0 // 4, :, s0 % 4]
    else:
        # a token's codes are one byte of every dword of four rows of 16 lane chunks
        v = v.flatten(-2).unflatten(-1, (p // 16, 4, 16, d // 32, 4))
        where = lambda blk, slot: (slice(None), blk, slice(None), slot // 16, slot // 4 % 4, slice(None), slice(None), 2 * (slot % 2) + slot % 4 // 2)  # noqa: E731
        v[where(b1, s1)] = v[where(b0, s0)]
        pool["ks"][:, b1, :, :, s1] = pool["ks"][:, b0, :, :, s0]
        pool["vs"][:, b1, :, s1] = pool["vs"][:, b0, :, s0]
        old, new = (pool["kf"][:, blk, :, slot // 16] >> (slot % 16).int()[:, None, None] & 1 for blk, slot in ((b1, s1), (b0, s0)))  # [row][layer][head]
        layer, head = (torch.arange(n, device="cuda") for n in pool["kf"].shape[:3:2])
        pool["kf"].index_put_((layer[:, None], b1[:, None, None], head, (s1 // 16)[:, None, None]), (new - old) << (s1 % 16).int()[:, None, None], accumulate=True)
    return s.start + count


def _frequencies(case):
    """Radians a position of every pair, and the factor on cosine and sine."""
    r, base, factor = case["rope_dim"], case["base"], case["factor"]
    if case["scaling"] == "base" and r > 2:
        base *= factor ** (r / (r - 2))
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    f, kind, size = base ** (-2 * i / r), case["scaling"], 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "bands":
        turns = LENGTH * f / (2 * math.pi)
        keep = ((turns - LOW[kind]) / (HIGH[kind] - LOW[kind])).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    elif kind == "yarn":
        at = lambda turns: r * math.log(LENGTH / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(at(HIGH[kind])), 0), min(math.ceil(at(LOW[kind])), r - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        size = 0.1 * math.log(factor) + 1
    return f, size


def _plain_rope(s):
    c = s.case
    f, size = _frequencies(c)
    angle = s.pos.double()[:, None] * f
    cos, sin = ((size * x).float()[:, None] for x in (angle.cos(), -angle.sin() if c["inverse"] else angle.sin()))
    r = c["rope_dim"]

    def turn(x):
        y = x.float()
        a, b = (y[..., :r // 2], y[..., r // 2:r]) if c["layout"] == "half" else (y[..., :r:2], y[..., 1:r:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([a, b] if c["layout"] == "half" else [torch.stack([a, b], -1).flatten(-2)], -1).to(x.dtype), x[..., r:]

    return {"q": torch.cat(turn(s.q), -1), "k": torch.cat(turn(s.k), -1)}


# ---- the framework's calls -------------------------------------------------------------------


def _vr():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vspec-engine_amd", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import vspec_rocm

    return vspec_rocm


def _pool_of(vr, case, parts):
    kind = {"f32": vr.KV_F32, "f16": vr.KV_F16, "int4": vr.KV_INT4}[case["kv"]]
    return vr.PagedPool.over(kind, case["block"], case["kv_heads"], case["head_dim"], parts["k"], parts["v"], parts.get("ks"), parts.get("vs"), parts.get("kf"))


def _own(s):
    vr, c = _vr(), s.case
    if c["kind"] == "tree":
        numerics = vr.NUMERICS_3BIT if c["numerics"] == "3bit" else vr.NUMERICS_PLAIN
        return vr.paged_tree_attention(s.handle, s.tables, s.start, s.q, tree_mask=s.mask, tree_lens=s.lens, max_start_pos=s.max_start, numerics=numerics)
    if c["kind"] == "accept":
        return vr.kv_accept(s.layers, s.tables, s.start, s.path, c["nodes"]).long()
    layout = vr.ROPE_HALF if c["layout"] == "half" else vr.ROPE_INTERLEAVED
    scaling = {"none": vr.ROPE_SCALE_NONE, "linear": vr.ROPE_SCALE_LINEAR, "base": vr.ROPE_SCALE_BASE, "bands": vr.ROPE_SCALE_BANDS, "yarn": vr.ROPE_SCALE_YARN}[c["scaling"]]
    q, k = vr.rope(s.pos, s.q, s.k, rope_dim=c["rope_dim"], base=c["base"], layout=layout, scaling=scaling, factor=c["factor"], trained_len=LENGTH,
                   low=LOW.get(c["scaling"], 0.0), high=HIGH.get(c["scaling"], 0.0), inverse=c["inverse"])
    return {"q": q, "k": k}


def run(state):
    kind = state.case["kind"]
    if own:
        got = _own(state)
    else:
        got = (_plain_tree if kind == "tree" else _plain_accept if kind == "accept" else _plain_rope)(state)
    if kind == "accept":
        # bits of the rows: what was moved has to be what was there
        return {"lens": got, **{n: x.view(torch.int16) if x.dtype == torch.float16 else x.view(torch.int32) if x.dtype == torch.float32 else x for n, x in state.pool.items()}}
    return got


# ---- what a pass cannot do without, and what it gives in 64 bits -------------------------------


def _row_bytes(case):
    d = case["head_dim"]
    return {"f32": 4 * d, "f16": 2 * d, "int4": d // 2 + d // 16}[case["kv"]]


def work(case):
    d = case["head_dim"]
    if case["kind"] == "rope":
        size = 2 if case["io"] == "f16" else 4
        rows = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * rows * d * size + 4 * case["tokens"], "flops": 3 * rows * case["rope_dim"]}
    starts = _starts(case)
    if case["kind"] == "accept":
        r = random.Random(case["mix"] + 2)
        moved = sum(sum(n != i for i, n in enumerate(_path(r, case["nodes"], case["path"]))) for _ in starts)
        return {"bytes": 4 * moved * case["layers"] * case["kv_heads"] * _row_bytes(case) + 4 * case["batch"] * (case["path"] + 2), "flops": 0}
    trees = _trees(case)
    slots = sum(n + m for n, (m, _) in zip(starts, trees))
    seen = sum(n * m + sum(bin(x).count("1") for x in bits) for n, (m, bits) in zip(starts, trees))
    io = 2 * case["batch"] * case["nodes"] * case["q_heads"] * d * (2 if case["io"] == "f16" else 4)
    return {"bytes": 2 * slots * case["kv_heads"] * _row_bytes(case) + io, "flops": 4 * d * case["q_heads"] * seen}


def _limited(x, three_bit):
    """Rows held to 4.5 standard deviations about zero, and in 3-bit mode to 16."""
    bound = torch.clamp(4.5 * torch.sqrt(((x - x.mean(-1, keepdim=True)) ** 2).mean(-1, keepdim=True)), min=1e-6)
    if three_bit:
        bound = torch.clamp(bound, max=16.0)
    return torch.minimum(torch.maximum(x, -bound), bound)


def _stored(case, x):
    if case["kv"] != "int4":
        return x.double()
    code, scale = _quantised(x)
    return (code.double() * scale.double()[..., None]).flatten(-2)


def _exact_tree(case, seed):
    heads, n, three = case["kv_heads"], case["nodes"], case["numerics"] == "3bit"
    group = case["q_heads"] // heads
    q = _limited(_queries(case, seed).double(), three)
    out = torch.zeros_like(q)
    for b, (start, (m, bits)) in enumerate(zip(_starts(case), _trees(case))):
        if not m:
            continue
        k, v = (_stored(case, x[:start + m]) for x in _cached(case, seed, b, start + n))
        k, v = _limited(k, three).permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
        hidden = torch.zeros((m, start + m), dtype=torch.float64)
        for i in range(m):
            for j in range(m):
                if not bits[i] >> j & 1:
                    hidden[i, start + j] = -math.inf
        score = torch.matmul(q[b, :m].view(m, heads, group, -1).permute(1, 2, 0, 3).reshape(heads, group * m, -1), k) * case["head_dim"] ** -0.5
        if three:
            score = score.clamp(min=-24.0, max=24.0)
        weight = (score.view(heads, group, m, -1) + hidden.cuda()).softmax(-1)
        out[b, :m] = torch.matmul(weight.flatten(1, 2), v).view(heads, group, m, -1).permute(2, 0, 1, 3).reshape(m, case["q_heads"], -1)
    return out


def _exact_rope(case, seed):
    pos, q, k = _rope_inputs(case, seed)
    r, base, factor, kind = case["rope_dim"], case["base"], case["factor"], case["scaling"]
    if kind == "base" and r > 2:
        base = base * factor ** (r / (r - 2))
    speed, size = [], 1.0 + 0.1 * math.log(factor) if kind == "yarn" else 1.0
    for i in range(r // 2):
        f = math.exp(-2.0 * i / r * math.log(base))
        share = 1.0  # of the pair's own speed
        if kind == "linear":
            share = 0.0
        elif kind == "bands":
            length = 2 * math.pi / f  # positions a turn
            share = 0.0 if length > LENGTH / LOW[kind] else 1.0 if length < LENGTH / HIGH[kind] else (LENGTH / length - LOW[kind]) / (HIGH[kind] - LOW[kind])
        elif kind == "yarn":
            ends = [r * math.log(LENGTH / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (HIGH[kind], LOW[kind])]
            lo, hi = max(0, math.floor(ends[0])), min(r - 1, math.ceil(ends[1]))
            share = 1.0 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))
        speed.append(f * share + f / factor * (1 - share))
    turn = torch.polar(torch.full((len(pos), r // 2), size, dtype=torch.float64, device="cuda"),
                       pos.double()[:, None] * torch.tensor(speed, dtype=torch.float64, device="cuda") * (-1 if case["inverse"] else 1))
    got = {}
    for name, x in (("q", q), ("k", k)):
        y = x.double()
        pairs = y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else y[..., :r].unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        y[..., :r] = (z.transpose(-1, -2) if case["layout"] == "half" else z).flatten(-2)
        got[name] = y.contiguous()
    return got


def exact(case, seed):
    # moved rows are bits: they have no value to compute
    return _exact_tree(case, seed) if case["kind"] == "tree" else _exact_rope(case, seed) if case["kind"] == "rope" else None
