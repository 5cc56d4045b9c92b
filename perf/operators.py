"""Speculative decoding over the slot cache: what is timed, and its plain form.

A step that checks a tree of drafted tokens per sequence: its block tables and
slots (``step_tables``), the attention of every node over the cached context
and its own ancestors (``v1_tree_attention``), the walk that finds the accepted
path (``tree_accept``) and the move of that path's slots to consecutive
positions (``commit_slots``).  ``listed()`` names the sizes in use, ``draw()``
the ranges they stand for, ``exact()`` the attention in 64 bits from the slots'
bytes.  The other operators give whole numbers, which have to be equal.
"""
import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
RAW = 16  # bits of raw fp16 slots


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one user, a small tree over a short conversation: latency
        dict(name="tree_one_user", op="tree", batch=1, hkv=8, group=4, d=128, kb=4, vb=4, vrot=False, page=16, lo=900,
             hi=900, nodes=8, chain=False, ragged=False, window=0, dtype="bf16"),
        # one layer of a server's step: 16 sequences, up to 32 nodes each, the default 3-bit cache
        dict(name="tree_batch", op="tree", batch=16, hkv=8, group=4, d=128, kb=3, vb=3, vrot=True, page=16, lo=1024,
             hi=6000, nodes=32, chain=False, ragged=True, window=0, dtype="bf16"),
        # two long conversations, large trees of an odd size
        dict(name="tree_long", op="tree", batch=2, hkv=8, group=4, d=128, kb=4, vb=2, vrot=True, page=16, lo=65536,
             hi=131072, nodes=61, chain=False, ragged=False, window=0, dtype="bf16"),
        # a chain of a few drafted tokens for many sequences, 64-wide heads
        dict(name="chain_d64", op="tree", batch=24, hkv=8, group=4, d=64, kb=4, vb=4, vrot=False, page=16, lo=700,
             hi=6000, nodes=5, chain=True, ragged=True, window=0, dtype="fp16"),
        # 256-wide heads, a sliding-window layer
        dict(name="tree_d256_window", op="tree", batch=5, hkv=4, group=2, d=256, kb=4, vb=3, vrot=False, page=32, lo=301,
             hi=9001, nodes=25, chain=False, ragged=True, window=4096, dtype="bf16"),
        # a boundary layer: raw fp16 slots
        dict(name="tree_raw", op="tree", batch=12, hkv=8, group=4, d=128, kb=RAW, vb=RAW, vrot=False, page=16, lo=500,
             hi=5000, nodes=20, chain=False, ragged=True, window=0, dtype="bf16"),
        # a server's decode step: 64 requests with an 8-node tree each, blocks taken and given back
        dict(name="step_decode", op="step", batch=64, most=8, hi=8192, page=16),
        # a chunked-prefill step of nine prompts
        dict(name="step_prefill", op="step", batch=9, most=4096, hi=16384, page=16),
        # three users' small trees
        dict(name="accept_small", op="accept", batch=3, nodes=8, vocab=50),
        # a full batch of large trees
        dict(name="accept_batch", op="accept", batch=64, nodes=61, vocab=4),
        # 32 layers of 3-bit slots
        dict(name="commit_layers", op="commit", batch=16, layers=32, hkv=8, slot=128, page=16, hi=200, nodes=32),
        # a few layers of raw 256-wide heads, one user
        dict(name="commit_raw", op="commit", batch=1, layers=4, hkv=4, slot=1024, page=32, hi=700, nodes=9),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "tree", "tree", "step", "accept", "commit"))
    if op == "step":
        batch = _log(rng, 1, 256)
        most = _log(rng, 1, min(4096, 65536 // batch))
        return dict(op=op, batch=batch, most=most, hi=_log(rng, max(16, most), 16384), page=rng.choice((16, 16, 32, 64)))
    if op == "accept":
        return dict(op=op, batch=_log(rng, 1, 64), nodes=_log(rng, 1, 100), vocab=rng.choice((2, 4, 50, 128256)))
    if op == "commit":
        hkv, slot = rng.choice(((8, 128), (8, 64), (4, 256), (2, 512), (4, 1024)))
        return dict(op=op, batch=_log(rng, 1, 16), layers=_log(rng, 1, 40), hkv=hkv, slot=slot, page=rng.choice((16, 32)),
                    hi=_log(rng, 20, 200), nodes=_log(rng, 1, 64))
    hkv, group = rng.choice(((8, 4), (8, 4), (8, 1), (4, 7), (4, 2), (2, 8), (8, 5)))
    d = rng.choice((64, 128, 128, 256))
    kb, vb = rng.choice(((4, 2), (3, 3), (4, 4), (3, 4), (2, 4), (1, 2), (8, 8), (RAW, RAW)))
    nodes = _log(rng, 1, 100)
    hi = _log(rng, 20, 32768)
    most = 40_000_000 // max(nodes, 16) // max(d, 128) * 128 // (hkv * group) // hi
    window = rng.choice((0, 0, 0, 128, 1024))
    return dict(op=op, batch=_log(rng, 1, max(1, min(48, most))), hkv=hkv, group=group, d=d, kb=kb, vb=vb,
                vrot=kb != RAW and rng.random() < 0.5, page=rng.choice((16, 16, 32, 64)), lo=rng.choice((hi, max(1, hi // 3), 0)), hi=hi, nodes=nodes,
                chain=rng.random() < 0.3, ragged=rng.random() < 0.5, window=window,
                dtype=rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32")))


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _dev(x, dtype=None):
    return torch.as_tensor(x, dtype=dtype).to(DEV)


def _hadamard(d, dtype):
    h = torch.ones(1, 1, dtype=dtype, device=DEV)
    while h.shape[0] < d:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / math.sqrt(d)


def _levels(d, bits):
    """Sorted Lloyd-Max levels of a normal coordinate of variance 1 / d."""
    n = 1 << bits
    cut = np.array([-8.0, *np.linspace(-2.5, 2.5, n - 1), 8.0])
    pdf, cdf = lambda x: np.exp(-x * x / 2) / math.sqrt(2 * math.pi), np.vectorize(lambda x: 0.5 * math.erfc(-x / math.sqrt(2)))
    for _ in range(60):
        lev = (pdf(cut[:-1]) - pdf(cut[1:])) / np.maximum(cdf(cut[1:]) - cdf(cut[:-1]), 1e-30)
        cut[1:-1] = (lev[1:] + lev[:-1]) / 2
    return _dev(np.sort(lev) / math.sqrt(d), torch.float32)


def _bytes_of(codes, bits):
    """Little-endian bit strings of codes [n, h, d] as bytes."""
    b = (codes[..., None] >> torch.arange(bits, device=DEV, dtype=torch.uint8)) & 1
    b = b.flatten(-2).view(*codes.shape[:2], -1, 8) << torch.arange(8, device=DEV, dtype=torch.uint8)
    return b.sum(-1, dtype=torch.uint8) if bits != 8 else codes


def _fields(*xs):
    return torch.stack(xs, -1).to(torch.float16).view(torch.uint8)


def _slots(c, k, v, lev, had, slot):
    """Slots [n, hkv, slot] of keys and values [n, hkv, d], as the store writes them."""
    if c["kb"] == RAW:
        return torch.cat((k.to(torch.float16).view(torch.uint8), v.to(torch.float16).view(torch.uint8)), -1)
    norm = k.norm(dim=-1, keepdim=True)
    y = (k / (norm + 1e-8)) @ had
    kc = torch.bucketize(y, (lev[1:] + lev[:-1]) / 2).to(torch.uint8)
    if c["vrot"]:
        v = v @ had
    lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    top = (1 << c["vb"]) - 1
    scale = (hi - lo).clamp(min=1e-6) / top
    vc = ((v - lo) / scale + 0.5).clamp(0, top).to(torch.uint8)
    row = torch.cat((_bytes_of(kc, c["kb"]), _fields(norm[..., 0]), _bytes_of(vc, c["vb"]), _fields(scale[..., 0], lo[..., 0])), -1)
    return torch.nn.functional.pad(row, (0, slot - row.shape[-1]))


def _table(seed, need, most, page):
    """Block table of sequences of ``need`` tokens whose pages are scattered over a pool, and the pool's size."""
    g = torch.Generator().manual_seed(int(seed) + 1)
    blocks = [(n + page - 1) // page for n in need]
    nb = sum((n + page - 1) // page for n in most) + 3
    perm = torch.randperm(nb, generator=g).to(torch.int32)
    bt = torch.zeros(len(need), max(max(blocks), 1), dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt.to(DEV), nb


def _trees(seed, counts, chain):
    """Parents of every node (parent before child, the root first) and, per node, the words of its ancestors' bits."""
    r = np.random.RandomState((int(seed) + 3) % (1 << 32))
    words = (max(counts) + 63) // 64
    parents, masks = [], []
    for n in counts:
        par = [-1] + [i - 1 if chain else int(r.randint(max(0, (i - 1) // 3), i)) for i in range(1, n)]
        anc = []
        for i in range(n):
            anc.append((anc[par[i]] if i else 0) | 1 << i)
        parents += par
        masks += [[(a >> 64 * w) & 0xFFFFFFFFFFFFFFFF for w in range(words)] for a in anc]
    mask = torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64))
    return np.array(parents, dtype=np.int32), mask


def _starts(counts):
    return _dev(np.concatenate(([0], np.cumsum(counts))), torch.int32)


def _counts(n, lo, hi):
    """Tokens of n sequences, in lo .. hi: of one case always the same, so that its tensors keep their shapes."""
    return [int(x) for x in np.random.RandomState(n * 1000 + hi).randint(lo, hi + 1, n)]


def _prepare_tree(c, seed):
    g, dt, hkv, d, page = _gen(seed), DTYPES[c["dtype"]], c["hkv"], c["d"], c["page"]
    r = np.random.RandomState((int(seed) + 2) % (1 << 32))
    ctx = [int(x) for x in r.randint(c["lo"], c["hi"] + 1, c["batch"])]
    counts = _counts(c["batch"], 1, c["nodes"]) if c["ragged"] else [c["nodes"]] * c["batch"]
    lens = [a + n for a, n in zip(ctx, counts)]
    bt, nb = _table(seed, lens, [c["hi"] + c["nodes"]] * c["batch"], page)
    raw = c["kb"] == RAW
    data = 4 * d if raw else d * (c["kb"] + c["vb"]) // 8 + 6
    slot = 1 << (data - 1).bit_length()
    lev, had = (None if raw else _levels(d, c["kb"])), _hadamard(d, torch.float32)
    cache = torch.zeros(nb * page, hkv, slot, dtype=torch.uint8, device=DEV)
    for i, n in enumerate(lens):
        for a in range(0, n, 16384):
            m = min(n, a + 16384) - a
            k = torch.randn(m, hkv, d, generator=g, device=DEV)
            k[..., 3::37] *= 3.0  # a few channels larger than the others, as trained models have them
            v = torch.randn(m, hkv, d, generator=g, device=DEV)
            pos = torch.arange(a, a + m, device=DEV)
            cache[bt[i][pos // page].long() * page + pos % page] = _slots(c, k, v, lev, had, slot)
    _, mask = _trees(seed, counts, c["chain"])
    # a sliding-window layer: each node sees the context from its own position - window + 1 on
    depth = (mask.view(-1, 1, mask.shape[1]) >> torch.arange(64).view(1, 64, 1) & 1).sum((1, 2))
    at = torch.tensor(np.repeat(ctx, counts)) + depth
    start = (at - c["window"]).clamp(min=0).to(torch.int32).to(DEV) if c["window"] else None
    q = torch.randn(sum(counts), hkv * c["group"], d, generator=g, device=DEV) * 1.5
    return SimpleNamespace(c=c, q=q.to(dt), cache=cache.view(nb, page, hkv, slot), bt=bt, lens=_dev(lens, torch.int32),
                           qsl=_starts(counts), lev=lev, mask=None if c["chain"] else mask.to(DEV), start=start,
                           most=max(counts), longest=max(lens), scale=1 / math.sqrt(d))


def _prepare_step(c, seed):
    """Two steps of a server that follow each other over and over: a third of the requests end in the one and
    begin in the other, the others grow by what the first step accepted."""
    r = np.random.RandomState((int(seed) + 2) % (1 << 32))
    n, page, most = c["batch"], c["page"], c["most"]
    past = r.randint(0, c["hi"] - most + 1, n)
    new, new2 = np.array(_counts(n, 1, most)), np.array(_counts(n, 0, most))
    ends = r.rand(n) < 1 / 3
    past2 = np.where(ends, 0, np.minimum(past + r.randint(1, new + 1), c["hi"] - most))
    width = (c["hi"] + page - 1) // page
    have = (past + page - 1) // page
    pool = n * (width + 2)
    perm = r.permutation(pool).astype(np.int32)
    bt = np.full((n, width), -1, dtype=np.int32)
    at = 0
    for i, h in enumerate(have):
        bt[i, :h] = perm[at:at + h]
        at += h
    free = np.full(pool, -1, dtype=np.int32)
    free[:pool - at] = perm[at:]
    steps = []
    for p, q in ((past, new), (past2, new2)):
        depths = np.concatenate([np.arange(x) // 2 for x in q]).astype(np.int32) if q.sum() else np.zeros(0, np.int32)
        steps.append((_starts(q), _dev(p, torch.int32), int(q.sum()) + 3, _dev(np.concatenate((depths, [0, 0, 0])), torch.int32)))
    return SimpleNamespace(c=c, steps=steps, turn=0, bt=_dev(bt), free=_dev(free), count=_dev([pool - at], torch.int32),
                           have=_dev(have, torch.int32))


def _prepare_accept(c, seed):
    r = np.random.RandomState((int(seed) + 2) % (1 << 32))
    counts = _counts(c["batch"], max(1, c["nodes"] // 2), c["nodes"])
    parents, _ = _trees(seed, counts, False)
    total = sum(counts)
    tokens = r.randint(0, c["vocab"], total)
    wanted = r.randint(0, c["vocab"], total)
    first = np.repeat(np.concatenate(([0], np.cumsum(counts)[:-1])), counts)
    child = np.arange(total) - first > 0
    # the drafter is right for two nodes in three: its token is what the model answers after the node's parent
    hit = child & (r.rand(total) < 2 / 3)
    tokens[hit] = wanted[(first + parents)[hit]]
    return SimpleNamespace(c=c, tokens=_dev(tokens), parents=_dev(parents), wanted=_dev(wanted), qsl=_starts(counts),
                           most=c["nodes"])


def _prepare_commit(c, seed):
    g, page = _gen(seed), c["page"]
    r = np.random.RandomState((int(seed) + 2) % (1 << 32))
    past = [int(x) for x in r.randint(0, c["hi"] + 1, c["batch"])]
    bt, nb = _table(seed, [p + c["nodes"] for p in past], [c["hi"] + c["nodes"]] * c["batch"], page)
    path = np.full((c["batch"], c["nodes"]), -1, dtype=np.int32)
    count = np.zeros(c["batch"], dtype=np.int32)
    for i in range(c["batch"]):
        at = [0]
        while len(at) < 12:  # a child a few nodes on, until the tree or the luck ends
            nxt = at[-1] + int(r.randint(1, 5))
            if nxt >= c["nodes"] or r.rand() < 0.2:
                break
            at.append(nxt)
        path[i, :len(at)], count[i] = at, len(at)
    caches = torch.randint(0, 256, (c["layers"], nb, page, c["hkv"], c["slot"]), generator=g, device=DEV, dtype=torch.uint8)
    return SimpleNamespace(c=c, caches=caches, layers=list(caches.unbind(0)), bt=bt, past=_dev(past, torch.int32),
                           path=_dev(path), count=_dev(count))


def prepare(case, seed):
    return {"tree": _prepare_tree, "step": _prepare_step, "accept": _prepare_accept,
            "commit": _prepare_commit}[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# one pass: the framework's calls
# ---------------------------------------------------------------------------

def _package():
    at = os.path.join(os.getcwd(), "fused-turboquant_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from fused_turboquant import steps, v1
    return steps, v1


def _own(s):
    steps, v1 = _package()
    c = s.c
    if c["op"] == "tree":
        return v1.v1_tree_attention(s.q, s.cache, s.bt, s.lens, s.qsl, s.lev, c["kb"], c["vb"], tree_mask=s.mask,
                                    scale=s.scale, v_rotate=c["vrot"], kv_start=s.start, max_query_len=s.most,
                                    max_seq_len=s.longest, sorted_centroids=True)
    if c["op"] == "step":
        qsl, past, total, depths = s.steps[s.turn]
        s.turn ^= 1
        r = steps.step_tables(qsl, past, s.bt, c["page"], total, depths=depths, num_blocks=s.have, free_blocks=s.free,
                              free_count=s.count)
        return r.slot_mapping, r.positions, r.token_request, r.seq_lens, r.missing, s.bt, s.have, s.free, s.count
    if c["op"] == "accept":
        r = steps.tree_accept(s.tokens, s.parents, s.wanted, s.qsl, s.most)
        return r.path, r.counts, r.tokens
    steps.commit_slots(s.layers, s.bt, s.past, s.path, s.count)
    return s.caches


# ---------------------------------------------------------------------------
# one pass: the plain form
# ---------------------------------------------------------------------------

def _unpack(rows, first, n, bits):
    """n little-endian codes of ``bits`` bits from byte ``first`` of rows [..., slot], as float32."""
    if bits == 8:
        return rows[..., first:first + n].float()
    at = torch.arange(n, device=DEV) * bits
    lo, hi = rows[..., first + at // 8], rows[..., first + (at + bits - 1) // 8]
    return (((lo.to(torch.int16) | hi.to(torch.int16) << 8) >> (at % 8).to(torch.int16)) & ((1 << bits) - 1)).float()


def _half(rows, first, n):
    return rows[..., first:first + 2 * n].contiguous().view(torch.float16).float()


def _plain_tree(s):
    c, d, hkv, page = s.c, s.c["d"], s.c["hkv"], s.c["page"]
    B, G, width, total = s.bt.shape[0], s.c["group"], s.bt.shape[1] * s.c["page"], s.q.shape[0]
    rows = s.cache[s.bt.long()].view(B, width, hkv, -1).transpose(1, 2)  # [B, hkv, L, slot]
    if c["kb"] == RAW:
        k, v = _half(rows, 0, d), _half(rows, 2 * d, d)
    else:
        kb, vb, at = c["kb"], c["vb"], d * c["kb"] // 8
        k = s.lev[_unpack(rows, 0, d, kb).to(torch.int32)]
        k = k * (_half(rows, at, 1) / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-16))
        f = at + 2 + d * vb // 8
        v = _unpack(rows, at + 2, d, vb) * _half(rows, f, 1) + _half(rows, f + 2, 1)
    # queries padded to one tree size: [B, hkv, N G, d]
    n = s.qsl[1:] - s.qsl[:-1]
    node = torch.arange(s.most, device=DEV)
    live = node[None] < n[:, None]
    row = (s.qsl[:-1, None] + node[None]).clamp(max=total - 1).long()
    q = s.q.float()
    had = _hadamard(d, torch.float32)
    if c["kb"] != RAW:
        q = q @ had
    q = q[row].view(B, s.most, hkv, G, d).transpose(1, 2).reshape(B, hkv, s.most * G, d)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(s.scale).view(B, hkv, s.most, G, width)
    # a node sees the context from its start on, and the nodes of its mask
    pos = torch.arange(width, device=DEV)
    rel = pos[None] - (s.lens - n)[:, None]
    if s.mask is None:
        tree = rel[:, None] <= node[:, None]
    else:
        words = s.mask[row].gather(2, (rel.clamp(0, s.mask.shape[1] * 64 - 1) >> 6)[:, None].expand(-1, s.most, -1).long())
        tree = (words >> (rel & 63)[:, None].long() & 1) != 0
    past = rel[:, None] < 0
    if s.start is not None:
        past = past & (pos >= s.start[row][..., None])
    sees = torch.where(rel[:, None] < 0, past, tree & (rel < n[:, None])[:, None])[:, None, :, None]
    p = p.masked_fill_(~sees, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    mass = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, s.most * G, width), v).view(B, hkv, s.most, G, d) / torch.where(mass == 0, 1.0, mass)
    if c["vrot"]:
        o = o @ had
    return o.transpose(1, 2).reshape(B, s.most, hkv * G, d)[live].to(s.q.dtype)


def _plain_step(s):
    bs, width = s.c["page"], s.bt.shape[1]
    qsl, past, total, depths = s.steps[s.turn]
    s.turn ^= 1
    lens = past + (qsl[1:] - qsl[:-1])
    want, have, pool = ((lens + bs - 1) // bs).clamp(max=width), s.have.clone(), s.free.numel()
    missing = ((lens + bs - 1) // bs - want).sum()
    # released blocks go on top of the free list in the order of the requests, new ones come from its top
    page = torch.arange(width, device=DEV, dtype=torch.int32)[None]
    gone = (page >= want[:, None]) & (page < have[:, None])
    rank = gone.flatten().cumsum(0).view_as(gone) - 1
    count = s.count.clone()
    at = torch.where(gone, count + rank, pool)
    stack = torch.cat((s.free, s.free.new_zeros(1))).index_put_((at,), s.bt)
    avail = count + gone.sum()
    take = (page >= have[:, None]) & (page < want[:, None])
    rank = take.flatten().cumsum(0).view_as(take) - 1
    given = take & (rank < avail)
    s.bt.copy_(torch.where(given, stack[(avail - 1 - rank).clamp(0, pool)], s.bt))
    s.have.copy_(torch.minimum(have, want) + given.sum(1))
    s.count.copy_(avail - given.sum())
    i = torch.arange(pool, device=DEV)
    s.free.copy_(torch.where((i >= count) & (i < s.count), stack[:-1], s.free))
    t = torch.arange(total, device=DEV, dtype=torch.int32)
    b = torch.searchsorted(qsl, t, right=True) - 1
    live = t < qsl[-1]
    b = torch.where(live, b, 0)
    where = past[b] + t - qsl[b]
    held = live & (where // bs < s.have[b])
    slot = s.bt[b, (where // bs).clamp(max=width - 1)].long() * bs + where % bs
    return (torch.where(held, slot, -1), torch.where(live, past[b] + depths, 0).long(),
            torch.where(live, b, -1).to(torch.int32), lens, (missing + take.sum() - given.sum()).to(torch.int32).view(1),
            s.bt, s.have, s.free, s.count)


def _plain_accept(s):
    B, n = s.qsl.numel() - 1, s.qsl[1:] - s.qsl[:-1]
    node = torch.arange(s.most, device=DEV)
    live = node[None] < n[:, None]
    row = torch.where(live, s.qsl[:-1, None] + node[None], 0).long()
    parent = torch.where(live, s.parents[row], -1).long()
    answer = s.wanted[row]
    child = live & (node > 0) & (parent >= 0)
    tok = s.tokens[row]
    hit = child & (tok == answer.gather(1, parent.clamp(min=0)))
    # of siblings with the same token the first counts
    same = (parent[:, :, None] == parent[:, None, :]) & (hit[:, :, None] & hit[:, None, :]) & (node[:, None] > node[None, :])
    hit = hit & ~same.any(2)
    # reached from the root by such children: powers of the edges, doubled until they cover the longest path
    edge = torch.zeros(B, s.most, s.most, device=DEV)
    edge.scatter_(2, parent.clamp(min=0)[..., None], hit[..., None].float())
    edge = ((edge + torch.eye(s.most, device=DEV)) > 0).float()
    doublings = max(1, (s.most - 1).bit_length())
    for _ in range(doublings):
        edge = (torch.matmul(edge, edge) > 0).float()
    done = live & (edge[:, :, 0] > 0)
    path = torch.where(done, node, s.most).sort(1).values
    ok = path < s.most
    tokens = torch.where(ok, answer.gather(1, path.clamp(max=s.most - 1)), -1)
    return torch.where(ok, path, -1).to(torch.int32), done.sum(1).to(torch.int32), tokens


def _plain_commit(s):
    bs = s.c["page"]
    j = torch.arange(s.path.shape[1], device=DEV)
    moved = j[None] < s.count[:, None]
    flat = s.caches.view(s.c["layers"], -1, s.c["hkv"] * s.c["slot"])
    rows = torch.arange(s.bt.shape[0], device=DEV)[:, None]

    def slots(at):
        return s.bt[rows, (at // bs).long()].long() * bs + at % bs

    src = slots(s.past[:, None] + torch.where(moved, s.path, 0)).flatten()
    dst = slots(s.past[:, None] + torch.where(moved, j, 0).to(torch.int32)).flatten()
    flat[:, dst] = flat[:, src]
    return s.caches


@torch.no_grad()
def run(s):
    if own:
        return _own(s)
    return {"tree": _plain_tree, "step": _plain_step, "accept": _plain_accept, "commit": _plain_commit}[s.c["op"]](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(c):
    n = c["batch"]
    if c["op"] == "step":
        tok = n * c["most"] / 2
        return {"bytes": 24 * tok + 24 * n, "flops": 0}
    if c["op"] == "accept":
        return {"bytes": n * c["nodes"] * 0.75 * 20 + n * (c["nodes"] * 12 + 8), "flops": 0}
    if c["op"] == "commit":
        # about three moved tokens a sequence, read and written
        return {"bytes": 2 * n * min(c["nodes"], 4) * 0.75 * c["layers"] * c["hkv"] * c["slot"] + 8 * n, "flops": 0}
    hkv, d = c["hkv"], c["d"]
    hq = hkv * c["group"]
    ctx = (c["lo"] + c["hi"]) / 2
    nodes = (1 + c["nodes"]) / 2 if c["ragged"] else c["nodes"]
    if c["window"]:
        ctx = min(ctx, c["window"])
    slot = 4 * d if c["kb"] == RAW else d * (c["kb"] + c["vb"]) / 8 + 6
    size = 4 if c["dtype"] == "fp32" else 2
    return {"bytes": n * ((ctx + nodes) * (hkv * slot + 4 / c["page"]) + nodes * hq * d * 2 * size),
            "flops": 4.0 * n * nodes * (ctx + nodes / 2) * hq * d}


# ---------------------------------------------------------------------------
# the attention in 64 bits
# ---------------------------------------------------------------------------

def _codes64(rows, first, n, bits):
    """The bits of each code, summed with their weights."""
    at = 8 * first + torch.arange(n, device=DEV)[:, None] * bits + torch.arange(bits, device=DEV)[None]
    bit = (rows[:, at // 8] >> (at % 8).to(torch.uint8)) & 1
    return (bit.long() << torch.arange(bits, device=DEV)).sum(-1)


def _half64(rows, first):
    return rows[:, first:first + 2].contiguous().view(torch.float16).double()


@torch.no_grad()
def exact(case, seed):
    c = case
    if c["op"] != "tree":
        return None
    s = _prepare_tree(c, seed)
    d, page, G = c["d"], c["page"], c["group"]
    had = _hadamard(d, torch.float64)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    at, lens = s.qsl.tolist(), s.lens.tolist()
    for b, length in enumerate(lens):
        a, n = at[b], at[b + 1] - at[b]
        ctx = length - n
        pos = torch.arange(length, device=DEV)
        slots = s.bt[b][pos // page].long() * page + pos % page
        sees = torch.ones(n, length, dtype=torch.bool, device=DEV)
        if s.start is not None:
            sees &= pos[None] >= s.start[a:a + n, None]
        for j in range(n):
            sees[:, ctx + j] = torch.arange(n, device=DEV) >= j if s.mask is None else (s.mask[a:a + n, j // 64] >> (j % 64)) & 1 != 0
        for h in range(c["hkv"]):
            rows = s.cache.flatten(0, 1)[slots, h]
            if c["kb"] == RAW:
                k = rows[:, :2 * d].contiguous().view(torch.float16).double()
                v = rows[:, 2 * d:4 * d].contiguous().view(torch.float16).double()
            else:
                nk = d * c["kb"] // 8
                f = nk + 2 + d * c["vb"] // 8
                table = s.lev.double()[_codes64(rows, 0, d, c["kb"])]
                k = table / (table.square().sum(1, keepdim=True) + 1e-16).sqrt() * _half64(rows, nk) @ had.T
                v = _codes64(rows, nk + 2, d, c["vb"]) * _half64(rows, f) + _half64(rows, f + 2)
                if c["vrot"]:
                    v = v @ had.T
            for i in range(G):
                w = s.q[a:a + n, h * G + i].double() @ k.T * s.scale
                w = torch.softmax(w.masked_fill(~sees, -math.inf), -1)
                out[a:a + n, h * G + i] = torch.nan_to_num(w) @ v
    return out
