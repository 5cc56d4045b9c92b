"""The steps around a speculative decode's attention (``steps``): block tables
and slots from lengths, the accepted path of a tree, and the move of its slots,
against plain Python over lists.  Whole numbers and bytes: everything is equal."""
import numpy as np
import pytest
import torch

I32 = torch.int32


def _plain_tables(qsl, past, table, bs, total, depths=None, held=None, free=None):
    """The same from lists; table, held and free change in place."""
    width = len(table[0]) if table else 0
    lens = [p + b - a for p, a, b in zip(past, qsl[:-1], qsl[1:])]
    missing = 0
    if held is not None:
        want = [min(-(-n // bs), width) for n in lens]
        missing = sum(-(-n // bs) - w for n, w in zip(lens, want))
        for i, w in enumerate(want):
            free.extend(table[i][w:held[i]])
            held[i] = min(held[i], w)
        for i, w in enumerate(want):
            while held[i] < w:
                if not free:
                    missing += w - held[i]
                    break
                table[i][held[i]] = free.pop()
                held[i] += 1
    slots, pos, req = [-1] * total, [0] * total, [-1] * total
    for b in range(len(past)):
        for i, t in enumerate(range(qsl[b], min(qsl[b + 1], total))):
            at = past[b] + i
            page = at // bs
            req[t], pos[t] = b, past[b] + (depths[t] if depths is not None else i)
            if page < (held[b] if held is not None else width) and table[b][page] >= 0:
                slots[t] = table[b][page] * bs + at % bs
    return slots, pos, req, lens, [missing]


def _dev(x, cuda, dtype=I32):
    return torch.tensor(x, dtype=dtype, device=cuda)


def _check(got, want):
    for name, g, w in zip(got._fields, got, want):
        assert g.tolist() == list(w), name


@pytest.mark.gpu
@pytest.mark.parametrize("B,most,bs,pad", [(1, 1, 16, 0), (3, 5, 16, 2), (7, 40, 1, 0), (64, 8, 16, 3), (5, 700, 48, 1),
                                           (300, 20, 32, 0), (2, 5000, 16, 7), (4096, 2, 16, 1)])
def test_tables_without_a_free_list(cuda, B, most, bs, pad):
    from fused_turboquant import steps
    r = np.random.RandomState(B)
    past, new = r.randint(0, 300, B), r.randint(0, most + 1, B)
    qsl = [0] + np.cumsum(new).tolist()
    width = int((past + new).max()) // bs  # the longest one's last tokens may have no page
    table = r.randint(-1, 10 ** 6, (B, max(width, 1))).tolist()
    total = qsl[-1] + pad
    depths = r.randint(0, 50, total).tolist()
    bt = _dev(table, cuda)
    for dep in (None, depths):
        got = steps.step_tables(_dev(qsl, cuda), _dev(past, cuda), bt, bs, total, depths=None if dep is None else _dev(dep, cuda))
        _check(got, _plain_tables(qsl, past.tolist(), table, bs, total, dep))
    assert bt.tolist() == table
    wide = torch.full((B, bt.shape[1] + 5), 77, dtype=I32, device=cuda)  # rows apart
    wide[:, 2:-3] = bt
    got2 = steps.step_tables(_dev(qsl, cuda), _dev(past, cuda), wide[:, 2:-3], bs, total, depths=_dev(depths, cuda))
    _check(got2, [g.tolist() for g in got])


@pytest.mark.gpu
@pytest.mark.parametrize("B,most,bs,pages,short,strided", [
    (1, 30, 16, 2, True, False), (3, 5, 16, 9, False, True), (9, 40, 16, 16, True, False), (33, 9, 4, 60, True, True),
    (64, 8, 16, 156, False, False), (5, 3000, 16, 871, True, False), (1024, 20, 16, 4280, False, False),
    (4096, 4, 16, 3122, True, False), (4, 0, 16, 7, False, False)])
def test_tables_grow_and_shrink(cuda, B, most, bs, pages, short, strided):
    """Twelve steps of requests that grow, end and begin; a short list runs out, and what it lacked is given later."""
    from fused_turboquant import steps
    r = np.random.RandomState(B + most)
    width = (3 * most + 40) // bs + 1
    pool = r.permutation(pages).tolist()
    table, held, free = [[-1] * width for _ in range(B)], [0] * B, list(pool)
    bt, hd = _dev(table, cuda), _dev(held, cuda)
    fb, fc = _dev(pool, cuda), _dev([len(pool)], cuda)
    if strided:
        room = torch.full((B, width + 3), -5, dtype=I32, device=cuda)
        room[:, :width] = bt
        bt = room[:, :width]
    past, ran_out = np.zeros(B, dtype=int), False
    for step in range(12):
        new = r.randint(0, most + 1, B)
        ends = r.rand(B) < 0.3
        past = np.where(ends, 0, past)
        new = np.where(ends & (r.rand(B) < 0.5), 0, new)
        qsl = [0] + np.cumsum(new).tolist()
        total = qsl[-1] + 2
        got = steps.step_tables(_dev(qsl, cuda), _dev(past, cuda), bt, bs, total, num_blocks=hd, free_blocks=fb, free_count=fc)
        want = _plain_tables(qsl, past.tolist(), table, bs, total, None, held, free)
        _check(got, want)
        assert bt.tolist() == table and hd.tolist() == held and fc.item() == len(free)
        assert fb[:len(free)].tolist() == free
        assert sorted(free + [x for row, h in zip(table, held) for x in row[:h]]) == sorted(pool)
        ran_out = ran_out or want[4][0] > 0
        past = past + r.randint(0, new + 1)  # what the step accepted
        past = np.minimum(past, 2 * most + 40)
    assert ran_out == short


@pytest.mark.gpu
def test_tables_of_nothing(cuda):
    from fused_turboquant import steps
    z = torch.zeros(0, dtype=I32, device=cuda)
    got = steps.step_tables(_dev([0], cuda), z, torch.zeros(0, 4, dtype=I32, device=cuda), 16, 3)
    _check(got, ([-1] * 3, [0] * 3, [-1] * 3, [], [0]))
    got = steps.step_tables(_dev([0], cuda), z, torch.zeros(0, 4, dtype=I32, device=cuda), 16, 0, num_blocks=z, free_blocks=_dev([4], cuda),
                            free_count=_dev([1], cuda))
    _check(got, ([], [], [], [], [0]))
    got = steps.step_tables(_dev([0, 2], cuda), _dev([0], cuda), torch.zeros(1, 0, dtype=I32, device=cuda), 16, 2)
    _check(got, ([-1, -1], [0, 1], [0, 0], [2], [0]))


def _plain_accept(tokens, parents, targets, qsl, width):
    paths, counts, out = [], [], []
    for a, b in zip(qsl[:-1], qsl[1:]):
        n, path = min(b - a, width), []
        cur = 0 if n > 0 else n
        while cur < n:
            path.append(cur)
            cur = next((j for j in range(cur + 1, n) if parents[a + j] == cur and tokens[a + j] == targets[a + cur]), n)
        paths.append(path + [-1] * (width - len(path)))
        counts.append(len(path))
        out.append([targets[a + i] for i in path] + [-1] * (width - len(path)))
    return paths, counts, out


@pytest.mark.gpu
@pytest.mark.parametrize("B,nodes,vocab,width", [(1, 1, 5, 1), (3, 8, 2, 8), (64, 61, 2, 61), (5, 300, 2, 300), (2, 2048, 1, 2048),
                                                 (9, 40, 3, 17), (4, 64, 2, 100), (300, 5, 2, 5)])
def test_accept(cuda, B, nodes, vocab, width):
    from fused_turboquant import steps
    r = np.random.RandomState(nodes)
    counts = r.randint(0, nodes + 1, B)
    counts[0] = nodes
    qsl = [0] + np.cumsum(counts).tolist()
    parents = [p for n in counts for p in [-1] + [int(r.randint(max(0, i - 4), i)) for i in range(1, n)]][:qsl[-1]] if qsl[-1] else []
    parents = []
    for n in counts:
        parents += [(-1 if i == 0 else int(r.randint(max(0, i - 4), i))) for i in range(n)]
    tokens, targets = r.randint(0, vocab, qsl[-1]) + 2 ** 40, r.randint(0, vocab, qsl[-1]) + 2 ** 40
    got = steps.tree_accept(_dev(tokens, cuda, torch.int64), _dev(parents, cuda), _dev(targets, cuda, torch.int64), _dev(qsl, cuda), width)
    _check(got, _plain_accept(tokens.tolist(), parents, targets.tolist(), qsl, width))


@pytest.mark.gpu
def test_accept_odd_trees(cuda):
    """Equal siblings, parents at or behind their child, a root whose own entries could match, no sequences."""
    from fused_turboquant import steps
    parents = [0, 0, 0, 2, 1, 9, -1, 4]
    tokens, targets = [7, 7, 7, 7, 7, 7, 7, 7], [7] * 8
    got = steps.tree_accept(_dev(tokens, cuda, torch.int64), _dev(parents, cuda), _dev(targets, cuda, torch.int64), _dev([0, 8], cuda), 8)
    _check(got, _plain_accept(tokens, parents, targets, [0, 8], 8))
    assert got.path[0, :4].tolist() == [0, 1, 4, 7]
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    got = steps.tree_accept(none, none.to(I32), none, _dev([0], cuda), 4)
    assert got.path.shape == (0, 4) and got.counts.numel() == 0


def _plain_commit(cache, table, past, path, counts):
    nb, bs = cache.shape[:2]
    flat = cache.copy()
    for b in range(len(past)):
        before = flat.copy()
        last = -1
        for j in range(min(counts[b], path.shape[1])):
            if path[b, j] <= last:
                break
            last = path[b, j]
            where = [(past[b] + x) for x in (last, j)]
            ids = [table[b][w // bs] if w // bs < len(table[b]) else -1 for w in where]
            if all(0 <= i < nb for i in ids):
                flat[ids[1], where[1] % bs] = before[ids[0], where[0] % bs]
    return flat


@pytest.mark.gpu
@pytest.mark.parametrize("layers,hkv,slot,bs,B,nodes", [(1, 8, 128, 16, 3, 9), (3, 2, 52, 16, 5, 40), (70, 1, 64, 32, 2, 7),
                                                        (2, 4, 1024, 16, 1, 61), (2, 3, 36, 48, 40, 5), (1, 16, 512, 16, 2, 700)])
def test_commit(cuda, layers, hkv, slot, bs, B, nodes):
    from fused_turboquant import steps
    r = np.random.RandomState(layers + nodes)
    past = r.randint(0, 100, B)
    pages = (past + nodes + bs - 1) // bs
    nb = int(pages.sum()) + 2
    perm, at = r.permutation(nb), 0
    table = np.full((B, int(pages.max())), -1, dtype=np.int32)
    for i, n in enumerate(pages):
        table[i, :n] = perm[at:at + n]
        at += n
    table[-1, -1] = nb + 3 if nodes > 8 else table[-1, -1]  # a page past the cache
    path, counts = np.full((B, nodes), -1, dtype=np.int32), np.zeros(B, dtype=np.int32)
    for i in range(B):
        n = r.randint(0, nodes + 1)
        got = np.sort(r.permutation(nodes)[:n])
        path[i, :n], counts[i] = got, n
    if B > 2:
        path[0, :4], counts[0] = [0, 3, 3, 4], 4          # an entry that does not ascend
        counts[1] = nodes + 50                            # -1 ends a path too
    caches = [torch.randint(0, 256, (nb, bs, hkv, slot), dtype=torch.uint8) for _ in range(layers)]
    want = [_plain_commit(c.numpy(), table, past, path, counts) for c in caches]
    for shift in (0, 4):  # the cache itself, and a view whose slots are 4 bytes off
        dev = []
        for c in caches:
            room = torch.full((nb, bs, hkv, slot + shift), 9, dtype=torch.uint8, device=cuda)
            room[..., shift:] = c.to(cuda)
            dev.append(room[..., shift:])
        steps.commit_slots(dev, _dev(table, cuda), _dev(past, cuda), _dev(path, cuda), _dev(counts, cuda))
        for d, w in zip(dev, want):
            assert np.array_equal(d.cpu().numpy(), w)
    steps.commit_slots([], _dev(table, cuda), _dev(past, cuda), _dev(path, cuda), _dev(counts, cuda))


@pytest.mark.gpu
def test_steps_captured_and_replayed(cuda):
    """A whole step's bookkeeping in a graph, on a state that the replays move on."""
    from fused_turboquant import steps
    B, N, bs, width = 4, 6, 16, 20
    r = np.random.RandomState(1)
    pool = r.permutation(70)
    state = dict(bt=_dev(np.full((B, width), -1), cuda), hd=_dev([0] * B, cuda), fb=_dev(pool, cuda), fc=_dev([70], cuda),
                 past=_dev([0, 15, 30, 47], cuda))
    qsl, parents = _dev(np.arange(B + 1) * N, cuda), _dev([-1, 0, 0, 1, 2, 3] * B, cuda)
    tokens, targets = (torch.zeros(B * N, dtype=torch.int64, device=cuda) for _ in range(2))
    cache = torch.randint(0, 256, (70, bs, 2, 64), dtype=torch.uint8, device=cuda)

    def step(s, c):
        t = steps.step_tables(qsl, s["past"], s["bt"], bs, B * N, num_blocks=s["hd"], free_blocks=s["fb"], free_count=s["fc"])
        a = steps.tree_accept(tokens, parents, targets, qsl, N)
        steps.commit_slots([c], s["bt"], s["past"], a.path, a.counts)
        s["past"].add_(a.counts)
        return (*t, *a)

    other = {k: v.clone() for k, v in state.items()}
    spare = cache.clone()
    begin = {k: v.clone() for k, v in state.items()}
    step(state, cache)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(state, cache)
    for k in state:
        state[k].copy_(begin[k])
    cache.copy_(spare)
    for rep in range(5):
        tokens.copy_(torch.from_numpy(r.randint(0, 2, B * N)))
        targets.copy_(torch.from_numpy(r.randint(0, 2, B * N)))
        want = step(other, spare)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), rep
        assert all(torch.equal(state[k], other[k]) for k in state) and torch.equal(cache, spare), rep


def _tab(**change):
    z = lambda *s: torch.zeros(*s, dtype=I32)  # noqa: E731
    return {**dict(query_start_loc=z(3), past_lens=z(2), block_table=z(2, 4), block_size=16, num_tokens=4), **change}


@pytest.mark.parametrize("change,match", [
    (dict(query_start_loc=torch.zeros(2, dtype=I32)), "query_start_loc"), (dict(past_lens=torch.zeros(2)), "past_lens"),
    (dict(block_table=torch.zeros(3, 4, dtype=I32)), "block_table"), (dict(block_table=torch.zeros(4, 2, dtype=I32).t()), "rows"),
    (dict(block_table=torch.zeros(1, 4, dtype=I32).expand(2, 4)), "overlap"),
    (dict(block_size=0), "block_size"), (dict(num_tokens=-1), "num_tokens"), (dict(depths=torch.zeros(3, dtype=I32)), "depths"),
    (dict(num_blocks=torch.zeros(2, dtype=I32)), "go together"),
    (dict(num_blocks=torch.zeros(2, dtype=I32), free_blocks=torch.zeros(9, dtype=I32), free_count=torch.zeros(2, dtype=I32)), "free_count"),
    (dict(num_blocks=torch.zeros(4, dtype=I32)[::2], free_blocks=torch.zeros(9, dtype=I32), free_count=torch.zeros(1, dtype=I32)), "num_blocks"),
    (dict(past_lens=torch.zeros(4097, dtype=I32), query_start_loc=torch.zeros(4098, dtype=I32)), "4096"),
])
def test_table_refusals(change, match):
    from fused_turboquant import steps
    with pytest.raises(ValueError, match=match):
        steps.step_tables(**_tab(**change))


def test_accept_and_commit_refusals():
    from fused_turboquant import _lib, steps
    i64, z = torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=I32)
    qsl = torch.tensor([0, 4], dtype=I32)
    for args, match in (((i64, z[:3], i64, qsl, 4), "one entry"), ((z, z, i64, qsl, 4), "tokens"), ((i64, i64, i64, qsl, 4), "parents"),
                        ((i64, z, i64, qsl, 0), "max_nodes"), ((i64, z, i64, qsl, 2049), "max_nodes"), ((i64, z, i64, qsl[:0], 4), "B \\+ 1")):
        with pytest.raises(ValueError, match=match):
            steps.tree_accept(*args)
    with pytest.raises(_lib.FusedTQError):
        steps.tree_accept(i64, z, i64, qsl, 4)
    with pytest.raises(_lib.FusedTQError):
        steps.step_tables(**_tab())
    c = torch.zeros(2, 16, 1, 64, dtype=torch.uint8)
    bt, past, path, cnt = torch.zeros(1, 2, dtype=I32), torch.zeros(1, dtype=I32), torch.zeros(1, 3, dtype=I32), torch.zeros(1, dtype=I32)
    for args, match in ((([c, c], bt, past, path, cnt), "twice"), (([c, c[:1].clone()], bt, past, path, cnt), "one shape"),
                        (([c.float()], bt, past, path, cnt), "uint8"), (([c[..., ::2]], bt, past, path, cnt), "contiguous"),
                        (([c], bt.long(), past, path, cnt), "block_table"), (([c], bt, past, path[0], cnt), "path"),
                        (([c], bt, torch.zeros(2, dtype=I32), path, cnt), "past_lens")):
        with pytest.raises(ValueError, match=match):
            steps.commit_slots(*args)
    with pytest.raises(_lib.FusedTQError):
        steps.commit_slots([c], bt, past, path, cnt)


@pytest.mark.gpu
@pytest.mark.parametrize("spoil,match", [
    (lambda c: [c[0], c[0]], "twice"), (lambda c: [c[0], c[1][:3]], "one shape"), (lambda c: [c[0], c[1].int()], "uint8"),
    (lambda c: [c[0], c[1].transpose(1, 2)], "one shape"), (lambda c: [c[0], c[1].cpu()], "one device"),
    (lambda c: [c[0][0], c[1]], "uint8"), (lambda c: [c[0][..., ::2], c[1][..., ::2]], "contiguous")])
def test_commit_refuses_caches_on_the_device(cuda, spoil, match):
    from fused_turboquant import steps
    caches = [torch.randint(0, 256, (4, 16, 16, 64), dtype=torch.uint8, device=cuda) for _ in range(2)]
    was = [c.clone() for c in caches]
    i32 = dict(dtype=I32, device=cuda)
    args = (torch.zeros(1, 4, **i32), torch.zeros(1, **i32), torch.tensor([[0, 2, 3]], **i32), torch.full((1,), 3, **i32))
    with pytest.raises(ValueError, match=match):
        steps.commit_slots(spoil(caches), *args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(caches, was))
