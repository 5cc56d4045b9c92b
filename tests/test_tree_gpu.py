"""Tree attention (``v1_tree_attention``): several query tokens a sequence over
their stored slots, against attention in 64 bits over the same cache bytes.

Tolerances, as the 2-norm of the error over the 2-norm of the result.  An output
type rounds by at most half a step (bf16 2^-8, fp16 2^-11, fp32 2^-24).  fp32
outputs: every operand is carried as f16 hi + lo (2^-22) and sums in fp32, so
the rest stays below 1e-5.  16-bit outputs: keys may be f16 table values and
weights f16 numbers, each off by 2^-11 at most.  The errors of a score's terms
add up as the roundings of independent values do, to at most e = 2^-11 scale
||q_i k_i||, a weight is off by a factor of 1 + 2 e + 2^-11, and the output by
that share of sum p |v|; ``want`` computes both from the data.
"""
import math

import numpy as np
import pytest
import torch

from oracle import tq_oracle as O

RAW = 16
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Case:
    """Sequences of ``ctx[b]`` context positions and ``counts[b]`` nodes, stored through the library's own stores."""

    def __init__(self, cuda, d, kb, vb, hkv, G, ctx, counts, page=16, vrot=False, lloyd=False, fp8=False, kind="rht", seed=0,
                 pad=0, spare=3):
        from fused_turboquant import raw as R, v1 as V1
        g = torch.Generator().manual_seed(seed)
        self.d, self.kb, self.vb, self.hkv, self.G = d, kb, vb, hkv, G
        self.lens = [a + n for a, n in zip(ctx, counts)]
        self.ctx, self.counts = list(ctx), list(counts)
        pages = [(n + page - 1) // page for n in self.lens]
        nb = sum(pages) + spare
        perm = torch.randperm(nb, generator=g).to(torch.int32)
        self.bt = torch.full((len(ctx), max(max(pages), 1)), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(pages):
            self.bt[i, :n] = perm[at:at + n]
            at += n
        self.layer = None if kb == RAW else V1.TurboQuantV1Layer(d, kb, vb, v_rotate=vrot, device=cuda, v_lloyd_max=lloyd,
                                                                 key_fp8=fp8, kind=kind)
        slot = (4 * d if kb == RAW else V1.slot_bytes(d, kb, vb, fp8)) + pad
        slot += -slot % 4
        self.cache = torch.randint(0, 256, (nb, page, hkv, slot), dtype=torch.uint8, generator=g).to(cuda)
        for i, n in enumerate(self.lens):
            if n == 0:
                continue
            k = torch.randn(n, hkv, d, generator=g)
            k[:: 37] *= 6.0  # outlier keys
            v = torch.randn(n, hkv, d, generator=g) + 0.5
            pos = torch.arange(n)
            slots = (self.bt[i].long()[pos // page] * page + pos % page).to(cuda)
            kd, vd = k.to(torch.bfloat16).to(cuda), v.to(torch.bfloat16).to(cuda)
            if self.layer is None:
                R.raw_store(kd, vd, self.cache, slots)
            else:
                self.layer.store(kd, vd, self.cache, slots)
        self.bt = self.bt.to(cuda)
        self.sl = torch.tensor(self.lens, dtype=torch.int32, device=cuda)
        self.qsl = torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device=cuda)
        self.T = sum(counts)
        self.q = torch.randn(self.T, hkv * G, d, generator=g).to(cuda)
        self.scale = 1 / math.sqrt(d)

    def trees(self, seed=1, words=None):
        """Masks of random trees (each node its ancestors and itself)."""
        r = np.random.RandomState(seed)
        words = words or max((max(self.counts + [1]) + 63) // 64, 1)
        rows = []
        for n in self.counts:
            anc = []
            for i in range(n):
                anc.append((anc[r.randint(max(0, i // 3 - 1), i)] if i else 0) | 1 << i)
            rows += anc
        return self.words(rows, words)

    def words(self, rows, words):
        m = np.array([[(x >> 64 * w) & (2 ** 64 - 1) for w in range(words)] for x in rows], dtype=np.uint64).reshape(-1, words)
        return torch.from_numpy(m.view(np.int64)).to(self.q.device)

    def run(self, mask=None, q=None, **kw):
        from fused_turboquant import v1 as V1
        q = self.q if q is None else q
        if self.layer is None:
            return V1.v1_tree_attention(q, self.cache, self.bt, self.sl, self.qsl, None, RAW, RAW, tree_mask=mask, **kw)
        return self.layer.tree(q, self.cache, self.bt, self.sl, self.qsl, tree_mask=mask, **kw)

    def want(self, mask=None, start=None, q=None):
        """(output, log-sum-exps, tolerance share of 16-bit operands) in 64 bits."""
        c, L = self.cache.cpu().numpy(), self.layer
        q = (self.q if q is None else q).double().cpu().numpy()
        rot = None
        if L is None:
            k_all, v_all = O.raw_unpack(c, self.d)
        else:
            k_all, v_all = O.v1_dequant(c, self.d, self.kb, self.vb, None if L.key_fp8 else L.centroids.cpu().numpy(), True,
                                        L.v_lloyd_max, L.key_fp8)
            rot = O.sylvester(self.d) / math.sqrt(self.d) if L.rotation is None else L.rotation.cpu().double().numpy()
            q = q @ rot
        bt, page, nb = self.bt.cpu().numpy(), c.shape[1], c.shape[0]
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        size, worst = np.zeros(q.shape), 0.0
        words = None if mask is None else mask.cpu().numpy().view(np.uint64)
        t = 0
        for b, n in enumerate(self.counts):
            pos = np.arange(self.lens[b])
            page_of = pos // page
            ids = np.where(page_of < bt.shape[1], bt[b][np.minimum(page_of, bt.shape[1] - 1)], -1)
            held = (ids >= 0) & (ids < nb)
            for i in range(n):
                rel = pos - self.ctx[b]
                if words is None:
                    sees = rel <= i
                else:
                    bits = [j for j in range(n) if j // 64 < words.shape[1] and int(words[t][j // 64]) >> (j % 64) & 1]
                    sees = (rel < 0) | np.isin(rel, bits)
                sees &= held & ~((rel < 0) & (pos < (0 if start is None else int(start[t]))))
                at, off = ids[sees], pos[sees] % page
                for h in range(q.shape[1]):
                    if not sees.any():
                        continue
                    k, v = k_all[at, off, h // self.G], v_all[at, off, h // self.G]
                    s = k @ q[t, h] * self.scale
                    worst = max(worst, float(np.sqrt((k * k) @ (q[t, h] * q[t, h])).max() * self.scale))
                    m = s.max()
                    p = np.exp(s - m)
                    lse[t, h] = m + np.log(p.sum())
                    out[t, h] = p / p.sum() @ v
                    size[t, h] = p / p.sum() @ np.abs(v)
                t += 1
        share = (2.0 ** -11 + 2 * 2.0 ** -11 * worst) * np.linalg.norm(size) / max(np.linalg.norm(out), 1e-30)
        if L is not None and L.v_rotate:
            out = out @ rot.T
        return out, lse, share


def _rel(got, want):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    return float(np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30))


CASES = [
    # d, kb, vb, hkv, G, contexts, nodes, page, vrot, lloyd, fp8, kind
    (128, 4, 4, 2, 4, [37, 0, 200], [9, 1, 33], 16, False, False, False, "rht"),
    (128, 3, 3, 2, 4, [31, 32, 33], [1, 31, 32], 32, True, False, False, "rht"),   # tile and workgroup edges
    (128, 4, 2, 1, 8, [1500], [16], 16, True, False, False, "rht"),                # several splits
    (128, 2, 4, 2, 7, [64, 5], [19, 40], 64, False, False, False, "rht"),          # a group that does not divide the columns
    (128, 3, 4, 1, 1, [90], [150], 16, True, False, False, "rht"),                 # three mask words
    (128, 4, 4, 2, 4, [90, 70], [20, 7], 16, True, False, False, "planar"),        # a matrix un-rotation
    (128, 4, 4, 2, 2, [90, 40], [20, 33], 16, True, True, False, "rht"),           # Lloyd-Max V
    (128, 3, 4, 1, 4, [77], [20], 16, True, True, False, "rht"),                   # ... with a smaller table than its codes
    (64, 4, 4, 2, 4, [63, 64, 65, 0], [1, 5, 33, 2], 16, False, False, False, "rht"),
    (64, 3, 2, 1, 16, [700], [9], 128, True, False, False, "rht"),
    (64, 2, 3, 2, 4, [129, 3], [64, 65], 16, True, False, False, "rht"),
    (256, 4, 3, 2, 2, [95, 31], [33, 8], 16, True, False, False, "rht"),
    (256, 2, 2, 1, 5, [640], [14], 16, False, False, False, "rht"),
    (256, 3, 4, 1, 4, [100], [6], 16, True, True, False, "rht"),
    (128, 1, 1, 2, 4, [77, 20], [20, 3], 16, True, False, False, "rht"),
    (256, 1, 3, 1, 4, [77], [20], 16, False, False, False, "rht"),
    (64, 4, 1, 1, 4, [77], [20], 16, False, False, False, "rht"),
    (128, 8, 8, 1, 4, [77, 300], [20, 4], 16, False, False, False, "rht"),
    (64, 8, 8, 1, 4, [77], [20], 16, True, False, True, "rht"),                    # fp8 keys
    (256, 8, 8, 1, 2, [50], [12], 32, True, False, False, "rht"),
    (64, RAW, RAW, 2, 4, [77, 5], [20, 9], 16, False, False, False, "rht"),        # raw fp16 slots
    (128, RAW, RAW, 2, 8, [300, 0], [20, 40], 16, False, False, False, "rht"),
    (256, RAW, RAW, 1, 2, [77], [40], 16, False, False, False, "rht"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("d,kb,vb,hkv,G,ctx,counts,page,vrot,lloyd,fp8,kind", CASES)
def test_tree_matches_64_bits(cuda, d, kb, vb, hkv, G, ctx, counts, page, vrot, lloyd, fp8, kind, tree):
    c = Case(cuda, d, kb, vb, hkv, G, ctx, counts, page, vrot, lloyd, fp8, kind, seed=d + sum(ctx))
    mask = c.trees() if tree else None
    lse = torch.empty(c.T, hkv * G, device=cuda)
    want, wlse, share = c.want(mask)
    for splits in (1, 3):
        got = c.run(mask, num_splits=splits, lse=lse)
        print(f"[tree d{d} k{kb}v{vb} G{G} {counts} splits {splits}] rel {_rel(got, want):.2e}", flush=True)
        assert got.dtype == torch.float32 and _rel(got, want) < 1e-5
        assert np.abs(lse.cpu().numpy() - wlse).max() < 1e-4
    for dtype in (torch.bfloat16, torch.float16):
        q = c.q.to(dtype)
        want, _, share = c.want(mask, q=q)
        got = c.run(mask, q=q)
        err = _rel(got.float(), want)
        print(f"[tree {dtype}] rel {err:.2e} of {HALF[dtype] + share:.2e}", flush=True)
        assert got.dtype == dtype and err < HALF[dtype] + share


@pytest.mark.gpu
@pytest.mark.parametrize("d,kb,vb", [(64, 4, 4), (128, 3, 3), (128, RAW, RAW), (256, 4, 2)])
def test_starts_and_masks_that_leave_rows_empty(cuda, d, kb, vb):
    c = Case(cuda, d, kb, vb, 1, 4, [70, 0, 40], [12, 9, 5], seed=3)
    r = np.random.RandomState(5)
    rows = [int(r.randint(0, 2 ** 30)) | int(r.randint(0, 2)) << 63 for _ in range(c.T)]  # bits past the nodes count for nothing
    for t in (0, 4, 13, 14, 21):
        rows[t] = 0
    start = r.randint(-2, 75, c.T)
    start[0], start[4], start[22] = 70, 2 ** 31 - 1, 40
    start = torch.tensor(start, dtype=torch.int32, device=cuda)
    mask = c.words(rows, 1)
    want, wlse, _ = c.want(mask, start)
    empty = np.isneginf(wlse)
    assert empty[[0, 4, 13, 14]].all() and not empty.all()
    for splits in (1, 4):
        lse = torch.empty(c.T, 4, device=cuda)
        got = c.run(mask, kv_start=start, num_splits=splits, lse=lse)
        assert _rel(got, want) < 1e-5
        assert (got.cpu().numpy()[empty] == 0).all() and np.array_equal(np.isneginf(lse.cpu().numpy()), empty)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2])
def test_empty_sequences_and_rows_behind_the_last(cuda, splits):
    """Sequences without nodes, and padding tokens, whose rows stay as they were."""
    c = Case(cuda, 128, 4, 4, 1, 4, [50, 40, 0, 33], [3, 0, 0, 6], seed=4)
    q = torch.cat((c.q, torch.full((5, 4, 128), float("nan"), device=cuda)))
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device=cuda)
    c.run(None, q=q, out=out, lse=lse, num_splits=splits)
    assert _rel(out[:9], c.want()[0]) < 1e-5
    assert (out[9:] == 7).all() and (lse[9:] == 7).all()
    none = Case(cuda, 64, 3, 3, 1, 2, [5, 0], [0, 0], seed=4)
    assert none.run().shape == (0, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("d,kb,vb", [(128, 4, 4), (64, RAW, RAW), (256, 8, 8)])
def test_pages_that_are_missing_hide_their_positions(cuda, d, kb, vb):
    c = Case(cuda, d, kb, vb, 2, 2, [160], [10], seed=5)
    c.bt[0, 2], c.bt[0, 5] = -1, c.cache.shape[0] + 7
    assert _rel(c.run(), c.want()[0]) < 1e-5
    c.bt = c.bt[:, :9].contiguous()  # the last pages, some nodes among them, are past the table
    assert _rel(c.run(), c.want()[0]) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("d,kb,vb,pad", [(128, 4, 4, 0), (128, 3, 3, 4), (64, 2, 2, 8), (256, 4, 3, 20), (128, RAW, RAW, 16)])
def test_cache_and_query_strides(cuda, d, kb, vb, pad):
    """Slots at 4-byte offsets, heads and positions apart, queries that are views."""
    c = Case(cuda, d, kb, vb, 2, 4, [45, 100], [9, 14], seed=6, pad=pad)
    want = c.run()
    nb, bs, hkv, slot = c.cache.shape
    wide = torch.zeros(nb, bs + 1, hkv + 1, slot + 12, dtype=torch.uint8, device=cuda)
    view = wide[:, :bs, 1:, 8:8 + slot]
    view.copy_(c.cache)
    c.cache = view
    assert torch.equal(c.run(), want)
    big = torch.zeros(c.T, c.q.shape[1] + 2, d, device=cuda)
    big[:, 1:-1] = c.q
    assert torch.equal(c.run(q=big[:, 1:-1]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("d,kb,vb", [(64, 4, 4), (128, 3, 3), (256, 4, 3), (128, 8, 8)])
def test_fields_of_hidden_positions_may_hold_anything(cuda, d, kb, vb):
    """NaN and infinite norms, scales and minima behind a start, beyond the nodes and in unseen nodes."""
    c = Case(cuda, d, kb, vb, 1, 4, [40], [12], seed=7)
    start = torch.full((12,), 9, dtype=torch.int32, device=cuda)
    rows = [1 << i | 1 for i in range(12)]  # nodes 1 .. 10 are seen by themselves alone
    mask = c.words(rows, 1)
    want = c.run(mask, kv_start=start)
    lay = c.layer
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=torch.float16, device=cuda).view(torch.uint8)
    nk = d * kb // 8
    v0 = nk + 2 + d * vb // 8
    for pos in (0, 5, 8, 45, 52, 60):
        if pos >= c.bt.shape[1] * 16:
            continue
        s = c.cache[c.bt[0, pos // 16].long(), pos % 16, 0]
        s[nk:nk + 2] = bad[:2]
        s[v0:v0 + 4] = bad[2:6]
    got = c.run(mask, kv_start=start)
    keep = [i for i in range(12) if i != 5]  # position 45 is node 5
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[5]).all()
    assert lay is not None


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_an_infinite_raw_value_stays_in_the_rows_that_attend_it(cuda, d):
    c = Case(cuda, d, RAW, RAW, 1, 2, [40], [12], seed=8)
    mask = c.words([1 << i | 1 for i in range(12)], 1)
    want = c.run(mask)
    v = c.cache[c.bt[0, 2].long(), 13, 0].view(torch.float16)  # position 45, node 5
    v[d + 5], v[2 * d - 1] = float("inf"), float("nan")
    got = c.run(mask)
    keep = [i for i in range(12) if i != 5]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[5][:, [5, d - 1]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("past", [40, 3000])
def test_nan_and_huge_queries_stay_in_their_rows(cuda, past):
    c = Case(cuda, 128, 4, 4, 1, 4, [past], [20], seed=9)
    for dtype in (torch.float32, torch.bfloat16):
        q = c.q.to(dtype)
        want = c.run(q=q)
        odd = q.clone()
        odd[7, 2, 5] = float("nan")
        odd[3, 1] *= 1e6  # beyond f16 once scaled
        got = c.run(q=odd)
        assert torch.isnan(got[7, 2]).all() and torch.isfinite(got[3, 1]).all()
        got[7, 2], got[3, 1] = want[7, 2], want[3, 1]
        assert _rel(got.float(), want.double().cpu().numpy()) < 1e-6
    one = c.q.clone()
    one[3, 1] *= 1e4
    w, _, _ = c.want(q=one)
    assert _rel(c.run(q=one)[3, 1], w[3, 1]) < 1e-3  # a score error of 2^-22 of scores near 1e4


@pytest.mark.gpu
@pytest.mark.parametrize("below", [20, 24])
@pytest.mark.parametrize("d,bits", [(64, RAW), (128, RAW), (64, 4), (128, 4), (256, 8)])
def test_one_dominant_key_and_a_long_tail(cuda, d, bits, below):
    """One key takes most of the weight; 30000 others, ``below`` log2 units under it, together still move the output."""
    from fused_turboquant import raw as R
    past, n, G = 30000, 4, 2
    c = Case(cuda, d, bits, bits, 1, G, [past], [n], seed=10)
    g = torch.Generator().manual_seed(d)
    k, v = torch.randn(past + n, 1, d, generator=g) * 0.02, torch.randn(past + n, 1, d, generator=g) * 0.5 + 0.5
    u = torch.randn(d, generator=g)
    u /= u.norm()
    k[0, 0] = 30 * u
    c.q = (torch.randn(n, G, d, generator=g) * 0.05 + u * (below * math.log(2) * math.sqrt(d) / 30)).to(cuda)
    pos = torch.arange(past + n, device=cuda)
    slots = c.bt[0].long()[pos // 16] * 16 + pos % 16
    (R.raw_store if bits == RAW else lambda *a: c.layer.store(*a))(k.to(cuda), v.to(cuda), c.cache, slots)
    err = _rel(c.run(), c.want()[0])
    print(f"[tree tail d{d} bits {bits} below {below}] rel {err:.2e}", flush=True)
    assert err < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("d,kb,vb", [(64, 4, 2), (128, 3, 4), (256, 2, 2), (128, 8, 8)])
def test_one_token_equals_decode_and_a_chain_equals_a_chunk(cuda, d, kb, vb):
    from fused_turboquant import v1 as V1
    c = Case(cuda, d, kb, vb, 2, 4, [100, 0, 33], [1, 1, 1], vrot=True, seed=11)
    dec = c.layer.decode(c.q, c.cache, c.bt, c.sl)
    f16_keys = d == 128 and kb < 8  # the decode kernel's
    assert _rel(c.run(), dec.double().cpu().numpy()) < (5e-4 if f16_keys else 1e-5)
    c = Case(cuda, d, kb, vb, 2, 4, [100], [37], vrot=True, seed=12)
    chunk = V1.v1_chunk_attention(c.q, c.cache, c.bt[0], 100, c.layer.centroids, kb, vb, c.scale, v_rotate=True)
    assert _rel(c.run(), chunk.double().cpu().numpy()) < (5e-4 if f16_keys else 1e-5)


@pytest.mark.gpu
def test_a_cache_past_32_bits(cuda):
    """Byte offsets beyond 2^32 in the cache."""
    c = Case(cuda, 64, 4, 4, 1, 2, [40], [5], seed=13)
    want = c.run()
    nb = (5 << 30) // (c.cache.shape[1] * c.cache.shape[3])
    big = torch.empty(nb, *c.cache.shape[1:], dtype=torch.uint8, device=cuda)
    ids = torch.arange(nb - 1, nb - 1 - c.bt.shape[1], -1, dtype=torch.int32, device=cuda)[None]
    big[ids.long()] = c.cache[c.bt.long()]
    c.cache, c.bt = big, ids.contiguous()
    assert torch.equal(c.run(), want)


@pytest.mark.gpu
def test_another_stream_and_a_launch_size_that_is_too_small(cuda):
    """The call runs on the current stream; max_query_len and max_seq_len only size the launch."""
    c = Case(cuda, 128, 3, 3, 2, 4, [300, 20], [40, 9], seed=14)
    mask = c.trees()
    want = c.run(mask, num_splits=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = c.q + 0
        got = c.run(mask, q=q, num_splits=2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert torch.equal(c.run(mask, max_query_len=1, max_seq_len=1, num_splits=2), want)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 4])
def test_captured_and_replayed(cuda, splits):
    """Two graphs that share a workspace, replayed in turn with eager calls between."""
    from fused_turboquant import v1 as V1
    c = Case(cuda, 128, 4, 4, 2, 4, [500, 100], [16, 7], seed=15)
    mask = c.trees()
    ws = torch.empty(V1.workspace_bytes(c.T, 8, 128, splits), dtype=torch.uint8, device=cuda)
    outs = [torch.empty_like(c.q) for _ in range(2)]

    def call(i):
        c.run(mask if i else None, out=outs[i], workspace=ws, num_splits=splits)

    graphs = []
    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i)
        graphs.append(g)
    for rep in range(3):
        c.q.copy_(torch.randn(c.q.shape, generator=torch.Generator().manual_seed(rep)))
        want = [c.run(mask if i else None, num_splits=splits) for i in range(2)]
        torch.cuda.synchronize()
        for i in (0, 1):
            outs[i].zero_()
            graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def _args(d=64, T=4, B=2):
    from fused_turboquant import v1 as V1
    i32 = torch.int32
    return dict(query=torch.zeros(T, 4, d), kv_cache=torch.zeros(4, 16, 2, V1.slot_bytes(d, 4, 4) + 2, dtype=torch.uint8),
                block_table=torch.zeros(B, 2, dtype=i32), seq_lens=torch.zeros(B, dtype=i32),
                query_start_loc=torch.zeros(B + 1, dtype=i32), centroids=torch.zeros(16), key_bits=4, value_bits=4)


@pytest.mark.parametrize("change,match", [
    (dict(key_bits=5), "key_bits"), (dict(key_bits=8), "8-bit"), (dict(value_bits=RAW), "key_bits"),
    (dict(key_bits=RAW, value_bits=4), "raw"), (dict(key_bits=RAW, value_bits=RAW, v_rotate=True), "raw"),
    (dict(key_bits=RAW, value_bits=RAW), "slot"), (dict(centroids=torch.zeros(8)), "centroids"), (dict(centroids=None), "centroids"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "int32"), (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "block_table"),
    (dict(query_start_loc=torch.zeros(2, dtype=torch.int32)), "query_start_loc"),
    (dict(tree_mask=torch.zeros(4, dtype=torch.int64)), "tree_mask"), (dict(tree_mask=torch.zeros(3, 1, dtype=torch.int64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(4, 1, dtype=torch.int32)), "tree_mask"), (dict(tree_mask=torch.zeros(4, 0, dtype=torch.int64)), "tree_mask"),
    (dict(kv_start=torch.zeros(2, dtype=torch.int32)), "kv_start"), (dict(lse=torch.zeros(4, 3)), "lse"),
    (dict(max_query_len=0), "max_query_len"), (dict(kv_cache=torch.zeros(4, 16, 2, 8, dtype=torch.uint8)), "slot"),
])
def test_tree_refusals(change, match):
    """Refused before a device is asked for."""
    from fused_turboquant import v1 as V1
    with pytest.raises(ValueError, match=match):
        V1.v1_tree_attention(**{**_args(), **change})


def test_tree_runs_on_devices_only():
    from fused_turboquant import _lib, v1 as V1
    with pytest.raises(_lib.FusedTQError, match="ROCm"):
        V1.v1_tree_attention(**_args())
    with pytest.raises(ValueError, match="head_dim"):
        V1.v1_tree_attention(**{**_args(), "query": torch.zeros(4, 4, 96)})


def test_tree_split_counts():
    from fused_turboquant import v1 as V1
    assert V1.default_tree_splits(0, 0, 32, 8, 128, 4, 4, 100) == 1
    for args in ((1, 8, 32, 8, 128, 4, 4, 131072), (64, 8, 32, 8, 128, 3, 3, 100), (1, 1, 8, 8, 64, 16, 16, 1 << 30)):
        assert 1 <= V1.default_tree_splits(*args) <= 64
