"""Tree attention of many and uneven sequences, whose parts the device cuts, of
lengths that change under a captured graph, and of 16-bit outputs beside fields
that are not finite; step tables at the end of the int32 range."""
import numpy as np
import pytest
import torch

from test_tree_gpu import HALF, RAW, Case, _rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,kb,vb", [(64, 4, 4), (128, 2, 3), (64, RAW, RAW), (64, 8, 8)])
@pytest.mark.parametrize("splits", [None, 1, 2, 7, 64])
def test_many_and_uneven_sequences(cuda, d, kb, vb, splits):
    """More sequences than a wave has lanes, some without tokens, one much longer than the rest."""
    r = np.random.RandomState(d + kb)
    B = 150
    counts = r.randint(0, 4, B)
    counts[[0, 63, 64, 149]] = [1, 0, 3, 2]
    ctx = r.randint(0, 100, B)
    ctx[100], counts[100] = 2500, 3
    c = Case(cuda, d, kb, vb, 1, 2, ctx.tolist(), counts.tolist(), seed=20)
    mask = c.trees()
    lse = torch.empty(c.T, 2, device=cuda)
    want, wlse, _ = c.want(mask)
    got = c.run(mask, num_splits=splits, lse=lse)
    assert _rel(got, want) < 1e-5 and np.abs(lse.cpu().numpy() - wlse).max() < 1e-4
    for dtype in (torch.bfloat16, torch.float16):
        q = c.q.to(dtype)
        want, _, share = c.want(mask, q=q)
        got = c.run(mask, q=q, num_splits=splits, max_query_len=3, max_seq_len=2503)
        assert _rel(got.float(), want) < HALF[dtype] + share


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_starts_behind_one_another(cuda, dtype):
    """Starts that fall from token to token: a sequence's parts begin at its first token's."""
    c = Case(cuda, 128, 4, 4, 1, 2, [900, 40], [40, 3], seed=21)  # 80 columns: two blocks of 64
    start = torch.tensor([20 * (39 - i) for i in range(40)] + [39, 0, 50], dtype=torch.int32, device=cuda)
    q = c.q.to(dtype)
    want, _, share = c.want(None, start, q=q)
    for splits in (1, 3, 16):
        err = _rel(c.run(q=q, kv_start=start, num_splits=splits).float(), want)
        assert err < (1e-5 if dtype == torch.float32 else HALF[dtype] + share), splits


@pytest.mark.parametrize("splits", [1, 6])
def test_captured_lengths_that_change(cuda, splits):
    from fused_turboquant import v1 as V1
    c = Case(cuda, 128, 4, 4, 2, 4, [1500, 900, 60], [12, 12, 12], seed=22)
    q, out = c.q.to(torch.bfloat16), torch.empty(36, 8, 128, dtype=torch.bfloat16, device=cuda)
    ws = torch.empty(V1.workspace_bytes(36, 8, 128, splits), dtype=torch.uint8, device=cuda)
    call = lambda o: c.run(q=q, out=o, workspace=ws, num_splits=splits, max_query_len=12)
    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for lens, counts in (([1512, 912, 72], [12, 12, 12]), ([300, 900, 2], [5, 12, 2]), ([0, 912, 40], [0, 7, 12]),
                         ([1512, 1, 0], [12, 1, 0])):
        c.lens, c.counts, c.ctx = lens, counts, [n - k for n, k in zip(lens, counts)]
        c.sl.copy_(torch.tensor(lens, dtype=torch.int32))
        c.qsl.copy_(torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32))
        eager = torch.full_like(out, 7.0)
        call(eager)
        torch.cuda.synchronize()
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        n = sum(counts)
        assert (out[n:] == 7.0).all()  # rows behind the last sequence
        want, _, share = c.want(q=q)
        assert _rel(out[:n].float(), want[:n]) < HALF[torch.bfloat16] + share


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,kb,vb,lloyd", [(64, 4, 4, False), (128, 3, 3, False), (256, 4, 3, False), (128, 8, 8, False),
                                           (128, 1, 2, False), (128, 4, 4, True)])
def test_fields_of_hidden_positions(cuda, d, kb, vb, lloyd, dtype):
    c = Case(cuda, d, kb, vb, 1, 4, [40], [12], vrot=lloyd, lloyd=lloyd, seed=23)
    start = torch.full((12,), 9, dtype=torch.int32, device=cuda)
    mask = c.words([1 << i | 1 for i in range(12)], 1)
    q = c.q.to(dtype)
    want = c.run(mask, q=q, kv_start=start)
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=torch.float16, device=cuda).view(torch.uint8)
    nk = d * kb // 8
    v0 = nk + 2 + d * vb // 8
    for pos in (0, 5, 8, 45, 52, 60):
        if pos >= c.bt.shape[1] * 16:
            continue
        s = c.cache[c.bt[0, pos // 16].long(), pos % 16, 0]
        s[nk:nk + 2] = bad[:2]
        s[v0:v0 + 4] = bad[2:6]
    got = c.run(mask, q=q, kv_start=start)
    keep = [i for i in range(12) if i != 5]  # position 45 is node 5
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[5]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_raw_values_that_are_not_finite(cuda, d, dtype):
    c = Case(cuda, d, RAW, RAW, 1, 2, [40], [12], seed=24)
    mask = c.words([1 << i | 1 for i in range(12)], 1)
    q = c.q.to(dtype)
    want = c.run(mask, q=q)
    v = c.cache[c.bt[0, 2].long(), 13, 0].view(torch.float16)  # position 45, node 5
    v[d + 5], v[2 * d - 1] = float("inf"), float("nan")
    got = c.run(mask, q=q)
    keep = [i for i in range(12) if i != 5]
    assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[5][:, [5, d - 1]]).any()


@pytest.mark.parametrize("listed", [False, True])
def test_step_tables_at_the_end_of_int32(cuda, listed):
    """Lengths past 2^31 - 1 count as that; no position past the table has a slot."""
    from fused_turboquant import steps
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    past = [2 ** 31 - 5, 3, 2 ** 31 - 1]
    bt = i32([[4, 5, 6, 7], [1, 2, -1, -1], [8, 9, 10, 11]])
    kw = dict(num_blocks=i32([4, 1, 4]), free_blocks=i32([20, 21, 22]), free_count=i32([1])) if listed else {}
    got = steps.step_tables(i32([0, 10, 12, 13]), i32(past), bt, 16, 14, **kw)
    assert got.seq_lens.tolist() == [2 ** 31 - 1, 5, 2 ** 31 - 1]
    assert got.slot_mapping.tolist() == [-1] * 10 + [19, 20, -1, -1]
    assert got.positions.tolist() == [past[0] + i for i in range(10)] + [3, 4, past[2], 0]
    lacked = 2 * (2 ** 27 - 4) if listed else 0
    assert got.missing.tolist() == [lacked]
    if listed:
        assert kw["num_blocks"].tolist() == [4, 1, 4] and kw["free_count"].tolist() == [1]


@pytest.mark.parametrize("q_type,out_type", [(torch.float32, torch.bfloat16), (torch.float32, torch.float16),
                                             (torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                             (torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("d,kb,vb,kind", [(64, 4, 4, "rht"), (128, 3, 2, "rht"), (256, 2, 4, "rht"), (128, 8, 8, "rht"),
                                          (128, RAW, RAW, "rht"), (64, 3, 3, "planar"), (256, 4, 4, "iso_full")])
def test_query_and_output_types(cuda, d, kb, vb, kind, q_type, out_type):
    c = Case(cuda, d, kb, vb, 1, 4, [70, 300], [20, 3], vrot=kb != RAW, kind=kind, seed=25)
    q, mask = c.q.to(q_type), c.trees()
    want, _, share = c.want(mask, q=q)
    for splits in (1, 4):
        out = torch.empty(c.T, 4, d, dtype=out_type, device=cuda)
        assert c.run(mask, q=q, out=out, num_splits=splits) is out
        assert _rel(out.float(), want) < (1e-5 if out_type == torch.float32 else HALF[out_type] + share)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,kb,vb", [(64, 4, 4), (128, 2, 2), (256, 3, 4), (64, RAW, RAW), (128, 8, 8)])
def test_queries_beyond_f16(cuda, d, kb, vb, dtype):
    """Rows that f16 cannot hold are scaled for the products; the others stay what they were."""
    c = Case(cuda, d, kb, vb, 1, 4, [50], [20], seed=26)
    q = c.q.to(dtype)
    want = c.run(q=q)
    odd = q.clone()
    for row, head in ((0, 0), (3, 1), (19, 3)):  # a column of several waves
        odd[row, head] *= 1e6
    got = c.run(q=odd)
    assert torch.isfinite(got).all()
    for row, head in ((0, 0), (3, 1), (19, 3)):
        got[row, head] = want[row, head]
    assert _rel(got.float(), want.double().cpu().numpy()) < 1e-6
