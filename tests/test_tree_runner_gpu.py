"""Trees of drafted tokens through the attention backend and the model runner:
one step stores the nodes, attends by the tree's mask, walks the accepted paths
and moves their slots, and the tokens are those of plain greedy decoding."""
import math
from types import SimpleNamespace

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the package on sys.path)

TREES = {"chain": [-1, 0, 1, 2], "tree": [-1, 0, 0, 1, 1, 2, 3, 6], "root": [-1]}


def _env(monkeypatch, boundary="0", **kw):
    for k, v in dict(TURBOQUANT_BOUNDARY_PROTECT=boundary, TURBOQUANT_V_ROTATE="1", TURBOQUANT_V_LLOYD_MAX="0",
                     TURBOQUANT_KIND="rht", TURBOQUANT_DEFER_PREFILL="0", **kw).items():
        monkeypatch.setenv(k, v)


@pytest.mark.parametrize("n", [1, 5, 63, 64, 65, 130])
def test_tree_shape(n):
    from fused_turboquant.steps import tree_shape
    g = torch.Generator().manual_seed(n)
    parents = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, n)]
    depths, mask = tree_shape(parents)
    assert depths.dtype == torch.int32 and mask.dtype == torch.int64 and tuple(mask.shape) == (n, (n + 63) // 64)
    for i in range(n):
        path, p = set(), i
        while p >= 0:
            path.add(p)
            p = parents[p]
        assert int(depths[i]) == len(path) - 1
        assert {j for j in range(64 * mask.shape[1]) if (int(mask[i, j // 64]) >> (j % 64)) & 1} == path


@pytest.mark.parametrize("parents", [[], [0], [-1, -1], [-1, 1], [-1, 2, 0]])
def test_tree_shape_refuses(parents):
    from fused_turboquant.steps import tree_shape
    with pytest.raises(ValueError):
        tree_shape(parents)


def _md(dev, n, context, window_positions, words=1, **kw):
    qsl = torch.tensor([0, n], dtype=torch.int32, device=dev)
    md = dict(num_actual_tokens=n, is_prefill=False, num_decodes=1, num_decode_tokens=n,
              seq_lens=torch.tensor([context + n], dtype=torch.int32, device=dev),
              block_table=torch.arange(8, dtype=torch.int32, device=dev)[None], query_start_loc=qsl, max_query_len=n,
              max_seq_len=128, slot_mapping=torch.arange(context, context + n, device=dev),
              tree_mask=torch.ones(n, words, dtype=torch.int64, device=dev), token_positions=window_positions)
    md.update(kw)
    return SimpleNamespace(**md)


def test_impl_refusals(monkeypatch):
    from fused_turboquant.vllm_plugin.v1_backend import FusedTurboQuantV1Backend as Backend, FusedTurboQuantV1Impl as Impl
    _env(monkeypatch)
    q, kv = torch.zeros(6, 4 * 64), torch.zeros(6, 2 * 64)
    cache = torch.zeros(Backend.get_kv_cache_shape(8, 16, 2, 64, "turboquant_4bit_nc"), dtype=torch.uint8)
    make = lambda **kw: Impl(4, 64, 0.125, 2, kv_cache_dtype="turboquant_4bit_nc", **kw)
    call = lambda impl, md: impl.forward(SimpleNamespace(), q, kv, kv, cache, md, output=torch.zeros_like(q))
    with pytest.raises(ValueError, match="token_positions"):
        call(make(sliding_window=32), _md("cpu", 6, 10, None))
    with pytest.raises(NotImplementedError, match="window"):
        call(make(sliding_window=5), _md("cpu", 6, 10, torch.arange(10, 16)))
    with pytest.raises(NotImplementedError, match="decode-only"):
        call(make(), _md("cpu", 6, 10, None, is_prefill=True))
    monkeypatch.setenv("TURBOQUANT_DEFER_PREFILL", "1")
    with pytest.raises(NotImplementedError, match="DEFER"):
        call(make(), _md("cpu", 6, 10, None))


def test_runner_refusals():
    from fused_turboquant.vllm_plugin.runner import LlamaDecoder, LlamaSpec, ModelRunner
    spec = LlamaSpec(num_layers=1, hidden=64, num_heads=2, num_kv_heads=1, head_dim=64, ffn=64, vocab=31, max_positions=64)
    model = LlamaDecoder(spec, "cpu", dtype=torch.float32)
    first, bt = torch.zeros(1, dtype=torch.int64), torch.arange(2, dtype=torch.int32)[None]
    run = ModelRunner(model, max_batch=1, max_context=32, backend="dense")
    with pytest.raises(NotImplementedError):
        run.start_tree(bt, first, [4], 8, [-1, 0], use_graph=False)
    run = ModelRunner(model, max_batch=1, max_context=32, kv_cache_dtype="turboquant_4bit_nc")
    with pytest.raises(ValueError, match="context"):
        run.start_tree(bt, first, [4], 27, [-1, 0], use_graph=False)  # 33 positions
    with pytest.raises(ValueError, match="parents"):
        run.start_tree(bt, first, [4], 8, [-1, 1], use_graph=False)
    run.start_tree(bt, first, [4], 26, [-1, 0], use_graph=False)
    with pytest.raises(ValueError, match="drafted"):
        run.tree_step(torch.zeros(1, 2, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["turboquant_3bit_nc", "auto"])
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("flat", [False, True])
def test_impl_tree(cuda, monkeypatch, kind, window, flat):
    """The backend's tree step is v1_tree_attention of the layer's slots: a
    code layer and a raw boundary layer, with and without a window, into an
    output of the query's type and (``flat`` False) another's."""
    from fused_turboquant import v1 as V1
    from fused_turboquant.steps import tree_shape
    from fused_turboquant.vllm_plugin.v1_backend import FusedTurboQuantV1Backend as Backend, FusedTurboQuantV1Impl as Impl
    _env(monkeypatch, boundary="fp16")
    hq, hkv, d, n, ctx = 8, 2, 128, 8, 77
    impl = Impl(hq, d, d ** -0.5, hkv, kv_cache_dtype=kind, sliding_window=window)
    cache = torch.zeros(Backend.get_kv_cache_shape(8, 16, hkv, d, kind), dtype=torch.uint8, device=cuda)
    if kind == "auto" and cache.shape[-1] < 4 * d:
        cache = torch.zeros(*cache.shape[:3], 4 * d, dtype=torch.uint8, device=cuda)
    g = torch.Generator().manual_seed(3)
    layer = SimpleNamespace()
    k, v = (torch.randn(ctx + n, hkv * d, generator=g).to(cuda, torch.bfloat16) for _ in range(2))
    impl.do_kv_cache_update(layer, k, v, cache, torch.arange(ctx + n, device=cuda))
    q = torch.randn(n, hq * d, generator=g).to(cuda, torch.bfloat16)
    depths, mask = tree_shape(TREES["tree"])
    depths, mask = depths.to(cuda), mask.to(cuda)
    md = _md(cuda, n, ctx, ctx + depths.long(), tree_mask=mask)
    out = torch.empty(n, hq * d, dtype=torch.bfloat16 if flat else torch.float32, device=cuda)
    impl.forward(layer, q, k[-n:], v[-n:], cache, md, output=out)
    start = None if window is None else (ctx + depths - window + 1).clamp(min=0).to(torch.int32)
    raw = kind == "auto"
    cent = None if raw else layer._fused_tq_state.centroids
    bits = (V1.RAW_BITS, V1.RAW_BITS) if raw else (impl.key_bits, impl.value_bits)
    want = V1.v1_tree_attention(q.view(n, hq, d), cache, md.block_table, md.seq_lens, md.query_start_loc, cent, *bits,
                                tree_mask=mask, scale=d ** -0.5, v_rotate=not raw, kv_start=start, max_query_len=n,
                                max_seq_len=128)
    torch.cuda.synchronize()
    assert torch.equal(out, want.view(n, hq * d).to(out.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", list(TREES))
def test_tree_decoding_is_greedy_decoding(cuda, monkeypatch, shape):
    """Three requests of different lengths, drafts of which some are the model's
    own next tokens: eager tree decoding and the captured step give the same
    tokens, those of plain decoding.

    Both runs multiply in fp32 or in fp16 parts with fp32-level products (64-wide
    heads): the logits, of unit variance, differ by some 1e-4, or 1e-2 where a
    stored code falls on the other side of its threshold.  A request is compared
    up to the first step whose two best plain logits are closer than 2e-2."""
    from fused_turboquant.vllm_plugin.runner import LlamaDecoder, LlamaSpec, ModelRunner
    _env(monkeypatch)
    new, parents = 24, TREES[shape]
    spec = LlamaSpec(num_layers=2, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, ffn=512, vocab=257,
                     max_positions=128)
    model = LlamaDecoder(spec, cuda, dtype=torch.float32, seed=1)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 257, (m,), generator=g).to(cuda) for m in (21, 9, 30)]
    run = ModelRunner(model, max_batch=3, max_context=80, kv_cache_dtype="turboquant_4bit_nc")
    run.keep_logits = True
    plain = run.generate(prompts, new, use_graph=False)
    gaps = [(lambda t: (t[:, 0] - t[:, 1]))(x.topk(2, dim=-1).values) for x in run.logits]
    gaps = torch.stack(gaps, dim=1).cpu()  # [3, new]: the prefill's, then the steps'
    assert tuple(gaps.shape) == (3, new)
    run.keep_logits = False
    depth = [0]
    for p in parents[1:]:
        depth.append(depth[p] + 1)
    steps = []

    def draft(tokens, lens):
        steps.append(lens.tolist())
        r = torch.Generator().manual_seed(len(steps))
        out = torch.randint(0, 257, (3, len(parents) - 1), generator=r)
        for b, m in enumerate(lens.tolist()):
            for i in range(1, len(parents)):
                right = m + depth[i] - 1
                if right < new and float(torch.rand(1, generator=r)) < 0.6:
                    out[b, i - 1] = int(plain[b, right])
        return out.to(cuda)

    got = {}
    for graph in (False, True):
        run.reset()
        steps.clear()
        got[graph] = run.generate_tree(prompts, new, parents, draft, use_graph=graph)
        torch.cuda.synchronize()
        if shape == "root":
            assert len(steps) == new - 1
        else:
            assert len(steps) < new - 1  # paths of more than their root
        print(f"[tree decoding {shape}] graph {graph}: {len(steps)} steps for {new - 1} tokens", flush=True)
    assert torch.equal(got[False], got[True])
    compared = 0
    for b in range(3):
        close = (gaps[b] < 2e-2).nonzero()
        upto = int(close[0]) if close.numel() else new
        assert torch.equal(got[True][b, :upto], plain[b, :upto]), b
        compared += upto
    assert compared >= 12
    assert math.isfinite(float(gaps.min()))
