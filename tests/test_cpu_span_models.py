"""Models with capped scores, a distance bias and packed documents: training on the CPU, the serving engine, tensor parallel ranks."""
import random

import pytest
import torch

from dist_utils import run_ranks
from rumus_b200.models import GPT, GPTConfig, Llama, LlamaConfig
from rumus_b200.ops import functional as F


def _gpt(**kw):
    torch.manual_seed(3)
    m = GPT(GPTConfig(vocab_size=50, seq_len=24, d_model=32, num_heads=4, num_layers=2, ffn_dim=64, **kw)).double()
    m.init_weights(0.3)
    return m


def _llama(**kw):
    torch.manual_seed(3)
    m = Llama(LlamaConfig(vocab_size=50, seq_len=24, d_model=32, num_heads=4, num_kv_heads=2, num_layers=2, ffn_dim=64, **kw)).double()
    m.init_weights(0.3)
    return m


@pytest.mark.parametrize("make,kw", [(_gpt, dict(alibi=True, attn_cap=2.0)), (_llama, dict(attn_cap=2.0)), (_llama, dict(alibi=True))])
def test_packed_documents_are_what_they_are_alone(make, kw):
    """Without absolute positions a document in a pack has the logits that it has alone, and so have its gradients."""
    model = make(**kw)
    g = torch.Generator().manual_seed(1)
    parts = [torch.randint(0, 50, (1, n), generator=g) for n in (7, 1, 12)]
    docs = torch.tensor([[0] * 7 + [1] + [2] * 12 + [-1] * 4])
    idx = torch.cat(parts + [torch.zeros(1, 4, dtype=torch.long)], 1)
    packed = model(idx, spans=F.document_spans(docs))
    alone = [model(p) for p in parts]
    if make is _gpt:
        for a, lo in zip(alone, (0, 7, 8)):
            assert torch.allclose(packed[:, lo:lo + a.shape[1]], a, atol=1e-10)
    else:                       # rotations are relative: the angles of far positions round differently
        for a, lo in zip(alone, (0, 7, 8)):
            assert torch.allclose(packed[:, lo:lo + a.shape[1]], a, atol=1e-5)
    gp = torch.autograd.grad(packed[:, :20].square().sum(), list(model.parameters()), allow_unused=True)
    ga = torch.autograd.grad(sum(a.square().sum() for a in alone), list(model.parameters()), allow_unused=True)
    for p, a in zip(gp, ga):
        assert (p is None) == (a is None) and (p is None or torch.allclose(p, a, rtol=1e-4, atol=1e-4))


def test_without_options_models_are_as_they_were():
    plain, capped = _gpt(), _gpt(attn_cap=1e9)
    idx = torch.randint(0, 50, (2, 24), generator=torch.Generator().manual_seed(0))
    assert torch.allclose(plain(idx), capped(idx), atol=1e-8)
    assert torch.allclose(plain(idx), plain(idx, spans=F.document_spans(torch.zeros(2, 24, dtype=torch.long))), atol=1e-10)
    assert set(plain.state_dict()) == set(capped.state_dict())
    assert set(plain.state_dict()) - set(_gpt(alibi=True).state_dict()) == {"pos_emb.weight"}
    n = sum(p.numel() for p in _gpt(alibi=True).parameters())
    assert n == _gpt(alibi=True).cfg.num_params()


def test_model_gradients_against_differences():
    model = _gpt(alibi=True, attn_cap=1.5)
    idx = torch.randint(0, 50, (1, 9), generator=torch.Generator().manual_seed(0))
    spans = F.document_spans(torch.tensor([[0, 0, 0, 1, 1, 1, 1, -1, -1]]), torch.tensor([[1, 1, 0, 1, 0, 0, 0, 0, 0]], dtype=torch.bool))
    w = model.blocks[0].attn.qkv_weight

    def loss():
        return model(idx, spans=spans)[:, :7].square().sum()

    (g,) = torch.autograd.grad(loss(), w)
    d = torch.randn(w.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    h = 1e-6
    with torch.no_grad():
        w += h * d
        up = loss()
        w -= 2 * h * d
        down = loss()
        w += h * d
    want = (up - down) / (2 * h)
    assert abs((g * d).sum() - want) < 1e-6 * abs(want)


def test_masks_and_spans_do_not_mix():
    m = _gpt().blocks[0].attn
    x = torch.randn(1, 4, 32, dtype=torch.float64)
    with pytest.raises(ValueError):
        m(x, torch.zeros(4, 4, dtype=torch.float64), spans=torch.zeros(4, 2, dtype=torch.int32))


@pytest.mark.parametrize("kw", [dict(attn_cap=1.0), dict(alibi=True), dict(attn_cap=1.0, alibi=True)])
@pytest.mark.parametrize("head_major", [False, True])
def test_engine_batches_as_it_runs_alone(kw, head_major):
    """Prompts in chunks beside decoded tokens give what each request gives alone (whole prompts, other layout)."""
    from rumus_b200.serve import Engine, ServeConfig
    r = random.Random(0)
    reqs = {i + 1: ([r.randrange(256) for _ in range(r.randint(5, 150))], r.randint(3, 8)) for i in range(4)}

    def engine(**more):
        mc = LlamaConfig(vocab_size=256, seq_len=256, d_model=128, num_heads=4, num_kv_heads=2, num_layers=2, ffn_dim=256, **kw)
        return Engine(ServeConfig(model=mc, num_blocks=64, block_size=16, max_batch=4, dtype=torch.float32, scale_dtype=torch.float32, **more))

    def drain(e):
        outs = {}
        while e.has_work():
            for rid in e.step():
                outs[rid] = e.requests.pop(rid).output
        return outs

    e = engine(token_budget=64, kv_head_major=head_major)
    for rid, (p, n) in reqs.items():
        assert e.add_request(rid, p, n)
    together = drain(e)
    alone = engine(token_budget=4096)
    for rid, (p, n) in reqs.items():
        alone.add_request(rid, p, n)
        assert drain(alone)[rid] == together[rid]


def _tp_worker(rank, world, kw):
    from rumus_b200.models.llama_parallel import ParallelLlamaStage
    from rumus_b200.parallel.topology import build_topology
    from rumus_b200.parallel.tp import TPContext
    topo = build_topology(tp=2, pp=1)
    cfg = LlamaConfig(vocab_size=64, seq_len=8, d_model=32, num_heads=4, num_kv_heads=2, num_layers=2, ffn_dim=64, **kw)
    torch.manual_seed(11)
    dense = Llama(cfg)
    stage = ParallelLlamaStage(cfg, TPContext(group=topo.tp_group, mode="nccl"), 0, 1)
    stage.load_dense(dense.state_dict())
    x = torch.randn(16, 32, generator=torch.Generator().manual_seed(12))
    rows = slice(rank * 8, rank * 8 + 8)                 # a block's stream is sharded by tokens
    got = stage.blocks[0](x[rows], 2, 8)
    want = dense.blocks[0](x.view(2, 8, 32)).view(16, 32)[rows]
    assert torch.allclose(got, want, atol=1e-5)
    return True


@pytest.mark.parametrize("kw", [dict(attn_cap=0.5, alibi=True)])
def test_tensor_parallel_heads_keep_their_slopes(kw):
    assert all(run_ranks(_tp_worker, 2, kw))
