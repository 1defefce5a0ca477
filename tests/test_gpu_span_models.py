"""Models with capped scores, a distance bias and packed documents on the GPU: a training step against the same model on the CPU in 64 bits, the
serving engine with and without captured decode steps."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("kind,kw", [("gpt", dict(alibi=True)), ("gpt", dict(attn_cap=4.0)), ("llama", dict(attn_cap=4.0)), ("llama", dict(alibi=True, attn_cap=4.0))])
def test_a_packed_training_step(kind, kw):
    """Loss and gradients of bfloat16 on the GPU against 64 bits on the CPU with the same weights.  A value in bfloat16 is off by 2^-9 on
    average; a gradient passes some twenty roundings in two layers, which add up like a random walk: 2^-9 sqrt(20) = 0.9 %, and three times that bounds it."""
    from rumus_b200.models import GPT, GPTConfig, Llama, LlamaConfig
    from rumus_b200.ops import functional as F, native
    torch.manual_seed(0)
    if kind == "gpt":
        make = lambda **m: GPT(GPTConfig(vocab_size=96, seq_len=200, d_model=256, num_heads=4, num_layers=2, ffn_dim=512, **kw), **m)      # noqa: E731
    else:
        make = lambda **m: Llama(LlamaConfig(vocab_size=96, seq_len=200, d_model=256, num_heads=2, num_kv_heads=1, num_layers=2, ffn_dim=512, **kw), **m)   # noqa: E731
    ref = make().double()
    ref.init_weights(0.06)
    for p in ref.parameters():
        p.data = p.data.bfloat16().double()
    model = make(device="cuda", dtype=torch.bfloat16)
    model.load_state_dict({k: v.bfloat16() for k, v in ref.state_dict().items()})
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, 96, (2, 201), generator=g)
    docs = torch.tensor([[0] * 64 + [1] * 130 + [-1] * 6, [0] * 1 + [1] * 100 + [2] * 99])
    prefix = torch.zeros(2, 200, dtype=torch.bool)
    prefix[0, 64:90] = True
    want = ref(tok[:, :-1], tok[:, 1:], spans=F.document_spans(docs, prefix))
    want.backward()
    got = model(tok[:, :-1].cuda(), tok[:, 1:].cuda(), spans=F.document_spans(docs.cuda(), prefix.cuda()))
    got.backward()
    assert native.read_status() == 0
    assert abs(got.item() - want.item()) < 0.02 * want.item()
    grads = dict(ref.named_parameters())
    for n, p in model.named_parameters():
        assert torch.isfinite(p.grad).all() and _rel(p.grad, grads[n].grad) < 0.027, (n, _rel(p.grad, grads[n].grad))


def _engine(graphs, kw, head_major=False):
    from rumus_b200.models.llama import LlamaConfig
    from rumus_b200.serve import Engine, ServeConfig
    mc = LlamaConfig(vocab_size=512, seq_len=1024, d_model=512, num_heads=8, num_kv_heads=2, num_layers=2, ffn_dim=512, **kw)
    cfg = ServeConfig(model=mc, num_blocks=256, block_size=16, max_batch=8, token_budget=256, cuda_graphs=graphs, kv_head_major=head_major)
    return Engine(cfg, torch.device("cuda"), seed=3)


@pytest.mark.parametrize("kw", [dict(attn_cap=2.0), dict(alibi=True), dict(attn_cap=2.0, alibi=True)])
@pytest.mark.parametrize("head_major", [False, True])
def test_engine_in_portions_as_in_one(kw, head_major):
    """Logits of a prompt's last place: fed whole, in portions, and token by token through captured decode steps, are one function."""
    from rumus_b200.ops import native
    g = torch.Generator().manual_seed(0)
    prompt = torch.randint(0, 512, (300,), generator=g).tolist()
    whole = _engine(False, kw).feed([(1, prompt, [299])])
    parts = _engine(True, kw, head_major)
    parts.feed([(1, prompt[:130], [])])
    parts.feed([(1, prompt[130:290], []), (2, prompt[:1], [])])
    for t in range(290, 300):
        last = parts.feed([(1, prompt[t:t + 1], [0])])
    assert parts.graph_replays == 10 and native.read_status() == 0
    # heads of 64, weights and results rounded to bfloat16 on both ways: 2^-9 per rounding, some sixteen of them in two layers
    assert _rel(last, whole) < 3 * 2 ** -9 * 4


def test_engine_serves_requests():
    e = _engine(True, dict(attn_cap=2.0, alibi=True))
    r = random.Random(0)
    want = {}
    for i in range(6):
        want[i + 1] = r.randint(4, 12)
        e.add_request(i + 1, [r.randrange(512) for _ in range(r.randint(1, 500))], want[i + 1])
    outs = {}
    while e.has_work():
        for rid in e.step():
            outs[rid] = e.requests.pop(rid).output
    from rumus_b200.ops import native
    assert {k: len(v) for k, v in outs.items()} == want and e.sched.free_blocks() == 256 and native.read_status() == 0


def test_fsdp_step_of_a_packed_model():
    """A step through FSDP (one rank) moves the weights as Adam on the plain model does."""
    from rumus_b200.models import GPT, GPTConfig
    from rumus_b200.ops import functional as F, native
    from rumus_b200.parallel import FSDP
    torch.manual_seed(0)
    model = GPT(GPTConfig(vocab_size=96, seq_len=128, d_model=256, num_heads=2, num_layers=2, ffn_dim=512, attn_cap=5.0, alibi=True), device="cuda",
                dtype=torch.bfloat16)
    eng = FSDP(model, lr=1e-3)
    tok = torch.randint(0, 96, (2, 129), device="cuda")
    spans = F.document_spans((torch.arange(128, device="cuda") // 40).expand(2, 128))
    before = {k: v.clone() for k, v in model.state_dict().items()}
    for _ in range(2):
        eng.zero_grad()
        loss = model(tok[:, :-1], tok[:, 1:], spans=spans)
        loss.backward()
        eng.step()
    after = model.state_dict()
    assert torch.isfinite(loss) and all(torch.isfinite(v.float()).all() for v in after.values()) and native.read_status() == 0
    assert all(not torch.equal(before[k], after[k]) for k in before if k.endswith("proj.weight"))


def test_forward_is_captured_first_and_replayed():
    """Nothing of a biased layer is made in its first call: that one can be a captured one."""
    from rumus_b200 import nn
    from rumus_b200.ops import functional as F
    m = nn.MultiheadAttention(128, 2, device="cuda", dtype=torch.bfloat16, attn_cap=5.0, alibi=True)
    other = nn.MultiheadAttention(128, 2, device="cuda", dtype=torch.bfloat16, attn_cap=5.0, alibi=True)
    x = torch.randn(2, 100, 128, device="cuda").bfloat16()
    spans = F.document_spans(torch.zeros(2, 100, dtype=torch.int64, device="cuda"))
    with torch.no_grad():
        other(x, spans=spans)                       # libraries and kernels are loaded
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x, spans=spans)
        for _ in range(2):
            x.copy_(torch.randn(2, 100, 128, device="cuda").bfloat16())
            graph.replay()
            assert torch.equal(y, m(x, spans=spans))
