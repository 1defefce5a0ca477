"""Sharded training on packed documents: two ranks against one plain model with Adam, the same spans."""
import pytest
import torch

from dist_utils import run_ranks

STEPS, WORLD = 3, 2


def _model():
    from rumus_b200.models import GPT, GPTConfig
    torch.manual_seed(0)
    return GPT(GPTConfig(vocab_size=64, seq_len=16, d_model=32, num_heads=2, num_layers=3, ffn_dim=64, attn_cap=3.0, alibi=True))


def _data():
    """Tokens and the documents that they are packed in, others in every row."""
    g = torch.Generator().manual_seed(5)
    tok = torch.randint(0, 64, (STEPS, WORLD * 2, 17), generator=g)
    docs = (torch.rand(STEPS, WORLD * 2, 16, generator=g) < 0.25).long().cumsum(-1)
    return tok, docs


def _worker(rank, world, reshard):
    from rumus_b200.ops import functional as F
    from rumus_b200.parallel import FSDP
    model = _model()
    eng = FSDP(model, lr=1e-2, reshard_after_forward=reshard)
    tok, docs = _data()
    mine, losses = slice(rank * 2, rank * 2 + 2), []
    for t, d in zip(tok[:, mine], docs[:, mine]):
        eng.zero_grad()
        loss = model(t[:, :-1], t[:, 1:], spans=F.document_spans(d))
        loss.backward()
        eng.step()
        losses.append(loss.item())
    with eng.summon_full_params():
        return losses, {k: v.clone() for k, v in model.state_dict().items()}


@pytest.mark.parametrize("reshard", [False, True])
def test_two_ranks_step_as_one_model_does(reshard):
    from rumus_b200.ops import functional as F
    from rumus_b200.optim import Adam
    out = run_ranks(_worker, WORLD, reshard)
    ref = _model()
    opt = Adam(ref.parameters(), lr=1e-2)
    apart = []
    for step, (t, d) in enumerate(zip(*_data())):
        opt.zero_grad()
        loss = ref(t[:, :-1], t[:, 1:], spans=F.document_spans(d))
        loss.backward()
        # losses of 4 from sums of some hundred fp32 numbers; weights that differ by less than 2e-5
        assert abs(sum(o[0][step] for o in out) / WORLD - loss.item()) < 1e-4
        with torch.no_grad():
            apart.append(abs(ref(t[:, :-1], t[:, 1:]).item() - loss.item()))
        opt.step()
    assert min(apart) > 1e-3                             # a wrapper that dropped the spans would be seen
    for k, v in ref.state_dict().items():
        assert torch.equal(out[0][1][k], out[1][1][k]), k
        if not k.endswith("k_proj.bias"):                # exact gradient is zero (softmax ignores a key bias): Adam amplifies rounding noise
            assert torch.allclose(out[0][1][k], v, atol=2e-5), k
