"""A dense Llama trains on the GPU (its rotation works in place on the projection's output)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gradients_against_the_cpu():
    from rumus_b200.models import Llama, LlamaConfig
    from rumus_b200.ops import native
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=96, seq_len=64, d_model=256, num_heads=2, num_kv_heads=2, num_layers=2, ffn_dim=256)
    ref = Llama(cfg)
    ref.init_weights(0.06)
    for p in ref.parameters():
        p.data = p.data.bfloat16().float()
    model = Llama(cfg, device="cuda", dtype=torch.bfloat16)
    model.load_state_dict({k: v.bfloat16() for k, v in ref.state_dict().items()})
    tok = torch.randint(0, 96, (2, 65), generator=torch.Generator().manual_seed(1))
    ref(tok[:, :-1], tok[:, 1:]).backward()
    model(tok[:, :-1].cuda(), tok[:, 1:].cuda()).backward()
    assert native.read_status() == 0
    grads = dict(ref.named_parameters())
    for n, p in model.named_parameters():
        want = grads[n].grad.double()
        # some twenty roundings to bfloat16 in two layers, 2^-9 each on average: 0.9 % as a random walk, and three times that
        assert ((p.grad.double().cpu() - want).norm() / want.norm()).item() < 0.027, n
