"""An FSDP step of a packed model on the GPU (one rank) against a plain model with the same weights, tokens and spans."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_losses_and_first_step():
    from rumus_b200.models import GPT, GPTConfig
    from rumus_b200.ops import functional as F, native
    from rumus_b200.parallel import FSDP

    def make():
        torch.manual_seed(0)
        return GPT(GPTConfig(vocab_size=96, seq_len=128, d_model=256, num_heads=2, num_layers=2, ffn_dim=512, attn_cap=5.0, alibi=True), device="cuda",
                   dtype=torch.bfloat16)

    plain, model = make(), make()
    eng = FSDP(model, lr=1e-3)
    tok = torch.randint(0, 96, (2, 129), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    spans = F.document_spans((torch.arange(128, device="cuda") // 40).expand(2, 128))
    want = plain(tok[:, :-1], tok[:, 1:], spans=spans)
    want.backward()
    eng.zero_grad()
    got = model(tok[:, :-1], tok[:, 1:], spans=spans)
    got.backward()
    eng.step()
    # the same kernels on the same numbers
    assert torch.equal(got.detach(), want.detach())
    with torch.no_grad():
        assert abs(plain(tok[:, :-1], tok[:, 1:]).item() - want.item()) > 1e-3        # spans matter
    grads = {n: p.grad.double() for n, p in plain.named_parameters()}
    weights = {n: p.detach().double() for n, p in plain.named_parameters()}          # it has not stepped
    after = dict(model.named_parameters())
    checked = 0
    for n, g in grads.items():
        if not n.startswith("blocks.") or g.dim() != 2:
            continue
        # Adam's first step: m / sqrt(v) with both corrected is g / |g|, 1e-8 beside it; gradients of the same kernels on the same numbers are the same.  A
        # weight in bfloat16 is off by half a step, 2^-8 of itself, the 32-bit arithmetic of the step by less than 2e-3 of lr (its powers of the betas).
        old, step = weights[n], 1e-3 * g / (g.abs() + 1e-8)
        off = (after[n].detach().double() - (old - step)).abs()
        assert (off <= 2.0 ** -8 * (old - step).abs() + 2e-6).all(), (n, off.max().item())
        checked += 1
    assert checked >= 2 * 4 and native.read_status() == 0
