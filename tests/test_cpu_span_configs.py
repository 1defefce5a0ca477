"""Configurations that the span attention kernels or its formula do not take are refused where they are built or called, with a reason."""
import math

import pytest
import torch

from rumus_b200.models import GPT, GPTConfig, Llama, LlamaConfig
from rumus_b200.models.llama_parallel import ParallelLlamaBlock
from rumus_b200.nn import MultiheadAttention, TransformerBlock
from rumus_b200.ops import span
from rumus_b200.serve import ServeConfig
from rumus_b200.serve.llama import Int4LlamaShard


def _config(heads=4, dtype=torch.bfloat16, **kw):
    mc = LlamaConfig(vocab_size=64, seq_len=64, d_model=256, num_heads=heads, num_kv_heads=heads, num_layers=1, ffn_dim=128, **kw)
    return ServeConfig(model=mc, num_blocks=8, block_size=16, max_batch=2, token_budget=32, dtype=dtype)


# 32 bits, heads of 256 and of 4
@pytest.mark.parametrize("heads,dtype", [(4, torch.float32), (1, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("kw", [dict(attn_cap=5.0), dict(alibi=True)])
def test_a_served_model_is_refused_when_it_is_built(heads, dtype, kw):
    with pytest.raises(TypeError, match="multiple of 8"):
        Int4LlamaShard(_config(heads, dtype, **kw), torch.device("cuda"))


def test_on_the_cpu_it_is_served():
    assert Int4LlamaShard(_config(64, torch.float32, attn_cap=5.0), torch.device("cpu")).shaped


@pytest.mark.parametrize("D,dtypes", [(64, (torch.float32,) * 3), (60, (torch.bfloat16,) * 3), (136, (torch.float16,) * 3),
                                      (64, (torch.bfloat16, torch.float16, torch.bfloat16))])
def test_the_forward_launch_checks_types_and_sizes(D, dtypes):
    q, k, v = (torch.zeros(1, 4, 2, D, dtype=t) for t in dtypes)
    with pytest.raises(TypeError, match="multiple of 8"):
        span.span_forward(q, k, v, None, True, 1.0, 0.0, None)


# "no cap" is zero: what is below it, or no number, would have meant it too
@pytest.mark.parametrize("cap", [-30.0, math.nan, math.inf, 1e300, 1e-46])
def test_models_refuse_caps_that_are_none(cap):
    from types import SimpleNamespace
    gpt = dict(vocab_size=50, seq_len=24, d_model=32, num_heads=4, num_layers=1, ffn_dim=64, attn_cap=cap)
    llama = LlamaConfig(num_kv_heads=4, **gpt)
    for make in (lambda: MultiheadAttention(32, 4, attn_cap=cap), lambda: TransformerBlock(32, 4, attn_cap=cap), lambda: GPT(GPTConfig(**gpt)), lambda: Llama(llama),
                 lambda: ParallelLlamaBlock(llama, SimpleNamespace(world=1, rank=0)),
                 lambda: Int4LlamaShard(_config(dtype=torch.float32, attn_cap=cap), torch.device("cpu"))):
        with pytest.raises(ValueError, match="cap"):
            make()
