"""What span attention's launchers refuse before they look for a GPU."""
import pytest
import torch

from rumus_b200.ops import native


# addresses as they are asked for, and one of them off: 20 comes before anything is launched
@pytest.mark.parametrize("name,off", [("q", 2), ("k", 8), ("v", 8), ("out", 4), ("part_o", 8)])
def test_decoding_refuses_addresses_that_its_loads_and_stores_do_not_take(name, off):
    at = dict(q=1 << 20, k=2 << 20, v=3 << 20, out=4 << 20, part_o=5 << 20)
    at[name] += off
    rc = native.lib().rb_span_decode(native.dtype_code(torch.bfloat16), 0, at["q"], 128, 64, at["k"], at["v"], 6 << 20, 7 << 20, None, None, at["out"],
                                     at["part_o"], 8 << 20, 1, 2, 1, 64, 64, 4, 4, 9, 1.0, 0.0, None)
    assert rc == 20


def test_decoding_refuses_results_at_an_odd_address():
    from rumus_b200.ops.span import span_decode
    q, pages = torch.randn(1, 2, 8).bfloat16(), torch.randn(2, 4, 2, 8).bfloat16()
    flat = torch.zeros(64, dtype=torch.bfloat16)
    first = next(i for i in range(4) if flat[i:].data_ptr() % 8)
    tables, ctx = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([8], dtype=torch.int32)
    with pytest.raises(ValueError, match="8-byte"):
        span_decode(q, pages, pages, tables, ctx, 8, out=flat[first:first + 16].view(1, 2, 8))
