"""GPU tests of the 4-bit cache at the edges of what its calls allow."""
import pytest
import torch

from test_gpu_kv4 import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [16, 17, 63, 64, 500])
@pytest.mark.parametrize("max_tokens", [0, 1, 64])
def test_a_call_without_sequences(tokens, max_tokens):
    """Nothing is written, whatever number of query rows there is."""
    from oxicuda_b200 import ops
    c = Case([5], [0], 2, 64, 64, 16)
    q = torch.ones(tokens, 8, 64, dtype=torch.bfloat16, device="cuda")
    home, lse = torch.full_like(q, 2.0), torch.full((tokens, 8), 2.0, device="cuda")
    nobody = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.kv4_attention_workspace_bytes(c.cache, c.table[:0], c.lens[:0], nobody, tokens, 8, max_tokens) == 0
    ops.kv4_attention(q, c.cache, c.table[:0], c.lens[:0], nobody, max_tokens=max_tokens, out=home, lse=lse)
    assert (home == 2).all() and (lse == 2).all()
