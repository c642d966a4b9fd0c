"""The paged 4-bit KV cache on the GPU at the edges of what its entry points take."""
import pytest
import torch

import kv4_util as U
import spindle_b200 as sg
from test_kv4_gpu import TYPES, case, check, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_tok,heads,group", [(1, 1, 1), (1, 2, 7), (3, 2, 2), (2000, 4, 8)])
def test_attention_without_requests(dev, dtype, n_tok, heads, group):
    # tokens that belong to no request, and no request at all
    cache = sg.Kv4Cache(2, heads, 64, 16, device=dev)
    q = torch.randn(n_tok, heads * group, 64, device=dev).to(dtype)
    lse = torch.zeros(n_tok, heads * group, device=dev)
    for width in (0, 3):
        out = sg.kv4_attention(cache, q, ints([0], dev), ints([], dev), torch.empty(0, width, dtype=torch.int32, device=dev), lse=lse)
        assert (out == 0).all() and torch.isneginf(lse).all()
    sg.device_status()
