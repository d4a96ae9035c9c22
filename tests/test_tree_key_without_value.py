"""Keys and values come together: a call with one of them is refused, as the
rows of neither could be written."""

from __future__ import annotations

import pytest
import torch

from micro_vllm_amd.attention.operators.mi355x_tree import MI355XTreeAttentionOperator, hip_tree_attention
from test_tree_refusals import metadata


@pytest.mark.parametrize("call", [hip_tree_attention, MI355XTreeAttentionOperator()], ids=["function", "operator"])
@pytest.mark.parametrize("missing", ["key", "value"])
def test_one_without_the_other(call, missing):
    token = torch.zeros((1, 1, 16), dtype=torch.bfloat16)
    cache = torch.zeros((2, 1, 16, 1, 16), dtype=torch.bfloat16)
    key, value = (None, token) if missing == "key" else (token, None)
    with pytest.raises(ValueError, match="key and value"):
        call(token, key, value, cache, metadata())
