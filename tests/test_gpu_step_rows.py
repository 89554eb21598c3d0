"""A step of no rows through its operators, and one beside it with rows (needs an MI355X)."""

import pytest
import torch

from mlx_tree_spec_amd import attention_inputs, next_tokens
from test_gpu_step import D, DEV, DIM, HEADS, KV, Model, batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(0,), (2, 0)])
def test_no_rows(lead):
    model = Model()
    x = torch.empty(*lead, DIM, dtype=torch.bfloat16, device=DEV)
    none = torch.empty(lead, dtype=torch.int32, device=DEV)
    q, k, v, gate = attention_inputs(x, model.attn[0], none, none)
    assert q.shape == gate.shape == (*lead, HEADS, D) and k.shape == v.shape == (*lead, KV, D)
    tokens, logprobs = next_tokens(x, model.head, torch.empty(lead, device=DEV), temperature=0.7)
    assert tokens.shape == logprobs.shape == lead and tokens.dtype == torch.int64


def test_leading_shape():
    model = Model()
    x, positions, adapters, *_ = batch(12, 3)
    want = attention_inputs(x, model.attn[0], positions, adapters)
    got = attention_inputs(x.reshape(3, 4, DIM), model.attn[0], positions.reshape(3, 4), adapters.reshape(3, 4))
    for a, b in zip(got, want):
        assert a.shape[:2] == (3, 4) and torch.equal(a.reshape(b.shape), b)
