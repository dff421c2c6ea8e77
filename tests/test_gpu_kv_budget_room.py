"""The KV manager with a budget in slots that have just enough room."""
from types import SimpleNamespace

import pytest
import torch

from tests import test_gpu_kv_budget_turns as T

DEV = "cuda"


def test_a_slot_without_room_for_budget_and_slack_is_refused():
    from kinetics_amd.batch_cache import PagedBatchKVManager

    cfg = SimpleNamespace(num_attention_heads=4, num_key_value_heads=2, head_dim=128, hidden_size=512, num_hidden_layers=1)
    for tokens, budget, slack in ((256, 256, 1), (256, 250, 7), (250, 200, 57), (4096, 4096, 64)):
        with pytest.raises(ValueError, match="kv_budget_slack"):
            PagedBatchKVManager(cfg, max_batch_size=2, max_seq_len=tokens, device="cpu", dtype=torch.bfloat16, kv_budget=budget,
                                kv_budget_slack=slack)


@pytest.mark.gpu
def test_budget_and_slack_that_fill_the_slot():
    """The pages hold exactly budget + slack tokens: no step ever lacks room."""
    torch.manual_seed(4)
    m = T.manager(slack=16, max_seq_len=T.N + 16)
    assert m.pages_per_slot * T.PS == T.N + 16
    T.prefill(m, 0, 64)
    T.prefill(m, 2, 80)
    idx = torch.tensor([2, 0], device=DEV)
    for _ in range(50):
        for layer in range(T.L):
            T.step(m, layer, [2, 0], idx)
    m.pool.raise_on_overflow()
