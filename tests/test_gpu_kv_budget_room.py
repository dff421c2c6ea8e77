"""The KV manager with a budget in slots that have just enough room, and under another default dtype."""
import math
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


def grown(m, slot, tokens):
    """The slot with `tokens` tokens, more than the budget, by decoding."""
    T.prefill(m, slot, T.N)
    idx = torch.tensor([slot], device=DEV)
    for _ in range(tokens - T.N):
        for layer in range(T.L):
            m.compute_attention(T.fresh(1, T.HQ, 1, T.D), T.fresh(1, T.HKV, 1, T.D), T.fresh(1, T.HKV, 1, T.D), layer, idx)
    assert all(int(m.kv_offset[layer][slot]) == tokens for layer in range(T.L))


def cut(k, v, sc):
    """What a sequence keeps of its keys and values, head by head."""
    n = k.shape[1]
    rows = []
    for h in range(T.HKV):
        mid = T.SINK + torch.sort(sc[h, T.SINK:n - T.LOCAL], descending=True, stable=True).indices[:T.N - T.SINK - T.LOCAL]
        rows.append(torch.cat([torch.arange(T.SINK, device=DEV), mid.sort().values, torch.arange(n - T.LOCAL, n, device=DEV)]))
    return tuple(torch.stack([x[h, r] for h, r in enumerate(rows)]) for x in (k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [64, 49, 48, 10])
def test_a_chunk_behind_a_slot_in_its_slack(chunk):
    """A slot needs pages for the budget plus the longest chunk: one that is in its slack is cut before the chunk where
    it would not fit otherwise, and attends to all it has where it does."""
    torch.manual_seed(5)
    m = T.manager(slack=17, max_seq_len=T.N + 64)
    grown(m, 1, 80)
    for layer in range(T.L):
        q, k, v = T.fresh(1, T.HQ, chunk, T.D), T.fresh(1, T.HKV, chunk, T.D), T.fresh(1, T.HKV, chunk, T.D)
        kc, vc, sc = T.cached(m, layer, 1)
        if 80 + chunk > T.N + 64:
            kc, vc = cut(kc, vc, sc)
        out = m.compute_attention(q, k, v, layer, torch.tensor([1], device=DEV))
        want, _, tol = T.attend(q[0], torch.cat([kc, k[0].double()], 1), torch.cat([vc, v[0].double()], 1))
        assert bool(((out[0].double() - want).abs() <= tol).all()), layer
        assert int(m.kv_offset[layer][1]) == T.N
    m.pool.raise_on_overflow()


@pytest.mark.gpu
def test_a_chunk_that_cannot_fit_changes_nothing():
    from kinetics_amd import _lib

    torch.manual_seed(6)
    m = T.manager(slack=17, max_seq_len=T.N + 64, max_batch=2)
    grown(m, 1, 80)
    one = torch.tensor([1], device=DEV)

    def unchanged(n):
        before = [T.cached(m, layer, 1) for layer in range(T.L)]
        with pytest.raises((ValueError, _lib.KineticsError)):
            m.compute_attention(T.fresh(1, T.HQ, n, T.D), T.fresh(1, T.HKV, n, T.D), T.fresh(1, T.HKV, n, T.D), 0, one)
        for layer in range(T.L):
            assert all(torch.equal(a, b) for a, b in zip(before[layer], T.cached(m, layer, 1)))

    unchanged(65)                                    # more than the slot holds even after a cut
    m = T.manager(slack=17, max_seq_len=T.N + 64, max_batch=2, kv_pool_pages=8)
    grown(m, 1, 80)
    T.prefill(m, 0, 40)                              # 5 + 3 pages: the pool is used up
    unchanged(60)                                    # would be cut to 64 first, but there are no pages for 124 tokens


@pytest.mark.gpu
def test_prefill_under_another_default_dtype():
    """Model loaders set the default dtype; the log-sum-exp is fp32 whatever it is."""
    torch.manual_seed(7)
    m = T.manager(slack=8)
    q, k, v = T.fresh(1, T.HQ, 100, T.D), T.fresh(1, T.HKV, 100, T.D), T.fresh(1, T.HKV, 100, T.D)
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        out = m.compute_attention(q, k, v, 0, torch.tensor([0], device=DEV))
    finally:
        torch.set_default_dtype(old)
    want, _, tol = T.attend(q[0], k[0].double(), v[0].double())
    assert bool(((out[0].double() - want).abs() <= tol).all()) and math.isfinite(float(m.scores[0].sum()))
