"""The KV manager with a budget (kv_budget): what it keeps, and that it attends to exactly that."""
import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PS, L, HQ, HKV, D = 16, 2, 4, 2, 128
G = HQ // HKV


def manager(**kw):
    from kinetics_amd.batch_cache import PagedBatchKVManager

    cfg = SimpleNamespace(num_attention_heads=HQ, num_key_value_heads=HKV, head_dim=D, hidden_size=HQ * D, num_hidden_layers=L)
    args = dict(kv_budget=64, kv_budget_sink=4, kv_budget_local=16, kv_budget_slack=5)
    args.update(kw)
    return PagedBatchKVManager(cfg, max_batch_size=5, max_seq_len=PS * 16, device=DEV, dtype=torch.bfloat16, **args)


def cached(m, layer, slot):
    """(keys, values, scores) that the slot holds, [Hkv, tokens, ...] in 64 bits."""
    n = int(m.kv_offset[layer][slot])
    pages = m.pool.slot_table[slot, : (n + PS - 1) // PS].long()
    flat = m.kv_cache[layer][pages].transpose(0, 1).reshape(2, -1, HKV, D)[:, :n].double()
    return flat[0].transpose(0, 1), flat[1].transpose(0, 1), m.scores[layer][slot, :, :n].double()


def attend(q, k, v, causal_from=None):
    """q [Hq, s, D] over k, v [Hkv, t, D]; rows see causal_from + row + 1 tokens (None: all)."""
    s, t = q.shape[1], k.shape[1]
    x = torch.matmul(q.double().reshape(HKV, G * s, D), k.transpose(1, 2).contiguous()).view(HKV, G, s, t) / math.sqrt(D)
    if causal_from is not None:
        x = x.masked_fill(torch.arange(t, device=DEV)[None, :] > causal_from + torch.arange(s, device=DEV)[:, None], -math.inf)
    w = torch.softmax(x, -1)
    return torch.matmul(w.view(HKV, G * s, t), v).view(HQ, s, D).transpose(0, 1).reshape(s, HQ * D), w.sum((1, 2))


def fresh(*shape):
    return torch.randn(*shape, device=DEV).to(torch.bfloat16)


def test_prefill_and_decode_within_a_budget():
    torch.manual_seed(0)
    m = manager()
    fed = {}
    lens = {}

    def remember(layer, slot, k):                    # k [Hkv, s, D]
        old = fed.get((layer, slot))
        fed[layer, slot] = k if old is None else torch.cat([old, k], 1)

    def check_kept(layer, slot):
        """Each head holds an ascending subset of what was fed: the first 4, the newest 16, one row each."""
        k = cached(m, layer, slot)[0]
        all_k = fed[layer, slot].double()
        for h in range(HKV):
            where = [int((all_k[h] == row).all(1).nonzero()[0, 0]) for row in k[h]]
            assert where == sorted(set(where)), "order"
            assert where[:4] == [0, 1, 2, 3] and where[-16:] == list(range(all_k.shape[1] - 16, all_k.shape[1]))

    def prefill(slot, n):
        for layer in range(L):
            q, k, v = fresh(1, HQ, n, D), fresh(1, HKV, n, D), fresh(1, HKV, n, D)
            offset = int(m.kv_offset[layer][slot])
            kc, vc, sc = cached(m, layer, slot)
            out = m.compute_attention(q, k, v, layer, torch.tensor([slot], device=DEV))
            remember(layer, slot, k[0])
            want, w = attend(q[0], torch.cat([kc, k[0].double()], 1), torch.cat([vc, v[0].double()], 1), offset)
            assert torch.allclose(out[0].double(), want, rtol=2e-2, atol=2e-2)
            w[:, :offset] += sc
            got = cached(m, layer, slot)[2]
            if offset + n > 64:
                assert int(m.kv_offset[layer][slot]) == 64
                check_kept(layer, slot)
                # the heaviest of the middle stayed, with their weights, and nothing is left behind them
                mid = w[:, 4:offset + n - 16]
                top = torch.sort(mid, 1, descending=True).values[:, :64 - 20]
                kept = torch.sort(got[:, 4:48], 1, descending=True).values
                assert torch.allclose(kept, top, rtol=1e-4, atol=1e-6)
                assert bool((m.scores[layer][slot, :, 64:] == 0).all())
            else:
                assert int(m.kv_offset[layer][slot]) == offset + n
                assert torch.allclose(got, w, rtol=1e-4, atol=1e-6)
        lens[slot] = int(m.kv_offset[0][slot])

    prefill(3, 40)
    prefill(3, 100)          # behind 40: cut to 64
    prefill(1, 64)           # exactly the budget
    prefill(4, 200)
    prefill(3, 30)           # a chunk behind a slot that was cut
    for step in range(1, 13):
        active = torch.tensor([4, 1, 3], device=DEV) if step < 9 else torch.tensor([3, 4], device=DEV)
        for layer in range(L):
            n = active.numel()
            q, k, v = fresh(n, HQ, 1, D), fresh(n, HKV, 1, D), fresh(n, HKV, 1, D)
            before = [cached(m, layer, int(s)) for s in active]
            out = m.compute_attention(q, k, v, layer, active)
            for i, s in enumerate(active.tolist()):
                remember(layer, s, k[i])
                kc, vc, sc = before[i]
                want, w = attend(q[i], torch.cat([kc, k[i].double()], 1), torch.cat([vc, v[i].double()], 1))
                assert torch.allclose(out[i].double(), want, rtol=2e-2, atol=2e-2), (step, layer, s)
                expect = kc.shape[1] + 1
                if step % 5 == 0:
                    expect = min(expect, 64)
                    check_kept(layer, s) if expect == 64 else None
                else:
                    w[:, :-1] += sc
                    assert torch.allclose(cached(m, layer, s)[2], w, rtol=1e-4, atol=1e-6)
                assert int(m.kv_offset[layer][s]) == expect
    m.clear_cache(3)
    assert all(bool((m.scores[layer][3] == 0).all()) for layer in range(L))
    fed.pop((0, 3)), fed.pop((1, 3))
    prefill(3, 70)
    m.pool.raise_on_overflow()


def test_a_sequence_without_pages_keeps_its_count():
    """An exhausted pool makes a sequence inert for the step; the eviction of that step must not forget it."""
    from kinetics_amd import _lib

    torch.manual_seed(1)
    m = manager(kv_budget=32, kv_budget_local=8, kv_budget_slack=1, kv_pool_pages=4)
    one = torch.tensor([0], device=DEV)
    m.compute_attention(fresh(1, HQ, 32, D), fresh(1, HKV, 32, D), fresh(1, HKV, 32, D), 0, one)
    two = torch.tensor([1], device=DEV)
    m.compute_attention(fresh(1, HQ, 32, D), fresh(1, HKV, 32, D), fresh(1, HKV, 32, D), 0, two)   # the pool is used up
    both = torch.tensor([0, 1], device=DEV)
    out = m.compute_attention(fresh(2, HQ, 1, D), fresh(2, HKV, 1, D), fresh(2, HKV, 1, D), 0, both)   # both want a third page
    assert int(torch.count_nonzero(out)) == 0
    assert m.kv_offset[0][:2].tolist() == [33, 33]
    with pytest.raises(_lib.KineticsError):
        m.pool.raise_on_overflow()


def test_refusals():
    for bad in (dict(kv_budget=20), dict(kv_budget_sink=-1), dict(kv_budget_slack=0)):
        with pytest.raises(ValueError):
            manager(**bad)
    for policy in (dict(attn_block_topk=2, attn_local=4), dict(attn_topk=8, attn_local=4), dict(attn_local=4),
                   dict(attn_block_topk=2, attn_local=4, attn_stride=8)):
        with pytest.raises(NotImplementedError):
            manager(**policy)
