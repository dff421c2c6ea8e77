"""The KV manager with a budget, decoding different sets of slots in different ways: no sequence ever holds more than the
budget and the slack, in any layer."""
import math
import random
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PS, L, HQ, HKV, D = 16, 2, 4, 2, 128
G = HQ // HKV
N, SINK, LOCAL = 64, 4, 16


def manager(slack, max_batch=5, max_seq_len=PS * 16, **kw):
    from kinetics_amd.batch_cache import PagedBatchKVManager

    cfg = SimpleNamespace(num_attention_heads=HQ, num_key_value_heads=HKV, head_dim=D, hidden_size=HQ * D, num_hidden_layers=L)
    return PagedBatchKVManager(cfg, max_batch_size=max_batch, max_seq_len=max_seq_len, device=DEV, dtype=torch.bfloat16, kv_budget=N,
                               kv_budget_sink=SINK, kv_budget_local=LOCAL, kv_budget_slack=slack, **kw)


def cached(m, layer, slot):
    """(keys, values, scores) that the slot holds, [Hkv, tokens, ...] in 64 bits."""
    n = int(m.kv_offset[layer][slot])
    pages = m.pool.slot_table[slot, : (n + PS - 1) // PS].long()
    flat = m.kv_cache[layer][pages].transpose(0, 1).reshape(2, -1, HKV, D)[:, :n].double()
    return flat[0].transpose(0, 1), flat[1].transpose(0, 1), m.scores[layer][slot, :, :n].double()


def attend(q, k, v):
    """(out [s, Hq * D], weights received [Hkv, t], bound) of q [Hq, s, D] over k, v [Hkv, t, D], the rows the newest."""
    s, t = q.shape[1], k.shape[1]
    x = torch.matmul(q.double().reshape(HKV, G * s, D), k.transpose(1, 2).contiguous()).view(HKV, G, s, t) / math.sqrt(D)
    x = x.masked_fill(torch.arange(t, device=DEV)[None, :] > t - s + torch.arange(s, device=DEV)[:, None], -math.inf)
    w = torch.softmax(x, -1)
    flat = lambda y: y.view(HQ, s, D).transpose(0, 1).reshape(s, HQ * D)  # noqa: E731
    out, mag = (flat(torch.matmul(w.view(HKV, G * s, t), y)) for y in (v, v.abs()))
    # result and, with more than 32 rows, weights rounded once to bf16; scores: 132 roundings of sums of at most 128 * 25 / sqrt(128)
    return out, w.sum((1, 2)), 2.0 ** -8 * 1.01 * (out.abs() + (mag if G * s > 32 else 0)) + 2 * 132 * 2.0 ** -24 * 283 * mag


def fresh(*shape):
    return torch.randn(*shape, device=DEV).to(torch.bfloat16)


def step(m, layer, slots, batch_idx):
    """One decoded token for each of the slots; checks output, scores and what is kept.  A sequence of N + slack is cut to N."""
    n, slack = len(slots), m.budget_slack
    q, k, v = fresh(n, HQ, 1, D), fresh(n, HKV, 1, D), fresh(n, HKV, 1, D)
    before = [cached(m, layer, s) for s in slots]
    out = m.compute_attention(q, k, v, layer, batch_idx)
    for i, s in enumerate(slots):
        kc, vc, sc = before[i]
        keys = torch.cat([kc, k[i].double()], 1)
        want, w, tol = attend(q[i], keys, torch.cat([vc, v[i].double()], 1))
        assert bool(((out[i].double() - want).abs() <= tol).all()), (layer, s, kc.shape[1])
        w[:, :-1] += sc
        got_k, _, got_s = cached(m, layer, s)
        length = keys.shape[1]
        if length < N + slack:
            assert int(m.kv_offset[layer][s]) == length, (layer, s, length)
            assert torch.allclose(got_s, w, rtol=1e-4, atol=1e-6)
            continue
        assert int(m.kv_offset[layer][s]) == N, (layer, s, length)
        for h in range(HKV):
            where = [int((keys[h] == row).all(1).nonzero()[0, 0]) for row in got_k[h]]
            assert where == sorted(set(where)) and where[:SINK] == list(range(SINK))
            assert where[-LOCAL:] == list(range(length - LOCAL, length))
            top = torch.sort(w[h, SINK:length - LOCAL], descending=True).values[:N - SINK - LOCAL]
            assert torch.allclose(torch.sort(got_s[h, SINK:N - LOCAL], descending=True).values, top, rtol=1e-4, atol=1e-6)
        assert bool((m.scores[layer][s, :, N:] == 0).all())


def prefill(m, slot, n):
    for layer in range(L):
        m.compute_attention(fresh(1, HQ, n, D), fresh(1, HKV, n, D), fresh(1, HKV, n, D), layer, torch.tensor([slot], device=DEV))


def test_two_batches_in_turn():
    """Micro-batches decoded alternately, with an even slack: each has its steps on odd or on even counts only."""
    torch.manual_seed(0)
    m = manager(slack=8)
    for slot, n in ((0, 64), (1, 70), (2, 40), (3, 61)):
        prefill(m, slot, n)
    sets = [[0, 2], [3, 1]]
    idx = [torch.tensor(s, device=DEV) for s in sets]
    for i in range(2 * 30):
        for layer in range(L):
            step(m, layer, sets[i % 2], idx[i % 2])
    m.pool.raise_on_overflow()


@pytest.mark.parametrize("slack", [1, 2, 6])
def test_a_new_batch_idx_object_for_every_layer(slack):
    torch.manual_seed(1)
    m = manager(slack)
    prefill(m, 4, 63)
    prefill(m, 1, 66)
    for i in range(3 * slack + 4):
        for layer in range(L):
            step(m, layer, [4, 1], torch.tensor([4, 1], device=DEV))


def test_random_subsets_of_the_slots():
    torch.manual_seed(2)
    rng = random.Random(2)
    m = manager(slack=4)
    for slot in range(5):
        prefill(m, slot, rng.randint(50, 90))
    for i in range(60):
        slots = rng.sample(range(5), rng.randint(1, 5))
        idx = torch.tensor(slots, device=DEV)
        for layer in range(L):
            step(m, layer, slots, idx)
    m.pool.raise_on_overflow()


def test_a_captured_step_replays_over_several_slacks():
    """One decode step recorded as a HIP graph cuts the sequences that need it in every replay, as eager steps do."""
    slots = [3, 0, 4]
    managers = [manager(slack=5) for _ in range(2)]
    for m in managers:
        torch.manual_seed(3)
        for slot, n in zip(slots, (64, 30, 90)):
            prefill(m, slot, n)
    g, e = managers
    idx = torch.tensor(slots, device=DEV)
    qs, ks, vs = ([fresh(3, h, 1, D) for _ in range(L)] for h in (HQ, HKV, HKV))

    def run(m):
        return [m.compute_attention(qs[layer], ks[layer], vs[layer], layer, idx) for layer in range(L)]

    run(g), run(e)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            outs = run(g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for i in range(50):
        for t in qs + ks + vs:
            t.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = run(e)
        torch.cuda.synchronize()
        for layer in range(L):
            assert int(g.kv_offset[layer].max()) < N + 5, (i, layer)
            assert torch.equal(got[layer], want[layer]), (i, layer)
            assert torch.equal(g.kv_offset[layer], e.kv_offset[layer]) and torch.equal(g.scores[layer], e.scores[layer])
    for m in managers:
        m.pool.raise_on_overflow()
