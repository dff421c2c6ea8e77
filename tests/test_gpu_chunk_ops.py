"""Attention of a chunk of new tokens, the weight it gave to the cached tokens, eviction by that weight and the q/k norm +
split with rotary positions, through the public entry points against plain float64 forms (tests/chunk_reference.py,
where the error bounds are derived)."""
import math

import pytest
import torch

from tests import chunk_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from kinetics_amd import ops as _ops

    return _ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def attend(ops, pb, num_splits=0, **mods):
    lse = torch.full(pb.q.shape[:2], 7.0, device=DEV)
    out = torch.full_like(pb.q, 5.0)
    got = ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, out=out, lse=lse,
                                    first_page_offset=pb.offset, num_splits=num_splits, **mods)
    assert got is out
    return out, lse


def check_attention(pb, out, lse, **mods):
    want, wlse, tol, ltol = R.attention(pb, **mods)
    rows = slice(pb.ends[0], pb.ends[-1])
    err = (out.double() - want)[rows].abs()
    assert bool((err <= tol[rows]).all()), f"out: worst error / bound {float((err / tol[rows]).max())}"
    w, z = wlse[rows], lse.double()[rows]
    assert torch.equal(w == -math.inf, z == -math.inf)
    fin = w > -math.inf
    lerr = (w[fin] - z[fin]).abs()
    assert bool((lerr <= ltol[rows][fin]).all()), f"lse: worst error {float(lerr.max()) if lerr.numel() else 0}"
    assert bool((out[pb.ends[-1]:] == 5.0).all()) and bool((lse[pb.ends[-1]:] == 7.0).all())  # rows of no sequence


SHAPES = [
    # lens, news, hq, hkv, d, page, dtype, offset
    ([1], [1], 1, 1, 128, 16, "bf16", 0),
    ([1, 2, 17], [1, 2, 17], 4, 1, 64, 16, "f16", 0),
    ([300, 64, 65, 1, 512], [1, 1, 1, 1, 1], 4, 1, 128, 16, "bf16", 0),
    ([300, 64, 65, 1, 512], [1, 1, 1, 1, 1], 16, 1, 64, 32, "bf16", 12),
    ([0, 130, 0, 77], [0, 3, 0, 0], 6, 2, 128, 64, "f16", 0),
    ([257], [257], 4, 1, 128, 16, "bf16", 0),
    ([400, 33, 129], [200, 33, 1], 8, 2, 128, 32, "bf16", 0),
    ([400, 33, 129], [200, 33, 1], 5, 1, 64, 128, "f16", 5),
    ([1000, 999], [40, 5], 12, 4, 128, 128, "f16", 100),
    ([700], [129], 3, 3, 64, 64, "bf16", 63),
    ([260] * 70, [1] * 69 + [9], 4, 2, 64, 16, "bf16", 3),
]
MODS = [
    dict(),
    dict(window=1),
    dict(window=50, prefix_lens=True),
    dict(softcap=5.0),
    dict(slopes=True, prefix_lens=True),
    dict(softcap=30.0, window=130, slopes=True, sm_scale=0.2),
]


def with_tensors(pb, mods):
    mods = dict(mods)
    if mods.get("slopes"):
        mods["slopes"] = 2.0 ** (-8.0 * torch.arange(1, pb.hq + 1, device=DEV, dtype=torch.float32) / pb.hq)
    if mods.get("prefix_lens"):
        mods["prefix_lens"] = i32([(31 * (i + 1)) % (n + 20) for i, n in enumerate(pb.lens)])   # some longer than the sequence
    return mods


@pytest.mark.parametrize("mods", MODS, ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_chunk_attention(ops, case, mods):
    lens, news, hq, hkv, d, page, dtype, offset = SHAPES[case]
    pb = R.problem(case, lens, news, hq, hkv, d, page, dtype, offset, tail_rows=2)
    mods = with_tensors(pb, mods)
    out, lse = attend(ops, pb, **mods)
    check_attention(pb, out, lse, **mods)


@pytest.mark.parametrize("splits", [1, 2, 3, 16])
@pytest.mark.parametrize("window", [0, 90])
def test_chunk_attention_in_spans(ops, splits, window):
    """Any number of spans of the keys, more of them than tiles too, gives the same answer within the bounds."""
    pb = R.problem(31, [900, 40, 0, 333], [1, 40, 0, 100], 8, 2, 128, 16, "bf16", 4, tail_rows=3)
    out, lse = attend(ops, pb, num_splits=splits, window=window)
    check_attention(pb, out, lse, window=window)
    again, lse2 = attend(ops, pb, num_splits=splits, window=window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("mods", [dict(), dict(window=700), dict(softcap=20.0, prefix_lens=True)], ids=["plain", "window", "cap-prefix"])
def test_chunk_attention_decode_and_prompts_in_one_call(ops, mods):
    """Long single-token rows are cut into more spans than the prompt's rows, which may have one."""
    pb = R.problem(32, [5000, 3001, 900, 17, 4097], [1, 2, 100, 1, 8], 4, 1, 128, 16, "bf16", tail_rows=1)
    mods = with_tensors(pb, mods)
    assert ops.chunk_workspace_bytes(pb.q.shape[0], 5, 4, 1, pb.max_pages) > 0
    out, lse = attend(ops, pb, **mods)
    check_attention(pb, out, lse, **mods)
    again, lse2 = attend(ops, pb, **mods)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("hq,hkv", [(24, 1), (64, 1), (66, 2), (128, 1)])
def test_large_groups(ops, hq, hkv):
    """More query heads per KV head than the decode kernels take: rows are (token, head) pairs."""
    pb = R.problem(33, [150, 40], [7, 40], hq, hkv, 64, 16, "bf16", 3)
    mods = with_tensors(pb, dict(slopes=True, window=60))
    out, lse = attend(ops, pb, **mods)
    check_attention(pb, out, lse, **mods)
    sc = torch.zeros(2, hkv, 160, device=DEV)
    want, tol = R.mass(pb, lse, sc, **mods)
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=3, **mods)
    assert bool(((sc.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("cap", [0.5, 3.0, 1000.0])
def test_caps_below_and_above_the_scores(ops, cap):
    """Every form of the tanh: scores far below the cap, near it and far above it, within one block too."""
    pb = R.problem(34, [300, 257], [64, 1], 4, 1, 128, 16, "bf16")
    pb.q[::3] *= 0.02
    pb.q[1::7] *= 8
    out, lse = attend(ops, pb, softcap=cap)
    check_attention(pb, out, lse, softcap=cap)
    sc = torch.zeros(2, 1, 300, device=DEV)
    want, tol = R.mass(pb, lse, sc, softcap=cap)
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, softcap=cap)
    assert bool(((sc.double() - want).abs() <= tol).all())


def test_chunk_attention_more_rows_than_tokens(ops):
    """Rows in front of a sequence see nothing: zeros and -inf; a prefix does not change that."""
    pb = R.problem(5, [3, 0, 40], [9, 4, 41], 4, 1, 128, 16, "bf16")
    for mods in (dict(), dict(prefix_lens=i32([2, 5, 7]))):
        out, lse = attend(ops, pb, **mods)
        check_attention(pb, out, lse, **mods)
        assert bool((out[:6] == 0).all()) and bool((lse[:6] == -math.inf).all())
        assert bool((out[9:13] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("news", [[1, 3], [150, 70]])
def test_chunk_attention_never_touches_what_is_not_seen(ops, news, dtype):
    """NaN and infinities in unlisted pages, behind the last token, in padding slots and in tokens outside the window or
    behind a row change nothing."""
    pb = R.problem(6, [333, 258], news, 8, 2, 128, 32, dtype, 9)
    want, wl = attend(ops, pb, window=40)
    clean = pb.kv.clone()
    listed = torch.zeros(pb.total_pages, dtype=torch.bool, device=DEV)
    listed[pb.ids.long()] = True
    poison = torch.tensor([math.nan, math.inf, -math.inf, math.nan], device=DEV, dtype=pb.dt)
    pb.kv[~listed] = math.nan
    for b, n in enumerate(pb.lens):
        first = pb.ids[pb.starts[b]].long()
        pb.kv[first, :, :pb.offset] = math.nan
        end = n + pb.offset - (pb.counts[b] - 1) * pb.page
        pb.kv[pb.ids[pb.starts[b + 1] - 1].long(), :, end:] = math.inf
        unseen = torch.arange(0, n - pb.news[b] - 39, device=DEV)       # older than the oldest row's window
        page, slot = R.slot_of(pb, b, unseen)
        pb.kv[page, :, slot] = poison[unseen % 4][:, None, None, None]
    got, gl = attend(ops, pb, window=40)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    # one new token's value is infinite: rows in front of it are as they were, its own and the later ones show it
    pb.kv = clean
    b, t = 1, pb.lens[1] - 1
    page, slot = R.slot_of(pb, b, torch.tensor([t - 1, t], device=DEV))
    pb.kv[page[1], 1, slot[1], 0, 5] = math.inf
    got, _ = attend(ops, pb)
    ref, _, tol, _ = R.attention(pb)
    last = pb.ends[2] - 1
    assert bool((got[last, :4, 5] == math.inf).all())
    err = (got.double() - ref).abs() <= tol
    err[last, :4, 5] = True
    assert bool(err.all())
    pb.kv[page[0], 1, slot[0], 0, 5] = -math.inf
    pb.kv[page[0], 1, slot[0], 0, 99] = math.nan
    got, _ = attend(ops, pb)
    assert bool(got[last, :4, 5].isnan().all()) and bool(got[last - 1:last + 1, :4, 99].isnan().all())
    if pb.news[1] > 1:
        assert bool((got[last - 1, :4, 5] == -math.inf).all())
    err = (got.double() - ref).abs() <= tol
    err[last - 1:last + 1, :4] = True
    assert bool(err.all())


def test_chunk_attention_skips_pages_outside_the_cache(ops):
    """Tokens of a page id outside the cache are seen by nobody: the same as an equal sequence without them (no mask by
    position applies to what is left)."""
    for news in ([1], [40]):
        pb = R.problem(8, [160], news, 4, 1, 128, 16, "bf16")
        bad = pb.ids.clone()
        bad[2], bad[5] = -1, pb.total_pages
        lse = torch.empty(pb.q.shape[:2], device=DEV)
        out = ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, bad, pb.ptr, pb.last, pb.max_pages, lse=lse)
        gone = [i for i in range(160) if i // 16 in (2, 5)]
        for head in range(4):
            s, _, (page, slot, h) = R.scores(pb, 0, head)
            s[:, gone] = -math.inf
            w = torch.softmax(s, 1)
            want = w @ pb.kv[page, 1, slot, h].double()
            assert torch.allclose(out[:, head].double(), want, rtol=2e-2, atol=2e-2)
            assert torch.allclose(lse[:, head].double(), torch.logsumexp(s, 1), rtol=0, atol=1e-4)


def test_chunk_attention_nan_in_a_seen_key_or_a_query_shows(ops):
    pb = R.problem(9, [70, 50], [70, 1], 4, 1, 128, 16, "bf16")
    page, slot = R.slot_of(pb, 0, torch.tensor([30], device=DEV))
    pb.kv[page[0], 0, slot[0], 0, 3] = math.nan
    pb.q[70, 2, 7] = math.nan
    out, lse = attend(ops, pb)
    assert not bool(out[:30].isnan().any()) and bool(out[30:70].isnan().all()) and bool(lse[30:70].isnan().all())
    assert bool(out[70, 2].isnan().all()) and not bool(out[70, [0, 1, 3]].isnan().any())


def test_chunk_attention_large_scores(ops):
    """Scores in the hundreds, rising and falling along the keys: the running maximum has to follow."""
    pb = R.problem(10, [500], [80], 4, 1, 128, 16, "bf16")
    ramp = torch.linspace(-3, 3, 500, device=DEV).roll(113)
    page, slot = R.slot_of(pb, 0, torch.arange(500, device=DEV))
    pb.kv[page, 0, slot, 0] = (pb.kv[page, 0, slot, 0].float() + ramp[:, None] * torch.sign(pb.q[0, 0].float())).to(pb.dt)
    for scale in (0.0, 1.0):
        out, lse = attend(ops, pb, sm_scale=scale)
        check_attention(pb, out, lse, sm_scale=scale)


def test_single_tokens_agree_with_dense_decode(ops):
    """One token per sequence is the dense decode of the same cache."""
    pb = R.problem(11, [700, 31, 16, 257], [1] * 4, 8, 2, 128, 16, "bf16")
    out, lse = attend(ops, pb)
    l2 = torch.empty_like(lse)
    ref = ops.dense_paged_decode(pb.q, pb.kv, pb.ids, pb.ptr, pb.last, pb.max_pages, lse=l2)
    assert torch.allclose(out.float(), ref.float(), rtol=2e-2, atol=2e-2) and torch.allclose(lse, l2, rtol=0, atol=1e-4)


def test_offsets_beyond_32_bits(ops):
    """A cache of more than 2^32 elements, the sequences on its last pages."""
    pb = R.problem(12, [200, 90], [100, 1], 8, 8, 128, 16, "bf16")
    small = pb.kv
    n = 2 ** 32 // (2 * 16 * 8 * 128) + 40
    big = torch.empty(n, 2, 16, 8, 128, dtype=pb.dt, device=DEV)
    shift = n - small.shape[0]
    big[shift:] = small
    want, wl = attend(ops, pb)
    sc = torch.rand(2, 8, 256, device=DEV)
    sc2 = sc.clone()
    lse = wl.clone()
    ops.attention_mass(pb.q, small, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    kept, lens = ops.evict_tokens(small, sc, pb.ids, pb.ptr, pb.last, 64)
    pb.kv, pb.ids = big, pb.ids + shift
    got, gl = attend(ops, pb)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    ops.attention_mass(pb.q, big, lse, sc2, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    kept2, lens2 = ops.evict_tokens(big, sc2, pb.ids, pb.ptr, pb.last, 64)
    assert torch.equal(sc, sc2) and torch.equal(kept, kept2) and torch.equal(big[shift:], small)


@pytest.mark.parametrize("mods", MODS, ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_mass(ops, case, mods):
    lens, news, hq, hkv, d, page, dtype, offset = SHAPES[case]
    pb = R.problem(100 + case, lens, news, hq, hkv, d, page, dtype, offset)
    mods = with_tensors(pb, mods)
    _, lse = attend(ops, pb, **mods)
    sc = torch.rand(len(lens), hkv, max(lens) + 5, device=DEV)
    want, tol = R.mass(pb, lse, sc, **mods)
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=offset, **mods)
    err = (sc.double() - want).abs()
    assert bool((err <= tol).all()), f"worst error / bound {float((err / tol).max())}"
    # every row gives one whole unit of weight
    if not mods:
        start_free = torch.zeros_like(sc)
        ops.attention_mass(pb.q, pb.kv, lse, start_free, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=offset)
        for b, n in enumerate(news):
            total = start_free[b].double().sum(1)
            assert torch.allclose(total, torch.full_like(total, float(n * hq // hkv)), rtol=1e-4, atol=1e-6)


def test_attention_mass_by_slot_and_what_it_leaves_alone(ops):
    pb = R.problem(40, [100, 260, 33, 64], [3, 100, 0, 1], 4, 2, 128, 16, "bf16", 4)
    _, lse = attend(ops, pb)
    slots = [5, 9, 2, 0]                                  # 9: not a row block; 2: brings no rows
    sc = torch.rand(6, 2, 300, device=DEV)
    before = sc.clone()
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=4, slot_ids=i32(slots))
    want, tol = R.mass(pb, lse, before, blocks=slots)
    assert bool(((sc.double() - want).abs() <= tol).all())
    for s in (1, 2, 3, 4):
        assert torch.equal(sc[s], before[s])
    assert torch.equal(sc[5, :, 100:], before[5, :, 100:])
    # a planning number that is too small costs time only; a sequence longer than the rows of scores is left alone
    sc2 = before.clone()
    ops.attention_mass(pb.q, pb.kv, lse, sc2, pb.q_indptr, pb.ids, pb.ptr, pb.last, 1, first_page_offset=4, slot_ids=i32(slots))
    assert torch.equal(sc, sc2)
    short = torch.rand(4, 2, 200, device=DEV)
    was = short.clone()
    ops.attention_mass(pb.q, pb.kv, lse, short, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=4)
    assert torch.equal(short[1], was[1]) and not torch.equal(short[0], was[0])


def test_attention_mass_empty_rows_and_poison(ops):
    """Rows that saw nothing (lse -inf) give nothing, NaN in unseen tokens stays out."""
    pb = R.problem(41, [3, 120], [9, 30], 4, 1, 128, 16, "bf16", 2)
    _, lse = attend(ops, pb, window=20)
    sc = torch.zeros(2, 1, 130, device=DEV)
    want, tol = R.mass(pb, lse, sc, window=20)
    unseen = torch.arange(0, 120 - 30 - 19, device=DEV)
    page, slot = R.slot_of(pb, 1, unseen)
    pb.kv[page, :, slot] = math.nan
    pb.kv[pb.ids[pb.starts[2] - 1].long(), :, (120 + 2) % 16:] = math.nan
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=2, window=20)
    assert bool(((sc.double() - want).abs() <= tol).all())


EVICT = [
    # lens, hkv, d, page, dtype, offset, budget, sink, local
    ([1], 1, 128, 16, "bf16", 0, 1, 0, 0),
    ([2, 3, 1], 2, 64, 16, "f16", 0, 1, 1, 0),
    ([100, 64, 65, 0, 300], 1, 128, 16, "bf16", 0, 64, 4, 16),
    ([100, 64, 65, 0, 300], 4, 64, 32, "f16", 12, 64, 0, 64),
    ([5000, 4097], 2, 128, 64, "bf16", 0, 2048, 4, 64),
    ([9001, 130], 3, 64, 128, "bf16", 100, 129, 0, 1),
    ([1100] * 40, 1, 128, 16, "f16", 0, 1024, 4, 32),
    ([700], 8, 128, 16, "bf16", 3, 699, 1, 1),
]


@pytest.mark.parametrize("scores", ["spread", "ties"])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict_tokens(ops, case, scores):
    lens, hkv, d, page, dtype, offset, budget, sink, local = EVICT[case]
    pb = R.problem(200 + case, lens, [0] * len(lens), hkv, hkv, d, page, dtype, offset)
    g = torch.Generator().manual_seed(case)
    sc = torch.randn(len(lens), hkv, max(lens) + 3, generator=g)
    if scores == "ties":
        sc = (sc * 1.5).round()                       # few values, -0 and +0 among them
        sc[:, :, ::7] *= 0.0
        sc[:, :, 5::90] = math.inf
        sc[:, :, 11::70] = -math.inf
        sc[:, :, 3::50] = math.nan
    sc = sc.to(DEV)
    kv, out, kept, lens_after = R.evict(pb, sc, budget, sink, local)
    # into a tensor of its own ...
    cache, separate = pb.kv.clone(), sc.clone()
    k1, n1 = ops.evict_tokens(cache, sc, pb.ids, pb.ptr, pb.last, budget, sink_tokens=sink, local_tokens=local,
                              first_page_offset=offset, scores_out=separate)
    assert torch.equal(n1, lens_after) and torch.equal(k1, kept)
    assert torch.equal(cache.view(torch.int16), kv.view(torch.int16))
    assert torch.equal(separate.view(torch.int32), out.view(torch.int32))
    # ... and in place
    cache, same = pb.kv.clone(), sc.clone()
    k2, n2 = ops.evict_tokens(cache, same, pb.ids, pb.ptr, pb.last, budget, sink_tokens=sink, local_tokens=local,
                              first_page_offset=offset)
    assert torch.equal(k2, kept) and torch.equal(n2, lens_after)
    assert torch.equal(cache.view(torch.int16), kv.view(torch.int16)) and torch.equal(same.view(torch.int32), out.view(torch.int32))


def test_evict_tokens_by_slot_and_out_of_contract_sequences(ops):
    pb = R.problem(50, [200, 300, 90, 500], [0] * 4, 2, 2, 128, 16, "bf16")
    slots = [3, -1, 0, 1]                 # -1: no scores; the last sequence is longer than a row of them
    sc = torch.randn(4, 2, 400, device=DEV)
    kv, out, kept, lens = R.evict(pb, sc, 80, 4, 8, blocks=slots)
    k, n = ops.evict_tokens(pb.kv, sc, pb.ids, pb.ptr, pb.last, 80, sink_tokens=4, local_tokens=8, slot_ids=i32(slots))
    assert torch.equal(k, kept) and torch.equal(n, lens) and torch.equal(pb.kv, kv) and torch.equal(sc, out)
    assert lens.tolist() == [80, 300, 80, 500]


def test_evict_tokens_with_a_page_outside_the_cache(ops):
    """Rows from or to a bad page are not moved; everything else is."""
    pb = R.problem(51, [320], [0], 1, 1, 128, 16, "bf16")
    sc = torch.randn(1, 1, 320, device=DEV)
    kv, out, kept, _ = R.evict(pb, sc, 100, 4, 8)
    bad = pb.ids.clone()
    bad[3], bad[10] = 10 ** 6, -5
    k, _ = ops.evict_tokens(pb.kv, sc.clone(), bad, pb.ptr, pb.last, 100, sink_tokens=4, local_tokens=8)
    assert torch.equal(k, kept)
    for dst, src in enumerate(kept[0, 0].tolist()):
        if dst // 16 not in (3, 10) and src // 16 not in (3, 10):
            page, slot = R.slot_of(pb, 0, torch.tensor([dst], device=DEV))
            assert torch.equal(pb.kv[page[0], :, slot[0]], kv[page[0], :, slot[0]])


ROPE = [
    # tokens, hq, hkv, d, dtype, sections, interleaved, far
    (1, 1, 1, 64, "bf16", [32], False, 10),
    (7, 4, 1, 128, "f16", [64], False, 40960),
    (130, 4, 1, 128, "bf16", [24, 20, 20], True, 2 ** 31 - 1),
    (33, 32, 8, 128, "bf16", [16, 24, 24], False, 1000000),
    (65, 5, 2, 64, "f16", [8, 12], True, 100000),
    (5, 40, 8, 64, "bf16", [0, 32], False, 5000),
]


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("case", range(len(ROPE)))
def test_qkv_norm_rope_split(ops, case, norm):
    tokens, hq, hkv, d, dtype, sections, interleaved, far = ROPE[case]
    g = torch.Generator().manual_seed(case)
    dt = R.DT[dtype]
    wide = (2 * torch.randn(tokens, (hq + 2 * hkv) * d + 64, generator=g)).to(dt).to(DEV)
    qkv = wide[:, 8:8 + (hq + 2 * hkv) * d]               # a view with a row stride
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(dt).to(DEV) if norm else None
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(dt).to(DEV) if norm else None
    pos = torch.randint(-min(far, 2 ** 31 - 2) // 3, far, (len(sections), tokens), generator=g, dtype=torch.int64).to(torch.int32).to(DEV)
    freq, axis = ops.rope_table(d, theta=1e6, sections=sections, interleaved=interleaved, device=DEV)
    q, k, v = ops.qkv_norm_rope_split(qkv, qw, kw, 1e-6, pos if len(sections) > 1 else pos[0], freq, axis, hq, hkv)
    inv = [1e6 ** (-2.0 * i / d) for i in range(d // 2)]
    wq, wk, wv = R.rope(qkv, qw, kw, 1e-6, pos, inv, axis.tolist(), hq, hkv, d)
    assert q.is_contiguous() and q.shape == (tokens, hq, d) and k.shape == (tokens, hkv, d)
    assert torch.equal(v.double(), wv)
    half = torch.finfo(dt).eps / 2
    for got, want in ((q, wq), (k, wk)):
        # one rounding; in front of it fp32: the norm (2^-20), the angle (2^-26 of a turn and, for |position| up to 2^31,
        # the 2^-53 of a float64 frequency: below 2^-20 radians together), two products
        mag = torch.sqrt(want[..., :d // 2] ** 2 + want[..., d // 2:] ** 2).repeat(1, 1, 2)
        bound = half * want.abs() * 1.01 + 2.0 ** -18 * mag + (2.0 ** -25 if dt is torch.float16 else 0.0)
        assert bool(((got.double() - want).abs() <= bound).all())


def test_rope_leaves_unturned_pairs_alone_and_matches_the_split_without_positions(ops):
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(9, 6 * 128, generator=g).to(torch.bfloat16).to(DEV)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    freq, axis = ops.rope_table(128, sections=[0], device=DEV)        # no pair is turned
    pos = torch.full((9,), 12345, dtype=torch.int32, device=DEV)
    got = ops.qkv_norm_rope_split(qkv, w, w, 1e-6, pos, freq, axis, 4, 1)
    want = ops.qkv_norm_split(qkv, w, w, 1e-6, 4, 1)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # position 0 turns nothing either
    freq, axis = ops.rope_table(128, device=DEV)
    got = ops.qkv_norm_rope_split(qkv, w, w, 1e-6, torch.zeros_like(pos), freq, axis, 4, 1)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_empty_batches(ops):
    pb = R.problem(60, [40], [0], 4, 1)
    out = ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    assert out.shape == (0, 4, 128)
    sc = torch.rand(1, 1, 50, device=DEV)
    was = sc.clone()
    ops.attention_mass(pb.q, pb.kv, torch.empty(0, 4, device=DEV), sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    assert torch.equal(sc, was)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    k, n = ops.evict_tokens(pb.kv, torch.empty(0, 1, 8, device=DEV), empty, none, empty, 8, sink_tokens=1, local_tokens=1)
    assert k.shape == (0, 1, 8) and n.shape == (0,)
    freq, axis = ops.rope_table(128, device=DEV)
    q, k, v = ops.qkv_norm_rope_split(torch.empty(0, 6 * 128, dtype=torch.bfloat16, device=DEV), None, None, 1e-6,
                                      torch.empty(0, dtype=torch.int32, device=DEV), freq, axis, 4, 1)
    assert q.shape == (0, 4, 128) and v.shape == (0, 1, 128)


def test_captured_replays_and_another_stream(ops):
    """The whole run in one HIP graph, replayed with new inputs between eager work, against the eager calls."""
    pb = R.problem(70, [600, 90], [64, 1], 8, 2, 128, 16, "bf16")
    ws = torch.empty(max(16, ops.chunk_workspace_bytes(pb.q.shape[0], 2, 8, 2, pb.max_pages)), dtype=torch.uint8, device=DEV)
    lse = torch.empty(pb.q.shape[:2], device=DEV)
    out = torch.empty_like(pb.q)
    sc = torch.zeros(2, 2, 640, device=DEV)
    kept = torch.empty(2, 2, 128, dtype=torch.int32, device=DEV)
    lens = torch.empty(2, dtype=torch.int32, device=DEV)
    first = pb.kv.clone()

    def step():
        ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, out=out, lse=lse, workspace=ws)
        ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
        ops.evict_tokens(pb.kv, sc, pb.ids, pb.ptr, pb.last, 128, kept=kept, new_lens=lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        torch.manual_seed(i)
        pb.q.normal_()
        pb.kv.copy_(first)
        sc.fill_(0.5)
        step()
        torch.cuda.synchronize()
        want = [x.clone() for x in (out, lse, sc, kept, lens, pb.kv)]
        pb.kv.copy_(first)
        sc.fill_(0.5)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, (out, lse, sc, kept, lens, pb.kv)):
            assert torch.equal(a, b)


def test_two_streams_at_once(ops):
    """Two chunks on two streams, each with its own workspace (allocated by the call), give what they give alone."""
    a = R.problem(71, [3000], [2], 8, 2, 128, 16, "bf16")
    b = R.problem(72, [2000, 100], [64, 100], 8, 2, 128, 16, "bf16")
    want = [attend(ops, a), attend(ops, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        got = []
        for s, pb in ((s1, a), (s2, b)):
            with torch.cuda.stream(s):
                got.append(attend(ops, pb))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_opcheck(ops):
    """Schemas, fake kernels and mutation annotations of the four operators under AOT dispatch."""
    from torch.library import opcheck

    pb = R.problem(73, [100, 40], [3, 1], 4, 2, 128, 16, "bf16")
    table = (pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    lse = torch.empty(pb.q.shape[:2], device=DEV)
    k = torch.ops.kinetics
    opcheck(k.paged_chunk_attention.default, (pb.q, pb.kv, *table), dict(lse=lse, window=30))
    ops.paged_chunk_attention(pb.q, pb.kv, *table, lse=lse)
    opcheck(k.attention_mass.default, (pb.q, pb.kv, lse, torch.rand(2, 2, 128, device=DEV), *table))
    opcheck(k.evict_tokens.default, (pb.kv, torch.rand(2, 2, 128, device=DEV), pb.ids, pb.ptr, pb.last, 64))
    freq, axis = ops.rope_table(128, device=DEV)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    opcheck(k.qkv_norm_rope_split.default, (torch.randn(5, 6 * 128, device=DEV).bfloat16(), w, w, 1e-6, i32([0, 5, 2, 9, 1]), freq, axis, 4, 1))
    opcheck(k.qkv_norm_rope_split.default, (torch.randn(5, 6 * 128, device=DEV).bfloat16(), None, None, 1e-6, i32([0, 5, 2, 9, 1]), freq, axis, 4, 1))


def test_the_run_of_them(ops):
    """Prompt in two chunks (rotary split, ragged append, attention, mass), eviction, then a decoded token: every step
    against the plain forms on the same cache."""
    hq, hkv, d, page, budget = 8, 2, 128, 16, 96
    g = torch.Generator().manual_seed(80)
    dt = torch.bfloat16
    kv = torch.zeros(40, 2, page, hkv, d, dtype=dt, device=DEV)
    table = torch.randperm(40, generator=g)[:20].to(torch.int32).to(DEV)
    qw, kw = (torch.ones(d, dtype=dt, device=DEV) for _ in range(2))
    freq, axis = ops.rope_table(d, sections=[24, 20, 20], device=DEV)
    sc = torch.zeros(1, hkv, 320, device=DEV)
    have = pos0 = 0
    for step, n in enumerate((130, 70, 1)):
        qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).to(dt).to(DEV)
        pos = (pos0 + torch.arange(n, dtype=torch.int32)).repeat(3, 1).to(DEV)
        q, k, v = ops.qkv_norm_rope_split(qkv, qw, kw, 1e-6, pos, freq, axis, hq, hkv)
        pos0 += n
        have += n
        pages = (have + page - 1) // page
        ids, ptr, last = table[:pages].contiguous(), i32([0, pages]), i32([have - (pages - 1) * page])
        ind = i32([0, n])
        ops.append_paged_kv_ragged(k, v, ind, kv, None, ids, ptr, last)
        pb = R.SimpleNamespace(lens=[have], news=[n], counts=[pages], starts=[0, pages], ends=[0, n], hq=hq, hkv=hkv, d=d, page=page,
                               offset=0, dt=dt, kv=kv, q=q, ids=ids, ptr=ptr, last=last, q_indptr=ind, max_pages=pages, total_pages=40)
        out, lse = attend(ops, pb)
        check_attention(pb, out, lse)
        want, tol = R.mass(pb, lse, sc)
        ops.attention_mass(q, kv, lse, sc, ind, ids, ptr, last, pages)
        assert bool(((sc.double() - want).abs() <= tol).all())
        if step == 1:
            wkv, wsc, wkept, _ = R.evict(pb, sc, budget, 4, 16)
            kept, lens = ops.evict_tokens(kv, sc, ids, ptr, last, budget, sink_tokens=4, local_tokens=16)
            assert torch.equal(kept, wkept) and torch.equal(kv, wkv) and torch.equal(sc, wsc)
            have = int(lens[0])
            assert have == budget


def test_refusals(ops):
    pb = R.problem(90, [40, 20], [3, 1], 4, 1)
    a = (pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    with pytest.raises(TypeError):
        ops.paged_chunk_attention(pb.q.half(), *a[1:])
    with pytest.raises(ValueError, match="contiguous"):
        ops.paged_chunk_attention(torch.cat([pb.q, pb.q], 2)[..., :128], *a[1:])
    with pytest.raises(ValueError, match="page_indptr"):
        ops.paged_chunk_attention(pb.q, pb.kv, i32([0, 4]), *a[3:])
    for bad in (dict(window=-1), dict(softcap=-1.0), dict(softcap=math.inf), dict(sm_scale=-0.1), dict(sm_scale=math.nan),
                dict(first_page_offset=16), dict(num_splits=-1), dict(num_splits=5000), dict(slopes=torch.ones(3, device=DEV)),
                dict(prefix_lens=i32([1])), dict(out=torch.empty_like(pb.q[:2])), dict(lse=torch.empty(4, 3, device=DEV))):
        with pytest.raises(ValueError):
            ops.paged_chunk_attention(*a, **bad)
    from kinetics_amd import _lib

    with pytest.raises(_lib.KineticsError, match="WORKSPACE"):
        ops.paged_chunk_attention(*a, num_splits=2, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    lse = torch.zeros(4, 4, device=DEV)
    with pytest.raises(ValueError):
        ops.attention_mass(pb.q, pb.kv, lse, torch.zeros(1, 1, 64, device=DEV), *a[2:])
    with pytest.raises(TypeError):
        ops.attention_mass(pb.q, pb.kv, lse, torch.zeros(2, 1, 64, device=DEV, dtype=torch.float64), *a[2:])
    sc = torch.zeros(2, 1, 64, device=DEV)
    for bad in (dict(budget=0), dict(budget=8, sink_tokens=5, local_tokens=4), dict(budget=8, sink_tokens=-1, local_tokens=0),
                dict(budget=40, kept=torch.empty(2, 1, 8, dtype=torch.int32, device=DEV)), dict(budget=40, scores_out=sc[:1])):
        with pytest.raises(ValueError):
            ops.evict_tokens(pb.kv, sc, pb.ids, pb.ptr, pb.last, **bad)
    both = torch.zeros(3, 1, 64, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.evict_tokens(pb.kv, both[:2], pb.ids, pb.ptr, pb.last, 40, scores_out=both[1:])
    freq, axis = ops.rope_table(128, device=DEV)
    qkv = torch.zeros(3, 6 * 128, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    for args in ((qkv, w, None, 1e-6, i32([0, 1, 2]), freq, axis, 4, 1), (qkv, w, w, 1e-6, i32([0, 1]), freq, axis, 4, 1),
                 (qkv, w, w, 1e-6, i32([0, 1, 2]), freq[:40], axis[:40], 4, 1), (qkv, w, w, -1.0, i32([0, 1, 2]), freq, axis, 4, 1),
                 (qkv, w, w, 1e-6, i32([0, 1, 2]), freq, axis, 5, 1)):
        with pytest.raises(ValueError):
            ops.qkv_norm_rope_split(*args)


@pytest.mark.parametrize("group", [1, 3, 4])
@pytest.mark.parametrize("news", [1, 3, 50, 170])
def test_infinite_keys_with_no_weight(ops, news, group):
    """Keys whose scores are -inf for every row have weight 0, in tiles that are full of rows and in those that are not."""
    pb = R.problem(91, [300, 200], [news, news], group, 1, 128, 16, "bf16")
    pb.q[..., 0] = pb.q[..., 0].abs() + 0.25
    for b, t in ((0, 5), (0, 140), (0, 299), (1, 40)):
        page, slot = R.slot_of(pb, b, torch.tensor([t], device=DEV))
        pb.kv[page, 0, slot, 0, 0] = -math.inf
    out, lse = attend(ops, pb)
    check_attention(pb, out, lse)
    start = torch.rand(2, 1, 310, device=DEV)
    sc = start.clone()
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    want, tol = R.mass(pb, lse, start)
    assert bool(((sc.double() - want).abs() <= tol).all())
    assert float(sc[0, 0, 5]) == float(start[0, 0, 5]) and float(sc[1, 0, 40]) == float(start[1, 0, 40])


def test_q_indptr_that_does_not_ascend_stays_inside(ops):
    """Out of contract, but no row is written that the table does not name."""
    pb = R.problem(92, [40, 40], [3, 0], 4, 1, 128, 16, "bf16", tail_rows=197)
    out = torch.full_like(pb.q, 5.0)
    ops.paged_chunk_attention(pb.q, pb.kv, i32([200, 0, 3]), pb.ids, pb.ptr, pb.last, pb.max_pages, out=out)
    assert bool((out[3:] == 5.0).all())


def test_thousands_of_sequences(ops):
    """More sequences than the 64 x 64 that two steps of the search for a row tile's sequence cover."""
    lens = [(7 * i) % 4 if i % 5 else 0 for i in range(4200)] + [33]
    news = [min(n, (i // 3) % 3) for i, n in enumerate(lens)]
    pb = R.problem(93, lens, news, 2, 1, 64, 16, "f16")
    out, lse = attend(ops, pb)
    check_attention(pb, out, lse)
    sc = torch.zeros(len(lens), 1, 40, device=DEV)
    ops.attention_mass(pb.q, pb.kv, lse, sc, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages)
    want, tol = R.mass(pb, lse, torch.zeros_like(sc))
    assert bool(((sc.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("n,budget", [(20000, 5000), (17000, 16900), (700, 300)])
def test_evict_tokens_whose_scores_differ_in_their_last_bits(ops, n, budget):
    """Every digit of the search is needed, and more keys than it ranks at once share the upper ones."""
    pb = R.problem(94, [n], [0], 1, 1, 64, 64, "bf16", 7)
    g = torch.Generator().manual_seed(94)
    for spread in (3000, 40):
        sc = (1.0 + torch.randint(0, spread, (1, 1, n + 5), generator=g).double() * 2.0 ** -23).float().to(DEV)
        kv, scores, kept, lens = R.evict(pb, sc, budget, 4, 100)
        got, new = ops.evict_tokens(pb.kv, sc, pb.ids, pb.ptr, pb.last, budget, sink_tokens=4, local_tokens=100, first_page_offset=7)
        assert torch.equal(got, kept) and torch.equal(new, lens) and torch.equal(sc, scores)
        assert torch.equal(pb.kv.view(torch.int16), kv.view(torch.int16))
