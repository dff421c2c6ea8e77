"""How many bits the weights of the chunk attention keep, against float64 forms whose bounds count the roundings there are."""
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


def attend(ops, pb, **mods):
    return ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, first_page_offset=pb.offset, **mods)


def plain(pb, narrow, **mods):
    """(out, bound) in float64.  The bound: the result's rounding; scores (twice, score and maximum); exp2, the quotient and the joins
    2^-17; sums of n weights and products in fp32, an eighth and a quarter of them one after the other, below n * 2^-25; the
    weights themselves: more than 32 rows, one rounding to the element type; up to 32, two parts of it, 2^-18.  In float16 a part is
    never finer than 2^-38 of the row's reference weight, and a result never finer than 2^-25."""
    rows = pb.q.shape[0]
    out = torch.zeros(rows, pb.hq, pb.d, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    half = torch.finfo(pb.dt).eps / 2
    for b, n in enumerate(pb.news):
        for head in range(pb.hq if n else 0):
            s, off, (page, slot, h) = R.scores(pb, b, head, **mods)
            r = slice(pb.ends[b], pb.ends[b + 1])
            w = torch.softmax(s, 1)
            v = pb.kv[page, 1, slot, h].double()
            v = torch.where(v.isfinite(), v, torch.zeros_like(v))
            out[r, head] = w @ v
            mag = w @ v.abs()
            rel = 2 * off + 2.0 ** -17 + s.shape[1] * 2.0 ** -25 + (2.0 ** -18 if narrow else half * 1.01)
            tol[r, head] = half * 1.01 * (out[r, head].abs() + rel * mag) + rel * mag + 1e-30
            if pb.dt is torch.float16:
                tol[r, head] += 2.0 ** -38 * v.abs().sum(0) + 2.0 ** -25
    return out, tol


def check(pb, got, narrow=True, **mods):
    want, tol = plain(pb, narrow, **mods)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst error / bound {float((err / tol).max())}"


@pytest.mark.parametrize("mods", [dict(), dict(softcap=30.0), dict(window=150), dict(num_splits=3)], ids=["plain", "cap", "window", "spans"])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_weights_of_few_rows_are_not_rounded_to_the_element_type(ops, dtype, d, mods):
    """Values that cancel under the weights: a weight of 16 bits would leave its rounding in the result."""
    n = 402
    pb = R.problem(1, [n] * 12, [1] * 12, 4, 1, d, 16, dtype, 3)
    tok = torch.arange(n, device=DEV)
    pb.q.zero_()
    pb.q[:, :, 0] = torch.tensor([1.0, 1.125, 0.875, 1.5], device=DEV, dtype=pb.dt)
    for b in range(12):
        page, slot = R.slot_of(pb, b, tok)
        u = (0.31 + 0.53 * b)
        k = torch.zeros(n, d, dtype=pb.dt, device=DEV)
        k[1::2, 0] = -u
        p = math.exp(float(k[1, 0]) / math.sqrt(d))
        v = torch.ones(n, d, dtype=pb.dt, device=DEV)
        v[1::2] = -((1 + 2.0 ** -7 * torch.linspace(-1, 1, d, device=DEV)) / p).to(pb.dt)
        pb.kv[page, 0, slot, 0], pb.kv[page, 1, slot, 0] = k, v
    got = attend(ops, pb, **mods)
    mods.pop("num_splits", None)
    check(pb, got, **mods)


@pytest.mark.parametrize("lens,news,hq,hkv,d,page,offset", [
    ([700, 31, 1, 257], [1] * 4, 8, 2, 128, 16, 0),
    ([900, 64, 40], [8, 3, 1], 4, 1, 64, 64, 9),
    ([333], [32], 2, 2, 128, 32, 5),
    ([600] * 40, [1] * 40, 16, 1, 64, 16, 0),
])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_few_rows(ops, dtype, lens, news, hq, hkv, d, page, offset):
    pb = R.problem(2, lens, news, hq, hkv, d, page, dtype, offset)
    check(pb, attend(ops, pb))
    mods = dict(window=100, prefix_lens=torch.tensor([(i * 7) % 50 for i in range(len(lens))], dtype=torch.int32, device=DEV),
                slopes=2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float32) / hq))
    check(pb, attend(ops, pb, **mods), **mods)


@pytest.mark.parametrize("news", [1, 5, 64, 200])
@pytest.mark.parametrize("extra", [False, True])
def test_many_small_weights_in_float16(ops, news, extra):
    """One heavy token with a value of 0 and thousands of weight 2^-26: their values are the whole result."""
    n = 4000
    pb = R.problem(3, [n], [news], 4, 1, 128, 16, "f16")
    page, slot = R.slot_of(pb, 0, torch.arange(n, device=DEV))
    k, v = torch.zeros(n, 128, dtype=pb.dt, device=DEV), torch.full((n, 128), 1000.0, dtype=pb.dt, device=DEV)
    k[0, 0], v[0] = 25.75, 0.0
    v[1:, 64:] *= 1 + torch.rand(n - 1, 64, device=DEV).to(pb.dt)
    pb.kv[page, 0, slot, 0], pb.kv[page, 1, slot, 0] = k, v
    pb.q.zero_()
    pb.q[:, :, 0] = torch.tensor([8.0, 7.5, 4.0, 8.25], device=DEV, dtype=pb.dt)
    mods = dict(softcap=200.0) if extra else {}
    check(pb, attend(ops, pb, **mods), narrow=news * 4 <= 32, **mods)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("news", [1, 40])
@pytest.mark.parametrize("power", [6, 9, 11, 12, 13, 14, 15])
def test_scores_of_many_millions(ops, power, news, dtype):
    """Far apart, so that every row gets the value of its largest score, whatever fp32 makes of its last digits."""
    n = 700
    pb = R.problem(6, [n], [news], 4, 1, 128, 16, dtype)
    g = torch.Generator().manual_seed(6)
    step = 64 + 64 * torch.randperm(n, generator=g).to(DEV)                  # up to 44864, some not exact in 16 bits
    page, slot = R.slot_of(pb, 0, torch.arange(n, device=DEV))
    k = torch.zeros(n, 128, dtype=pb.dt, device=DEV)
    k[:, 0] = step.to(pb.dt)
    pb.kv[page, 0, slot, 0] = k
    pb.q.zero_()
    pb.q[:, :, 0] = torch.tensor([1.0, -1.0, 0.5, 0.75], device=DEV, dtype=pb.dt) * 2.0 ** power
    got = attend(ops, pb)
    v = pb.kv[page, 1, slot, 0]
    for r in range(news):
        for head in range(4):
            s = k[:n - news + r + 1, 0].double() * float(pb.q[r, head, 0])
            top = (s == s.max()).nonzero()[:, 0]
            want = v[top].double().mean(0)
            assert bool(((got[r, head].double() - want).abs() <= torch.finfo(pb.dt).eps * (want.abs() + v[top].double().abs().amax(0))).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("news", [1, 7, 60])
def test_infinite_values_that_every_row_sees(ops, news, dtype):
    """Values that are infinite or NaN in blocks without a mask reach their own column alone, with their sign."""
    pb = R.problem(4, [900, 300], [news, news], 4, 1, 128, 16, dtype)
    for b, t, col, x in ((0, 100, 5, math.inf), (0, 333, 7, -math.inf), (0, 64, 9, math.nan), (0, 400, 11, math.inf), (0, 17, 11, -math.inf),
                         (1, 40, 127, math.inf), (1, 41, 127, math.inf)):
        page, slot = R.slot_of(pb, b, torch.tensor([t], device=DEV))
        pb.kv[page, 1, slot, 0, col] = x
    got = attend(ops, pb)
    a, b = got[:news], got[news:]
    assert bool((a[:, :, 5] == math.inf).all()) and bool((a[:, :, 7] == -math.inf).all()) and bool((b[:, :, 127] == math.inf).all())
    assert bool(a[:, :, [9, 11]].isnan().all())
    want, tol = plain(pb, news * 4 <= 32)
    ok = (got.double() - want).abs() <= tol
    ok[:news, :, [5, 7, 9, 11]] = True
    ok[news:, :, 127] = True
    assert bool(ok.all())


def test_more_tokens_than_one_batch_of_page_ids(ops):
    """Every span of the keys walks over many blocks; one span too."""
    pb = R.problem(5, [9000, 4200], [1, 2], 4, 1, 64, 16, "bf16", 7)
    for splits in (0, 1):
        check(pb, attend(ops, pb, num_splits=splits))
