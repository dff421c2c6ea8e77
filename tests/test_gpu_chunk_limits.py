"""The chunk operators at the ends of their ranges."""
import math

import pytest
import torch

from tests import chunk_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("softcap", [1.0, 1e-7, 1.4e-8, 1e-8, 1e-12, 1e-30])
@pytest.mark.parametrize("news", [1, 40])
def test_mass_of_scores_of_zero_under_any_cap(softcap, news):
    """A score of 0 stays 0 under a cap whose short form has coefficients beyond fp32; other scores are at the cap."""
    from kinetics_amd import ops

    pb = R.problem(1, [300, 130], [news, news], 4, 1, 128, 16, "bf16")
    pb.q[:news] = 0.0
    lse = torch.empty(pb.q.shape[:2], device=DEV)
    ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, lse=lse, softcap=softcap)
    start = torch.rand(2, 1, 310, device=DEV)
    want, tol = R.mass(pb, lse, start, softcap=softcap)
    got = start.clone()
    ops.attention_mass(pb.q, pb.kv, lse, got, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, softcap=softcap)
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [128, 64])
def test_a_pair_that_is_not_turned_keeps_its_elements(d, dtype):
    """Whatever its partner is: an infinity or NaN in the other half is no part of it."""
    from kinetics_amd import ops

    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(5, 6 * d, generator=g).to(R.DT[dtype]).to(DEV)
    x = qkv.view(5, 6, d)
    x[0, 0, d // 2 - 1], x[1, 4, d - 1], x[2, 3, d - 2] = math.inf, math.nan, -math.inf
    freq, axis = ops.rope_table(d, sections=[3], device=DEV)
    pos = torch.arange(5, dtype=torch.int32, device=DEV) * 7
    q, k, v = ops.qkv_norm_rope_split(qkv, None, None, 1e-6, pos, freq, axis, 4, 1)
    got = torch.cat([q, k, v], 1).double()
    same = [i for i in range(d) if i % (d // 2) >= 3]
    assert torch.equal(got[:, :, same].nan_to_num(nan=7e7), x[:, :, same].double().nan_to_num(nan=7e7))
    want = R.rope(qkv, None, None, 1e-6, pos, [1e6 ** (-2.0 * i / d) for i in range(d // 2)], axis.tolist(), 4, 1, d)
    turned = [i for i in range(d) if i % (d // 2) < 3]
    mag = x[:, :5].double().abs().nan_to_num(0, 0, 0).amax(-1, keepdim=True) * 1.5
    err = (got[:, :5] - torch.cat(want[:2], 1)).abs()[..., turned]
    assert bool((err <= (torch.finfo(R.DT[dtype]).eps / 2 + 2.0 ** -18) * mag).all())


def test_mass_of_many_long_page_lists():
    """512 sequences of 8 heads planned for 2^22 tokens each: more (sequence, head, tile) triples than a grid holds workgroups."""
    from kinetics_amd import ops

    lens = [0] * 512
    lens[3], lens[511] = 700, 40
    news = [0] * 512
    news[3], news[511] = 2, 1
    pb = R.problem(3, lens, news, 8, 8, 64, 16, "bf16")
    lse = torch.empty(pb.q.shape[:2], device=DEV)
    ops.paged_chunk_attention(pb.q, pb.kv, pb.q_indptr, pb.ids, pb.ptr, pb.last, pb.max_pages, lse=lse)
    start = torch.rand(512, 8, 704, device=DEV)
    want, tol = R.mass(pb, lse, start)
    ops.attention_mass(pb.q, pb.kv, lse, start, pb.q_indptr, pb.ids, pb.ptr, pb.last, 2 ** 18)
    assert bool(((start.double() - want).abs() <= tol).all())
