"""The chunk operators at the ends of their ranges."""
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
