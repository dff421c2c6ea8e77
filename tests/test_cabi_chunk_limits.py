"""Sizes that no launch of the chunk operators can hold, without a GPU."""
import pytest

from kinetics_amd import _lib
from tests.test_cabi_chunk import A, chunk, evict, mass, rope


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_launches_beyond_what_a_grid_holds_are_refused(lib):
    """A grid has fewer than 2^32 threads; nothing is launched for a call that would need more, in any of its kernels."""
    assert evict(lib, B=1 << 18, Hkv=4, blocks=1 << 18) == _lib.KIN_ERR_UNSUPPORTED
    assert evict(lib, B=1 << 21, Hkv=1, D=64, blocks=1 << 21) == _lib.KIN_ERR_UNSUPPORTED
    assert chunk(lib, B=1 << 22, Hq=4, Hkv=4, nnz=1) == _lib.KIN_ERR_UNSUPPORTED
    # the join of the spans: head_dim / 4 threads to a (row, head)
    assert chunk(lib, nnz=1 << 25, B=1, splits=2, ws=A, wsb=1 << 60) == _lib.KIN_ERR_UNSUPPORTED
    assert mass(lib, B=1 << 22, Hq=4, Hkv=4, blocks=1 << 22) == _lib.KIN_ERR_UNSUPPORTED
    assert rope(lib, T=1 << 24, Hq=32, Hkv=8, stride=48 * 128) == _lib.KIN_ERR_UNSUPPORTED
    assert rope(lib, T=1 << 26) == _lib.KIN_ERR_UNSUPPORTED
