"""The chunk operators without a GPU: argument errors of the C entry points, workspace sizes, the rotary table, fake kernels."""
import math

import pytest
import torch

from kinetics_amd import _lib

A = 0x1000  # a non-null, 16-byte aligned dummy address; never dereferenced on these paths


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def chunk(lib, q=A, kv=A, ind=A, idx=A, ptr=A, last=A, out=A, ws=None, wsb=0, nnz=64, B=2, Hq=4, Hkv=1, D=128, ps=16, P=8, mp=4, offset=0,
          scale=0.0, cap=0.0, window=0, splits=1, f16=False):
    fn = lib.kin_paged_chunk_attention_f16 if f16 else lib.kin_paged_chunk_attention
    return fn(q, kv, ind, idx, ptr, last, None, None, out, None, ws, wsb, nnz, B, Hq, Hkv, D, ps, P, mp, offset, scale, cap, window,
              splits, None)


@pytest.mark.parametrize("f16", [False, True])
def test_chunk_attention_argument_errors(lib, f16):
    for name in ("q", "kv", "ind", "idx", "ptr", "last", "out"):
        assert chunk(lib, f16=f16, **{name: None}) == _lib.KIN_ERR_NULL_POINTER, name
    assert (b"_f16" in lib.kin_last_error()) == f16
    for bad in (dict(B=-1), dict(nnz=-1), dict(Hkv=0), dict(Hq=5, Hkv=2), dict(P=0), dict(mp=0), dict(offset=16), dict(offset=-1),
                dict(window=-1), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.inf),
                dict(cap=math.nan), dict(splits=-1), dict(splits=1025)):
        assert chunk(lib, f16=f16, **bad) == _lib.KIN_ERR_BAD_SHAPE, bad
    for bad in (dict(D=96), dict(ps=24), dict(nnz=1 << 40), dict(Hq=40000, Hkv=1, nnz=1)):
        assert chunk(lib, f16=f16, **bad) == _lib.KIN_ERR_UNSUPPORTED, bad
    for bad in (dict(q=A + 2), dict(kv=A + 8), dict(out=A + 4)):
        assert chunk(lib, f16=f16, **bad) == _lib.KIN_ERR_MISALIGNED, bad
    assert chunk(lib, f16=f16, splits=2) == _lib.KIN_ERR_WORKSPACE
    need = lib.kin_chunk_workspace_bytes(64, 2, 4, 1, 4, 16, 128, 2)
    assert need == 64 * 4 * (2 * 129 + 1) * 4
    assert chunk(lib, f16=f16, splits=2, ws=A, wsb=need - 1) == _lib.KIN_ERR_WORKSPACE
    assert chunk(lib, f16=f16, splits=2, ws=A + 8, wsb=need) == _lib.KIN_ERR_MISALIGNED
    assert chunk(lib, f16=f16, B=0) == _lib.KIN_OK and chunk(lib, f16=f16, nnz=0, Hq=64) == _lib.KIN_OK


def test_chunk_workspace_bytes(lib):
    size = lib.kin_chunk_workspace_bytes
    assert size(0, 1, 4, 1, 100, 16, 128, 0) == 0 and size(5, 0, 4, 1, 100, 16, 128, 0) == 0 and size(5, 2, 4, 3, 100, 16, 128, 0) == 0
    assert size(8, 8, 4, 1, 16, 16, 128, 0) == 0                      # 256 tokens: one span of 4 tiles
    assert size(8, 8, 4, 1, 257, 16, 128, 0) == 8 * 4 * (17 * 129 + 1) * 4
    assert size(65536, 8, 32, 8, 512, 16, 128, 0) == 0                # prompts that fill the GPU by themselves
    assert size(64, 64, 32, 8, 512, 16, 64, 0) > 0                    # decode of uneven sequences


def mass(lib, q=A, kv=A, lse=A, sc=A, ind=A, nnz=64, B=2, Hq=4, Hkv=1, D=128, P=8, mp=4, cap=0.0, window=0, blocks=2, stride=64,
         slots=None):
    return lib.kin_attention_mass(q, kv, lse, sc, ind, A, A, A, None, None, nnz, B, Hq, Hkv, D, 16, P, mp, 0, 0.0, cap, window, blocks,
                                  stride, slots, None)


def test_attention_mass_argument_errors(lib):
    for name in ("q", "kv", "lse", "sc", "ind"):
        assert mass(lib, **{name: None}) == _lib.KIN_ERR_NULL_POINTER, name
    for bad in (dict(nnz=-1), dict(window=-2), dict(cap=-1.0), dict(blocks=1), dict(blocks=-1), dict(stride=0), dict(slots=A, blocks=0)):
        assert mass(lib, **bad) == _lib.KIN_ERR_BAD_SHAPE, bad
    assert mass(lib, D=256) == _lib.KIN_ERR_UNSUPPORTED
    assert mass(lib, Hq=129) == _lib.KIN_ERR_UNSUPPORTED
    assert mass(lib, B=1 << 20, Hq=64, Hkv=64, blocks=1 << 20, mp=1 << 20) == _lib.KIN_ERR_UNSUPPORTED
    assert mass(lib, kv=A + 2) == _lib.KIN_ERR_MISALIGNED
    assert mass(lib, B=0, blocks=0) == _lib.KIN_OK and mass(lib, nnz=0) == _lib.KIN_OK


def evict(lib, kv=A, sc=A, out=A, kept=A, lens=A, B=2, Hkv=1, D=128, ps=16, P=8, offset=0, budget=32, sink=4, local=8, blocks=2, stride=64,
          slots=None):
    return lib.kin_evict_tokens(kv, sc, out, A, A, A, kept, lens, B, Hkv, D, ps, P, offset, budget, sink, local, blocks, stride, slots, None)


def test_evict_tokens_argument_errors(lib):
    for name in ("kv", "sc", "out", "kept", "lens"):
        assert evict(lib, **{name: None}) == _lib.KIN_ERR_NULL_POINTER, name
    for bad in (dict(B=-1), dict(Hkv=0), dict(P=0), dict(offset=16), dict(budget=0), dict(sink=-1), dict(local=-1), dict(sink=25),
                dict(sink=2 ** 31 - 1, local=2 ** 31 - 1), dict(blocks=1), dict(stride=0), dict(slots=A, blocks=0)):
        assert evict(lib, **bad) == _lib.KIN_ERR_BAD_SHAPE, bad
    assert evict(lib, D=80) == _lib.KIN_ERR_UNSUPPORTED and evict(lib, ps=8) == _lib.KIN_ERR_UNSUPPORTED
    assert evict(lib, P=1 << 40) == _lib.KIN_ERR_UNSUPPORTED
    assert evict(lib, kv=A + 4) == _lib.KIN_ERR_MISALIGNED
    assert evict(lib, B=0, blocks=0) == _lib.KIN_OK


def rope(lib, qkv=A, stride=768, qw=A, kw=A, pos=A, axes=1, freq=A, axis=A, q=A, k=A, v=A, T=2, Hq=4, Hkv=1, D=128, eps=1e-6):
    return lib.kin_qkv_norm_rope_split(qkv, stride, qw, kw, eps, pos, axes, freq, axis, q, k, v, T, Hq, Hkv, D, None)


def test_qkv_norm_rope_split_argument_errors(lib):
    for name in ("qkv", "kw", "pos", "freq", "axis", "q", "k", "v"):
        assert rope(lib, **{name: None}) == _lib.KIN_ERR_NULL_POINTER, name
    for bad in (dict(T=-1), dict(Hq=0), dict(axes=0), dict(stride=760), dict(stride=772), dict(eps=-1.0), dict(eps=math.nan)):
        assert rope(lib, **bad) == _lib.KIN_ERR_BAD_SHAPE, bad
    assert rope(lib, D=96) == _lib.KIN_ERR_UNSUPPORTED
    assert rope(lib, q=A + 2) == _lib.KIN_ERR_MISALIGNED
    assert rope(lib, T=0) == _lib.KIN_OK and rope(lib, T=0, qw=None, kw=None) == _lib.KIN_OK


def test_rope_table():
    from kinetics_amd import ops

    freq, axis = ops.rope_table(128, theta=1e6, sections=[24, 20, 20], device="cpu")
    assert freq.dtype == torch.int64 and axis.dtype == torch.int32 and axis.tolist() == [0] * 24 + [1] * 20 + [2] * 20
    for i in (0, 1, 40, 63):
        turns = (int(freq[i]) % 2 ** 64) / 2.0 ** 64
        assert math.isclose(turns * 2 * math.pi, 1e6 ** (-2 * i / 128), rel_tol=1e-14)
    _, axis = ops.rope_table(64, sections=[4, 8, 20], interleaved=True, device="cpu")
    assert axis.tolist() == [0, 1, 2] * 4 + [1, 2] * 4 + [2] * 12
    _, axis = ops.rope_table(64, sections=[3, 5], device="cpu")
    assert axis.tolist() == [0] * 3 + [1] * 5 + [-1] * 24
    freq, axis = ops.rope_table(64, inv_freq=[-2.5 + i for i in range(32)], device="cpu")        # negative, and more than a turn
    for i in range(32):
        turns = (int(freq[i]) % 2 ** 64) / 2.0 ** 64
        assert math.isclose(turns, ((-2.5 + i) / (2 * math.pi)) % 1.0, rel_tol=1e-12)
    for bad in (dict(sections=[40]), dict(sections=[-1, 5]), dict(sections=[]), dict(inv_freq=[1.0]), dict(inv_freq=[math.inf] * 32)):
        with pytest.raises(ValueError):
            ops.rope_table(64, device="cpu", **bad)


def test_chunk_ops_have_fake_kernels_and_refuse_cpu_tensors():
    from kinetics_amd import ops

    meta = dict(device="meta")
    q = torch.empty(5, 4, 128, dtype=torch.bfloat16, **meta)
    kv = torch.empty(8, 2, 16, 1, 128, dtype=torch.bfloat16, **meta)
    i = torch.empty(3, dtype=torch.int32, **meta)
    two = torch.empty(2, dtype=torch.int32, **meta)
    assert torch.ops.kinetics.paged_chunk_attention(q, kv, i, i, i, two, 4).shape == q.shape
    sc = torch.empty(2, 1, 64, **meta)
    assert torch.ops.kinetics.attention_mass(q, kv, torch.empty(5, 4, **meta), sc, i, i, i, two, 4) is None
    kept, lens = torch.ops.kinetics.evict_tokens(kv, sc, i, i, two, 32)
    assert kept.shape == (2, 1, 32) and kept.dtype == torch.int32 and lens.shape == (2,)
    qkv = torch.empty(3, 6 * 128, dtype=torch.float16, **meta)
    f = torch.empty(64, dtype=torch.int64, **meta)
    a, b, c = torch.ops.kinetics.qkv_norm_rope_split(qkv, None, None, 1e-6, i, f, torch.empty(64, dtype=torch.int32, **meta), 4, 1)
    assert a.shape == (3, 4, 128) and b.shape == c.shape == (3, 1, 128) and a.dtype == torch.float16
    cpu = torch.zeros(5, 4, 128, dtype=torch.bfloat16)
    ckv = torch.zeros(8, 2, 16, 1, 128, dtype=torch.bfloat16)
    ci = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_chunk_attention(cpu, ckv, ci, ci, ci, ci[:2], 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.evict_tokens(ckv, torch.zeros(2, 1, 64), ci, ci, ci[:2], 32)
    with pytest.raises(ValueError, match="GPU"):
        ops.qkv_norm_rope_split(torch.zeros(3, 768, dtype=torch.bfloat16), None, None, 1e-6, ci, *ops.rope_table(128, device="cpu"), 4, 1)


def test_scales_out_of_range(lib):
    """A scale or cap whose fp32 factors overflow would turn a score of 0 into NaN: refused."""
    for bad in (dict(cap=1e-40), dict(scale=3e38), dict(scale=1e30, cap=1e-9)):
        assert chunk(lib, **bad) == _lib.KIN_ERR_BAD_SHAPE, bad
    assert mass(lib, cap=1e-40) == _lib.KIN_ERR_BAD_SHAPE
    assert chunk(lib, cap=1e-30, nnz=0) == _lib.KIN_OK and chunk(lib, scale=1e30, nnz=0) == _lib.KIN_OK


def test_chunk_workspace_bytes_of_the_longest_page_list(lib):
    size = lib.kin_chunk_workspace_bytes
    for ps in (16, 128):
        assert size(1, 1, 4, 1, 2 ** 31 - 1, ps, 128, 0) == 4 * (64 * 129 + 1) * 4      # at most 64 spans
        assert size(10 ** 6, 1, 4, 1, 2 ** 31 - 1, ps, 128, 0) == 0                       # one span of all of it
