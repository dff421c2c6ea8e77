"""Plain float64 forms of the chunk operators (attention of a chunk, the weight it gave, eviction, the rotary split)
and seeded problems for them, for the GPU tests.  Straight from the definitions, one sequence and head at a time."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def problem(seed, lens, news, hq=4, hkv=1, d=128, page=16, dtype="bf16", offset=0, extra_pages=3, tail_rows=0, device="cuda"):
    """A paged cache holding ``lens`` tokens per sequence, the last ``news`` of them new; pages in random order."""
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    counts = [(n + offset + page - 1) // page if n else 0 for n in lens]
    total = sum(counts) + extra_pages
    ids = torch.randperm(total, generator=g)[: sum(counts)].to(torch.int32)
    starts, ends = [0], [0]
    for c, n in zip(counts, news):
        starts.append(starts[-1] + c)
        ends.append(ends[-1] + n)
    kv = torch.randn(total, 2, page, hkv, d, generator=g)
    kv[:, 1] += 0.25
    q = 1.5 * torch.randn(ends[-1] + tail_rows, hq, d, generator=g)
    last = [n + offset - (c - 1) * page if c else 1 for n, c in zip(lens, counts)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return SimpleNamespace(lens=list(lens), news=list(news), counts=counts, starts=starts, ends=ends, hq=hq, hkv=hkv, d=d, page=page,
                           offset=offset, dt=dt, kv=kv.to(dt).to(device), q=q.to(dt).to(device), ids=ids.to(device), ptr=i32(starts),
                           last=i32(last), q_indptr=i32(ends), max_pages=max(counts + [1]), device=device, total_pages=total)


def slot_of(pb, b, t):
    """(page, slot) of tokens ``t`` of sequence b."""
    at = t + pb.offset
    return pb.ids.long()[pb.starts[b] + at // pb.page], at % pb.page


def scores(pb, b, head, softcap=0.0, window=0, slopes=None, prefix_lens=None, sm_scale=0.0):
    """float64 scores [new, tokens] of one query head (-inf: not seen), and how far fp32 arithmetic may be off on one."""
    n, length, dev = pb.news[b], pb.lens[b], pb.q.device
    h = head // (pb.hq // pb.hkv)
    tok = torch.arange(length, device=dev)
    page, slot = slot_of(pb, b, tok)
    k = pb.kv[page, 0, slot, h].double()
    q = pb.q[pb.ends[b]:pb.ends[b + 1], head].double()
    scale = sm_scale if sm_scale > 0 else 1.0 / math.sqrt(pb.d)
    s = (q @ k.t()) * scale
    # products of 16-bit elements are exact in fp32; d of them are summed (d roundings at most), then scaled
    off = (pb.d + 4) * 2.0 ** -24 * float(torch.nan_to_num((q.abs() @ k.abs().t()), 0, 0, 0).max() if n and length else 0.0) * scale
    if softcap > 0:
        s = softcap * torch.tanh(s / softcap)
        off += softcap * 2.0 ** -21       # tanh: 3 units in the last place, two products
    p = (length - n + torch.arange(n, device=dev))[:, None]
    dist = p - tok[None, :]
    if slopes is not None:
        s = s - float(slopes[head]) * dist.abs()
    seen = (dist >= 0) & ((dist < window) if window else torch.ones_like(dist, dtype=torch.bool))
    if prefix_lens is not None:
        seen = seen | (tok[None, :] < min(max(int(prefix_lens[b]), 0), length))
    seen = seen & (p >= 0)
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    if slopes is not None and bool(seen.any()):
        # the bias is rounded at the size of the score it makes; scores far below the row's largest have no weight
        top = s.amax(1, keepdim=True)
        near = torch.where(seen & (s > top - 60), s.abs(), torch.zeros_like(s)).max()
        off += 3 * 2.0 ** -24 * (float(near) + float(slopes[head]) * float(torch.where(seen & (s > top - 60), dist.abs(), 0).max()))
    return s, off, (page, slot, h)


def attention(pb, **mods):
    """(out, lse, bound of |out error|, bound of |lse error|) in float64; rows of no sequence are NaN."""
    rows = pb.q.shape[0]
    out = torch.full((rows, pb.hq, pb.d), math.nan, dtype=torch.float64, device=pb.q.device)
    lse = torch.full((rows, pb.hq), math.nan, dtype=torch.float64, device=pb.q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    half = torch.finfo(pb.dt).eps / 2
    for b, n in enumerate(pb.news):
        for head in range(pb.hq if n else 0):
            s, off, (page, slot, h) = scores(pb, b, head, **mods)
            r = slice(pb.ends[b], pb.ends[b + 1])
            if s.shape[1] == 0:
                out[r, head], lse[r, head] = 0.0, -math.inf
                continue
            z = torch.logsumexp(s, 1)
            w = torch.where(s > -math.inf, torch.exp(s - z[:, None]), torch.zeros_like(s))
            v = pb.kv[page, 1, slot, h].double()
            out[r, head] = w @ torch.nan_to_num(v, 0, 0, 0)
            lse[r, head] = z
            mag = w @ torch.nan_to_num(v, 0, 0, 0).abs()
            # a weight: off by 2 * off relatively (score and maximum), rounded once to the element type (and in float16 never
            # finer than 2^-25 of the largest weight); exp2, the sums and the quotient: 2^-18; the result: rounded once
            tol[r, head] = (half * (1 + 2.0 ** -6) + 2 * off + 2.0 ** -18) * mag + half * out[r, head].abs() + 1e-30
            if pb.dt is torch.float16:
                tol[r, head] += 2.0 ** -25 * (w > 0).double() @ torch.nan_to_num(v, 0, 0, 0).abs() + 2.0 ** -25
            ltol[r, head] = off + 2.0 ** -20 * (1 + torch.nan_to_num(z, 0, 0, 0).abs())
    return out, lse, tol, ltol


def mass(pb, lse, start, blocks=None, **mods):
    """(scores, bound) in float64 after the chunk's weights were added to ``start``; ``lse`` as the operator is given it."""
    out = start.double().clone()
    tol = torch.zeros_like(out)
    for b, n in enumerate(pb.news):
        blk = b if blocks is None else blocks[b]
        if n == 0 or not 0 <= blk < out.shape[0] or pb.lens[b] > out.shape[2]:
            continue
        for head in range(pb.hq):
            s, off, (_, _, h) = scores(pb, b, head, **mods)
            z = lse[pb.ends[b]:pb.ends[b + 1], head].double()[:, None]
            w = torch.where((s > -math.inf) & (z > -math.inf), torch.exp(s - z), torch.zeros_like(s)).sum(0)
            big = float(torch.nan_to_num(z, 0, 0, 0).abs().max()) + 1.0
            out[blk, h, :pb.lens[b]] += w
            # a weight: its score's error, the roundings of score and lse in log2 units, exp2
            tol[blk, h, :pb.lens[b]] += w * (off + 2.0 ** -21 * big)
    group = pb.hq // pb.hkv
    n_max = max(pb.news + [1]) * group
    return out, tol + (n_max / 32 + 24) * 2.0 ** -24 * out.abs() + 1e-30     # at most rows / 32 + 16 + a few additions


def evict(pb, sc, budget, sink, local, blocks=None):
    """(kv, scores, kept, new_lens) after the eviction, from the definition."""
    kv, out = pb.kv.clone(), sc.clone()
    kept = torch.full((len(pb.lens), pb.hkv, budget), -1, dtype=torch.int32, device=sc.device)
    new = []
    for b, n in enumerate(pb.lens):
        blk = b if blocks is None else blocks[b]
        known = 0 <= blk < sc.shape[0] and n <= sc.shape[2]
        new.append(min(n, budget) if known else n)
        if not known:
            continue
        for h in range(pb.hkv):
            if n <= budget:
                kept[b, h, :n] = torch.arange(n, dtype=torch.int32, device=sc.device)
                continue
            x = sc[blk, h, :n].tolist()
            mid = sorted(range(sink, n - local), key=lambda i: (-math.inf if math.isnan(x[i]) else -x[i], 0 if math.isnan(x[i]) else 1, i))
            keep = sorted(list(range(sink)) + mid[:budget - sink - local] + list(range(n - local, n)))
            src = torch.tensor(keep, device=sc.device)
            kept[b, h] = src.to(torch.int32)
            (sp, ss), (dp, ds) = slot_of(pb, b, src), slot_of(pb, b, torch.arange(budget, device=sc.device))
            kv[dp, :, ds, h] = pb.kv[sp, :, ss, h]
            out[blk, h, :n] = 0
            out[blk, h, :budget] = sc[blk, h, src]
    return kv, out, kept, torch.tensor(new, dtype=torch.int32, device=sc.device)


def rope(qkv, qw, kw, eps, positions, inv_freq, axis, hq, hkv, d):
    """(q, k, v) in float64; inv_freq: Python floats; axis: list of ints (-1: not turned)."""
    t = qkv.shape[0]
    x = qkv.double().reshape(t, hq + 2 * hkv, d)
    pos = positions.reshape(-1, t).tolist()
    cos = torch.ones(t, d // 2, dtype=torch.float64)
    sin = torch.zeros(t, d // 2, dtype=torch.float64)
    for i in range(d // 2):
        if 0 <= axis[i] < len(pos):
            for r in range(t):
                a = math.fmod(pos[axis[i]][r] * inv_freq[i], 2 * math.pi)
                cos[r, i], sin[r, i] = math.cos(a), math.sin(a)
    cos, sin = cos.to(qkv.device)[:, None], sin.to(qkv.device)[:, None]
    parts = []
    for heads, w in ((x[:, :hq], qw), (x[:, hq:hq + hkv], kw)):
        if w is not None:
            heads = heads * torch.rsqrt((heads ** 2).mean(-1, keepdim=True) + eps) * w.double()
        lo, hi = heads[..., :d // 2], heads[..., d // 2:]
        parts.append(torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1))
    return parts[0], parts[1], x[:, hq + hkv:]
