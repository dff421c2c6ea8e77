"""Measured cases of the serving operators around a paged KV cache: attention of a chunk of new tokens, the weight that
each cached token received, eviction by that weight, and the q/k norm + split with rotary positions of several axes.

``own`` false: the operators in plain torch operations, in 32 bits; true: the calls a serving program makes."""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# --------------------------------------------------------------------------------------------------------- the cases

def _chunk(name, lens, news, hq, hkv, d, page, dtype, **mods):
    """lens: tokens per sequence after the append; news: how many of them are new."""
    c = dict(name=name, op="chunk", lens=",".join(map(str, lens)), news=",".join(map(str, news)), hq=hq, hkv=hkv, d=d, page=page,
             dtype=dtype, softcap=0.0, window=0, slopes=False, prefix=0, offset=0)
    c.update(mods)
    return c


def _mass(name, lens, news, hq, hkv, d, page, dtype, **mods):
    return dict(_chunk(name, lens, news, hq, hkv, d, page, dtype, **mods), op="mass")


def _evict(name, lens, hkv, d, page, dtype, budget, sink, local, offset=0):
    return dict(name=name, op="evict", lens=",".join(map(str, lens)), hkv=hkv, d=d, page=page, dtype=dtype, budget=budget, sink=sink,
                local=local, offset=offset)


def _rope(name, tokens, hq, hkv, d, dtype, sections, interleaved, far, norm=True):
    return dict(name=name, op="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, dtype=dtype, sections=",".join(map(str, sections)),
                interleaved=interleaved, far=far, norm=norm)


def _spread(n, lo, hi, step):
    """n lengths between lo and hi, in no order, most of them odd."""
    return [lo + (i * step) % (hi - lo + 1) for i in range(n)]


def listed():
    return [
        # the smallest call: 8 sequences of up to 4096 tokens take one token each (latency counts)
        _chunk("chunk: 8 single tokens", _spread(8, 513, 4097, 1031), [1] * 8, 4, 1, 128, 16, "bf16"),
        # continuous batching: 60 sequences decode while 4 prompts enter in chunks, all in one call
        _chunk("chunk: 60 decode + 4 prefill", _spread(60, 301, 8201, 2311) + [512, 2048, 1203, 700], [1] * 60 + [512, 512, 203, 37], 32, 8, 64, 16, "f16"),
        # a chunk of a long prompt on the one-GPU share of a tensor-parallel model: 2048 new tokens behind 30720 cached ones
        _chunk("chunk: 2048 after 30720", [32768], [2048], 4, 1, 128, 16, "bf16"),
        # a whole prompt of 8192 tokens with every head on one GPU
        _chunk("chunk: 8192 from nothing", [8192], [8192], 32, 8, 128, 16, "bf16"),
        # capped scores and a sliding window, large pages, groups of 8
        _chunk("chunk: capped, window 1024", [9001, 6007], [2047, 1023], 32, 4, 128, 64, "bf16", softcap=50.0, window=1024),
        # distance bias with a prefix that sees itself whole (an image in front of the text), odd sizes
        _chunk("chunk: distance bias, prefix", [2111, 777, 1500], [1111, 777, 300], 12, 2, 64, 32, "f16", slopes=True, prefix=577),
        # one token each of 256 sequences: how much weight every cached token received
        _mass("mass: 256 single tokens", _spread(256, 1025, 8193, 3001), [1] * 256, 4, 1, 128, 16, "bf16"),
        # the weights of a whole chunk of a prompt, scores capped
        _mass("mass: 2048 after 6144", [8192], [2048], 32, 8, 128, 16, "bf16", softcap=30.0),
        # long contexts cut to 4096 tokens per head after their prompts
        _evict("evict: 4 x 16384 to 4096", [16384, 16001, 12345, 16384], 8, 128, 16, "bf16", 4096, 4, 64),
        # a serving batch whose slots have outgrown their budget by one block each; some have not
        _evict("evict: 96 x 1100 to 1024", _spread(96, 900, 1160, 37), 1, 128, 16, "f16", 1024, 4, 32),
        # one decode step of the large batch: one token per sequence, text positions on one axis
        _rope("rope: 4096 tokens, one axis", 4096, 4, 1, 128, "bf16", [64], False, 40960),
        # a prompt with images and video: time, height and width, far positions, every head
        _rope("rope: 8191 tokens, three axes", 8191, 32, 8, 128, "bf16", [24, 20, 20], True, 1000000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "mass", "evict", "rope"])
    d, dtype, page = rng.choice([64, 128]), rng.choice(["bf16", "f16"]), rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "rope":
        axes = rng.choice([1, 2, 3])
        cut = sorted(rng.sample(range(1, d // 2), axes - 1))
        sections = [b - a for a, b in zip([0] + cut, cut + [d // 2])]
        return _rope("", _log(rng, 1, 8000), hq, hkv, d, dtype, sections, rng.random() < 0.5, _log(rng, 1000, 2000000), rng.random() < 0.8)
    if op == "evict":
        sink, local = rng.choice([0, 1, 4]), rng.choice([0, 1, 17, 64])
        budget = sink + local + _log(rng, 1, 4000)
        n = _log(rng, 1, max(1, 40000 // (budget + 600)))
        lens = [max(1, rng.randint(budget // 2, 3 * budget)) for _ in range(n)]
        return _evict("", lens, hkv, d, page, dtype, budget, sink, local, rng.choice([0, 0, 12]))
    mods = dict(softcap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, _log(rng, 1, 3000)]), slopes=rng.random() < 0.3,
                prefix=rng.choice([0, 0, _log(rng, 1, 1000)]), offset=rng.choice([0, 0, 12]))
    if rng.random() < 0.5:  # single tokens, now and then a few
        n = _log(rng, 1, 64)
        news = [rng.choice([1, 1, 1, rng.randint(0, 9)]) for _ in range(n)]
        lens = [max(k, _log(rng, 1, 16000)) for k in news]
    else:  # chunks of prompts
        n = rng.randint(1, 4)
        news = [_log(rng, 2, 1500) for _ in range(n)]
        lens = [k + rng.choice([0, _log(rng, 1, 9000)]) for k in news]
    return (_chunk if op == "chunk" else _mass)("", lens, news, hq, hkv, d, page, dtype, **mods)


def _ints(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------------------------------------------ their inputs

def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(case, g):
    """A paged cache with its page table, pages in no order and a few of them unused."""
    lens, page, off = _ints(case["lens"]), case["page"], case["offset"]
    counts = [(n + off + page - 1) // page for n in lens]
    total = sum(counts) + 5
    ids = torch.randperm(total, device=DEV, generator=g)[: sum(counts)].to(torch.int32)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    shape = (total, 2, page, case["hkv"], case["d"])
    kv = torch.empty(shape, dtype=DT[case["dtype"]], device=DEV)
    kv.normal_(generator=g)
    kv[:, 0] *= 1.0 + torch.rand(case["hkv"], case["d"], device=DEV, generator=g).to(kv.dtype)  # keys have louder channels
    return dict(lens=lens, counts=counts, starts=starts, kv=kv, ids=ids, indptr=_i32(starts),
                last=_i32([n + off - (c - 1) * page for n, c in zip(lens, counts)]), max_pages=max(counts))


def _heads(case, s, g):
    news, hq, d = _ints(case["news"]), case["hq"], case["d"]
    ends = [0]
    for n in news:
        ends.append(ends[-1] + n)
    q = torch.empty(ends[-1], hq, d, dtype=DT[case["dtype"]], device=DEV)
    q.normal_(generator=g)
    s.update(news=news, ends=ends, q=q, q_indptr=_i32(ends), slopes=None, prefix=None,
             scale=1.0 / math.sqrt(d), mods=dict(softcap=case["softcap"], window=case["window"], first_page_offset=case["offset"]))
    if case["slopes"]:
        s["slopes"] = 2.0 ** (-8.0 * (torch.arange(hq, device=DEV, dtype=torch.float32) + 1) / hq)
    if case["prefix"]:
        s["prefix"] = _i32([min(n, case["prefix"] + 3 * i) for i, n in enumerate(s["lens"])])
    s["mods"].update(slopes=s["slopes"], prefix_lens=s["prefix"])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    if op == "rope":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        sections = _ints(case["sections"])
        dt = DT[case["dtype"]]
        s = dict(case=case, qkv=torch.randn(t, (hq + 2 * hkv) * d, device=DEV, generator=g).mul_(2.0).to(dt), qw=None, kw=None)
        if case["norm"]:
            s["qw"] = (1.0 + 0.2 * torch.randn(d, device=DEV, generator=g)).to(dt)
            s["kw"] = (1.0 + 0.2 * torch.randn(d, device=DEV, generator=g)).to(dt)
        s["pos"] = torch.randint(0, case["far"], (len(sections), t), device=DEV, generator=g, dtype=torch.int32)
        s["inv"], s["axis"] = _frequencies(d, sections, case["interleaved"])
        if own:
            from kinetics_amd import ops

            s["freq"], s["freq_axis"] = ops.rope_table(d, theta=THETA, sections=sections, interleaved=case["interleaved"], device=DEV)
        return s
    s = _cache(case, g)
    s["case"] = case
    top = max(s["lens"])
    if op == "evict":
        # what tokens gathered over a while: most very little, some a great deal
        s["scores"] = torch.empty(len(s["lens"]), case["hkv"], top + 7, device=DEV).normal_(generator=g).mul_(2.0).exp_()
        if own:
            s["scores_out"] = s["scores"].clone()
        return s
    _heads(case, s, g)
    if op == "mass":
        s["scores"] = torch.rand(len(s["lens"]), case["hkv"], top + 7, device=DEV, generator=g)
        s["lse"] = _plain_attention(s)[1]
    elif own:
        from kinetics_amd import ops

        need = ops.chunk_workspace_bytes(s["q"].shape[0], len(s["lens"]), case["hq"], case["hkv"], s["max_pages"], case["page"], case["d"])
        s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    return s


# --------------------------------------------------------------------------------------------------- the plain forms

THETA = 1000000.0


def _frequencies(d, sections, interleaved):
    """Radians per position of every pair (i, i + d/2), and the axis whose position turns it."""
    inv = THETA ** (-torch.arange(d // 2, device=DEV, dtype=torch.float64) * 2 / d)
    if not interleaved:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    else:  # the axes in turn, as long as they have pairs left
        left, axis = list(sections), []
        while len(axis) < d // 2:
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    axis.append(a)
    return inv, torch.tensor(axis, device=DEV)


def _rows(s, b):
    """Keys and values of sequence b, [Hkv, tokens, D] in 32 bits."""
    kv, off, n = s["kv"], s["case"]["offset"], s["lens"][b]
    pages = kv[s["ids"][s["starts"][b]:s["starts"][b + 1]].long()]
    flat = pages.transpose(0, 1).reshape(2, -1, kv.shape[3], kv.shape[4])[:, off:off + n]
    return flat[0].float().transpose(0, 1).contiguous(), flat[1].float().transpose(0, 1).contiguous()


def _plain_scores(s, b, h, k):
    """Scores of the new tokens of sequence b under KV head h, [group, new, tokens]; -inf where a token is not seen."""
    c = s["case"]
    group, n, length = c["hq"] // c["hkv"], s["news"][b], s["lens"][b]
    q = s["q"][s["ends"][b]:s["ends"][b + 1], h * group:(h + 1) * group].float().transpose(0, 1).reshape(group * n, c["d"])
    x = (q @ k[h].t()).view(group, n, length) * s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    at = torch.arange(length - n, length, device=DEV)[:, None]
    j = torch.arange(length, device=DEV)[None, :]
    if s["slopes"] is not None:
        x = x - s["slopes"][h * group:(h + 1) * group, None, None] * (at - j).abs()
    seen = j <= at
    if c["window"]:
        seen = seen & (at - j < c["window"])
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"][b])
    return x.masked_fill(~seen, float("-inf"))


def _plain_attention(s):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    out = torch.zeros_like(s["q"])
    lse = torch.full(s["q"].shape[:2], float("-inf"), device=DEV)
    for b, n in enumerate(s["news"]):
        if n == 0:
            continue
        k, v = _rows(s, b)
        rows = slice(s["ends"][b], s["ends"][b + 1])
        for h in range(c["hkv"]):
            heads = slice(h * group, (h + 1) * group)
            x = _plain_scores(s, b, h, k)
            m = x.amax(-1, keepdim=True)
            p = torch.exp(x - m)
            total = p.sum(-1, keepdim=True)
            o = (p.view(group * n, -1) @ v[h]).view(group, n, -1) / total
            out[rows, heads] = o.transpose(0, 1).to(out.dtype)
            lse[rows, heads] = (m + torch.log(total))[..., 0].t()
    return out, lse


def _plain_mass(s):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    for b, n in enumerate(s["news"]):
        if n == 0:
            continue
        k, _ = _rows(s, b)
        lse = s["lse"][s["ends"][b]:s["ends"][b + 1]]
        for h in range(c["hkv"]):
            x = _plain_scores(s, b, h, k)
            w = torch.exp(x - lse[:, h * group:(h + 1) * group].t()[..., None])
            s["scores"][b, h, :s["lens"][b]] += w.sum((0, 1))
    return s["scores"]


def _plain_evict(s):
    c = s["case"]
    kv, budget, sink, local, off, page = s["kv"], c["budget"], c["sink"], c["local"], c["offset"], c["page"]
    scores = s["scores"].clone()
    kept = torch.full((len(s["lens"]), c["hkv"], budget), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(s["lens"]):
        if n <= budget:
            kept[b, :, :n] = torch.arange(n, device=DEV)
            continue
        x = s["scores"][b, :, :n]
        best = sink + torch.argsort(x[:, sink:n - local], dim=1, descending=True, stable=True)[:, :budget - sink - local]
        fixed = torch.cat([torch.arange(sink, device=DEV), torch.arange(n - local, n, device=DEV)]).expand(c["hkv"], -1)
        src = torch.cat([best, fixed], 1).sort(1).values                      # [Hkv, budget], ascending
        kept[b] = src.to(torch.int32)
        ids = s["ids"][s["starts"][b]:s["starts"][b + 1]].long()
        dst = torch.arange(budget, device=DEV).expand_as(src)
        heads = torch.arange(c["hkv"], device=DEV)[:, None]
        rows = kv[ids[(src + off) // page], :, (src + off) % page, heads]     # [Hkv, budget, 2, D]
        kv[ids[(dst + off) // page], :, (dst + off) % page, heads] = rows
        scores[b, :, :budget] = x.gather(1, src)
        scores[b, :, budget:n] = 0
    return dict(kv=kv, kept=kept, scores=scores, lens=torch.tensor([min(n, budget) for n in s["lens"]], dtype=torch.int32, device=DEV))


def _plain_rope(s):
    c = s["case"]
    t, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    x = s["qkv"].view(t, hq + 2 * hkv, d)
    qk = x[:, :hq + hkv].float()
    if c["norm"]:
        w = torch.cat([s["qw"].float().expand(hq, d), s["kw"].float().expand(hkv, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    angle = s["pos"].double()[s["axis"]].t() * s["inv"]                       # [tokens, d/2], 64 bits: positions are far
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    lo, hi = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(x.dtype)
    return qk[:, :hq].contiguous(), qk[:, hq:].contiguous(), x[:, hq + hkv:].contiguous()


# ----------------------------------------------------------------------------------------------------------- a pass

def run(s):
    c = s["case"]
    if not own:
        return {"chunk": _plain_attention, "mass": _plain_mass, "evict": _plain_evict, "rope": _plain_rope}[c["op"]](s)
    from kinetics_amd import ops

    if c["op"] == "chunk":
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
        out = ops.paged_chunk_attention(s["q"], s["kv"], s["q_indptr"], s["ids"], s["indptr"], s["last"], s["max_pages"], lse=lse,
                                        workspace=s["workspace"], **s["mods"])
        return out, lse
    if c["op"] == "mass":
        ops.attention_mass(s["q"], s["kv"], s["lse"], s["scores"], s["q_indptr"], s["ids"], s["indptr"], s["last"], s["max_pages"],
                           **s["mods"])
        return s["scores"]
    if c["op"] == "evict":
        kept, lens = ops.evict_tokens(s["kv"], s["scores"], s["ids"], s["indptr"], s["last"], c["budget"], sink_tokens=c["sink"],
                                      local_tokens=c["local"], first_page_offset=c["offset"], scores_out=s["scores_out"])
        return dict(kv=s["kv"], kept=kept, scores=s["scores_out"], lens=lens)
    return ops.qkv_norm_rope_split(s["qkv"], s["qw"], s["kw"], 1e-6, s["pos"], s["freq"], s["freq_axis"], c["hq"], c["hkv"])


def _pairs(case):
    """(query, key) pairs that are seen, and the keys that any query sees."""
    pairs = keys = 0
    for b, (length, n) in enumerate(zip(_ints(case["lens"]), _ints(case["news"]))):
        w = case["window"] or length
        prefix = min(length, case["prefix"] + 3 * b) if case["prefix"] else 0
        for p in range(length - n, length):
            lo = max(0, p - w + 1)
            pairs += p + 1 - lo + min(prefix, lo) + max(0, prefix - p - 1)
        if n:
            first = max(0, length - n - w + 1)
            keys += length - first + min(prefix, first)
    return pairs, keys


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * (case["hq"] + 2 * case["hkv"]) * case["d"]
        axes = len(_ints(case["sections"]))
        return {"bytes": 4 * n + 4 * axes * case["tokens"], "flops": 8 * n}
    hkv, d = case["hkv"], case["d"]
    if case["op"] == "evict":
        read = moved = 0
        for n in _ints(case["lens"]):
            read += n if n > case["budget"] else 0
            moved += case["budget"] - case["sink"] if n > case["budget"] else 0
        return {"bytes": hkv * (8 * read + 4 * case["budget"] * len(_ints(case["lens"])) + moved * 2 * 2 * d * 2), "flops": 0}
    pairs, keys = _pairs(case)
    rows = sum(_ints(case["news"])) * case["hq"]
    if case["op"] == "mass":
        return {"bytes": rows * (2 * d + 4) + keys * hkv * (2 * d + 8), "flops": 2 * d * case["hq"] * pairs}
    return {"bytes": rows * (4 * d + 4) + keys * hkv * 4 * d, "flops": 4 * d * case["hq"] * pairs}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits

def _token(s, b, t):
    """Where token t of sequence b lies: (page, slot)."""
    at = t + s["case"]["offset"]
    return s["ids"].long()[s["starts"][b] + at // s["case"]["page"]], at % s["case"]["page"]


def _exact_weights(s, b, head, first, count):
    """Scores of `count` rows from row `first` of sequence b for one query head, float64, and the seen tokens' mask."""
    c = s["case"]
    length = s["lens"][b]
    h = head // (c["hq"] // c["hkv"])
    tokens = torch.arange(length, device=DEV)
    page, slot = _token(s, b, tokens)
    k = s["kv"][page, 0, slot, h].double()
    q = s["q"][s["ends"][b] + first:s["ends"][b] + first + count, head].double()
    x = torch.mm(q, k.t()) / math.sqrt(c["d"])
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    p = (length - s["news"][b] + first + torch.arange(count, device=DEV)).unsqueeze(1)
    dist = p - tokens
    if c["slopes"]:
        x -= s["slopes"][head].double() * dist.abs()
    see = (dist >= 0) & (dist < (c["window"] or length + 1))
    if c["prefix"]:
        see |= (tokens < min(length, c["prefix"] + 3 * b)).unsqueeze(0)
    return torch.where(see, x, torch.full_like(x, -math.inf)), (page, slot, h)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    if c["op"] == "rope":
        t, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
        x = s["qkv"].double().reshape(t, -1, d)
        parts = []
        for heads, w in ((x[:, :hq], s["qw"]), (x[:, hq:hq + hkv], s["kw"])):
            if w is not None:
                heads = heads / torch.sqrt((heads * heads).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            z = torch.complex(heads[..., :d // 2], heads[..., d // 2:])
            turn = torch.stack([s["pos"][int(a)].double() * float(f) for a, f in zip(s["axis"], s["inv"])], 1)
            z = z * torch.polar(torch.ones_like(turn), turn)[:, None]
            parts.append(torch.cat([z.real, z.imag], -1))
        return parts[0], parts[1], x[:, hq + hkv:].contiguous()
    if c["op"] == "evict":
        kv, scores = s["kv"].double(), s["scores"].double()
        was_kv, was_scores = kv.clone(), scores.clone()
        for b, n in enumerate(s["lens"]):
            if n <= c["budget"]:
                continue
            for h in range(c["hkv"]):
                x = was_scores[b, h, :n].clone()
                x[:c["sink"]] = math.inf
                x[n - c["local"]:] = math.inf
                cut = torch.topk(x, c["budget"]).values[-1]
                over = x > cut
                same = (x == cut) & ((x == cut).cumsum(0) <= c["budget"] - over.sum())
                src = torch.nonzero(over | same)[:, 0]
                (sp, ss), (dp, ds) = _token(s, b, src), _token(s, b, torch.arange(c["budget"], device=DEV))
                kv[dp, :, ds, h] = was_kv[sp, :, ss, h]
                scores[b, h, :n] = 0
                scores[b, h, :c["budget"]] = was_scores[b, h, src]
        return dict(kv=kv, kept=None, scores=scores, lens=None)
    nnz, hq, d = s["q"].shape
    if c["op"] == "mass":
        scores = s["scores"].double()
        lse = s["lse"].double()
    out = torch.zeros(nnz, hq, d, dtype=torch.float64, device=DEV)
    total = torch.full((nnz, hq), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["news"]):
        for head in range(hq):
            for first in range(0, n, 4096):
                count = min(4096, n - first)
                x, (page, slot, h) = _exact_weights(s, b, head, first, count)
                rows = slice(s["ends"][b] + first, s["ends"][b] + first + count)
                if c["op"] == "mass":
                    scores[b, h, :s["lens"][b]] += torch.exp(x - lse[rows, head].unsqueeze(1)).sum(0)
                else:
                    z = torch.logsumexp(x, 1)
                    total[rows, head] = z
                    out[rows, head] = torch.mm(torch.exp(x - z.unsqueeze(1)), s["kv"][page, 1, slot, h].double())
    return scores if c["op"] == "mass" else (out, total)
