"""The steps between a layer's q/k/v projection and its output projection, as measurable cases.

* ``rope``: rotary positions of a matrix of heads, out of place.
* ``append``: keys and values of new tokens into a paged cache with the rotation on the way, queries rotated beside them; with the
  per-head norm of queries and keys or without it.
* ``attn``: attention of new tokens over the paged cache: single tokens, chunks, or both in one batch.
* ``step``: the append and the attention one after the other, as a layer runs them.

Sequences hold `lens` tokens, the last `news` of which are new. A token of a sequence of n is visible to the one at position p if it
is not behind it, and with a window w > 0 if it is fewer than w positions before it.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
THETA = 1e7


# ------------------------------------------------------------------ cases ---

def _rope(name, tokens, heads, dim, rot, interleaved=False, x16=False, out16=True, far=0, scaling="none"):
    return dict(name=name, kind="rope", tokens=tokens, heads=heads, dim=dim, rot=rot, interleaved=interleaved, x16=x16,
                out16=out16, far=far, scaling=scaling)


def _paged(name, kind, seqs, heads, kv_heads, dim, length, new, page=64, head_major=False, rot=0, norm=False, x16=False,
           window=0, ragged=True):
    return dict(name=name, kind=kind, seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, length=length, new=new, page=page,
                head_major=head_major, rot=rot, norm=norm, x16=x16, window=window, ragged=ragged)


def listed():
    return [
        # queries and keys of a single token: nothing but the latency of one call
        _rope("rope_token", 1, 40, 128, 128),
        # queries of a long prompt at far positions, frequencies stretched for a long context
        _rope("rope_prompt", 8192, 32, 128, 128, interleaved=True, x16=True, far=120000, scaling="yarn"),
        # one token of each of 48 streams: projections in f32, heads normed, a quarter of a head rotated
        _paged("append_tokens", "append", 48, 16, 4, 256, 2000, 1, page=64, rot=64, norm=True),
        # three ragged prompts written at once, projections in bf16, small pages
        _paged("append_prompts", "append", 3, 32, 8, 128, 2600, 2600, page=16, head_major=True, rot=128, x16=True),
        # single-stream decode with a short context: latency
        _paged("attn_token", "attn", 1, 32, 8, 128, 777, 1, page=16),
        # single-stream decode with a long context: the cache read once, by all of the chip
        _paged("attn_token_long", "attn", 1, 32, 8, 128, 130001, 1),
        # 64 streams with contexts of every length up to 12000
        _paged("attn_tokens", "attn", 64, 32, 8, 128, 12000, 1),
        # wide heads, as the layer widths of 4096 and 1024 have them with 256 per head
        _paged("attn_tokens_256", "attn", 24, 16, 4, 256, 9000, 1, page=128, head_major=True),
        # a chunk of a long prompt over what is cached of it
        _paged("attn_chunk", "attn", 1, 32, 8, 128, 33024, 1024),
        # a whole prompt, wide heads
        _paged("attn_prompt_256", "attn", 1, 16, 4, 256, 4096, 4096, page=32),
        # a batch of short ragged chunks over ragged contexts, in a layer with a sliding window
        _paged("attn_mixed", "attn", 9, 32, 8, 128, 3900, 300, page=16, window=1024),
        # the step of one layer for 32 streams: append, then attention
        _paged("step_tokens", "step", 32, 32, 8, 128, 4000, 1, rot=128, norm=True),
    ]


def _between(rng, lo, hi):
    """In [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rope", "append", "attn", "attn", "attn", "attn", "step"))
    dim = rng.choice((64, 96, 128, 128, 128, 192, 256, 256))
    rot = rng.choice((dim, dim, dim // 2, dim // 4))
    if kind == "rope":
        c = _rope("", _between(rng, 1, 8192), rng.randint(1, 32), dim, rot, rng.random() < 0.5, rng.random() < 0.5,
                  rng.random() < 0.6, rng.choice((0, 0, 5000, 120000, 1000000)),
                  rng.choice(("none", "none", "linear", "yarn")))
    else:
        kv_heads = rng.randint(1, 8)
        heads = kv_heads * rng.randint(1, 8)
        page = rng.choice((16, 16, 32, 48, 64, 64, 128, 256))
        how = rng.choice(("tokens", "tokens", "few", "chunk")) if kind != "append" else rng.choice(("tokens", "chunk"))
        if how == "tokens":
            seqs, new, length = _between(rng, 1, 96), 1, _between(rng, 1, 24000)
            length = max(1, min(length, 1000000 // seqs))
        elif how == "few":
            seqs, new, length = _between(rng, 1, 32), rng.randint(2, 8), _between(rng, 16, 12000)
            length = max(new, min(length, 300000 // seqs))
        else:
            seqs, new = _between(rng, 1, 6), _between(rng, 9, 2048)
            new = min(new, 6000 // seqs)
            length = max(new, min(_between(rng, 16, 24000), 40000000 // (seqs * new)))
        c = _paged("", kind, seqs, heads, kv_heads, dim, length, new, page, rng.random() < 0.5,
                   0 if kind == "attn" else rot, kind != "attn" and rng.random() < 0.5,
                   kind != "attn" and rng.random() < 0.5,
                   _between(rng, 128, 4096) if kind != "append" and rng.random() < 0.2 else 0, rng.random() < 0.8)
    del c["name"]
    return c


def lengths(c):
    """(tokens, new tokens) of each sequence: the first has `length` and `new`, the others of a ragged batch any share of them."""
    n = c["seqs"]
    if not c["ragged"]:
        return [c["length"]] * n, [c["new"]] * n
    share = [((i * 7919) % 1009) / 1009.0 for i in range(n)]
    news = [max(1, c["new"] - int(s * c["new"])) for s in share]
    lens = [max(w, c["length"] - int(((i * 4051) % 997) / 997.0 * c["length"])) for i, w in enumerate(news)]
    return lens, news


# ----------------------------------------------------------------- inputs ---

def frequencies(rot, scaling):
    """(radians a position of each pair, factor of the rotated values): the base's powers, or stretched for contexts four times as
    long: all of them, or by parts, the waves that fit 32 times into a context of 32768 as they are, those that do not fit once
    divided by four, a ramp between them."""
    pairs = rot // 2
    i = torch.arange(pairs, dtype=torch.float64)
    w = THETA ** (-2.0 * i / rot)
    if scaling == "linear":
        return w / 4.0, 1.0
    if scaling == "yarn":
        def pair_of(turns):
            return rot * math.log(32768 / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))
        lo, hi = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return w / 4.0 * ramp + w * (1.0 - ramp), 0.1 * math.log(4.0) + 1.0
    return w, 1.0


_runtime = []


def runtime():
    """The process's runtime, in encode-only mode: calls return once they are on the runtime's stream."""
    if not _runtime:
        from tessl_b200 import nn

        rt = nn.Runtime()
        rt.set_encode_only(True)
        _runtime.append(rt)
    return _runtime[0]


class _State:
    pass


def prepare(case, seed):
    c, s = case, _State()
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float32)
                * std).to(dtype)

    s.case = c
    s.inputs = torch.bfloat16 if c["x16"] else torch.float32
    if c["kind"] == "rope":
        s.x = normal(c["tokens"], c["heads"], c["dim"], dtype=s.inputs)
        s.positions = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
        s.positions += c["far"] + int(torch.randint(0, 1000, (1,), device="cuda", generator=gen))
        s.out = torch.zeros(s.x.shape, device="cuda", dtype=torch.bfloat16 if c["out16"] else torch.float32)
    else:
        lens, news = lengths(c)
        s.total, s.max_len, s.max_new = sum(news), max(lens), max(news)
        need = [-(-n // c["page"]) for n in lens]
        pages = sum(need)
        order = torch.randperm(pages, device="cuda", generator=gen, dtype=torch.int32)
        # a table of the longest sequence's width; what a shorter one does not use names its own first page
        s.width = max(need)
        at = torch.tensor(need).cumsum(0) - torch.tensor(need)
        col = torch.arange(s.width)[None, :].expand(c["seqs"], -1)
        s.table = order[(at[:, None] + torch.where(col < torch.tensor(need)[:, None], col, 0)).cuda()].contiguous()
        s.kv_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        s.starts = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32).cuda()
        shape = (pages, c["kv_heads"], c["page"], c["dim"]) if c["head_major"] else (pages, c["page"], c["kv_heads"], c["dim"])
        s.pages = pages
        s.k, s.v = normal(*shape, dtype=torch.bfloat16), normal(*shape, dtype=torch.bfloat16)
        s.q16 = torch.zeros(s.total, c["heads"], c["dim"], device="cuda", dtype=torch.bfloat16)
        if c["kind"] == "attn":
            s.q16 = normal(s.total, c["heads"], c["dim"], dtype=torch.bfloat16)
        else:  # a row of the fused projection: queries, keys, values
            s.qkv = normal(s.total, (c["heads"] + 2 * c["kv_heads"]) * c["dim"], dtype=s.inputs)
            s.q_norm, s.k_norm = normal(c["dim"], std=0.1), normal(c["dim"], std=0.1)
        s.out = torch.zeros(s.total, c["heads"], c["dim"], device="cuda", dtype=torch.bfloat16)
    if c["kind"] == "rope" or c["rot"]:
        w, s.factor = frequencies(c["rot"], c.get("scaling", "none"))
        s.w = w.cuda()
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


def _handles(s):
    """The library's views of the same memory, which a program keeps."""
    from tessl_b200 import nn

    c, rt, buf = s.case, runtime(), nn.GpuBuffer.from_torch
    s.rt = rt
    s.rope = None
    if c["kind"] == "rope" or c["rot"]:
        scaling = {"none": None, "linear": nn.RopeScaling("linear", 4.0),
                   "yarn": nn.RopeScaling("yarn", 4.0, 32768)}[c.get("scaling", "none")]
        s.rope = nn.rope_plan(rt, c["rot"], THETA, interleaved=c.get("interleaved", False), scaling=scaling)
    if c["kind"] == "rope":
        s.b_x, s.b_pos, s.b_out = buf(s.x), buf(s.positions), buf(s.out)
        return
    s.cache = nn.PagedKv(buf(s.k), buf(s.v), s.pages, c["page"], c["kv_heads"], c["dim"],
                         nn.KV_HEAD_MAJOR if c["head_major"] else nn.KV_TOKEN_MAJOR)
    s.seqs = nn.PagedSeqs(buf(s.table), buf(s.kv_lens), None if s.max_new == 1 else buf(s.starts), c["seqs"], s.width)
    s.b_q16, s.b_out = buf(s.q16), buf(s.out)
    if c["kind"] != "attn":
        b, size = buf(s.qkv), s.qkv.element_size()
        q, kv = c["heads"] * c["dim"] * size, c["kv_heads"] * c["dim"] * size
        rest = (s.total - 1) * (q + 2 * kv)
        s.row = s.qkv.shape[1]
        s.b_q, s.b_k, s.b_v = b.view(0, rest + q), b.view(q, rest + kv), b.view(q + kv, rest + kv)
        s.norms = nn.QkNorm(buf(s.q_norm), buf(s.k_norm), EPS) if c["norm"] else None
    if c["kind"] != "append":
        s.work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, s.total, c["heads"], s.cache, s.seqs))


# -------------------------------------------------------------------- run ---

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from tessl_b200 import nn

    c = s.case
    if c["kind"] == "rope":
        nn.rope(s.rt, s.b_x, s.b_pos, s.b_out, s.rope, c["tokens"], c["heads"], c["dim"], c["x16"], c["out16"])
        return s.out
    if c["kind"] != "attn":
        nn.kv_append_paged(s.rt, s.b_q, s.b_k, s.b_v, s.b_q16, s.cache, s.seqs, s.rope, s.norms, s.total, c["heads"],
                           s.row, s.row, s.row, c["x16"])
    if c["kind"] != "append":
        nn.attn_paged(s.rt, s.b_q16, s.cache, s.seqs, s.b_out, s.work, s.total, c["heads"], c["dim"] ** -0.5, True, c["window"])
    return _outputs(s)


def _outputs(s):
    kind = s.case["kind"]
    if kind == "attn":
        return s.out
    if kind == "append":
        return {"q": s.q16, "k": s.k, "v": s.v}
    return {"q": s.q16, "k": s.k, "v": s.v, "out": s.out}


def _rotate(x, positions, w, factor, interleaved):
    """x f32 [tokens, heads, dim]: the first 2 * len(w) of each head turned by position * w radians."""
    n = 2 * w.shape[0]
    angle = positions.double()[:, None] * w[None, :]
    cos, sin = ((f(angle) * factor).float()[:, None, :] for f in (torch.cos, torch.sin))
    r = x[..., :n]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., : n // 2], r[..., n // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((r, x[..., n:]), dim=-1)


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * (1.0 + weight)


def _places(s):
    """Of every new token: its sequence and its position there."""
    row = torch.arange(s.total, device="cuda")
    seq = torch.searchsorted(s.starts[1:].contiguous(), row, right=True)
    pos = s.kv_lens.long()[seq] - s.starts.long()[seq + 1] + row
    return seq, pos


def _run_plain(s):
    c = s.case
    if c["kind"] == "rope":
        s.out.copy_(_rotate(s.x.float(), s.positions, s.w, s.factor, c["interleaved"]))
        return s.out
    if c["kind"] != "attn":
        _append_plain(s)
    if c["kind"] != "append":
        _attend_plain(s)
    return _outputs(s)


def _append_plain(s):
    c = s.case
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    seq, pos = _places(s)
    x = s.qkv.float().view(s.total, h + 2 * kvh, d)
    q, k, v = x[:, :h], x[:, h:h + kvh], x[:, h + kvh:]
    if c["norm"]:
        q, k = _normed(q, s.q_norm), _normed(k, s.k_norm)
    s.q16.copy_(_rotate(q, pos, s.w, s.factor, False))
    k = _rotate(k, pos, s.w, s.factor, False).bfloat16()
    page, slot = s.table.long()[seq, pos // c["page"]], pos % c["page"]
    if c["head_major"]:
        s.k[page, :, slot], s.v[page, :, slot] = k, v.bfloat16()
    else:
        s.k[page, slot], s.v[page, slot] = k, v.bfloat16()


def _attend_plain(s):
    c = s.case
    n, h, kvh, d, page = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    j = torch.arange(s.max_len, device="cuda")
    pages, slot = s.table.long()[:, j // page], (j % page)[None, :].expand(n, -1)
    keys, values = ((t[pages, :, slot] if c["head_major"] else t[pages, slot]).float().transpose(1, 2) for t in (s.k, s.v))
    i = torch.arange(s.max_new, device="cuda")
    news = (s.starts[1:] - s.starts[:-1]).long()
    rows = s.starts[:-1].long()[:, None] + i[None, :]  # [n, max_new]
    live = i[None, :] < news[:, None]
    q = s.q16[rows.clamp(max=s.total - 1)].float().view(n, s.max_new, kvh, h // kvh, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kvh, (h // kvh) * s.max_new, d)
    scores = (q @ keys.transpose(2, 3)).view(n, kvh, h // kvh, s.max_new, s.max_len).mul_(d ** -0.5)
    pos = (s.kv_lens.long() - news)[:, None] + i[None, :]
    seen = (j[None, None, :] <= pos[:, :, None])
    if c["window"]:
        seen &= j[None, None, :] > pos[:, :, None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    o = (scores.view(n, kvh, -1, s.max_len) @ values).view(n, kvh, h // kvh, s.max_new, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s.max_new, h, d)
    s.out[rows[live]] = o[live].bfloat16()


# ------------------------------------------------------------------- work ---

def work(case):
    c = case
    if c["kind"] == "rope":
        values = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": values * ((2 if c["x16"] else 4) + (2 if c["out16"] else 4)) + 4 * c["tokens"],
                "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    lens, news = lengths(c)
    h, kvh, d, w = c["heads"], c["kv_heads"], c["dim"], c["window"]
    total, pages = sum(news), sum(-(-n // c["page"]) for n in lens)
    nbytes = flops = 0
    if c["kind"] != "attn":
        values = total * (h + 2 * kvh) * d
        nbytes += values * (2 if c["x16"] else 4) + values * 2 + 4 * (total + pages)
        flops += total * (h + kvh) * (3 * c["rot"] + (4 * d if c["norm"] else 0))
    if c["kind"] != "append":
        nbytes += 2 * total * h * d * 2 + 4 * pages
        for n, m in zip(lens, news):
            first = n - m  # position of the first new token
            if w == 0:
                seen, reach = m * first + m * (m + 1) // 2, n
            else:
                full = max(0, n - max(first, w))  # rows that see a whole window
                part = range(first, n - full)
                seen, reach = full * w + sum(p + 1 for p in part), n - max(0, first + 1 - w)
            nbytes += 2 * reach * kvh * d * 2
            flops += 4 * seen * h * d
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ exact ---

def exact(case, seed):
    """The definitions, one sequence and one key head at a time, in 64 bits. What the cache and the queries hold in bf16 is part of
    the step's definition: its attention reads those."""
    global own
    c = case
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    f64 = torch.float64

    def turned(x, positions):
        """Pair i of a head as a complex number, times factor * exp(i angle)."""
        n = 2 * s.w.shape[0]
        turn = torch.polar(torch.full_like(s.w, s.factor)[None].expand(len(positions), -1).contiguous(), positions.to(f64)[:, None] * s.w)
        first = torch.arange(0, n, 2, device="cuda") if c.get("interleaved") else torch.arange(n // 2, device="cuda")
        second = first + (1 if c.get("interleaved") else n // 2)
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None, :]
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if c["kind"] == "rope":
        return turned(s.x.to(f64), s.positions)
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    lens, news = lengths(c)
    starts = [0]
    for m in news:
        starts.append(starts[-1] + m)
    caches = {"k": s.k.to(f64) if c["kind"] != "attn" else s.k, "v": s.v.to(f64) if c["kind"] != "attn" else s.v}
    q_of = s.q16.to(f64)

    def slots(b, first, last):
        p = torch.arange(first, last, device="cuda")
        return s.table[b].long()[p // c["page"]], p % c["page"]

    if c["kind"] != "attn":
        for b in range(c["seqs"]):
            x = s.qkv[starts[b]:starts[b + 1]].to(f64).view(news[b], h + 2 * kvh, d)
            q, k, v = x.split((h, kvh, kvh), dim=1)
            if c["norm"]:
                q, k = (t / (t.square().sum(-1, keepdim=True) / d + EPS).sqrt() * (1 + g.to(f64)) for t, g in ((q, s.q_norm), (k, s.k_norm)))
            at = torch.arange(lens[b] - news[b], lens[b], device="cuda")
            q_of[starts[b]:starts[b + 1]] = turned(q, at)
            page, slot = slots(b, lens[b] - news[b], lens[b])
            for name, t in (("k", turned(k, at)), ("v", v)):
                if c["head_major"]:
                    caches[name][page, :, slot] = t
                else:
                    caches[name][page, slot] = t
    if c["kind"] == "append":
        return {"q": q_of, **caches}
    out = torch.zeros(s.total, h, d, device="cuda", dtype=f64)
    g = h // kvh
    for b in range(c["seqs"]):
        page, slot = slots(b, 0, lens[b])
        pos = torch.arange(lens[b] - news[b], lens[b], device="cuda").repeat_interleave(g)
        j = torch.arange(lens[b], device="cuda")
        hidden = j[None, :] > pos[:, None]
        if c["window"]:
            hidden |= j[None, :] <= pos[:, None] - c["window"]
        for e in range(kvh):
            k, v = ((caches[n][page, e, slot] if c["head_major"] else caches[n][page, slot, e]).bfloat16().to(f64) for n in ("k", "v"))
            q = q_of[starts[b]:starts[b + 1], e * g:(e + 1) * g].bfloat16().to(f64).reshape(-1, d)
            z = (q @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[starts[b]:starts[b + 1], e * g:(e + 1) * g] = (torch.softmax(z, dim=-1) @ v).view(news[b], g, d)
    if c["kind"] == "attn":
        return out
    return {"q": q_of, **caches, "out": out}
