"""What stands between a layer's q/k/v and output projections, as measurable cases.

Every case is a dict of plain values; its "kind" names the operator:

  rope    RMS norm of each query and key head and the position rotation, fp32 rows in and out
  append  keys and values of new tokens into a paged cache of e4m3 codes with one power-of-two scale for each page and head,
          the key's norm and rotation applied on the way; "q" says that the queries are normed and rotated in the same call
  attend  causal attention of each sequence's newest rows over that cache, optionally over a window of the latest keys

A batch has "seqs" sequences of ragged lengths up to "kv" tokens, of which up to "rows" each are the call's own; "idle" adds a
sequence without tokens or rows, as a serving program's unused slot.  Lengths follow from the case alone, values and the order of
pages from the seed.  All of it is made on the GPU.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
# query heads, key/value heads, head width
H06 = {"hq": 16, "hkv": 8, "d": 128}   # a 0.6B model's layer
H8 = {"hq": 32, "hkv": 8, "d": 128}    # an 8B model's layer
H64 = {"hq": 14, "hkv": 2, "d": 64}    # a small model with seven query heads to a key head
H256 = {"hq": 8, "hkv": 4, "d": 256}   # wide heads


def listed():
    return [
        # one decoded token of a 0.6B model: latency
        {"name": "rope_decode_0.6b", "kind": "rope", "rows": 1, **H06, "norm": True, "rot": 128, "pairs": False, "far": 4096},
        # a prompt through an 8B layer: bandwidth
        {"name": "rope_prompt_4096", "kind": "rope", "rows": 4096, **H8, "norm": True, "rot": 128, "pairs": False, "far": 4096},
        # an odd number of rows far into a long context, half of each head rotated as neighbouring pairs
        {"name": "rope_far_77", "kind": "rope", "rows": 77, **H64, "norm": False, "rot": 32, "pairs": True, "far": 1000000},
        # one decoded token of one user: query, key and value in one call
        {"name": "append_decode_0.6b", "kind": "append", "seqs": 1, "kv": 301, "rows": 1, **H06, "page": 64, "norm": True,
         "rot": 128, "pairs": False, "q": True, "vhalf": True, "idle": False},
        # a decode step of 64 users, each in the middle of a page
        {"name": "append_decode_64_users", "kind": "append", "seqs": 64, "kv": 2048, "rows": 1, **H8, "page": 16, "norm": False,
         "rot": 128, "pairs": True, "q": True, "vhalf": False, "idle": True},
        # three ragged prompts behind cached prefixes
        {"name": "append_prompts", "kind": "append", "seqs": 3, "kv": 2500, "rows": 2048, **H8, "page": 64, "norm": True,
         "rot": 128, "pairs": False, "q": False, "vhalf": False, "idle": False},
        # a conversation's first words: latency
        {"name": "attend_short_0.6b", "kind": "attend", "seqs": 1, "kv": 40, "rows": 1, **H06, "page": 64, "window": 0,
         "half": False, "idle": False},
        # a decode step of 64 users with ragged contexts: bandwidth
        {"name": "attend_decode_64_users", "kind": "attend", "seqs": 64, "kv": 8192, "rows": 1, **H8, "page": 64, "window": 0,
         "half": False, "idle": True},
        # one user far into a long document: the work has to be split along the cache
        {"name": "attend_long_131072", "kind": "attend", "seqs": 1, "kv": 131072, "rows": 1, **H8, "page": 64, "window": 0,
         "half": False, "idle": False},
        # checking drafts of up to five tokens for 16 users, wide heads, a sliding window
        {"name": "attend_verify_5", "kind": "attend", "seqs": 16, "kv": 3001, "rows": 5, **H256, "page": 32, "window": 1024,
         "half": False, "idle": False},
        # prefill of one prompt for the matrix-core projections, which take bf16: bound by the products
        {"name": "attend_prompt_4096", "kind": "attend", "seqs": 1, "kv": 4096, "rows": 4096, **H8, "page": 64, "window": 0,
         "half": True, "idle": False},
        # ragged chunks of three prompts behind long prefixes, in fp32
        {"name": "attend_chunks_500", "kind": "attend", "seqs": 3, "kv": 6001, "rows": 500, **H64, "page": 16, "window": 0,
         "half": False, "idle": True},
    ]


def _log(rng, lo, hi):
    """An integer from [lo, hi], its logarithm spread evenly."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST_TOKENS = 64 * 8192 * 8 * 128  # cached values of the 64 users' decode step
MOST_PAIRS = 32 * 4096 * 4096 * 128  # query rows times keys times width of the 4096-token prompt


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend"])
    heads = dict(rng.choice([H06, H8, H64, H256, {"hq": 8, "hkv": 8, "d": 64}, {"hq": 24, "hkv": 2, "d": 128}]))
    width = heads["hkv"] * heads["d"]
    rot = rng.choice([heads["d"], heads["d"], heads["d"] // 2])
    turn = {"norm": rng.random() < 0.5, "rot": rot, "pairs": rng.random() < 0.5}
    if kind == "rope":
        return {"kind": kind, "rows": _log(rng, 1, 4096), **heads, **turn, "far": _log(rng, 4096, 1000000)}
    seqs = rng.choice([1, 1, _log(rng, 2, 100)])
    page = rng.choice([16, 32, 64])
    idle = rng.random() < 0.3
    if kind == "append":
        rows = rng.choice([1, _log(rng, 2, 8), min(_log(rng, 9, 4096), max(9, 6000 // seqs))])
        kv = min(rows + _log(rng, 1, 8192), max(rows, (1 << 27) // (seqs * width)))
        return {"kind": kind, "seqs": seqs, "kv": kv, "rows": rows, **heads, "page": page, **turn, "q": rng.random() < 0.5,
                "vhalf": rng.random() < 0.5, "idle": idle}
    kv = min(_log(rng, 1, 131072), max(1, MOST_TOKENS // (seqs * width)))
    rows = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 4096)])
    rows = max(1, min(rows, kv, MOST_PAIRS // (seqs * heads["hq"] * kv * heads["d"])))
    return {"kind": kind, "seqs": seqs, "kv": kv, "rows": rows, **heads, "page": page,
            "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "half": rng.random() < 0.5, "idle": idle}


def _lengths(c):
    """(rows, tokens) of each sequence: the first has the most of both, the others down to a quarter."""
    rows = [max(1, int(c["rows"] * (1 - 0.75 * (s * 0.4142 % 1)))) for s in range(c["seqs"])]
    lens = [max(rows[s], int(c["kv"] * (1 - 0.75 * (s * 0.618 % 1)))) for s in range(c["seqs"])]
    if c["idle"]:  # an unused slot in the middle of the batch
        at = c["seqs"] // 2
        rows.insert(at, 0)
        lens.insert(at, 0)
    return rows, lens


# ---------------------------------------------------------------- inputs

class _State:
    def __init__(self, case):
        self.case, self.kept = case, None


def _normal(shape, g, strong=0.0):
    x = torch.randn(*shape, device="cuda", generator=g)
    if strong:
        x = x * torch.where(torch.rand(shape[-1], device="cuda", generator=g) < 0.02, strong, 1.0)
    return x


def _inputs(case, seed):
    """The tensors of a case by name, from the seed alone (prepare() and exact() share it)."""
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, d = {}, c["d"]
    if c["kind"] != "attend":
        t["freq"] = (10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])).float()
        if c["norm"]:
            t["qw"] = torch.rand(d, device="cuda", generator=g) + 0.5
            t["kw"] = torch.rand(d, device="cuda", generator=g) + 0.5
    if c["kind"] == "rope":
        R = c["rows"]
        # q and k are columns of one projection's output
        t["qk"] = _normal((R, (c["hq"] + c["hkv"]) * d), g, 8.0)
        t["pos"] = torch.randint(0, c["far"], (R,), device="cuda", generator=g, dtype=torch.int32)
        return t
    rows, lens = _lengths(c)
    P, S, R = c["page"], len(rows), sum(rows)
    need = [-(-n // P) for n in lens]
    pages, wide = sum(need) + 3, max(need) + 1
    order = torch.randperm(pages, device="cuda", generator=g).int()
    need_t = torch.tensor(need, device="cuda")
    first = torch.cumsum(need_t, 0) - need_t
    col = torch.arange(wide, device="cuda")[None, :]
    # columns behind a sequence's pages hold -1, as a serving program leaves them
    t["table"] = torch.where(col < need_t[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).int().contiguous()
    t["len"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
    t["start"] = torch.tensor([sum(rows[:s]) for s in range(S + 1)], device="cuda", dtype=torch.int32)
    for n in ("k", "v"):
        codes = torch.empty(pages, c["hkv"], P, d, device="cuda", dtype=torch.float8_e4m3fn)
        step = max(1, (1 << 28) // (c["hkv"] * P * d))  # in pieces, so that the fp32 values fit easily
        for a in range(0, pages, step):
            b = min(pages, a + step)
            codes[a:b] = (_normal((b - a, c["hkv"], P, d), g) * 60.0).clamp(-448, 448).to(torch.float8_e4m3fn)
        t[n + "c"] = codes
        t[n + "s"] = torch.exp2(torch.randint(-7, -4, (pages, c["hkv"]), device="cuda", generator=g).float())
    if c["kind"] == "attend":
        t["q"] = _normal((R, c["hq"] * d), g) * 2.0
    else:
        t["k"] = _normal((R, c["hkv"] * d), g, 8.0)
        v = _normal((R, c["hkv"] * d), g)
        t["v"] = v.half() if c["vhalf"] else v
        if c["q"]:
            t["q"] = _normal((R, c["hq"] * d), g, 8.0)
    return t


def prepare(case, seed):
    s = _State(case)
    s.t = _inputs(case, seed)
    c = case
    if c["kind"] == "rope":
        s.qo = torch.empty(c["rows"], c["hq"] * c["d"], device="cuda")
        s.ko = torch.empty(c["rows"], c["hkv"] * c["d"], device="cuda")
    elif c["kind"] == "attend":
        s.out = torch.empty(*s.t["q"].shape, device="cuda", dtype=torch.bfloat16 if c["half"] else torch.float32)
    elif c["q"]:
        s.qo = torch.empty_like(s.t["q"])
    return s


# ---------------------------------------------------------------- the plain forms

def _turned(x, heads, pos, c, w, freq):
    """Rows of heads, normed where w is given, rotated to their positions."""
    x = x.reshape(x.shape[0], heads, c["d"])
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    angle = pos.double()[:, None] * freq.double()
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    rot, h = c["rot"], c["rot"] // 2
    if c["pairs"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _places(t, R):
    """Sequence, position and index within the sequence of each of the R rows."""
    row = torch.arange(R, device="cuda")
    seq = torch.bucketize(row, t["start"][1:].long(), right=True)
    within = row - t["start"][seq]
    n = (t["start"][1:] - t["start"][:-1])[seq]
    return seq, t["len"][seq] - n + within, within


def _grow(codes, scale, x, page, offset, first):
    """Writes x [R, heads, d] at (page, offset); each touched page and head gets the scale that its old and new values need."""
    peak = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    m, e = torch.frexp(peak)
    need = torch.exp2((e - torch.where(m <= 0.875, 9, 8)).clamp(min=-100).float())
    need = torch.where(peak > 0, need, torch.full_like(need, 2.0 ** -100))
    head = offset == first  # the first new row of each page
    p, kept = page[head], first[head]
    old = torch.where(kept[:, None] > 0, scale[p], torch.zeros_like(scale[p]))
    new = torch.maximum(old, need[p])
    was = codes[p].float() * (old / new)[:, :, None, None]
    keep = torch.arange(codes.shape[2], device="cuda")[None, :] < kept[:, None]
    codes[p] = torch.where(keep[:, None, :, None], was, codes[p].float()).to(codes.dtype)
    scale[p] = new
    heads = torch.arange(x.shape[1], device="cuda")
    codes[page[:, None], heads[None, :], offset[:, None]] = (x / scale[page][:, :, None]).to(codes.dtype)


def _plain_append(s):
    c, t = s.case, s.t
    R, P = t["k"].shape[0], c["page"]
    seq, pos, within = _places(t, R)
    page = t["table"][seq, pos // P].long()
    offset = pos % P
    first = torch.clamp(offset - within, min=0)  # where the call's own rows begin in this page
    k = _turned(t["k"], c["hkv"], pos, c, t.get("kw"), t["freq"])
    _grow(t["kc"], t["ks"], k, page, offset, first)
    _grow(t["vc"], t["vs"], t["v"].float().reshape(R, c["hkv"], c["d"]), page, offset, first)
    if c["q"]:
        s.qo = _turned(t["q"], c["hq"], pos, c, t.get("qw"), t["freq"]).reshape(R, -1)


def _plain_attend(s):
    c, t = s.case, s.t
    R, P, S = t["q"].shape[0], c["page"], t["len"].shape[0]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    seq, pos, within = _places(t, R)
    most, wide = c["rows"], -(-max(_lengths(c)[1]) // P)
    table = t["table"][:, :wide].clamp(min=0).long()

    def read(n):  # [sequences, heads, tokens, d]
        x = t[n + "c"][table].float() * t[n + "s"][table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(S, hkv, wide * P, d)
    q = torch.zeros(S, hkv, hq // hkv, most, d, device="cuda")
    at = torch.full((S, most), -1, device="cuda", dtype=pos.dtype)
    q[seq, :, :, within] = t["q"].reshape(R, hkv, hq // hkv, d)
    at[seq, within] = pos
    score = torch.matmul(q.reshape(S, hkv, -1, d), read("k").transpose(2, 3).contiguous()) * d ** -0.5
    score = score.reshape(S, hkv, hq // hkv, most, wide * P)
    key = torch.arange(wide * P, device="cuda")
    seen = key[None, None] <= at[:, :, None]
    if c["window"]:
        seen &= key[None, None] > at[:, :, None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.reshape(S, hkv, -1, wide * P), read("v")).reshape(S, hkv, hq // hkv, most, d)
    out = out / torch.where(total == 0, 1.0, total)
    return out[seq, :, :, within].reshape(R, hq * d).to(s.out.dtype)


# ---------------------------------------------------------------- one pass

def _handles(s):
    """The buffers, views and kernels that a program keeps beside its tensors."""
    from edgerunner_amd import (Buffer, HeadRows, KV8AppendKernel, KV8AttentionKernel, KV8Batch, KV8Cache, QKNormRopeKernel,
                                Rope, default_context)
    from edgerunner_amd._ffi import er_buffer
    ctx, c, t, k = default_context(), s.case, s.t, {}

    def buf(x):
        return Buffer(ctx, er_buffer(x.data_ptr(), x.numel() * x.element_size()), owned=False)

    def optional(name):
        return buf(t[name]) if name in t else None
    if c["kind"] != "attend":
        k["rope"] = Rope(buf(t["freq"]), c["rot"], c["pairs"])
        k["qw"], k["kw"] = optional("qw"), optional("kw")
    if c["kind"] == "rope":
        width, each = (c["hq"] + c["hkv"]) * c["d"], c["hq"] * c["d"]
        both = buf(t["qk"])
        k["kernel"] = QKNormRopeKernel(ctx)
        k["q"], k["k"] = HeadRows(both, c["hq"], width), HeadRows(both.view(4 * each), c["hkv"], width)
        k["qo"], k["ko"] = HeadRows(buf(s.qo), c["hq"], each), HeadRows(buf(s.ko), c["hkv"], c["hkv"] * c["d"])
        k["pos"] = buf(t["pos"])
        return k
    rows, lens = _lengths(c)
    k["cache"] = KV8Cache(buf(t["kc"]), buf(t["vc"]), buf(t["ks"]), buf(t["vs"]), t["kc"].shape[0], c["hkv"], c["page"], c["d"])
    k["batch"] = KV8Batch(buf(t["table"]), buf(t["len"]), buf(t["start"]), len(rows), t["table"].shape[1], sum(rows), max(rows),
                          max(lens))
    if c["kind"] == "append":
        k["kernel"] = KV8AppendKernel(ctx)
        k["k"], k["v"] = HeadRows(buf(t["k"]), c["hkv"], c["hkv"] * c["d"]), HeadRows(buf(t["v"]), c["hkv"], c["hkv"] * c["d"])
        k["q"] = HeadRows(buf(t["q"]), c["hq"], c["hq"] * c["d"]) if c["q"] else None
        k["qo"] = HeadRows(buf(s.qo), c["hq"], c["hq"] * c["d"]) if c["q"] else None
    else:
        k["kernel"] = KV8AttentionKernel(ctx)
        k["q"], k["out"] = HeadRows(buf(t["q"]), c["hq"], c["hq"] * c["d"]), HeadRows(buf(s.out), c["hq"], c["hq"] * c["d"])
        k["scratch"] = ctx.alloc(max(16, k["kernel"].workspaceBytes(k["cache"], k["batch"], c["hq"])))
    return k


def run(s):
    c = s.case
    if own:
        if s.kept is None:
            s.kept = _handles(s)
        k = s.kept
        if c["kind"] == "rope":
            k["kernel"].encode(None, k["q"], k["k"], k["qo"], k["ko"], k["pos"], c["rows"], c["d"], k["rope"], k["qw"], k["kw"],
                               EPS)
        elif c["kind"] == "append":
            k["kernel"].encode(None, k["cache"], k["batch"], k["k"], k["v"], k["rope"], kNorm=k["kw"], q=k["q"], qOut=k["qo"],
                               qNorm=k["qw"] if c["q"] else None, eps=EPS, vHalf=c["vhalf"])
        else:
            k["kernel"].encode(None, k["cache"], k["batch"], k["q"], k["out"], c["d"] ** -0.5, window=c["window"],
                               workspace=k["scratch"], outBF16=c["half"])
    elif c["kind"] == "rope":
        each = c["hq"] * c["d"]
        pos, qk = s.t["pos"], s.t["qk"]
        s.qo = _turned(qk[:, :each], c["hq"], pos, c, s.t.get("qw"), s.t["freq"]).reshape(c["rows"], -1)
        s.ko = _turned(qk[:, each:], c["hkv"], pos, c, s.t.get("kw"), s.t["freq"]).reshape(c["rows"], -1)
    elif c["kind"] == "append":
        _plain_append(s)
    else:
        s.out = _plain_attend(s)
    if c["kind"] == "rope":
        return {"q": s.qo, "k": s.ko}
    if c["kind"] == "attend":
        return {"out": s.out}
    out = {n: s.t[n] for n in ("kc", "ks", "vc", "vs")}
    return {**out, "q": s.qo} if c["q"] else out


# ---------------------------------------------------------------- what a pass cannot do without

def _seen(c):
    """(keys that some row of the sequence reaches, pairs of a row and a key) over all sequences."""
    keys = pairs = 0
    for n, m in zip(*_lengths(c)):
        w = c["window"] or m
        keys += min(m, n + w - 1) if n else 0
        full = max(0, min(n, m - w))  # rows that see a whole window
        pairs += full * w + sum(m - n + i + 1 for i in range(n - full))
    return keys, pairs


def work(case):
    c = case
    if c["kind"] == "rope":
        values = c["rows"] * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": 8 * values, "flops": 10 * values}
    rows, lens = _lengths(c)
    R = sum(rows)
    if c["kind"] == "append":
        values = R * c["hkv"] * c["d"]
        nbytes = values * (4 + (2 if c["vhalf"] else 4) + 2) + (8 * R * c["hq"] * c["d"] if c["q"] else 0)
        return {"bytes": nbytes, "flops": 20 * values}
    keys, pairs = _seen(c)
    return {"bytes": 2 * keys * c["hkv"] * c["d"] + R * c["hq"] * c["d"] * (4 + (2 if c["half"] else 4)),
            "flops": 4 * pairs * c["hq"] * c["d"]}


# ---------------------------------------------------------------- the same in 64 bits

def _rotate64(x, pos, c, w, freq):
    """One row at a time is one matrix: each pair of columns turns by its angle.  x [R, H, d]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["d"] + EPS) * w.double()
    y = x.clone()
    for i in range(c["rot"] // 2):
        a, b = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + c["rot"] // 2)
        z = torch.polar(torch.ones_like(pos, dtype=torch.float64), pos.double() * freq[i].double())[:, None]
        turned = torch.complex(x[..., a], x[..., b]) * z
        y[..., a], y[..., b] = turned.real, turned.imag
    return y


def _code64(x):
    """The e4m3 value nearest to each x of up to 448 in size, ties to the even one: three bits behind the first, steps of 2^-9 at the least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    c, t, d = case, _inputs(case, seed), case["d"]
    if c["kind"] == "rope":
        x = t["qk"].reshape(c["rows"], -1, d)
        return {"q": _rotate64(x[:, :c["hq"]], t["pos"], c, t.get("qw"), t["freq"]).flatten(1),
                "k": _rotate64(x[:, c["hq"]:], t["pos"], c, t.get("kw"), t["freq"]).flatten(1)}
    rows, lens = _lengths(c)
    P, hkv, G = c["page"], c["hkv"], c["hq"] // c["hkv"]
    pos = torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(rows, lens)])
    if c["kind"] == "append":
        R, out = len(pos), {}
        new = {"k": _rotate64(t["k"].reshape(R, hkv, d), pos, c, t.get("kw"), t["freq"]), "v": t["v"].reshape(R, hkv, d).double()}
        for n in ("k", "v"):
            # the codes' values, in units of the page's scale
            values, scale = t[n + "c"].double(), t[n + "s"].double()
            row = 0
            for s, (count, m) in enumerate(zip(rows, lens)):
                for p in range((m - count) // P, -(-m // P)) if count else ():
                    page, a, b = int(t["table"][s, p]), max(m - count, p * P), min(m, p * P + P)
                    x = new[n][row + a - (m - count):row + b - (m - count)].transpose(0, 1)  # [heads, tokens, d]
                    peak = x.abs().amax((1, 2)) / 448
                    grown = torch.exp2(torch.ceil(torch.log2(peak.clamp(min=2.0 ** -100))))
                    old = scale[page].clone() if a > p * P else torch.zeros_like(grown)
                    scale[page] = torch.maximum(old, grown)
                    values[page, :, :a - p * P] = _code64(values[page, :, :a - p * P] * (old / scale[page])[:, None, None])
                    values[page, :, a - p * P:b - p * P] = _code64(x / scale[page][:, None, None])
                row += count
            out[n + "c"], out[n + "s"] = values, scale
        if c["q"]:
            out["q"] = _rotate64(t["q"].reshape(R, -1, d), pos, c, t.get("qw"), t["freq"]).flatten(1)
        return out
    parts = []
    row = 0
    for s, (n, m) in enumerate(zip(rows, lens)):
        if not n:
            continue
        pages = t["table"][s, :-(-m // P)].long()
        o = torch.empty(n, c["hq"], d, device="cuda", dtype=torch.float64)
        at = torch.arange(m - n, m, device="cuda")[:, None]
        key = torch.arange(m, device="cuda")[None]
        hidden = (key > at) | (key <= at - (c["window"] or m + 1))
        for h in range(hkv):
            k, v = ((t[x + "c"][pages, h].double() * t[x + "s"][pages, h].double()[:, None, None]).flatten(0, 1)[:m] for x in "kv")
            q = t["q"][row:row + n].reshape(n, c["hq"], d)[:, h * G:(h + 1) * G].double()
            for g in range(G):
                p = torch.softmax((q[:, g] @ k.T.contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                o[:, h * G + g] = p @ v
        parts.append(o.flatten(1))
        row += n
    return {"out": torch.cat(parts)}
