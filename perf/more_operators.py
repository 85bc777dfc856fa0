"""What a step that drafts tokens, streams without end or answers under rules needs beside the cache's operators, as measurable cases.

Every case is a dict of plain values; its "kind" names the operator:

  attend  attention over the paged cache of e4m3 codes where not every earlier token is visible: a "window" of the latest tokens and the
          first "sinks" ones, or (where "tree") the tokens before the call's rows and, among the rows, each one's ancestors in a tree of
          drafted tokens and itself; window and sinks may join a tree
  accept  the walk down a tree of drafted tokens along the chosen ones, and the moves that leave the cache with the kept ones alone
  choose  penalties for tokens of the context, biases and a mask of allowed tokens on logits, and the largest that is left

A batch has "seqs" sequences of ragged lengths up to "kv" tokens, of which up to "rows" each are the call's own; "idle" adds a
sequence without tokens or rows, as a serving program's unused slot.  Lengths follow from the case alone; values, trees and the order
of pages from the seed.  All of it is made on the GPU.
"""
from __future__ import annotations

import math

import torch

own = False

# query heads, key/value heads, head width
H06 = {"hq": 16, "hkv": 8, "d": 128}   # a 0.6B model's layer
H8 = {"hq": 32, "hkv": 8, "d": 128}    # an 8B model's layer
H64 = {"hq": 14, "hkv": 2, "d": 64}    # a small model with seven query heads to a key head
H256 = {"hq": 8, "hkv": 4, "d": 256}   # wide heads


def listed():
    return [
        # one user of a 0.6B model far into an endless stream: a window and the first tokens; latency
        {"name": "sinks_one_131072", "kind": "attend", "tree": False, "seqs": 1, "kv": 131072, "rows": 1, **H06, "page": 64,
         "window": 1020, "sinks": 4, "half": False, "idle": False},
        # a decode step of 48 users with ragged streams behind a long window: bandwidth
        {"name": "sinks_decode_48_users", "kind": "attend", "tree": False, "seqs": 48, "kv": 20000, "rows": 1, **H8, "page": 64,
         "window": 8192, "sinks": 4, "half": False, "idle": True},
        # a chunk of a prompt behind what came before it, for the matrix-core projections: bound by the products
        {"name": "sinks_chunk_2048", "kind": "attend", "tree": False, "seqs": 1, "kv": 12001, "rows": 2048, **H8, "page": 32,
         "window": 4096, "sinks": 16, "half": True, "idle": False},
        # one user's tree of 26 drafts in a short conversation: latency
        {"name": "tree_26_one_user", "kind": "attend", "tree": True, "seqs": 1, "kv": 1001, "rows": 26, **H06, "page": 64,
         "window": 0, "sinks": 0, "half": False, "idle": False},
        # ragged trees of 32 users: 128 columns of a key head, one pass over each cache
        {"name": "tree_32_users", "kind": "attend", "tree": True, "seqs": 32, "kv": 6000, "rows": 32, **H8, "page": 16,
         "window": 0, "sinks": 0, "half": False, "idle": True},
        # trees of 64 nodes over long documents, for projections that take bf16
        {"name": "tree_64_long", "kind": "attend", "tree": True, "seqs": 4, "kv": 40001, "rows": 64, **H64, "page": 64,
         "window": 0, "sinks": 0, "half": True, "idle": False},
        # what one user keeps of 26 drafts: latency
        {"name": "accept_one_user", "kind": "accept", "seqs": 1, "kv": 1001, "rows": 26, **H06, "page": 64, "idle": False},
        # what 64 users keep of up to 64 drafts each
        {"name": "accept_64_users", "kind": "accept", "seqs": 64, "kv": 2500, "rows": 64, **H8, "page": 16, "idle": True},
        # one user's next token under penalties: latency
        {"name": "choose_one_user", "kind": "choose", "seqs": 1, "rows": 1, "vocab": 151936, "past": 301, "penal": True, "bias": 0,
         "allowed": False, "tree": False, "write": False, "idle": False},
        # a decode step of 64 users, each with penalties, a few biases and a grammar
        {"name": "choose_64_users", "kind": "choose", "seqs": 64, "rows": 1, "vocab": 128256, "past": 4096, "penal": True, "bias": 100,
         "allowed": True, "tree": False, "write": True, "idle": True},
        # every node of 8 users' trees under its own state of the grammar, the path to it in its context
        {"name": "choose_trees_256", "kind": "choose", "seqs": 8, "rows": 32, "vocab": 128256, "past": 1500, "penal": True, "bias": 0,
         "allowed": True, "tree": True, "write": True, "idle": False},
        # a small odd vocabulary, masks alone
        {"name": "choose_masked_5", "kind": "choose", "seqs": 5, "rows": 1, "vocab": 32003, "past": 0, "penal": False, "bias": 0,
         "allowed": True, "tree": False, "write": False, "idle": False},
    ]


def _log(rng, lo, hi):
    """An integer from [lo, hi], its logarithm spread evenly."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST_TOKENS = 48 * 8192 * 8 * 128  # cached values that the 48 users' decode step reads
MOST_PAIRS = 32 * 2048 * 4096 * 128  # query rows times visible keys times width of the prompt's chunk
MOST_LOGITS = 256 * 128256


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "accept", "choose", "choose"])
    seqs, idle = rng.choice([1, 1, _log(rng, 2, 64)]), rng.random() < 0.3
    if kind == "choose":
        tree = rng.random() < 0.4
        rows = _log(rng, 2, 64) if tree else 1
        vocab = _log(rng, 1000, 200000)
        seqs = max(1, min(seqs, MOST_LOGITS // (vocab * rows)))
        return {"kind": kind, "seqs": seqs, "rows": rows, "vocab": vocab, "past": rng.choice([0, _log(rng, 1, 8192)]),
                "penal": rng.random() < 0.7, "bias": rng.choice([0, _log(rng, 1, 300)]), "allowed": rng.random() < 0.6, "tree": tree,
                "write": rng.random() < 0.6, "idle": idle}
    heads = dict(rng.choice([H06, H8, H64, H256, {"hq": 8, "hkv": 8, "d": 64}, {"hq": 24, "hkv": 2, "d": 128}]))
    width, page = heads["hkv"] * heads["d"], rng.choice([16, 32, 64])
    if kind == "accept":
        rows = _log(rng, 2, 128)
        kv = rows + min(_log(rng, 1, 8192), max(1, (1 << 27) // (seqs * width)))
        return {"kind": kind, "seqs": seqs, "kv": kv, "rows": rows, **heads, "page": page, "idle": idle}
    tree = rng.random() < 0.5
    window = rng.choice([0, _log(rng, 16, 4096)]) if tree else _log(rng, 16, 8192)
    sinks = rng.choice([0, 1, 4, _log(rng, 2, 200)]) if tree else rng.choice([1, 4, _log(rng, 2, 200)])
    kv = min(_log(rng, 1, 131072), max(1, (1 << 30) // (seqs * width)))  # what the pool holds
    seen = min(kv, window + sinks) if window else kv
    if seqs * seen * width > MOST_TOKENS:
        kv = seen = max(1, MOST_TOKENS // (seqs * width))
    rows = _log(rng, 2, 128) if tree else rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 2048)])
    rows = max(1, min(rows, kv, MOST_PAIRS // (seqs * heads["hq"] * seen * heads["d"])))
    return {"kind": kind, "tree": tree, "seqs": seqs, "kv": kv, "rows": rows, **heads, "page": page, "window": window, "sinks": sinks,
            "half": rng.random() < 0.5, "idle": idle}


def _lengths(c):
    """(rows, tokens) of each sequence: the first has the most of both, the others down to a quarter."""
    rows = [max(1, int(c["rows"] * (1 - 0.75 * (s * 0.4142 % 1)))) for s in range(c["seqs"])]
    most = c["past"] if c["kind"] == "choose" else c["kv"]
    lens = [int(most * (1 - 0.75 * (s * 0.618 % 1))) for s in range(c["seqs"])]
    if c["kind"] != "choose":  # the rows are the newest tokens
        lens = [max(r, m) for r, m in zip(rows, lens)]
    if c["idle"]:  # an unused slot in the middle of the batch
        at = c["seqs"] // 2
        rows.insert(at, 0)
        lens.insert(at, 0)
    return rows, lens


# ---------------------------------------------------------------- inputs

class _State:
    def __init__(self, case):
        self.case, self.kept = case, None


def _normal(shape, g):
    return torch.randn(*shape, device="cuda", generator=g)


def _words(bits):
    """Truth values [..., n] as 32-bit words [..., ceil(n / 32)], the first the lowest bit."""
    n = bits.shape[-1]
    padded = torch.zeros(*bits.shape[:-1], -(-n // 32) * 32, device=bits.device, dtype=torch.int64)
    padded[..., :n] = bits
    words = (padded.unflatten(-1, (-1, 32)) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def _trees(rows, g, vocab):
    """Trees of the rows of each sequence, as a drafting program hands them over: parents (-1 for a sequence's first row, else an
    earlier row of it), tokens, and for each row the rows that it sees, its ancestors and itself."""
    S, most, R = len(rows), max(rows), sum(rows)
    i = torch.arange(most, device="cuda")
    parent = torch.clamp((torch.rand(S, most, device="cuda", generator=g, dtype=torch.float64) * i).long(), max=most - 1)
    parent[:, 0] = -1
    up = torch.nn.functional.one_hot(parent.clamp(min=0), most).double()
    up[:, 0] = 0
    seen = torch.matrix_power(up + torch.eye(most, device="cuda", dtype=torch.float64), most) > 0
    live = i[None] < torch.tensor(rows, device="cuda")[:, None]
    token = torch.randint(0, vocab, (R,), device="cuda", generator=g, dtype=torch.int32)
    return {"parent": parent[live].int(), "token": token, "seen": _words(seen[live]), "depth": (seen[live].sum(-1) - 1).int()}


def _starts(rows):
    return torch.tensor([sum(rows[:s]) for s in range(len(rows) + 1)], device="cuda", dtype=torch.int32)


def _inputs(case, seed):
    """The tensors of a case by name, from the seed alone (prepare() and exact() share it)."""
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, lens = _lengths(c)
    S, R = len(rows), sum(rows)
    t = {"start": _starts(rows), "len": torch.tensor(lens, device="cuda", dtype=torch.int32)}
    if c["kind"] == "choose":
        V = c["vocab"]
        t["logits"] = _normal((R, V), g) * 3.0
        if c["tree"]:
            t |= _trees(rows, g, V)
        if c["penal"]:
            # a text's tokens: few of them often
            t["past"] = (torch.rand(S, max(1, c["past"]), device="cuda", generator=g) ** 4 * V).int().clamp(max=V - 1)
            spread = torch.tensor([[0.3, 0.6, 0.2]], device="cuda")
            t["penalty"] = torch.tensor([[1.0, 0.0, 0.0]], device="cuda") + spread * torch.rand(S, 3, device="cuda", generator=g)
        if c["bias"]:
            t["bias_token"] = torch.randint(0, V, (S, c["bias"]), device="cuda", generator=g, dtype=torch.int32)
            t["bias"] = _normal((S, c["bias"]), g) * 4.0
            t["bias_len"] = torch.randint(0, c["bias"] + 1, (S,), device="cuda", generator=g, dtype=torch.int32)
        if c["allowed"]:
            # grammars allow most tokens, or some, or few; in a tree every ninth node is a dead end
            share = torch.tensor([0.9, 0.3, 0.01], device="cuda")[torch.randint(0, 3, (R, 1), device="cuda", generator=g)]
            if c["tree"]:
                share[torch.arange(R, device="cuda") % 9 == 8] = 0.0
            t["allowed"] = _words(torch.rand(R, V, device="cuda", generator=g) < share)
        return t
    P, d, hkv = c["page"], c["d"], c["hkv"]
    need = [-(-n // P) for n in lens]
    pages, wide = sum(need) + 3, max(need) + 1
    order = torch.randperm(pages, device="cuda", generator=g).int()
    need_t = torch.tensor(need, device="cuda")
    first = torch.cumsum(need_t, 0) - need_t
    col = torch.arange(wide, device="cuda")[None, :]
    # columns behind a sequence's pages hold -1, as a serving program leaves them
    t["table"] = torch.where(col < need_t[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).int().contiguous()
    for n in ("k", "v"):
        codes = torch.empty(pages, hkv, P, d, device="cuda", dtype=torch.float8_e4m3fn)
        step = max(1, (1 << 28) // (hkv * P * d))  # in pieces, so that the fp32 values fit easily
        for a in range(0, pages, step):
            b = min(pages, a + step)
            codes[a:b] = (_normal((b - a, hkv, P, d), g) * 60.0).clamp(-448, 448).to(torch.float8_e4m3fn)
        t[n + "c"] = codes
        t[n + "s"] = torch.exp2(torch.randint(-7, -4, (pages, hkv), device="cuda", generator=g).float())
    if c["kind"] == "accept" or c["tree"]:
        t |= _trees(rows, g, 150000)
        seq = torch.repeat_interleave(torch.arange(S, device="cuda"), torch.tensor(rows, device="cuda"))
        t["position"] = ((t["len"] - (t["start"][1:] - t["start"][:-1]))[seq] + t["depth"]).int()
    if c["kind"] == "accept":
        # at most nodes the model chooses one of the drafts that follow, at some another token
        luck = torch.rand(R, device="cuda", generator=g)
        above = t["start"][seq].long() + t["parent"]
        above = torch.where(t["parent"] >= 0, above, R)
        best = torch.full((R + 1,), -1.0, device="cuda").scatter_reduce_(0, above, luck, "amax")
        picked = (best[above] == luck) & (above < R)
        follow = torch.full((R + 1,), -1, device="cuda", dtype=torch.int32)
        follow[torch.where(picked, above, R)] = torch.where(picked, t["token"], -1)
        other = torch.randint(0, 150000, (R,), device="cuda", generator=g, dtype=torch.int32)
        lucky = (torch.rand(R, device="cuda", generator=g) < 0.85) & (follow[:R] >= 0)
        t["chosen"] = torch.where(lucky, follow[:R], other)
    else:
        t["q"] = _normal((R, c["hq"] * d), g) * 2.0
    return t


def prepare(case, seed):
    s = _State(case)
    s.t = _inputs(case, seed)
    c, R, S = case, int(sum(_lengths(case)[0])), len(_lengths(case)[0])
    if c["kind"] == "attend":
        s.out = torch.empty(*s.t["q"].shape, device="cuda", dtype=torch.bfloat16 if c["half"] else torch.float32)
    elif c["kind"] == "accept":
        s.path = torch.full((R,), -1, device="cuda", dtype=torch.int32)
        s.count, s.next, s.left = (torch.zeros(S, device="cuda", dtype=torch.int32) for _ in range(3))
    else:
        s.chosen = torch.empty(R, device="cuda", dtype=torch.int32)
        s.out = torch.empty_like(s.t["logits"]) if c["write"] else None
    return s


# ---------------------------------------------------------------- the plain forms

def _places(t, R):
    """Sequence of each of the R rows, and its index within the sequence."""
    row = torch.arange(R, device="cuda")
    seq = torch.bucketize(row, t["start"][1:].long(), right=True)
    return seq, row - t["start"][seq]


def _bits(words, n):
    """The truth values that 32-bit words hold, the first n."""
    return ((words[..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(-2)[..., :n].bool()


def _plain_attend(s):
    c, t = s.case, s.t
    R, P, S = t["q"].shape[0], c["page"], t["len"].shape[0]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    seq, within = _places(t, R)
    rows, lens = _lengths(c)
    most, wide = max(rows), -(-max(lens) // P)
    table = t["table"][:, :wide].clamp(min=0).long()
    base = (t["len"] - (t["start"][1:] - t["start"][:-1]))[seq][:, None]

    def read(n):  # [sequences, heads, tokens, d]
        x = t[n + "c"][table].float() * t[n + "s"][table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(S, hkv, wide * P, d)
    key = torch.arange(wide * P, device="cuda")[None]
    at = t["position"][:, None] if c["tree"] else base + within[:, None]
    near = key > at - (c["window"] or wide * P)
    if c["tree"]:
        draft = key - base
        drafted = torch.gather(_bits(t["seen"], most), 1, draft.clamp(0, most - 1)) & (draft >= 0) & (draft < most)
        seen = ((key < base) & (near | (key < c["sinks"]))) | drafted
    else:
        seen = (key <= at) & (near | (key < c["sinks"]))
    shown = torch.zeros(S, most, wide * P, device="cuda", dtype=torch.bool)
    shown[seq, within] = seen
    q = torch.zeros(S, hkv, hq // hkv, most, d, device="cuda")
    q[seq, :, :, within] = t["q"].reshape(R, hkv, hq // hkv, d)
    score = torch.matmul(q.reshape(S, hkv, -1, d), read("k").transpose(2, 3).contiguous()) * d ** -0.5
    score = score.reshape(S, hkv, hq // hkv, most, wide * P)
    score.masked_fill_(~shown[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.reshape(S, hkv, -1, wide * P), read("v")).reshape(S, hkv, hq // hkv, most, d)
    out = out / torch.where(total == 0, 1.0, total)
    return out[seq, :, :, within].reshape(R, hq * d).to(s.out.dtype)


def _put(codes, scale, x, page, offset, first):
    """Writes x [R, heads, d] at (page, offset), of which the call's slots begin at `first` in each page; touched pages and heads get
    the scale that their earlier and their new values need."""
    peak = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    m, e = torch.frexp(peak)
    need = torch.exp2((e - torch.where(m <= 0.875, 9, 8)).clamp(min=-100).float())
    need = torch.where(peak > 0, need, torch.full_like(need, 2.0 ** -100))
    head = offset == first
    p, kept = page[head], first[head]
    old = torch.where(kept[:, None] > 0, scale[p], torch.zeros_like(scale[p]))
    new = torch.maximum(old, need[p])
    was = codes[p].float() * (old / new)[:, :, None, None]
    keep = torch.arange(codes.shape[2], device="cuda")[None, :] < kept[:, None]
    codes[p] = torch.where(keep[:, None, :, None], was, codes[p].float()).to(codes.dtype)
    scale[p] = new
    heads = torch.arange(x.shape[1], device="cuda")
    codes[page[:, None], heads[None, :], offset[:, None]] = (x / scale[page][:, :, None]).to(codes.dtype)


def _plain_accept(s):
    c, t = s.case, s.t
    R, P, S = t["parent"].shape[0], c["page"], t["len"].shape[0]
    seq, within = _places(t, R)
    most = max(_lengths(c)[0])
    n = t["start"][1:] - t["start"][:-1]
    base = t["len"] - n

    def padded(x, empty):
        y = torch.full((S, most), empty, device="cuda", dtype=torch.int64)
        y[seq, within] = x.long()
        return y
    parent, token, chosen = padded(t["parent"], -2), padded(t["token"], -2), padded(t["chosen"], -3)
    # a row follows its parent if it holds the token chosen there, the lowest that does
    follows = (parent >= 0) & (token == torch.gather(chosen, 1, parent.clamp(min=0))) & (token >= 0)
    i = torch.arange(most, device="cuda")
    lower = (parent[:, :, None] == parent[:, None, :]) & (token[:, :, None] == token[:, None, :]) & (i[None, :] < i[:, None])
    follows &= ~lower.any(-1)
    follows[:, 0] = True
    up = torch.nn.functional.one_hot(parent.clamp(min=0), most).double() * (parent >= 0)[..., None]
    line = torch.matrix_power(up + torch.eye(most, device="cuda", dtype=torch.float64), most) > 0  # ancestors and itself
    kept = ~(line & ~follows[:, None, :]).any(-1) & (i[None] < n[:, None]) & line[:, :, 0]
    count = kept.sum(-1)
    rank = torch.cumsum(kept, -1) - 1
    path = torch.full((S, most), -1, device="cuda", dtype=torch.int64)
    path.scatter_(1, torch.where(kept, rank, most - 1), torch.where(kept, i[None], -1))
    path[torch.arange(S, device="cuda"), most - 1] = torch.where(count == most, most - 1, -1)
    last = torch.gather(path, 1, (count - 1).clamp(min=0)[:, None])
    s.next = torch.where(count > 0, torch.gather(chosen, 1, last.clamp(min=0))[:, 0], -1).int()
    s.path, s.count, s.left = path[seq, within].int(), count.int(), (base + count).int()
    # tokens from the first one that changes its place on
    moved = (path != i[None]) & (path >= 0)
    first = torch.where(moved.any(-1), moved.int().argmax(-1), most)
    which, rank = torch.nonzero(moved)[:, 0], torch.nonzero(moved)[:, 1]
    source = base[which] + path[which, rank]
    place = base[which] + rank
    page_of, slot_of = t["table"][which, source // P].long(), source % P
    page, offset = t["table"][which, place // P].long(), place % P
    begins = torch.clamp(offset - (rank - first[which]), min=0)
    for n in ("k", "v"):
        x = t[n + "c"][page_of, :, slot_of].float() * t[n + "s"][page_of][..., None]
        _put(t[n + "c"], t[n + "s"], x, page, offset, begins)


def _plain_choose(s):
    c, t = s.case, s.t
    x = t["logits"]
    R, V = x.shape
    S = t["len"].shape[0]
    seq, within = _places(t, R)
    if c["penal"]:
        known = torch.arange(t["past"].shape[1], device="cuda")[None] < t["len"][:, None]
        times = torch.zeros(S, V, device="cuda").scatter_add_(1, t["past"].long(), known.float())[seq]
        if c["tree"]:
            most = max(_lengths(c)[0])
            at = t["start"][seq].long()[:, None] + torch.arange(most, device="cuda")[None]
            times.scatter_add_(1, t["token"][at.clamp(max=R - 1)].long(), _bits(t["seen"], most).float())
        p = t["penalty"][seq]
        y = torch.where(x > 0, x / p[:, 0:1], x * p[:, 0:1]) - (p[:, 1:2] + p[:, 2:3] * times)
        x = torch.where(times > 0, y, x)
    if c["bias"]:
        # the last entry of a token counts
        entry = torch.arange(1, c["bias"] + 1, device="cuda")[None] * (torch.arange(c["bias"], device="cuda")[None] < t["bias_len"][:, None])
        last = torch.zeros(S, V, device="cuda", dtype=torch.int64).scatter_reduce_(1, t["bias_token"].long(), entry, "amax")
        extra = torch.gather(torch.nn.functional.pad(t["bias"], (1, 0)), 1, last)[seq]
        x = torch.where(last[seq] > 0, x + extra, x)
    token = torch.arange(V, device="cuda")
    if c["allowed"]:
        allowed = _bits(t["allowed"], V)
        x = x.masked_fill(~allowed, -math.inf)
        token = torch.where(allowed, token, V)
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, token, V).amin(-1)
    s.chosen = torch.where(first < V, first, -1).int()
    s.out = x


# ---------------------------------------------------------------- one pass

def _handles(s):
    """The buffers, views and kernels that a program keeps beside its tensors."""
    from edgerunner_amd import (Buffer, Drafts, HeadRows, KV8AcceptKernel, KV8AttentionKernel, KV8Batch, KV8Cache, LogitChoiceKernel,
                                LogitRules, default_context)
    from edgerunner_amd._ffi import er_buffer
    ctx, c, t, k = default_context(), s.case, s.t, {}

    def buf(x):
        return Buffer(ctx, er_buffer(x.data_ptr(), x.numel() * x.element_size()), owned=False)

    def optional(name):
        return buf(t[name]) if name in t else None
    rows, lens = _lengths(c)
    R = sum(rows)
    drafted = c["kind"] == "accept" or c["tree"]
    k["drafts"] = Drafts(buf(t["seen"]), t["seen"].shape[1], position=optional("position"), parent=buf(t["parent"]),
                         token=buf(t["token"])) if drafted else None
    if c["kind"] == "choose":
        k["kernel"] = LogitChoiceKernel(ctx)
        k["logits"], k["chosen"], k["out"] = buf(t["logits"]), buf(s.chosen), buf(s.out) if c["write"] else None
        k["rules"] = LogitRules(buf(t["start"]), len(rows), max(rows), penalty=optional("penalty"), history=optional("past"),
                                historyLen=buf(t["len"]) if c["penal"] else None,
                                historyStride=t["past"].shape[1] if c["penal"] else 0, biasToken=optional("bias_token"),
                                bias=optional("bias"), biasLen=optional("bias_len"), biasStride=c["bias"], allowed=optional("allowed"),
                                allowedStride=t["allowed"].shape[1] if c["allowed"] else 0)
        k["scratch"] = ctx.alloc(max(16, k["kernel"].workspaceBytes(R, c["vocab"])))
        return k
    k["cache"] = KV8Cache(buf(t["kc"]), buf(t["vc"]), buf(t["ks"]), buf(t["vs"]), t["kc"].shape[0], c["hkv"], c["page"], c["d"])
    k["batch"] = KV8Batch(buf(t["table"]), buf(t["len"]), buf(t["start"]), len(rows), t["table"].shape[1], R, max(rows), max(lens))
    if c["kind"] == "accept":
        k["kernel"] = KV8AcceptKernel(ctx)
        k["chosen"], k["path"], k["count"], k["next"], k["left"] = (buf(x) for x in (t["chosen"], s.path, s.count, s.next, s.left))
        return k
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
        if c["kind"] == "attend":
            k["kernel"].encode(None, k["cache"], k["batch"], k["q"], k["out"], c["d"] ** -0.5, window=c["window"],
                               workspace=k["scratch"], outBF16=c["half"], sinks=c["sinks"], drafts=k["drafts"])
        elif c["kind"] == "accept":
            k["kernel"].encode(None, k["cache"], k["batch"], k["drafts"], k["chosen"], k["path"], k["count"], k["next"], k["left"])
        else:
            k["kernel"].encode(None, k["logits"], s.t["logits"].shape[0], c["vocab"], k["rules"], drafts=k["drafts"], out=k["out"],
                               chosen=k["chosen"], workspace=k["scratch"])
    elif c["kind"] == "attend":
        s.out = _plain_attend(s)
    elif c["kind"] == "accept":
        _plain_accept(s)
    else:
        _plain_choose(s)
    if c["kind"] == "attend":
        return {"out": s.out}
    if c["kind"] == "accept":
        return {**{n: s.t[n] for n in ("kc", "ks", "vc", "vs")}, "path": s.path, "count": s.count, "next": s.next, "left": s.left}
    return {"chosen": s.chosen, "out": s.out} if c["write"] else {"chosen": s.chosen}


# ---------------------------------------------------------------- what a pass cannot do without

def _seen(c):
    """(keys that some row of the sequence reaches, pairs of a row and a key, at the most) over all sequences."""
    keys = pairs = 0
    for n, m in zip(*_lengths(c)):
        if not n:
            continue
        before = m - n
        if c["tree"]:
            far = min(before, c["window"] + c["sinks"]) if c["window"] else before
            keys += far + n
            pairs += n * far + n * min(n, 2 * n.bit_length())  # a random tree's depth
        else:
            far = c["window"] + c["sinks"]
            keys += min(m, far + n - 1)
            pairs += sum(min(before + i + 1, far) for i in range(n))
    return keys, pairs


def work(case):
    c = case
    rows, lens = _lengths(c)
    R = sum(rows)
    if c["kind"] == "choose":
        V = c["vocab"]
        nbytes = R * V * (8 if c["write"] else 4) + (R * -(-V // 32) * 4 if c["allowed"] else 0) + 4 * sum(lens) * c["penal"] + 4 * R
        return {"bytes": nbytes + 8 * len(rows) * c["bias"] // 2, "flops": R * V * (1 + c["allowed"])}
    if c["kind"] == "accept":
        kept = sum(min(n, 2) for n in rows)  # about two moves a sequence
        return {"bytes": 16 * R + 4 * kept * c["hkv"] * c["d"], "flops": 4 * kept * c["hkv"] * c["d"] + R}
    keys, pairs = _seen(c)
    return {"bytes": 2 * keys * c["hkv"] * c["d"] + R * c["hq"] * c["d"] * (4 + (2 if c["half"] else 4)),
            "flops": 4 * pairs * c["hq"] * c["d"]}


# ---------------------------------------------------------------- the same in 64 bits

def _code64(x):
    """The e4m3 value nearest to each x of up to 448 in size, ties to the even one: three bits behind the first, steps of 2^-9 at the least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _line(parent, i):
    """A row and its ancestors, from it upwards."""
    while i >= 0:
        yield i
        i = parent[i]


def _exact_attend(c, t):
    rows, lens = _lengths(c)
    P, hkv, G, d = c["page"], c["hkv"], c["hq"] // c["hkv"], c["d"]
    parent = t["parent"].tolist() if c["tree"] else None
    parts, row = [], 0
    for s, (n, m) in enumerate(zip(rows, lens)):
        if not n:
            continue
        pages = t["table"][s, :-(-m // P)].long()
        o = torch.empty(n, c["hq"], d, device="cuda", dtype=torch.float64)
        at = torch.arange(m - n, m, device="cuda")[:, None]
        key = torch.arange(m, device="cuda")[None]
        if c["tree"]:
            above = parent[row:row + n]
            lines = [list(_line(above, i)) for i in range(n)]
            at = torch.tensor([[m - n + len(x) - 1] for x in lines], device="cuda")
            hidden = (key >= m - n) | ((key <= at - (c["window"] or m + 1)) & (key >= c["sinks"]))
            pairs = torch.tensor([(i, m - n + j) for i, x in enumerate(lines) for j in x], device="cuda")
            hidden[pairs[:, 0], pairs[:, 1]] = False
        else:
            hidden = (key > at) | ((key <= at - c["window"]) & (key >= c["sinks"]))
        for h in range(hkv):
            k, v = ((t[x + "c"][pages, h].double() * t[x + "s"][pages, h].double()[:, None, None]).flatten(0, 1)[:m] for x in "kv")
            q = t["q"][row:row + n].reshape(n, c["hq"], d)[:, h * G:(h + 1) * G].double()
            for g in range(G):
                p = torch.softmax((q[:, g] @ k.T.contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                o[:, h * G + g] = p @ v
        parts.append(o.flatten(1))
        row += n
    return {"out": torch.cat(parts)}


def _exact_accept(c, t):
    rows, lens = _lengths(c)
    P, row = c["page"], 0
    parent, token, chosen = t["parent"].tolist(), t["token"].tolist(), t["chosen"].tolist()
    out = {n + x: t[n + x].double() for n in "kv" for x in "cs"}
    path, count, after, left = [], [], [], []
    for s, (n, m) in enumerate(zip(rows, lens)):
        line, cur = ([0], 0) if n else ([], -1)
        while cur >= 0:
            cur = next((r for r in range(n) if parent[row + r] == cur and token[row + r] == chosen[row + cur] >= 0), -1)
            line += [cur] if cur >= 0 else []
        path += line + [-1] * (n - len(line))
        count.append(len(line))
        after.append(chosen[row + line[-1]] if n else -1)
        base = m - n
        left.append(base + len(line))
        changed = [j for j, r in enumerate(line) if r != j]
        if changed:
            table = t["table"][s].tolist()
            for n_ in "kv":
                codes, scale = out[n_ + "c"], out[n_ + "s"]
                values = [codes[table[(base + r) // P], :, (base + r) % P] * scale[table[(base + r) // P]][:, None] for r in line]
                a = base + changed[0]
                for p in range(a // P, (base + len(line) - 1) // P + 1):
                    lo, hi = max(a, p * P), min(base + len(line), p * P + P)
                    x = torch.stack(values[lo - base:hi - base], 1)  # [heads, tokens, d]
                    peak = x.abs().amax((1, 2)) / 448
                    grown = torch.exp2(torch.ceil(torch.log2(peak.clamp(min=2.0 ** -100))))
                    page, kept = table[p], lo - p * P
                    old = scale[page].clone() if kept else torch.zeros_like(grown)
                    scale[page] = torch.maximum(old, grown)
                    codes[page, :, :kept] = _code64(codes[page, :, :kept] * (old / scale[page])[:, None, None])
                    codes[page, :, kept:kept + hi - lo] = _code64(x / scale[page][:, None, None])
        row += n
    whole = {"path": path, "count": count, "next": after, "left": left}
    return {**out, **{n: torch.tensor(x, device="cuda", dtype=torch.int32) for n, x in whole.items()}}


def _exact_choose(c, t):
    rows, lens = _lengths(c)
    V, row, ys, chosen = c["vocab"], 0, [], []
    for s, n in enumerate(rows):
        for i in range(n):
            y = t["logits"][row + i].double()
            if c["penal"]:
                context = t["past"][s, :lens[s]].long()
                if c["tree"]:
                    line = list(_line(t["parent"][row:row + n].tolist(), i))
                    context = torch.cat([context, t["token"][row:row + n][torch.tensor(line, device="cuda")].long()])
                times = torch.bincount(context, minlength=V).double()
                rep, presence, frequency = t["penalty"][s].double()
                less = torch.where(y > 0, y / rep, y * rep) - presence - frequency * times
                y = torch.where(times > 0, less, y)
            if c["bias"]:
                for token, b in dict(zip(t["bias_token"][s, :t["bias_len"][s]].tolist(), t["bias"][s].tolist())).items():
                    y[token] += b
            able = torch.arange(V, device="cuda")
            if c["allowed"]:
                words = t["allowed"][row + i].repeat_interleave(32)[:V] >> (able % 32).int()
                y = torch.where(words & 1 == 1, y, -math.inf)
                able = able[words & 1 == 1]
            # the choice is among the values as they are stored
            best = y.float()[able]
            chosen.append(int(able[torch.nonzero(best == best.max())[0, 0]]) if len(able) else -1)
            ys.append(y if c["write"] else None)
        row += n
    chosen = torch.tensor(chosen, device="cuda", dtype=torch.int32)
    return {"chosen": chosen, "out": torch.stack(ys)} if c["write"] else {"chosen": chosen}


def exact(case, seed):
    t = _inputs(case, seed)
    return {"attend": _exact_attend, "accept": _exact_accept, "choose": _exact_choose}[case["kind"]](case, t)
