"""The operators of drafting and verifying over a paged cache whose speed is measured, with
their plain forms and their 64-bit results.

  rotary   rotary positions of queries and keys, forward or forward and backward
  append   paged_append: norms, rotation and storing of new tokens into a cache of pages
  attend   paged_attention of single tokens, drafted trees or chunks of prompts over pages
  verify   verify_drafts: drafted trees against the target's probabilities
  keep     paged_keep: the accepted branch moved into place in every layer

Sizes are those of this repository's benchmark and model defaults (8 query and 4 key heads
of 96, 64 sequences decoding over some 2048 positions, 8 layers, a vocabulary of 6400) and
generic ones around them.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

PKG = Path(__file__).resolve().parent.parent / "minimind-mhc_amd"
if str(PKG) not in sys.path:
    sys.path.insert(0, str(PKG))

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# ------------------------------------------------------------------ the cases

def _rotary(name, tokens, heads=8, kv=4, hd=96, rd=96, dtype="bf16", pairs="half", scaled=False, train=True):
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "kv": kv, "hd": hd, "rd": rd,
            "dtype": dtype, "pairs": pairs, "scaled": scaled, "train": train}


def _append(name, seqs, tokens, past, page, heads=8, kv=4, hd=96, rd=96, dtype="bf16", pairs="half", norm=True):
    """tokens: new ones of all sequences; past: keys of a sequence before them, at most."""
    return {"name": name, "kind": "append", "seqs": seqs, "tokens": tokens, "past": past, "page": page,
            "heads": heads, "kv": kv, "hd": hd, "rd": rd, "dtype": dtype, "pairs": pairs, "norm": norm}


def _attend(name, seqs, tokens, past, page, heads=8, kv=4, hd=96, dtype="bf16", width=0):
    """width: of the drafted tree (a node's parent is one of so many before it); 0: causal."""
    return {"name": name, "kind": "attend", "seqs": seqs, "tokens": tokens, "past": past, "page": page,
            "heads": heads, "kv": kv, "hd": hd, "dtype": dtype, "width": width}


def _verify(name, seqs, tokens, vocab, dtype="f32", width=1, mode="sample"):
    """mode: "sample" (against the draft's probabilities), "certain" (drafts without them) or
    "greedy"."""
    return {"name": name, "kind": "verify", "seqs": seqs, "tokens": tokens, "vocab": vocab, "dtype": dtype,
            "width": width, "mode": mode}


def _keep(name, seqs, tokens, past, page, layers=8, kv=4, hd=96, dtype="bf16"):
    return {"name": name, "kind": "keep", "seqs": seqs, "tokens": tokens, "past": past, "page": page,
            "layers": layers, "kv": kv, "hd": hd, "dtype": dtype}


def listed():
    return [
        # queries and keys of a training step's layer, whole heads in halves
        _rotary("rotary_train", 16384),
        # the trainers' 32 bits: half of each wide head, interleaved, at far, scaled positions
        _rotary("rotary_partial", 4001, heads=16, kv=2, hd=128, rd=64, dtype="f32", pairs="interleaved", scaled=True),
        # a decode step's new tokens of 64 sequences
        _append("append_decode", 64, 64, 2100, 64),
        # prompts of different lengths into small pages, without norms
        _append("append_prompts", 16, 8191, 1, 16, heads=16, kv=2, hd=128, rd=64, dtype="f16",
                pairs="interleaved", norm=False),
        # the decode step's attention, the lengths all different
        _attend("attend_decode", 64, 64, 2175, 64),
        # a step of drafted trees for the same batch
        _attend("attend_trees", 64, 1024, 2175, 16, width=4),
        # one long conversation with a large tree
        _attend("attend_long", 1, 64, 65001, 256, heads=16, kv=2, hd=128, dtype="f16", width=6),
        # chunks of prompts behind what is cached
        _attend("attend_chunks", 6, 3001, 4100, 64, heads=8, kv=8, hd=64),
        # chains of seven drafts for 64 sequences, sampled
        _verify("verify_chains", 64, 512, 6400),
        # trees over a wide, odd vocabulary, half the probabilities' bits
        _verify("verify_trees", 16, 512, 50257, dtype="bf16", width=5),
        # the accepted branches of a batch's trees
        _keep("keep_trees", 64, 1024, 2175, 16),
        # of one conversation
        _keep("keep_one", 1, 33, 9001, 256, layers=24, kv=2, hd=128, dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "verify", "keep"])
    half = rng.choice(["bf16", "bf16", "f16"])
    heads, kv = rng.choice([(8, 4), (8, 4), (8, 8), (8, 2), (8, 1), (6, 2), (16, 2), (12, 4)])
    hd = rng.choice([64, 96, 96, 128])
    rd, pairs = hd // rng.choice([1, 1, 2, 4]), rng.choice(["half", "half", "interleaved"])
    seqs, page = _log_int(rng, 1, 64), rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "rotary":
        c = _rotary("", _log_int(rng, 1, 16384), heads, kv, hd, rd, rng.choice([half, half, "f32"]), pairs,
                    rng.random() < 0.3, rng.random() < 0.6)
    elif kind == "verify":
        vocab = rng.choice([6400, 6400, 6401, 1000, 32000, 50257])
        nodes = _log_int(rng, 1, max(1, min(64, 512 * 50257 // (vocab * seqs))))
        c = _verify("", seqs, max(seqs, seqs * nodes - rng.randrange(2)), vocab, rng.choice([half, "f32", "f32"]),
                    rng.choice([1, 1, 3, 6]), rng.choice(["sample", "sample", "certain", "greedy"]))
    elif kind == "keep":
        c = _keep("", seqs, max(seqs, seqs * _log_int(rng, 1, 64) - rng.randrange(2)),
                  _log_int(rng, 1, max(64, 65536 // seqs)), page, rng.choice([4, 8, 16]), kv, hd, half)
    else:
        past = _log_int(rng, 1, max(4096, 131072 // seqs))
        what = rng.random()
        new = 1 if what < 0.35 else _log_int(rng, 2, 100) if what < 0.75 else _log_int(rng, 2, max(2, 4096 // seqs))
        tokens = max(seqs, seqs * new - (rng.randrange(2) if new > 1 else 0))
        if kind == "append":
            c = _append("", seqs, tokens, past, page, heads, kv, hd, rd, half, pairs, rng.random() < 0.7)
        else:
            tree = 0.35 <= what < 0.75 and rng.random() < 0.8
            c = _attend("", seqs, tokens, past, page, heads, kv, hd, half, rng.choice([1, 3, 6]) if tree else 0)
    del c["name"]
    return c


def draw(rng):
    top = [work(c) for c in listed()]
    flops, moved = max(w["flops"] for w in top), max(w["bytes"] for w in top)
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= moved:
            return c


def _lengths(total, n):
    """n lengths with that sum, no two more than one apart."""
    return [total // n + (i < total % n) for i in range(n)]


def _spans(case):
    """(keys before, new tokens) of each sequence; they follow from the case alone."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["tokens"], case["past"]))
    new = _lengths(case["tokens"], case["seqs"])
    if case["kind"] == "append" and case["past"] == 1:  # whole prompts, of different lengths
        new = [max(1, n - d) for n, d in zip(new, (rng.randint(0, max(n - 1, 0)) for n in new))]
        new[0] += case["tokens"] - sum(new)
        return [(0, n) for n in new]
    past = [rng.randint(case["past"] // 3, case["past"]) for _ in new]
    past[-1] = case["past"]
    return list(zip(past, new))


def _parents(case):
    """The parents of each sequence's nodes (-1 for the first)."""
    out = []
    for i, n in enumerate(_lengths(case["tokens"], case["seqs"])):
        rng = random.Random("%d %d %d" % (i, n, case["width"]))
        out.append([-1] + [rng.randrange(max(0, j - case["width"]), j) for j in range(1, n)])
    return out


def _paths(case):
    """The accepted nodes of each sequence: the root, some of the first branch, then nodes of
    others."""
    out = []
    for i, n in enumerate(_lengths(case["tokens"], case["seqs"])):
        rng = random.Random("%d %d kept" % (i, n))
        kept = rng.randint(1, max(1, min(n // 2, 12)))
        same = rng.randint(1, kept)
        out.append(list(range(same)) + sorted(rng.sample(range(kept, n), kept - same)))
    return out


# ------------------------------------------------------------------- the work

def work(case):
    """Each input read once, each output written once; the products under the mask."""
    k, e, T = case["kind"], 4 if case["dtype"] == "f32" else 2, case["tokens"]
    if k == "rotary":
        n, both = T * (case["heads"] + case["kv"]), 2 if case["train"] else 1
        return {"bytes": 2 * both * n * case["hd"] * e + T * (4 * case["rd"] + 8), "flops": 3 * both * n * case["rd"]}
    if k == "append":
        H, KV, hd = case["heads"], case["kv"], case["hd"]
        return {"bytes": 2 * T * (H + 2 * KV) * hd * e + T * 4 * case["rd"],
                "flops": T * (H + KV) * (3 * case["rd"] + (4 * hd if case["norm"] else 0))}
    if k == "attend":
        H, KV, hd, spans = case["heads"], case["kv"], case["hd"], _spans(case)
        seen = sum(p * n for p, n in spans)
        if case["width"]:
            seen += sum(_depth(ps) for ps in _parents(case))
        else:
            seen += sum(n * (n + 1) // 2 for _, n in spans)
        return {"bytes": (2 * T * H + 2 * sum(p + n for p, n in spans) * KV) * hd * e, "flops": 4 * seen * H * hd}
    if k == "keep":
        rows = sum(sum(a != b for a, b in enumerate(p)) for p in _paths(case))
        return {"bytes": 4 * rows * case["layers"] * case["kv"] * case["hd"] * e + 4 * T, "flops": 0}
    # the last node's rows; greedy: the rows on the way, half the longest branch
    rows = 2 if case["mode"] == "sample" else 1
    if case["mode"] == "greedy":
        rows = 1 + max(_depth(ps, True) for ps in _parents(case)) / 2
    return {"bytes": int(case["seqs"] * case["vocab"] * e * rows) + 16 * T, "flops": int(2 * case["seqs"] * case["vocab"] * rows)}


def _depth(parents, most=False):
    """The nodes that all nodes see of their tree, themselves among them (most: one does)."""
    d = []
    for p in parents:
        d.append(1 if p < 0 else d[p] + 1)
    return max(d) if most else sum(d)


# ----------------------------------------------------------------- the inputs

def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _on_gpu(ints, dtype=torch.int32):
    return torch.tensor(ints, dtype=dtype, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, dtype, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def _tables(positions, rd, scaled):
    """cos and sin [positions, rd / 2] of angles in 64 bits; scaled: slow pairs sixteen times
    slower, for contexts longer than the trained one, and everything a tenth longer."""
    freq = 1e6 ** (-torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)
    if scaled:
        freq = torch.where(2 * math.pi / freq > 2048, freq / 16, freq)
    a = torch.outer(torch.arange(positions, device="cuda", dtype=torch.float64), freq)
    m = 1.1 if scaled else 1.0
    return (m * a.cos()).float(), (m * a.sin()).float()


def _bits(case):
    """The drafted trees as bits: which of its sequence's new rows each row sees."""
    words = (max(_lengths(case["tokens"], case["seqs"])) + 63) // 64
    rows = []
    for ps in _parents(case):
        seen = []
        for j, p in enumerate(ps):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        rows += seen
    full = (1 << 64) - 1
    return _on_gpu([[(w if w < 1 << 63 else w - (1 << 64)) for w in ((r >> 64 * i) & full for i in range(words))]
                    for r in rows], torch.int64)


def _pages(s, g, seed, case, planes):
    """Pages of the cache, in no order, and the table of which are whose."""
    page, spans = case["page"], s["spans"]
    need = [(p + n + page - 1) // page for p, n in spans]
    wide = max(need) + 1
    order = list(range(sum(need) + 3))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (wide - n))
        at += n
    s["table"] = _on_gpu(table)
    s["lengths"] = _on_gpu([p for p, _ in spans])
    s["cu"] = _on_gpu(_starts([n for _, n in spans]))
    return _normal(g, DT[case["dtype"]], planes, len(order), page, case["kv"], case["hd"])


def prepare(case, seed):
    g, k, dt = _gen(seed), case["kind"], DT[case["dtype"]]
    s = {"case": case}
    if k == "rotary":
        T, hd = case["tokens"], case["hd"]
        table = 32768 if case["scaled"] else max(2048, T)
        s["cos"], s["sin"] = _tables(table, case["rd"], case["scaled"])
        # packed sequences, some behind a past
        starts = [0]
        while starts[-1] < T:
            starts.append(starts[-1] + 1 + T // 5)
        rng = random.Random(seed)
        at = [torch.arange(b - a, device="cuda") + rng.randint(0, table - (b - a))
              for a, b in zip(starts, [min(x, T) for x in starts[1:]])]
        s["positions"] = torch.cat(at)
        for t, n in (("q", case["heads"]), ("k", case["kv"])):
            s[t], s["g" + t] = _normal(g, dt, T, n, hd), _normal(g, dt, T, n, hd)
            s[t].requires_grad_(case["train"])
        return s
    if k == "verify":
        T, V, n = case["tokens"], case["vocab"], case["seqs"]
        s["cu"] = _on_gpu(_starts(_lengths(T, n)))
        s["parents"] = None if case["width"] == 1 else _on_gpu(sum(_parents(case), []))
        logits = torch.randn(T, V, generator=g, device="cuda").mul_(4.0)
        rough = logits + torch.randn(T, V, generator=g, device="cuda").mul_(0.6)
        s["probs"], q = (x.softmax(-1).to(dt) for x in (logits, rough))
        at = _starts(_lengths(T, n))
        up = [a + max(p, 0) for a, ps in zip(at, _parents(case)) for p in ps]
        up = _on_gpu(up, torch.int64)
        if case["mode"] == "sample":  # drafted by the draft's probabilities at the parent
            s["tokens"] = torch.multinomial(q.float()[up], 1, generator=g)[:, 0]
        else:  # siblings the draft's most probable ones, in turn
            turn, seen = [], {}
            for p in up.tolist():
                turn.append(seen.get(p, 0))
                seen[p] = turn[-1] + 1
            best = rough.topk(max(turn) + 1, -1).indices[up]
            s["tokens"] = best.gather(1, _on_gpu(turn, torch.int64)[:, None])[:, 0].contiguous()
        s["draft"] = q if case["mode"] == "sample" else None
        s["u"] = None if case["mode"] == "greedy" else torch.rand(T, generator=g, device="cuda")
        return s
    if k == "keep":
        s["spans"] = _spans(case)
        s["pages"] = _pages(s, g, seed, case, 2 * case["layers"])
        s["kept"] = _on_gpu([len(p) for p in _paths(case)])
        s["path"] = _on_gpu(sum((p + [-1] * (n - len(p)) for p, (_, n) in zip(_paths(case), s["spans"])), []))
        return s
    H, KV, hd, T = case["heads"], case["kv"], case["hd"], case["tokens"]
    s["spans"] = _spans(case)
    both = _pages(s, g, seed, case, 2)
    s["k_pages"], s["v_pages"] = both.unbind(0)
    s["q"] = _normal(g, dt, T, H, hd, std=1.3)
    if k == "attend":
        s["k_pages"].mul_(1.3)
        s["tree"] = _bits(case) if case["width"] else None
        return s
    s["k"], s["v"] = _normal(g, dt, T, KV, hd, std=1.3), _normal(g, dt, T, KV, hd)
    s["cos"], s["sin"] = _tables(max(p + n for p, n in s["spans"]), case["rd"], False)
    for t in ("q_gain", "k_gain"):
        s[t] = (1 + _normal(g, torch.float32, hd, std=0.2)).to(dt) if case["norm"] else None
    return s


# -------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, rd, pairs, back=False):
    """x [rows, heads, hd] in 32 bits, turned by the rows' angles (back: by their opposites)."""
    c, s = cos[:, None], -sin[:, None] if back else sin[:, None]
    if pairs == "half":
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([y, x[..., rd:]], -1)


def _plain_rotary(s):
    case = s["case"]
    c, n = s["cos"][s["positions"]], s["sin"][s["positions"]]
    out = {t: _rotate(s[t].detach().float(), c, n, case["rd"], case["pairs"]).to(s[t].dtype) for t in "qk"}
    if case["train"]:
        for t in ("gq", "gk"):
            out[t] = _rotate(s[t].float(), c, n, case["rd"], case["pairs"], back=True).to(s[t].dtype)
    return out


def _key_rows(s, keys):
    """The rows in the pages (as one long tensor) of the given keys of each sequence."""
    page = s["case"]["page"]
    out = []
    for i, (a, b) in enumerate(keys):
        at = torch.arange(a, b, device="cuda")
        out.append(s["table"][i, at // page].long() * page + at % page)
    return out


def _plain_append(s):
    case = s["case"]
    at = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in s["spans"]])
    c, n = s["cos"][at], s["sin"][at]
    res = {}
    for t in "qk":
        x = s[t].float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s[t + "_gain"].float()
        res[t] = _rotate(x, c, n, case["rd"], case["pairs"]).to(s[t].dtype)
    rows = torch.cat(_key_rows(s, [(p, p + n) for p, n in s["spans"]]))
    s["k_pages"].flatten(0, 1)[rows] = res["k"]
    s["v_pages"].flatten(0, 1)[rows] = s["v"]
    return {"q": res["q"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _unseen(s, i, at, past, new):
    """[new, keys] of sequence i, whose rows begin at `at`: the keys that a row does not see."""
    col = torch.arange(past + new, device="cuda")
    if s["tree"] is None:
        return col > past + torch.arange(new, device="cuda")[:, None]
    j = torch.arange(new, device="cuda")
    own_rows = (s["tree"][at:at + new][:, j // 64] >> (j % 64)) & 1
    return torch.cat([torch.zeros(new, past, dtype=torch.bool, device="cuda"), own_rows == 0], 1)


def _plain_attend(s):
    case, at = s["case"], 0
    rep, scale = case["heads"] // case["kv"], 1.0 / math.sqrt(case["hd"])
    out = torch.empty_like(s["q"])
    rows = _key_rows(s, [(0, p + n) for p, n in s["spans"]])
    for i, (past, new) in enumerate(s["spans"]):
        q = s["q"][at:at + new].float().transpose(0, 1)
        k, v = (s[t].flatten(0, 1)[rows[i]].float().transpose(0, 1).repeat_interleave(rep, 0)
                for t in ("k_pages", "v_pages"))
        a = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
        a.masked_fill_(_unseen(s, i, at, past, new), -math.inf)
        a = torch.exp(a - a.amax(-1, keepdim=True))
        a = a / a.sum(-1, keepdim=True)
        out[at:at + new] = torch.matmul(a, v).transpose(0, 1).to(out.dtype)
        at += new
    return {"out": out}


def _plain_verify(s):
    """All sequences at once, a node at a time.  In 64 bits: cumulated probabilities are compared."""
    case, probs, draft, u = s["case"], s["probs"], s["draft"], s["u"]
    V, n = case["vocab"], case["seqs"]
    lens = _lengths(case["tokens"], n)
    first = s["cu"][:-1].long()
    count = s["cu"].diff().long()
    cur = torch.zeros_like(first)
    kept = torch.ones_like(first)
    path = torch.full((case["tokens"],), -1, dtype=torch.int32, device="cuda")
    path[first] = 0
    p = probs[first].double()
    q = draft[first].double() if draft is not None else None
    a, c = torch.zeros(n, 1, dtype=torch.float64, device="cuda"), torch.ones(n, 1, dtype=torch.float64, device="cuda")
    index = torch.arange(V, device="cuda")
    for j in range(1, max(lens)):
        row = first + torch.clamp(torch.full_like(first, j), max=count - 1)
        parent = s["parents"][row].long() if s["parents"] is not None else torch.full_like(first, j - 1)
        mine = (parent == cur) & (j < count)
        x = s["tokens"][row][:, None]
        px = p.gather(1, x)
        if u is None:
            top = torch.where(p == p.amax(1, keepdim=True), index, V).amin(1)
            ok = mine & (top == x[:, 0])
        elif draft is None:
            ok = mine & (u[row, None].double() * c < px)[:, 0]
            gone = (mine & ~ok)[:, None]
            c = torch.where(gone, c - px, c)
            p = torch.where(gone & (index == x), 0.0, p)
        else:
            qx = q.gather(1, x)
            ok = mine & (u[row, None].double() * qx * c < (px - a * qx).clamp_min(0))[:, 0]
            gone = (mine & ~ok)[:, None]
            a = torch.where(gone, a + c, a)
            c = torch.where(gone, (p - a * q).clamp_min(0).sum(1, keepdim=True), c)
        cur = torch.where(ok, j, cur)
        at = first + torch.minimum(kept, count - 1)
        path[at] = torch.where(ok, j, path[at]).to(torch.int32)
        kept = kept + ok
        p = torch.where(ok[:, None], probs[first + cur].double(), p)
        if draft is not None:
            q = torch.where(ok[:, None], draft[first + cur].double(), q)
        a, c = torch.where(ok[:, None], 0.0, a), torch.where(ok[:, None], 1.0, c)
    if u is None:
        token = torch.where(p == p.amax(1, keepdim=True), index, V).amin(1)
    else:
        w = p if draft is None else (p - a * q).clamp_min(0)
        w = torch.where((w.sum(1, keepdim=True) > 0), w, probs[first + cur].double())
        cum = w.cumsum(1)
        past = cum > u[first, None].double() * cum[:, -1:]
        last = torch.where(w > 0, index, -1).amax(1)
        token = torch.minimum(torch.where(past & (w > 0), index, V).amin(1), last)
    return {"kept": kept.to(torch.int32), "path": path, "next": token}


def _plain_keep(s):
    flat = s["pages"].flatten(1, 2)
    src, dst = [], []
    paths = _paths(s["case"])
    for i, (past, _) in enumerate(s["spans"]):
        both = _key_rows({**s, "table": s["table"][i:i + 1]}, [(past, past + len(paths[i]))])
        dst.append(both[0])
    page = s["case"]["page"]
    at = 0
    for i, (past, new) in enumerate(s["spans"]):
        key = past + s["path"][at:at + len(paths[i])].long()
        src.append(s["table"][i, key // page].long() * page + key % page)
        at += new
    flat[:, torch.cat(dst)] = flat[:, torch.cat(src)]
    return {"pages": s["pages"], "lengths": s["lengths"] + s["kept"]}


# ------------------------------------------------------------------------ run

def run(s):
    case, k = s["case"], s["case"]["kind"]
    if not own:
        with torch.no_grad():
            return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend,
                    "verify": _plain_verify, "keep": _plain_keep}[k](s)
    inter = case.get("pairs") == "interleaved"
    if k == "rotary":
        from model.rotary import rotary
        if not case["train"]:
            with torch.inference_mode():
                return dict(zip("qk", rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=inter)))
        out = rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=inter)
        grads = torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))
        return dict(zip(("q", "k", "gq", "gk"), (out[0].detach(), out[1].detach(), *grads)))
    with torch.inference_mode():
        if k == "append":
            from model.paged import paged_append
            q = paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["cu"],
                             s["cos"], s["sin"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS, interleaved=inter)
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if k == "attend":
            from model.paged import paged_attention
            return {"out": paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["cu"],
                                           tree=s["tree"])}
        if k == "verify":
            from model.speculative import verify_drafts
            return dict(zip(("kept", "path", "next"),
                            verify_drafts(s["probs"], s["tokens"], s["cu"], parents=s["parents"],
                                          draft_probs=s["draft"], uniforms=s["u"])))
        from model.paged import paged_keep
        return {"pages": s["pages"], "lengths": paged_keep(s["pages"], s["table"], s["lengths"], s["cu"], s["kept"],
                                                           s["path"])}


# ------------------------------------------------- the results, in 64 bits

def _turn(x, angle_cos, angle_sin, pairs):
    """Each pair of x [rows, heads, rd] as a complex number times cos + i sin."""
    z = torch.view_as_complex(x.unflatten(-1, (2, -1)).transpose(-1, -2).contiguous() if pairs == "half"
                              else x.unflatten(-1, (-1, 2)).contiguous())
    z = z * torch.complex(angle_cos, angle_sin)[:, None]
    z = torch.view_as_real(z)
    return z.transpose(-1, -2).flatten(-2) if pairs == "half" else z.flatten(-2)


def _exact_rotary(case, s):
    c, n = (s[t].double()[s["positions"]] for t in ("cos", "sin"))
    out, rd = {}, case["rd"]
    for t in "qk":
        x = s[t].detach().double().requires_grad_()
        y = torch.cat([_turn(x[..., :rd], c, n, case["pairs"]), x[..., rd:]], -1)
        out[t] = y.detach()
        if case["train"]:
            out["g" + t], = torch.autograd.grad(y, x, s["g" + t].double())
    return {t: out[t] for t in (("q", "k", "gq", "gk") if case["train"] else "qk")}


def _exact_append(case, s):
    page, rd = case["page"], case["rd"]
    pages = {t: s[t + "_pages"].double() for t in "kv"}
    table, row, qs = s["table"].tolist(), 0, []
    for i, (past, new) in enumerate(s["spans"]):
        sl = slice(row, row + new)
        c, n = (s[t][past:past + new].double() for t in ("cos", "sin"))
        for t in "qk":
            x = s[t][sl].double()
            if case["norm"]:
                x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * s[t + "_gain"].double()
            x = torch.cat([_turn(x[..., :rd], c, n, case["pairs"]), x[..., rd:]], -1)
            if t == "q":
                qs.append(x)
        for b in range(past // page, (past + new - 1) // page + 1):
            lo, hi = max(past, b * page), min(past + new, b * page + page)
            there = slice(lo - b * page, hi - b * page)
            pages["k"][table[i][b], there] = x[lo - past:hi - past]
            pages["v"][table[i][b], there] = s["v"][row + lo - past:row + hi - past].double()
        row += new
    return {"q": torch.cat(qs), "k_pages": pages["k"], "v_pages": pages["v"]}


def _exact_attend(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    rep, row, parents = case["heads"] // case["kv"], 0, _parents(case) if case["width"] else None
    for i, (past, new) in enumerate(s["spans"]):
        need = (past + new + case["page"] - 1) // case["page"]
        k, v = (s[t][s["table"][i, :need].long()].flatten(0, 1)[:past + new] for t in ("k_pages", "v_pages"))
        hidden = torch.ones(new, past + new, dtype=torch.bool).triu(past + 1)
        for j, p in enumerate(parents[i] if parents is not None else []):
            hidden[j, past:] = hidden[p, past:] if p >= 0 else True
            hidden[j, past + j] = False
        hidden = hidden.cuda()
        for h in range(case["heads"]):
            S = s["q"][row:row + new, h].double() @ k[:, h // rep].double().t() * case["hd"] ** -0.5
            out[row:row + new, h] = torch.softmax(S.masked_fill(hidden, -math.inf), -1) @ v[:, h // rep].double()
        row += new
    return {"out": out}


def _exact_verify(case, s):
    """A sequence at a time, walking its tree."""
    tokens, at = s["tokens"].tolist(), s["cu"].tolist()
    u = s["u"].double().tolist() if s["u"] is not None else None
    path, kept, following = [], [], []
    for i, parents in enumerate(_parents(case)):
        base, node, walk = at[i], 0, [0]
        while True:
            p = s["probs"][base + node].double()
            left, token, norm = p, None, 1.0
            if u is None:
                token = int((p == p.max()).nonzero()[0])
            q = s["draft"][base + node].double() if s["draft"] is not None else None
            step = None
            for child in (j for j, up in enumerate(parents) if up == node):
                x = tokens[base + child]
                if u is None:
                    good = x == token
                else:  # left is what the rejected ones before leave, norm its sum
                    good = u[base + child] * (float(q[x]) if q is not None else 1.0) * norm < float(left[x])
                if good:
                    step = child
                    break
                if u is not None and q is not None:
                    left = (left - norm * q).clamp_min(0)
                    norm = float(left.sum())
                elif u is not None:
                    norm -= float(left[x])
                    left = left.clone()
                    left[x] = 0.0
            if step is None:
                break
            node = step
            walk.append(node)
        if u is not None:
            run_sum = (left if float(left.sum()) > 0 else p).cumsum(0)
            token = int((run_sum > u[base] * run_sum[-1]).nonzero()[0])
        kept.append(len(walk))
        path += walk + [-1] * (len(parents) - len(walk))
        following.append(token)
    return {"kept": _on_gpu(kept), "path": _on_gpu(path), "next": _on_gpu(following, torch.int64)}


def _exact_keep(case, s):
    pages, table, page = s["pages"].double(), s["table"].tolist(), case["page"]
    for i, ((past, _), path) in enumerate(zip(s["spans"], _paths(case))):
        for j, node in enumerate(path):
            a, b = past + node, past + j
            pages[:, table[i][b // page], b % page] = pages[:, table[i][a // page], a % page].clone()
    return {"pages": pages, "lengths": _on_gpu([p + len(path) for (p, _), path in zip(s["spans"], _paths(case))])}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend,
            "verify": _exact_verify, "keep": _exact_keep}[case["kind"]](case, s)
