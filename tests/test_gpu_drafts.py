"""Verification of drafted tokens against a walk over each tree in float64 on the CPU."""
from __future__ import annotations

import math
import random

import pytest
import torch

from model.speculative import verify_drafts

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def walk(p, q, tokens, parents, u):
    """(path, next token) of one sequence: rows p, q of float64 lists' tensors, on the CPU.  The
    remaining distribution is formed anew, and divided by its sum, after every rejection."""
    def clean(x):
        return torch.where((x > 0) & torch.isfinite(x), x, torch.zeros_like(x))

    def first_largest(x):
        there = x[~x.isnan()]
        return int((x == there.max()).nonzero()[0]) if len(there) else -1
    node, path, n, V = 0, [0], len(tokens), p.shape[1]
    while True:
        left = clean(p[node])
        norm = 1.0
        step = None
        for j in range(node + 1, n):
            up = parents[j] if parents is not None else j - 1
            if up != node:
                continue
            x = tokens[j]
            if u is None:
                ok = x >= 0 and x == first_largest(p[node])
            elif not 0 <= x < V:
                ok = False
            elif q is None:
                ok = u[j] * norm < float(left[x])
            else:
                ok = u[j] * float(clean(q[node])[x]) * norm < float(left[x])
            if ok:
                step = j
                break
            if u is not None and q is not None:
                left = (left - norm * clean(q[node])).clamp_min(0)
                norm = float(left.sum())
            elif u is not None and 0 <= x < V:
                norm -= float(left[x])
                left = left.clone()
                left[x] = 0
        if step is None:
            break
        node = step
        path.append(node)
    if u is None:
        return path, first_largest(p[node])
    if not float(left.sum()) > 0:
        left = clean(p[node])
    if not float(left.sum()) > 0:
        return path, -1
    run = left.cumsum(0)
    past = ((run > u[0] * run[-1]) & (left > 0)).nonzero()
    return path, int(past[0]) if len(past) else int((left > 0).nonzero()[-1])


def trees(lens, width, seed):
    rng = random.Random(seed)
    return sum(([-1] + [rng.randrange(max(0, j - width), j) for j in range(1, n)] if n else [] for n in lens), [])


def make(dev, dtype, lens, V, width, mode, seed=0, noise=0.5):
    torch.manual_seed(seed)
    T = sum(lens)
    logits = torch.randn(T, V) * 3
    rough = logits + noise * torch.randn(T, V)
    p, q = logits.softmax(-1).to(dtype), rough.softmax(-1).to(dtype)
    parents = trees(lens, width, seed)
    tokens, at = torch.zeros(T, dtype=torch.int64), 0
    for n in lens:
        for j in range(1, n):
            up = at + parents[at + j]
            turn = sum(parents[at + i] == parents[at + j] for i in range(1, j))
            tokens[at + j] = (torch.multinomial(q[up].float(), 1)[0] if mode == "sample"
                              else rough[up].topk(min(turn + 1, V)).indices[-1])
        at += n
    u = torch.rand(T)
    return p, (q if mode == "sample" else None), tokens, parents, (None if mode == "greedy" else u)


def check(dev, lens, p, q, tokens, parents, u, behind=0):
    cu = ints([0] + torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist(), dev)
    on = lambda t: None if t is None else t.to(dev)
    up = None if parents is None else ints(parents, dev)
    kept, path, following = verify_drafts(on(p), on(tokens), cu, parents=up, draft_probs=on(q), uniforms=on(u))
    at = 0
    for i, n in enumerate(lens):
        sl = slice(at, at + n)
        if n == 0:
            assert int(kept[i]) == 0 and int(following[i]) == -1
            continue
        want, token = walk(p[sl].double(), None if q is None else q[sl].double(), tokens[sl].tolist(),
                           None if parents is None else parents[at:at + n], None if u is None else u[sl].double().tolist())
        assert path[sl].tolist() == want + [-1] * (n - len(want)), i
        assert (int(kept[i]), int(following[i])) == (len(want), token), i
        at += n
    assert path[at:].tolist() == [-1] * (len(path) - at)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,V", [([1], 100), ([5, 1, 0, 9], 6400), ([8] * 20, 257), ([60, 70], 1000), ([7, 3], 50257),
                                    ([12, 30], 16385), ([4, 4], 1), ([6], 7), ([3, 200], 33)])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("mode", ["sample", "certain", "greedy"])
@pytest.mark.parametrize("width", [1, 5])
def test_against_the_walk(dev, lens, V, dtype, mode, width):
    p, q, tokens, parents, u = make(dev, dtype, lens, V, width, mode, seed=V + width)
    check(dev, lens, p, q, tokens, parents, u)
    if width == 1:
        check(dev, lens, p, q, tokens, None, u)


@pytest.mark.gpu
def test_many_nodes_and_siblings(dev):
    """More nodes than are fetched at a time, more rejected siblings than are kept at hand, and the
    same token twice among siblings."""
    torch.manual_seed(1)
    V, n = 300, 2500
    for mode in ("sample", "certain", "greedy"):
        p, q, tokens, _, u = make(dev, F32, [n], V, 2, mode)
        wide = [-1] + [0] * 1500 + [random.Random(j).choice([0, 1500, j - 1]) for j in range(1501, n)]
        tokens = torch.randint(0, V, (n,))
        if u is not None:
            u[:1490] = 0.999999
        check(dev, [n], p, q, tokens, wide, u)
        check(dev, [n], p, q, tokens, None, u)


@pytest.mark.gpu
def test_edges(dev):
    """Tokens and parents that are none, numbers at 0 and 1, empty and senseless probabilities, ties."""
    V = 40
    p, q, tokens, parents, u = make(dev, F32, [6] * 8, V, 3, "sample")
    tokens[3], tokens[8], tokens[9] = -1, V, 2 ** 60
    parents[10], parents[14], parents[20] = 5, -3, 2 ** 31 - 1
    u[12:18] = 0.0
    u[18:24] = 1.0
    p[24:30] = 0.0
    p[30:36] = math.nan
    p[36], q[37], p[38, 5], p[39, :20] = -1.0, 0.0, math.inf, 0.25
    u[41] = math.nan
    for args in ((q, u), (None, u), (None, None)):
        check(dev, [6] * 8, p, args[0], tokens, parents, args[1])
    same = torch.full((4, 9), 0.125)
    check(dev, [4], same, None, torch.zeros(4, dtype=torch.int64), None, None)
    check(dev, [4], same, same, torch.zeros(4, dtype=torch.int64), None, torch.full((4,), 0.5))


@pytest.mark.gpu
def test_rows_behind_and_bounds(dev):
    p, q, tokens, parents, u = (x.to(dev) if torch.is_tensor(x) else x for x in make(dev, F32, [5, 6], 50, 2, "sample"))
    up = ints(parents, dev)
    kept, path, nxt = verify_drafts(p, tokens, ints([0, 5], dev), up, q, u)
    full = verify_drafts(p, tokens, ints([0, 5, 11], dev), up, q, u)
    assert int(kept[0]) == int(full[0][0]) and path[5:].tolist() == [-1] * 6 and torch.equal(path[:5], full[1][:5])
    assert [t.shape for t in verify_drafts(p, tokens, ints([0], dev), up, q, u)] == [(0,), (11,), (0,)]
    assert verify_drafts(p, tokens, ints([0], dev), up, q, u)[1].tolist() == [-1] * 11
    for ends in ([-5, 500, 2 ** 31 - 1], [0, 9, 3], [7, 7, 7]):
        assert verify_drafts(p, tokens, ints(ends, dev), up, q, u)[0].shape == (2,)
    empty = verify_drafts(p[:0], tokens[:0], ints([0, 0], dev), up[:0], q[:0], u[:0])
    assert empty[0].tolist() == [0] and empty[2].tolist() == [-1]


@pytest.mark.gpu
def test_strides_and_mixed_types(dev):
    p, q, tokens, parents, u = make(dev, F32, [9, 9], 101, 3, "sample")
    wide = torch.full((18, 150), 9.0)
    wide[:, 20:121] = p
    check(dev, [9, 9], wide.to(dev)[:, 20:121].cpu(), q, tokens, parents, u)
    cu = ints([0, 9, 18], dev)
    up, want = ints(parents, dev), None
    for pp in (p.to(dev), wide.to(dev)[:, 20:121], p.t().contiguous().to(dev).t()):
        got = verify_drafts(pp, tokens.to(dev), cu, up, q.to(dev), u.to(dev).double())
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_q = q.to(BF)
    kept = verify_drafts(p.to(dev), tokens.to(dev), cu, up, check_q.to(dev), u.to(dev))
    check(dev, [9, 9], p, check_q.float(), tokens, parents, u)
    again = verify_drafts(p.to(dev), tokens.to(dev), cu, up, check_q.float().to(dev), u.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(kept, again))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["sample", "certain"])
def test_the_targets_distribution(dev, mode):
    """The first accepted token, or the next one where none was, over many random numbers: counts of
    the target's probabilities (each within 5 standard deviations; with 12 tokens one in 10^5 runs
    would not be, and the numbers are the same on every run)."""
    torch.manual_seed(11)
    N, V = 40000, 12
    target, draft = torch.softmax(torch.randn(V), 0), torch.softmax(torch.randn(V), 0)
    p, q = target.expand(3 * N, V).contiguous().to(dev), draft.expand(3 * N, V).contiguous().to(dev)
    if mode == "sample":
        tokens = torch.multinomial(draft, 3 * N, replacement=True)
    else:
        tokens = torch.tensor([0, 4, 7]).repeat(N)
    up = ints([-1, 0, 0] * N, dev)
    kept, path, following = verify_drafts(p, tokens.to(dev), ints(list(range(0, 3 * N + 1, 3)), dev), up,
                                          q if mode == "sample" else None, torch.rand(3 * N, device=dev))
    rows = path.view(N, 3)[:, 1].long()
    first = torch.where(kept > 1, tokens.to(dev).view(N, 3).gather(1, rows.clamp_min(0)[:, None])[:, 0], following)
    count = torch.bincount(first, minlength=V).double().cpu()
    t = target.double()
    assert bool(((count - N * t).abs() <= 5 * (N * t * (1 - t)).sqrt()).all())
