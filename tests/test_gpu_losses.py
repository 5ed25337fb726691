"""The losses' kernels against their formulas in float64 on the CPU: vocabularies and rows
off 16-byte boundaries, labels that do not count, masked and lowest logits, empty sequences,
all three types, the gradients against the formulas' and against differences."""
from __future__ import annotations

import math

import pytest
import torch

from model.losses import balance_loss, preference_loss, token_logprobs

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = {F32: 2.0 ** -24, BF: 2.0 ** -8, F16: 2.0 ** -11}  # half a step of each type
IGN = -100


def _logits(T, V, dtype, dev, seed=0, pad=0, offset=0):
    torch.manual_seed(seed)
    whole = torch.randn(T, V + pad).mul_(3.0).to(dtype)
    labels = torch.randint(0, V, (T,))
    labels[torch.rand(T) < 0.3] = IGN
    store = torch.empty(whole.numel() + offset, dtype=dtype, device=dev)
    x = store[offset:].view(T, V + pad).copy_(whole)[:, :V]
    return x, labels.to(dev)


def _exact_logprobs(x, labels):
    lp = torch.log_softmax(x.detach().double().cpu(), -1)
    y = labels.cpu()
    p, hot = lp.exp(), torch.nn.functional.one_hot(y.clamp_min(0), x.shape[1])
    m = (y != IGN).double()
    return (lp * hot).nan_to_num(0.0, 0.0, 0.0).sum(-1) * m, (hot - p) * m[:, None]


def _lp_close(got, want):
    # lp = (x - max) - log(sum): an argument of the exponentials is off by |x - max| half
    # steps of fp32 and a sum of V = 2^16 terms in 256 chains by 2^8 of them: under 2^-15 together
    got = got.detach().double().cpu()
    assert bool(((got - want).abs() <= 2.0 ** -15 + 2.0 ** -22 * want.abs()).all())


def _grad_close(got, want, f, dtype):
    # one rounding to the type, and p off by the log-probability's error
    got, f = got.detach().double().cpu(), f.abs()
    bar = EPS[dtype] * want.abs() + 2.0 ** -15 * f + (2.0 ** -25 if dtype == F16 else 0.0)
    assert bool(((got - want).abs() <= bar).all()), float(((got - want).abs() - bar).max())


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,dtype,pad,offset", [
    (1, 1, F32, 0, 0), (3, 2, BF, 0, 0), (7, 7, F16, 0, 1), (5, 64, BF, 0, 3), (33, 6400, BF, 0, 0),
    (9, 6401, F16, 0, 0), (4, 6400, F32, 3, 1), (6, 50257, F32, 0, 0), (5, 50257, BF, 0, 5), (2, 255, F32, 0, 2),
    (300, 100, F16, 28, 0), (2, 131072, BF, 0, 0), (17, 2050, BF, 6, 7)])
def test_token_logprobs(dev, T, V, dtype, pad, offset):
    x, labels = _logits(T, V, dtype, dev, pad=pad, offset=offset)
    labels[0] = V - 1
    want, dwant = _exact_logprobs(x, labels)
    with torch.no_grad():
        _lp_close(token_logprobs(x, labels), want)
    x = x.detach().requires_grad_()
    lp = token_logprobs(x, labels)
    _lp_close(lp, want)
    g = torch.randn(T)
    got, = torch.autograd.grad(lp, x, g.to(dev))
    assert got.dtype == dtype and got.shape == x.shape
    _grad_close(got, dwant * g[:, None], g.double()[:, None], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_masked_logits(dev, dtype):
    """-inf and the type's lowest value as masks: of some columns, and of all but one, and a
    whole row of the lowest value, which is uniform."""
    low, V = torch.finfo(dtype).min, 100
    x = torch.randn(6, V).to(dtype)
    x[0, 50:], x[1, 50:] = -math.inf, low
    x[2, 1:], x[3, 1:] = -math.inf, low
    x[4] = low
    labels = torch.tensor([3, 3, 0, 0, 7, 1])
    want, dwant = _exact_logprobs(x, labels)
    x = x.to(dev).requires_grad_()
    lp = token_logprobs(x, labels.to(dev))
    _lp_close(lp, want)
    got, = torch.autograd.grad(lp.sum(), x)
    _grad_close(got, dwant, torch.ones(6, 1, dtype=torch.float64), dtype)


@pytest.mark.gpu
def test_labels_out_of_range_and_uncounted_rows(dev):
    x, _ = _logits(5, 40, F32, dev)
    x[1] = math.nan  # of a row that does not count: never read
    labels = torch.tensor([40, IGN, -1, 2 ** 40, 39], device=dev)
    x.requires_grad_()
    lp = token_logprobs(x, labels)
    assert lp.isnan().tolist() == [True, False, True, True, False] and float(lp[1]) == 0.0
    g, = torch.autograd.grad(lp.sum(), x)
    assert not bool(g[1].any()) and bool(g[4].isfinite().all())
    assert float(token_logprobs(x.detach(), torch.full((5,), 7, device=dev), 7).abs().sum()) == 0.0


@pytest.mark.gpu
def test_shapes_and_strides(dev):
    x, labels = _logits(24, 130, BF, dev)
    want = token_logprobs(x, labels)
    got = token_logprobs(x.view(2, 3, 4, 130), labels.view(2, 3, 4))
    assert got.shape == (2, 3, 4) and torch.equal(got.view(-1), want)
    turned = x.t().contiguous().t()
    assert torch.equal(token_logprobs(turned, labels), want)
    wide = torch.zeros(4, 9, 130, dtype=BF, device=dev)
    wide[:, :6] = x.view(4, 6, 130)  # rows that no one stride joins
    assert torch.equal(token_logprobs(wide[:, :6], labels.view(4, 6)).reshape(-1), want)
    leaf = wide.clone().requires_grad_()
    g, = torch.autograd.grad(token_logprobs(leaf[:, :6], labels.view(4, 6)).sum(), leaf)
    ref = x.clone().requires_grad_()
    h, = torch.autograd.grad(token_logprobs(ref, labels).sum(), ref)
    assert torch.equal(g[:, :6].reshape(24, 130), h) and not bool(g[:, 6:].any())
    assert token_logprobs(x[:0], labels[:0]).shape == (0,)


def _exact_preference(lp, counted, lengths, ref, beta, e, average):
    """(loss, rewards, factor of each row) in float64."""
    P, at, S, rows = len(lengths) // 2, 0, [], []
    for n in lengths:
        s = slice(at, at + n)
        c = max(int(counted[s].sum()), 1) if average else 1
        S.append(lp[s].sum() / c)
        rows.append((s, c))
        at += n
    r = beta * (torch.stack(S) - ref.double())
    z = r[:P] - r[P:]
    ls = torch.nn.functional.logsigmoid
    dz = (e * torch.sigmoid(z) - (1 - e) * torch.sigmoid(-z)) * beta / P
    f = torch.zeros_like(lp)
    for i, (s, c) in enumerate(rows):
        f[s] = (dz[i] if i < P else -dz[i - P]) / c
    return -((1 - e) * ls(z) + e * ls(-z)).mean(), r, f


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,V,dtype,e,average,behind", [
    ([1, 1], 8, F32, 0.0, False, 0), ([5, 0, 3, 9], 100, BF, 0.1, False, 4),
    ([700, 300, 1, 257, 64, 900], 64, F16, 0.0, True, 0), ([0, 0], 16, F32, 0.3, True, 2),
    ([3] * 400, 33, F32, 0.1, True, 5)])
def test_preference_loss(dev, lengths, V, dtype, e, average, behind):
    T, P = sum(lengths) + behind, len(lengths) // 2
    x, labels = _logits(T, V, dtype, dev, offset=1)
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    lp, dlp = _exact_logprobs(x, labels)
    counted = labels.cpu() != IGN
    base = _exact_preference(lp, counted, lengths, torch.zeros(2 * P), 1.0, e, average)[1]
    ref = (base + torch.randn(2 * P) * 5).float()
    loss, r, f = _exact_preference(lp, counted, lengths, ref, 0.3, e, average)
    x = x.detach().requires_grad_()
    got, chosen, rejected = preference_loss(x, labels, cu, ref.to(dev), 0.3, e, average)
    assert not chosen.requires_grad and not rejected.requires_grad
    # a sum's terms are off by 2^-15 each, and by 2^-22 of their size
    n = max(max(lengths), 1) if not average else 1
    bar = 0.3 * (2.0 ** -15 * n + 2.0 ** -22 * float(base.abs().max())) + 2.0 ** -23 * r.abs()
    off = (torch.cat([chosen, rejected]).double().cpu() - r).abs()
    assert bool((off <= bar).all())
    tol = 2 * float(bar.max()) + 2.0 ** -22 * float(loss)
    assert abs(float(got) - float(loss)) <= tol
    g = torch.full((), 512.0, device=dev)
    dx, = torch.autograd.grad(got, x, g)
    # a factor is off by what its sigmoid's argument is, at a slope of one
    want = dlp * f[:, None] * 512
    bar = tol * 512 * 0.3 / P * dlp.abs() + 2.0 ** -22 * want.abs()
    bar += EPS[dtype] * want.abs() + 2.0 ** -15 * 512 * f.abs()[:, None] + (2.0 ** -25 if dtype == F16 else 0)
    assert bool(((dx.double().cpu() - want).abs() <= bar).all())
    with torch.no_grad():
        again = preference_loss(x, labels, cu, ref.to(dev), 0.3, e, average)
    assert all(torch.equal(a, b) for a, b in zip(again, (got, chosen, rejected)))


@pytest.mark.gpu
def test_preference_differences(dev):
    """The loss along a direction, against its gradient: fp32 logits, a step of 2^-6, whose
    third-order term is under 2^-12 of the slope, and rounding of the loss 2^-23 / 2^-6."""
    x, labels = _logits(60, 50, F32, dev)
    cu = torch.tensor([0, 20, 35, 41, 60], dtype=torch.int32, device=dev)
    ref = torch.full((4,), -30.0, device=dev)
    x.requires_grad_()
    g, = torch.autograd.grad(preference_loss(x, labels, cu, ref, 0.1, 0.05)[0], x)
    with torch.no_grad():
        d = g / g.norm()
        up, down = (float(preference_loss(x + s * d, labels, cu, ref, 0.1, 0.05)[0]) for s in (2.0 ** -6, -2.0 ** -6))
    slope = (up - down) / 2.0 ** -5
    assert abs(slope - float(g.norm())) <= 2.0 ** -10 * abs(slope) + 2.0 ** -16


def _exact_balance(x, index, lengths, coef):
    x, index = x.detach().double().cpu(), index.cpu()
    E, at, loss, counts, g = x.shape[1], 0, 0.0, [], torch.zeros_like(x)
    real = max(sum(n > 0 for n in lengths), 1)
    for n in lengths:
        s = slice(at, at + n)
        counts.append(torch.bincount(index[s].reshape(-1), minlength=E))
        if n:
            f = counts[-1].double() / n
            loss += coef * E * float((f * x[s].mean(0)).sum()) / real
            g[s] = coef * E * f / (n * real)
        at += n
    return loss, torch.stack(counts), g


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,E,K,dtype,behind", [
    ([1], 1, 1, F32, 0), ([100], 4, 1, BF, 0), ([4097], 8, 2, BF, 0), ([333], 7, 3, F16, 0),
    ([20000], 64, 6, F32, 0), ([5, 0, 300, 1], 8, 2, F32, 9), ([64] * 50, 16, 4, BF, 0),
    ([700, 65], 300, 8, F32, 1), ([0, 0], 8, 2, BF, 3), ([50], 4096, 2, F32, 0)])
@pytest.mark.parametrize("packed", [False, True])
def test_balance_loss(dev, lengths, E, K, dtype, behind, packed):
    if not packed and (len(lengths) > 1 or behind):
        pytest.skip("one sequence of all rows")
    torch.manual_seed(0)
    T = sum(lengths) + behind
    x = torch.randn(T, E + 3, device=dev).softmax(-1).to(dtype)[:, :E].requires_grad_()  # rows a stride apart
    index = torch.randint(0, E, (T, K), device=dev)
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=dev) if packed else None
    loss, counts = balance_loss(x, index, 0.01, cu)
    want, wcounts, wg = _exact_balance(x, index, lengths, 0.01)
    assert torch.equal(counts.cpu(), wcounts if packed else wcounts[0])
    # sums of up to 2^8 terms in fp32 chains, then 64 bits, and one rounding
    assert abs(float(loss) - want) <= 2.0 ** -15 * abs(want)
    s = 2.0 ** 12  # a loss scale, for fp16
    g, = torch.autograd.grad(loss, x, torch.full((), s, device=dev))
    assert g.dtype == dtype
    bar = (EPS[dtype] + 2.0 ** -22) * wg * s + (2.0 ** -25 if dtype == F16 else 0.0)
    assert bool(((g.double().cpu() - wg * s).abs() <= bar).all())
    again = balance_loss(x.detach(), index, 0.01, cu)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts)


@pytest.mark.gpu
def test_balance_ignores_foreign_experts(dev):
    x = torch.rand(50, 8, device=dev)
    index = torch.randint(0, 8, (50, 2), device=dev)
    want = torch.bincount(index[:, 0], minlength=8)
    index[:, 1] = torch.tensor([-1, 8, 2 ** 40, -2 ** 40, 1 << 32], device=dev).repeat(10)
    assert torch.equal(balance_loss(x, index, 1.0)[1], want)


@pytest.mark.gpu
def test_no_rows_and_no_sequences(dev):
    x, y = torch.zeros(0, 10, device=dev, requires_grad=True), torch.zeros(0, dtype=torch.int64, device=dev)
    lp = token_logprobs(x, y)
    assert lp.shape == (0,) and torch.autograd.grad(lp.sum(), x)[0].shape == (0, 10)
    cu, ref = torch.zeros(3, dtype=torch.int32, device=dev), torch.tensor([1.0, 3.0], device=dev)
    loss, c, r = preference_loss(x, y, cu, ref, 0.5)
    assert abs(float(loss) - math.log1p(math.exp(-1.0))) <= 2.0 ** -22 and float(c) == -0.5 and float(r) == -1.5
    assert torch.autograd.grad(loss, x)[0].shape == (0, 10)
    s = torch.rand(7, 4, device=dev, requires_grad=True)
    k = torch.zeros(7, 1, dtype=torch.int64, device=dev)
    for bounds in ([0], [0, 0, 0]):
        loss, counts = balance_loss(s, k, 1.0, torch.tensor(bounds, dtype=torch.int32, device=dev))
        assert float(loss) == 0.0 and counts.shape == (len(bounds) - 1, 4) and not bool(counts.any())
        assert not bool(torch.autograd.grad(loss, s)[0].any())
    loss, counts = balance_loss(s[:0], k[:0], 1.0)
    assert float(loss) == 0.0 and not bool(counts.any())


@pytest.mark.gpu
def test_logits_past_32_bits(dev):
    """Rows past 2^31 elements, both ways."""
    V = 65536
    T = (1 << 31) // V + 6
    x = torch.zeros(T, V, dtype=BF, device=dev)
    tail = torch.randn(4, V, device=dev).to(BF)
    x[-4:] = tail
    labels = torch.full((T,), IGN, device=dev)
    labels[-4:] = torch.tensor([0, 5, V - 1, 77], device=dev)
    want, dwant = _exact_logprobs(tail, labels[-4:])
    x.requires_grad_()
    lp = token_logprobs(x, labels)
    _lp_close(lp[-4:], want)
    g, = torch.autograd.grad(lp.sum(), x)
    _grad_close(g[-4:], dwant, torch.ones(4, 1, dtype=torch.float64), BF)
    assert not bool(g[:100].any())
