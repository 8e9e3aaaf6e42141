"""The HIP kernel of ops.distill against the reference in 64 bits."""
import pytest
import torch

from metaopt_amd.ops import distill, lm

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(P, rows, V, K, dtype, top=torch.float32, missing=True, seed=0):
    torch.manual_seed(seed + V + K)
    R = P * rows
    x = (2 * torch.randn(R, V, device=DEV)).to(dtype)
    t = (3 * torch.randn(R, K, device=DEV)).to(top)
    index = torch.randint(0, V, (R, K), device=DEV, dtype=torch.int32)
    y = torch.randint(0, V, (R,), device=DEV, dtype=torch.int32)
    if missing and R > 3:
        y[1], y[2], y[R - 1] = -100, V, -1
        if K:
            index[0], index[2] = -1, -1                    # (row 2 has neither label nor teacher)
            index[3] = index[3, 0].clone()                 # one place K times
            index[R - 1, K // 2:] = V + 7
            y[3] = index[3, 0]
    return x, y, t, index


def _check(x, y, t, index, rows, tau, alpha, scale=1.0, weight=None):
    P, V = x.shape[0] // rows, x.shape[1]
    full = lambda v: v.double() if torch.is_tensor(v) else v  # noqa: E731
    xd = x.detach().double().requires_grad_(True)
    want = distill.distill_ref(xd, y, t.double(), index, rows, full(tau), full(alpha))
    w = torch.ones(P, device=DEV) if weight is None else weight
    gw, = torch.autograd.grad(want, xd, w.double() * scale)
    leaf = x.detach().requires_grad_(True)
    args = (y, t, index, rows, tau, alpha, scale)
    got = distill.distill_loss(leaf, *args, unit_weights=weight is None)
    g, = torch.autograd.grad(got, leaf, w)
    with torch.no_grad():
        alone = distill.distill_loss(leaf, *args)
    assert torch.equal(got, alone)
    # a row's sums have at most V / 256 + 64 additions in 32 bits, an exponential is good to 2^-20:
    # logs and quotients of them to e; the row's loss has 1 + 3 tau^2 such parts
    e = (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -18
    tt = tau.double().repeat_interleave(rows)[:, None] if torch.is_tensor(tau) else tau
    top = float(tau.max()) if torch.is_tensor(tau) else tau
    tol = rows * e * (1 + 3 * top * top) + 2.0 ** -20 * want.detach().abs()
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= tol).all()
    # gradient: one rounding, and e of the parts that it is the difference of
    u = torch.finfo(x.dtype).eps / 2
    xx = xd.detach()
    parts = (xx.softmax(1) + top * (xx / tt).softmax(1))
    ones = torch.ones_like(t, dtype=torch.float64)
    at = index.long().clamp(0, V - 1) if t.shape[1] else index.long()
    parts.scatter_add_(1, at, top * ones)
    parts.scatter_add_(1, y.long().clamp(0, V - 1)[:, None], torch.ones(len(y), 1, device=DEV, dtype=torch.float64))
    size = scale * w.double().abs().repeat_interleave(rows)[:, None]
    step = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    over = (g.double() - gw).abs() - (u * gw.abs() + 2 * e * size * parts + step)
    assert torch.isfinite(g).all() and over.max().item() <= 0, over.max().item()
    return got, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P,rows,V,K", [
    (1, 1, 1, 1), (1, 5, 7, 3), (2, 4, 512, 8), (1, 4, 1000, 64), (3, 4, 2047, 5), (2, 5, 2049, 1),
    (1, 4, 4096, 257), (1, 5, 8191, 40), (1, 4, 16390, 1024), (1, 4, 32000, 64), (1, 4, 50001, 16),
    (1, 4, 140001, 300)])
def test_distill_loss(P, rows, V, K, dtype):
    _check(*_case(P, rows, V, K, dtype), rows, 2.0, 0.6, scale=0.5)


@pytest.mark.parametrize("top", TYPES)
@pytest.mark.parametrize("tau,alpha", [(1.0, 0.5), (0.5, 1.0), (3.0, 0.0), (1.0, 1.0)])
def test_distill_mix_and_teacher_types(tau, alpha, top):
    x, y, t, index = _case(2, 6, 3001, 33, torch.bfloat16, top)
    _check(x, y, t, index, 6, tau, alpha)
    if alpha == 1.0:                      # labels do not matter, and neither what they say
        a = distill.distill_loss(x, y, t, index, 6, tau, alpha)
        b = distill.distill_loss(x, torch.full_like(y, -1), t, index, 6, tau, alpha)
        assert torch.equal(a, b)


def test_distill_per_trial_mix_and_weights():
    x, y, t, index = _case(3, 5, 2500, 20, torch.float32)
    tau = torch.tensor([1.0, 2.0, 4.0], device=DEV)
    alpha = torch.tensor([0.0, 0.5, 1.0], device=DEV)
    _check(x, y, t, index, 5, tau, alpha, weight=torch.tensor([2.0, 0.0, -1.5], device=DEV))
    _check(x, y, t, index, 5, tau, 0.3)
    _check(x, y, t, index, 5, 2.0, alpha)


@pytest.mark.parametrize("dtype", TYPES)
def test_distill_takes_views(dtype):
    """Rows of a wider tensor, at any element's alignment; columns that are not contiguous."""
    x, y, t, index = _case(1, 6, 1003, 9, dtype)
    want = _check(x, y, t, index, 6, 2.0, 0.5)
    wide = torch.full((6, 1100), 50.0, device=DEV, dtype=dtype)
    for off in (0, 1, 3, 8):
        wide.fill_(50.0)
        wide[:, off:off + 1003] = x
        got = _check(wide[:, off:off + 1003], y, t, index, 6, 2.0, 0.5)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    turned = x.t().contiguous().t()
    got = _check(turned, y, t.t().contiguous().t(), index, 6, 2.0, 0.5)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_distill_in_place_and_rows_of_nothing():
    x, y, t, index = _case(2, 6, 777, 12, torch.bfloat16)
    y[2], index[2] = -1, -1
    x[2] = float("nan")                                      # neither label nor teacher: not looked at
    leaf = x.clone().requires_grad_(True)
    h = leaf * 1
    loss = distill.distill_loss(h, y, t, index, 6, 2.0, 0.5, unit_weights=True, inplace=True)
    g, = torch.autograd.grad(loss.sum(), leaf)
    loss2 = distill.distill_loss(leaf, y, t, index, 6, 2.0, 0.5)
    g2, = torch.autograd.grad(loss2.sum(), leaf)
    assert torch.equal(loss, loss2) and torch.equal(g, g2) and torch.isfinite(loss).all()
    assert (g[2] == 0).all() and torch.equal(h.detach(), g)
    with pytest.raises(ValueError, match="leaf"):
        distill.distill_loss(leaf, y, t, index, 6, unit_weights=True, inplace=True)


def test_distill_masked_logits_and_teacher():
    """-inf logits (a masked vocabulary) take part in nothing; -inf teacher entries neither."""
    x, y, t, index = _case(1, 6, 900, 10, torch.float32, missing=False)
    x[:, 500:] = float("-inf")
    y %= 500
    index %= 500
    want = _check(x[:, :500].contiguous(), y, t, index, 6, 2.0, 0.5)
    leaf = x.requires_grad_(True)
    got = distill.distill_loss(leaf, y, t, index, 6, 2.0, 0.5)
    g, = torch.autograd.grad(got.sum(), leaf)
    torch.testing.assert_close(got, want[0], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(g[:, :500], want[1], rtol=1e-4, atol=1e-6)
    assert (g[:, 500:] == 0).all()
    t[:, 4:] = float("-inf")
    t[1] = float("-inf")
    cut = index.clone()
    cut[:, 4:], cut[1] = -1, -1
    with torch.no_grad():
        assert torch.equal(distill.distill_loss(x, y, t, index, 6), distill.distill_loss(x, y, t, cut, 6))


def test_distill_without_teacher_is_cross_entropy():
    x, y, _, _ = _case(2, 8, 4096, 1, torch.bfloat16, missing=False)
    none = torch.empty(16, 0, device=DEV), torch.empty(16, 0, device=DEV, dtype=torch.int32)
    got = distill.distill_loss(x, y, *none, 8, alpha=0.0)
    torch.testing.assert_close(got, lm.ce_eval(x.clone(), y, 8), rtol=1e-5, atol=1e-4)
    _check(x, y, *none, 8, 2.0, 0.5)


def test_distill_replays_in_a_graph():
    x, y, t, index = _case(2, 16, 1500, 8, torch.bfloat16)
    leaf, one = x.requires_grad_(True), torch.ones(2, device=DEV)

    def step(unit):
        loss = distill.distill_loss(leaf, y, t, index, 16, 2.0, 0.5, 1 / 16, unit_weights=unit)
        return [loss] + list(torch.autograd.grad(loss, leaf, one))
    for unit in (False, True):
        step(unit)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(unit)
        for i in range(3):
            with torch.no_grad():
                leaf.copy_(torch.randn(*x.shape, device=DEV))
                index.copy_(torch.randint(-3, 1500, index.shape, device=DEV, dtype=torch.int32))
            want = [w.detach().clone() for w in step(unit)]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_distill_empty_and_refusals():
    x = torch.zeros(0, 5, device=DEV, requires_grad=True)
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    loss = distill.distill_loss(x, e, torch.zeros(0, 2, device=DEV), torch.zeros(0, 2, dtype=torch.int32, device=DEV), 4)
    assert tuple(loss.shape) == (0,)
    assert tuple(torch.autograd.grad(loss.sum(), x)[0].shape) == (0, 5)
    with pytest.raises(ValueError, match="float64"):
        distill.distill_loss(torch.zeros(2, 5, device=DEV).double(), torch.zeros(2, dtype=torch.int32, device=DEV),
                             torch.zeros(2, 2, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV), 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("offset", [0.0, 24.0, -24.0, 1000.0, -1000.0, 30000.0, -30000.0])
def test_distill_loss_of_shifted_logits(offset, dtype):
    """Rows of which one logit stands out by 6 to 16, all shifted by ``offset``: the loss does not go with
    it.  (fp16 logits at 1000 and 30000 are multiples of 1/2 and 16: what they are is what counts.)

    z, the sum of exponentials relative to the largest logit m, is 1 and a rest: at most 17 values of a thread
    and 10 more sums round to 2^-24 of about 1, an exponential e^d is off by (2 |d| + 4) 2^-24 of itself.
    log z and x - m are rounded, and their difference."""
    torch.manual_seed(5)
    R, V, K, tau = 64, 1001, 6, 2.0
    x = torch.randn(R, V, device=DEV)
    y = torch.randint(0, V, (R,), device=DEV, dtype=torch.int32)
    x[torch.arange(R, device=DEV), y.long()] = torch.linspace(9, 19, R, device=DEV)
    x = (x + offset).to(dtype)
    index = torch.randint(0, V, (R, K), device=DEV, dtype=torch.int32)
    index[:, 0] = y
    top = torch.randn(R, K, device=DEV)
    top[:, 0] += 8
    d = x.double() - x.double().amax(1, keepdim=True)
    f, exp = 2.0 ** -24, lambda a: a.exp() * (2 * a.abs() + 4)  # noqa: E731

    def log_sum(a):
        z = a.exp().sum(1)
        return z.log(), f * (27 * z + exp(a).sum(1) - 4 + 2 * z.log().abs()) / z
    lz, tol = log_sum(d)
    dy = d.gather(1, y.long()[:, None])[:, 0]
    want, tol = lz - dy, tol + f * (2 * dy.abs() + 2 * (lz - dy).abs())
    with torch.no_grad():
        got = distill.distill_loss(x, y, top, index, 1, tau, 0.0).double()
    assert (got >= 0).all()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()
    # the teacher's: q_k = e^t_k / z_q, sum q_k (t_k - (x_k - m) / tau) - log z_q + log z_tau
    lt, tol = log_sum(d / tau)
    t = (top.double() - top.double().amax(1, keepdim=True)) / tau
    lq, tol_q = log_sum(t)
    part = t - d.gather(1, index.long()) / tau
    q = t.softmax(1)
    want = tau * tau * ((q * part).sum(1) - lq + lt)
    tol = tol + tol_q + f * ((q * part.abs() * (2 * t.abs() + 4 + 16)).sum(1) + (q * (t.abs() + part.abs()) * 4).sum(1)
                             + 2 * (lq.abs() + lt.abs() + (q * part).sum(1).abs()))
    with torch.no_grad():
        got = distill.distill_loss(x, y, top, index, 1, tau, 1.0).double()
    assert ((got - want).abs() <= tau * tau * tol).all(), ((got - want).abs() / (tau * tau * tol)).max().item()


def test_distill_loss_of_a_low_temperature_and_far_logits():
    """m / tau past 2^31: sums, losses and gradients are those of the differences to the largest logit."""
    x = 10000.0 + torch.randn(8, 500, device=DEV)
    y = torch.zeros(8, device=DEV, dtype=torch.int32)
    index = x.topk(3, 1).indices.int()
    top = torch.zeros(8, 3, device=DEV)
    leaf = x.requires_grad_(True)
    loss = distill.distill_loss(leaf, y, top, index, 8, 1e-6, 0.5)
    g, = torch.autograd.grad(loss.sum(), leaf)
    with torch.no_grad():
        alone = distill.distill_loss(leaf[:, :], y, top, index, 8, 1e-6, 0.0)
    # the student at this temperature is its largest logit alone: a tau (1 - 1 / 3), and -a tau / 3 twice
    assert torch.isfinite(loss).all() and torch.isfinite(g).all()
    soft = 0.5 * 1e-6 * (2.0 / 3)
    hard = 0.5 * (x.detach().double().softmax(1) - torch.nn.functional.one_hot(y.long(), 500))
    best = x.argmax(1, keepdim=True)
    want = hard.gather(1, best) + soft
    assert ((g.gather(1, best) - want).abs() <= 2.0 ** -20 * want.abs()).all()
    # tau^2 times differences of logits / tau of at most 4 / tau
    assert ((loss - 0.5 * alone).abs() <= 0.5 * 8 * 4e-6 + 2.0 ** -20 * alone).all()
