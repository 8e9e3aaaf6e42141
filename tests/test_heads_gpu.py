"""The HIP kernels of ops.heads against the references in 64 bits.

Tolerances count roundings.  ``u`` is half a step of the 16-bit type (eps / 2); every output is
rounded once (u |value|), probabilities and score gradients once more on their way into a matrix
product (u of each term's magnitude), the rest is 32-bit arithmetic, whose bounds are written where
they are used."""
import math

import pytest
import torch

from metaopt_amd.ops import heads

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float16


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(*shape, dtype, scale=1.0, mean=0.0):
    return (torch.randn(*shape, device=DEV) * scale + mean).to(dtype)


def _within(got, want, tol, what):
    """|got - want| <= tol everywhere (and nothing but numbers)."""
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    over = ((got.double() - want).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0, f"{what}: {over} over its tolerance"


# ------------------------------------------------------------------------------- norm + rotation
def _qk_case(P, n, T, H, KV, D, dtype):
    torch.manual_seed(P + 10 * T + H)
    cos, sin = heads.rope_tables(T + 3, D, device=DEV)
    return (_rand(n * T, (H + 2 * KV) * D, dtype=dtype), _rand(P, D, dtype=dtype, scale=0.3, mean=1),
            _rand(P, D, dtype=dtype, scale=0.3, mean=1), cos, sin)


def _qk_oracle(qkv, wq, wk, cos, sin, T, H, KV, il, dq, dk, dv, eps=1e-5):
    """Reference outputs and gradients in 64 bits with their tolerances."""
    u = _u(qkv.dtype)
    x, a, b = (t.detach().double().requires_grad_(True) for t in (qkv, wq, wk))
    q, k, v = heads.qk_norm_rope_ref(x, a, b, cos.double(), sin.double(), T, H, KV, eps, il)
    grads = torch.autograd.grad([q, k, v], [x, a, b], [t.double() for t in (dq, dk, dv)])
    # a head's sum of D squares, root, two products and the rotation: under 2^-18 of its largest
    # value, one rounding behind them
    outs = [(t.detach(), u * t.detach().abs() + 2.0 ** -18 * t.detach().abs().amax(-1, keepdim=True))
            for t in (q, k, v)]
    # dx = r (u - x^ m): both terms are at most |w| |dy| r resp. |x^| max|w dy| sqrt(D) r
    n, D, P = qkv.shape[0] // T, wq.shape[1], wq.shape[0]
    xs = x.detach().view(n * T, H + 2 * KV, D)
    r = (xs.square().mean(-1, keepdim=True) + eps).rsqrt()
    d = torch.cat([dq, dk, dv], 1).double().transpose(1, 2).reshape(n * T, H + 2 * KV, D)
    top = d.abs().amax(-1, keepdim=True) * 1.5 * float(torch.cat([wq, wk]).detach().abs().max())
    size = r * top * (1 + (xs * r).abs().amax(-1, keepdim=True))
    dx_tol = u * grads[0].abs() + (2.0 ** -17 * size).expand_as(xs).reshape(n * T, -1)
    # dw: every lane adds its terms one by one (under 4096 here), then a tree: 2^-24 a step of the
    # magnitudes' sum; the terms themselves are good to 2^-20
    mags = (d.abs().amax(-1, keepdim=True) * 1.5 * (xs * r).abs())
    per = mags.view(P, -1, H + 2 * KV, D).sum(1)
    steps = 2.0 ** -20 + F32 * (n * T * (H + 2 * KV) / 16 / P + 64)
    dw_tol = [u * g.abs() + steps * per[:, s].sum(1) for g, s in
              zip(grads[1:], (slice(0, H), slice(H, H + KV)))]
    return outs, list(zip(grads, [dx_tol] + dw_tol))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("P,n,T,H,KV,D", [
    (1, 1, 1, 1, 1, 64), (2, 4, 7, 4, 2, 64), (3, 3, 33, 3, 3, 128), (1, 2, 130, 8, 1, 128),
    (8, 16, 64, 12, 12, 64), (1, 1, 1, 5, 5, 128)])
def test_qk_norm_rope(P, n, T, H, KV, D, il, dtype):
    qkv, wq, wk, cos, sin = _qk_case(P, n, T, H, KV, D, dtype)
    d = [_rand(n, h, T, D, dtype=dtype) for h in (H, KV, KV)]
    leaves = [t.requires_grad_(True) for t in (qkv, wq, wk)]
    out = heads.qk_norm_rope(*leaves, cos, sin, T, H, KV, il=il)
    grads = torch.autograd.grad(out, leaves, d)
    outs, back = _qk_oracle(qkv, wq, wk, cos, sin, T, H, KV, il, *d)
    assert torch.equal(out[2].double(), outs[2][0])
    for got, (want, tol), what in zip(list(out) + list(grads), outs + back,
                                      ("q", "k", "v", "dqkv", "dwq", "dwk")):
        _within(got, want, tol, what)


def test_qk_norm_rope_takes_rows_of_a_wider_activation_and_zero_rows():
    T, H, D = 5, 2, 64
    cos, sin = heads.rope_tables(T, D, device=DEV)
    wide = _rand(4 * T, 3 * H * D + 24, dtype=BF)
    odd = _rand(4 * T, 3 * H * D + 3, dtype=BF)
    w = _rand(2, D, dtype=BF)
    for src in (wide[:, 8:-16], odd[:, :-3], wide[:, 1:3 * H * D + 1]):
        got = heads.qk_norm_rope(src, w, w, cos, sin, T, H)
        want = heads.qk_norm_rope(src.contiguous(), w, w, cos, sin, T, H)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    zero = torch.zeros(4 * T, 3 * H * D, device=DEV, dtype=BF, requires_grad=True)
    out = heads.qk_norm_rope(zero, w, w, cos, sin, T, H)
    assert all((t == 0).all() for t in out)
    g, = torch.autograd.grad(out, [zero], [torch.zeros_like(t) for t in out])
    assert (g == 0).all()
    empty = heads.qk_norm_rope(zero[:0], w, w, cos, sin, T, H)
    assert [tuple(t.shape) for t in empty] == [(0, H, T, D)] * 3


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T,D,il", [(1, 64, True), (3, 128, False), (1, 128, True), (2, 64, False)])
def test_qk_norm_rope_cached(T, D, il, dtype):
    torch.manual_seed(T + D)
    P, n, H, KV, cap = 2, 6, 4, 2, 9
    cos, sin = heads.rope_tables(8, D, device=DEV)               # one position less than the cache
    rows = _rand(n * T, (H + 2 * KV) * D, dtype=dtype)
    wq, wk = (_rand(P, D, dtype=dtype, scale=0.3, mean=1) for _ in range(2))
    start = torch.tensor([0, 5, -1, 7, 8, 1 << 30], dtype=torch.int32, device=DEV)
    caches = [_rand(n, cap, KV, D, dtype=dtype).transpose(1, 2) for _ in range(2)]   # strided
    want = [c.clone() for c in caches]
    q = heads.qk_norm_rope_cached(rows, wq, wk, cos, sin, T, H, *caches, start, il=il)
    ref = [c.double().cpu() for c in want]
    ref_q = heads.qk_norm_rope_cached(rows.double().cpu(), wq.double().cpu(), wk.double().cpu(), cos.cpu(),
                                      sin.cpu(), T, H, *ref, start.cpu(), il=il)
    u = _u(dtype)
    for got, wanted in ((q, ref_q), (caches[0], ref[0]), (caches[1], ref[1])):
        wanted = wanted.to(DEV)
        _within(got, wanted, u * wanted.abs() + 2.0 ** -18 * wanted.abs().amax(-1, keepdim=True), "cached")
    for b in range(n):                                            # every other place is untouched
        mine = set(range(int(start[b]), int(start[b]) + T)) & set(range(8))
        other = [p for p in range(cap) if p not in mine]
        for c, w in zip(caches, want):
            assert torch.equal(c[b, :, other], w[b, :, other])


def test_heads_refuse_on_the_gpu():
    cos, sin = heads.rope_tables(2, 32, device=DEV)
    x = torch.zeros(2, 96, device=DEV, dtype=BF)
    w = torch.ones(1, 32, device=DEV, dtype=BF)
    with pytest.raises(ValueError, match="head dimensions"):
        heads.qk_norm_rope(x, w, w, cos, sin, 2, 1)
    q = torch.zeros(1, 1, 2, 64, device=DEV)
    with pytest.raises(ValueError, match="bfloat16"):
        heads.window_attention(q, q, q)
    with pytest.raises(ValueError, match="is on"):
        heads.window_attention(q.half(), q.half().cpu(), q.half().cpu())


# ------------------------------------------------------------------------------- attention
def _attention_oracle(q, k, v, do, window, sinks, start, lengths, scale=None):
    """(o, dq, dk, dv) in 64 bits and their tolerances."""
    u = _u(q.dtype)
    B, H, Tq, D = q.shape
    KV, Tk = k.shape[1:3]
    G = H // KV
    scale = 1 / math.sqrt(D) if scale is None else scale
    first = start if torch.is_tensor(start) else torch.full(
        (B,), Tk - Tq if start is None else start, device=DEV, dtype=torch.int32)
    last = (first + Tq if lengths is None else lengths)
    see = heads.window_mask(Tq, Tk, window or Tq + Tk, sinks, first, last, DEV)[:, None, None]
    real = see.any(-1, keepdim=True)
    live = (torch.arange(Tk, device=DEV) < last[:, None])[:, None, :, None]
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    kd, vd = (torch.where(live, t.detach().double(), zero)[:, :, None] for t in (k, v))
    qd = torch.where(real, q.detach().double().view(B, KV, G, Tq, D), zero)
    s = (qd @ kd.transpose(-1, -2)) * scale
    p = s.masked_fill(~see, -math.inf).masked_fill(~real, 0).softmax(-1) * real * see
    o = p @ vd
    # scores: D products added in 32 bits; p's relative error is twice that (itself and the sum),
    # the exponential's own and the reference point's 2^-20
    es = (2 * D * F32 * scale * (qd.abs() @ kd.abs().transpose(-1, -2)) * see).amax() + 2.0 ** -20
    # fp16 below 2^-14 rounds by up to 2^-25, whatever the value: the forward's probabilities are
    # relative to a sum of at least 1, the backward's 2^12 times theirs, score gradients as they are
    # (bf16: an exponential under 2^-126 is 0)
    sub = 2.0 ** -25 if q.dtype == FP else 2.0 ** -126
    o_tol = u * o.abs() + (u + es) * (p @ vd.abs()) + sub * (see.double() @ vd.abs())
    rows = lambda t: t.reshape(B, H, Tq, D).transpose(1, 2).reshape(B * Tq, H * D)  # noqa: E731
    # (fp16 values below 2^-14 are multiples of 2^-24: rounding is off by up to half of that, 2^-25)
    res = [(rows(o), rows(o_tol) + torch.finfo(q.dtype).tiny * u)]
    if do is None:
        return res
    # the backward adds a score's products onto minus its row's log-sum (in base 2, at most the largest
    # score's and the logarithm of the keys): a rounding of that size for each 16 of D, and two more
    es = es + (D / 16 + 2) * F32 * (1.4427 * ((s * see).abs().amax() + math.log(Tk)) + 1)
    dod = torch.where(real, do.detach().double().view(B, Tq, H, D).transpose(1, 2).reshape(B, KV, G, Tq, D), zero)
    dv = (p.transpose(-1, -2) @ dod).sum(2)
    dv_tol = u * dv.abs() + (u + es) * (p.transpose(-1, -2) @ dod.abs()).sum(2)
    seen = (see & real).double().expand(B, KV, G, Tq, Tk)
    dv_tol = dv_tol + sub * (2.0 ** -12 if q.dtype == FP else 1) * (seen.transpose(-1, -2) @ dod.abs()).sum(2)
    dp = dod @ vd.transpose(-1, -2)
    delta = (dod * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # dP and D: D products in 32 bits; D is formed from o before its rounding
    e_ds = p * (2 * D * F32 * (dod.abs() @ vd.abs().transpose(-1, -2))
                + (dod.abs() * (o_tol - u * o.abs())).sum(-1, keepdim=True)) + (u + es) * ds.abs()
    e_ds = e_ds + seen * (sub + 2.0 ** -126 * (dp - delta).abs())
    dq, dq_e = ds @ kd * scale, e_ds @ kd.abs() * scale
    dk = (ds.transpose(-1, -2) @ qd).sum(2) * scale
    dk_e = (e_ds.transpose(-1, -2) @ qd.abs()).sum(2) * scale
    tiny = torch.finfo(q.dtype).tiny * u                      # fp16: half a subnormal step
    return res + [(dq.reshape(B, H, Tq, D), (u * dq.abs() + dq_e).reshape(B, H, Tq, D) + tiny),
                  (dk, u * dk.abs() + dk_e + tiny), (dv, dv_tol + tiny)]


def _attention_case(B, H, KV, Tq, Tk, D, dtype, seed=0):
    torch.manual_seed(seed + Tq + Tk + H)
    return (_rand(B, H, Tq, D, dtype=dtype), _rand(B, KV, Tk, D, dtype=dtype),
            _rand(B, KV, Tk, D, dtype=dtype), _rand(B * Tq, H * D, dtype=dtype))


def _check(q, k, v, do, window, sinks, start=None, lengths=None, scale=None):
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = heads.window_attention(*leaves, window, sinks, scale, start, lengths)
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():
        plain = heads.window_attention(*leaves, window, sinks, scale, start, lengths)
    want = _attention_oracle(q, k, v, do, window, sinks, start, lengths, scale)
    for got, (w, tol), what in zip((o,) + grads, want, ("o", "dq", "dk", "dv")):
        _within(got, w, tol, what)
    _within(plain, *want[0], "o without gradients")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,window,sinks", [
    (1, 1, 0), (1, 5, 3), (2, 1, 1), (31, 7, 2), (32, 32, 0), (33, 16, 40), (64, None, 0),
    (65, 64, 1), (127, 20, 5), (128, None, 0), (129, 100, 4), (200, 33, 33), (257, 64, 65),
    (300, 1, 0), (300, 1, 4), (300, 299, 1), (300, 300, 4), (300, 2000, 4), (333, 32, 130)])
def test_window_attention_self(T, window, sinks, D, dtype):
    _check(*_attention_case(2, 3, 3, T, T, D, dtype), window, sinks)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("H,KV,D,T,window,sinks", [
    (4, 2, 64, 150, 40, 3), (6, 1, 128, 140, 33, 0), (8, 1, 64, 70, None, 0), (5, 5, 128, 129, 128, 2)])
def test_window_attention_shared_heads_and_padding(H, KV, D, T, window, sinks, dtype):
    q, k, v, do = _attention_case(6, H, KV, T, T, D, dtype)
    lengths = torch.tensor([0, 1, T, T // 2, T - 1, T + 50], dtype=torch.int32, device=DEV)
    _check(q, k, v, do, window, sinks, lengths=lengths)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,H,KV,D,T,window,sinks", [
    (1, 2, 1, 64, 1100, 100, 4), (1, 1, 1, 128, 1500, 200, 70), (3, 4, 2, 128, 700, 256, 2),
    (1, 4, 1, 64, 1025, 1000, 1), (140, 2, 2, 64, 600, 70, 9)])
def test_window_attention_in_shares(B, H, KV, D, T, window, sinks, dtype):
    """Queries of a key block, and those far behind the sinks, shared among workgroups."""
    _check(*_attention_case(B, H, KV, T, T, D, dtype), window, sinks)


@pytest.mark.parametrize("Tq,Tk,H,KV,D", [
    (1, 1, 2, 2, 64), (1, 500, 4, 4, 64), (1, 700, 8, 1, 128), (2, 300, 6, 2, 64), (5, 333, 8, 4, 128),
    (16, 129, 1, 1, 64), (17, 400, 3, 1, 64), (40, 200, 4, 2, 128), (1, 3000, 16, 1, 64),
    (3, 2600, 15, 3, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (64, 4), (1, 0), (200, 70)])
def test_window_attention_over_a_cache(Tq, Tk, H, KV, D, window, sinks):
    q, k, v, do = _attention_case(5, H, KV, Tq, Tk, D, BF if D == 64 else FP)
    _check(q, k, v, do, window, sinks)
    start = torch.tensor([0, Tk - Tq, Tk // 2, -1, Tk - 1], dtype=torch.int32, device=DEV)
    _check(q, k, v, do, window, sinks, start=start)
    _check(q, k, v, do, window, sinks, start=start, scale=0.3,
           lengths=torch.tensor([Tq, Tk, Tk // 2 + 1, Tk, 0], dtype=torch.int32, device=DEV))


def test_window_attention_ignores_what_padding_holds():
    q, k, v, do = _attention_case(3, 4, 2, 100, 100, 64, BF)
    lengths = torch.tensor([70, 0, 100], dtype=torch.int32, device=DEV)
    want = []
    for bad in (0.0, float("nan"), float("inf")):
        leaves = []
        for t in (q, k, v):
            t = t.clone()
            t[0, :, 70:], t[1] = bad, bad
            leaves.append(t.requires_grad_(True))
        d = do.clone()
        d.view(3, 100, -1)[0, 70:], d.view(3, 100, -1)[1] = bad, bad
        o = heads.window_attention(*leaves, 30, 4, lengths=lengths)
        want.append([o] + list(torch.autograd.grad(o, leaves, d)))
        step = heads.window_attention(leaves[0][:, :, 69:70], leaves[1], leaves[2], 30, 4,
                                      start=lengths - 1)
        want[-1].append(step)
    for other in want[1:]:
        assert all(torch.equal(a, b) for a, b in zip(want[0], other))
    assert (want[0][0].view(3, 100, -1)[0, 70:] == 0).all() and (want[0][0].view(3, 100, -1)[1] == 0).all()
    assert (want[0][1][0, :, 70:] == 0).all() and (want[0][2][1] == 0).all()


def test_window_attention_takes_strides_and_broadcast_heads():
    torch.manual_seed(3)
    B, T, H, KV, D = 2, 90, 4, 2, 64
    rows = _rand(B, T, (H + 2 * KV) * D, dtype=BF)
    q, k, v = (rows[..., a:b].view(B, T, -1, D).transpose(1, 2) for a, b in
               ((0, H * D), (H * D, (H + KV) * D), ((H + KV) * D, (H + 2 * KV) * D)))
    do = _rand(B * T, H * D, dtype=BF)
    _check(q.detach(), k.detach(), v.detach(), do, 17, 2)
    # one key head expanded over the batch: its gradient is the sum
    one = _rand(1, 1, T, D, dtype=BF).requires_grad_(True)
    o = heads.window_attention(q, one.expand(B, KV, T, D), v, 17, 2)
    g, = torch.autograd.grad(o, [one], do)
    full = one.detach().expand(B, KV, T, D).contiguous().requires_grad_(True)
    gf, = torch.autograd.grad(heads.window_attention(q, full, v, 17, 2), [full], do)
    _within(g, gf.double().sum((0, 1), keepdim=True), 8 * _u(BF) * gf.double().abs().sum((0, 1), keepdim=True), "dk")
    # rows that are not 16-byte aligned, and heads in another order of dimensions
    flat = _rand(B * H * T * D + 1, dtype=BF)[1:].view(B, H, T, D)
    a = heads.window_attention(flat, k, v, 17, 2)
    assert torch.equal(a, heads.window_attention(flat.clone(), k, v, 17, 2))
    cols = _rand(B, H, D, T, dtype=BF).transpose(2, 3)
    assert torch.equal(heads.window_attention(cols, k, v, 17, 2),
                       heads.window_attention(cols.contiguous(), k, v, 17, 2))


def test_window_attention_large_scores_and_equal_scores():
    """Scores of both signs up to hundreds (a softmax of one key) and all-equal scores."""
    q, k, v, do = _attention_case(1, 2, 2, 200, 200, 64, BF)
    _check(q * 8, k * 8, v, do, 90, 4)
    _check(torch.zeros_like(q), k, v, do, 90, 4)
    _check(-k[:, :, :].clone() * 20, k * 20, v, do, 50, 0)
    for scale in (1e-6, 1e-20, 4.0):
        _check(*_attention_case(1, 2, 1, 300, 300, 64, FP), 90, 4, scale=scale)
        _check(*_attention_case(1, 2, 1, 300, 300, 128, BF), 90, 4, scale=scale)


def test_window_attention_is_deterministic_and_replays_in_a_graph():
    q, k, v, do = _attention_case(4, 6, 2, 300, 300, 64, BF)
    lengths = torch.tensor([300, 7, 0, 155], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        o = heads.window_attention(*leaves, 40, 4, lengths=lengths)
        return [o] + list(torch.autograd.grad(o, leaves, do))
    first = [t.detach().clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(_rand(*q.shape, dtype=BF))
            lengths.copy_(torch.tensor([300 - i, 7 + i, i, 150], dtype=torch.int32, device=DEV))
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_empty_batches_and_caches():
    q = torch.zeros(0, 2, 3, 64, device=DEV, dtype=BF, requires_grad=True)
    o = heads.window_attention(q, q, q, 2, 1)
    assert tuple(o.shape) == (0, 128)
    assert tuple(torch.autograd.grad(o.sum(), q)[0].shape) == tuple(q.shape)
    q, k = torch.ones(2, 2, 3, 64, device=DEV, dtype=BF), torch.ones(2, 2, 0, 64, device=DEV, dtype=BF)
    assert (heads.window_attention(q, k, k) == 0).all()


def test_offsets_past_32_bits():
    """A cache whose last sequence and rows lie beyond 2^31 elements."""
    D, Tk, n = 128, 1 << 20, 18
    k = torch.zeros(n, 1, Tk, D, device=DEV, dtype=BF)
    assert k.numel() > (1 << 31)
    torch.manual_seed(1)
    tail = _rand(1, 1, 600, D, dtype=BF)
    k[-1, :, Tk - 600:] = tail
    q = _rand(n, 2, 1, D, dtype=BF)
    o = heads.window_attention(q, k, k, 500, 2)
    want = _attention_oracle(q[-1:], torch.cat([k[-1:, :, :2], tail], 2), torch.cat([k[-1:, :, :2], tail], 2),
                             None, 500, 2, None, None)
    _within(o[-1:], *want[0], "o")
    x, w = _rand(n, 4 * D, dtype=BF), torch.ones(1, D, device=DEV, dtype=BF)
    cos, sin = heads.rope_tables(2, D, device=DEV)
    big = (torch.cat([cos] * 1)[:1].expand(Tk, -1).contiguous(), sin[:1].expand(Tk, -1).contiguous())
    kc = heads.qk_norm_rope(x, w, w, cos, sin, 1, 2, 1)
    v = torch.zeros_like(k)
    heads.qk_norm_rope_cached(x, w, w, *big, 1, 2, k, v,
                              torch.full((n,), Tk - 1, device=DEV, dtype=torch.int32))
    assert torch.equal(v[:, :, Tk - 1], kc[2][:, :, 0])
    assert torch.equal(k[:, :, Tk - 1], kc[1][:, :, 0])          # (the angle of every row is 0)
    assert not v[:, :, :Tk - 1].any()


def test_cached_heads_with_tables_of_no_position():
    """Every token is outside tables that hold no position: zeros, and the caches stay."""
    rows, w = _rand(4, 6 * 64, dtype=BF), torch.ones(1, 64, device=DEV, dtype=BF)
    caches = [_rand(2, 2, 4, 64, dtype=BF) for _ in "kv"]
    before = [c.clone() for c in caches]
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    q = heads.qk_norm_rope_cached(rows, w, w, *heads.rope_tables(0, 64, device=DEV), 2, 2, *caches, start)
    assert tuple(q.shape) == (2, 2, 2, 64) and not q.any()
    assert all(torch.equal(a, b) for a, b in zip(caches, before))


def test_forward_mode_is_refused():
    """(a dual tensor does not require a gradient, and its tangent must not get lost)"""
    q = _rand(1, 2, 4, 64, dtype=BF)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            heads.window_attention(dual, q, q)
        heads.window_attention(q, q, q)


def _eighths(*shape, most):
    """fp16 values that are multiples of 1/8 of at most ``most``: exact at any power of two in range."""
    return (torch.randn(*shape, device=DEV) * 8).round().clamp(-8 * most, 8 * most).div(8).half()


@pytest.mark.parametrize("B,H,KV,T,D,window,sinks", [
    (2, 3, 3, 300, 64, 100, 4), (1, 4, 1, 300, 128, None, 0), (1, 4, 2, 1100, 64, 100, 4), (1, 4, 1, 1300, 128, 1000, 2),
    (1, 2, 2, 40, 64, None, 0)])
@pytest.mark.parametrize("power", [-13, -10, 8])
def test_window_attention_fp16_gradients_follow_the_incoming_size(power, B, H, KV, T, D, window, sinks):
    """Gradients are linear in the output's: do 2^power gives 2^power of what do gives, exactly before the
    last rounding, if score gradients lose nothing on the way whatever their size.  That rounding is off by
    u of the value or, in the subnormal range, by 2^-25, once on either side.

    (Scores 8 q k / 64 of size 1; queries, keys and 8 / 64 leave gradients of a size of about 1 for do of
    size 1, so at 2^-13 a score gradient is about 2^-20, the gradients about 2^-13.)"""
    torch.manual_seed(T + D)
    q, k, v = (_rand(B, h, T, D, dtype=FP, scale=s) for h, s in ((H, 0.125), (KV, 0.125), (KV, 1.0)))
    do = _eighths(B * T, H * D, most=4)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = heads.window_attention(*leaves, window, sinks, scale=8.0)
    want, got = (torch.autograd.grad(o, leaves, d, retain_graph=True) for d in (do, do * 2.0 ** power))
    assert torch.equal(do * 2.0 ** power * 2.0 ** -power, do)
    for g, w, name in zip(got, want, ("dq", "dk", "dv")):
        w, back = w.double(), g.double() * 2.0 ** -power
        tol = 2 * _u(FP) * w.abs() * (1 + _u(FP)) + 2.0 ** -25 * (1 + 2.0 ** -power)
        _within(back, w, tol, name)


@pytest.mark.parametrize("D,T,window", [(64, 700, 90), (128, 900, 200)])
def test_window_attention_fp16_gradients_of_rows_of_unlike_sizes(D, T, window):
    """Rows of do of 1 and of 2^-13 in one sequence: dq of the small ones, and dk of keys that only these
    see, are what they are where all rows are small."""
    torch.manual_seed(T)
    q, k, v = (_rand(1, 2, T, D, dtype=FP, scale=s) for s in (0.125, 0.125, 1.0))
    do = _eighths(T, 2 * D, most=4)
    small, mixed = do * 2.0 ** -13, do.clone()
    mixed[:T // 2] *= 2.0 ** -13
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = heads.window_attention(*leaves, window, scale=8.0)
    a, b = (torch.autograd.grad(o, leaves, d, retain_graph=True) for d in (mixed, small))
    cut = T // 2 - window                           # keys seen by queries in front of T / 2 only
    assert torch.equal(a[0][:, :, :T // 2], b[0][:, :, :T // 2])
    assert torch.equal(a[1][:, :, :cut], b[1][:, :, :cut]) and a[1][:, :, :cut].any()
    assert torch.equal(a[2][:, :, :cut], b[2][:, :, :cut])


@pytest.mark.parametrize("T", [60, 500])
def test_window_attention_fp16_large_score_gradients(T):
    """Score gradients past fp16's largest value (65504), whose sums of products over 16 are not."""
    q, k, v, do = _attention_case(1, 2, 2, T, T, 64, FP)
    _check(q, k, (v * 32).half(), (do * 256).half(), 50, 2, scale=0.0625)


def _once_rounded(q, k, v, do, window, sinks, scale=None, start=None, lengths=None):
    """(want, tolerance) of o (and dq, dk, dv) where outputs are rounded to 16 bits and nothing in front of
    them is: probabilities and score gradients enter their products in two 16-bit pieces, off by u u."""
    u, (B, H, Tq, D), (KV, Tk) = _u(q.dtype), q.shape, k.shape[1:3]
    want = [w for w, _ in _attention_oracle(q, k, v, do, window, sinks, start, lengths, scale)]
    scale = 1 / math.sqrt(D) if scale is None else scale
    first = torch.full((B,), Tk - Tq, device=DEV) if start is None else start
    see = heads.window_mask(Tq, Tk, window or Tq + Tk, sinks, first, first + Tq if lengths is None else lengths,
                            DEV)[:, None, None]
    some = see.any(-1, keepdim=True)
    kd, vd = k.detach().double()[:, :, None], v.detach().double()[:, :, None]
    qd = q.detach().double().view(B, KV, H // KV, Tq, D)
    s = (qd @ kd.transpose(-1, -2)) * scale
    p = s.masked_fill(~see, -math.inf).masked_fill(~some, 0).softmax(-1) * see
    o = p @ vd
    # a score is D products summed in 32 bits, an exponential is good to 2^-20; the second piece of an fp16
    # value below 2^-14 is off by 2^-25 of what the row's largest probability (at least 1 / 256) is taken as
    es = (2 * D * F32 * scale * (qd.abs() @ kd.abs().transpose(-1, -2)) * see).amax() + 2.0 ** -20
    sub = 2.0 ** -25 if q.dtype == FP else 2.0 ** -126
    tiny = torch.finfo(q.dtype).tiny * u
    rough = (u * u + es) * (p @ vd.abs()) + sub * (see.double() @ vd.abs())
    rows = lambda t: t.reshape(B, H, Tq, D).transpose(1, 2).reshape(B * Tq, H * D)  # noqa: E731
    tols = [rows(u * o.abs() + rough) + tiny]
    if do is not None:
        # (as in the oracle: the log-sum's rounding, added to a score 16 products at a time)
        es = es + (D / 16 + 2) * F32 * (1.4427 * ((s * see).abs().amax() + math.log(Tk)) + 1)
        dod = do.double().view(B, Tq, H, D).transpose(1, 2).reshape(B, KV, H // KV, Tq, D)
        dp, delta = dod @ vd.transpose(-1, -2), (dod * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        low = sub * (2.0 ** -12 if q.dtype == FP else 1)
        dv = (u * u + es) * (p.transpose(-1, -2) @ dod.abs()) + low * (see.double().transpose(-1, -2) @ dod.abs())
        # D: from o and what its rounding left off, itself rounded
        e_ds = p * (2 * D * F32 * (dod.abs() @ vd.abs().transpose(-1, -2))
                    + (dod.abs() * (rough + u * u * o.abs() + sub)).sum(-1, keepdim=True))
        e_ds = e_ds + (u * u + es) * ds.abs() + see * (2.0 ** -32 * ds.abs().amax() + 2.0 ** -126)
        tols += [u * want[1].abs() + (e_ds @ kd.abs() * scale).reshape(B, H, Tq, D) + tiny,
                 u * want[2].abs() + (e_ds.transpose(-1, -2) @ qd.abs()).sum(2) * scale + tiny,
                 u * want[3].abs() + dv.sum(2) + tiny]
    return list(zip(want, tols))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,H,KV,T,D,window,sinks", [
    (2, 3, 3, 1, 64, 4, 1), (2, 3, 3, 33, 64, 16, 40), (2, 4, 2, 300, 64, 100, 4), (1, 4, 1, 257, 128, None, 0),
    (1, 4, 2, 1100, 64, 100, 4), (1, 2, 1, 1300, 128, 200, 70)])
def test_window_attention_rounds_once(B, H, KV, T, D, window, sinks, dtype):
    q, k, v, do = _attention_case(B, H, KV, T, T, D, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = heads.window_attention(*leaves, window, sinks)
    got = (o,) + torch.autograd.grad(o, leaves, do)
    for g, (w, tol), name in zip(got, _once_rounded(q, k, v, do, window, sinks), ("o", "dq", "dk", "dv")):
        _within(g, w, tol, name)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,H,KV,Tq,Tk,D,window,sinks", [
    (3, 4, 4, 1, 500, 64, None, 0), (2, 8, 2, 1, 3000, 128, None, 0), (3, 6, 3, 2, 900, 64, 128, 4),
    (1, 16, 1, 1, 5000, 128, 2000, 33), (2, 2, 2, 40, 700, 64, 300, 2)])
def test_window_attention_over_a_cache_rounds_once(B, H, KV, Tq, Tk, D, window, sinks, dtype):
    q, k, v, _ = _attention_case(B, H, KV, Tq, Tk, D, dtype)
    with torch.no_grad():
        got = heads.window_attention(q, k, v, window, sinks)
    (want, tol), = _once_rounded(q, k, v, None, window, sinks)
    _within(got, want, tol, "o")
