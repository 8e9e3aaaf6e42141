"""ops.heads and ops.distill on the CPU: the references against loops over their definitions, their
gradients against differences, and what the entry points refuse."""
import ctypes
import math

import pytest
import torch

from metaopt_amd.ops import _lib, distill, heads, lm


def _rand(*shape, dtype=torch.float64):
    return torch.randn(*shape, dtype=dtype)


# ------------------------------------------------------------------------------- definitions
@pytest.mark.parametrize("il", [False, True])
def test_qk_norm_rope_is_the_formula(il):
    torch.manual_seed(0)
    P, n, T, H, KV, D = 2, 4, 3, 4, 2, 8
    qkv, wq, wk = _rand(n * T, (H + 2 * KV) * D), _rand(P, D), _rand(P, D)
    cos, sin = heads.rope_tables(8, D)
    q, k, v = heads.qk_norm_rope(qkv, wq, wk, cos, sin, T, H, KV, eps=1e-3, il=il)
    for b in range(n):
        for t in range(T):
            for h in range(H + 2 * KV):
                x = qkv[b * T + t, h * D:(h + 1) * D]
                if h >= H + KV:
                    assert torch.equal(v[b, h - H - KV, t], x)
                    continue
                w = (wq if h < H else wk)[b // (n // P)]
                y = x / math.sqrt(float((x * x).mean()) + 1e-3) * w
                z = torch.empty(D, dtype=torch.float64)
                for j in range(D // 2):
                    i0, i1 = (2 * j, 2 * j + 1) if il else (j, j + D // 2)
                    c, s = float(cos[t, j]), float(sin[t, j])
                    z[i0], z[i1] = y[i0] * c - y[i1] * s, y[i1] * c + y[i0] * s
                got = q[b, h, t] if h < H else k[b, h - H, t]
                torch.testing.assert_close(got, z, rtol=1e-12, atol=1e-12)


def test_qk_norm_rope_gradients_match_differences():
    torch.manual_seed(1)
    P, n, T, H, KV, D = 2, 2, 3, 2, 1, 4
    cos, sin = heads.rope_tables(T, D)
    args = [t.requires_grad_(True) for t in (_rand(n * T, (H + 2 * KV) * D), _rand(P, D), _rand(P, D))]
    for il in (False, True):
        assert torch.autograd.gradcheck(
            lambda x, a, b: heads.qk_norm_rope(x, a, b, cos, sin, T, H, KV, il=il), args)


@pytest.mark.parametrize("T", [1, 2])
def test_cached_heads_are_the_whole_sequence_s(T):
    """Tokens added T at a time leave in the cache what one call over the sequence gives."""
    torch.manual_seed(2)
    P, n, L, H, KV, D = 2, 4, 6, 4, 2, 8
    qkv, wq, wk = _rand(n * L, (H + 2 * KV) * D), _rand(P, D), _rand(P, D)
    cos, sin = heads.rope_tables(L, D)
    want = heads.qk_norm_rope(qkv, wq, wk, cos, sin, L, H, KV)
    kc, vc = torch.full((n, KV, L + 2, D), 9.0, dtype=torch.float64), \
        torch.full((n, KV, L + 2, D), 9.0, dtype=torch.float64)
    for t in range(0, L, T):
        rows = qkv.view(n, L, -1)[:, t:t + T].reshape(n * T, -1)
        start = torch.full((n,), t, dtype=torch.int32)
        q = heads.qk_norm_rope_cached(rows, wq, wk, cos, sin, T, H, kc, vc, start)
        torch.testing.assert_close(q, want[0][:, :, t:t + T])
    torch.testing.assert_close(kc[:, :, :L], want[1])
    torch.testing.assert_close(vc[:, :, :L], want[2])
    assert (kc[:, :, L:] == 9).all() and (vc[:, :, L:] == 9).all()


def test_cached_heads_leave_out_positions_that_are_not_there():
    torch.manual_seed(3)
    n, T, H, D, cap = 4, 2, 2, 8, 5
    rows, w = _rand(n * T, 3 * H * D), _rand(1, D)
    cos, sin = heads.rope_tables(4, D)
    kc, vc = torch.zeros(n, H, cap, D, dtype=torch.float64), torch.zeros(n, H, cap, D, dtype=torch.float64)
    start = torch.tensor([-1, 3, 4, 0], dtype=torch.int32)
    q = heads.qk_norm_rope_cached(rows, w, w, cos, sin, T, H, kc, vc, start)
    there = {(0, 1): 0, (1, 0): 3, (3, 0): 0, (3, 1): 1}      # (sequence, token): position
    for b in range(n):
        for t in range(T):
            assert (q[b, :, t].abs().sum() > 0) == ((b, t) in there)
    written = [(b, p) for b in range(n) for p in range(cap) if kc[b, :, p].abs().sum() > 0]
    assert written == sorted((b, p) for (b, _), p in there.items())


def _naive_attention(q, k, v, window, sinks, scale, start, lengths):
    B, H, Tq, D = q.shape
    KV, Tk = k.shape[1:3]
    o = torch.zeros(B, Tq, H, D, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            for t in range(Tq):
                i = start[b] + t
                js = [j for j in range(min(Tk, lengths[b])) if 0 <= i < min(Tk, lengths[b]) and j <= i
                      and (window is None or i - j < window or j < sinks)]
                if js:
                    kk, vv = k[b, h // (H // KV), js], v[b, h // (H // KV), js]
                    p = (kk @ q[b, h, t] * scale).softmax(0)
                    o[b, t, h] = p @ vv
    return o.view(B * Tq, H * D)


@pytest.mark.parametrize("Tq,Tk,window,sinks,start,lengths", [
    (5, 5, None, 0, None, None), (6, 6, 2, 0, None, None), (7, 7, 2, 1, None, [0, 1, 7]),
    (7, 7, 1, 3, None, [4, 9, 2]), (2, 9, 3, 2, None, None), (1, 9, 4, 1, [0, 5, 8], None),
    (3, 6, 2, 2, [-1, 5, 9], None), (3, 6, 2, 2, -2, None), (4, 6, 3, 1, [0, 1, 2], [2, 3, 6])])
def test_window_attention_is_the_formula(Tq, Tk, window, sinks, start, lengths):
    torch.manual_seed(4)
    B, H, KV, D = 3, 4, 2, 8
    q, k, v = _rand(B, H, Tq, D), _rand(B, KV, Tk, D), _rand(B, KV, Tk, D)
    first = [Tk - Tq] * B if start is None else start if isinstance(start, list) else [start] * B
    last = [f + Tq for f in first] if lengths is None else lengths
    tensor = lambda x: torch.tensor(x, dtype=torch.int32) if isinstance(x, list) else x  # noqa: E731
    o = heads.window_attention(q, k, v, window, sinks, start=tensor(start), lengths=tensor(lengths))
    want = _naive_attention(q, k, v, window, sinks, 1 / math.sqrt(D), first, last)
    torch.testing.assert_close(o, want, rtol=1e-12, atol=1e-12)


def test_window_attention_ignores_what_padding_holds():
    torch.manual_seed(5)
    B, H, T, D = 2, 2, 6, 8
    q, k, v = (_rand(B, H, T, D) for _ in range(3))
    lengths = torch.tensor([3, 0], dtype=torch.int32)
    want = heads.window_attention(q, k, v, 2, 1, lengths=lengths)
    leaves = []
    for t in (q, k, v):
        t = t.clone()
        t[0, :, 3:], t[1] = float("nan"), float("inf")
        leaves.append(t.requires_grad_(True))
    got = heads.window_attention(*leaves, 2, 1, lengths=lengths)
    assert torch.equal(got, want) and (got.view(B, T, -1)[0, 3:] == 0).all()
    for g in torch.autograd.grad(got[:3].sum(), leaves):
        assert torch.isfinite(g).all() and (g[0, :, 3:] == 0).all() and (g[1] == 0).all()


def test_window_attention_gradients_match_differences():
    torch.manual_seed(6)
    q, k, v = _rand(2, 4, 5, 3), _rand(2, 2, 5, 3), _rand(2, 2, 5, 3)
    lengths = torch.tensor([5, 3], dtype=torch.int32)
    assert torch.autograd.gradcheck(
        lambda a, b, c: heads.window_attention(a, b, c, 2, 1, lengths=lengths),
        [t.requires_grad_(True) for t in (q, k, v)])


def test_plain_causal_window_is_lm_attention():
    torch.manual_seed(7)
    q, k, v = (_rand(2, 3, 64, 64, dtype=torch.float32) for _ in range(3))
    torch.testing.assert_close(heads.window_attention(q, k, v), lm.attention(q, k, v))


def _naive_distill(x, y, t, index, tau, a):
    V = len(x)
    lp1, lpt = x.log_softmax(0), (x / tau).log_softmax(0)
    loss = 0.0
    if 0 <= y < V:
        loss += (1 - a) * -float(lp1[y])
    there = [k for k, i in enumerate(index) if 0 <= i < V]
    if there:
        lq = (t[there] / tau).log_softmax(0)
        loss += a * tau * tau * sum(float(l.exp() * (l - lpt[index[k]])) for l, k in zip(lq, there))
    return loss


def test_distill_loss_is_the_formula():
    torch.manual_seed(8)
    P, rows, V, K = 2, 4, 11, 3
    x, t = _rand(P * rows, V), _rand(P * rows, K)
    index = torch.randint(0, V, (P * rows, K), dtype=torch.int32)
    index[1] = -1
    index[2, 1] = V
    index[3] = index[3, 0]                                   # one place three times
    y = torch.randint(0, V, (P * rows,), dtype=torch.int32)
    y[1], y[5] = -100, V
    tau, a = torch.tensor([1.0, 2.5]), torch.tensor([0.25, 1.0])
    got = distill.distill_loss(x, y, t, index, rows, tau, a)
    for p in range(P):
        want = sum(_naive_distill(x[r], int(y[r]), t[r], index[r].tolist(), float(tau[p]), float(a[p]))
                   for r in range(p * rows, (p + 1) * rows))
        assert abs(float(got[p]) - want) < 1e-10


def test_distill_loss_gradients_match_differences():
    torch.manual_seed(9)
    x, t = _rand(4, 7).requires_grad_(True), _rand(4, 3)
    index = torch.tensor([[0, 1, 1], [-1, 2, 6], [-1, -1, -1], [5, 5, 5]], dtype=torch.int32)
    y = torch.tensor([0, -1, 3, 6], dtype=torch.int32)
    assert torch.autograd.gradcheck(
        lambda z: distill.distill_loss(z, y, t, index, 2, 1.7, 0.4), [x])
    grad, = torch.autograd.grad(distill.distill_loss(x, y, t, index, 2, 1.7, 0.4).sum(), x)
    scaled, = torch.autograd.grad(
        distill.distill_loss(x, y, t, index, 2, 1.7, 0.4, grad_scale=0.5).sum(), x)
    torch.testing.assert_close(scaled, 0.5 * grad)


def test_distill_without_teacher_is_cross_entropy():
    torch.manual_seed(10)
    x = _rand(6, 9, dtype=torch.float32)
    y = torch.randint(0, 9, (6,), dtype=torch.int32)
    none = torch.empty(6, 0), torch.empty(6, 0, dtype=torch.int32)
    got = distill.distill_loss(x, y, *none, 3, alpha=0.0)
    torch.testing.assert_close(got, lm.cross_entropy(x, y, 3))


# ------------------------------------------------------------------------------- refusals
def _qk_args(**kw):
    d = dict(qkv=torch.zeros(4, 32), wq=torch.ones(1, 8), wk=torch.ones(1, 8),
             cos=torch.zeros(2, 4), sin=torch.zeros(2, 4), T=2, H=2)
    return dict(d, **kw)


@pytest.mark.parametrize("bad,match", [
    (dict(qkv=torch.zeros(4, 33)), "columns"), (dict(qkv=torch.zeros(5, 48)), "whole sequences"),
    (dict(qkv=torch.zeros(4, 48), T=0), "positive"), (dict(qkv=torch.zeros(4, 48), T=4), "tables"),
    (dict(qkv=torch.zeros(4, 56), H=3, kv_heads=2), "multiple"),
    (dict(qkv=torch.zeros(4, 48), cos=torch.zeros(2, 3)), "table"),
    (dict(qkv=torch.zeros(4, 48), sin=torch.zeros(2, 4).double()), "table"),
    (dict(qkv=torch.zeros(4, 48), wk=torch.ones(2, 8)), "trials"),
    (dict(qkv=torch.zeros(4, 48).half()), "one type"), (dict(qkv=torch.zeros(2, 2, 48)), "rows")])
def test_qk_norm_rope_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        heads.qk_norm_rope(**_qk_args(**bad))


@pytest.mark.parametrize("bad,match", [
    (dict(start=torch.zeros(2)), "int32"), (dict(start=torch.zeros(3, dtype=torch.int32)), "int32"),
    (dict(kcache=torch.zeros(2, 2, 4, 8), vcache=torch.zeros(2, 2, 5, 8)), "alike"),
    (dict(kcache=torch.zeros(3, 2, 4, 8), vcache=torch.zeros(3, 2, 4, 8)), "sequences"),
    (dict(kcache=torch.zeros(2, 2, 4, 8).half(), vcache=torch.zeros(2, 2, 4, 8).half()), "type"),
    (dict(kcache=torch.zeros(1, 2, 4, 8).expand(2, 2, 4, 8)), "written"),
    (dict(zip(("kcache", "vcache"), [torch.zeros(2, 2, 4, 8)] * 2)), "written")])
def test_qk_norm_rope_cached_refuses(bad, match):
    d = _qk_args(qkv=torch.zeros(4, 48), kcache=torch.zeros(2, 2, 4, 8), vcache=torch.zeros(2, 2, 4, 8),
                 start=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match=match):
        heads.qk_norm_rope_cached(**dict(d, **bad))


@pytest.mark.parametrize("bad,match", [
    (dict(q=torch.zeros(1, 3, 4, 8)), "multiple"), (dict(q=torch.zeros(2, 2, 4, 8)), "fit"),
    (dict(q=torch.zeros(2, 4, 8)), "B, H"), (dict(q=torch.zeros(1, 2, 4, 8).half()), "one type"),
    (dict(window=0), "window"), (dict(sinks=-1), "sinks"), (dict(scale=0.0), "positive"),
    (dict(scale=float("inf")), "positive"), (dict(scale=1e-38), "positive"), (dict(start=torch.zeros(1)), "int32"),
    (dict(start=1 << 40), "position"), (dict(lengths=torch.zeros(2, dtype=torch.int32)), "int32"),
    (dict(lengths=torch.zeros(1, dtype=torch.int64)), "int32")])
def test_window_attention_refuses(bad, match):
    d = dict(q=torch.zeros(1, 2, 4, 8), k=torch.zeros(1, 2, 4, 8), v=torch.zeros(1, 2, 4, 8))
    with pytest.raises(ValueError, match=match):
        heads.window_attention(**dict(d, **bad))


@pytest.mark.parametrize("bad,match", [
    (dict(labels=torch.zeros(4)), "int32"), (dict(labels=torch.zeros(3, dtype=torch.int32)), "int32"),
    (dict(top_index=torch.zeros(4, 2, dtype=torch.int64)), "int32"),
    (dict(top_values=torch.zeros(4, 3)), "one shape"),
    (dict(top_values=torch.zeros(4, 2, requires_grad=True)), "detach"),
    (dict(top_values=torch.zeros(4, 1025), top_index=torch.zeros(4, 1025, dtype=torch.int32)), "1024"),
    (dict(rows_per_trial=3), "whole trials"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(alpha=1.5), "alpha"),
    (dict(alpha=torch.zeros(3)), "alpha"), (dict(alpha=torch.zeros(2).double()), "alpha"),
    (dict(temperature=torch.ones(2, requires_grad=True)), "detach"), (dict(inplace=True), "unit_weights"),
    (dict(logits=torch.zeros(4)), "vocabulary")])
def test_distill_loss_refuses(bad, match):
    d = dict(logits=torch.zeros(4, 5), labels=torch.zeros(4, dtype=torch.int32),
             top_values=torch.zeros(4, 2), top_index=torch.zeros(4, 2, dtype=torch.int32),
             rows_per_trial=2)
    with pytest.raises(ValueError, match=match):
        distill.distill_loss(**dict(d, **bad))


def test_cached_heads_with_tables_of_no_position():
    """No position is inside tables that hold none: nothing is written, every query is 0."""
    kc, vc = torch.full((2, 2, 4, 8), 9.0), torch.full((2, 2, 4, 8), 9.0)
    cos, sin = heads.rope_tables(0, 8)
    q = heads.qk_norm_rope_cached(torch.ones(4, 48), torch.ones(1, 8), torch.ones(1, 8), cos, sin, 2, 2, kc, vc,
                                  torch.zeros(2, dtype=torch.int32))
    assert tuple(q.shape) == (2, 2, 2, 8) and not q.any()
    assert (kc == 9).all() and (vc == 9).all()


def test_cached_heads_do_not_launch_with_tables_of_no_position(monkeypatch):
    """The kernel reads row 0 of the tables for a token that has no position."""
    monkeypatch.setattr(heads, "_hip", lambda t, op="": True)
    monkeypatch.setattr(heads, "_call", lambda *args: pytest.fail("launched"))
    rows, w = torch.ones(4, 384, dtype=torch.bfloat16), torch.ones(1, 64, dtype=torch.bfloat16)
    caches = [torch.full((2, 2, 4, 64), 9.0, dtype=torch.bfloat16) for _ in "kv"]
    cos, sin = heads.rope_tables(0, 64)
    q = heads.qk_norm_rope_cached(rows, w, w, cos, sin, 2, 2, *caches, torch.zeros(2, dtype=torch.int32))
    assert tuple(q.shape) == (2, 2, 2, 64) and not q.any() and all((c == 9).all() for c in caches)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of nothing: only where nothing can be launched")
def test_the_kernel_s_entry_refuses_tables_of_no_position():
    one = ctypes.c_int32(0)
    args = [None, 384, None, None, None, None, ctypes.addressof(one), None, None, None, heads._Strides6(), 4, 2, 2, 2,
            4, 64, 0, 4, 1e-5, 0, 0, None]
    assert _lib.get_lib().mopt_qk_norm_rope_fwd(*args) == 1      # (1: refused on the host, in front of the launch)


def test_cached_heads_of_tokens_without_a_position_are_zero_whatever_the_row_holds():
    rows = torch.full((2, 48), float("nan"))
    cos, sin = heads.rope_tables(4, 8)
    kc, vc = torch.zeros(2, 2, 4, 8), torch.zeros(2, 2, 4, 8)
    q = heads.qk_norm_rope_cached(rows, torch.ones(1, 8), torch.ones(1, 8), cos, sin, 1, 2, kc, vc,
                                  torch.tensor([4, -1], dtype=torch.int32))
    assert (q == 0).all() and not kc.any() and not vc.any()


# ------------------------------------------------------------------------------- forward mode
def _forward_mode_calls():
    """(name, call of one tensor, the tensor): each differentiable argument of the operators."""
    torch.manual_seed(12)
    bf = torch.bfloat16
    cos, sin = heads.rope_tables(2, 64)
    qkv, w = _rand(4, 384, dtype=bf), _rand(1, 64, dtype=bf)
    start = torch.zeros(2, dtype=torch.int32)
    caches = [_rand(2, 2, 4, 64, dtype=bf) for _ in "kv"]
    q, k = _rand(1, 2, 4, 64, dtype=bf), _rand(1, 1, 4, 64, dtype=bf)
    x, top = _rand(4, 9, dtype=torch.float32), _rand(4, 3, dtype=torch.float32)
    y, index = torch.zeros(4, dtype=torch.int32), torch.arange(12, dtype=torch.int32).view(4, 3) % 9
    tau, alpha = torch.ones(2), torch.full((2,), 0.5)

    def rope(qkv=qkv, wq=w, wk=w, cos=cos, sin=sin):
        return heads.qk_norm_rope(qkv, wq, wk, cos, sin, 2, 2)

    def cached(qkv=qkv, wq=w, wk=w, cos=cos, sin=sin, kc=caches[0], vc=caches[1]):
        return heads.qk_norm_rope_cached(qkv, wq, wk, cos, sin, 2, 2, kc, vc, start)

    def attention(q=q, k=k, v=k):
        return heads.window_attention(q, k, v, 2, 1)

    def loss(x=x, top=top, tau=tau, alpha=alpha):
        return distill.distill_loss(x, y, top, index, 2, tau, alpha)
    for f, args in ((rope, dict(qkv=qkv, wq=w, wk=w, cos=cos, sin=sin)),
                    (cached, dict(qkv=qkv, wq=w, wk=w, cos=cos, sin=sin, kc=caches[0], vc=caches[1])),
                    (attention, dict(q=q, k=k, v=k)), (loss, dict(x=x, top=top, tau=tau, alpha=alpha))):
        for name, t in args.items():
            yield f"{f.__name__}-{name}", (lambda t, f=f, name=name: f(**{name: t})), t


CALLS = {name: (call, t) for name, call, t in _forward_mode_calls()}


@pytest.mark.parametrize("name", CALLS)
def test_kernels_refuse_forward_mode_derivatives(name, monkeypatch):
    """A dual tensor does not require a gradient: a call that looks at that alone would drop its
    tangent, which counts as a derivative of 0."""
    call, t = CALLS[name]
    for module in (heads, distill):
        monkeypatch.setattr(module, "_hip", lambda t, op="": True)
        monkeypatch.setattr(module, "_call", lambda *args: pytest.fail("launched"))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)


def test_references_have_forward_mode_derivatives():
    torch.manual_seed(13)
    q, d = _rand(1, 2, 4, 8), _rand(1, 2, 4, 8)
    with torch.autograd.forward_ad.dual_level():
        o = heads.window_attention(torch.autograd.forward_ad.make_dual(q, d), q, q, 2, 1)
        got = torch.autograd.forward_ad.unpack_dual(o).tangent
    h = 1e-6
    ends = [heads.window_attention(q + s * d, q, q, 2, 1) for s in (h, -h)]
    torch.testing.assert_close(got, (ends[0] - ends[1]) / (2 * h), rtol=1e-6, atol=1e-8)


# ------------------------------------------------------------------------------- memory of the caches
def _cached_call(kc, vc, qkv=None):
    n, KV, _, D = kc.shape
    rows = torch.ones(n, 3 * KV * D) if qkv is None else qkv
    return heads.qk_norm_rope_cached(rows, torch.ones(1, D), torch.ones(1, D), *heads.rope_tables(4, D), 1, KV, kc, vc,
                                     torch.zeros(n, dtype=torch.int32))


def _overlapping():
    flat = torch.zeros(4096)
    yield "shifted", flat[:128].view(2, 2, 4, 8), flat[8:136].view(2, 2, 4, 8)
    yield "one element", flat[:128].view(2, 2, 4, 8), flat[127:255].view(2, 2, 4, 8)
    wide = torch.zeros(2, 2, 4, 16)
    yield "columns", wide[..., :8], wide[..., 7:15]
    yield "another order", flat[:128].view(2, 2, 4, 8), flat[64:192].view(2, 4, 2, 8).transpose(1, 2)
    yield "heads of one cache", flat.as_strided((2, 2, 4, 8), (64, 16, 8, 1)), flat[2048:2176].view(2, 2, 4, 8)
    yield "sequences of the other", flat[2048:2176].view(2, 2, 4, 8), flat.as_strided((2, 2, 4, 8), (24, 32, 8, 1))


@pytest.mark.parametrize("name,kc,vc", list(_overlapping()))
def test_overlapping_caches_are_refused(name, kc, vc):
    """Both are written at once: where they share memory the last write wins."""
    with pytest.raises(ValueError, match="written"):
        _cached_call(kc, vc)


def test_caches_over_the_activation_are_refused():
    flat = torch.ones(512)
    for at in (0, 95):
        with pytest.raises(ValueError, match="written"):
            _cached_call(flat[at:at + 128].view(2, 2, 4, 8), torch.zeros(2, 2, 4, 8), flat[:96].view(2, 48))
        with pytest.raises(ValueError, match="written"):
            _cached_call(torch.zeros(2, 2, 4, 8), flat[at:at + 128].view(2, 2, 4, 8), flat[:96].view(2, 48))
    _cached_call(flat[96:224].view(2, 2, 4, 8), flat[224:352].view(2, 2, 4, 8), flat[:96].view(2, 48))


@pytest.mark.parametrize("layout", ["halves", "columns", "by sequence", "by head", "by position", "transposed"])
def test_caches_side_by_side_in_one_tensor_are_taken(layout):
    shape, pick = {
        "halves": ((2, 2, 2, 4, 8), lambda t: (t[0], t[1])), "columns": ((2, 2, 4, 16), lambda t: (t[..., :8], t[..., 8:])),
        "by sequence": ((2, 2, 2, 4, 8), lambda t: (t[:, 0], t[:, 1])),
        "by head": ((2, 4, 4, 8), lambda t: (t[:, ::2], t[:, 1::2])),
        "by position": ((2, 2, 8, 8), lambda t: (t[:, :, :4], t[:, :, 4:])),
        "transposed": ((2, 4, 4, 8), lambda t: (t[:, :, :2].transpose(1, 2), t[:, :, 2:].transpose(1, 2)))}[layout]
    kc, vc = pick(torch.zeros(shape))
    apart = [torch.zeros(2, 2, 4, 8) for _ in "kv"]
    assert torch.equal(_cached_call(kc, vc), _cached_call(*apart))
    assert torch.equal(kc, apart[0]) and torch.equal(vc, apart[1]) and kc.any() and vc.any()


# ------------------------------------------------------------------------------- writes that autograd has to see
def test_distill_in_place_marks_the_logits_as_written(monkeypatch):
    """Another operation that kept the logits for its backward says so, as after any write in place."""
    monkeypatch.setattr(distill, "_hip", lambda t, op="": True)
    monkeypatch.setattr(distill, "_call", lambda x, name, *args: None)
    leaf = torch.randn(4, 5, requires_grad=True)
    y, top, index = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    for inplace in (False, True):
        h = leaf * 2
        other = (h * h).sum()
        loss = distill.distill_loss(h.view(4, 5), y, top, index, 2, unit_weights=True, inplace=inplace)
        g, = torch.autograd.grad(loss.sum(), h, retain_graph=True)        # (its own backward runs)
        assert (g.data_ptr() == h.data_ptr()) == inplace
        if not inplace:
            torch.autograd.grad(other, leaf)
            continue
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(other, leaf)
    with torch.no_grad():                              # without a gradient nothing is written
        before = h._version
        distill.distill_loss(h, y, top, index, 2, unit_weights=True, inplace=True)
        assert h._version == before


@pytest.mark.parametrize("kernel", [False, True])
def test_cached_heads_mark_the_caches_as_written(kernel, monkeypatch):
    """Attention over the caches keeps them for its backward, which a later write into them would falsify."""
    if kernel:
        monkeypatch.setattr(heads, "_hip", lambda t, op="": True)
        monkeypatch.setattr(heads, "_call", lambda *args: None)
    bf, w = torch.bfloat16, torch.ones(1, 64, dtype=torch.bfloat16)
    kc, vc = (torch.randn(2, 1, 4, 64).to(bf) for _ in "kv")
    q = torch.randn(2, 1, 1, 64).to(bf).requires_grad_(True)
    start = torch.full((2,), 2, dtype=torch.int32)
    if kernel:
        o = heads._WindowAttention.apply(q, kc, vc, 9, 0, 0.125, start, 3, None)
    else:
        o = (q * kc).sum() + (q * vc).sum()
    before = kc._version, vc._version
    heads.qk_norm_rope_cached(torch.ones(2, 192, dtype=bf), w, w, *heads.rope_tables(4, 64), 1, 1, kc, vc, start)
    assert kc._version > before[0] and vc._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.float().sum(), q)
