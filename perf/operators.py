"""The LM operators' cases, plain forms and exact forms: query / key head norms with the position
rotation (``qk_norm_rope``), sliding-window attention with sink tokens (``window_attention``) and
distillation from a teacher's top logits (``distill_loss``).

``own`` selects the framework's kernels; otherwise the same values come from elementary torch
operations in 32 bits, rounded once at the end.  A step that trains returns its gradients, a step
that extends a cache returns the cache.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    """Cases; sizes are those of the LM presets (12 heads of 64, 512 positions, 64 sequences of a
    population of 8, vocabulary 32000; the tiny preset's 4096) and generic ones around them."""
    return [
        # one layer's heads of the 125M population: 8 trials x 8 sequences x 512 tokens
        rope("rope-train-lm", trials=8, seqs=64, tokens=512, heads=12, kv_heads=12, dim=64),
        # grouped heads of 128, rotate-half pairs, an odd length
        rope("rope-train-grouped", trials=1, seqs=3, tokens=4001, heads=20, kv_heads=4, dim=128,
             dtype="fp16", interleaved=False),
        # one new token of 64 sequences, written into their caches
        rope("rope-step", trials=8, seqs=64, tokens=1, heads=12, kv_heads=12, dim=64, cache=1024,
             grad=False),
        # the 125M population's attention with a window
        window("window-train-lm", seqs=64, heads=12, kv_heads=12, dim=64, queries=512, keys=512,
               window=128, sinks=4),
        # one long sequence, grouped heads of 128
        window("window-train-long", seqs=1, heads=16, kv_heads=4, dim=128, queries=8192,
               keys=8192, window=1024, sinks=4),
        # a padded batch of odd lengths (0 and 1 among them)
        window("window-train-ragged", seqs=7, heads=6, kv_heads=2, dim=64, queries=777, keys=777,
               window=100, sinks=3, dtype="fp16", ragged=True),
        # a prompt read without gradients
        window("window-prompt", seqs=4, heads=12, kv_heads=12, dim=64, queries=4096, keys=4096,
               window=512, sinks=16, grad=False),
        # one token of 64 sequences over their caches
        window("window-step", seqs=64, heads=12, kv_heads=4, dim=64, queries=1, keys=4096,
               window=1024, sinks=4, grad=False, ragged=True),
        # one token of one sequence over all of a long cache: no window
        window("window-step-long", seqs=1, heads=32, kv_heads=8, dim=128, queries=1, keys=32768,
               window=0, sinks=0, grad=False),
        # the 125M population's step: 32768 rows of 32000 logits
        distill("distill-train-lm", trials=8, rows=4096, vocab=32000, top=64),
        # a micro step: latency
        distill("distill-small", trials=4, rows=64, vocab=4096, top=8),
        # rows of odd length in 32 bits, with rows without labels or teacher
        distill("distill-odd", trials=1, rows=1023, vocab=49999, top=37, dtype="fp32",
                missing=True),
    ]


def rope(name, trials, seqs, tokens, heads, kv_heads, dim, dtype="bf16", interleaved=True,
         cache=0, grad=True):
    return _named(name, op="rope", trials=trials, seqs=seqs, tokens=tokens, heads=heads,
                  kv_heads=kv_heads, dim=dim, dtype=dtype, interleaved=interleaved, cache=cache,
                  grad=grad)


def window(name, seqs, heads, kv_heads, dim, queries, keys, window, sinks, dtype="bf16",
           grad=True, ragged=False):
    return _named(name, op="window", seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim,
                  queries=queries, keys=keys, window=window, sinks=sinks, dtype=dtype, grad=grad,
                  ragged=ragged)


def distill(name, trials, rows, vocab, top, dtype="bf16", missing=False, grad=True):
    return _named(name, op="distill", trials=trials, rows=rows, vocab=vocab, top=top, dtype=dtype,
                  missing=missing, grad=grad)


def _named(name, **case):
    return dict(case, name=name) if name else case


def _spread(rng, lo, hi):
    """A size in [lo, hi], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope-step", "window", "window-forward", "window-step", "distill"])
    dim, dtype = rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    kv = rng.randint(1, 12 if dim == 64 else 8)
    heads = kv * rng.randint(1, min(8, 24 // kv))
    if op == "rope":
        trials, tokens = rng.randint(1, 8), _spread(rng, 1, 2048)
        room = 32768 * 36 * 64 // (tokens * (heads + 2 * kv) * dim)
        seqs = trials * _spread(rng, 1, max(1, min(64, room) // trials))
        return rope(None, trials, seqs, tokens, heads, kv, dim, dtype, rng.random() < 0.5)
    if op == "rope-step":
        trials = rng.randint(1, 8)
        return rope(None, trials, trials * _spread(rng, 1, 16), rng.randint(1, 4), heads, kv, dim,
                    dtype, rng.random() < 0.5, cache=rng.randint(8, 1024), grad=False)
    sinks = rng.choice([0, 1, 4, rng.randint(1, 80)])
    if op in ("window", "window-forward"):
        tokens = _spread(rng, 1, 4096)
        seqs = _spread(rng, 1, max(1, min(64, (1 << 28) // (heads * tokens * tokens))))
        return window(None, seqs, heads, kv, dim, tokens, tokens, _spread(rng, 1, 2048), sinks,
                      dtype, op == "window", rng.random() < 0.5)
    if op == "window-step":
        keys = _spread(rng, 1, 16384)
        seqs = _spread(rng, 1, max(1, min(128, (1 << 28) // (keys * kv * dim))))
        return window(None, seqs, heads, kv, dim, min(keys, rng.choice([1, 1, 2, 3])), keys,
                      rng.choice([0, _spread(rng, 16, 4096)]), sinks, dtype, False, True)
    vocab = _spread(rng, 1000, 130000)
    trials = rng.randint(1, 8)
    rows = _spread(rng, 1, max(1, (1 << 28) // (vocab * trials)))
    return distill(None, trials, min(rows, 4096), vocab, rng.randint(1, 128),
                   rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5, rng.random() < 0.7)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"rope": _prepare_rope, "window": _prepare_window,
            "distill": _prepare_distill}[case["op"]](case, g)


def _randn(g, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    return x.mul_(scale).add_(mean).to(dtype)


def _prepare_rope(c, g):
    dt, n, T, H, KV, D = DTYPES[c["dtype"]], c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    reach = c["cache"] or T
    angle = (torch.arange(reach, dtype=torch.float64)[:, None]
             * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)[None])
    s = dict(case=c, cos=angle.cos().float().cuda(), sin=angle.sin().float().cuda(),
             qkv=_randn(g, n * T, (H + 2 * KV) * D, dtype=dt),
             wq=_randn(g, c["trials"], D, dtype=dt, scale=0.2, mean=1.0),
             wk=_randn(g, c["trials"], D, dtype=dt, scale=0.2, mean=1.0))
    if c["cache"]:
        s["kcache"], s["vcache"] = (_randn(g, n, KV, reach, D, dtype=dt) for _ in range(2))
        s["start"] = torch.randint(0, reach - T + 1, (n,), generator=g, device="cuda",
                                   dtype=torch.int32)
    if c["grad"]:
        s["d"] = [_randn(g, n, h, T, D, dtype=dt) for h in (H, KV, KV)]
        for name in ("qkv", "wq", "wk"):
            s[name].requires_grad_(True)
    return s


def _lengths(c):
    """Lengths of a padded batch: spread over 0 ... keys, or over what a step has (its own tokens
    at least) ... keys."""
    n, lo = c["seqs"], 0 if c["queries"] == c["keys"] else c["queries"]
    if not c["ragged"]:
        return [c["keys"]] * n
    got = [lo + round((c["keys"] - lo) * i / max(1, n - 1)) for i in range(n)]
    if n > 2 and lo == 0:
        got[1] = 1
    return got


def _prepare_window(c, g):
    dt, n, H, KV, D = DTYPES[c["dtype"]], c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    q = _randn(g, n, H, c["queries"], D, dtype=dt)
    k, v = (_randn(g, n, KV, c["keys"], D, dtype=dt) for _ in range(2))
    lengths = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    lengths = lengths[torch.randperm(n, generator=g, device="cuda")]
    s = dict(case=c, q=q, k=k, v=v, lengths=lengths, start=None)
    if c["queries"] != c["keys"]:
        s["start"] = lengths - c["queries"]
    if c["grad"]:
        s["do"] = _randn(g, n * c["queries"], H * D, dtype=dt)
        for name in ("q", "k", "v"):
            s[name].requires_grad_(True)
    return s


def _prepare_distill(c, g):
    R, V, K = c["trials"] * c["rows"], c["vocab"], c["top"]
    logits = _randn(g, R, V, dtype=DTYPES[c["dtype"]], scale=2.0)
    index = torch.randint(0, V, (R, K), generator=g, device="cuda")
    top = _randn(g, R, K, scale=2.0, mean=6.0).sort(1, descending=True).values
    # the student half agrees with its teacher
    logits.scatter_(1, index, (0.5 * top + _randn(g, R, K)).to(logits.dtype))
    labels = index[:, 0].clone()
    if c["missing"]:
        cut = torch.rand(R, generator=g, device="cuda")
        labels[cut < 0.2] = -100
        keep = torch.randint(0, K + 1, (R, 1), generator=g, device="cuda")
        index[torch.arange(K, device="cuda")[None] >= keep] = -1
    return dict(case=c, logits=logits.requires_grad_(c["grad"]), labels=labels.int(),
                index=index.int(), top=top.to(torch.bfloat16 if c["dtype"] == "bf16" else
                                              torch.float32),
                temperature=2.0, alpha=0.7, weight=torch.ones(c["trials"], device="cuda"))


# ------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return {"rope": _own_rope, "window": _own_window,
                "distill": _own_distill}[state["case"]["op"]](state)
    with torch.no_grad():
        return {"rope": _plain_rope, "window": _plain_window,
                "distill": _plain_distill}[state["case"]["op"]](state)


def _own_rope(s):
    from metaopt_amd.ops import heads
    c = s["case"]
    if c["cache"]:
        q = heads.qk_norm_rope_cached(s["qkv"], s["wq"], s["wk"], s["cos"], s["sin"], c["tokens"],
                                      c["heads"], s["kcache"], s["vcache"], s["start"], eps=EPS,
                                      il=c["interleaved"])
        return q, s["kcache"], s["vcache"]
    out = heads.qk_norm_rope(s["qkv"], s["wq"], s["wk"], s["cos"], s["sin"], c["tokens"],
                             c["heads"], c["kv_heads"], eps=EPS, il=c["interleaved"])
    return list(out) + list(torch.autograd.grad(out, [s["qkv"], s["wq"], s["wk"]], s["d"]))


def _own_window(s):
    from metaopt_amd.ops import heads
    c = s["case"]
    o = heads.window_attention(s["q"], s["k"], s["v"], window=c["window"] or None,
                               sinks=c["sinks"], start=s["start"],
                               lengths=s["lengths"] if c["ragged"] else None)
    if not c["grad"]:
        return o
    return [o] + list(torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"]))


def _own_distill(s):
    from metaopt_amd.ops import distill
    c = s["case"]
    loss = distill.distill_loss(s["logits"], s["labels"], s["top"], s["index"], c["rows"],
                                temperature=s["temperature"], alpha=s["alpha"],
                                grad_scale=1.0 / c["rows"], unit_weights=True)
    if not c["grad"]:
        return loss
    return [loss] + list(torch.autograd.grad(loss, [s["logits"]], s["weight"]))


# ------------------------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, interleaved):
    """x [..., D] rotated by the angles of its pairs."""
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)


def _plain_norm_turn(x, w, cos, sin, interleaved):
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _turn(x * rstd * w, cos, sin, interleaved)


def _plain_norm_turn_back(x, w, cos, sin, interleaved, d):
    """(dx, terms of dw)"""
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    hat, dy = x * rstd, _turn(d, cos, -sin, interleaved)
    dhat = dy * w
    return rstd * (dhat - hat * (dhat * hat).mean(-1, keepdim=True)), dy * hat


def _plain_rope(s):
    c = s["case"]
    n, T, H, KV, D = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    dt, il = s["qkv"].dtype, c["interleaved"]
    x = s["qkv"].float().view(n, T, H + 2 * KV, D).transpose(1, 2)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    wq, wk = (w.float().repeat_interleave(n // c["trials"], 0)[:, None, None]
              for w in (s["wq"], s["wk"]))
    cos, sin = s["cos"][:T], s["sin"][:T]
    if c["cache"]:
        at = s["start"].long()[:, None] + torch.arange(T, device="cuda")
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    zq = _plain_norm_turn(q, wq, cos, sin, il).to(dt)
    zk = _plain_norm_turn(k, wk, cos, sin, il).to(dt)
    if c["cache"]:
        seq = torch.arange(n, device="cuda")[:, None]
        s["kcache"][seq, :, at] = zk.transpose(1, 2)
        s["vcache"][seq, :, at] = v.transpose(1, 2).to(dt)
        return zq, s["kcache"], s["vcache"]
    dq, tq = _plain_norm_turn_back(q, wq, cos, sin, il, s["d"][0].float())
    dk, tk = _plain_norm_turn_back(k, wk, cos, sin, il, s["d"][1].float())
    dx = torch.cat([dq, dk, s["d"][2].float()], 1).transpose(1, 2).reshape(n * T, -1)
    dw = [t.double().reshape(c["trials"], -1, D).sum(1).to(dt) for t in (tq, tk)]
    return [zq, zk, v.to(dt).contiguous(), dx.to(dt)] + dw


def _plain_window(s):
    c = s["case"]
    n, H, KV, D, Tq, Tk = (c[k] for k in ("seqs", "heads", "kv_heads", "dim", "queries", "keys"))
    dt, G, scale = s["q"].dtype, H // KV, 1.0 / math.sqrt(D)
    first = s["start"].long() if s["start"] is not None else torch.zeros(n, dtype=torch.long, device="cuda")
    i = (first[:, None] + torch.arange(Tq, device="cuda"))[:, None, None, :, None]
    j = torch.arange(Tk, device="cuda")
    near = i - j < c["window"] if c["window"] else j >= 0
    sees = (j <= i) & (i < s["lengths"].view(n, 1, 1, 1, 1)) & (near | (j < c["sinks"]))
    q = s["q"].float().reshape(n, KV, G * Tq, D)
    k, v = s["k"].float(), s["v"].float()
    x = (torch.matmul(q, k.transpose(2, 3)) * scale).view(n, KV, G, Tq, Tk)
    x = torch.where(sees, x, x.new_tensor(-math.inf))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = (e / torch.where(total == 0, torch.ones_like(total), total)).view(n, KV, G * Tq, Tk)
    o = torch.matmul(p, v)

    def rows(t):      # [n, KV, G Tq, D] -> [n Tq, H D]
        return t.view(n, H, Tq, D).transpose(1, 2).reshape(n * Tq, H * D).to(dt)
    if not c["grad"]:
        return rows(o)
    do = s["do"].float().view(n, Tq, H, D).transpose(1, 2).reshape(n, KV, G * Tq, D)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k).view(n, H, Tq, D)
    dk = torch.matmul(ds.transpose(2, 3), q)
    return [rows(o), dq.to(dt), dk.to(dt), dv.to(dt)]


def _plain_distill(s):
    c, x, tau, a = s["case"], s["logits"].float(), s["temperature"], s["alpha"]
    rows, gs = c["rows"], 1.0 / s["case"]["rows"]
    labels, index = s["labels"].long()[:, None], s["index"].long()
    has_label, has_top = labels >= 0, index >= 0
    y, at = labels.clamp(min=0), index.clamp(min=0)
    x = x - x.amax(1, keepdim=True)
    e1, et = torch.exp(x), torch.exp(x / tau)
    z1, zt = e1.sum(1, keepdim=True), et.sum(1, keepdim=True)
    ce = (torch.log(z1) - x.gather(1, y)) * has_label
    t = torch.where(has_top, s["top"].float() / tau, torch.full_like(index, -1e30, dtype=torch.float32))
    t = t - t.amax(1, keepdim=True)
    w = torch.exp(t) * has_top
    zw = w.sum(1, keepdim=True)
    has_row = zw > 0
    zw = torch.where(has_row, zw, torch.ones_like(zw))
    w = w / zw
    kl = (w * (t - torch.log(zw) - x.gather(1, at) / tau + torch.log(zt))).sum(1, keepdim=True)
    loss = (1 - a) * ce + a * tau * tau * kl
    loss = loss.double().view(-1, rows).sum(1).float()
    if not c["grad"]:
        return loss
    grad = (1 - a) * has_label * (e1 / z1) + a * tau * has_row * (et / zt)
    grad.scatter_add_(1, y, -(1 - a) * has_label.float())
    grad.scatter_add_(1, at, -a * tau * w)
    return [loss, (grad * gs).to(s["logits"].dtype)]


# ------------------------------------------------------------------------------------ work
def _pairs(c):
    """Visible (query, key) pairs of one head over the batch, and the keys that are read."""
    W, S = c["window"] or c["keys"], c["sinks"]

    def sum_to(m, most):         # min(1, most) + ... + min(m, most)
        return m * (m + 1) // 2 if m <= most else most * (most + 1) // 2 + (m - most) * most

    def upto(m):                 # pairs of the queries at positions 0 ... m - 1
        return sum_to(m, W) + sum_to(max(0, m - W), S)

    def low(n):                  # the window's first key
        return max(0, first(n) - W + 1)

    def first(n):
        return 0 if c["queries"] == c["keys"] else n - c["queries"]
    lengths = [n for n in _lengths(c) if n > first(n)]
    return (sum(upto(n) - upto(first(n)) for n in lengths),
            sum(n - low(n) + min(S, low(n)) for n in lengths))


def work(case):
    c = case
    if c["op"] == "rope":
        rows, size = c["seqs"] * c["tokens"], 2
        every, turned = (c["heads"] + 2 * c["kv_heads"]) * c["dim"], (c["heads"] + c["kv_heads"]) * c["dim"]
        moved = 2 * every + (2 * every + turned if c["grad"] else 0)
        return {"bytes": rows * moved * size, "flops": rows * turned * (30 if c["grad"] else 10)}
    if c["op"] == "window":
        pairs, keys = _pairs(c)
        queries, D = c["seqs"] * c["queries"] * c["heads"], c["dim"]
        moved = 2 * queries * D + 2 * keys * c["kv_heads"] * D
        if c["grad"]:
            moved += 2 * queries * D + 2 * c["seqs"] * c["kv_heads"] * c["keys"] * D
        return {"bytes": 2 * moved, "flops": pairs * c["heads"] * D * (14 if c["grad"] else 4)}
    size = 4 if c["dtype"] == "fp32" else 2
    n = c["trials"] * c["rows"]
    return {"bytes": n * c["vocab"] * size * (2 if c["grad"] else 1) + n * c["top"] * 8,
            "flops": n * c["vocab"] * (12 if c["grad"] else 6)}


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    def _rope(s):
        """The rotation as a complex product, the norm's derivative from its Jacobian."""
        c = s["case"]
        n, T, H, KV, D = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        pos = torch.arange(T, device="cuda").expand(n, T)
        if c["cache"]:
            pos = pos + s["start"].long()[:, None]
        unit = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, :, None]   # [n, T, 1, D/2]
        trial = torch.arange(n, device="cuda") // (n // c["trials"])

        def pairs(t):
            t = t.reshape(*t.shape[:-1], D // 2, 2) if c["interleaved"] else \
                t.reshape(*t.shape[:-1], 2, D // 2).transpose(-1, -2)
            return torch.complex(t[..., 0].contiguous(), t[..., 1].contiguous())

        def flat(z):
            t = torch.stack([z.real, z.imag], -1 if c["interleaved"] else -2)
            return t.reshape(*t.shape[:-2], D)
        x = s["qkv"].detach().double().view(n, T, H + 2 * KV, D)
        out, back, dws = [], [], []
        spans = [(0, H, s["wq"]), (H, H + KV, s["wk"])]
        for i, (a, b, w) in enumerate(spans):
            h, w = x[:, :, a:b], w.detach().double()[trial][:, None, None]
            r = 1.0 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
            out.append(flat(pairs(h * r * w) * unit).transpose(1, 2))
            if c["grad"]:
                d = flat(pairs(s["d"][i].double().transpose(1, 2)) * unit.conj())
                dws.append((d * h * r).sum((1, 2)).view(c["trials"], -1, D).sum(1))
                u = d * w
                back.append(r * u - h * r ** 3 * (u * h).sum(-1, keepdim=True) / D)
        v = x[:, :, H + KV:].transpose(1, 2)
        if c["cache"]:
            kc, vc = s["kcache"].double(), s["vcache"].double()
            for b, first in enumerate(s["start"].tolist()):
                kc[b, :, first:first + T], vc[b, :, first:first + T] = out[1][b], v[b]
            return out[0], kc, vc
        back.append(s["d"][2].double().transpose(1, 2))
        return [out[0], out[1], v, torch.cat(back, 2).reshape(n * T, -1)] + dws

    def _window(s):
        """Sequence by sequence and a few queries at a time, over the keys that any of them sees."""
        c = s["case"]
        n, H, KV, D, Tq, Tk = (c[k] for k in ("seqs", "heads", "kv_heads", "dim", "queries", "keys"))
        G, W, S = H // KV, c["window"] or Tk, c["sinks"]
        o = torch.zeros(n, H, Tq, D, dtype=torch.float64, device="cuda")
        dq, dk, dv = torch.zeros_like(o), *(torch.zeros(n, KV, Tk, D, dtype=torch.float64, device="cuda")
                                            for _ in range(2))
        start = s["start"].tolist() if s["start"] is not None else [0] * n
        for b, length in enumerate(s["lengths"].tolist()):
            for t0 in range(0, min(Tq, length - start[b]), 256):
                t1 = min(t0 + 256, Tq, length - start[b])
                i = torch.arange(start[b] + t0, start[b] + t1, device="cuda")
                low = max(0, int(i[0]) - W + 1)
                js = torch.cat([torch.arange(min(S, low), device="cuda"),
                                torch.arange(low, int(i[-1]) + 1, device="cuda")])
                ago = i[:, None] - js
                hide = (ago < 0) | ((ago >= W) & (js >= S))
                q = s["q"][b, :, t0:t1].double().view(KV, G, -1, D) / math.sqrt(D)
                k, v = (s[x][b][:, js].double()[:, None].expand(-1, G, -1, -1) for x in ("k", "v"))
                p = (q @ k.transpose(-1, -2)).masked_fill(hide, -math.inf).softmax(-1)
                o[b, :, t0:t1] = (p @ v).view(H, -1, D)
                if c["grad"]:
                    do = s["do"].view(n, Tq, H, D)[b, t0:t1].double().transpose(0, 1).reshape(KV, G, -1, D)
                    dp = do @ v.transpose(-1, -2)
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                    dq[b, :, t0:t1] = (ds @ k).view(H, -1, D) / math.sqrt(D)
                    dk[b].index_add_(1, js, (ds.transpose(-1, -2) @ q).sum(1))
                    dv[b].index_add_(1, js, (p.transpose(-1, -2) @ do).sum(1))
        o = o.transpose(1, 2).reshape(n * Tq, H * D)
        return [o, dq, dk, dv] if c["grad"] else o

    def _distill(s):
        c, tau, a = s["case"], s["temperature"], s["alpha"]
        R, V = s["logits"].shape
        loss = torch.empty(R, dtype=torch.float64, device="cuda")
        grad = torch.empty(R, V, dtype=torch.float64, device="cuda") if c["grad"] else None
        for r0 in range(0, R, 4096):
            r = slice(r0, r0 + 4096)
            x = s["logits"][r].detach().double()
            y, at = s["labels"][r].long(), s["index"][r].long()
            hard = torch.zeros_like(x)
            hard[y >= 0, y[y >= 0]] = 1.0
            soft = torch.zeros_like(x)
            score = s["top"][r].double().div(tau).masked_fill(at < 0, -math.inf)
            some = (at >= 0).any(1)
            q = torch.zeros_like(score)
            q[some] = score[some].softmax(1)
            soft.scatter_add_(1, at.clamp(min=0), q)
            lp1, lpt = x.log_softmax(1), (x / tau).log_softmax(1)
            inner = torch.where(q > 0, q.log(), torch.zeros_like(q)).mul(q).sum(1) - (soft * lpt).sum(1)
            loss[r] = (1 - a) * -(hard * lp1).sum(1) + a * tau * tau * inner
            if c["grad"]:
                d = (1 - a) * (hard.sum(1, keepdim=True) * lp1.exp() - hard)
                d += a * tau * (soft.sum(1, keepdim=True) * lpt.exp() - soft)
                grad[r] = d / c["rows"]
        loss = loss.view(c["trials"], -1).sum(1)
        return [loss, grad] if c["grad"] else loss

    s = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _rope, "window": _window, "distill": _distill}[case["op"]](s)
