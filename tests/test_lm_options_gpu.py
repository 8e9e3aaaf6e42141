"""Head norms, windowed attention and distillation together on the GPU: the chain that a training
step runs, a prompt against its tokens one by one, and the population LM that calls them."""
import dataclasses

import numpy as np
import pytest
import torch

from metaopt_amd.models.llama import PRESETS, PopulationLM, SyntheticLM
from metaopt_amd.ops import distill, heads
from metaopt_amd.ops.gemm import pbmm
from metaopt_amd.ops.population import MemberConfig

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
U = 2.0 ** -8


def _off(got, want):
    """|got - want| relative to |want|, as norms."""
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("T,H,KV,D,window,sinks", [(77, 4, 2, 64, 20, 3), (200, 2, 1, 128, 64, 0),
                                                   (1, 4, 4, 64, 5, 1)])
def test_from_the_projection_to_the_loss(T, H, KV, D, window, sinks):
    """qkv -> normed, rotated heads -> attention -> logits -> distillation, and back.

    Normed queries and keys have norms of about sqrt(D) / 4 and sqrt(D) (the weights' sizes), each
    off by U: scores of q k / sqrt(D) are off by at most 2 U sqrt(D) / 4 <= 5.7 U, and so are,
    relatively, probabilities.  A gradient meets them three times (the forward's output in D, P and
    dS) and at most 12 more tensors rounded once (q, k, v, P, o, logits, their gradient, do, dS, the
    attention's gradients, dqkv or dw, the head): 30 U as norms."""
    torch.manual_seed(T)
    P, n, V, K = 2, 3, 504, 9
    R = P * n * T
    cos, sin = heads.rope_tables(T, D, device=DEV)
    rand = lambda *s, scale=1.0, mean=0.0: (  # noqa: E731
        torch.randn(*s, device=DEV) * scale + mean).to(BF).requires_grad_(True)
    qkv, head = rand(R, (H + 2 * KV) * D), rand(P, H * D, V, scale=(H * D) ** -0.5)
    wq, wk = rand(P, D, scale=0.02, mean=0.25), rand(P, D, scale=0.1, mean=1)
    y = torch.randint(0, V, (R,), device=DEV, dtype=torch.int32)
    index = torch.randint(0, V, (R, K), device=DEV, dtype=torch.int32)
    top = torch.randn(R, K, device=DEV)
    tau, alpha = torch.tensor([1.0, 2.5], device=DEV), torch.tensor([0.3, 0.8], device=DEV)
    lengths = torch.tensor([T, max(1, T // 2), T, T, 1, T], device=DEV, dtype=torch.int32)

    q, k, v = heads.qk_norm_rope(qkv, wq, wk, cos, sin, T, H, KV)
    o = heads.window_attention(q, k, v, window, sinks, start=0, lengths=lengths)
    logits = pbmm(o.view(P, n * T, H * D), head).view(R, V)
    loss = distill.distill_loss(logits, y, top, index, n * T, tau, alpha, grad_scale=1 / (n * T),
                                unit_weights=True, inplace=True)
    leaves = [qkv, wq, wk, head]
    grads = torch.autograd.grad(loss.sum(), leaves)

    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    x, a, b, h = exact
    q, k, v = heads.qk_norm_rope_ref(x, a, b, cos, sin, T, H, KV)
    o = heads.window_attention_ref(q, k, v, window, sinks, start=0, lengths=lengths)
    logits = (o.view(P, n * T, H * D) @ h).view(R, V)
    want = distill.distill_ref(logits, y, top.double(), index, n * T, tau.double(), alpha.double())
    exact = torch.autograd.grad(want.sum() / (n * T), exact)
    assert ((loss - want).abs() <= 30 * U * want.abs()).all()
    for name, g, e in zip(("qkv", "wq", "wk", "head"), grads, exact):
        assert torch.isfinite(g).all(), name
        if T == 1 and name in ("wq", "wk"):      # one key: nothing depends on them
            assert e.norm() == 0 and g.double().norm() <= 30 * U * exact[0].norm() * D ** 0.5
        else:
            assert _off(g, e) <= 30 * U, (name, _off(g, e))


@pytest.mark.parametrize("H,KV,D,window,sinks", [(4, 2, 64, 20, 3), (3, 3, 128, None, 0)])
def test_a_prompt_and_its_tokens_one_by_one(H, KV, D, window, sinks):
    torch.manual_seed(H)
    n, T = 3, 70
    cos, sin = heads.rope_tables(T, D, device=DEV)
    qkv = torch.randn(n, T, (H + 2 * KV) * D, device=DEV).to(BF)
    wq, wk = (torch.randn(1, D, device=DEV).to(BF) for _ in "qk")
    caches = [[torch.zeros(n, KV, T, D, device=DEV, dtype=BF) for _ in "kv"] for _ in range(2)]
    zero = torch.zeros(n, dtype=torch.int32, device=DEV)
    q = heads.qk_norm_rope_cached(qkv.flatten(0, 1), wq, wk, cos, sin, T, H, *caches[0], zero)
    whole = heads.window_attention(q, *caches[0], window, sinks, start=zero).view(n, T, H * D)
    for t in range(T):
        at = zero + t
        one = heads.qk_norm_rope_cached(qkv[:, t], wq, wk, cos, sin, 1, H, *caches[1], at)
        assert torch.equal(one, q[:, :, t:t + 1])
        o = heads.window_attention(one, *caches[1], window, sinks, start=at)
        # both are rounded once, as are both's probabilities: 4 U of the largest value at most
        assert ((o - whole[:, t]).float().abs() <= 4 * U * caches[0][1].abs().max().float()).all(), t
    assert all(torch.equal(a, b) for a, b in zip(*caches))


FULL = dict(qk_norm=True, kv_heads=1, window=20, sinks=3)
OPTIONS = [(FULL, (0.4, 2.0)), (dict(window=20), None), (dict(n_heads=1, qk_norm=True), (1.0, 1.0))]


def _population(options, distilled, device=DEV, graph=True, lr=2e-3):
    pop = PopulationLM(2, dataclasses.replace(PRESETS["micro"], **options), batch_size=4, device=device,
                       distill=distilled, use_graph=graph)
    for s in range(2):
        pop.set_member(s, MemberConfig(width=128, lr=lr * (s + 1), seed=7 + s, beta2=0.95))
    return pop


def _data(distilled):
    return SyntheticLM(512, 64, 4, n_tokens=1 << 14, seed=0, device=DEV,
                       teacher_top=6 if distilled else 0)


@pytest.mark.parametrize("options,distilled", OPTIONS)
def test_population_gradients_match_the_reference_backend(options, distilled):
    """About 40 tensors lie between a weight and the loss in a model of 2 layers, each rounded once
    here and once there: 80 U as norms."""
    gpu, cpu = _population(options, distilled, graph=False), _population(options, distilled, "cpu")
    with torch.no_grad():
        cpu.p32.copy_(gpu.master_flat().cpu())
        cpu.p16.copy_(gpu.p16.cpu())
    x, y = _data(distilled).batch(0)
    host = tuple(t.cpu() for t in y) if isinstance(y, tuple) else y.cpu()
    gpu.train_step(x, y)
    cpu.train_step(x.cpu(), host)
    assert np.abs(gpu.train_loss() / cpu.train_loss() - 1).max() <= 80 * U
    for (name, _, _), (o, k) in zip(gpu.specs, gpu.segments):
        want = cpu.g16[o:o + 2 * k].double()
        assert _off(gpu.g16[o:o + 2 * k].cpu(), want) <= 80 * U, name


@pytest.mark.parametrize("options,distilled", OPTIONS)
def test_population_steps_replay(options, distilled):
    """A captured step, replayed with evaluations and another population's eager steps between, has
    the eager step's gradients bit for bit (at fixed weights: the norm that the optimizer clips by is
    summed by atomics, as is the cross-entropy's loss: 256 terms in any order)."""
    pops = [_population(options, distilled, graph=g, lr=0.0) for g in (True, False)]
    with torch.no_grad():
        pops[1].p16.copy_(pops[0].p16)
        pops[1].master_buf.copy_(pops[0].master_buf)
    data = _data(distilled)
    for step in range(4):
        for pop in pops:
            pop.train_step(*data.batch(step))
        a, b = (pop.train_loss() for pop in pops)
        for pop in pops:
            pop.evaluate(*data.validation())
        assert torch.equal(pops[0].g16, pops[1].g16), step
        assert np.abs(a - b).max() <= (0 if distilled else 2 * 256 * 2.0 ** -24 * b.max()), step
    assert pops[0].g16.float().abs().sum() > 0


def test_mix_is_read_by_the_captured_step():
    """alpha and temperature, written in place, reach the replays."""
    pops = [_population(FULL, (0.9, 1.0), graph=g, lr=0.0) for g in (True, False)]
    with torch.no_grad():
        pops[1].p16.copy_(pops[0].p16)
        pops[1].master_buf.copy_(pops[0].master_buf)
    data, seen = _data(True), []
    for step in range(3):
        for pop in pops:
            pop.alpha[1] = 0.1 * step
            pop.temperature[0] = 1.0 + step
            pop.train_step(*data.batch(0))
        seen.append(pops[0].train_loss())
        assert np.array_equal(seen[-1], pops[1].train_loss())
    assert len({s[0] for s in seen}) == len({s[1] for s in seen}) == 3


def test_greedy_continuations():
    pop = _population(FULL, None)
    prompt = _data(False).batch(0)[0][:3, :30]
    got = pop.greedy(prompt, 7)
    assert got.shape == (2, 3, 7) and got.dtype == torch.int32
    tok = pop._expand(prompt, torch.int32)
    for step in range(7):
        with torch.no_grad():
            last = pop._logits(tok, pop._attention).view(2, 3, -1, 512)[:, :, -1].float()
        # of about 20 tensors in front of the logits each is rounded once on either way
        top = last.amax(-1)
        chosen = last.gather(-1, got[:, :, step:step + 1].long())[..., 0]
        assert (top - chosen <= 2 * 40 * U * last.abs().amax()).all()
        tok = torch.cat([tok, got[:, :, step:step + 1]], -1)


def _with_weights(pop, std, seed=1):
    """Matrices of N(0, std), norms of N(1, 0.2), as 16-bit values, the same on either device."""
    rng = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, w in pop.W.items():
            t = torch.randn(w.shape, generator=rng) * (0.2 if "norm" in name else std) + ("norm" in name)
            w.copy_(t.to(BF))
    return pop


@pytest.mark.parametrize("options,distilled,wrong", [
    (FULL, (0.4, 2.0), [dict(window=19), dict(window=21), dict(sinks=2), dict(sinks=4)]),
    (dict(window=20, sinks=3), None, [dict(window=19), dict(sinks=2)]),
    (dict(n_heads=1, qk_norm=True), (1.0, 1.0), [dict(window=48)])])
def test_population_gradients_tell_a_token_more_or_less(options, distilled, wrong):
    """Loss and gradients of the population against the model in 64 bits with the same 16-bit weights, and
    how far those of a window or sinks one token off are (where all 64 are seen: of a window of 48).

    About 40 tensors between a weight and the loss are rounded once, each value by at most U of it and, over
    values, by U / sqrt(3) at the root of the mean square; independent, they add up to sqrt(40 / 3) U =
    1.4 %.  Two layers' norms and softmaxes pass errors on about as they are: 12 U = 4.7 % is three times
    that.  The mean loss is such a sum over 512 tokens, each off by 1.4 % of its logits' size at most."""
    limit = 12 * U
    x, y = _data(distilled).batch(0)
    host = tuple(t.cpu() for t in y) if isinstance(y, tuple) else y.cpu()
    gpu = _with_weights(_population(options, distilled, graph=False), 0.06)
    loss = gpu._loss(x, y, True)
    loss.backward(torch.ones_like(loss))

    def exact(**changes):
        pop = _population(dict(options, **changes), distilled, "cpu")
        pop.W = {k: w.detach().double().requires_grad_(True) for k, w in _with_weights(pop, 0.06).W.items()}
        loss = pop._loss(x.cpu(), host, True)
        loss.sum().backward()
        return loss.detach(), {k: w.grad for k, w in pop.W.items()}
    want, grads = exact()
    assert ((loss.detach().cpu() - want).abs() <= limit / 3 * want.abs()).all()
    far = {k: _off(gpu.W[k].grad.cpu(), g) for k, g in grads.items()}
    assert max(far.values()) <= limit, far
    for changes in wrong:
        other = exact(**changes)[1]
        assert max(_off(other[k], g) for k, g in grads.items()) > 2 * limit, changes


def test_a_trial_s_mix_is_in_its_checkpoints():
    """... and a captured step reads what was loaded."""
    pops = [_population(FULL, (0.4, 2.0), graph=g, lr=0.0) for g in (True, False)]
    data, seen = _data(True), []
    for pop in pops:
        pop.alloc_ckpt_pool(1)
        pop.train_step(*data.batch(0))
        pop.alpha[0], pop.temperature[0] = 0.75, 3.5
        meta, = pop.save_states([(0, 0)])
        pop.set_member(0, MemberConfig(width=128, lr=0.0, seed=7, beta2=0.95))
        assert (pop.alpha[0].item(), pop.temperature[0].item()) == (torch.tensor(0.4).item(), 2.0)
        pop.load_states([(1, meta)])
        assert (pop.alpha[1].item(), pop.temperature[1].item()) == (0.75, 3.5)
        pop.train_step(*data.batch(0))
        seen.append(pop.train_loss())
    assert np.array_equal(*seen) and seen[0][0] != seen[0][1]
