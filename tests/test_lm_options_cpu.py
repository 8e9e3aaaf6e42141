"""The population LM's attention options, distillation and continuations on the CPU backend."""
import dataclasses
import math

import numpy as np
import pytest
import torch

from metaopt_amd.models.hyper import HypergradLM
from metaopt_amd.models.llama import PRESETS, PopulationLM, SyntheticLM, param_specs
from metaopt_amd.ops.population import MemberConfig
from metaopt_amd.worker import tasks

MICRO = PRESETS["micro"]
FULL = dict(qk_norm=True, kv_heads=1, window=20, sinks=3)


def _population(distill=None, **options):
    pop = PopulationLM(2, dataclasses.replace(MICRO, **options), batch_size=2, device="cpu",
                       distill=distill)
    for s in range(2):
        pop.set_member(s, MemberConfig(width=128, lr=1e-3, seed=3 + s, beta2=0.95))
    return pop


def _in_64_bits(pop):
    pop.W = {k: w.detach().double().requires_grad_(True) for k, w in pop.W.items()}
    return pop


def test_presets_have_none_of_them():
    shapes = {n: s for n, s, _ in param_specs(MICRO)}
    assert shapes["l0.wqkv"] == (128, 384) and not any("q_norm" in n for n in shapes)
    assert all(c.plain_attention for c in PRESETS.values())
    shapes = {n: s for n, s, _ in param_specs(dataclasses.replace(MICRO, **FULL))}
    assert shapes["l0.wqkv"] == (128, 256) and shapes["l1.k_norm"] == (64,)


@pytest.mark.parametrize("options,match", [
    (dict(kv_heads=3, qk_norm=True), "not a multiple"), (dict(kv_heads=0, qk_norm=True), "not a multiple"),
    (dict(kv_heads=1), "needs qk_norm"), (dict(sinks=2), "beyond a window"),
    (dict(n_heads=1), "head_dim"), (dict(n_heads=4, qk_norm=True), "head_dim"),
    (dict(window=0), "window"), (dict(window=8, sinks=-1), "sinks"), (dict(seq_len=100, window=8), "seq_len")])
def test_refused_options(options, match):
    with pytest.raises(ValueError, match=match):
        _population(**options)


def test_refused_calls():
    for bad in ((1.5, 1.0), (0.5, 0.0)):
        with pytest.raises(ValueError, match="alpha in"):
            _population(distill=bad)
    with pytest.raises(ValueError, match="hypergradients"):
        HypergradLM(1, dataclasses.replace(MICRO, window=8), device="cpu")
    data = SyntheticLM(512, 64, 2, n_tokens=1 << 12)
    with pytest.raises(ValueError, match="top values"):
        _population(distill=(0.5, 1.0)).train_step(*data.batch(0))
    tok = data.batch(0)[0]
    with pytest.raises(ValueError, match="qk_norm"):
        _population(window=8).greedy(tok[:, :4], 2)
    for cut, steps in ((0, 2), (4, 0), (64, 2)):
        with pytest.raises(ValueError, match="a prompt and a step"):
            _population(**FULL).greedy(tok[:, :cut], steps)


@pytest.mark.parametrize("options", [
    dict(window=20, sinks=3), dict(qk_norm=True), FULL, dict(n_heads=1, qk_norm=True, window=9)])
@pytest.mark.parametrize("distill", [None, (0.4, 2.0)])
def test_steps_run(options, distill):
    pop = _population(distill, **options)
    data = SyntheticLM(512, 64, 2, n_tokens=1 << 12, teacher_top=5 if distill else 0)
    before = pop.p32.clone()
    for step in range(2):
        pop.train_step(*data.batch(step))
    assert np.isfinite(pop.train_loss()).all() and np.isfinite(pop.evaluate(*data.validation())[0]).all()
    moved = {n: not torch.equal(before[o:o + 2 * k], pop.p32[o:o + 2 * k])
             for (n, _, _), (o, k) in zip(pop.specs, pop.segments)}
    assert all(moved.values()), moved


@pytest.mark.parametrize("distill", [None, (0.4, 2.0)])
def test_gradients_match_differences(distill):
    pop = _in_64_bits(_population(distill, **FULL))
    data = SyntheticLM(512, 64, 2, n_tokens=1 << 12, teacher_top=5 if distill else 0)
    x, y = data.batch(0)
    pop._loss(x, y, True).sum().backward()
    rng = torch.Generator().manual_seed(0)
    scale = 1.0 / (x.numel())       # gradients are those of the mean over a trial's rows
    for name in ("l0.q_norm", "l1.k_norm", "l0.wqkv", "l1.wo", "head", "embed"):
        w = pop.W[name]
        d = torch.randn(w.shape, generator=rng, dtype=torch.float64)
        d /= d.norm()
        with torch.no_grad():
            h = 1e-3
            ends = []
            for sign in (h, -h):
                w += sign * d
                ends.append(pop._loss(x, y, True).sum().item() * scale)
                w -= sign * d
        slope = (ends[0] - ends[1]) / (2 * h)
        # some of the reference's pieces compute in 32 bits: 2^-24 x ~100 operations of a mean loss of
        # about 6, over 2 h: 2e-2 x 2^-10; the third derivative's share is h^2
        assert abs(slope - (w.grad * d).sum().item()) <= 6 * 100 * 2.0 ** -24 / (2 * h) / 10 + 1e-4, name


def test_window_over_all_tokens_is_plain_attention():
    """Nothing out of the window: the plain model's loss, to the rounding of its 16-bit tensors."""
    plain, wide = _population(), _population(window=64, sinks=1)
    with torch.no_grad():
        wide.p16.copy_(plain.p16)
    data = SyntheticLM(512, 64, 2, n_tokens=1 << 12)
    a, b = (p.evaluate(*data.validation())[0] for p in (plain, wide))
    # logits of about 1, each off by a few half steps: far under one such step of the mean loss
    assert np.abs(a - b).max() <= 2.0 ** -8 * math.log(512)


def test_greedy_is_the_whole_pass_again():
    pop = _in_64_bits(_population(**FULL))
    prompt = SyntheticLM(512, 64, 3, n_tokens=1 << 12).batch(0)[0][:, :30]
    got = pop.greedy(prompt, 6)
    assert got.shape == (2, 3, 6) and got.dtype == torch.int32
    tok = pop._expand(prompt, torch.int32)
    for step in range(6):
        with torch.no_grad():
            last = pop._logits(tok, pop._attention).view(2, 3, -1, 512)[:, :, -1]
        top = last.topk(2).values
        best = last.argmax(-1)
        # (some of the reference's pieces compute in 32 bits: a tie may go either way)
        sure = top[..., 0] - top[..., 1] > 1e-4
        assert sure.any()
        assert torch.equal(got[:, :, step][sure], best[sure].int())
        tok = torch.cat([tok, got[:, :, step:step + 1]], -1)


def test_synthetic_teacher():
    plain = SyntheticLM(512, 64, 4, n_tokens=1 << 12, seed=5)
    data = SyntheticLM(512, 64, 4, n_tokens=1 << 12, seed=5, teacher_top=8)
    (x, y), (x2, (y2, values, index)) = plain.batch(1), data.batch(1)
    assert torch.equal(x, x2) and torch.equal(y, y2)
    assert values.shape == index.shape == (4, 64, 8) and index.dtype == torch.int32
    assert (values.double().exp().sum(-1) - 1).abs().max() <= 16 * 2.0 ** -24
    assert (values[..., :-1] >= values[..., 1:]).all()
    assert (index == y[..., None]).any(-1).all()           # every next token is one of them
    assert SyntheticLM(512, 64, 4, n_tokens=1 << 12, teacher_top=3).batch(0)[1][1].shape == (4, 64, 3)
    assert len(data.validation()) == 2 and data.validation()[1].shape == (4, 64)


def test_task_builds_them():
    task, pop, data = tasks.get("lm-tiny").build(2, "cpu", 0, n_tokens=1 << 12, batch_size=2,
                                                 model=dict(qk_norm=True, window=64, sinks=2),
                                                 distill=(0.5, 2.0), teacher_top=4)
    assert pop.cfg.window == 64 and pop.cfg.qk_norm and pop.distill
    for s in range(2):
        pop.set_member(s, task.member_config({"/lr": 1e-3, "/steps": 1}, s))
    pop.train_step(*data.batch(0))
    assert np.isfinite(pop.train_loss()[0])


def _with_weights(pop, std, seed=1):
    """Matrices of N(0, std), norms of N(1, 0.2): weights with which every part counts."""
    rng = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, w in pop.W.items():
            w.copy_(torch.randn(w.shape, generator=rng) * (0.2 if "norm" in name else std) + ("norm" in name))
    return pop


@pytest.mark.parametrize("options", [FULL, dict(window=20, sinks=3)])
@pytest.mark.parametrize("distill", [None, (0.4, 2.0)])
def test_gradients_have_the_slope_s_size_and_direction(options, distill):
    """Along a gradient the loss rises by its norm: no other direction is as steep, and a gradient that is
    scaled or lacks a part is told by it.

    The loss, of at most 12 for 512 tokens, passes some 32-bit pieces: 16 roundings of it are 1.2e-5 at
    most, over 2 h 6e-4.  The third derivative's share, h^2 of the slope's size times what a step of 1
    changes of it (some tens), is under 1 %."""
    pop = _with_weights(_in_64_bits(_population(distill, **options)), 0.15)
    x, y = SyntheticLM(512, 64, 2, n_tokens=1 << 12, teacher_top=5 if distill else 0).batch(0)
    loss = lambda: pop._loss(x, y, True).sum() / x.numel()  # noqa: E731
    pop._loss(x, y, True).sum().backward()     # (gradients are those of the mean over a trial's rows)
    h = 1e-2
    for name, w in pop.W.items():
        size = w.grad.norm().item()
        assert size > 0.03, name               # (well over what the tolerance leaves open)
        with torch.no_grad():
            d = h * w.grad / size
            ends = [(w.add_(s * d), loss().item(), w.sub_(s * d))[1] for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * h)
        assert abs(slope - size) <= 0.01 * size + 16 * 12 * 2.0 ** -24 / (2 * h), (name, slope, size)


def test_a_window_over_all_tokens_is_plain_attention_and_a_shorter_one_is_not():
    """Rows of logits, in 64 bits but for the plain attention's 32: 2^-24 times some hundred operations."""
    x = SyntheticLM(512, 64, 2, n_tokens=1 << 12).batch(0)[0]

    def logits(**options):
        pop = _with_weights(_in_64_bits(_population(**options)), 0.15)
        with torch.no_grad():
            return pop._logits(pop._expand(x, torch.int32), pop._attention)
    plain = logits()
    off = {w: ((logits(window=w, sinks=s) - plain).norm() / plain.norm()).item()
           for w, s in ((64, 1), (63, 0), (5, 0))}
    assert off[64] <= 500 * 2.0 ** -24
    assert off[63] > 20 * 500 * 2.0 ** -24 and off[5] > 0.1, off


def test_greedy_forms_logits_of_last_tokens_only(monkeypatch):
    """A prompt's other rows, vocabulary wide, are the largest tensors there would be."""
    from metaopt_amd.models import llama
    pop = _population(**FULL)
    prompt = SyntheticLM(512, 64, 3, n_tokens=1 << 12).batch(0)[0][:, :30]
    rows, lin = [], llama._lin

    def watched(x, w):
        if w is pop.W["head"]:
            rows.append(x.shape[1])
        return lin(x, w)
    monkeypatch.setattr(llama, "_lin", watched)
    pop.greedy(prompt, 4)
    assert rows == [3] * 4, rows


def test_a_trial_s_mix_goes_where_its_weights_go():
    """alpha and temperature of a trial are in its checkpoints, in what is sent to another rank and in copies
    between slots; a new trial has those that the population was built with."""
    pop = _population((0.4, 2.0), **FULL)
    pop.alloc_ckpt_pool(2)
    mix = lambda s, p=pop: (p.alpha[s].item(), p.temperature[s].item())  # noqa: E731
    first = (pytest.approx(0.4), 2.0)
    assert [mix(0), mix(1)] == [first] * 2
    pop.alpha[0], pop.temperature[0] = 0.75, 3.5
    meta, = pop.save_states([(0, 1)])
    sent = pop.unpack_state(pop.pack_state(pop.pool_state(meta)).clone())
    state = pop.slot_state(0)
    pop.set_member(0, MemberConfig(width=128, lr=1e-3, seed=9))
    assert mix(0) == first
    pop.load_states([(1, meta)])
    assert [mix(0), mix(1)] == [first, (0.75, 3.5)]
    pop.load_slot_state(0, state)
    assert mix(0) == (0.75, 3.5)
    pop.set_member(1, MemberConfig(width=128, lr=1e-3, seed=10))
    pop.copy_member(0, 1)
    assert mix(1) == (0.75, 3.5)
    other = _population((0.1, 1.0), **FULL)
    other.load_slot_state(0, sent)
    assert mix(0, other) == (0.75, 3.5) and mix(1, other) == (pytest.approx(0.1), 1.0)
    tensors = pop.c4_send_tensors(meta)
    got = other._c4_header()
    got.copy_(tensors[1])
    other.alloc_ckpt_pool(1)
    other._ck[0].copy_(tensors[0])
    other.load_states([(1, other.c4_finish(0, [other._ck[0], got]))])
    assert mix(1, other) == (0.75, 3.5)
    # a state of a population without a mix (or from before it was kept) leaves the slot's
    plain = _population(None, **FULL)
    assert plain.n_aux == 0
    other.load_slot_state(0, plain.slot_state(0))
    assert mix(0, other) == (0.75, 3.5)
