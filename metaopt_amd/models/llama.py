"""Llama-style decoder LMs trained as device populations (BASELINE.json configs 4 and 5).

``PopulationLM`` keeps ``capacity`` trials of ONE architecture on a GPU.  Every parameter tensor
is stacked over the population (``[P, ...]``), so a step is a handful of batched launches
regardless of ``P``:

* GEMMs: ``pbmm`` over the population dimension -- the hand-written gfx950 population GEMM
  (``ops/gemm.py`` -> ``csrc/pgemm.hip`` ``pgemm_big_kernel``: bf16 MFMA 16x16x32, f32
  accumulation, the SwiGLU and RoPE epilogues fused); no library GEMM runs in the step;
* embedding gather/scatter, RMSNorm, RoPE + head split, causal flash attention, SwiGLU, the
  vocabulary cross-entropy and the per-trial fused AdamW: hand-written gfx950 kernels
  (:mod:`metaopt_amd.ops.lm`);
* parameters live in flat buffers -- bf16 working copy ``p16`` (autograd leaves are views of it,
  with their ``.grad`` pre-bound to views of the flat bf16 gradient ``g16``), the f32 master
  (on the GPU split: ``p16`` is its high half, ``plo`` the int16 low half), AdamW moments
  ``m``/``v`` -- so the optimizer is ONE fused kernel over all tensors and trials,
  and a checkpoint / PBT exploit copy of a trial is a fixed set of contiguous slices.

The member interface (``set_member``, ``update_hparams``, ``save_states``/``load_states``,
``evaluate_async``, ...) is the one :class:`~metaopt_amd.worker.population_sweep.PopulationSweep`
drives for the MLP population, so the same sweep runs ASHA / PBT / TPE over LMs.

Options of :class:`LMConfig` (off in the presets): RMS norms of the query and key heads
(``qk_norm``), fewer key heads than query heads (``kv_heads``), a sliding attention window with sink
tokens (``window``, ``sinks``) -- :mod:`metaopt_amd.ops.heads`; ``PopulationLM(distill=...)`` trains
on a teacher's top logits beside the labels (:mod:`metaopt_amd.ops.distill`), and
:meth:`PopulationLM.greedy` continues prompts over a key / value cache.

Presets: ``llama-125m`` (d 768, 12 layers, 12 heads, SwiGLU 2048, vocab 32000; ~134M params with
an untied head) and ``tiny-2layer`` (the 2-layer LM of config 4).
"""
from __future__ import annotations

import dataclasses
import math
from dataclasses import dataclass
from typing import ClassVar, Dict, Optional, Tuple

import numpy as np
import torch

from ..ops import heads
from ..ops import lm as ops
from ..ops.distill import distill_loss
from ..ops.gemm import pbmm
from ..ops.population import MemberConfig
from .flatpop import FlatPopulation

@dataclass
class LMConfig:
    vocab: int = 32000
    d_model: int = 768
    n_layers: int = 12
    n_heads: int = 12
    ffn: int = 2048
    seq_len: int = 512
    rope_base: float = 10000.0
    norm_eps: float = 1e-5
    init_std: float = 0.02
    qk_norm: bool = False              # RMS norm, with a weight, of every query and key head
    kv_heads: Optional[int] = None     # key / value heads (None: n_heads); needs qk_norm
    window: Optional[int] = None       # tokens a query sees back, itself included (None: all)
    sinks: int = 0                     # first tokens seen whatever the window

    @property
    def head_dim(self) -> int:
        return self.d_model // self.n_heads

    @property
    def key_heads(self) -> int:
        return self.n_heads if self.kv_heads is None else self.kv_heads

    @property
    def plain_attention(self) -> bool:
        """Causal attention over all tokens without head norms or shared key heads."""
        return not self.qk_norm and self.key_heads == self.n_heads and self.window is None

    def check_heads(self) -> None:
        if self.key_heads < 1 or self.n_heads % self.key_heads:
            raise ValueError(f"{self.n_heads} heads are not a multiple of {self.key_heads} key heads")
        if self.key_heads != self.n_heads and not self.qk_norm:
            raise ValueError("kv_heads needs qk_norm")
        if (self.window is not None and self.window < 1) or self.sinks < 0:
            raise ValueError(f"window {self.window}, sinks {self.sinks}")
        if self.sinks and self.window is None:
            raise ValueError("sinks are seen beyond a window: give one")


PRESETS = {
    "llama-125m": LMConfig(),
    "tiny-2layer": LMConfig(vocab=4096, d_model=256, n_layers=2, n_heads=4, ffn=704,
                            seq_len=256),
    "micro": LMConfig(vocab=512, d_model=128, n_layers=2, n_heads=2, ffn=256, seq_len=64),
}


def param_specs(cfg: LMConfig):
    """(name, per-trial shape, init) of every tensor; init = ('normal', std) or ('ones',)."""
    d, F, V, L = cfg.d_model, cfg.ffn, cfg.vocab, cfg.n_layers
    out_std = cfg.init_std / math.sqrt(2 * L)
    specs = [("embed", (V, d), ("normal", cfg.init_std))]
    qkv = (cfg.n_heads + 2 * cfg.key_heads) * cfg.head_dim
    for l in range(L):
        specs += [(f"l{l}.attn_norm", (d,), ("ones",)),
                  (f"l{l}.wqkv", (d, qkv), ("normal", cfg.init_std)),
                  (f"l{l}.wo", (d, d), ("normal", out_std)),
                  (f"l{l}.mlp_norm", (d,), ("ones",)),
                  (f"l{l}.wgu", (d, 2 * F), ("normal", cfg.init_std)),
                  (f"l{l}.wdown", (F, d), ("normal", out_std))]
    specs += [("final_norm", (d,), ("ones",)), ("head", (d, V), ("normal", cfg.init_std))]
    if cfg.qk_norm:        # together: one run of the gradient buffer to clear
        specs += [(f"l{l}.{kind}_norm", (cfg.head_dim,), ("ones",)) for l in range(L) for kind in "qk"]
    return specs


def _lin(x, w):
    """Population linear layer; the weight gradient goes straight into the leaf's preset
    ``.grad`` (a view of the flat gradient buffer the fused AdamW reads)."""
    return pbmm(x, w, w.grad if w.requires_grad else None)


class PopulationLM(FlatPopulation):
    """``capacity`` Llama-style LM trials of one architecture (AdamW, per-trial lr / betas /
    weight decay, per-trial gradient clipping)."""

    optimizer = "adamw"
    secondary = "ppl"

    def __init__(self, capacity: int, config="tiny-2layer", batch_size: int = 8,
                 seq_len: Optional[int] = None, device="cuda", max_grad_norm: float = 1.0,
                 eval_batch: Optional[int] = None, use_graph: bool = True,
                 moment_dtype: Optional[torch.dtype] = None,
                 distill: Optional[Tuple[float, float]] = None):
        """``distill``: (alpha, temperature) of :func:`~metaopt_amd.ops.distill.distill_loss` --
        training batches are then (tokens, (labels, teacher's top logits, their indices)), as
        ``SyntheticLM(teacher_top=...)`` gives them.  ``self.alpha`` and ``self.temperature`` hold
        one value a trial and may be written in place between steps; they go with the trial's
        weights into checkpoints and copies, and a new trial (``set_member``) has those given here."""
        if moment_dtype is not None:       # AdamW first-moment storage (mopt sweep --dtype)
            self.moment_dtype = moment_dtype
        self.cfg = PRESETS[config] if isinstance(config, str) else config
        if seq_len is not None:
            self.cfg = dataclasses.replace(self.cfg, seq_len=seq_len)
        c = self.cfg
        c.check_heads()
        if c.head_dim not in ((64, 128) if c.qk_norm else (64,)) or c.seq_len % 64:
            raise ValueError("the attention kernel needs head_dim 64 (128 too with qk_norm) and "
                             "seq_len % 64 == 0")
        self.batch_size = int(batch_size)          # sequences per trial per step
        self.eval_batch = int(eval_batch or batch_size)
        self.tokens_per_step = self.batch_size * c.seq_len
        self.distill = distill is not None
        if self.distill:
            self._first_mix = alpha, temperature = tuple(float(x) for x in distill)
            if not (0.0 <= alpha <= 1.0 and temperature > 0.0):
                raise ValueError(f"distill {distill}: (alpha in [0, 1], temperature > 0)")
        super().__init__(capacity, device=device, max_grad_norm=max_grad_norm,
                         use_graph=use_graph)
        self.cos, self.sin = (ops.rope_tables(c.seq_len, c.rope_base, device=self.device)
                              if not c.qk_norm else
                              heads.rope_tables(c.seq_len, c.head_dim, c.rope_base, self.device))
        if self.distill:
            self.alpha, self.temperature = self.A["mix"][:, 0], self.A["mix"][:, 1]
            for slot in range(self.capacity):
                self.init_aux(slot)

    def aux_specs(self):
        return [("mix", 4)] if self.distill else []      # alpha, temperature (copied 4 values at a time)

    def init_aux(self, slot: int) -> None:
        if self.distill:
            for i, x in enumerate(self._first_mix):
                self.A["mix"][slot, i] = x

    def param_specs(self):
        return param_specs(self.cfg)

    # AdamW first moment in bf16 (28 -> 24 bytes per parameter per step)
    moment_dtype = torch.bfloat16

    def direct_grads(self):
        # projections (pgemm grad_out), norms and the embedding (cast into the .grad views); the
        # head norms' gradients are added by autograd
        return {name for name, _, _ in self.specs if not name.endswith((".q_norm", ".k_norm"))}

    def rows_per_batch(self, x) -> int:
        return int(x.numel())

    def train_rows(self) -> int:
        return self.tokens_per_step

    def _loss(self, tok: torch.Tensor, labels, train: bool):
        top = None
        if isinstance(labels, tuple):
            labels, *top = labels
        tok, labels = self._expand(tok, torch.int32), self._expand(labels, torch.int32)
        P, rpt, V = self.capacity, tok.numel() // self.capacity, self.cfg.vocab
        logits = self._logits(tok.view(P, -1, self.cfg.seq_len), self._attention)
        labels = labels.reshape(-1)
        if not train:
            return ops.ce_eval(logits, labels, rpt)
        if not self.distill:
            return ops.cross_entropy(logits, labels, rpt, grad_scale=1.0 / rpt, unit_weights=True)
        if top is None:
            raise ValueError("distillation takes batches (tokens, (labels, top values, top indices))")
        values, index = (self._expand(t, kind).reshape(P * rpt, -1)
                         for t, kind in zip(top, (None, torch.int32)))
        return distill_loss(logits, labels, values, index, rpt, self.temperature.contiguous(),
                            self.alpha.contiguous(), grad_scale=1.0 / rpt, unit_weights=True,
                            inplace=True)

    def _logits(self, tok: torch.Tensor, attend, last: bool = False):
        """Rows of logits of the tokens ``[P, sequences, T]`` (``last``: of each sequence's last
        token); ``attend(l, h, T)``: layer l's attention output of the normalised rows h."""
        c, P, W = self.cfg, self.capacity, self.W
        R, T, d = tok.numel(), tok.shape[-1], c.d_model
        rpt = R // P
        x = ops.embedding(tok.reshape(-1), W["embed"], rpt)
        # every residual add is fused into the pre-norm that follows it (ops.add_rmsnorm); the
        # embedding's two gradients (residual stream, first norm) meet in that norm's backward
        x, h = ops.rmsnorm_pass(x, W["l0.attn_norm"], rpt, c.norm_eps)
        for l in range(c.n_layers):
            o = attend(l, h.view(P, rpt, d), T)
            x, h = ops.add_rmsnorm(x, _lin(o.view(P, rpt, d), W[f"l{l}.wo"]).view(R, d),
                                   W[f"l{l}.mlp_norm"], rpt, c.norm_eps)
            # gate / up columns interleaved in 16-column groups: the SwiGLU runs in the GEMM
            # epilogues (ops.swiglu_mlp)
            y = ops.swiglu_mlp(h.view(P, rpt, d), W[f"l{l}.wgu"], W[f"l{l}.wdown"])
            nxt = W[f"l{l + 1}.attn_norm"] if l + 1 < c.n_layers else W["final_norm"]
            x, h = ops.add_rmsnorm(x, y.view(R, d), nxt, rpt, c.norm_eps)
        h = h.view(P, -1, T, d)[:, :, -1] if last else h.view(P, rpt, d)
        return _lin(h, W["head"]).view(-1, c.vocab)

    def _attention(self, l, h, T):
        c, W = self.cfg, self.W
        if c.plain_attention:
            # interleaved-pair RoPE applied by the QKV GEMM's epilogue and, backward, by the
            # attention kernels' gradient outputs (ops.qkv_rope_attention)
            return ops.qkv_rope_attention(h, W[f"l{l}.wqkv"], self.cos, self.sin, T, c.n_heads)
        if c.qk_norm:
            qkv = _lin(h, W[f"l{l}.wqkv"]).flatten(0, 1)
            q, k, v = heads.qk_norm_rope(qkv, W[f"l{l}.q_norm"], W[f"l{l}.k_norm"], self.cos, self.sin,
                                         T, c.n_heads, c.key_heads, c.norm_eps, il=True)
        else:
            q, k, v = ops.qkv_rope(h, W[f"l{l}.wqkv"], self.cos, self.sin, T, c.n_heads)
        return heads.window_attention(q, k, v, c.window, c.sinks)

    @torch.no_grad()
    def greedy(self, tok: torch.Tensor, steps: int) -> torch.Tensor:
        """The ``steps`` most likely next tokens, one after another, ``[P, sequences, steps]`` of
        every trial for the prompts ``tok`` ``[sequences, T]``, over a cache of keys and values
        (``qk_norm`` models; ``T + steps <= seq_len + 1``)."""
        c, P, W = self.cfg, self.capacity, self.W
        n, T = tok.shape
        if not c.qk_norm:
            raise ValueError("continuations need a model with qk_norm")
        if T < 1 or steps < 1 or T + steps > c.seq_len + 1:
            raise ValueError(f"{T} + {steps} tokens: a prompt and a step at least, and at most "
                             f"{c.seq_len + 1}")
        shape = (c.n_layers, P * n, c.key_heads, T + steps - 1, c.head_dim)
        kcache, vcache = (torch.zeros(shape, dtype=W["embed"].dtype, device=self.device)
                          for _ in "kv")
        start = torch.zeros(P * n, dtype=torch.int32, device=self.device)

        def attend(l, h, T):
            qkv = _lin(h, W[f"l{l}.wqkv"]).flatten(0, 1)
            q = heads.qk_norm_rope_cached(qkv, W[f"l{l}.q_norm"], W[f"l{l}.k_norm"], self.cos, self.sin,
                                          T, c.n_heads, kcache[l], vcache[l], start, c.norm_eps, il=True)
            return heads.window_attention(q, kcache[l], vcache[l], c.window, c.sinks, start=start)
        out, tok = [], self._expand(tok, torch.int32)
        for _ in range(steps):
            logits = self._logits(tok, attend, last=True).view(P, n, 1, c.vocab)
            start += tok.shape[-1]
            tok = logits.argmax(-1).to(torch.int32)
            out.append(tok)
        return torch.cat(out, -1)


class SyntheticLM:
    """Token streams from a fixed random sparse bigram model (so the loss can fall well below
    ``log(vocab)``): every token has ``branch`` likely successors.  Pre-generated on the host
    with numpy (vectorised over many chains), stored on the device, sliced per step.

    ``teacher_top``: training batches are (tokens, (labels, values, indices)) with the model's own
    largest log-probabilities of each next token, that many or ``branch`` of them (a successor may
    come twice), for ``PopulationLM(distill=...)``."""

    def __init__(self, vocab: int, seq_len: int, batch_size: int, n_tokens: int = 1 << 21,
                 branch: int = 8, seed: int = 0, device=None, n_val_seq: Optional[int] = None,
                 teacher_top: int = 0):
        rng = np.random.default_rng(seed)
        self.vocab, self.seq_len, self.batch_size = vocab, seq_len, batch_size
        succ = rng.integers(0, vocab, size=(vocab, branch))
        probs = rng.dirichlet(np.full(branch, 0.5), size=vocab)
        cdf = np.cumsum(probs, 1)
        L = seq_len + 1
        n_seq = max(batch_size * 4, n_tokens // L)
        toks = np.empty((n_seq, L), dtype=np.int32)
        toks[:, 0] = rng.integers(0, vocab, size=n_seq)
        for t in range(1, L):
            u = rng.random(n_seq)
            prev = toks[:, t - 1]
            k = (u[:, None] > cdf[prev]).sum(1).clip(max=branch - 1)
            toks[:, t] = succ[prev, k]
        dev = torch.device(device) if device is not None else torch.device("cpu")
        n_val = n_val_seq or batch_size
        self.train = torch.from_numpy(toks[n_val:]).to(dev)
        self.val = torch.from_numpy(toks[:n_val]).to(dev)
        self.n_batches = len(self.train) // batch_size
        self.top = None
        if teacher_top:
            order = np.argsort(-probs, 1, kind="stable")[:, :teacher_top]
            with np.errstate(divide="ignore"):
                values = np.log(np.take_along_axis(probs, order, 1)).astype(np.float32)
            index = np.take_along_axis(succ, order, 1).astype(np.int32)
            self.top = torch.from_numpy(values).to(dev), torch.from_numpy(index).to(dev)

    def batch(self, step: int):
        i = step % self.n_batches
        b = self.train[i * self.batch_size:(i + 1) * self.batch_size]
        if self.top is not None:
            return b[:, :-1], (b[:, 1:], *(t[b[:, :-1].long()] for t in self.top))
        return b[:, :-1], b[:, 1:]

    def validation(self):
        return self.val[:, :-1], self.val[:, 1:]


LM_PBT_PRIORS = {
    "/lr": "loguniform(1e-4, 3e-3)",
    "/weight_decay": "loguniform(1e-3, 0.3)",
    "/beta1": "uniform(0.8, 0.95)",
    "/steps": "fidelity(200, 2000, 2)",
}


@dataclass
class LMSweepTask:
    """Maps trial parameters to LM population members (AdamW lr / wd / beta1)."""

    priors: Dict[str, str] = dataclasses.field(default_factory=lambda: dict(LM_PBT_PRIORS))
    # key(params) == param_key(params, fidelity): the sweep may derive it from points directly
    key_by_params: ClassVar[bool] = True
    fidelity: str = "/steps"
    secondary_stat: str = "val_ppl"
    d_model: int = 768
    member_defaults: Dict = dataclasses.field(default_factory=lambda: {"beta2": 0.95})

    def member_config(self, params: Dict, seed: int) -> MemberConfig:
        return MemberConfig(width=self.d_model, lr=float(params["/lr"]),
                            momentum=float(params.get("/beta1", 0.9)),
                            weight_decay=float(params.get("/weight_decay", 0.0)),
                            dropout=0.0, seed=int(seed) & 0x7FFFFFFF, **self.member_defaults)

    def budget(self, params: Dict) -> int:
        return int(params[self.fidelity])

    def key(self, params: Dict) -> str:
        from .mlp import param_key
        return param_key(params, self.fidelity)

    @staticmethod
    def seed_of(key: str) -> int:
        return int(key[:8], 16)
