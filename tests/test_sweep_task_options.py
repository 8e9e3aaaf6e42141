"""``mopt sweep --task-options``: the options of the LM tasks from the command line."""
import json

import pytest

from metaopt_amd.cli import main
from metaopt_amd.worker import tasks

OPTIONS = {"model": {"qk_norm": True, "kv_heads": 1, "window": 24, "sinks": 2}, "distill": [0.4, 2.0],
           "teacher_top": 5}


def test_a_sweep_trains_a_population_with_its_options(capsys, monkeypatch):
    """Four steps of two trials of the smallest preset, on the CPU backend."""
    built = []

    def build(population, device, seed, **kw):
        built.append(tasks._lm(population, "cpu", seed, preset="micro", seq_len=64, batch_size=2, n_tokens=1 << 12, **kw))
        return built[-1]
    spec = tasks.get("lm-tiny")
    monkeypatch.setattr(spec, "build", build)
    assert main(["--debug", "sweep", "-n", "sweep-lm-options", "--task", "lm-tiny", "--algo", "random", "--population",
                 "2", "--sync-every", "2", "--steps", "4", "--max-trials", "4", "--task-options", json.dumps(OPTIONS),
                 "--lr~loguniform(1e-4, 1e-3)", "--steps~fidelity(8, 8, 2)"]) == 0
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1])["experiment"]["name"] == "sweep-lm-options"
    (task, pop, data), = built
    assert (pop.cfg.qk_norm, pop.cfg.kv_heads, pop.cfg.window, pop.cfg.sinks) == (True, 1, 24, 2)
    assert pop.distill and pop.alpha.tolist() == [pytest.approx(0.4)] * 2 and data.top[0].shape[1] == 5


@pytest.mark.parametrize("task,text,match", [
    ("lm-tiny", "{", "JSON"), ("lm-tiny", "[1]", "JSON"), ("lm-tiny", '{"depth": 3}', "not known"),
    ("mlp", '{"model": {}}', "not known"), ("lm-tiny", '{"model": {"widow": 3}}', "widow")])
def test_refused_task_options(task, text, match):
    with pytest.raises(ValueError, match=match):
        main(["--debug", "sweep", "-n", "sweep-bad-options", "--task", task, "--population", "2", "--task-options", text])
