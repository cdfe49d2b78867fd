"""Step times and throughput of the trainer do not count ``--score-every``."""

from __future__ import annotations

import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The trainer with scores that take a second longer.
SLOW_SCORES = """
import importlib.util, sys, time
spec = importlib.util.spec_from_file_location("train_gpt", sys.argv[1])
trainer = importlib.util.module_from_spec(spec)
spec.loader.exec_module(trainer)
real = trainer.token_logprobs
def slow(*args, **kwargs):
    time.sleep(1.0)
    return real(*args, **kwargs)
trainer.token_logprobs = slow
trainer.main(sys.argv[2:])
"""


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("timing", ["device", "host"])
def test_scores_are_not_timed(device, timing, tmp_path):
    if device == "cpu" and timing == "device":
        pytest.skip("no device time on CPU")
    path = tmp_path / "m.jsonl"
    args = ["--layers", "1", "--embd", "64", "--heads", "2", "--vocab", "256", "--seq-len", "32", "--batch-size", "2",
            "--steps", "4", "--score-every", "2", "--timing", timing, "--metrics-jsonl", str(path)]
    env = dict(os.environ, OMP_NUM_THREADS="2")
    if device == "cpu":
        env["CUDA_VISIBLE_DEVICES"] = ""
        args += ["--backend", "gloo"]
    proc = subprocess.run([sys.executable, "-c", SLOW_SCORES, os.path.join(ROOT, "examples", "train_gpt.py"), *args],
                          capture_output=True, text=True, timeout=300, env=env, cwd=ROOT)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-3000:]
    recs = [json.loads(line) for line in path.read_text().splitlines()]
    assert sum(r.get("event") == "score" for r in recs) == 2
    # two seconds of scores over four steps would show as 500 ms a step
    times = [r["ms_per_step"] for r in recs if "ms_per_step" in r]
    assert len(times) >= 2 and all(t < 400 for t in times), recs
