"""Data parallelism of the transformer operators' callers on the CPU: FusedMuon, the fused residual sums, predictions."""
import json
import os
import subprocess
import sys

import pytest

import _muon_dist_workers as W
from distributed_pytorch_amd import launch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("backend", ["gloo", "native"])
def test_muon_and_fused_residual_sums_under_ddp(tmp_path, backend):
    launch.spawn(W.train, 2, (2, launch.free_port(), str(tmp_path), backend))
    W.check(str(tmp_path), 2)


def _lines(path):
    return [json.loads(line) for line in path.read_text().splitlines()]


def _check_lines(lines, n):
    assert [v["sample"] for v in lines] == list(range(n))
    for v in lines:
        assert len(set(v["top"])) == 5 and v["top_logprob"] == sorted(v["top_logprob"], reverse=True) and v["logprob"] <= 0.0


def test_predictions_of_ranks_that_validate_different_samples(tmp_path):
    """The AMP script's ranks write a file each."""
    out, port = tmp_path / "pred.jsonl", str(launch.free_port())
    procs = []
    for r in range(2):
        env = dict(os.environ, WORLD_SIZE="2", RANK=str(r), LOCAL_RANK=str(r), MASTER_ADDR="127.0.0.1", MASTER_PORT=port)
        procs.append(subprocess.Popen(
            [sys.executable, os.path.join(ROOT, "scripts", "imagenet_ddp_apex.py"), "--synthetic", "-a", "squeezenet1_1", "-b", "8", "-p",
             "1", "--cpu", "--steps", "2", "--synthetic-size", "64", "--synthetic-val-size", "16", "--num-classes", "10", "--epochs", "1",
             "--opt-level", "O0", "--local_rank", str(r), "--dist-backend", "gloo", "--predictions", str(out), "--optimizer", "muon",
             "--lr", "0.001", "--out-dir", str(tmp_path / "out")], env=env, cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    for p in procs:
        _, err = p.communicate(timeout=300)
        assert p.returncode == 0, err[-2000:]
    assert not out.exists()
    for r in range(2):
        _check_lines(_lines(tmp_path / ("pred.jsonl.rank%d" % r)), 8)


def test_predictions_of_ranks_that_validate_the_same_samples(tmp_path):
    out = tmp_path / "pred.jsonl"
    r = subprocess.run(
        [sys.executable, os.path.join(ROOT, "scripts", "imagenet_ddp.py"), "--synthetic", "-a", "squeezenet1_1", "-b", "16", "-p", "1", "--cpu",
         "--steps", "2", "--synthetic-size", "64", "--synthetic-val-size", "16", "--num-classes", "10", "--epochs", "1", "--dist-url",
         "tcp://127.0.0.1:%d" % launch.free_port(), "--dist-backend", "gloo", "--world-size", "1", "--rank", "0", "--lr", "0.001",
         "--optimizer", "muon", "--predictions", str(out), "--out-dir", str(tmp_path / "out")],
        env=dict(os.environ, DPA_NPROC_PER_NODE="2"), cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert sorted(p.name for p in tmp_path.glob("pred*")) == ["pred.jsonl"]
    _check_lines(_lines(out), len(_lines(out)))
    assert len(_lines(out)) >= 8
