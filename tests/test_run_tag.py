"""The default name of a run, under which its checkpoints lie, tells runs of
other models apart."""
import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARGS = ["--dnn", "lstm", "--dataset", "ptb", "--device", "cpu", "--no-amp",
        "--num-workers", "0", "--batch-size", "2", "--max-epochs", "1",
        "--iters-per-epoch", "1", "--n-samples", "4"]


def tag(monkeypatch, *extra):
    import train
    monkeypatch.setattr(sys, "argv", ["train.py", *extra])
    return train.default_run_tag(train.parse_args(), 1)


def test_tags_of_other_models_differ(monkeypatch):
    base = ["--dnn", "lstm", "--dataset", "ptb"]
    tags = [tag(monkeypatch, *base, *extra) for extra in (
        [], ["--ffn-mult", "1"], ["--ffn-mult", "4"],
        ["--ffn-mult", "4", "--act8"])]
    assert len(set(tags)) == 4


def test_tag_without_the_block_is_as_before(monkeypatch):
    assert tag(monkeypatch, "--dnn", "lstm", "--dataset", "ptb",
               "--batch-size", "20", "--density", "0.01",
               "--compression", "gtopk") == "lstm-ptb-bs20-rho0.01-gtopk-n1"


@pytest.mark.parametrize("first,then", [([], ["--ffn-mult", "1"]),
                                        (["--ffn-mult", "1"], [])])
def test_resume_leaves_another_models_checkpoint(tmp_path, first, then):
    for extra in (first, [*then, "--resume"]):
        r = subprocess.run(
            [sys.executable, os.path.join(REPO, "train.py"), *ARGS, *extra,
             "--checkpoint-dir", str(tmp_path)],
            cwd=REPO, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
