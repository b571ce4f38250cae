"""The default name of a run, under which its checkpoints lie, tells runs of
other models apart."""
import sys

import pytest
from torch import nn

from gtopkssgd_amd.checkpoint import latest_checkpoint, save_checkpoint


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
def test_resume_leaves_another_models_checkpoint(tmp_path, monkeypatch, first,
                                                 then):
    base = ["--dnn", "lstm", "--dataset", "ptb"]
    tags = [tag(monkeypatch, *base, *extra) for extra in (first, then)]
    path = save_checkpoint(str(tmp_path), tags[0], 0, nn.Linear(2, 2))
    assert latest_checkpoint(str(tmp_path), tags[0]) == path
    assert latest_checkpoint(str(tmp_path), tags[1]) is None
