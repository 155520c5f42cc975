"""A checkpoint is never on disk before the answers of the batches that a resumed run would not repeat."""
from __future__ import annotations

import pytest
import torch

from proteus_b200 import run_atlas as R


class _Done:
    """An event whose copies are under way until they are waited for."""

    def __init__(self):
        self.waited = False

    def query(self):
        return self.waited

    def synchronize(self):
        self.waited = True


def _pending(answers, *batches):
    for b in batches:
        answers._pending.append((b, {"tok": torch.arange(b + 1)}, _Done()))


def test_answers_are_written_before_the_checkpoint(tmp_path, monkeypatch):
    order = []
    save = R.atomic_save
    monkeypatch.setattr(R, "atomic_save", lambda obj, path: (save(obj, path), order.append(path.name)))
    answers = R.ReadoutWriter(tmp_path / "readout")
    ck = tmp_path / "ckpt"
    ck.mkdir()
    w = R.CheckpointWriter(ck, keep=2, answers=answers)
    _pending(answers, 0, 1)
    answers.drain(2)  # the loop's own: leaves the newest two, whose copies are not done
    w.save({"atlas": {}, "next_batch": 2, "args_key": "k"}, ck / "ckpt_2.pt")
    w.wait()
    assert order == ["0.pt", "1.pt", "ckpt_2.pt"]
    _pending(answers, 2)
    w.save({"atlas": {}, "next_batch": 3, "args_key": "k"}, ck / "ckpt_3.pt")
    w.wait()
    assert order[3:] == ["2.pt", "ckpt_3.pt"] and not answers._pending


def test_answers_that_cannot_be_written_leave_no_checkpoint(tmp_path):
    """The run ends with the error, and a resumed one starts from the checkpoint before."""
    answers = R.ReadoutWriter(tmp_path / "readout")
    w = R.CheckpointWriter(tmp_path, keep=2, answers=answers)
    answers.d = tmp_path / "gone"
    _pending(answers, 0)
    with pytest.raises((FileNotFoundError, RuntimeError), match="does not exist|No such file"):
        w.save({"atlas": {}, "next_batch": 1, "args_key": "k"}, tmp_path / "ckpt_1.pt")
    w.wait()
    assert not list(tmp_path.glob("ckpt_*"))
