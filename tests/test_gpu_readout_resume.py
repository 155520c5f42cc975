"""run_atlas --readout stopped dead right behind a checkpoint, then resumed: every batch has its answers."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

# The process ends where the second checkpoint has reached the disk; the loop's own writing of answers is held up, as by
# a slow disk, so that only what a checkpoint waits for is there.
STOPPED = """
import os, sys
from proteus_b200 import run_atlas as R
drain, save = R.ReadoutWriter.drain, R.CheckpointWriter.save
R.ReadoutWriter.drain = lambda self, keep: drain(self, keep) if keep == 0 else None
def stop(self, obj, path, after=None):
    save(self, obj, path, after)
    self.wait()
    if obj["next_batch"] >= 4:
        os._exit(7)
R.CheckpointWriter.save = stop
R.main(sys.argv[1:])
"""


def test_every_batch_has_its_answers_after_a_stop_behind_a_checkpoint(tmp_path):
    args = ["--model", "8M", "--data", "synthetic:60:3", "--device", "cuda:0", "--dtype", "fp32", "--tokens-per-batch", "4096",
            "--pilot-tokens", "4096", "--K", "8", "--Kr", "4", "--ckpt-every", "2", "--attn", "rows", "--readout", "2"]

    def run(out, *more, code=None):
        cmd = [sys.executable, *(["-c", code] if code else ["-m", "proteus_b200.run_atlas"]), *args, "--out", str(out), *more]
        r = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=600)
        assert r.returncode == (7 if code else 0), r.stdout[-2000:] + r.stderr[-3000:]

    run(tmp_path / "whole")
    run(tmp_path / "cut", code=STOPPED)
    assert (tmp_path / "cut" / "ckpt" / "ckpt_4.pt").exists()
    run(tmp_path / "cut", "--resume")
    want = {p.name for p in (tmp_path / "whole" / "readout").glob("*.pt")}
    assert len(want) > 4 and {p.name for p in (tmp_path / "cut" / "readout").glob("*.pt")} == want
    for name in want:
        a, b = torch.load(tmp_path / "whole" / "readout" / name), torch.load(tmp_path / "cut" / "readout" / name)
        assert all(torch.equal(a[k], b[k]) for k in a)
