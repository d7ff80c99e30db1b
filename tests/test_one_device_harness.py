"""Ranks on a device are not started again after the runtime's queue abort, and the case that met it stays skipped."""
import os
import subprocess
import sys

import pytest
from torch.multiprocessing.spawn import ProcessExitedException

from tests import spawn_one_device as sod
from tests.test_harness import _worker

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ranks_on_a_device_are_not_started_again(tmp_path, monkeypatch):
    """(The workers only say what the runtime would: no device is used here.)"""
    monkeypatch.setattr(sod, "RETRIES", [])
    monkeypatch.setattr(sod, "GPU_TEST", True)
    starts = []

    def make_args():
        starts.append(1)
        return str(tmp_path / "a"), True
    with pytest.raises(RuntimeError, match="not started again") as failure:
        sod.spawn_ranks(_worker, make_args, 2)
    assert isinstance(failure.value.__cause__, ProcessExitedException)
    assert len(starts) == 1 and sod.RETRIES == []


def test_the_case_that_aborted_is_skipped():
    case = "test_svgd_resnet50_sharded_one_device"
    p = subprocess.run([sys.executable, "-m", "pytest", os.path.join(ROOT, "tests", "test_dist_fullsize_gpu.py"), "-q", "-rs", "-p", "no:cacheprovider",
                        "-k", f"{case} and alltoall-8"], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=300)
    text = p.stdout.decode()
    assert p.returncode == 0 and "1 skipped" in text and "cause not shown" in text, text[-1500:]
