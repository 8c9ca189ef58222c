"""Builds and runs the C++ program that drives the feed-forward operators through the host-side mirror."""
import subprocess

import pytest

from test_hostapi import _build


def test_compiles_without_gpu(tmp_path):
    _build("test_feed_forward", tmp_path)


@pytest.mark.gpu
def test_on_gpu(tmp_path):
    out = subprocess.run([_build("test_feed_forward", tmp_path)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "feed forward ok" in out.stdout
