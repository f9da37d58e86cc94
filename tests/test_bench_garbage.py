"""bench.py leaves no long garbage collection to fall among its timed steps."""

import os
import subprocess
import sys

from conftest import ROOT


def test_what_is_loaded_is_left_out_of_later_collections():
    code = """
import gc
import inspect
import torch
import mrsa
import bench
assert "set_garbage_aside()" in inspect.getsource(bench.main)
before = len(gc.get_objects())
bench.set_garbage_aside()
assert gc.get_freeze_count() > before / 2, (before, gc.get_freeze_count())
assert len(gc.get_objects()) < before / 20, (before, len(gc.get_objects()))
"""
    package = next(p for p in os.listdir(ROOT) if p.startswith("mask-routed"))
    path = os.pathsep.join((ROOT, os.path.join(ROOT, package)))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300,
                   env={**os.environ, "PYTHONPATH": path})
