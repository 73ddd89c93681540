"""CPU tier: the tests of tests/test_gpu_blocks.py (same bodies, shapes and bounds) on the CPU wavefront emulator of tests/emu."""
import os
import shutil

import pytest

import emu_util

pytestmark = pytest.mark.skipif(not (shutil.which("clang++") or os.path.exists("/opt/rocm/lib/llvm/bin/clang++")),
                                reason="the emulator build needs a host clang++ (vector extensions, __bf16)")

_G = emu_util.load_copy("test_gpu_blocks", DEV="cpu")


@pytest.fixture(autouse=True)
def _emulated_library(monkeypatch):
    from refil_amd import blocks
    monkeypatch.setattr(blocks, "_require_gpu", lambda t, who: None)        # (the guard itself: tests/test_blocks_refusals.py)
    with emu_util.active():
        yield


for _k, _v in list(vars(_G).items()):
    if _k.startswith("test_"):
        globals()[_k] = _v
del _k, _v
