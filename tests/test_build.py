"""CPU tier: the product build (__graft_entry__.build, refil_amd/build.py) on a copy of the sources, with a stand-in for the compiler: it needs
nothing under tests/, runs no more compilers at a time than it may, and names a compiler that fails."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "refil_amd", "librefil_hip.so")

# A compiler that takes a moment and notes how many run beside it; linking hands out the library that is there already.
HIPCC = f"""#!{sys.executable}
import os, shutil, sys, time
out, box = sys.argv[sys.argv.index("-o") + 1], os.environ["HIPCC_BOX"]
if "-c" in sys.argv:
    me = os.path.join(box, f"run.{{os.getpid()}}")
    open(me, "w").close()
    time.sleep(0.1)
    n = sum(f.startswith("run.") for f in os.listdir(box))
    open(os.path.join(box, f"seen.{{n}}"), "w").close()
    os.remove(me)
    src = os.path.basename(sys.argv[sys.argv.index("-c") + 1])
    if src == os.environ.get("HIPCC_FAILS"):
        print("this source has a mistake")
        sys.exit(1)
    open(out, "w").close()
else:
    shutil.copyfile({LIB!r}, out)
"""


@pytest.fixture
def tree(tmp_path):
    """the product's sources without tests/, and a function that builds them"""
    for d in ("refil_amd", "include"):
        shutil.copytree(os.path.join(ROOT, d), tmp_path / d, ignore=shutil.ignore_patterns("build", "*.so", "*.so.*", "__pycache__"))
    shutil.copy(os.path.join(ROOT, "__graft_entry__.py"), tmp_path)
    box = tmp_path / "box"
    box.mkdir()
    (box / "hipcc").write_text(HIPCC)
    (box / "hipcc").chmod(0o755)

    def run(code="import __graft_entry__ as g; g.build()", **env):
        e = {k: v for k, v in os.environ.items() if k not in ("MAX_JOBS", "REFIL_EXTRA_FLAGS", "REFIL_SKIP_EMU_BUILD", "PYTHONPATH")}
        e.update(HIPCC=str(box / "hipcc"), HIPCC_BOX=str(box), PYTHONDONTWRITEBYTECODE="1", **env)
        return subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env=e, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    run.root, run.box = tmp_path, box
    return run


@pytest.mark.skipif(not os.path.exists(LIB), reason="librefil_hip.so is not built")
@pytest.mark.parametrize("emulator", [None, "raise ValueError('an instruction the emulator does not know')\n", "def build():\n    raise RuntimeError('no host compiler')\n"])
def test_the_product_build_does_not_depend_on_the_tests(tree, emulator):
    if emulator is not None:
        (tree.root / "tests" / "emu").mkdir(parents=True)
        (tree.root / "tests" / "emu" / "build_emu.py").write_text(emulator)
    r = tree()
    assert r.returncode == 0, r.stderr
    assert (tree.root / "refil_amd" / "librefil_hip.so").exists()
    assert ("did not build" in r.stderr) == (emulator is not None and os.path.exists("/opt/rocm/lib/llvm/bin/clang++"))


def _most(box):
    return max(int(f.name.split(".")[1]) for f in box.iterdir() if f.name.startswith("seen."))


def test_compilers_at_a_time(tree):
    code = "from refil_amd import build; build.build(force=True)"
    r = tree(code, MAX_JOBS="2")
    assert r.returncode == 0, r.stderr
    assert _most(tree.box) <= 2
    r = tree(code)
    assert r.returncode == 0 and _most(tree.box) <= len(os.sched_getaffinity(0))


def test_a_failing_compiler_is_named(tree):
    code = "from refil_amd import build; build.build(force=True)"
    r = tree(code, HIPCC_FAILS="gru.hip", MAX_JOBS="1")
    assert r.returncode != 0 and "hipcc failed on gru.hip" in r.stderr and "this source has a mistake" in r.stderr
    assert not (tree.root / "refil_amd" / "build" / "gru.o").exists() and not (tree.root / "refil_amd" / "librefil_hip.so").exists()
    assert tree("from refil_amd import build; build.build()").returncode == 0
