"""What the build needs: the library a HIP compiler alone, the torch binding torch and a host compiler."""
import importlib.util
import os
import subprocess
import sys

import pytest

from spiky_amd import build

FILE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spiky_amd", "build.py")


@pytest.fixture
def made(monkeypatch):
    """The files that compilers would have written, in their order."""
    made = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: made.append(os.path.basename(cmd[cmd.index("-o") + 1])))
    monkeypatch.setattr(os, "replace", lambda a, b: made.append(os.path.basename(b)))
    monkeypatch.setattr(build, "_hipcc", lambda: "hipcc")
    return made


def test_both_are_built_where_torch_is(made):
    assert build.build() == build.LIB and made.index("libspiky_lut.so") < made.index("_lm_torch.so") == len(made) - 1


def test_the_library_is_built_without_torch(made, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build() == build.LIB
    assert made[-1] == "libspiky_lut.so" and "without the torch binding" in capsys.readouterr().err
    with pytest.raises(RuntimeError, match="torch"):
        build.build_binding()


def test_the_library_alone_is_built_on_request(made):
    assert build.build(binding=False) == build.LIB and made[-1] == "libspiky_lut.so"


def test_the_file_runs_without_the_package():
    """As a host without torch runs it."""
    code = f"import runpy, sys; sys.modules['torch'] = None; runpy.run_path({FILE!r}); assert 'spiky_amd' not in sys.modules"
    subprocess.run([sys.executable, "-c", code], check=True)
