"""CPU: what build() takes for up to date, and modules built for another torch."""
import os
import subprocess
import sys

import pytest
import torch

import __graft_entry__ as entry
from pde_amd import _native as native
from conftest import ROOT


def writes(out, text):
    return [sys.executable, "-c", "import sys; open(sys.argv[1], 'w').write(sys.argv[2])", out, text]


def test_objects_go_by_their_command_line_too(tmp_path):
    src, out = tmp_path / "a.hip", str(tmp_path / "a.o")
    src.write_text("x")
    os.utime(src, (1, 1))
    deps = [str(src)]
    assert entry._compile(writes(out, "1"), out, deps, False)
    assert not entry._compile(writes(out, "1"), out, deps, False)              # nothing has changed
    assert entry._compile(writes(out, "1"), out, deps, True)                   # asked for
    assert entry._compile(writes(out, "2"), out, deps, False) and open(out).read() == "2"     # another flag
    os.utime(src)
    os.utime(out, (2, 2))
    assert entry._compile(writes(out, "2"), out, deps, False)                  # a newer source
    os.remove(out + ".cmd")
    assert entry._compile(writes(out, "2"), out, deps, False)                  # made before command lines were kept


def test_a_failed_compile_leaves_nothing_older(tmp_path):
    out = str(tmp_path / "a.o")
    entry._compile(writes(out, "1"), out, [], True)
    with pytest.raises(subprocess.CalledProcessError):
        entry._compile([sys.executable, "-c", "raise SystemExit(1)"], out, [], True)
    assert not os.path.exists(out) and not os.path.exists(out + ".cmd")


def test_build_compiles_every_unit_every_time(monkeypatch):
    ran = []
    monkeypatch.setattr(entry, "_compile", lambda cmd, out, deps, force: ran.append((os.path.basename(out), force)))
    monkeypatch.setattr(entry.subprocess, "check_call", lambda cmd: None)
    entry.build()
    units = [f + ".o" for f in os.listdir(os.path.join(ROOT, "pde_amd", "csrc")) if f.endswith(".hip")]
    assert sorted(ran) == sorted((name, True) for name in units + ["libpinnjet.so", "_tensorlist.so"])


def test_development_builds_have_every_unit():
    """tools/dev_build.sh links what it builds of pinnjet.hip with all the others: load_library takes no library with an entry point missing"""
    script = open(os.path.join(ROOT, "tools", "dev_build.sh")).read()
    named = set(script.split("for unit in ")[1].split(";")[0].split()) | {"pinnjet"}
    assert named == {f[:-4] for f in os.listdir(os.path.join(ROOT, "pde_amd", "csrc")) if f.endswith(".hip")}


@pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "pde_amd", "_tensorlist.so")), reason="_tensorlist.so not built")
def test_a_list_reader_for_another_torch_is_noticed(monkeypatch):
    assert native.load_tensorlist().torch_version == str(torch.__version__)
    monkeypatch.setattr(native, "_list", None)
    monkeypatch.setattr(torch, "__version__", "2.0.0")
    with pytest.raises(native.NativeError, match="another torch"):
        native.load_tensorlist()
