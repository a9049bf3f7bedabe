"""The autograd nodes stand apart: attention, decode, paging and the rest neither load nor build them."""

import pathlib
import subprocess
import sys

import pytest

from mfattn import build

PACKAGE = pathlib.Path(build.__file__).resolve().parents[1]


def _python(code):
    return subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(PACKAGE)!r})\n"
                           + code], capture_output=True, text=True)


def test_what_has_no_nodes_imports_without_them():
    proc = _python(
        "sys.modules['mfattn._nodes'] = None\n"
        "import mfattn\n"
        "from mfattn.kernels import attention, bidirectional, convolution, paged, prologue, rotary\n"
        "for name in ('normalization', 'embedding', 'distillation'):\n"
        "    try:\n"
        "        __import__('mfattn.kernels.' + name)\n"
        "    except ImportError:\n"
        "        continue\n"
        "    raise SystemExit(name + ' has lost its nodes')\n")
    assert proc.returncode == 0, proc.stderr + proc.stdout


def test_missing_nodes_say_how_they_are_built(tmp_path):
    proc = _python(
        "import pathlib\n"
        "there = pathlib.Path.exists\n"
        "pathlib.Path.exists = lambda p: p.name != '_mfnodes.so' and there(p)\n"
        "import mfattn\n"
        "try:\n"
        "    from mfattn.kernels import normalization\n"
        "except ImportError as e:\n"
        "    assert 'build them with' in str(e), e\n"
        "else:\n"
        "    raise SystemExit('imported')\n")
    assert proc.returncode == 0, proc.stderr + proc.stdout


@pytest.mark.parametrize("gone", ["Python.h", "torch"])
def test_the_library_is_built_without_the_nodes_headers(gone, tmp_path, monkeypatch, capsys):
    if gone == "Python.h":
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    else:
        monkeypatch.setitem(sys.modules, "torch", None)
    stale = tmp_path / "_mfnodes.so"
    stale.write_bytes(b"of another torch")
    monkeypatch.setattr(build, "NODES", stale)
    monkeypatch.setattr(build, "OUT", tmp_path / "lib.so")
    monkeypatch.setattr(build, "_compile", lambda src, obj: None)
    done = []

    def run(cmd, **kw):  # the link
        assert "-shared" in cmd and not any("nodes" in c for c in cmd), cmd
        pathlib.Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")
        done.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build(verbose=False) == tmp_path / "lib.so"
    assert len(done) == 1 and (tmp_path / "lib.so").exists()
    assert not stale.exists()
    assert "autograd nodes" in capsys.readouterr().err
