"""What the build decides about the binding to torch, with stand-ins for torch and the compiler."""

from __future__ import annotations

import os
import subprocess
import sys
import textwrap

from conftest import ROOT

# A build whose outputs go to argv[1], with a compiler that only writes its output file; prints one line per call.
RUN = """
import subprocess, sys
from pathlib import Path
from ntilang_b200 import build

out = Path(sys.argv[1])
build.BINDING, build.BUILD = out / "_paged.so", out / "_build"

def run(cmd, **kwargs):
    Path(cmd[cmd.index("-o") + 1]).write_text("compiled")
    print("compiled")
    return subprocess.CompletedProcess(cmd, 0, "", "")

subprocess.run = run
print("result", build.build_binding())
"""


def build(tmp_path, version, cuda):
    torch = tmp_path / "torch"
    (torch / "utils").mkdir(parents=True, exist_ok=True)
    (torch / "version.py").write_text(f"__version__ = {version!r}\ncuda = {cuda!r}\n")
    (torch / "__init__.py").write_text("from .version import __version__\nfrom . import version\n"
                                       "def compiled_with_cxx11_abi(): return True\n")
    (torch / "utils" / "__init__.py").write_text("")
    (torch / "utils" / "cpp_extension.py").write_text("def include_paths(): return []\n")
    env = {**os.environ, "PYTHONPATH": os.pathsep.join([str(tmp_path), str(ROOT)])}
    done = subprocess.run([sys.executable, "-c", textwrap.dedent(RUN), str(tmp_path)], env=env, capture_output=True,
                          text=True)
    assert done.returncode == 0, done.stderr
    *calls, result = done.stdout.split("\n")[:-1]
    return len(calls), result.removeprefix("result ")


def test_no_binding_for_a_torch_without_cuda(tmp_path):
    """There is no libc10_cuda to link: the library builds alone, as where torch is not installed."""
    assert build(tmp_path, "2.9.0+cpu", None) == (0, "None")
    assert build(tmp_path, "2.9.0+cu128", "12.8") == (1, str(tmp_path / "_paged.so"))


def test_the_binding_follows_torch(tmp_path):
    """Built for one torch and interpreter, it is built again for another, without --force."""
    built = str(tmp_path / "_paged.so")
    assert build(tmp_path, "2.9.0+cu128", "12.8") == (1, built)
    assert build(tmp_path, "2.9.0+cu128", "12.8") == (0, built)
    assert build(tmp_path, "2.10.0+cu128", "12.8") == (1, built)
    assert build(tmp_path, "2.10.0+cu128", "12.8") == (0, built)
    (tmp_path / "_build" / "_paged.torch").write_text("of another interpreter")
    assert build(tmp_path, "2.10.0+cu128", "12.8") == (1, built)
