"""What ``build_all`` builds, from the commands it issues: the C-ABI libraries on a machine without torch, the autograd
module beside them on one with torch, and the paths of the two C-ABI libraries as its result."""
import os
import sys

import pytest

from cbm4gnn_amd import build


@pytest.fixture
def commands(monkeypatch):
    """The commands that a build would run, none of them run."""
    seen = []
    monkeypatch.setattr(build, "_run", lambda cmd: seen.append(list(cmd)) or "")
    return seen


def outputs(commands):
    return [os.path.basename(c[c.index("-o") + 1]) for c in commands if "-shared" in c]


def test_without_torch(commands, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)         # import torch raises, as where there is none
    hip, host = build.build_all()
    assert (hip, host) == (build.HIP_LIB, build.HOST_LIB)
    assert sorted(outputs(commands)) == ["libcbm_hip.so", "libcbm_host.so"]
    assert not any("torch" in part for c in commands for part in c)


def test_with_torch(commands):
    hip, host = build.build_all()
    assert (hip, host) == (build.HIP_LIB, build.HOST_LIB)
    made = outputs(commands)
    assert sorted(made) == ["cbm_autograd.so", "libcbm_hip.so", "libcbm_host.so"]
    assert made.index("cbm_autograd.so") > made.index("libcbm_hip.so")      # which it is linked to


def test_a_failure_is_not_swallowed(commands, monkeypatch):
    def fail(verbose=False):
        raise RuntimeError("no compiler")
    for name in ("build_hip", "build_host", "build_autograd"):
        with monkeypatch.context() as m:
            m.setattr(build, name, fail)
            with pytest.raises(RuntimeError, match="no compiler"):
                build.build_all()


def test_the_compiler_from_the_path(commands, monkeypatch, tmp_path):
    """``HIPCC=hipcc``, a link to it, or a wrapper somewhere else: the headers are found all the same."""
    (tmp_path / "hipcc").symlink_to(build.HIPCC)
    wrapper = tmp_path / "wrapped" / "hipcc"
    wrapper.parent.mkdir()
    wrapper.write_text("#!/bin/sh\n")
    wrapper.chmod(0o755)
    monkeypatch.setenv("PATH", f"{tmp_path}:{os.environ['PATH']}")
    for name in ("hipcc", str(tmp_path / "hipcc"), str(wrapper)):
        monkeypatch.setattr(build, "HIPCC", name)
        commands.clear()
        build.build_autograd()
        dirs = [part[len("-isystem"):] for part in commands[0] if part.startswith("-isystem")]
        assert any(os.path.exists(os.path.join(d, "hip", "hip_runtime_api.h")) for d in dirs), name
