"""What the build counts as out of date (no GPU, no compiler)."""

import re

import pytest

from torchwarp_b200 import build


def test_every_included_header_is_a_dependency():
    headers = {p.resolve() for p in build._headers()}
    sources = list(build.CSRC.glob("*.cu")) + list(headers)
    assert sources
    for src in sources:
        for name in re.findall(r'^#include "([^"]+)"', src.read_text(), re.M):
            assert (src.parent / name).resolve() in headers, (src.name, name)


@pytest.fixture
def commands(tmp_path, monkeypatch):
    """A host build whose compiler is a note of its command."""
    ran = []

    class Result:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **_):
        ran.append(cmd)
        (tmp_path / "host.so").write_text("")
        return Result

    monkeypatch.setattr(build, "HOST_LIB", tmp_path / "host.so")
    monkeypatch.setattr(build, "HOST_STAMP", tmp_path / "host.stamp")
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(build.subprocess, "run", run)
    return ran


def test_host_extension_follows_torch(commands, monkeypatch):
    import torch
    assert build._build_host(False) is None and len(commands) == 1
    assert build._build_host(False) is None and len(commands) == 1
    monkeypatch.setattr(torch, "__version__", "0.0")
    assert build._build_host(False) is None and len(commands) == 2
    assert build._build_host(True) is None and len(commands) == 3


def test_failed_host_build_is_tried_again(commands, monkeypatch):
    assert build._build_host(False) is None

    class Failed:
        returncode, stdout, stderr = 1, "", "no"

    with monkeypatch.context() as m:
        m.setattr(build.subprocess, "run", lambda *_, **__: Failed)
        assert "no" in build._build_host(True)
    assert build._build_host(False) is None and len(commands) == 2
