"""When emmy_ptx/_paged.so is built anew: its sources, its command or torch changed."""

import os
from pathlib import Path

import pytest


@pytest.fixture
def built(monkeypatch):
    """__graft_entry__ with a compiler that only notes that it was called; the real files are put back."""
    import __graft_entry__ as g
    out = g.build_binding()
    stamp, calls = out.with_suffix(".built"), []
    before, text = out.stat(), stamp.read_text()
    monkeypatch.setattr(g, "build_library", lambda: g.PKG / "libemmyb200.so")
    monkeypatch.setattr(g.subprocess, "run", lambda cmd, check: calls.append(cmd))
    yield g, out, stamp, calls
    stamp.write_text(text)
    os.utime(out, ns=(before.st_atime_ns, before.st_mtime_ns))


def test_nothing_is_built_twice(built):
    g, out, stamp, calls = built
    assert g.build_binding() == out and not calls


def test_another_torch_builds_it_anew(built, monkeypatch):
    import torch
    g, out, stamp, calls = built
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "+other")
    g.build_binding()
    assert len(calls) == 1
    g.build_binding()
    assert len(calls) == 1
    monkeypatch.setattr(torch.version, "git_version", "0" * 40)
    g.build_binding()
    assert len(calls) == 2


def test_another_place_of_torch_or_no_record_builds_it_anew(built, monkeypatch):
    import torch
    g, out, stamp, calls = built
    stamp.unlink()
    g.build_binding()
    assert len(calls) == 1 and stamp.exists()
    monkeypatch.setattr(torch, "__file__", str(Path("/elsewhere/torch/__init__.py")))
    g.build_binding()
    assert len(calls) == 2


def test_a_newer_source_builds_it_anew(built):
    g, out, stamp, calls = built
    os.utime(out, (1, 1))
    g.build_binding()
    assert len(calls) == 1


def test_a_build_that_fails_is_not_taken_for_done(built, monkeypatch):
    g, out, stamp, calls = built
    os.utime(out, (1, 1))

    def fails(cmd, check):
        raise g.subprocess.CalledProcessError(1, cmd)
    monkeypatch.setattr(g.subprocess, "run", fails)
    with pytest.raises(g.subprocess.CalledProcessError):
        g.build_binding()
    assert not stamp.exists()
