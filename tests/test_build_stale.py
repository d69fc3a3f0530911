"""CPU: when the serving extension is built again."""
import sys

from computd_b200 import build


def test_the_extension_belongs_to_one_torch_and_python(tmp_path, monkeypatch):
    """Another torch or Python makes it stale, whatever the files' times say: importing it would fail
    with the advice to build it."""
    import torch

    so = tmp_path / "_serving.so"
    so.write_bytes(b"x")
    monkeypatch.setattr(build, "HOST_PATH", so)
    monkeypatch.setattr(build, "BUILD_DIR", tmp_path)
    monkeypatch.setattr(build, "_stale", lambda obj, deps: not obj.exists())
    assert build._host_stale()  # no word of what it was built for
    build._note_host()
    assert not build._host_stale()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9.9+cu999")
        assert build._host_stale()
    with monkeypatch.context() as m:
        m.setattr(sys, "version", "9.9 (another one)")
        assert build._host_stale()
    assert not build._host_stale()
    so.unlink()
    assert build._host_stale()
