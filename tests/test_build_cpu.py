"""When the library is built again."""
import os

from aethergraph_b200 import build


def test_stale_after_a_change_of_source_or_torch(tmp_path, monkeypatch):
    src = tmp_path / "csrc"
    src.mkdir()
    for name, path in (("CSRC", src), ("HERE", tmp_path), ("LIB", tmp_path / "lib.so"), ("OPS", tmp_path / "_ops.so"), ("OPS_TORCH", tmp_path / "_ops.torch")):
        monkeypatch.setattr(build, name, str(path))
    (src / "a.cu").write_text("")
    assert build._stale()  # nothing built
    (tmp_path / "lib.so").write_text("")
    (tmp_path / "_ops.so").write_text("")
    assert build._stale()  # nobody knows against which torch
    (tmp_path / "_ops.torch").write_text(build._torch_version())
    assert not build._stale()
    monkeypatch.setattr(build, "_torch_version", lambda: "0.0")
    assert build._stale()
    monkeypatch.undo()
    for name, path in (("CSRC", src), ("HERE", tmp_path), ("LIB", tmp_path / "lib.so"), ("OPS", tmp_path / "_ops.so"), ("OPS_TORCH", tmp_path / "_ops.torch")):
        monkeypatch.setattr(build, name, str(path))
    os.utime(src / "a.cu", (2e9, 2e9))
    assert build._stale()
