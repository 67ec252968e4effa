"""The library needs no torch: only its Python binding does."""
import sys

from gateddeltanet_b200 import build


def test_the_library_builds_without_torch(monkeypatch, tmp_path, capsys):
    build.build()
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "_ops_torch.so"))
    monkeypatch.setitem(sys.modules, "torch", None)  # its import fails
    assert build.build() == build.LIB
    assert "no torch" in capsys.readouterr().err and not (tmp_path / "_ops_torch.so").exists()
