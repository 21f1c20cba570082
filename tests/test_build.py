"""What the build does, without a compiler's run: which steps it takes, and when the binding counts as stale."""

import subprocess
import sys

import pytest

from exp3_b200 import _capi, build, paged


@pytest.fixture
def steps(monkeypatch):
    taken = []
    monkeypatch.setattr(build, "_build_library", lambda: taken.append("library"))
    monkeypatch.setattr(build, "_build_binding", lambda: taken.append("binding"))
    return taken


def test_the_library_needs_no_torch(steps, monkeypatch, capsys):
    build.build(force=True, library_only=True)
    assert steps == ["library"]
    monkeypatch.setattr(build.importlib.metadata, "version", _not_installed)
    build.build(force=True, verbose=True)
    assert steps == ["library", "library"] and "torch is not installed" in capsys.readouterr().out


def _not_installed(name):
    raise build.importlib.metadata.PackageNotFoundError(name)


def test_the_build_itself_does_not_import_torch():
    code = "import sys; sys.modules['torch'] = None; from exp3_b200 import build; print(build._stale())"
    assert subprocess.run([sys.executable, "-c", code], cwd=build.ROOT, capture_output=True, text=True).returncode == 0


def test_a_binding_that_does_not_build_leaves_the_library_built(steps, monkeypatch, capsys):
    def fails():
        raise RuntimeError("no compiler")

    monkeypatch.setattr(build, "_build_binding", fails)
    with pytest.raises(RuntimeError, match="no compiler"):
        build.build(force=True, verbose=True)
    assert steps == ["library"] and "libfpx.so" in capsys.readouterr().out


def test_a_binding_for_another_torch_is_stale(tmp_path, monkeypatch):
    binding = tmp_path / "_paged.so"
    binding.write_bytes(b"")
    monkeypatch.setattr(build, "BUILD", tmp_path)
    monkeypatch.setattr(build, "BINDING", binding)
    assert build._binding_stale()  # nothing says what it was built for
    (tmp_path / "paged_binding.txt").write_text(build._binding_for())
    assert not build._binding_stale()
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "9.9.9")
    assert build._binding_stale()


def test_a_binding_for_another_torch_is_not_used(monkeypatch):
    paged._binding()
    paged._binding.cache_clear()
    try:
        monkeypatch.setattr(paged.torch, "__version__", "9.9.9")
        with pytest.raises(_capi.FpxError, match="9.9.9"):
            paged._binding()
    finally:
        monkeypatch.undo()
        assert paged._binding().TORCH_VERSION == paged.torch.__version__
