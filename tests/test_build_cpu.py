"""CPU test of what the build compiles again, with the compilers replaced by a record of their calls."""
import pytest

from fav4_bshd import build as B


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """Names that the compilers were called for; the built files are empty."""
    names = []

    def run(cmd, log, name, verbose):
        names.append(name)
        (tmp_path / name).touch()

    monkeypatch.setattr(B, "BUILD", tmp_path)
    monkeypatch.setattr(B, "_run", run)
    monkeypatch.setattr(B, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    return names


def test_nothing_is_built_twice(compiled):
    B.build()
    assert compiled == [*B.TARGETS, B.BINDING]
    compiled.clear()
    B.build()
    assert compiled == []


def test_another_torch_needs_another_binding(compiled, monkeypatch):
    import importlib.metadata
    B.build()
    compiled.clear()
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0" if name == "torch" else version(name))
    B.build()
    assert compiled == [B.BINDING]
    compiled.clear()
    B.build()
    assert compiled == []


def test_a_torch_without_cuda_gets_no_binding(compiled, monkeypatch, tmp_path, capsys):
    # the libraries of the C ABI are built all the same
    import importlib.util
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "__init__.py").touch()
    cpu_only = importlib.util.spec_from_file_location("torch", tmp_path / "torch" / "__init__.py")
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: cpu_only)
    assert [p.name for p in B.build()] == list(B.TARGETS) == compiled
    assert "not built" in capsys.readouterr().err
