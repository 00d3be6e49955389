"""The build script's decisions, without compiling."""
import pytest

from laya_cuda import build as builder


@pytest.fixture
def compiled(monkeypatch, tmp_path):
    """The targets that a build would have made; the real ones are not touched."""
    made = []
    monkeypatch.setattr(builder, "TARGET", tmp_path / "liblaya_b200.so")
    monkeypatch.setattr(builder, "EXTENSION", tmp_path / builder.EXTENSION.name)
    monkeypatch.setattr(builder, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(builder.subprocess, "run", lambda cmd, check: open(made.append(cmd) or cmd[cmd.index("-o") + 1], "w").close())
    return made


def test_builds_what_is_missing_or_older_than_its_sources(compiled):
    assert builder.build() == builder.TARGET
    assert [cmd[0].rsplit("/")[-1] for cmd in compiled] == ["nvcc", "g++"]
    assert builder.TARGET.exists() and builder.EXTENSION.exists()
    builder.build()
    assert len(compiled) == 2
    builder.build(force=True)
    assert len(compiled) == 4


def test_without_pythons_headers_the_library_is_built_and_the_extension_left_out(compiled, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(builder.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    builder.EXTENSION.touch()
    assert builder.build(force=True) == builder.TARGET
    assert [cmd[0] for cmd in compiled] == ["nvcc"]
    assert builder.TARGET.exists() and not builder.EXTENSION.exists()
    assert "laya_cuda.mx8 not available" in capsys.readouterr().err


def test_the_extension_is_named_for_this_pythons_abi(compiled):
    import importlib.machinery
    suffix = importlib.machinery.EXTENSION_SUFFIXES[0]
    assert builder.EXTENSION.name == "_mx8" + suffix and "cpython" in suffix
    plain = builder.EXTENSION.with_name("_mx8.so")
    plain.touch()
    builder.build()
    assert builder.EXTENSION.exists() and not plain.exists()
