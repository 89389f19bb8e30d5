"""When the Python binding of the paged-cache operators is built; no compiler is run here."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("t4a_build", os.path.join(ROOT, "t4a-cuda-kernels_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(module, "BUILD", str(tmp_path / "objects"))
    os.makedirs(module.LIBDIR)
    os.makedirs(module.BUILD)
    module.commands = []

    def run(command):
        module.commands.append(command)
        open(os.path.join(module.LIBDIR, "_cache_torch.so"), "w").close()

    monkeypatch.setattr(module, "run", run)
    return module


def torch_at(monkeypatch, module, directory, version):
    os.makedirs(directory, exist_ok=True)
    for name, text in (("__init__.py", ""), ("version.py", f"__version__ = '{version}'\n")):
        with open(os.path.join(directory, name), "w") as f:
            f.write(text)
    spec = importlib.util.spec_from_file_location("torch", os.path.join(directory, "__init__.py"))
    monkeypatch.setattr(module.importlib.util, "find_spec", lambda name: spec)


def test_without_torch_the_library_is_built_alone(monkeypatch, build, capsys):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert build.build_binding("libt4a_b200.so") is None and build.commands == []
    assert "torch is not installed" in capsys.readouterr().err


def test_another_torch_is_built_for_anew(monkeypatch, build, tmp_path):
    torch_at(monkeypatch, build, str(tmp_path / "a" / "torch"), "2.11.0")
    out = build.build_binding("libt4a_b200.so")
    assert out == os.path.join(build.LIBDIR, "_cache_torch.so") and len(build.commands) == 1
    assert str(tmp_path / "a" / "torch" / "lib") in build.commands[0]
    build.build_binding("libt4a_b200.so")
    assert len(build.commands) == 1  # nothing changed
    torch_at(monkeypatch, build, str(tmp_path / "a" / "torch"), "2.12.0")
    build.build_binding("libt4a_b200.so")
    assert len(build.commands) == 2
    torch_at(monkeypatch, build, str(tmp_path / "b" / "torch"), "2.12.0")
    build.build_binding("libt4a_b200.so")
    assert len(build.commands) == 3 and str(tmp_path / "b" / "torch" / "lib") in build.commands[2]
