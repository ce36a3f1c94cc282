"""The build of the library and of the CPython module over it, without a GPU."""
import importlib.util
import os
import sysconfig

import pytest

from baremetalinferenceengine_b200 import build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """Builds go to a scratch folder; the commands that would run are recorded and not run."""
    ran = []
    for name in ("BUILD_DIR", "LIB_PATH", "BINDING_PATH"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    monkeypatch.setattr(build, "_run", lambda cmd: (ran.append(cmd), open(cmd[cmd.index("-o") + 1], "w").close()))
    return ran


@pytest.mark.parametrize("missing", ["torch", "Python's headers"])
def test_without_torch_or_pythons_headers_the_library_is_all(commands, monkeypatch, capsys, tmp_path, missing):
    build.build()
    assert [c for c in commands if c[0] == "g++"]  # with both the module is built
    commands.clear()
    os.remove(build.BINDING_PATH)
    if missing == "torch":
        real = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))
    else:
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: {"include": str(tmp_path)})
    assert build.build(force=True) == build.LIB_PATH and os.path.exists(build.LIB_PATH)
    assert not [c for c in commands if c[0] == "g++"] and not os.path.exists(build.BINDING_PATH)
    assert missing in capsys.readouterr().err


def test_a_module_made_for_another_torch_or_python_is_built_again(commands, monkeypatch, tmp_path):
    built = lambda: len([c for c in commands if c[0] == "g++"])  # noqa: E731
    build.build()
    assert built() == 1
    build.build()
    assert built() == 1
    torch = tmp_path / "torch"
    torch.mkdir()
    (torch / "version.py").write_text("__version__ = '0.0.1'\n")
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: type("Spec", (), {"origin": str(torch / "__init__.py")})
                        if name == "torch" else real(name, *a))
    build.build()
    assert built() == 2
    (torch / "version.py").write_text("__version__ = '0.0.2'\n")  # another one in its place
    build.build()
    assert built() == 3
    monkeypatch.setattr(build.sys.implementation, "cache_tag", "cpython-399")
    build.build()
    assert built() == 4
    build.build()
    assert built() == 4
