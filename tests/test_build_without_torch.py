"""Building the libraries needs no torch; the extension module that does is left out where there is none."""
import os
import subprocess
import sys
import sysconfig

import pytest

from friday_inference_engine_b200.ops import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def libraries_are_there(monkeypatch):
    monkeypatch.setattr(build, "ensure_engine_built", lambda progress=True: "engine")
    monkeypatch.setattr(build, "ensure_built", lambda fams, progress=True: None)


def test_everything_else_is_built_without_torch(libraries_are_there, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)       # (an import of it raises ImportError)
    made = build.build_all()
    assert made[0] == "engine" and len(made) > 10 and build.binding_path() not in made
    assert "left out: torch cannot be imported" in capsys.readouterr().err
    with pytest.raises(build.BuildError, match="torch cannot be imported"):
        build.ensure_binding_built()


def test_everything_else_is_built_without_pythons_headers(libraries_are_there, monkeypatch, tmp_path):
    pytest.importorskip("torch")
    paths = dict(sysconfig.get_paths(), include=str(tmp_path))
    monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: paths)
    assert build.binding_path() not in build.build_all(progress=False)
    with pytest.raises(build.BuildError):
        build.ensure_binding_built()


def test_the_command_for_cpp_users_ends_well_without_torch(tmp_path):
    """The documented command, in a process whose torch cannot be imported; the libraries are taken as built."""
    (tmp_path / "torch.py").write_text("raise ImportError('there is none here')\n")
    code = ("import sys; from friday_inference_engine_b200.ops import build as b; b.ensure_engine_built = lambda progress=True: 'engine'; "
            "b.ensure_built = lambda fams, progress=True: None; b.build_all(); assert 'torch' not in sys.modules")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(tmp_path), ROOT]))
    done = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    assert "left out: torch cannot be imported" in done.stderr
