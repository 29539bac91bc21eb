"""The build entry point compiles the product; test programs are built beside it where their files are there."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def entry(tmp_path, monkeypatch):
    """__graft_entry__ over an empty tree, with the product's own builds left out (they are not what is tested)."""
    spec = importlib.util.spec_from_file_location("graft_entry_under_test", os.path.join(ROOT, "__graft_entry__.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    import oracle
    from brotensor_b200 import build
    done = []
    monkeypatch.setattr(build, "build_all", lambda *a, **k: done.append("product"))
    monkeypatch.setattr(oracle, "build", lambda *a, **k: None)
    monkeypatch.setattr(oracle, "build_gpu", lambda *a, **k: None)
    monkeypatch.setattr(mod, "ROOT", str(tmp_path))
    mod.done, mod.tree = done, tmp_path
    return mod


def _builder(tree, name, body):
    (tree / "tests" / "cpp").mkdir(parents=True, exist_ok=True)
    (tree / "tests" / "cpp" / f"build_{name}.py").write_text(body)


def test_builds_without_any_tests(entry):
    entry.build()
    assert entry.done == ["product"]


def test_a_test_program_whose_source_or_builder_is_missing_is_left_out(entry):
    note = "import pathlib\ndef build():\n    pathlib.Path(__file__).with_suffix('.ran').touch()\n"
    for name in ("host_tests", "expert_tests"):
        _builder(entry.tree, name, note)
    cpp = entry.tree / "tests" / "cpp"
    (cpp / "host_tests.cpp").touch()
    (cpp / "other_tests.cpp").touch()  # no builder
    entry.build()
    assert (cpp / "build_host_tests.ran").exists() and not (cpp / "build_expert_tests.ran").exists()


def test_a_test_program_that_does_not_compile_is_an_error(entry):
    _builder(entry.tree, "host_tests", "def build():\n    raise RuntimeError('does not compile')\n")
    (entry.tree / "tests" / "cpp" / "host_tests.cpp").touch()
    with pytest.raises(RuntimeError, match="does not compile"):
        entry.build()
