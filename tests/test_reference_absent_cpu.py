"""CPU: what becomes of the tests and bench legs that run the reference's own
code where its libraries are not built."""
import ast

import pytest

import __graft_entry__ as entry
import bench
import conftest


@pytest.fixture
def roots(tmp_path, monkeypatch):
    """A tree without libraries, for the tests and the bench; returns its folder for them."""
    monkeypatch.setattr(conftest, "ROOT", tmp_path)
    monkeypatch.setattr(bench, "ROOT", tmp_path)
    libs = tmp_path / "oracle" / "_ref"
    libs.mkdir(parents=True)
    return libs


def test_absent_tree_skips_and_says_so(roots, monkeypatch):
    monkeypatch.setattr(entry, "reference_tree", lambda: None)
    assert "source tree is absent" in conftest.reference_absent()
    assert "source tree is absent" in bench.reference_missing()


def test_tree_without_libraries_is_not_skipped(roots, monkeypatch, tmp_path):
    monkeypatch.setattr(entry, "reference_tree", lambda: tmp_path)
    assert conftest.reference_absent() is None
    assert "make -C oracle" in bench.reference_missing()


def test_built_libraries_run(roots, monkeypatch):
    monkeypatch.setattr(entry, "reference_tree", lambda: None)
    for n in ("libinfengine_ref.so", "libref_model_ref.so"):
        (roots / n).touch()
    assert conftest.reference_absent() is None and bench.reference_missing() is None


def test_the_named_tests_are_those_that_load_the_libraries():
    """In each test file, a test is named exactly if it, or a helper it calls,
    loads a library of oracle/_ref."""
    for path in sorted(conftest.Path(__file__).parent.glob("test_gpu_*.py")):
        tree = ast.parse(path.read_text())
        functions = {f.name: f for f in tree.body if isinstance(f, ast.FunctionDef)}

        def loads(f, seen=()):
            calls = {n.func.id for n in ast.walk(f) if isinstance(n, ast.Call) and isinstance(n.func, ast.Name)}
            if "ref" in calls:
                return True
            names = {n.id for n in ast.walk(f) if isinstance(n, ast.Name)}
            if "REF" in names:
                return True
            return any(c in functions and c not in seen and loads(functions[c], (*seen, c)) for c in calls)

        for name, f in functions.items():
            if name.startswith("test_"):
                assert conftest.needs_reference(path, name) == loads(f), (path.name, name)
