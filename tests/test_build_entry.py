"""build() makes the product whatever tests lie in the tree: a program of theirs that cannot be built is reported, and fails its own tests only."""
import pytest

import __graft_entry__ as entry
import oracle
from vtl_amd import build as product
from vtl_amd import capi


@pytest.fixture
def other_tree(tmp_path, monkeypatch):
    """The tests' programs in a tree of its own, with the product taken as built."""
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    monkeypatch.setattr(product, "build_lib", lambda: capi.LIB_PATH)
    monkeypatch.setattr(oracle, "build", lambda force=False: None)
    for folder in ("host_cpp", "host_c"):
        (tmp_path / "tests" / folder).mkdir(parents=True)
    (tmp_path / "tests" / "host_c" / "Makefile").write_text("abi_check:\n\ttouch $@\n")
    return tmp_path / "tests"


def test_a_program_that_the_tests_do_not_know(other_tree, capsys):
    (other_tree / "host_cpp" / "Makefile").write_text("test_host_mirror:\n\ttouch $@\ntest_kv_mirror:\n\ttouch $@\n")
    entry.build()
    out = capsys.readouterr().out
    assert "not built: tests/host_cpp/test_mxfp4_mirror" in out and out.count("not built") == 1 and "built " + capi.LIB_PATH in out
    assert all((other_tree / p).exists() for p in ("host_cpp/test_host_mirror", "host_cpp/test_kv_mirror", "host_c/abi_check"))


def test_a_program_that_does_not_compile(other_tree, capsys):
    """It is not left as it was built from other sources."""
    (other_tree / "host_cpp" / "Makefile").write_text("test_host_mirror:\n\tfalse\ntest_kv_mirror test_mxfp4_mirror:\n\ttouch $@\n")
    (other_tree / "host_cpp" / "test_host_mirror").write_text("")
    entry.build()
    assert capsys.readouterr().out.count("not built") == 1 and not (other_tree / "host_cpp" / "test_host_mirror").exists()


def test_no_tests_at_all(tmp_path, monkeypatch, capsys):
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    monkeypatch.setattr(product, "build_lib", lambda: capi.LIB_PATH)
    monkeypatch.setattr(oracle, "build", lambda force=False: None)
    entry.build()
    assert capsys.readouterr().out.count("not built") == 4
