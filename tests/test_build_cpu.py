"""The entry point that says whether the sources build compiles them, whatever is built already."""
import __graft_entry__
from tf_repos_amd import build


def test_build_compiles_what_is_built(monkeypatch, tmp_path):
    calls = []
    monkeypatch.setattr(build, "build_library", lambda force=False, **kw: calls.append((force, kw.get("variant", ""))) or __file__)
    __graft_entry__.build()
    assert calls == [(True, ""), (True, "ieee")]
