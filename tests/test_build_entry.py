"""__graft_entry__: build() compiles every time it is called, the tests load what is built (CPU; make itself is not run)."""
import os

import __graft_entry__ as g


def test_every_build_compiles_the_projects_own_sources_again(monkeypatch):
    calls = []
    monkeypatch.setattr(g, "_make", lambda args, cwd: calls.append((args, os.path.relpath(cwd, g.ROOT))))
    g.build()
    own = [(a, d) for a, d in calls if "ref" not in a]
    assert {d for _, d in own} == {"nextpolish_amd/csrc", "oracle", "tests/model"} and all("-B" in a for a, _ in own), calls


def test_what_is_loaded_is_known_to_be_built():
    assert g.is_built()
    assert all(os.path.getsize(os.path.join(g.ROOT, p)) > 0 for p in g.BUILT)
