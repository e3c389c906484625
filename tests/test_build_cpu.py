"""The library is compiled every time that build() is called, not only where a source is newer."""
import subprocess

import __graft_entry__ as entry


def test_build_compiles_also_where_a_library_is_there(monkeypatch):
    calls = []
    monkeypatch.setattr(subprocess, "run", lambda args, **kw: calls.append((args, kw)))
    entry.build()
    assert len(calls) == 1 and calls[0][1] == {"check": True}
    assert calls[0][0][0] == "make" and "-B" in calls[0][0]
