"""What building the library compiles: everything when asked to, and whatever a change of source, header or flag touched."""
import os

import __graft_entry__ as entry
from dssm_amd import _lib
from dssm_amd import build as B


def test_the_entry_compiles_every_source(monkeypatch):
    seen = []
    monkeypatch.setattr(B, "build", lambda force=False, **kw: seen.append(force))
    monkeypatch.setattr(_lib, "load", lambda *a: None)
    monkeypatch.setattr(B.subprocess, "run", lambda *a, **kw: type("R", (), {"returncode": 0})())
    entry.build()
    assert seen == [True]


def test_a_change_of_the_flags_is_a_change_of_every_source(monkeypatch, tmp_path):
    made = []
    monkeypatch.setattr(B, "OBJ", str(tmp_path))
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **k: made.append(cmd) or type("R", (), {"returncode": 0})())
    obj = tmp_path / "embed.o"
    obj.write_text("")
    newest = max(os.path.getmtime(os.path.join(B.CSRC, f)) for f in os.listdir(B.CSRC))
    os.utime(obj, (newest + 10, newest + 10))
    real = B._mtime
    monkeypatch.setattr(B, "_mtime", lambda p: newest + (20 if p == B.__file__ else 0) if not p.endswith(".o") else real(p))
    B._compile("embed.hip", False)
    assert len(made) == 1
    monkeypatch.setattr(B, "_mtime", lambda p: newest if not p.endswith(".o") else real(p))
    B._compile("embed.hip", False)
    assert len(made) == 1
