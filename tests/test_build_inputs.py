"""The library is rebuilt when any file changes that its sources include."""

from __future__ import annotations

import os
import re

from vflash_b200 import build


def test_every_included_file_is_an_input():
    files = set(build._sources() + build._headers())
    for path in sorted(files):
        for name in re.findall(r'#include "([^"]+)"', path.read_text()):
            assert build.CSRC / name in files or build.INCLUDE / name in files, f"{path.name} includes {name}"


def test_a_changed_header_makes_the_library_stale(tmp_path, monkeypatch):
    """attention_plan.h as an example of the headers beside the sources."""
    header = tmp_path / "csrc" / "attention_plan.h"
    header.parent.mkdir()
    header.write_text("")
    library = tmp_path / "library.so"
    library.write_text("")
    monkeypatch.setattr(build, "CSRC", header.parent)
    monkeypatch.setattr(build, "INCLUDE", tmp_path)
    os.utime(library, (1000, 1000))
    os.utime(header, (2000, 2000))
    assert build._stale(library, build._headers())
