"""CPU test of what the build counts as newer than the built libraries."""

import os
import shutil

import pytest

from harp_amd import build

FILES = [p for d in (build.CSRC, build.INCLUDE) for p in sorted(d.iterdir()) if p.is_file()]


@pytest.mark.parametrize("source", FILES, ids=lambda p: p.name)
def test_every_source_and_header_counts(source, tmp_path, monkeypatch):
    for name in ("CSRC", "INCLUDE"):
        copy = tmp_path / name
        copy.mkdir()
        for p in getattr(build, name).iterdir():
            if p.is_file():
                shutil.copyfile(p, copy / p.name)
                os.utime(copy / p.name, (1000, 1000))
        monkeypatch.setattr(build, name, copy)
    for name in ("ABI_LIB", "OPS_LIB", "ASYNC_OPS_LIB", "BLOCK_OPS_LIB", "REQUEST_OPS_LIB"):
        lib = tmp_path / name
        lib.touch()
        os.utime(lib, (2000, 2000))
        monkeypatch.setattr(build, name, lib)
    assert not build.sources_newer_than_libs()
    mine = (build.CSRC if source.parent.name == "csrc" else build.INCLUDE) / source.name
    os.utime(mine, (3000, 3000))
    assert build.sources_newer_than_libs()
