"""Building a host library again in one process: what the entry point's build()
does when it is called twice, or after an edit."""
import ctypes
import os
import shutil

import pytest

from xrdslam_amd import build_torch_ext as ext

SOURCE = 'extern "C" int xrd_probe(void) { return %s; }\n'


def answer(lib, copy):
    """what the built library says (loaded from a copy: a loaded file's path
    is not looked at again)"""
    shutil.copy(lib, copy)
    return ctypes.CDLL(str(copy)).xrd_probe()


def test_a_forced_build_compiles_every_time(tmp_path, monkeypatch):
    monkeypatch.setattr(ext, 'OUT', str(tmp_path))
    lib, src = str(tmp_path / 'xrd_probe.so'), str(tmp_path / 'probe.cpp')
    for turn, value in enumerate((1, 1, 2)):
        with open(src, 'w') as f:
            f.write(SOURCE % value)
        if os.path.exists(lib):
            os.utime(lib, (1, 1))
        ext._build(lib, src, True, False)
        assert os.path.getmtime(lib) > 1
        assert answer(lib, tmp_path / f'copy{turn}.so') == value


def test_a_build_that_fails_leaves_the_library(tmp_path, monkeypatch):
    monkeypatch.setattr(ext, 'OUT', str(tmp_path))
    lib, src = str(tmp_path / 'xrd_probe2.so'), str(tmp_path / 'probe2.cpp')
    with open(src, 'w') as f:
        f.write(SOURCE % 5)
    ext._build(lib, src, False, False)
    with open(src, 'w') as f:
        f.write(SOURCE % 'no such name')
    with pytest.raises(Exception):
        ext._build(lib, src, True, False)
    assert answer(lib, tmp_path / 'copy.so') == 5


def test_an_unforced_build_keeps_what_is_newer(tmp_path, monkeypatch):
    monkeypatch.setattr(ext, 'OUT', str(tmp_path))
    lib, src = str(tmp_path / 'xrd_probe3.so'), str(tmp_path / 'probe3.cpp')
    with open(src, 'w') as f:
        f.write(SOURCE % 1)
    ext._build(lib, src, False, False)
    at = os.path.getmtime(lib) + 100
    os.utime(lib, (at, at))
    ext._build(lib, src, False, False)
    assert os.path.getmtime(lib) == at
