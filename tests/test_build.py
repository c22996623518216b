"""When the library is built anew."""
import os

import pytest

from imagesegmentation_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A library one second newer than build.py, its sources, a header and the ABI header older than both."""
    csrc = tmp_path / "package" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    files = {"source": csrc / "a.hip", "header": csrc / "a.h", "abi": tmp_path / "include" / "isg.h",
             "library": csrc.parent / "libisg.so"}
    now = os.path.getmtime(build.__file__)
    for name, path in files.items():
        path.write_text("")
        os.utime(path, (now, now + 1 if name == "library" else now - 100))
    monkeypatch.setattr(build, "_HERE", str(csrc.parent))
    monkeypatch.setattr(build, "CSRC", str(csrc))
    monkeypatch.setattr(build, "OUT", str(files["library"]))
    return files, now


def test_a_library_newer_than_everything_stays(tree):
    assert not build._stale()


@pytest.mark.parametrize("name", ["source", "header", "abi"])
def test_a_change_of_a_source_or_header_builds_it_anew(tree, name):
    files, now = tree
    os.utime(files[name], (now, now + 2))
    assert build._stale()


def test_a_change_of_the_flags_builds_it_anew(tree):
    files, now = tree
    os.utime(files["library"], (now, now - 1))  # older than build.py, newer than the sources
    assert build._stale()


def test_a_missing_library_is_built(tree):
    files, _ = tree
    files["library"].unlink()
    assert build._stale()
