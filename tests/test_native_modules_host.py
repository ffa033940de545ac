"""The native modules against another torch than they were built with: what does
not need calls.cpp's module keeps working, what does takes the longer way, and
building brings it up to date.  No GPU."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "memboost_b200")

USE = """
import warnings, sys, torch
{first}
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    import memboost_b200 as mb
seen = [str(w.message) for w in seen if "_calls.so" in str(w.message)]
assert len(seen) == {warned}, seen
assert {words!r} in "".join(seen), seen
assert mb.__file__.startswith({where!r}), mb.__file__
for call, words in ((lambda: mb.pack_2bit(torch.zeros(8, dtype=torch.uint8)), "multiple of 16"),
                    (lambda: mb.quantize_int8(torch.zeros(2, 16)), "x must be on CUDA")):
    try:
        call()
    except RuntimeError as e:
        assert words in str(e), e
    else:
        assert False, words
"""


def _run(where, first, warned, words):
    code = USE.format(first=first, warned=warned, words=words, where=where)
    r = subprocess.run([sys.executable, "-c", code], cwd=where, capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=where))
    assert r.returncode == 0, r.stderr


def test_as_built():
    _run(ROOT, "", 0, "")


def test_another_torch():
    _run(ROOT, "torch.__version__ = '1.0.0'", 1, "this is 1.0.0")


@pytest.mark.parametrize("what", ["empty", "not a library"])
def test_a_module_that_does_not_load(tmp_path, what):
    there = tmp_path / "memboost_b200"
    there.mkdir()
    for f in os.listdir(PKG):
        if f.endswith(".py") or f == "libmemboost_b200.so":
            os.symlink(os.path.join(PKG, f), there / f)
    (there / "_calls.so").write_bytes(b"" if what == "empty" else b"another torch's" * 100)
    _run(str(tmp_path), "", 1, "is not used")


def test_no_module_at_all(tmp_path):
    there = tmp_path / "memboost_b200"
    there.mkdir()
    for f in os.listdir(PKG):
        if f.endswith(".py") or f == "libmemboost_b200.so":
            os.symlink(os.path.join(PKG, f), there / f)
    r = subprocess.run([sys.executable, "-c", "import memboost_b200"], cwd=str(tmp_path),
                       capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=str(tmp_path)))
    assert r.returncode != 0 and "build it with" in r.stderr


def _builder():
    spec = importlib.util.spec_from_file_location("mb_build_tested", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_stale_when_torch_or_python_changed(tmp_path):
    import torch
    b = _builder()
    assert b._torch()[1] == str(torch.__version__)
    calls, stamp = tmp_path / "_calls.so", tmp_path / "_calls.for"
    b.CALLS, b.CALLS_FOR = str(calls), str(stamp)
    assert b._calls_stale("a")               # not there
    calls.write_bytes(b"x")                  # newer than its sources
    assert b._calls_stale("a")               # of nothing known
    stamp.write_text("a")
    assert not b._calls_stale("a")
    assert b._calls_stale("b")
    os.utime(calls, (1, 1))
    assert b._calls_stale("a")               # older than its sources
