"""build.py with and without the IQ2_XXS tables, by a stand-in compiler (an object holds its source's name, a library its
objects' names), and b200q.py's loading of a library that lacks operators."""
import importlib.util
import os
import subprocess
import time

import pytest

import b200q

PKG = os.path.dirname(b200q.__file__)
NVCC = """#!/usr/bin/env python3
import os, sys
a = sys.argv[1:]
out = a[a.index("-o") + 1]
if "-c" in a:
    open(out, "w").write(os.path.basename(a[a.index("-c") + 1]))
else:
    open(out, "w").write(" ".join(sorted(open(x).read() for x in a if x.endswith(".o"))))
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """a package of three sources, two of them table-free -> its build module"""
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    pkg, inc = tmp_path / "pkg", tmp_path / "include"
    (pkg / "csrc").mkdir(parents=True)
    inc.mkdir()
    for f in ("core.cu", "iq2.cu", "kv.cu", "common.cuh"):
        (pkg / "csrc" / f).write_text("")
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(NVCC)
    nvcc.chmod(0o755)
    for name, value in dict(HERE=pkg, ROOT=tmp_path, CSRC=pkg / "csrc", OUT=pkg / "libb200q.so", PART=pkg / m.os.path.basename(m.PART),
                            OBJ=pkg / "_build", TABLES=tmp_path / "tables.inc", NVCC=nvcc).items():
        monkeypatch.setattr(m, name, str(value))
    (tmp_path / "tables.inc").write_text("")
    return m


def touch(path):
    """newer than all that was written so far"""
    t = time.time() + 5
    while os.path.exists(path) and os.path.getmtime(path) >= t:
        t += 5
    os.utime(path, (t, t))


def holds(path):
    return open(path).read().split()


ALL, FREE = ["core.cu", "iq2.cu", "kv.cu"], ["core.cu", "kv.cu"]


def test_whole_library(tree):
    assert tree.build() == tree.OUT and holds(tree.OUT) == ALL and not os.path.exists(tree.PART)


def test_without_tables_a_fresh_prebuilt_library_is_used_and_a_stale_one_is_an_error(tree):
    tree.build()
    os.remove(tree.TABLES)
    assert tree.build() == tree.OUT and holds(tree.OUT) == ALL
    open(os.path.join(tree.CSRC, "kv.cu"), "a").write("// changed")
    with pytest.raises(RuntimeError, match="not of these sources"):
        tree.build()
    assert holds(tree.OUT) == ALL and not os.path.exists(tree.PART)   # neither replaced nor joined by less


def test_a_prebuilt_library_goes_by_the_sources_contents_else_by_their_times(tree):
    tree.build()
    os.remove(tree.TABLES)
    touch(os.path.join(tree.CSRC, "kv.cu"))   # as a copy of the tree does
    assert tree.build() == tree.OUT
    os.remove(tree.OUT + ".sources")
    with pytest.raises(RuntimeError, match="not of these sources"):
        tree.build()
    touch(tree.OUT)
    assert tree.build() == tree.OUT


def test_without_tables_and_library_the_part_goes_by_another_name_and_says_so(tree, capfd):
    os.remove(tree.TABLES)
    for _ in range(2):
        assert tree.build() == tree.PART and holds(tree.PART) == FREE and not os.path.exists(tree.OUT)
        assert "lacks the operators" in capfd.readouterr().err


def test_the_whole_library_comes_back_with_the_tables(tree):
    tables = open(tree.TABLES).read()
    tree.build()
    os.remove(tree.TABLES)
    os.remove(tree.OUT)
    touch(os.path.join(tree.CSRC, "kv.cu"))
    assert tree.build() == tree.PART
    open(tree.TABLES, "w").write(tables)
    assert tree.build() == tree.OUT and holds(tree.OUT) == ALL


def test_a_library_of_other_objects_is_linked_again(tree):
    """as one that lost a source has, or one left by a build that linked fewer under the same name"""
    tree.build()
    open(tree.OUT, "w").write("core.cu kv.cu")
    os.remove(tree.OUT + ".sources")
    touch(tree.OUT)
    assert tree.build() == tree.OUT and holds(tree.OUT) == ALL
    os.remove(os.path.join(tree.CSRC, "kv.cu"))
    touch(tree.OUT)
    tree.build()
    assert holds(tree.OUT) == ["core.cu", "iq2.cu"]


def few(tmp_path, name):
    """a library with three of the C ABI's functions"""
    src, out = tmp_path / "few.c", tmp_path / name
    src.write_text('int b200q_abi(void) { return 1; }\nint b200q_last_cuda_error(void) { return 0; }\n'
                   'const char* b200q_strerror(int s) { return "?"; }\n')
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(out)], check=True)
    return str(out)


def test_calling_an_operator_that_the_part_lacks_raises(tmp_path, monkeypatch):
    monkeypatch.setattr(b200q, "LIB_PATH", few(tmp_path, b200q.PART))
    monkeypatch.setattr(b200q, "_LIB", None)
    assert b200q.lib().b200q_abi() == 1
    with pytest.raises(b200q.B200QError, match="b200q_iq2_gemv: not in libb200q_tablefree.so") as e:
        b200q.lib().b200q_iq2_gemv(None, 0, 0, None, None, 0, None, 0, 0, None)
    assert e.value.status == b200q.EMISSING


def test_a_library_of_another_version_is_refused_when_it_is_loaded(tmp_path, monkeypatch):
    monkeypatch.setattr(b200q, "LIB_PATH", few(tmp_path, "libb200q.so"))
    monkeypatch.setattr(b200q, "_LIB", None)
    with pytest.raises(RuntimeError, match="lacks b200q_"):
        b200q.lib()
