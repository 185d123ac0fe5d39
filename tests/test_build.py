"""Host-only checks of build_library(): what it needs for what it builds.  The compilers are stand-ins that write their
output file; the package's own paths are turned to a folder of the test's."""
import json
import re
import sys
import warnings

import pytest

from tests.conftest import load_package

LIBRARIES = ("bshd", "serving", "mx4", "loader_kat", "mfma_ceiling")


def stand_in(path, status=0):
    path.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do\n  [ "$1" = -o ] && echo built > "$2"\n  shift\ndone\n'
                    f'echo "compiler says so" >&2\nexit {status}\n')
    path.chmod(0o755)
    return str(path)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """The binding's module, with its build folder and compilers in tmp_path."""
    module = load_package().fav4_bshd
    build = tmp_path / "build"
    for name in ("LIB_PATH", "SERVING_LIB_PATH", "MX4_LIB_PATH", "MX4_BLOCKS_PATH", "KAT_LIB_PATH", "CEILING_LIB_PATH",
                 "RESOURCE_LOG", "MANIFEST"):
        monkeypatch.setattr(module, name, build / getattr(module, name).name)
    monkeypatch.setattr(module, "_MX4_BLOCKS", None)
    monkeypatch.setenv("HIPCC", stand_in(tmp_path / "hipcc"))
    monkeypatch.setenv("CXX", stand_in(tmp_path / "cxx"))
    return module


def built(module):
    """The build as it ended, and the libraries that it left."""
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        module.build_library(module.LIB_PATH)
    said = [str(w.message) for w in seen if "fav4_mx4_blocks" in str(w.message)]
    names = {p.name for p in module.LIB_PATH.parent.glob("*.so")}
    return names, said, json.loads(module.MANIFEST.read_text())


def c_libraries(module):
    return {module.LIB_PATH.parent.joinpath(f"libfav4_{n}.so").name for n in LIBRARIES}


def test_builds_everything(tree):
    names, said, manifest = built(tree)
    assert names == c_libraries(tree) | {"fav4_mx4_blocks.so"} == set(manifest["libraries"]) and not said


def without_torch(tree, monkeypatch, tmp_path):
    monkeypatch.setitem(sys.modules, "torch", None)
    return "torch"


def without_a_compiler(tree, monkeypatch, tmp_path):
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    return "no-such-compiler"


@pytest.mark.parametrize("missing", [without_torch, without_a_compiler])
def test_the_c_libraries_need_hipcc_alone(tree, monkeypatch, tmp_path, missing):
    """The extension is left out, one of an earlier build too (its argument blocks may be others), and loading it says
    why."""
    tree.MX4_BLOCKS_PATH.parent.mkdir()
    tree.MX4_BLOCKS_PATH.write_text("of an earlier build")
    word = missing(tree, monkeypatch, tmp_path)
    names, said, manifest = built(tree)
    assert names == c_libraries(tree) == set(manifest["libraries"])
    assert len(said) == 1 and word in said[0]
    with pytest.raises(OSError, match=word):
        tree.load_mx4_blocks(tree.MX4_BLOCKS_PATH)


def test_an_extension_that_does_not_compile_is_an_error(tree, monkeypatch, tmp_path):
    """... after the libraries are built."""
    monkeypatch.setenv("CXX", stand_in(tmp_path / "bad", status=1))
    with pytest.raises(RuntimeError, match="compiler says so"):
        tree.build_library(tree.LIB_PATH)
    assert c_libraries(tree) <= {p.name for p in tree.LIB_PATH.parent.glob("*.so")}
    assert not tree.MX4_BLOCKS_PATH.exists()


@pytest.fixture(scope="module")
def extension():
    """The built extension's path (built here where one of the two is missing)."""
    pkg = load_package()
    if not pkg.fav4_bshd.MX4_BLOCKS_PATH.exists() or not pkg.MX4_LIB_PATH.exists():
        pkg.build_library()
    return pkg.fav4_bshd.MX4_BLOCKS_PATH


def test_an_extension_of_another_torch_is_refused(extension, monkeypatch):
    """It reads tensors by the C++ layout of the torch that it was built against."""
    import torch
    module = load_package().fav4_bshd
    monkeypatch.setattr(module, "_MX4_BLOCKS", None)
    built_for = module.load_mx4_blocks(extension).torch_version
    assert built_for == torch.__version__
    monkeypatch.setattr(module, "_MX4_BLOCKS", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(OSError, match=f"torch {re.escape(built_for)}, not 1.0.0"):
        module.load_mx4_blocks(extension)
    assert module._MX4_BLOCKS is None


def test_an_extension_that_does_not_load_is_an_oserror(tmp_path, monkeypatch):
    """As a build against another torch ends whose symbols are gone."""
    module = load_package().fav4_bshd
    monkeypatch.setattr(module, "_MX4_BLOCKS", None)
    path = tmp_path / "fav4_mx4_blocks.so"
    path.write_bytes(b"no library")
    with pytest.raises(OSError, match="does not load"):
        module.load_mx4_blocks(path)


def test_the_manifest_says_how_the_extension_was_built(tree):
    import torch
    manifest = built(tree)[2]["extension"]
    assert manifest["torch"] == torch.__version__
    assert manifest["command"][0].endswith("cxx") and any("mx4_blocks.cpp" in x for x in manifest["command"])


def test_the_manifest_of_a_build_without_it(tree, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert built(tree)[2]["extension"] is None
