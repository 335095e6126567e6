"""CPU: the script that builds a variant of the library with other flags for some files (scripts/build_variant.sh)."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


def test_a_variant_is_the_library_with_one_file_compiled_again(trag):
    lib = os.path.join(ROOT, "trueno-rag_amd", "lib")
    if not os.path.exists(HIPCC) or not os.path.exists(os.path.join(lib, "trag_api.o")):
        pytest.skip("the library's objects are not here")
    name = f"test_{os.getpid()}"
    out = os.path.join(ROOT, "trueno-rag_amd", "lib_var", name)
    try:
        r = subprocess.run(["bash", "-x", os.path.join(ROOT, "scripts", "build_variant.sh"), name, "-f", "trag_fuse_device.hip", "-DVARIANT=1"],
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        compiled = [line for line in r.stderr.splitlines() if HIPCC in line and "-DVARIANT=1" in line]
        assert len(compiled) == 1 and "-ffp-contract=off" in compiled[0] and "-packed-fp32-ops" in compiled[0]
        assert os.path.exists(os.path.join(out, "trag_fuse_device.o")) and not os.path.exists(os.path.join(out, "trag_api.o"))
        # every symbol is there, and every entry of the interface
        load = ("import sys; sys.path.insert(0, sys.argv[1]); from conftest import load_package as p; t = p(); t.lib(); "
                "assert 'lib_var' in t.lib_path()")
        r = subprocess.run([sys.executable, "-c", load, os.path.join(ROOT, "tests")], capture_output=True, text=True, timeout=300,
                           env=dict(os.environ, TRAG_LIB=os.path.join(out, "libtrag.so"), LD_BIND_NOW="1"))
        assert r.returncode == 0, r.stderr[-2000:]
    finally:
        shutil.rmtree(out, ignore_errors=True)
