"""The paged cache without a device: every entry point include/wsp_cache.h
declares is exported and has a ctypes signature, the structures are laid out
as the header has them, the C++ header compiles against the library, and every
refusal of the entry points comes back before anything is launched
(tests/cpp/cache_test.cu, compiled with the cache's host code).  On the GPU, the
program over the C++ header runs."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "wsp_cache.h")


def test_library_exports_every_declared_symbol():
    from whispereacp_b200._native import SIGNATURES, library
    names = set(re.findall(r"\b(wsp_[a-z_]+)\s*\(", re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)))
    assert {"wsp_cache_create", "wsp_cache_append", "wsp_cache_read", "wsp_cache_attend"} <= names
    for name in names:
        assert hasattr(library(), name), f"{name} is declared but not exported"
        assert name in SIGNATURES, f"{name} has no ctypes signature"


def test_the_structures_are_laid_out_as_the_header_has_them(tmp_path):
    import ctypes
    from whispereacp_b200 import _native as N
    source = tmp_path / "sizes.c"
    pairs = {"wsp_cache_shape": N.CCacheShape, "wsp_cache_memory": N.CCacheMemory, "wsp_cache_batch": N.CCacheBatch,
             "wsp_cache_rows": N.CCacheRows}
    lines = [f'printf("%zu", sizeof({c}));' + "".join(f'printf(" %zu", offsetof({c}, {f[0]}));' for f in p._fields_) +
             'printf("\\n");' for c, p in pairs.items()]
    source.write_text('#include "wsp_cache.h"\n#include <stdio.h>\nint main(void) {' + "".join(lines) + "return 0; }\n")
    program = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"), str(source),
                    "-o", str(program)], check=True)
    said = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, p in zip(said, pairs.values()):
        assert [int(x) for x in line.split()] == [ctypes.sizeof(p)] + [getattr(p, f[0]).offset for f in p._fields_]


def test_every_refusal_comes_before_any_launch(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc is not installed")
    program = os.path.join(str(tmp_path), "cache_test")
    library = os.path.join(ROOT, "whispereacp_b200")
    build = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-ccbin", "g++",
                            "--expt-relaxed-constexpr", "-o", program, os.path.join(ROOT, "tests", "cpp", "cache_test.cu"),
                            "-L", library, "-lwsp_b200", "-Xlinker", f"-rpath={library}"], capture_output=True, text=True)
    if build.returncode != 0:
        pytest.fail(build.stderr)
    run = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def compile_binding(out_dir) -> str:
    cuda = "/usr/local/cuda"
    library = os.path.join(ROOT, "whispereacp_b200")
    program = os.path.join(str(out_dir), "cache_binding_test")
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
                            "-I", os.path.join(cuda, "include"), os.path.join(ROOT, "tests", "cpp", "cache_binding_test.cpp"),
                            "-L", library, "-lwsp_b200", f"-Wl,-rpath,{library}", "-L", os.path.join(cuda, "lib64"),
                            "-lcudart", f"-Wl,-rpath,{os.path.join(cuda, 'lib64')}", "-o", program],
                           capture_output=True, text=True)
    if build.returncode != 0:
        pytest.fail(build.stderr)
    return program


def test_the_cpp_header_compiles_against_the_library(tmp_path):
    compile_binding(tmp_path)


@pytest.mark.gpu
def test_the_cache_through_the_cpp_header(tmp_path):
    run = subprocess.run([compile_binding(tmp_path)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def test_tensors_that_are_not_on_a_device_are_refused():
    torch = pytest.importorskip("torch")
    from whispereacp_b200 import CacheBatch, PagedCache
    with pytest.raises(ValueError, match="CUDA device"):
        PagedCache(torch.zeros(2, 1, 16, 64), torch.zeros(2, 1, 16, 64))
    with pytest.raises(ValueError, match="CUDA device"):
        CacheBatch(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="storage"):
        PagedCache.allocate(1, 1, 16, 64, storage="int4")
