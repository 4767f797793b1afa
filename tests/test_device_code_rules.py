"""CPU: what the HIP code of this repository must not contain, checked on its sources, build lines and the built library."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _texts(*patterns):
    """(path relative to the root, text) of every file the patterns match."""
    paths = sorted({p for pat in patterns for p in glob.glob(os.path.join(ROOT, pat))})
    assert paths
    return [(os.path.relpath(p, ROOT), open(p, errors="replace").read()) for p in paths]


def _hip_sources():
    return _texts("ais-catcher_amd/csrc/*.hip", "ais-catcher_amd/csrc/*.cpp", "ais-catcher_amd/csrc/*.h", "ais-catcher_amd/csrc/*.inc",
                  "tools/*.hip")


def test_no_writes_through_the_scalar_data_cache():
    """gfx950 has no working scalar store (it assembles and writes nothing): device code writes through vector stores only."""
    scalar_write = re.compile(r"\bs_((buffer_|scratch_)?(store|atomic)|dcache_(wb|discard))", re.I)
    for name, text in _hip_sources():
        assert not scalar_write.search(text), name


def test_streams_have_the_default_priority():
    """Work on streams of different queue priorities can stop for good on this hardware: no source asks for one."""
    sources = _texts("ais-catcher_amd/*.py", "ais-catcher_amd/host/*.cpp", "ais-catcher_amd/host/*.h", "integration/reference/Source/DSP/GPU/*",
                     "tools/*.py", "bench.py")
    for name, text in _hip_sources() + sources:
        assert not re.search(r"StreamCreateWithPriority|StreamPriorityRange|\bpriority\s*=|is_high_priority_stream", text), name


# Packed f32 (v_pk_add / v_pk_mul / v_pk_fma): some of its forms have given wrong results on gfx950 now and then.
PACKED_F32 = re.compile(r"\bv_pk_(add|mul|fma)_f32\b")


def test_no_packed_f32_written_by_hand():
    for name, text in _hip_sources():
        assert not PACKED_F32.search(text), name


def test_every_hip_build_line_turns_packed_f32_off():
    """hipcc -O3 makes packed f32 of ordinary float code, so every line that compiles HIP code carries the flag."""
    flag = "-Xclang -target-feature -Xclang -packed-fp32-ops"
    for name, text in _texts("ais-catcher_amd/csrc/Makefile", "tools/*.sh", "tools/*.hip"):
        for line in text.replace("\\\n", " ").splitlines():
            if "--offload-arch" in line:
                assert flag in re.sub(r"\s+", " ", line), (name, line)


def test_built_library_has_no_packed_f32(tmp_path):
    """The library as it was built: the gfx950 code object it carries, listed."""
    objdump = "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(os.path.join(ROOT, "ais-catcher_amd", "libaisgpu.so"), tmp_path)
    subprocess.run([objdump, "--offloading", lib], check=True, cwd=tmp_path, stdout=subprocess.DEVNULL)
    objects = [p for p in glob.glob(os.path.join(tmp_path, "libaisgpu.so.*gfx950*")) if os.path.getsize(p)]
    assert objects
    for p in objects:
        listing = subprocess.run([objdump, "-d", "--no-show-raw-insn", p], check=True, stdout=subprocess.PIPE, text=True).stdout
        assert listing.count("v_add_f32") > 1000  # (the listing is of the kernels)
        assert not PACKED_F32.search(listing), PACKED_F32.search(listing).group()
