"""CPU: what the HIP code of this repository must not contain, checked on its sources, build lines and the built library."""
import glob
import os
import re

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
