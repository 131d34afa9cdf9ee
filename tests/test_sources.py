"""What the tree's text may not hold, checked on the files themselves (CPU only).

Statements about the reference rest on its sources, build files and documents, never on what its prebuilt executables contain; GPU code
writes through the vector path only and holds no packed f32 instruction.
"""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SKIP_DIRS = {".git", "__pycache__", ".pytest_cache", "gpurun_out", "_work", "tmp_ab", "build"}


def _files(*suffixes):
    """Paths of the tree's text files with one of the suffixes (a name without a dot, such as Makefile, is its own suffix)."""
    for d, subdirs, names in os.walk(ROOT):
        subdirs[:] = sorted(s for s in subdirs if s not in SKIP_DIRS)
        for n in sorted(names):
            if n.endswith(suffixes):
                yield os.path.join(d, n)


def _hits(pattern, *suffixes):
    rx = re.compile(pattern)
    out = []
    for path in _files(*suffixes):
        with open(path, errors="replace") as f:
            out += ["%s:%d" % (os.path.relpath(path, ROOT), i) for i, line in enumerate(f, 1) if rx.search(line)]
    return out


def test_no_document_cites_the_contents_of_a_prebuilt_executable():
    """A tool's output on a shipped .exe / .dll, or its import table, is no source of a statement here."""
    reads = r"(?i)confirmed by `(strings|objdump|readelf|dumpbin)` on|(import|imports|symbol) visible in `[^`]*\.(exe|dll)"
    assert _hits(reads, ".md") == []


def test_no_gpu_code_writes_through_the_scalar_cache():
    """Scalar stores and atomics, the scalar cache's write-back and discard: in no source, script, test or kept patch, not as a comment."""
    writes = r"\b(?:s_(?:buffer_|scratch_)?(?:atomic|store)(?=_)|s_d" + r"cache_(?:wb|discard))"
    assert _hits(writes, ".hip", ".cpp", ".hpp", ".h", ".c", ".s", ".py", ".sh", ".patch", "Makefile", ".mk", ".txt") == []


PACKED_F32 = r"\bv_pk" + r"_(?:add|mul|fma)_f32\b"


def test_no_source_writes_packed_f32_instructions():
    """By hand: in no source, script or kept patch (some of their forms have given wrong results on this hardware)."""
    assert _hits(PACKED_F32, ".hip", ".cpp", ".hpp", ".h", ".c", ".s", ".py", ".sh", ".patch", "Makefile") == []


def test_every_hipcc_line_that_compiles_turns_packed_f32_off():
    """hipcc makes packed f32 instructions from ordinary float code too; the build files and tools that compile HIP code say not to."""
    missing = []
    for path in _files("Makefile", ".sh", ".py"):
        text = open(path, errors="replace").read().replace("\\\n", " ")
        if os.path.abspath(path) == os.path.abspath(__file__) or os.sep + "tests" + os.sep + "test_" in path:
            continue
        flags = "-packed-fp32-ops" in text
        for line in text.split("\n"):
            compiles = re.search(r"(\$\(HIPCC\)|bin/hipcc|env\[\"HIPCC\"\])", line) and "-shared" not in line and "?=" not in line and "setdefault" not in line
            if compiles and not line.lstrip().startswith("#") and not flags:
                missing.append("%s: %s" % (os.path.relpath(path, ROOT), line.strip()[:60]))
    assert missing == []


@pytest.mark.parametrize("name", ["slx_kernels", "slx_track", "slx_cloud", "slx_text", "slx_gather"])
def test_compiled_kernels_hold_no_packed_f32_instruction(name, tmp_path):
    """The device code of every kernel file, compiled by the library's own command line (`make -n`), holds none."""
    csrc = os.path.join(ROOT, "structured-light-calculation_amd", "csrc")
    dry = subprocess.run(["make", "-n", "-B", "-C", csrc, name + ".o"], capture_output=True, text=True, check=True).stdout
    cmd = next(ln for ln in dry.splitlines() if name + ".hip" in ln and " -c " in ln).split()
    if not os.path.exists(cmd[0]):
        pytest.skip("hipcc is not installed")
    out = str(tmp_path / "k.s")
    cmd = [a for a in cmd[:cmd.index("-o")] if a != "-c"] + ["-S", "--cuda-device-only", "-o", out]
    subprocess.run(cmd, cwd=csrc, check=True, stderr=subprocess.DEVNULL)
    with open(out) as f:
        text = f.read()
    assert "amdhsa.kernels" in text
    assert len(re.findall(PACKED_F32, text)) == 0
