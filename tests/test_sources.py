"""What the tree's text may not hold, checked on the files themselves (CPU only).

Statements about the reference rest on its sources, build files and documents, never on what its prebuilt executables contain; GPU code
writes through the vector path only.
"""
import os
import re

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
