"""What the sources of this repository must not contain, whatever they compute."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = (".py", ".c", ".cpp", ".h", ".hpp", ".hip", ".rs", ".toml", ".sh", ".s", ".S", ".ll", ".inc", "Makefile")
SKIP = {".git", ".pytest_cache", "__pycache__", "_work", "gpurun_out", "variants"}


def code_files():
    for folder, names, files in os.walk(ROOT):
        names[:] = [n for n in names if n not in SKIP]
        for f in files:
            path = os.path.join(folder, f)
            if f.endswith(CODE) and os.path.abspath(path) != os.path.abspath(__file__):
                yield path


def hits(pattern):
    found, scanned = [], 0
    for path in code_files():
        scanned += 1
        with open(path, errors="replace") as f:
            found += [f"{os.path.relpath(path, ROOT)}:{i}" for i, line in enumerate(f, 1) if pattern.search(line)]
    assert scanned > 40                                        # the walk found the sources
    return found


def test_no_code_reads_the_references_compiled_shaders():
    """The oracle is written from the GLSL sources; nothing opens or decodes the modules compiled from them."""
    assert hits(re.compile(r"\.spv\b|/spv\b|\bspir-?v", re.I)) == []


def test_no_code_writes_through_the_scalar_data_cache():
    """Device code writes through vector stores only (scalar stores, scalar atomics and the cache's write-back and discard
    are in no source, in inline assembly or comments): the timeline probes wrote their slots with scalar stores."""
    assert hits(re.compile(r"(\b|\\[nt])s_((buffer_|scratch_)?(store|atomic)|dcache_(wb|discard))")) == []
