"""Streams of different priorities have kept this chip waiting without end: nothing here makes a stream or a process group of another priority than
the default (a reading of the sources, no GPU needed)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OTHER = re.compile(r"hipStreamCreateWithPriority|cudaStreamCreateWithPriority|Stream\([^)]*priority\s*=|is_high_priority_stream\s*=\s*True")


def test_every_stream_has_the_default_priority():
    found = []
    for top in ("tf_repos_amd", "tools", "examples", "perf", "include", "oracle", ""):
        for folder, inner, names in os.walk(os.path.join(ROOT, top)):
            inner[:] = [] if not top else [d for d in inner if d not in ("_lib", "__pycache__")]
            for name in names:
                if name.endswith((".hip", ".h", ".cpp", ".py", ".sh")):
                    path = os.path.join(folder, name)
                    for i, line in enumerate(open(path, errors="replace"), 1):
                        if OTHER.search(line):
                            found.append("%s:%d" % (os.path.relpath(path, ROOT), i))
    assert not found, found
