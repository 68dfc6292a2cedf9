"""Kernels that may start before the one in front of them has ended, by their source: each waits for it before it touches
global memory, unconditionally.  (PTX promises the writes of earlier kernels to a grid that has executed the wait itself,
so that no run can show that a kernel does without it.)"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mercury_artifact_b200" / "csrc"
FILES = ["attn_paged_rows.cu", "attn_paged_tiles.cu", "kv_cache.cu", "merge.cu"]
ACCESS = re.compile(r"__ld|__st|atomic|cp_async|tma_load|paged_seq\(|paged_entry\(|\b(seq_lens|cu|table|open|tile_open|part_ml|part_o|tile_ml)\[")


def kernels(name):
    """(kernel, body) of every kernel of the file that is launched with launch_overlapped."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)
    for m in re.finditer(r"__global__\s+void(?:\s+__\w+__\([^()]*(?:\([^()]*\))?[^()]*\))*\s+(\w+)\s*\(", text):
        at = text.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        yield m.group(1), text[at + 1:end - 1]


@pytest.mark.parametrize("name", FILES)
def test_wait_comes_before_every_access(name):
    found = 0
    for kernel, body in kernels(name):
        if "grid_dependency_wait" not in body and "grid_dependents_launch" not in body:
            continue  # launched in the ordinary way
        found += 1
        wait = re.search(r"(?<=[;{}])\s*grid_dependency_wait\(\);", body)
        assert wait, f"{kernel}: no unconditional wait"
        before = body[:wait.start()]
        assert before.count("{") == before.count("}"), f"{kernel}: the wait is inside a block"
        assert not ACCESS.search(before), f"{kernel}: {ACCESS.search(before).group()} before the wait"
        assert body.count("grid_dependency_wait") == 1
    assert found >= 1
