"""The built kernel that moves kept tokens: its exchange between lanes runs with all of them
(CPU only: reads the objects that the build leaves)."""
import os
import re

import pytest

from test_mfma_shapes import LLVM, ROOT, disassembly

OBJECT = os.path.join(ROOT, "_build", "nx_evict.o")


def open_conditions(lines, kernel, op):
    """Of each `op` in functions whose names have `kernel` in them: how many s_and_saveexec are open."""
    found, inside, saved = [], False, []
    for line in lines:
        m = re.match(r"[0-9a-f]* ?<(\S+)>:|^(_Z\w+):", line)
        if m:
            inside, saved = kernel in (m[1] or m[2]), []
            continue
        text = line.split("//")[0].strip()
        m = re.match(r"s_and_saveexec_b64 (s\[\d+:\d+\])", text)
        if m:
            saved.append(m[1])
        m = re.match(r"s_or_b64 exec, exec, (s\[\d+:\d+\])", text)
        if m and m[1] in saved:
            del saved[saved.index(m[1]):]
        if inside and text.startswith(op):
            found.append(len(saved))
    return found


def test_conditions_are_counted():
    lines = ["0 <_Z1k>:", "s_and_saveexec_b64 s[2:3], vcc", "ds_bpermute_b32 v1, v1, v2",
             "s_and_saveexec_b64 s[4:5], vcc", "ds_bpermute_b32 v1, v1, v2", "s_or_b64 exec, exec, s[2:3]",
             "ds_bpermute_b32 v1, v1, v2", "8 <_Z1x>:", "ds_bpermute_b32 v1, v1, v2"]
    assert open_conditions(lines, "1k", "ds_bpermute_b32") == [1, 2, 0]


@pytest.mark.skipif(not all(map(os.path.exists, [OBJECT, f"{LLVM}/clang-offload-bundler"])),
                    reason="no built objects (run nexus_amd.build() first) or no ROCm LLVM tools")
def test_kept_tokens_chunks_are_compared_by_all_lanes(tmp_path):
    """A token's chunk is compared with the one before it, which the lane before hands over: the
    exchange is under the condition of the tokens' 32 threads and under no other, since what a
    lane that does not take part hands over is not defined."""
    found = open_conditions(disassembly(OBJECT, tmp_path), "k_evict_move", "ds_bpermute_b32")
    assert len(found) == 8  # two formats of four head sizes
    assert max(found) <= 1, found
