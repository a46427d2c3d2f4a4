"""No MFMA of the attention's built kernels runs while some of its wave's lanes are masked.

An MFMA ignores the mask of active lanes, but copies of its registers (accumulators that
live in the other register file among them) do not.  Conditions that a whole wave shares,
held in vector registers, become such masks: k_attn_tile on heads of 256 gave wrong rows
that way.  Whether a condition is scalar hangs on what the compiler can prove, and parity
tests of one build say nothing about the next.  This test reads the instructions of the
object that the build leaves in _build/ (CPU only).
"""
import os
import re

import pytest

from test_mfma_shapes import LLVM, ROOT, disassembly

OBJECT = os.path.join(ROOT, "_build", "nx_attn.o")


def functions(lines):
    """name -> [(address, instruction, address that it branches to or None)]"""
    out, body, start = {}, [], 0
    for line in lines:
        m = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if m:
            body, start = out.setdefault(m[2], []), int(m[1], 16)
            continue
        m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):[^<]*(?:<\S+?(?:\+0x([0-9a-f]+))?>)?$", line)
        if m:
            body.append((int(m[2], 16), m[1], start + int(m[3] or "0", 16) if "branch" in m[1] else None))
    return out


def masked_mfmas(body):
    """(the MFMAs that some way from the barrier before a kernel's first one, which whole
    waves pass, to the next barrier reaches between a narrowing of the mask and the place that takes
    it back, or behind a change of any other kind; all MFMAs)."""
    mfmas = [i for i, (_, text, _) in enumerate(body) if text.startswith("v_mfma")]
    if not mfmas:
        return [], 0
    index = {address: i for i, (address, _, _) in enumerate(body)}
    start = max((i for i in range(mfmas[0]) if body[i][1].startswith("s_barrier")), default=-1) + 1
    found, passed, ways = {}, set(), [(start, ())]  # (instruction, the masks that are saved before it)
    while ways:
        i, saved = ways.pop()
        while (i, saved) not in passed and i < len(body):
            passed.add((i, saved))
            _, text, target = body[i]
            op, _, rest = text.partition(" ")
            operands = [o.strip() for o in re.split(r",(?![^\[]*\])", rest)]
            if op in ("s_barrier", "s_endpgm"):
                break
            if op.startswith("v_mfma"):
                if saved:
                    found[i] = text
            elif op == "s_and_saveexec_b64":
                saved += (operands[0],)
            elif op.endswith("saveexec_b64") or operands[0].startswith("exec"):
                if op == "s_or_b64" and saved and operands[2] == saved[-1]:
                    saved = saved[:-1]
                elif not (op == "s_and_b64" and saved):  # (narrower still, until it is taken back)
                    saved = (None,)
            if target is not None:
                ways.append((index[target], saved))
            if op == "s_branch":
                break
            i += 1
    assert {i for i, _ in passed} >= set(mfmas), "MFMAs behind the next barrier"
    return [found[i] for i in sorted(found)], len(mfmas)


@pytest.mark.skipif(not (os.path.exists(OBJECT) and os.path.exists(f"{LLVM}/clang-offload-bundler")),
                    reason="no built object (run nexus_amd.build() first) or no ROCm LLVM tools")
def test_attention_mfmas_run_on_whole_waves(tmp_path):
    results = {name: masked_mfmas(body) for name, body in functions(disassembly(OBJECT, tmp_path)).items()}
    assert sum(count > 0 for _, count in results.values()) == 16  # two kernels, formats, four head sizes
    assert not {name: found[:4] for name, (found, _) in results.items() if found}


def listing(*instructions):
    """A function of 4-byte instructions; a branch ends in the number of its target."""
    out = ["0000000000001000 <f>:"]
    for i, text in enumerate(instructions):
        text, _, to = text.partition(" -> ")
        out.append(f"\t{text}   // {4096 + 4 * i:012X}: BF800000" + (f" <f+0x{4 * int(to):x}>" if to else ""))
    return functions(out)["f"]


def test_finds_a_masked_mfma():
    mfma = "v_mfma_f32_32x32x16_f16 v[0:15], v[16:19], v[20:23], v[0:15]"
    narrow, narrower, back = "s_and_saveexec_b64 s[4:5], vcc", "s_and_b64 exec, exec, s[2:3]", "s_or_b64 exec, exec, s[4:5]"
    move, other = "v_mov_b32_e32 v30, v31", "s_mov_b64 exec, s[2:3]"
    check = lambda *a: masked_mfmas(listing(*a))  # noqa: E731
    assert check("s_barrier", mfma, narrow, narrower, move, back, mfma) == ([], 2)
    assert check("s_barrier", narrow, mfma, back, mfma) == ([mfma], 2)
    assert check("s_barrier", narrow, narrower, move, mfma) == ([mfma], 1)
    assert check("s_barrier", mfma, other) == ([], 1)
    assert check("s_barrier", mfma, other, mfma) == ([mfma], 2)
    assert check(narrow, "s_barrier", mfma) == ([], 1)
    assert check(move) == ([], 0)
    # over a part that is apart in the listing, which comes back in front of the taking back, or behind it
    apart = ["s_barrier", narrow, "s_cbranch_execnz -> 6", back, mfma, "s_endpgm", move]
    assert check(*apart, "s_branch -> 3") == ([], 1)
    assert check(*apart, "s_branch -> 4") == ([mfma], 1)
