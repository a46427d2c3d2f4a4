"""The built kernels around the cache: MFMAs of one shape per accumulator, and no packed f32
instruction (CPU only: reads the objects that the build leaves)."""
import os

import pytest

from test_mfma_shapes import LLVM, ROOT, disassembly, mixed_chains

OBJECTS = {name: os.path.join(ROOT, "_build", f"nx_{name}.o") for name in ("rope", "logprobs", "evict", "mass")}


@pytest.mark.skipif(not all(map(os.path.exists, [*OBJECTS.values(), f"{LLVM}/clang-offload-bundler"])),
                    reason="no built objects (run nexus_amd.build() first) or no ROCm LLVM tools")
@pytest.mark.parametrize("name", OBJECTS)
def test_kernels(name, tmp_path):
    lines = disassembly(OBJECTS[name], tmp_path)
    found, count = mixed_chains(lines)
    assert (count > 0) == (name == "mass")
    assert not found, found[:4]
    assert not [line for line in lines if "v_pk_add_f32" in line or "v_pk_mul_f32" in line or "v_pk_fma_f32" in line]
