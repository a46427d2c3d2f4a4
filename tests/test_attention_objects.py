"""The attention's built kernels: MFMAs of one shape per accumulator, and no
packed f32 instruction (CPU only: reads the objects that the build leaves)."""
import os

import pytest

from test_mfma_shapes import LLVM, ROOT, disassembly, mixed_chains

OBJECT = os.path.join(ROOT, "_build", "nx_attn.o")


@pytest.mark.skipif(not (os.path.exists(OBJECT) and os.path.exists(f"{LLVM}/clang-offload-bundler")),
                    reason="no built object (run nexus_amd.build() first) or no ROCm LLVM tools")
def test_attention_kernels(tmp_path):
    lines = disassembly(OBJECT, tmp_path)
    found, count = mixed_chains(lines)
    assert count > 0
    assert not found, found[:4]
    assert not [line for line in lines if "v_pk_add_f32" in line or "v_pk_mul_f32" in line or "v_pk_fma_f32" in line]
