"""Limits that the calls around the cache document, as their plans have them (nexus_amd/csrc/nx_step_plan.hpp),
on the CPU."""
import os
import re

from test_kv_plan import needs_gxx
from test_mfma_shapes import ROOT
from test_step_plan import run


@needs_gxx
def test_rows_that_take_the_workspace_of_log_probabilities(tmp_path):
    """Those that the header names: up to so many rows, of more than so many logits."""
    text = re.sub(r"[\s*]+", " ", open(os.path.join(ROOT, "include", "nexus_hip.h")).read())
    assert "up to 512 rows of more than 4096 logits" in text
    run(tmp_path, r"""
  for (int rows : {1, 2, 61, 511, 512, 513, 600, 1023, 1024, 5000, 1 << 24})
    for (int vocab : {1, 100, 4095, 4096, 4097, 5000, 32000, 262144, 1 << 30})
      is((logprob_split(rows, vocab).parts > 1) == (rows <= 512 && vocab > 4096), "shared rows");
""")
