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


@needs_gxx
def test_weights_are_read_up_to_the_last_one(tmp_path):
    """Host calls read no weight behind the last sequence's last: a caller's rows may end there."""
    run(tmp_path, r"""
  const int lens[][5] = {{5, 3, 9, 2, 4}, {9, 9, 9, 9, 9}, {0, 7, 0, 0, 0}, {7, 0, 0, 0, 1}, {0, 0, 0, 0, 0}, {1, 2, 3, 4, 0}};
  for (auto &len : lens)
    for (int seqs = 1; seqs <= 5; ++seqs)
      for (int heads : {1, 2, 5}) {
        size_t width = 1, end = 0, stride = 0;
        for (int s = 0; s < seqs; ++s) width = std::max(width, (size_t)len[s]);
        for (size_t more : {0, 1, 40}) {
          stride = width + more;
          for (int s = 0; s < seqs; ++s)
            if (len[s]) end = ((size_t)s * heads + heads - 1) * stride + len[s];
          const WeightRows r = weight_rows(seqs, heads, [&](int s) { return (size_t)len[s]; });
          size_t read = r.rows ? (r.rows - 1) * stride + r.last : 0;
          if (r.rows > 1) read = std::max(read, (r.rows - 2) * stride + width);
          is(read == end, "all of them, and nothing behind");
          for (int s = 0; s < seqs; ++s)
            is(len[s] == 0 || (size_t)(s + 1) * heads < r.rows || ((size_t)(s + 1) * heads == r.rows && r.last == (size_t)len[s]),
               "each row has its own");
          end = 0;
        }
      }
""")
