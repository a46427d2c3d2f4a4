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


@needs_gxx
def test_weights_behind_the_last_one_are_no_overlap(tmp_path):
    """Host calls know where weights end: what lies behind the last sequence's last is another's."""
    run(tmp_path, r"""
  static float m[4096];
  static int32_t out[64];
  int32_t len[3] = {100, 50, 0}, pages[12] = {0, 1, 2, 3, 4, 5, -1, -1, -1, -1, -1, -1}, to[6] = {6, 7, 8, 9, 10, 11};
  nx_kv_batch b{3, 0, 4, nullptr, len, pages};
  EvictArgs a{to, 2, 40, 4, 8, m, 100, out, out + 32, nullptr, 40};
  // two heads: rows at 0, 100, 200, 300, the last with weights of 50
  auto evict = [&](long at) {
    a.new_mass = m + at;
    is(evict_check(&b, 32, 2, a, true).code == NX_OK, "looked at later");
    return evict_check_tables(b, 12, 32, a, 2).code;
  };
  is(evict(350) == NX_OK && evict(400) == NX_OK, "behind the last weight");
  is(evict(349) == NX_ERR_INVALID_ARG && evict(300) == NX_ERR_INVALID_ARG && evict(0) == NX_ERR_INVALID_ARG, "before it");
  EvictArgs e = a;  // rows at 0, 40, 80, 120 of new weights, and then the old ones
  e.new_mass = m, e.mass = m + 160;
  is(evict_check_tables(b, 12, 32, e, 2).code == NX_OK, "in front");
  e.mass = m + 159;
  is(evict_check_tables(b, 12, 32, e, 2).code == NX_ERR_INVALID_ARG, "into the last of them");
  e = a, e.new_mass = m + 100, e.mass_stride = e.new_mass_stride = 140;
  is(evict_check_tables(b, 12, 32, e, 2).code == NX_OK, "beside each other");
  a.new_mass = m + 600;
  is(evict_check(&b, 32, 2, a).code == NX_OK, "a device call with whole rows in front");
  a.new_mass = m + 350;
  is(evict_check(&b, 32, 2, a).code == NX_ERR_INVALID_ARG, "a device call does not know the lengths");

  int32_t rows[4] = {0, 2, 3, 3};
  nx_kv_batch s{3, 3, 4, rows, len, pages};
  auto mass = [&](const float *before, const float *to) { return mass_check_tables(s, 2, before, to, 100).code; };
  is(mass(m, m) == NX_OK && mass(nullptr, m) == NX_OK && mass(m, m + 349) == NX_OK, "in place, none, behind");
  is(mass(m, m + 348) == NX_ERR_INVALID_ARG && mass(m + 349, m) == NX_ERR_INVALID_ARG && mass(m + 350, m) == NX_OK, "in part");
  is(mass_check(&s, 2, 4, 256, 256, m, m, m + 349, 100).code == NX_ERR_INVALID_ARG, "whole rows");
  is(mass_check(&s, 2, 4, 256, 256, m, m, m + 349, 100, true).code == NX_OK, "looked at later");
""")
