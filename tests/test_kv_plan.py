"""The paged cache's layout and refusals (nexus_amd/csrc/nx_kv_plan.hpp), on the
CPU: the header is plain C++ and is compiled on its own with the host compiler.
"""
import os
import shutil
import subprocess

import pytest

import nexus_amd as nx

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nexus_amd", "csrc")
GXX = shutil.which("g++")
needs_gxx = pytest.mark.skipif(GXX is None, reason="no host C++ compiler")


def run(tmp_path, body):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text('#include <cstdio>\n#include <set>\n#include "nx_kv_plan.hpp"\nusing namespace nx;\n'
                   "int bad = 0;\n"
                   "void is(bool ok, const char *what) { if (!ok) { std::printf(\"%s\\n\", what); ++bad; } }\n"
                   "int main() {\n" + body + "\n  return bad ? 1 : 0;\n}\n")
    r = subprocess.run([GXX, "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, f"exit {r.returncode}\n{r.stdout[-2000:]}"


@needs_gxx
def test_layout_is_a_bijection(tmp_path):
    """Every (token, element) of a group has a place of its own, chunk order and
    row order included."""
    run(tmp_path, r"""
  for (int fmt : {NX_KV_F16, NX_KV_INT8}) {
    for (int t = 0; t < 32; ++t) is(kv_token(fmt, kv_row(fmt, t)) == t, "kv_token inverts kv_row");
    for (int D : {64, 96, 128, 256}) {
      std::set<int> k, v;
      for (int t = 0; t < 32; ++t)
        for (int d = 0; d < D; ++d) {
          k.insert(kv_key_at(fmt, t, d));
          v.insert(kv_value_at(D, t, d));
        }
      is((int)k.size() == 32 * D && *k.rbegin() == 32 * D - 1 && *k.begin() == 0, "keys");
      is((int)v.size() == 32 * D && *v.rbegin() == 32 * D - 1 && *v.begin() == 0, "values");
    }
  }
""")


@needs_gxx
def test_rows_put_eight_tokens_in_a_lane(tmp_path):
    """The accumulator of a 16-row tile holds rows 4 g .. 4 g + 3 in lane group g:
    the two tiles of a group give that lane tokens 8 g .. 8 g + 7, the value chunk
    it multiplies.  A 32-row tile: rows 8 a + 4 h + b in half h give it tokens
    16 s + 8 h .. + 7."""
    run(tmp_path, r"""
  for (int g = 0; g < 4; ++g)
    for (int u = 0; u < 2; ++u)
      for (int i = 0; i < 4; ++i) {
        const int m = 4 * g + i;  // row of tile u
        is(kv_token(NX_KV_F16, 16 * (m >> 3) + 8 * u + (m & 7)) == 8 * g + 4 * u + i, "f16, 16 rows");
        is(kv_token(NX_KV_INT8, 2 * m + u) == 8 * g + 4 * u + i, "int8, 16 rows");
      }
  for (int h = 0; h < 2; ++h)
    for (int i = 0; i < 16; ++i)
      is(kv_token(NX_KV_F16, (i / 4) * 8 + 4 * h + i % 4) == 16 * (i / 8) + 8 * h + i % 8, "32 rows");
""")


@needs_gxx
def test_geometry(tmp_path):
    run(tmp_path, r"""
  auto code = [](int fmt, int pages, int pt, int heads, int D) { return kv_check_geometry(fmt, pages, pt, heads, D).code; };
  for (int fmt : {NX_KV_F16, NX_KV_INT8})
    for (int pt : {32, 64, 1024})
      for (int D : {64, 96, 128, 256}) is(code(fmt, 1, pt, 1, D) == NX_OK, "taken");
  is(code(2, 1, 64, 1, 64) == NX_ERR_INVALID_ARG && code(-1, 1, 64, 1, 64) == NX_ERR_INVALID_ARG, "format");
  is(code(0, 0, 64, 1, 64) == NX_ERR_INVALID_ARG && code(0, -1, 64, 1, 64) == NX_ERR_INVALID_ARG, "pages");
  is(code(0, 1, 64, 0, 64) == NX_ERR_INVALID_ARG && code(0, 1, 64, 1, 0) == NX_ERR_INVALID_ARG, "zero");
  for (int pt : {1, 16, 48, 2048, 33}) is(code(0, 1, pt, 1, 64) == NX_ERR_UNSUPPORTED, "page size");
  for (int D : {32, 65, 80, 160, 512}) is(code(0, 1, 64, 1, D) == NX_ERR_UNSUPPORTED, "head_dim");
  is(code(0, 1, 64, 4097, 64) == NX_ERR_UNSUPPORTED, "heads");
  is(kv_plane_bytes(NX_KV_F16, 1 << 20, 64, 8, 128) == ((size_t)1 << 37), "bytes past 32 bits");
  is(kv_scale_bytes(NX_KV_F16, 10, 64, 8) == 0 && kv_scale_bytes(NX_KV_INT8, 10, 64, 8) == 20480, "scales");
""")


@needs_gxx
def test_batches(tmp_path):
    run(tmp_path, r"""
  int32_t rs[3] = {0, 1, 3}, len[2] = {70, 40}, pg[4] = {0, 1, 2, -7};
  nx_kv_batch b{2, 3, 2, rs, len, pg};
  auto shallow = [&](nx_kv_batch x) { return kv_check_batch(&x, 64).code; };
  is(kv_check_batch(nullptr, 64).code == NX_ERR_INVALID_ARG, "null batch");
  is(shallow(b) == NX_OK, "good");
  for (int i = 0; i < 3; ++i) {
    nx_kv_batch x = b;
    (i == 0 ? x.num_seqs : i == 1 ? x.num_tokens : x.max_pages) = -1;
    is(shallow(x) == NX_ERR_INVALID_ARG, "negative");
    x = b;
    (i == 0 ? x.row_start : i == 1 ? x.kv_len : x.pages) = nullptr;
    is(shallow(x) == NX_ERR_INVALID_ARG, "null array");
  }
  nx_kv_batch e{0, 3, 0, nullptr, nullptr, nullptr};
  is(shallow(e) == NX_OK, "no sequences");
  nx_kv_batch t{2, 0, 2, nullptr, nullptr, nullptr};
  is(shallow(t) == NX_OK, "no rows");
  nx_kv_batch z = b;
  z.max_pages = 0;
  is(shallow(z) == NX_ERR_SHAPE, "no pages");
  z.max_pages = INT32_MAX / 64;
  is(shallow(z) == NX_ERR_UNSUPPORTED, "2^31 tokens");
  z = b;
  z.num_tokens = (1 << 24) + 1;
  is(shallow(z) == NX_ERR_UNSUPPORTED, "rows");

  auto deep = [&](bool whole, bool writes) { return kv_check_tables(b, 3, 64, whole, writes).code; };
  is(deep(true, false) == NX_OK && deep(false, true) == NX_OK, "good tables");
  pg[0] = 3;  // a page that only attention needs (row 69 lies in page 1 of its sequence)
  is(deep(true, false) == NX_ERR_INVALID_ARG && deep(false, true) == NX_OK, "page behind the cache");
  pg[0] = 0; pg[1] = -1;
  is(deep(true, false) == NX_ERR_INVALID_ARG && deep(false, true) == NX_ERR_INVALID_ARG, "negative page");
  pg[1] = 1;
  len[1] = 1;
  is(deep(true, false) == NX_ERR_SHAPE, "fewer tokens than rows");
  len[1] = 129;
  is(deep(true, false) == NX_ERR_SHAPE, "longer than its pages");
  len[1] = -1;
  is(deep(true, false) == NX_ERR_SHAPE, "negative length");
  len[1] = 40;
  rs[2] = 4;
  is(deep(true, false) == NX_ERR_SHAPE, "rows behind the batch");
  rs[2] = 3; rs[1] = -1;
  is(deep(true, false) == NX_ERR_SHAPE, "rows before the batch");
  rs[1] = 1; rs[2] = 0;
  is(deep(true, false) == NX_ERR_SHAPE, "rows that decrease");
  rs[2] = 3;
  pg[2] = 1;  // both write page 1: tokens 5 and 38, 39
  is(deep(false, true) == NX_OK, "different tokens of a page");
  len[1] = 7;  // tokens 5 and 6
  is(deep(false, true) == NX_ERR_INVALID_ARG && deep(false, false) == NX_OK, "one place twice");
  rs[1] = 0;   // the first sequence has no rows: its table is not looked at
  pg[0] = pg[1] = -9;
  is(deep(true, true) == NX_OK, "a sequence left out");
""")


@needs_gxx
def test_tables_behind_a_window(tmp_path):
    """Pages that no row sees need not be there; each that some row sees does."""
    run(tmp_path, r"""
  for (int n : {1, 40})
    for (int window : {1, 64, 65, 200, INT_MAX})
      for (int sinks : {0, 1, 64, 65, INT_MAX})
        for (int missing = 0; missing < 6; ++missing) {
          const int len = 350;
          int rows[] = {0, n}, lens[] = {len}, pages[] = {0, 1, 2, 3, 4, 5};
          pages[missing] = -1;
          const nx_kv_batch b{1, n, 6, rows, lens, pages};
          bool seen = false;
          for (int p = len - n; p < len; ++p)
            for (int j = 64 * missing; j < 64 * (missing + 1); ++j)
              seen = seen || (j <= p && (p - j < window || j < sinks));
          is((kv_check_tables(b, 6, 64, true, false, window, sinks).code != NX_OK) == seen, "seen");
          is(kv_check_tables(b, 6, 64, true, false).code != NX_OK, "without a window");
        }
""")


@needs_gxx
def test_attention_arguments(tmp_path):
    run(tmp_path, r"""
  is(attn_check(8, 2, 0.1f, 0, 0).code == NX_OK && attn_check(2, 2, -3.f, 1, 0).code == NX_OK, "good");
  is(attn_check(0, 2, 0.1f, 0, 0).code == NX_ERR_INVALID_ARG, "no heads");
  is(attn_check(7, 2, 0.1f, 0, 0).code == NX_ERR_SHAPE, "uneven heads");
  is(attn_check(1, 2, 0.1f, 0, 0).code == NX_ERR_SHAPE, "fewer heads");
  is(attn_check(8, 2, NAN, 0, 0).code == NX_ERR_INVALID_ARG, "NaN scale");
  is(attn_check(8, 2, INFINITY, 0, 0).code == NX_ERR_INVALID_ARG, "infinite scale");
  is(attn_check(8, 2, 0.1f, -1, 0).code == NX_ERR_INVALID_ARG, "window");
  is(attn_check(8, 2, 0.1f, 4, -1).code == NX_ERR_INVALID_ARG, "sinks");
  is(kv_check_rows("x", 127, 128).code == NX_ERR_SHAPE && kv_check_rows("x", 128, 128).code == NX_OK, "stride");
""")


@needs_gxx
def test_key_spans(tmp_path):
    """The groups of a span hold every token that some row sees, in order, each
    once; rows before a sequence's first token see nothing and cost none."""
    run(tmp_path, r"""
  auto sees = [](int p, int j, int window, int sinks) {
    return j <= p && (window == 0 || (long)p - j < window || j < sinks);
  };
  for (int len : {0, 1, 31, 32, 33, 64, 100, 200})
    for (int pmin = -40; pmin < 210; pmin += 7)
      for (int width : {0, 1, 5, 33})
        for (int window : {0, 1, 2, 31, 32, 33, 90, 1000, INT_MAX})
          for (int sinks : {0, 1, 32, 33, 64, 500, INT_MAX}) {
            const int pmax = pmin + width;
            const KeySpan s = key_span(pmin, pmax, len, window, sinks);
            is(s.sinks >= 0 && s.sinks <= s.from && s.from <= s.to && s.to <= (len + 31) / 32, "in order");
            std::set<int> groups;
            for (int i = 0; i < s.count(); ++i) groups.insert(s.group(i));
            is((int)groups.size() == s.count(), "each once");
            for (int p = pmin; p <= pmax; ++p)
              for (int j = 0; j < len; ++j)
                if (sees(p, j, window, sinks)) is(groups.count(j / 32) == 1, "a token that is seen");
            if (pmax < 0) is(s.count() == 0, "rows before the first token");
          }
  // the longest sequences and windows
  const KeySpan far = key_span(INT_MAX - 70000, INT_MAX - 69999, INT_MAX - 65536, INT_MAX, INT_MAX);
  is(far.from == 0 && far.to == (INT_MAX - 69999) / 32 + 1, "far");
  is(key_span(-(1 << 24), 5, 6, INT_MAX, 0).count() == 1, "before the first token, wide window");
""")


@needs_gxx
def test_touched_groups_bound(tmp_path):
    run(tmp_path, r"""
  for (int first = 0; first < 64; ++first)
    for (int n = 1; n < 200; ++n)
      is((first + n - 1) / 32 - first / 32 + 1 <= kv_touched_groups(1, n), "groups of one sequence");
""")


@needs_gxx
def test_join_slots(tmp_path):
    """A join's slots add up only slots that there are, every row has one that does, and
    no slot is added twice; heads of 96 leave slots over."""
    run(tmp_path, r"""
  for (int D : {64, 96, 128, 256})
    for (int waves : {4, 8}) {
      const int slots = 64 * waves / (D / 4);
      for (int rows = 1; rows <= 128; ++rows)
        for (int parts : {2, 3, 4, 8, 9, 16, 17, 100, 512}) {
          const JoinSlots j = join_slots(slots, rows, parts);
          is(j.share >= 1 && (j.share & (j.share - 1)) == 0 && j.share <= slots && j.rows() >= 1, "share");
          int leads = 0;
          // (threads behind the last slot have numbers too)
          for (int slot = 0; slot <= slots; ++slot)
            if (j.leads(slot)) {
              is(slot / j.share == leads++, "rows in order");
              is(slot + j.share <= slots, "adds up slots that there are");
            }
          is(leads == j.rows(), "a leader each");
        }
    }
""")


@needs_gxx
def test_launches_of_the_largest_batches(tmp_path):
    """A launch has fewer than 2^32 threads, whatever the batch; the groups' numbers fit an int."""
    run(tmp_path, r"""
  for (int heads : {1, 7, 8, 32, 4096}) {
    const long at_once = kv_groups_at_once(heads);
    is(at_once >= 1 && at_once * heads * kMoveThreads <= UINT32_MAX, "threads of a launch");
    is((at_once + 1) * heads * kMoveThreads > UINT32_MAX, "as many as fit");
  }
  is(kv_touched_groups(1 << 20, 1 << 24) < INT32_MAX / 2, "the largest batch");
""")


def test_null_handles():
    """Refused without a device."""
    L = nx.lib()
    out = nx._vp()
    assert L.nx_kv_create(None, nx.KV_F16, 1, 64, 1, 128, out) == nx.NX_ERR_INVALID_ARG
    assert b"null context" in L.nx_last_error()
    assert L.nx_kv_info(None, None, None, None, None, None, None) == nx.NX_ERR_INVALID_ARG
    assert L.nx_kv_destroy(None) == nx.NX_OK
    b = nx.KvBatch(1, 1, 1, 0, 0, 0)
    for f in (L.nx_kv_write, L.nx_kv_write_dev, L.nx_kv_read, L.nx_kv_read_dev):
        assert f(None, None, b.ref, None, None, 128) == nx.NX_ERR_INVALID_ARG
    for f in (L.nx_attention, L.nx_attention_dev):
        assert f(None, None, b.ref, None, 128, 1, 1.0, 0, 0, None, 128) == nx.NX_ERR_INVALID_ARG
