"""What the calls around a step's cache accept and how they share their work out
(nexus_amd/csrc/nx_step_plan.hpp), on the CPU: the header is plain C++."""
import subprocess

from test_kv_plan import CSRC, GXX, needs_gxx


def run(tmp_path, body):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text('#include <cstdio>\n#include "nx_step_plan.hpp"\nusing namespace nx;\n'
                   "int bad = 0;\n"
                   "void is(bool ok, const char *what) { if (!ok) { std::printf(\"%s\\n\", what); ++bad; } }\n"
                   "int main() {\n" + body + "\n  return bad ? 1 : 0;\n}\n")
    r = subprocess.run([GXX, "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, f"exit {r.returncode}\n{r.stdout[-2000:]}"


@needs_gxx
def test_rows_overlap(tmp_path):
    run(tmp_path, r"""
  static float m[4096];
  auto o = [&](long a, size_t sa, size_t wa, long b, size_t sb, size_t wb, long rows) {
    const bool x = rows_overlap(m + a, sa, wa, m + b, sb, wb, rows);
    is(x == rows_overlap(m + b, sb, wb, m + a, sa, wa, rows), "symmetric");
    return x;
  };
  is(!o(0, 64, 16, 16, 64, 16, 8) && !o(0, 64, 16, 48, 64, 16, 8), "beside each other");
  is(o(0, 64, 17, 16, 64, 16, 8) && o(0, 64, 16, 49, 64, 16, 8), "into each other, and around the end");
  is(o(0, 64, 16, 128, 64, 16, 8) && o(0, 64, 16, 130, 64, 16, 8), "later rows");
  is(!o(0, 64, 16, 512, 64, 16, 8), "behind");
  is(o(0, 64, 16, 16, 80, 16, 8) && !o(0, 64, 16, 464, 80, 16, 8), "two strides");
  is(!o(0, 64, 16, 16, 80, 16, 1) && o(0, 64, 17, 16, 80, 16, 1), "one row");
  is(!o(0, 64, 0, 0, 64, 16, 8) && !o(0, 64, 16, 0, 64, 16, 0), "nothing");
  is(!rows_overlap(nullptr, 64, 16, m, 64, 16, 4), "null");
  is(rows_overlap(m, (size_t)1 << 40, 16, m + 1, (size_t)1 << 40, 16, 1 << 24), "past 64 bits of bytes");
""")


@needs_gxx
def test_every_logit_has_one_part(tmp_path):
    run(tmp_path, r"""
  for (int rows : {1, 2, 3, 7, 61, 300, 1023, 1024, 1025, 2047, 2048, 2049, 5000, 1 << 24})
    for (int vocab : {1, 2, 3, 4, 5, 1000, 1024, 1025, 2048, 2049, 4096, 32000, 100003, 131072, 200000, 1 << 30}) {
      const RowSplit s = logprob_split(rows, vocab);
      is(s.parts >= 1 && s.parts <= kLogprobParts && s.share % 4 == 0 && s.share > 0, "sizes");
      is((long)s.parts * s.share >= vocab && (long)(s.parts - 1) * s.share < vocab, "all, none empty");
      is(s.parts == 1 || (long)s.parts * rows <= kLogprobWgs, "the workspace has a record for each");
    }
""")


@needs_gxx
def test_gathered_weights_fit_their_workspace(tmp_path):
    run(tmp_path, r"""
  int slices = 0;
  for (int seqs : {1, 2, 17, 61, 300, 1 << 20})
    for (int rows : {1, 2, 5, 64, 300, 4093, 100000, 1 << 24})
      for (int kv_heads : {1, 2, 8, 12, 4096})
        for (int group : {1, 3, 4, 24})
          for (int groups : {1, 2, 17, 128, 1001, 4096, 200000, 67000000}) {
            const long heads = (long)kv_heads * group;
            if (rows * heads > INT32_MAX) continue;
            for (bool one : {false, true}) {
              const MassNarrow n = mass_narrow(seqs, rows, group, kv_heads, groups, one);
              is(n.heads >= 0 && n.heads <= kv_heads, "heads");
              if (n.heads == 0) continue;
              is(n.slots * ((size_t)groups * 32 + 2 * (size_t)n.chunks) <= kMassFloats, "scores fit");
              is((long)n.share * n.chunks >= groups && (long)n.share * (n.chunks - 1) < groups && n.share <= 64, "chunks");
              is((long)n.add_share * n.add_chunks >= groups && n.add_share <= 64 && n.add_chunks <= n.chunks, "sums");
              is((long)n.tiles * n.chunks * 256 < 1L << 32 && (long)seqs * n.heads * n.chunks * 256 < 1L << 32, "launch");
              is(n.slots >= (one ? (size_t)seqs * 16 : (size_t)rows * group) * n.heads, "rows");
              is(n.tiles >= (one ? (long)seqs : (long)rows * group / 16 + (seqs < rows ? seqs : 0)) * n.heads, "tiles");
            }
            for (int D : {64, 256}) {
              const MassWide w = mass_wide(seqs, rows, (int)heads, kv_heads, groups, D == 256 ? 4 : 8, D);
              slices += w.rows < rows;
              is(w.rows >= 1 && w.rows <= rows && w.query >= (size_t)w.rows * heads && w.query % 4 == 0, "rows");
              const long room = (long)kMassFloats - (long)w.query * (D + 2);
              is(room >= 0, "halves fit");
              is(w.key_parts == 1 || (long)w.rows * heads * w.key_parts * 2 <= room, "statistics fit");
              is((long)w.key_share * w.key_parts >= groups && (long)w.key_share * (w.key_parts - 1) < groups, "keys");
              is(w.row_parts == 1 || (long)seqs * kv_heads * w.row_parts * groups * 32 <= room, "sums fit");
              // a sequence's last tile may be short
              is(w.key_units >= kv_heads * ((long)w.rows * group / 128 + std::min(seqs, w.rows)) * w.key_parts, "units");
              const long blocks = ((long)w.rows * group + 31) / 32;
              // sequences of one row but for one, and of as many rows each
              const long most = std::min(seqs, w.rows), each = std::max(1, w.rows / seqs);
              auto parts = [&](long n) { return ((n * group + 31) / 32 + w.row_share - 1) / w.row_share; };
              const long tiles = kv_heads * (((long)groups + (D == 256 ? 3 : 7)) / (D == 256 ? 4 : 8));
              is(w.column_units >= tiles * ((most - 1) * parts(1) + parts(w.rows - most + 1)), "columns of one long");
              is(w.column_units >= tiles * most * parts(each), "columns of even ones");
              is((long)w.row_share * w.row_parts >= blocks && (long)w.row_share * (w.row_parts - 1) < blocks, "rows' parts");
            }
          }
  is(slices > 0, "some calls are in slices");
""")


@needs_gxx
def test_refusals(tmp_path):
    run(tmp_path, r"""
  static float m[1 << 16];
  static int32_t i[64];
  nx_rope r{64, 64, NX_ROPE_HALVES, 1e-6f, m, nullptr, nullptr};
  const RopeRows x{m, m + 512, m, m + 512, 1024, 1024, 1024, 1024};
  auto rope = [&](nx_rope q, int rows, int heads, int kv, RopeRows y) { return rope_check(&q, i, rows, heads, kv, y).code; };
  is(rope(r, 4, 8, 2, x) == NX_OK && rope(r, 0, 8, 2, {}) == NX_OK && rope(r, 4, 0, 0, {}) == NX_OK, "taken");
  is(rope_check(nullptr, i, 4, 8, 2, x).code == NX_ERR_INVALID_ARG, "null");
  is(rope_check(&r, nullptr, 4, 8, 2, x).code == NX_ERR_INVALID_ARG, "no positions");
  nx_rope still = r;
  still.rotary_dim = 0;
  is(rope_check(&still, nullptr, 4, 8, 2, x).code == NX_OK, "none needed");
  is(rope(r, 4, 9, 2, x) == NX_ERR_INVALID_ARG, "queries into keys");
  is(rope(r, 4, 17, 2, x) == NX_ERR_SHAPE, "rows overlap");
  is(rope(r, (1 << 24) + 1, 8, 2, x) == NX_ERR_UNSUPPORTED, "rows");
  RopeRows y = x;
  y.q_out = m + 4;
  is(rope(r, 4, 8, 2, y) == NX_ERR_INVALID_ARG, "beside itself");
  y.q_out = m + 8192, y.k_out = m + 8192 + 512;
  is(rope(r, 4, 8, 2, y) == NX_OK, "elsewhere");
  y.k_out = m + 8192 + 500;
  is(rope(r, 4, 8, 2, y) == NX_ERR_INVALID_ARG, "outputs into each other");

  auto lp = [&](size_t stride, int rows, int vocab, int given, int top) {
    return logprobs_check(m, stride, rows, vocab, i, given, m, top, i, m).code;
  };
  is(lp(64, 4, 64, 1, 64) == NX_OK && lp(64, 4, 64, 0, 0) == NX_OK, "taken");
  is(lp(63, 4, 64, 1, 4) == NX_ERR_SHAPE && lp(64, 4, 0, 1, 4) == NX_ERR_INVALID_ARG, "vocab");
  is(lp(64, 4, 64, 1, 65) == NX_ERR_UNSUPPORTED && lp((size_t)1 << 41, 4, 64, 1, 1) == NX_ERR_UNSUPPORTED, "sizes");
  is(lp((size_t)1 << 40, 4, 1 << 30, 1, 1) == NX_OK && lp((size_t)1 << 40, 4, (1 << 30) + 1, 1, 1) == NX_ERR_UNSUPPORTED,
     "logits");

  int32_t len[2] = {100, 50}, pages[8] = {0, 1, 2, 3, 4, 5, -1, -1}, to[4] = {6, 7, 8, 9};
  nx_kv_batch b{2, 0, 4, nullptr, len, pages};
  EvictArgs a{to, 2, 40, 4, 8, m, 100, i, i, m + 4096, 40};
  auto evict = [&](EvictArgs e) { return evict_check(&b, 32, 2, e).code; };
  auto tables = [&](EvictArgs e, int num = 10) { return evict_check_tables(b, num, 32, e).code; };
  is(evict(a) == NX_OK && tables(a) == NX_OK, "taken");
  EvictArgs e = a;
  e.sinks = 33;
  is(evict(e) == NX_ERR_SHAPE, "more than are kept");
  e.sinks = INT32_MAX, e.recent = INT32_MAX;
  is(evict(e) == NX_ERR_SHAPE, "past 31 bits");
  e = a, e.new_mass = m + 300;
  is(evict(e) == NX_ERR_INVALID_ARG, "over the old ones");
  e.new_mass = m + 400;
  is(evict(e) == NX_OK, "behind the old ones");
  for (int off : {-1, 0, 1}) {
    e = a, e.new_len = len + off;
    is(evict(e) == NX_ERR_INVALID_ARG, "lengths in place");
  }
  e = a, e.mass_stride = 99;
  is(evict(e) == NX_OK && tables(e) == NX_ERR_SHAPE, "fewer weights than tokens");
  is(tables(a, 9) == NX_ERR_INVALID_ARG && tables(a, 3) == NX_ERR_INVALID_ARG, "pages");
  for (int32_t bad : {7, 0, 5, -1, 10}) {
    to[2] = bad;
    is(tables(a) == NX_ERR_INVALID_ARG, "in use, or none");
  }
  to[2] = 8;
  len[0] = 129;
  is(tables(a) == NX_ERR_SHAPE, "longer than its pages");
  len[0] = -1;
  is(tables(a) == NX_ERR_SHAPE, "below 0");
  len[0] = 0, len[1] = 0;
  is(tables(a) == NX_OK, "no tokens");

  nx_kv_batch s{2, 3, 4, i, len, pages};
  auto mass = [&](int heads, size_t stride, const float *before, const float *out, size_t ms) {
    return mass_check(&s, 2, heads, stride, heads * 64, m, before, out, ms).code;
  };
  is(mass(4, 256, nullptr, m, 100) == NX_OK && mass(4, 256, m, m, 100) == NX_OK, "taken");
  is(mass(4, 256, m, m + 100, 100) == NX_ERR_INVALID_ARG && mass(4, 256, m, m + 400, 100) == NX_OK, "in part");
  is(mass(4, 255, nullptr, m, 100) == NX_ERR_SHAPE && mass(4, 256, nullptr, m, 0) == NX_ERR_SHAPE, "strides");
  s.num_tokens = 1 << 24;
  is(mass(256, 256 * 64, nullptr, m, 100) == NX_ERR_UNSUPPORTED, "rows");
""")
