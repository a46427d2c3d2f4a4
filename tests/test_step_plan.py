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
