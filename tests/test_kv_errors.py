"""Exceptions of the cache's and the attention's C entries (guarded, nx_kv_plan.hpp), on the
CPU: they become errors with a message of their own."""
import subprocess

from test_kv_plan import CSRC, GXX, needs_gxx

SOURCE = r"""
#include "nx_kv_plan.hpp"
static std::string last;
int nx::fail(int code, const std::string &msg) { last = msg; return code; }
using nx::guarded;
int main() {
  int bad = 0;
  last = "an earlier call's";
  bad += guarded([]() -> int { throw std::bad_alloc(); }) != NX_ERR_OOM || last != "out of memory";
  bad += guarded([]() -> int { throw 1; }) != NX_ERR_DEVICE || last != "internal error";
  bad += guarded([] { return nx::fail(NX_ERR_SHAPE, "why"); }) != NX_ERR_SHAPE || last != "why";
  bad += guarded([] { return 0; }) != 0;
  return bad;
}
"""


@needs_gxx
def test_exceptions_are_errors_with_messages(tmp_path):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(SOURCE)
    r = subprocess.run([GXX, "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(exe)]).returncode == 0
