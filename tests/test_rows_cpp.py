"""The row operators' C++ header, checked by the compiler: a caller compiles and
links against the public headers and libraries, and its refusals (made on the
host before any device call) arrive as the documented exceptions."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "powersparse_amd", "lib")

SOURCE = r"""
#include <cstdio>
#include <type_traits>

#include "PowerSparse_Rows.h"

using namespace PowerSparse;

static_assert(!std::is_copy_constructible<GradientList>::value, "");

// what a training step calls (not run here: it needs a GPU)
void Step(const ps_rows& table, const ps_ids& ids, const ps_rows& x, const ps_rows& xs,
          const ps_rows& y, const ps_rows& grad, int* order, int* position, int* offsets,
          float* weights, float* dweights, void* work, size_t bytes, const GradientList& list,
          float* norm) {
  EmbeddingLookup(table, ids, 2.f, x);
  ExpertSort(ids, 8, order, position, offsets, work, bytes);
  ExpertDispatch(x, position, 2, xs);
  ExpertCombine(xs, position, weights, 2, y);
  ExpertCombineGrad(y, xs, position, weights, 2, xs, dweights);
  ExpertDispatchGrad(xs, position, 2, x);
  EmbeddingGrad(ids, x, 2.f, grad, work, bytes);
  list.Norm(norm);
  list.Clip(1.f, norm);
  list.ClipNorm(1.f, norm);
}

template <typename F>
bool Refused(F f) {
  try {
    f();
  } catch (const std::invalid_argument& e) {
    std::printf("%s\n", e.what());
    return true;
  }
  return false;
}

int main(int argc, char**) {
  char* const far = reinterpret_cast<char*>(1ull << 32);  // never followed
  const ps_rows a{far, 4, 8, 8, PS_F32}, wrong{far + (1 << 20), 4, 9, 9, PS_F32};
  const ps_ids ids{far + (1 << 21), 4, PS_I32};
  if (argc > 100) Step(a, ids, a, a, a, a, 0, 0, 0, 0, 0, 0, 0, GradientList({}), 0);
  const bool ok = Refused([&] { EmbeddingLookup(a, ids, 1.f, wrong); }) &&
                  Refused([&] { EmbeddingGrad(ids, a, 1.f, wrong, far, 1 << 20); }) &&
                  Refused([&] { ExpertSort(ids, 0, nullptr, nullptr, nullptr, far, 0); }) &&
                  Refused([&] { ExpertCombine(a, nullptr, nullptr, 1, a); }) &&
                  Refused([&] { GradientList({{far, 4, PS_F32}}, {{far, 5, PS_F32}}); }) &&
                  Refused([&] { GradientList({{far, 4, 7}}); });
  return ok ? 0 : 1;
}
"""


def test_caller_compiles_links_and_is_refused(tmp_path):
    if not os.path.exists(os.path.join(LIB, "libpowersparse.so")):
        pytest.skip("host library not built")
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    src, exe = tmp_path / "caller.cpp", tmp_path / "caller"
    src.write_text(SOURCE)
    cmd = [cxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I" + os.path.join(ROOT, "include"),
           "-I" + os.path.join(ROOT, "powersparse_amd", "host"), str(src), "-o", str(exe),
           "-L" + LIB, "-lpowersparse", "-lpowersparse_hip", "-Wl,-rpath," + LIB]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert len(r.stdout.splitlines()) == 6
