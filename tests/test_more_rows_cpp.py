"""The C++ header's layer norm, router and AdamW, checked by the compiler: a caller compiles and
links against the public headers and libraries, and its refusals (made on the host before any
device call) arrive as the documented exceptions."""
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

static_assert(!std::is_copy_constructible<AdamWList>::value, "");

// what a training step calls (not run here: it needs a GPU)
void Step(const ps_rows& x, const ps_rows& y, const ps_rows& w, const ps_rows& logits, float* mean,
          float* rstd, int* ids, float* weights, int* counts, float* loss, void* work, size_t bytes,
          const AdamWList& list) {
  LayerNorm(x, &w, nullptr, 1e-5f, y);
  LayerNorm(x, &w, &w, 1e-5f, y, mean, rstd);
  ExpertRoute(logits, 2, ids, weights);
  ExpertRoute(logits, 2, ids, weights, counts, loss, work, bytes, nullptr, false);
  ExpertRouteGrad(logits, 2, ids, weights, counts, loss, logits);
  LayerNormGrad(y, x, &w, mean, rstd, x, &w, nullptr, work, bytes, true);
  ps_adamw_options o{};
  o.lr = 1e-3;
  o.beta1 = 0.9;
  o.beta2 = 0.999;
  o.eps = 1e-8;
  o.step = 1;
  o.grad_scale = 1.f;
  list.Step(o);
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
  float* const f = reinterpret_cast<float*>(far + (1 << 21));
  int* const i = reinterpret_cast<int*>(far + (1 << 22));
  if (argc > 100) Step(a, a, a, a, f, f, i, f, i, f, far, 0, AdamWList({}));
  ps_adamw_tensor t{};
  t.count = 4;
  const bool ok = Refused([&] { LayerNorm(a, nullptr, nullptr, 1e-5f, wrong); }) &&
                  Refused([&] { LayerNorm(a, &a, nullptr, 1e-5f, a); }) &&
                  Refused([&] { LayerNormGrad(a, a, nullptr, f, f, wrong, nullptr, nullptr, nullptr, 0); }) &&
                  Refused([&] { ExpertRoute(a, 9, i, f); }) &&
                  Refused([&] { ExpertRouteGrad(a, 2, i, f, nullptr, f, wrong); }) &&
                  Refused([&] { AdamWList({t}); }) &&
                  Refused([&] { AdamWList({}, PS_BF16); });
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
    assert len(r.stdout.splitlines()) == 7
