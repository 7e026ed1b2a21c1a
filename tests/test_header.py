"""Programs in C and C++ that use include/hypno_hip.h's structs compile without a warning."""
import os
import subprocess

import pytest

from conftest import ROOT

SET_AND_READ = r"""
#include <hypno_hip.h>
float first_scale(const hypno_hip_kv_cache *c);
float first_scale(const hypno_hip_kv_cache *c) {
  const float *k = c->k_scale, *v = c->v_scale;  /* 8-bit caches */
  return k[0] + v[0];
}
void set(hypno_hip_kv_cache *c, float *scales, void *fp16_scales);
void set(hypno_hip_kv_cache *c, float *scales, void *fp16_scales) {
  hypno_hip_kv_cache i8 = {HYPNO_HIP_KV_INT8, 0, 0, scales, scales + 64, 1, 2, 32, 64, 0, 0, 0, 0};
  *c = i8;
  c->k_scale = scales;
  c->v_scale = c->k_scale + 64;
  if (c->dtype == HYPNO_HIP_KV_FP4) c->k_scale = (float *)fp16_scales;
}
"""


@pytest.mark.parametrize("compiler,std", [("gcc", "c99"), ("gcc", "c11"), ("g++", "c++11"),
                                          ("g++", "c++17")])
def test_scales_of_a_cache(compiler, std):
    p = subprocess.run([compiler, "-x", "c++" if compiler == "g++" else "c", f"-std={std}", "-Wall",
                        "-Wextra", "-Werror", "-fsyntax-only", f"-I{os.path.join(ROOT, 'include')}",
                        "-"], input=SET_AND_READ, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr
