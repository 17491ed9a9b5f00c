"""CPU: limits and scales that only the GPU knows are for the launch of two products; every other launch refuses them before it
touches a device, instead of dropping them."""
import importlib
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "intel-extension-for-openxla_b200")

PROBE = r'''
#include <stdio.h>
#include "gemm_sm100.h"
using namespace ixk;
int main() {
  int limit = 1;
  float scale = 2.0f;
  for (int which = 0; which < 3; ++which) {
    gemm::Problem p;
    p.kind = gemm::kKindF16;
    p.ab_dtype = IXK_BF16;
    p.M = 16, p.N = 64, p.K = 64;
    if (which == 0) p.acc_scale_dev = &scale;
    if (which == 1) p.m_limit = &limit;
    if (which == 2) p.k_limit = &limit;
    DeviceInfo dev;
    dev.sm_count = 148;
    printf("%d %d %d\n", gemm::launch(p, dev, nullptr), gemm::launch_stream(p, 1, nullptr, dev, nullptr),
           gemm::run_problem(p, nullptr, 0, dev, nullptr));
  }
}
'''


def test_other_launches_refuse_what_only_the_gpu_knows(pkg):
    lib = pkg.load_library()._name
    nvcc = importlib.import_module(pkg.__name__ + ".build")._nvcc()
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.cu"), os.path.join(d, "probe")
        with open(src, "w") as f:
            f.write(PROBE)
        subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr",
                        "-I", os.path.join(ROOT, "include"), "-I", os.path.join(PACKAGE, "csrc"), src, "-o", exe, lib], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True, env={**os.environ, "LD_LIBRARY_PATH": os.path.dirname(lib)}).stdout
    assert out.split() == [str(pkg.IXK_INVALID_ARGUMENT)] * 9
