"""expert_mm_rule.h compiled for the host: which kernel multiplies a call of the experts' products."""
import ctypes
import functools
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FORWARD, SWIGLU, ROWS, WEIGHTS = range(4)

SOURCE = r"""
#include "expert_mm_rule.h"
extern "C" int takes_few(int kind, int experts, int rows, int n, int k, int cus) { return esmoe::expert_mm_takes_few(kind, experts, rows, n, k, cus); }
"""


@functools.lru_cache(maxsize=None)
def _rule():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "rule.cpp"), os.path.join(d, "rule.so")
        with open(src, "w") as f:
            f.write(SOURCE)
        csrc = os.path.join(ROOT, "expert_specialization_moe_amd", "csrc")
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{csrc}", src, "-o", lib], check=True)
        return ctypes.CDLL(lib)


def takes_few(kind, experts, rows, n, k, cus):
    return bool(_rule().takes_few(kind, experts, rows, n, k, cus))


def only_large(experts, rows, n, k, kinds=(FORWARD, SWIGLU, ROWS, WEIGHTS)):
    """Whether all these forms of a call go to the large kernel on this device."""
    import torch

    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return not any(takes_few(kind, experts, rows, n, k, cus) for kind in kinds)
