"""The lengths that attention over a cache cuts its keys into are worked out anew in the tile
kernels and in the join kernel. They must not depend on what the compiler contracts into fused
products and sums: the same source, compiled for the host with every contraction that the
library's own flags allow and with none, gives the same lengths."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _lines(tmp_path, contract):
    out = str(tmp_path / contract)
    subprocess.run([HIPCC, "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-O3", "-std=c++17", "-mfma",
                    f"-ffp-contract={contract}", "-I", os.path.join(ROOT, "qwen-image.cu_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "cache_ranges.cpp"), "-o", out], check=True)
    return subprocess.run([out], check=True, stdout=subprocess.PIPE, text=True).stdout.splitlines()


def test_lengths_do_not_depend_on_contraction(tmp_path):
    if " fma " not in open("/proc/cpuinfo").read():
        pytest.skip("needs a host with fused products")
    fused, plain = _lines(tmp_path, "fast-honor-pragmas"), _lines(tmp_path, "off")
    assert len(plain) == 2000
    assert fused == plain
