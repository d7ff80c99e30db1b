"""The fused SVGD step reads its coefficients from scalar registers, not one by one from lanes they were parked in: counted in the
compiler's output (the kernels build without a GPU)."""
import os
import re
import subprocess

import pytest

from tools import resource_usage

CSRC = resource_usage.CSRC


def kernels(source, tmp_path):
    out = os.path.join(str(tmp_path), "out.s")
    flags = [f for f in resource_usage.FLAGS if not f.startswith("-Rpass")]
    subprocess.run([resource_usage.HIPCC] + flags + ["--offload-device-only", "-S", os.path.join(CSRC, source), "-o", out], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    text = open(out).read()
    for name in re.findall(r"^(_ZN3bde17svgd_fused_kernel\S+):", text, re.M):
        body = text[text.index("\n" + name + ":"):]
        yield name, body[:body.index("s_endpgm")]


@pytest.mark.skipif(not os.path.exists(resource_usage.HIPCC), reason="no HIP compiler")
def test_the_fused_sgd_step_does_not_read_a_parked_lane_per_product(tmp_path):
    """2 M^2 coefficients do not fit the scalar registers at M >= 8; what does not is parked.  Wanted once per particle's terms, each
    comes back at most once for four products (plus what the scalar tail and the pointers need), not once for each product."""
    seen = 0
    for name, body in kernels("svgd_fused.hip", tmp_path):
        m, opt = (int(x) for x in re.match(r"_ZN3bde17svgd_fused_kernelILi(\d+)ELi(\d)", name).groups())
        if opt != 0:
            continue
        seen += 1
        lanes, products = len(re.findall(r"\bv_readlane", body)), len(re.findall(r"\bv_fma", body))
        assert lanes <= products, f"M = {m}: {lanes} lane reads for {products} products ({name})"
    assert seen == 48                                   # 16 particle counts, flat and segmented, and 8 of them with the Gram twice
