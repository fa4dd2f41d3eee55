"""The build refuses kernels of the matrix-core attention that spill registers."""
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "sparse-offload-infer_amd"
sys.path.insert(0, str(PKG))

import build  # noqa: E402

REMARK = """remark: a.hip:124:0: Function Name: {name} [-Rpass-analysis=kernel-resource-usage]
remark: a.hip:124:0:     TotalSGPRs: 79 [-Rpass-analysis=kernel-resource-usage]
remark: a.hip:124:0:     VGPRs: 256 [-Rpass-analysis=kernel-resource-usage]
remark: a.hip:124:0:     AGPRs: 172 [-Rpass-analysis=kernel-resource-usage]
remark: a.hip:124:0:     ScratchSize [bytes/lane]: {scratch} [-Rpass-analysis=kernel-resource-usage]
remark: a.hip:124:0:     SGPRs Spill: {sgpr} [-Rpass-analysis=kernel-resource-usage]
remark: a.hip:124:0:     VGPRs Spill: {vgpr} [-Rpass-analysis=kernel-resource-usage]
"""


def remarks(*kernels):
    return "".join(REMARK.format(**(dict(name=n, scratch=0, sgpr=0, vgpr=0) | d)) for n, d in kernels)


def test_what_counts_as_a_spill():
    assert build.spilling_kernels(remarks(("f", {}), ("g", {}))) == []
    for bad in (dict(scratch=16), dict(sgpr=3), dict(vgpr=1)):
        assert build.spilling_kernels(remarks(("f", {}), ("g", bad), ("h", {}))) == ["g"]


def test_remarks_that_are_missing_are_not_a_pass():
    for text in ("", "warning: something else\n", "remark: a.hip:1:0: Function Name: f [-Rpass-analysis=kernel-resource-usage]\n"):
        with pytest.raises(RuntimeError, match="remarks"):
            build.spilling_kernels(text)


def test_a_kernel_that_spills_fails_the_build(tmp_path):
    """64 accumulators of 16 registers where 4 waves share a SIMD's registers (128 each)."""
    src = tmp_path / "spill.hip"
    src.write_text("""#include <hip/hip_runtime.h>
extern "C" __global__ __launch_bounds__(256, 4) void spills(float* p, const float* q, int n) {
    float a[200];
    for (int i = 0; i < 200; ++i) a[i] = q[i * 256 + threadIdx.x];
    for (int k = 0; k < n; ++k)
#pragma unroll
        for (int i = 0; i < 200; ++i) a[i] = a[i] * a[(i * 7 + 3) % 200] + q[k];
    for (int i = 0; i < 200; ++i) p[i * 256 + threadIdx.x] = a[i];
}
""")
    out = tmp_path / "spill.o"
    with pytest.raises(RuntimeError, match="spills"):
        build.compile_hip(src, out, no_spills=True)
    assert not out.exists()
    build.compile_hip(src, out, no_spills=False)
    assert out.exists()


@pytest.mark.parametrize("source", build.NO_SPILLS)
def test_the_attention_kernels_do_not(source, tmp_path):
    build.compile_hip(build.CSRC / source, tmp_path / "k.o", no_spills=True)
    assert (tmp_path / "k.o").exists()
