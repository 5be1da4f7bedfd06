"""Static check of the gfx950 assembly of the tree attention kernels whose MFMAs
are inline asm: no instruction reads a result earlier than the wait states that
the compiler itself puts after a builtin MFMA of the same shape (a probe compile
measures that number), on any control-flow path, and where pages hold whole
tiles no register is spilled (a reload would wait for the loads to LDS in flight).  CPU only."""
import re
from pathlib import Path

import pytest

from ops_amd import build as sfa_build
from tests.test_isa_hazards import DRAIN, _device_asm, pytestmark, scan_result_reads  # noqa: F401

KERNELS = ("tree_pipe_kernel", "tree_mla_kernel")

PROBE = """#include <hip/hip_runtime.h>
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
__global__ void probe(float* o, const bf16x8* a, const bf16x8* b) {
  f32x4 c = {};
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[threadIdx.x], b[threadIdx.x], c, 0, 0, 0);
  o[threadIdx.x] = c[0] * 3.0f;
}
"""


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    src = [s for s in sfa_build.sources() if Path(s).stem == "sfa_tree"]
    assert len(src) == 1
    return _device_asm(Path(src[0]), tmp_path_factory.mktemp("tree"))


def _needed(tmp_path):
    src = tmp_path / "probe.hip"
    src.write_text(PROBE)
    lines = [l.strip() for l in _device_asm(src, tmp_path).split("\n") if l.startswith("\t")]
    i = next(j for j, l in enumerate(lines) if l.startswith("v_mfma_f32_16x16x32_bf16"))
    waits = 0
    for l in lines[i + 1:]:
        if l.startswith("v_"):
            return waits
        waits += int(l.split()[1]) + 1 if l.startswith("s_nop") else 1
    raise AssertionError("no VALU read after the probe MFMA")


def test_no_early_reads_of_results(asm, tmp_path):
    need = _needed(tmp_path)
    assert 4 <= need <= DRAIN, need
    names = [n for n in re.findall(r"^(_Z\S+):", asm, re.M) if any(k in n for k in KERNELS)]
    assert len(names) == 10, names  # two row counts x two head dims x two page forms, and the latent rows' two
    hits = scan_result_reads(asm, kernels=KERNELS, drain=need)
    assert not hits, "\n".join(f"{k[-60:]}: {m}  ->  {r}" for k, m, r in hits[:10])


def test_scanner_sees_these_kernels():
    planted = ("_Ztree_pipe_kernel_planted:\n\tv_mfma_f32_16x16x32_bf16 v[0:3], v[16:19], a[0:3], 0\n"
               "\tv_max_f32_e32 v20, v3, v3\n.Lfunc_end0:\n")
    assert [h[2] for h in scan_result_reads(planted, kernels=KERNELS, drain=8)] == ["v_max_f32_e32 v20, v3, v3"]


def test_no_spills(asm):
    """(of the forms for pages that hold whole tiles)"""
    seen = 0
    for m in re.finditer(r"\.name:\s+(_Z\S*tree_(?:pipe|mla)_kernelI\S*Lb1EE\S*)(.*?)\.vgpr_spill_count:\s+(\d+)", asm, re.S):
        seen += 1
        assert m.group(3) == "0", m.group(1)
    assert seen == 5
