"""Static check of the gfx950 assembly of the dense attention kernel that reads products'
results in inline asm: none earlier than the wait states that the compiler itself puts after
a builtin product of the same shape, on any control-flow path.  CPU only."""
import re
from pathlib import Path

import pytest

from ops_amd import build as sfa_build
from tests.test_isa_hazards import DRAIN, _device_asm, pytestmark, scan_result_reads  # noqa: F401

PROBE = """#include <hip/hip_runtime.h>
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
__global__ void probe(float* o, const bf16x8* a, const bf16x8* b) {
  f32x16 c = {};
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[threadIdx.x], b[threadIdx.x], c, 0, 0, 0);
  o[threadIdx.x] = c[0] * 3.0f;
}
"""


def _needed(tmp_path):
    src = tmp_path / "probe.hip"
    src.write_text(PROBE)
    lines = [l.strip() for l in _device_asm(src, tmp_path).split("\n") if l.startswith("\t")]
    i = next(j for j, l in enumerate(lines) if l.startswith("v_mfma_f32_32x32x16_bf16"))
    waits = 0
    for l in lines[i + 1:]:
        if l.startswith("v_"):
            return waits
        waits += int(l.split()[1]) + 1 if l.startswith("s_nop") else 1
    raise AssertionError("no VALU read after the probe MFMA")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    out = {}
    for stem in ("sfa_dense_wide", "sfa_dense_few", "sfa_dense_bwd"):
        src = [s for s in sfa_build.sources() if Path(s).stem == stem]
        assert len(src) == 1
        out[stem] = _device_asm(Path(src[0]), tmp_path_factory.mktemp(stem))
    return out


def test_no_early_reads_of_results(asm, tmp_path):
    need = _needed(tmp_path)
    assert 4 <= need <= DRAIN, need
    names = [n for n in re.findall(r"^(_Z\S+):", asm["sfa_dense_wide"], re.M) if "dense_wide_kernel" in n]
    assert len(names) == 8, names  # two head dims x two types x two forms of pages
    hits = scan_result_reads(asm["sfa_dense_wide"], kernels=("dense_wide_kernel",), drain=need)
    assert not hits, "\n".join(f"{k[-60:]}: {m}  ->  {r}" for k, m, r in hits[:10])


def test_rows_loaded_to_lds_do_not_wait_for_spills(asm):
    """No register of the kernels whose loops count their loads is spilled: a reload in a loop
    would wait for all of them.  (Forms for pages that hold whole tiles, 64 and 128 dims in the
    backward.)"""
    seen = {}
    for stem, pattern in (("sfa_dense_bwd", r"dense_(?:dq|dkv)_kernelI"), ("sfa_dense_few", r"dense_few_kernelI")):
        for m in re.finditer(r"\.name:\s+(_Z\S*" + pattern + r"\S*)(.*?)\.vgpr_spill_count:\s+(\d+)", asm[stem], re.S):
            seen[m.group(1)] = int(m.group(3))
    assert len(seen) >= 4 and not any(seen.values()), seen
