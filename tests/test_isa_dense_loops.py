"""Static check of the gfx950 assembly of dense attention of many rows: where pages hold whole
tiles of bf16 rows, and at 64 dims in every form, its loops reload no spilled register (a
reload waits for every load in flight, which they count).  CPU only."""
import re
from pathlib import Path

from ops_amd import build as sfa_build
from tests.test_isa_hazards import _device_asm, pytestmark  # noqa: F401


def _reloads_in_loops(body):
    block, n = "", 0
    for line in body.split("\n"):
        if re.match(r"(\.LBB|; %bb)", line):
            block = line
        elif "scratch_load" in line and "Loop" in block:
            n += 1
    return n


def test_no_reloads_in_the_loops_of_many_rows(tmp_path):
    src, = [s for s in sfa_build.sources() if Path(s).stem == "sfa_dense_wide"]
    asm = _device_asm(Path(src), tmp_path)
    seen = {}
    for m in re.finditer(r"^_Z\S*dense_wide_kernelI(\S+)Ev\S*:(.*?)^\.Lfunc_end", asm, re.S | re.M):
        seen[m.group(1)] = _reloads_in_loops(m.group(2))
    assert len(seen) == 8, seen  # head dims x types x forms of pages
    none = [k for k in seen if k.startswith("Li64E") or k == "Li128ELb0ELb1EE"]
    assert len(none) == 5 and not any(seen[k] for k in none), seen
