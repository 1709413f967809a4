"""Order of programmatic launches and tensor memory, read from the kernels' source: ``tcgen05.alloc`` is the library's
one wait without a limit, and some kernels allocate before they wait for their predecessor. So a kernel may release
its dependents (``griddep_launch_dependents``) only once its own block holds its columns: a successor that took them
first would wait for a predecessor that waits for them."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "mlx-generate-ctmr_b200" / "csrc"


def _kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for part in re.split(r"__global__", text)[1:]:
            body = part[:part.find("\n}\n")]
            name = re.search(r"(\w+_kernel\w*)\s*\(", body)
            if "tmem_alloc" in body:
                yield pytest.param(body, id=f"{path.stem}-{name.group(1) if name else '?'}")


KERNELS = list(_kernels())


def test_the_kernels_are_found():
    assert len(KERNELS) >= 7


@pytest.mark.parametrize("body", KERNELS)
def test_dependents_are_released_after_the_allocation(body):
    alloc, freed = body.index("tmem_alloc"), body.find("griddep_launch_dependents")
    assert freed > alloc
    assert "__syncthreads()" in body[alloc:freed]  # all of the block's warps are past it


@pytest.mark.parametrize("name", ["attention_packed", "adapter_linear"])
def test_warps_meet_between_a_wait_and_tensor_memory(name):
    """``tcgen05.ld`` and ``.st`` are for a whole warp at once; a wait that each lane leaves by itself does not
    bring the lanes back together, ``mbar_wait_warp`` does."""
    text = re.sub(r"//[^\n]*", "", (CSRC / f"{name}.cu").read_text())
    loads = [m.start() for m in re.finditer(r"tmem_ld(16|32)\(", text)]
    assert len(loads) >= 3
    for at in loads:
        assert re.findall(r"mbar_wait_\w+", text[:at])[-1] == "mbar_wait_warp"


@pytest.mark.parametrize("path", [p for p in sorted(CSRC.glob("*.cu")) if "tmem_ld" in p.read_text()], ids=lambda p: p.stem)
def test_accumulators_are_waited_for_by_whole_warps(path):
    """The barriers that announce an accumulator are waited for by the warps that then read it."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    assert not re.findall(r"mbar_wait_bounded\(\s*&?(?:tmem_full|o_full|s_full|acc_full|chunk_full)\b", text)


def test_warps_meet_before_sums_are_read_out():
    """The same for loads that are started and waited for apart (``tmem_ld16_start``)."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "scaled_linear.cu").read_text())
    loads = [m.start() for m in re.finditer(r"tmem_ld16_start\(", text)]
    assert len(loads) >= 3
    for at in loads:
        assert re.findall(r"mbar_wait_\w+", text[:at])[-1] == "mbar_wait_warp"
        # What a load gives is read after a wait for it, tied to that place.
        assert re.search(r"tmem_ld_wait\(\);\s*tmem_ld_fence16\(", text[at:])
