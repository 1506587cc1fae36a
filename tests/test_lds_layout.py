"""A kernel whose transfers write LDS has one object there, which therefore starts at
address 0: a transfer's LDS address is 16 bits, and the last buffer of the widest block
ends at 65536."""

import os

import pytest

from tests.test_wait_check import check_waits

OBJ = os.path.join(os.path.dirname(__file__), "..", "molla_amd", "csrc", "_obj")
KERNEL = "	.amdhsa_kernel _ZN2mi12_GLOBAL__N_1{}EvNS_7RowSegsEii\n		.amdhsa_group_segment_fixed_size {}\n	.end_amdhsa_kernel\n"
PREFILL, GROUP = "14prefill_kernelILi12ELi{}ELi{}ELi{}ELi{}EE", "12group_kernelILi14ELi{}ELi{}ELi{}ELi{}ELb0EE"


def run(name, size):
    return check_waits.check_lds(KERNEL.format(name, size).splitlines())


@pytest.mark.parametrize("name,size", [
    (PREFILL.format(1, 1, 4, 2), 32768), (PREFILL.format(2, 2, 4, 2), 65536), (GROUP.format(1, 1, 4, 2), 32768 + 256),
    (GROUP.format(1, 4, 8, 1), 131072 + 1024), (GROUP.format(2, 2, 4, 2), 65536 + 512)])
def test_one_object_passes(name, size):
    assert run(name, size) == (1, [])
    for other in (size + 4, size + 512, size - 256):
        seen, bad = run(name, other)
        assert seen == 1 and bad


def test_other_kernels_are_left_alone():
    assert run("19prefill_prep_kernelEPKfiiPh", 16) == (0, [])


@pytest.mark.parametrize("source", ["prefill", "experts_tile"])
def test_the_built_kernels(source):
    path = os.path.join(OBJ, f"{source}-hip-amdgcn-amd-amdhsa-gfx950.s")
    if not os.path.exists(path):
        pytest.skip("the library was not built here")
    with open(path) as f:
        seen, bad = check_waits.check_lds(f.read().splitlines())
    assert seen >= 24 and not bad, bad[:3]
