"""Arithmetic that the paged-cache kernels share between host and device, compiled for the host."""
import ctypes as C
import random
import subprocess

import pytest

from thor_megakernels_b200 import build

HARNESS = """
#include "paged_attention.cuh"
using namespace mk::paged;
extern "C" void fill(uint32_t stage, uint32_t parity, uint32_t k, uint32_t stages, uint32_t *out) {
    const RingFill f = ring_fill(stage, parity, k, stages);
    out[0] = f.stage;
    out[1] = f.parity;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    at = tmp_path_factory.mktemp("host")
    (at / "host.cu").write_text(HARNESS)
    subprocess.run([build.find_nvcc(), *build.NVCC_FLAGS, f"-I{build.CSRC}", "-shared", "-o", str(at / "host.so"), str(at / "host.cu")], check=True)
    return C.CDLL(str(at / "host.so"))


@pytest.mark.parametrize("stages", [2, 4])
def test_fills_under_way_are_found(host, stages):
    """The few-row kernel's ring, filled and consumed at random: what a warp that gives up has to wait for."""
    rng = random.Random(stages)
    stage = parity = fill = 0
    fills, under_way = [0] * stages, []   # per stage; (stage, phase) of those not consumed, oldest first
    out = (C.c_uint32 * 2)()
    for _ in range(500):
        while len(under_way) < stages and rng.random() < 0.7:
            under_way.append((fill, fills[fill]))
            fills[fill] += 1
            fill = (fill + 1) % stages
        for k, (at, phase) in enumerate(under_way):
            host.fill(stage, parity, k, stages, out)
            assert (out[0], out[1]) == (at, phase & 1)
        if under_way and rng.random() < 0.6:
            assert under_way.pop(0)[0] == stage
            stage += 1
            if stage == stages:
                stage, parity = 0, parity ^ 1
