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
extern "C" int held(long long length, int max_pages, int page_shift) { return held_length(length, max_pages, page_shift); }
extern "C" int tiles(int length, int count, int group, int rows, int rb, int tile) {
    return block_tiles(length, count, fast_div(group), rows, rb, tile);
}
extern "C" int units(int length, int count, int group, int rows, int tile, int extra, int kv_heads) {
    return sequence_units(length, count, fast_div(group), Cut{rows, tile, extra}, kv_heads);
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


@pytest.mark.parametrize("tile", [64, 128])
@pytest.mark.parametrize("length", [1, 63, 64, 65, 2 ** 20, 2 ** 31 - 65537, 2 ** 31 - 65536, 2 ** 31 - 129, 2 ** 31 - 64, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 40])
def test_lengths_up_to_the_largest_int(host, length, tile):
    """A table of 2^24 pages of 128 holds more positions than an int counts: no length makes its tiles negative."""
    host.held.argtypes = [C.c_longlong, C.c_int, C.c_int]
    held = host.held(length, 2 ** 24 + 3, 7)
    assert held == min(length, 2 ** 31 - 65536)
    want = -(-held // tile)
    assert host.tiles(held, 1, 4, 8, 0, tile) == want
    assert host.units(held, 1, 4, 8, tile, 1, 8) == 8 * (want + 1)
    assert host.held(length, 10, 4) == min(length, 160)
    assert host.held(-length, 10, 4) == 0
