"""Products of 8-bit rows: what every workgroup of a launch reads and makes, asked of the functions that the kernels themselves call, without a GPU: every block of the
result is made once by every part of k, the parts go through all of k, and every byte that is loaded, and every byte of the workspace, lies in its operand. (Not followed
here: the kernel that adds parts, the rows' and packing kernels, and the stores of the results, which check each row and column that they write.)"""
import ctypes
import random

import numpy as np
import pytest

MODES = {"store": 0, "add": 1, "gated": 2}
MOST_K = 131071
NOTHING = (2 ** 63 - 1, 0)


@pytest.fixture(scope="module")
def lib():
    from xeno_rt_amd.ops import build
    made = ctypes.CDLL(build.find_library() or build.build())
    made.xrt_linear_int8_workspace.restype = made.xrt_int8_stride.restype = made.xrt_int8_packed_rows.restype = ctypes.c_long
    made.xrt_linear_int8_reach.argtypes = [ctypes.c_int] * 4 + [ctypes.c_long, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    return made


class Reach:
    """What workgroup `number` of a product reaches."""

    def __init__(self, lib, m, n, k, mode, number):
        reach, room = np.zeros(14, dtype=np.int64), 512
        made = np.zeros((room, 3), dtype=np.int32)
        assert lib.xrt_linear_int8_reach(m, n, k, MODES[mode], number, reach.ctypes.data, made.ctypes.data, room) == 0
        self.a, self.w, self.a_scales, self.w_scales, self.sums = ((int(reach[2 * i]), int(reach[2 * i + 1])) for i in range(5))
        self.workgroups, self.parts, self.steps, count = (int(reach[i]) for i in range(10, 14))
        assert count <= room
        self.made = made[:count]


def inside(span, size):
    return span == NOTHING or 0 <= span[0] < span[1] <= size


def sizes(seed, count):
    spread = random.Random(seed)
    near = lambda low, high: min(high, max(low, int(round(2 ** spread.uniform(np.log2(low), np.log2(high))))))     # noqa: E731
    for _ in range(count):
        yield near(1, 6000), near(1, 12000), near(1, 20000), spread.choice(list(MODES))


ENDS = [(1, 1, 1, "add"), (1, 1, MOST_K, "gated"), (300, 17, MOST_K, "add"), (64, 20, MOST_K, "store"), (65, 9000, 1, "store"), (512, 4096, 14336, "add"), (512, 6144, 4096, "store"),
        (20000, 300, 100, "gated"), (36000, 24, 65536, "store"), (5, 36000, 65536, "store"), (333, 25600, 5120, "gated"), (4096, 6144, 4096, "store"), (100, 4096, 14336, "add")]


def check(lib, m, n, k, mode, numbers=None):
    stride, packed_rows = lib.xrt_int8_stride(k), lib.xrt_int8_packed_rows(n, int(mode == "gated"))
    first = Reach(lib, m, n, k, mode, 0)
    blocks, groups, workspace = -(-m // 16), packed_rows // 16, lib.xrt_linear_int8_workspace(m, n, k, MODES[mode])
    whole = numbers is None
    times, steps = (np.zeros((first.parts, blocks, groups), dtype=np.int32), np.zeros((blocks, groups), dtype=np.int64)) if whole else (None, None)
    for number in range(first.workgroups) if whole else numbers(first.workgroups):
        reach = Reach(lib, m, n, k, mode, number)
        assert inside(reach.a, m * stride) and inside(reach.w, packed_rows * stride), (m, n, k, mode, number)
        assert inside(reach.a_scales, m * 4) and inside(reach.w_scales, packed_rows * 4) and inside(reach.sums, workspace), (m, n, k, mode, number)
        if reach.a_scales != NOTHING:
            # a row's scales are fetched for all rows of a that the workgroup loads, and for all channels
            assert reach.a_scales[0] // 4 == reach.a[0] // stride and reach.a_scales[1] // 4 >= -(-reach.a[1] // stride), (m, n, k, mode, number)
            assert reach.w_scales[0] // 64 == reach.w[0] // (16 * stride) and reach.w_scales[1] // 64 >= -(-reach.w[1] // (16 * stride)), (m, n, k, mode, number)
        if whole and len(reach.made):
            part, block, group = reach.made.T
            np.add.at(times, (part, block, group), 1)
            np.add.at(steps, (block, group), reach.steps)
    if whole:
        assert (times == 1).all() and (steps == stride // 128).all(), (m, n, k, mode)
        assert (first.parts > 1) == (workspace > 0)


@pytest.mark.parametrize("seed", range(8))
def test_every_block_is_made_once_and_every_byte_is_inside(lib, seed):
    for size in sizes(seed, 12):
        check(lib, *size)


@pytest.mark.parametrize("size", ENDS, ids=str)
def test_the_ends_of_the_range(lib, size):
    check(lib, *size)


# 2^30 rows and more of one step along k: a row's scale lies 2^32 bytes and more behind the first one's
@pytest.mark.parametrize("m", [2 ** 30 - 300, 2 ** 30 + 4096, 2 ** 30 + 2 ** 29 + 77, 2 ** 31 - 300])
def test_rows_whose_scales_pass_2_to_the_32_bytes(lib, m):
    middle = 2 ** 30 // 256
    check(lib, m, 1, 64, "store", lambda workgroups: [0, 1, 7, workgroups // 2, *range(min(middle, workgroups) - 40, min(middle, workgroups)), *range(workgroups - 40, workgroups)])


def test_more_rows_than_32_bits_number_are_refused(lib):
    lib.xrt_last_error.restype = ctypes.c_char_p
    plan, at = (ctypes.c_int * 5)(), ctypes.c_void_p(1 << 20)
    for m, n, mode in ((2 ** 31 - 1, 1, "store"), (2 ** 31 - 256, 1, "add"), (1, 2 ** 30, "store"), (1, 2 ** 29, "gated"), (4096, 2 ** 31 - 1, "store")):
        assert lib.xrt_linear_int8_plan(m, n, 64, MODES[mode], plan) != 0 and lib.xrt_linear_int8_workspace(m, n, 64, MODES[mode]) == 0
        assert lib.xrt_linear_int8(at, at, at, at, at, 0, m, n, 64, MODES[mode], None, ctypes.c_long(0), None) != 0 and b"too many rows" in lib.xrt_last_error()


def test_more_threads_than_a_launch_counts_are_refused(lib):
    lib.xrt_last_error.restype = ctypes.c_char_p
    at = ctypes.c_void_p(1 << 20)
    for m, n, mode in ((1, 2 ** 27 + 16, "store"), (1, 2 ** 29 - 64, "add"), (16, 2 ** 26 + 64, "gated"), (2 ** 31 - 300, 1, "store")):
        assert lib.xrt_linear_int8(at, at, at, at, at, 0, m, n, 64, MODES[mode], None, ctypes.c_long(0), None) != 0
        assert b"too many tiles" in lib.xrt_last_error(), (m, n, mode)
    assert lib.xrt_pack_int8(at, at, at, at, 2 ** 29, 128, 0, None) != 0 and b"too many elements" in lib.xrt_last_error()
