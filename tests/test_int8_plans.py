"""Products of 8-bit rows: which kernel takes them, asked of the launchers without a GPU, and what their workgroups read and write, worked out here from the sizes:
every block of the result by one workgroup of every part, every byte inside the operands and the workspace."""
import ctypes
import random

import numpy as np
import pytest

MODES = {"store": 0, "add": 1, "gated": 2}
MOST_K = 131071


@pytest.fixture(scope="module")
def lib():
    from xeno_rt_amd.ops import build
    made = ctypes.CDLL(build.find_library() or build.build())
    made.xrt_linear_int8_workspace.restype = made.xrt_int8_stride.restype = made.xrt_int8_packed_rows.restype = ctypes.c_long
    return made


def plan_of(lib, m, n, k, mode):
    plan = (ctypes.c_int * 5)()
    assert lib.xrt_linear_int8_plan(m, n, k, MODES[mode], plan) == 0
    return dict(zip(("tile", "width", "blocks", "groups", "parts"), plan))


# By registers: up to 16, 32 and 64 rows; few tiles of 64 x 64 above. By LDS: all three heights, the narrow tile, k whole and in parts.
@pytest.mark.parametrize("m,n,k,mode,plan", [
    (1, 4096, 4096, "add", (0, 0, 1, 1, 1)), (16, 100, 9000, "store", (0, 0, 1, 1, 5)), (7, 297, 926, "store", (0, 0, 1, 1, 1)), (17, 6144, 4096, "store", (0, 0, 2, 2, 1)), (32, 14336, 4096, "gated", (0, 0, 2, 4, 1)),
    (33, 14336, 4096, "gated", (0, 0, 4, 4, 1)), (64, 4096, 14336, "add", (0, 0, 4, 4, 4)), (777, 1001, 2049, "store", (0, 0, 4, 4, 1)), (65, 24, 9000, "gated", (0, 0, 4, 4, 16)),
    (4096, 4096, 4096, "add", (256, 256, 0, 0, 1)), (4096, 14336, 4096, "gated", (256, 256, 0, 0, 1)), (333, 25600, 5120, "gated", (192, 256, 0, 0, 1)),
    (200, 14336, 4096, "gated", (128, 256, 0, 0, 1)), (128, 14336, 4096, "gated", (128, 128, 0, 0, 1)), (100, 4096, 14336, "add", (128, 128, 0, 0, 8)),
    (416, 1705, 987, "gated", (128, 128, 0, 0, 1)), (375, 1709, 6572, "gated", (128, 128, 0, 0, 3))])
def test_which_kernel_takes_a_product(lib, m, n, k, mode, plan):
    assert tuple(plan_of(lib, m, n, k, mode).values()) == plan


def tile_place(identity, tiles_m, tiles_n):
    total = tiles_m * tiles_n
    identity = identity % 8 * ((total + 7) // 8) + identity // 8
    if identity >= total:
        return None
    if tiles_m <= 4:
        return identity % tiles_m, identity // tiles_m, 0
    panel, inside = divmod(identity, 8 * tiles_m)
    width = min(8, tiles_n - panel * 8)
    return inside // width, panel * 8 + inside % width, 0


def part_place(identity, tiles_m, tiles_n, parts):
    tiles = tiles_m * tiles_n
    total = tiles * parts
    identity = identity % 8 * ((total + 7) // 8) + identity // 8
    if identity >= total:
        return None
    return identity % tiles % tiles_m, identity % tiles // tiles_m, identity // tiles


def dealt(plan, tiles_m, tiles_n, streamed_once):
    ids = (tiles_m * tiles_n * plan["parts"] + 7) // 8 * 8
    for identity in range(ids):
        if plan["parts"] == 1:
            place = tile_place(identity, tiles_m, tiles_n)
        elif streamed_once:
            place = (0, identity % tiles_n, identity // tiles_n) if identity < tiles_n * plan["parts"] else None
        else:
            place = part_place(identity, tiles_m, tiles_n, plan["parts"])
        if place is not None:
            yield place


def even_height(m, most):
    tiles = -(-m // most)
    return -(-(-(-m // tiles)) // 16) * 16


def inside(offsets, size, limit):
    return int(offsets.min()) >= 0 and int(offsets.max()) + size <= limit


def tile_in_lds(plan, tile_m, tile_n, part, m, groups, stride):
    """What a workgroup of the kernel with tiles in LDS loads from the rows, the weights and the scales (bytes), and the blocks of the result it writes."""
    bm, bn, units = plan["tile"], plan["width"], stride // 128
    height = even_height(m, bm)
    m0, first_group = tile_m * height, tile_n * bn // 16
    per = -(-units // plan["parts"])
    first_step = part * per if plan["parts"] > 1 else 0
    steps = min(per, units - first_step) if plan["parts"] > 1 else units
    assert steps > 0
    last_row, upper = min(height, m - m0) - 1, (height // 16 + 1) // 2
    missing = bm // 2 - upper * 16
    lane, rows_a, pieces_w = np.arange(64), [], []
    for wave in range(8):
        for half in range(2):
            def block_of(i, rows, blocks):
                count, p = rows // 16, min(i * 8 + wave, blocks - 1)
                return (p // count * rows + half * (rows // 2)) // 8 + p % count
            for i in range((bm // 16 + 7) // 8):
                block = block_of(i, bm // 2, bm // 16)
                rows_a.append(np.minimum(block * 8 + lane // 8 - (missing if block * 8 >= bm // 2 else 0), last_row) * stride + (lane % 8 ^ lane // 8) * 16)
            for i in range(bn // 128):
                block = block_of(i, bn // 4, bn // 16)
                pieces_w.append(min(block // 2, groups - 1 - first_group) * 16 * stride + block % 2 * 1024 + lane * 16)
    rows_a, pieces_w = m0 * stride + np.concatenate(rows_a), first_group * 16 * stride + np.concatenate(pieces_w)
    assert rows_a.max() - m0 * stride + units * 128 < 2 ** 32 and pieces_w.max() - first_group * 16 * stride + units * 2048 < 2 ** 32
    last = first_step + steps - 1
    loads_a, loads_w = np.concatenate([rows_a + first_step * 128, rows_a + last * 128]), np.concatenate([pieces_w + first_step * 2048, pieces_w + last * 2048])
    written = []
    for wave in range(8):
        blocks = upper if wave < 4 else height // 16 - upper
        wave_row, wave_group = m0 + (wave // 4) * upper * 16, first_group + wave % 4 * (bn // 64)
        row_end = min(wave_row + blocks * 16, min(m0 + height, m))
        assert wave_row - m0 + blocks * 16 <= 256
        written += [(row // 16, wave_group + j) for row in range(wave_row, row_end, 16) for j in range(bn // 64) if wave_group + j < groups]
    return loads_a, loads_w, written


def tile_in_registers(plan, tile_m, tile_n, part, m, groups, stride):
    units, mt, g, parts = stride // 128, plan["blocks"], plan["groups"], plan["parts"]
    lane, loads_a, loads_w, walked = np.arange(64), [], [], 0
    begin, end = units * part // parts, units * (part + 1) // parts
    for wave in range(8):
        first, after = begin + (end - begin) * wave // 8, begin + (end - begin) * (wave + 1) // 8
        walked += after - first
        for unit in {first, after - 1} if after > first else ():
            for i in range(mt):
                loads_a.append(np.minimum((tile_m * mt + i) * 16 + lane % 16, m - 1) * stride + unit * 128 + lane // 16 * 16 + 64)
                loads_a.append(loads_a[-1] - 64)
            for j in range(g):
                loads_w.append(min(tile_n * g + j, groups - 1) * 16 * stride + unit * 2048 + lane * 16 + 1024)
                loads_w.append(loads_w[-1] - 1024)
    assert walked == end - begin
    written = [(tile_m * mt + i, tile_n * g + j) for i in range(mt) for j in range(g) if tile_n * g + j < groups and (tile_m * mt + i) * 16 < m]
    return np.concatenate(loads_a), np.concatenate(loads_w), written


def sizes(seed, count):
    spread = random.Random(seed)
    near = lambda low, high: min(high, max(low, int(round(2 ** spread.uniform(np.log2(low), np.log2(high))))))     # noqa: E731
    for _ in range(count):
        yield near(1, 6000), near(1, 12000), near(1, 20000), spread.choice(list(MODES))
    for m, n, k in ((1, 1, 1), (1, 1, MOST_K), (300, 17, MOST_K), (64, 20, MOST_K), (65, 9000, 1), (512, 4096, 14336), (512, 6144, 4096), (20000, 300, 100),
                    (36000, 24, 65536), (5, 36000, 65536), (20000, 110000, 64)):
        yield m, n, k, "add"


@pytest.mark.parametrize("seed", range(12))
def test_every_block_is_made_once_and_every_access_is_inside(lib, seed):
    for m, n, k, mode in sizes(seed, 20):
        plan, stride = plan_of(lib, m, n, k, mode), lib.xrt_int8_stride(k)
        packed_rows = lib.xrt_int8_packed_rows(n, int(mode == "gated"))
        groups = packed_rows // 16
        assert stride % 128 == 0 and k <= stride < k + 128 and packed_rows >= (2 * n if mode == "gated" else n)
        in_lds = plan["tile"] > 0
        high, wide = (even_height(m, plan["tile"]), plan["width"]) if in_lds else (plan["blocks"] * 16, plan["groups"] * 16)
        tiles_m, tiles_n = -(-m // high), -(-packed_rows // wide)
        if in_lds:
            assert tiles_m == -(-m // plan["tile"])
        made = np.zeros((plan["parts"], -(-m // 16), groups), dtype=np.int32)
        places = list(dealt(plan, tiles_m, tiles_n, not in_lds and m <= 64))
        assert len(places) == len(set(places)) == tiles_m * tiles_n * plan["parts"]
        look = set(random.Random(seed).sample(places, min(len(places), 12))) | {places[0], places[-1], (tiles_m - 1, tiles_n - 1, plan["parts"] - 1)}
        for place in places:
            if place in look or len(places) <= 600:
                a, w, written = (tile_in_lds if in_lds else tile_in_registers)(plan, *place, m, groups, stride)
                assert not len(a) or (inside(a, 16, m * stride) and inside(w, 16, packed_rows * stride)), (m, n, k, mode, plan, place)
                for block in written:
                    made[(place[2], *block)] += 1
        if len(places) <= 600:
            assert (made == 1).all(), (m, n, k, mode, plan)
        need = lib.xrt_linear_int8_workspace(m, n, k, MODES[mode])
        assert need == (made.size * 64 * 16 if plan["parts"] > 1 else 0)


def test_bad_sizes_are_refused(lib):
    plan = (ctypes.c_int * 5)()
    for m, n, k in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, MOST_K + 1), (-1, 1, 1)):
        assert lib.xrt_linear_int8_plan(m, n, k, 0, plan) != 0 and lib.xrt_linear_int8_workspace(m, n, k, 0) == 0
    assert lib.xrt_linear_int8_plan(1, 1, 1, 0, None) != 0
