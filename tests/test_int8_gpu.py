"""Rows and weights in 8-bit integers: the kernels against plain arithmetic in 64 bits."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}         # half a step relative to the value


@pytest.fixture(scope="module")
def ops():
    from xeno_rt_amd.ops import load_ops
    return load_ops()


def rand(*shape, seed=0, scale=1.0, dtype=torch.float32):
    generator = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=generator) * scale).to(dtype)


def whole_numbers(rows, k, seed):
    """8-bit rows with every value from -128 to 127, and scales, as Int8Rows."""
    from xeno_rt_amd.ops import load_ops
    generator = torch.Generator(device=DEV).manual_seed(seed)
    made = load_ops().int8_rows(rows, k, DEV)
    made.values.zero_()
    made.values[:, :k] = torch.randint(-128, 128, (rows, k), device=DEV, generator=generator, dtype=torch.int8)
    made.scales.copy_(torch.rand(rows, device=DEV, generator=generator) * 0.05 + 0.001)
    return made


def plain_rows(y):
    """(values, scales) of float32 rows by the definition, with the float32 divisions that it names."""
    most = y.abs().amax(1)
    scales = most / torch.full_like(most, 127.0)                # (by a plain number torch would multiply with its reciprocal)
    values = torch.where(scales[:, None] > 0, y / scales[:, None], torch.zeros_like(y)).round().clamp(-127, 127)
    broken = ~torch.isfinite(y).all(1)
    scales[broken], values[broken] = float("nan"), 0.0
    return values, scales


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=7e30), torch.nan_to_num(b.float(), nan=7e30))


def padding_is_zero(rows):
    return not bool(rows.values[:, rows.k:].any())


# ---- rows to 8 bits ---------------------------------------------------------------------------------------------------------------------------------------------

# widths of one element, around a piece of eight, a step of 128 and what the threads of a row's workgroup keep (32768), odd ones; x float32 and bfloat16
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 8), (2, 127), (4, 128), (3, 129), (7, 515), (33, 4096), (2, 16391), (1, 32768), (2, 32769), (1, 40007), (300, 64)])
def test_rows_to_8_bits_are_those_of_the_definition(ops, rows, k, dtype):
    x = rand(rows, k, seed=rows + k, dtype=dtype)
    out = ops.int8_rows(rows, k, DEV)
    out.values.fill_(55)
    ops.quantize_int8(x, out)
    values, scales = plain_rows(x.float())
    assert torch.equal(out.values[:, :k].float(), values) and torch.equal(out.scales, scales) and padding_is_zero(out)


def test_rows_to_8_bits_at_the_edges_of_the_numbers(ops):
    k = 300
    x = rand(12, k, seed=3)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 17] = float("inf")
    x[3, 299] = float("nan")
    x[4, 0], x[4, 1] = float("-inf"), float("nan")
    x[5] *= 1e-42                                              # denormal magnitudes, and a scale that is denormal too
    x[6] = torch.full((k,), 1.4e-45, device=DEV)               # the smallest: its scale rounds to zero
    x[7] = torch.where(torch.arange(k, device=DEV) == 5, 3.0e38, x[7])
    x[8] = (torch.arange(k, device=DEV) % 255 - 127).float() * 0.5      # ties: halves of integers
    x[8, 0] = 127.0
    x[9] *= 3e38 / x[9].abs().max()
    x[10] = -1.0
    out = ops.int8_rows(12, k, DEV)
    ops.quantize_int8(x, out)
    values, scales = plain_rows(x)
    assert same(out.scales, scales)
    assert torch.equal(out.values[:, :k].float(), values)
    assert out.scales[6] == 0 and not out.values[6].any() and out.scales[5] > 0 and int(out.values.abs().max()) <= 127


def test_rows_to_8_bits_of_a_part_of_a_wider_matrix(ops):
    wide = rand(9, 1000, seed=4, dtype=torch.bfloat16)
    for columns in (slice(0, 300), slice(3, 404), slice(600, 1000)):
        x = wide[:, columns]
        out, copied = ops.int8_rows(9, x.shape[1], DEV), ops.int8_rows(9, x.shape[1], DEV)
        ops.quantize_int8(x, out)
        ops.quantize_int8(x.contiguous(), copied)
        assert torch.equal(out.values, copied.values) and torch.equal(out.scales, copied.scales)


@pytest.mark.parametrize("rows,k", [(1, 1), (5, 129), (33, 4096), (3, 40007)])
def test_values_of_8_bit_rows(ops, rows, k):
    q = whole_numbers(rows, k, seed=5)
    want = q.values[:, :k].float() * q.scales[:, None]
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.empty(rows, k, dtype=dtype, device=DEV)
        ops.dequantize_int8(q, out)
        assert torch.equal(out, want.to(dtype))


# ---- the norm ---------------------------------------------------------------------------------------------------------------------------------------------------

def exact_norm(x, gain):
    x, gain = x.double(), gain.double()
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * gain


def holds(out, y, rows, k):
    """The 8-bit rows stand for y (64 bits) as nearly as float32 arithmetic has to have it. The mean of k squares in float32 is off by a relative error of at
    most (k / threads + 16) half steps, which the root halves; with the four further roundings of y (rms, quotient, product, gain) 64 half steps cover every
    width here. The scale adds one, the quotient another, and 127 of them can move a value that stands nearer than that to a border."""
    scales = y.abs().amax(1) / 127.0
    assert bool(((out.scales.double() - scales).abs() <= 66 * STEP[torch.float32] * scales).all())
    quotient = y / scales[:, None]
    off = (out.values[:, :k].double() - quotient).abs()
    assert float(off.max()) <= 0.5 + 127 * 132 * STEP[torch.float32]
    assert padding_is_zero(out)


@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gain", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 9), (8, 128), (5, 1001), (8, 4096), (1001, 2049), (2, 32768), (2, 33003)])
def test_norm_with_8_bit_rows(ops, rows, k, gain, delta):
    x, weight = rand(rows, k, seed=1, scale=3.0), (rand(k, seed=2, scale=0.2) + 1.0).to(gain)
    add = None if delta is None else rand(rows, k, seed=3, dtype=delta)
    want = x + add.float() if add is not None else x.clone()
    out = ops.int8_rows(rows, k, DEV)
    out.values.fill_(55)
    ops.rmsnorm_int8(x, weight, EPS, out, delta=add)
    assert torch.equal(x, want)                                 # one float32 addition an element: no other result is right
    holds(out, exact_norm(want, weight), rows, k)


def test_norm_with_8_bit_rows_at_the_edges(ops):
    k = 520
    x = rand(6, k, seed=1)
    x[0] = 0.0
    x[1, 3] = float("inf")
    x[2, 4] = float("nan")
    x[3] *= 1e-30                                              # far below eps
    x[4] *= 1e18                                               # its squares do not fit float32: the mean is infinite and the norm zero
    weight = torch.ones(k, device=DEV)
    out = ops.int8_rows(6, k, DEV)
    ops.rmsnorm_int8(x, weight, EPS, out)
    assert out.scales[0] == 0 and not out.values[0].any()
    assert torch.isnan(out.scales[1:3]).all() and not out.values[1:3].any()
    kept = ops.int8_rows(2, k, DEV)
    ops.rmsnorm_int8(x[3::2].contiguous(), weight, EPS, kept)
    holds(kept, exact_norm(x[3::2], weight), 2, k)
    assert torch.equal(kept.values, out.values[3::2]) and torch.equal(kept.scales, out.scales[3::2])


def test_norm_of_chosen_rows(ops):
    x, weight = rand(10, 700, seed=1), rand(700, seed=2)
    before = x.clone()
    rows = torch.tensor([9, 0, 9, 10, -1, 4], dtype=torch.int32, device=DEV)
    every, out = ops.int8_rows(10, 700, DEV), ops.int8_rows(6, 700, DEV)
    ops.rmsnorm_int8(x, weight, EPS, every)
    ops.rmsnorm_int8(x, weight, EPS, out, rows=rows)
    there = [0, 1, 2, 5]
    assert torch.equal(out.values[there], every.values[rows[there].long()]) and torch.equal(out.scales[there], every.scales[rows[there].long()])
    assert torch.isnan(out.scales[3:5]).all() and not out.values[3:5].any() and torch.equal(x, before)


# ---- products ---------------------------------------------------------------------------------------------------------------------------------------------------

def exact_product(a, w):
    """The products by the definition in 64 bits (the sums are whole numbers far below 2^53), and what their magnitudes are."""
    sums = a.values[:, : a.k].double() @ w.values[:, : w.k].double().t()
    return sums * a.scales.double()[:, None] * w.scales.double()


def near(out, want, base=None):
    """Float32: the sum rounded once and two products (an addition: a further rounding of the result), then what out's type costs."""
    bound = 4 * STEP[torch.float32] * want.abs()
    if base is not None:
        want = base.double() + want
        bound = bound + STEP[torch.float32] * want.abs()
    if out.dtype == torch.bfloat16:
        bound = bound + 1.01 * STEP[torch.bfloat16] * want.abs()
    return bool(((out.double() - want).abs() <= bound + 1e-38).all())


# one row and one column, sizes around the tiles of 16, 64, 128 and 256 and around steps of 64 and 128 along k, long and short k, odd sizes of everything
SIZES = [(1, 1, 1), (1, 5, 64), (2, 16, 65), (3, 17, 127), (1, 4096, 4096), (5, 300, 129), (16, 1000, 512), (17, 48, 1000), (31, 130, 4100), (33, 512, 14336), (48, 4096, 256),
         (64, 257, 2048), (65, 640, 1024), (100, 1001, 777), (128, 128, 128), (129, 255, 300), (200, 3000, 512), (255, 256, 64), (256, 256, 640), (257, 513, 1280), (333, 1280, 5120),
         (512, 6144, 1024), (777, 1001, 2049), (1030, 2050, 384), (2048, 512, 2048), (9, 40000, 128), (300, 24, 9000),
         # 17 to 32 rows of many channels; the larger tiles, with rows and channels that do not fill the last one, one step along k and an odd number of them
         (20, 16400, 256), (300, 16000, 640), (500, 9000, 500), (1200, 8200, 256), (190, 40000, 100), (70, 5000, 8000), (2049, 7000, 384), (3333, 4111, 120), (800, 12345, 128), (1030, 20000, 128), (10, 100, 9000), (25, 3000, 200),
         # the narrow tiles, k whole and in two parts
         (416, 3410, 987), (375, 3418, 4200), (281, 4494, 5951)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_of_8_bit_rows(ops, m, n, k):
    a, w = whole_numbers(m, k, seed=m), whole_numbers(n, k, seed=n + 1)
    want, packed, base = exact_product(a, w), ops.pack_int8(w), rand(m, n, seed=5, scale=30.0)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m + 2, n), 77.0, dtype=dtype, device=DEV)
        ops.linear_int8(a, packed, out[1:m + 1])
        assert near(out[1:m + 1], want) and bool((out[0] == 77.0).all()) and bool((out[m + 1] == 77.0).all())
    added = base.clone()
    ops.linear_int8(a, packed, added, accumulate=True)
    assert near(added, want, base)


@pytest.mark.parametrize("m,n,k", [(m, (n + 1) // 2, k) for m, n, k in SIZES])
def test_gated_products_of_8_bit_rows(ops, m, n, k):
    a, w = whole_numbers(m, k, seed=m), whole_numbers(2 * n, k, seed=n + 1)
    w.scales.mul_(4.0 / (k ** 0.5 * 0.05 * 74 * 74 * 0.05))      # gates of some units, as a feed-forward has them
    both = exact_product(a, w)
    gate, up = both[:, :n], both[:, n:]
    want = gate * torch.sigmoid(gate) * up
    packed = ops.pack_int8(w, gated=True)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m + 2, n), 77.0, dtype=dtype, device=DEV)
        ops.linear_glu_int8(a, packed, out[1:m + 1])
        # gate's relative error e moves silu by at most (1 + |gate|) e; the exponential and the division have a few half steps of their own
        bound = (16 + 8 * gate.abs()) * STEP[torch.float32] * want.abs() + (1.01 * STEP[dtype] * want.abs() if dtype == torch.bfloat16 else 0) + 1e-30
        assert bool(((out[1:m + 1].double() - want).abs() <= bound).all())
        assert bool((out[0] == 77.0).all()) and bool((out[m + 1] == 77.0).all())


@pytest.mark.parametrize("n,k", [(700, 3000), (12000, 300)])
def test_a_row_has_the_same_bits_alone_and_among_others(ops, n, k):
    a, w = whole_numbers(600, k, seed=1), ops.pack_int8(whole_numbers(n, k, seed=2))
    gated = ops.pack_int8(whole_numbers(n, k, seed=3), gated=True)
    from xeno_rt_amd.ops.hip import Int8Rows
    results = []
    for rows in (600, 1, 16, 17, 64, 65, 130, 257):
        part = Int8Rows(a.values[:rows].contiguous(), a.scales[:rows].contiguous(), k)
        stored, added = torch.empty(rows, n, device=DEV), torch.ones(rows, n, device=DEV)
        pairs = torch.empty(rows, n // 2, device=DEV)
        ops.linear_int8(part, w, stored)
        ops.linear_int8(part, w, added, accumulate=True)
        ops.linear_glu_int8(part, gated, pairs)
        results.append((stored, added, pairs))
    for got in results[1:]:
        for x, all_rows in zip(got, results[0]):
            assert torch.equal(torch.nan_to_num(x, nan=7e30), torch.nan_to_num(all_rows[: x.shape[0]], nan=7e30))


def test_the_largest_sums_are_exact(ops):
    """-128 times -128, as many times as there may be: 2^31 - 2^14."""
    from xeno_rt_amd.ops.hip import INT8_MOST_K
    for m in (1, 40, 300):
        a, w = whole_numbers(m, INT8_MOST_K, seed=1), whole_numbers(20, INT8_MOST_K, seed=2)
        for rows in (a, w):
            rows.values[:, : rows.k] = -128
            rows.scales.fill_(1.0)
        out = torch.empty(m, 20, device=DEV)
        ops.linear_int8(a, ops.pack_int8(w), out)
        assert bool((out == float(torch.tensor(2 ** 14 * INT8_MOST_K, dtype=torch.float32))).all())


# rows, weights and a result of more than 2^31 bytes or elements: what lies last is made from what belongs to it
def test_offsets_that_pass_32_bits(ops):
    from xeno_rt_amd.ops.hip import Int8Rows
    picked = lambda rows, which: Int8Rows(rows.values[which].contiguous(), rows.scales[which].contiguous(), rows.k)          # noqa: E731
    long, short = whole_numbers(36000, 65536, seed=1), whole_numbers(24, 65536, seed=2)
    some = torch.tensor([0, 1, 17000, 32767, 32768, 35983, 35998, 35999], device=DEV)
    some_long = picked(long, some)
    out = torch.empty(36000, 24, device=DEV)
    ops.linear_int8(long, ops.pack_int8(short), out)
    assert near(out[some], exact_product(some_long, short))
    few, out = picked(short, torch.arange(5, device=DEV)), torch.empty(5, 36000, device=DEV)
    ops.linear_int8(few, ops.pack_int8(long), out)
    assert near(out[:, some], exact_product(few, some_long))
    x = torch.empty(36000, 65536, device=DEV)
    ops.dequantize_int8(long, x)
    assert torch.equal(x[some], some_long.values.float() * some_long.scales[:, None])
    again = ops.int8_rows(36000, 65536, DEV)
    ops.quantize_int8(x, again)
    values, scales = plain_rows(x[some])
    assert torch.equal(again.values[some].float(), values) and torch.equal(again.scales[some], scales)
    del x, again, long
    a, w = whole_numbers(20000, 64, seed=3), whole_numbers(110000, 64, seed=4)
    rows, columns = torch.tensor([0, 12345, 19998, 19999], device=DEV), torch.tensor([0, 1, 65536, 109983, 109999], device=DEV)
    want, out = exact_product(picked(a, rows), picked(w, columns)), torch.empty(20000, 110000, dtype=torch.bfloat16, device=DEV)
    ops.linear_int8(a, ops.pack_int8(w), out)
    assert near(out[rows][:, columns], want)


def test_rows_and_channels_without_a_scale(ops):
    """A NaN scale makes its row or its channel NaN and nothing else; a zero scale zeros."""
    for m in (3, 40, 300):
        a, w = whole_numbers(m, 200, seed=1), whole_numbers(50, 200, seed=2)
        a.scales[1], w.scales[7] = float("nan"), float("nan")
        a.scales[2] = 0.0
        out = torch.empty(m, 50, device=DEV)
        ops.linear_int8(a, ops.pack_int8(w), out)
        wrong = torch.isnan(out)
        assert bool(wrong[1].all()) and bool(wrong[:, 7].all()) and int(wrong.sum()) == 50 + m - 1
        assert not torch.nan_to_num(out[2]).any()


def test_weights_packed_from_floats(ops):
    for dtype in (torch.float32, torch.bfloat16):
        w, a = rand(70, 333, seed=1, dtype=dtype), whole_numbers(5, 333, seed=2)
        rows = ops.int8_rows(70, 333, DEV)
        ops.quantize_int8(w, rows)
        for gated in (False, True):
            one, two = ops.pack_int8(w, gated=gated), ops.pack_int8(rows, gated=gated)
            assert torch.equal(one.data, two.data) and torch.equal(one.scales, two.scales) and one.shape == (70, 333)


def test_what_lies_behind_the_columns_does_not_count(ops):
    for m in (3, 40, 300):
        for k in (1, 100, 130, 500):
            a, w = whole_numbers(m, k, seed=1), whole_numbers(40, k, seed=2)
            want, gated = torch.empty(m, 40, device=DEV), torch.empty(m, 20, device=DEV)
            ops.linear_int8(a, ops.pack_int8(w), want)
            ops.linear_glu_int8(a, ops.pack_int8(w, gated=True), gated)
            a.values[:, k:], w.values[:, k:] = 77, -99
            got, got_gated = torch.empty_like(want), torch.empty_like(gated)
            ops.linear_int8(a, ops.pack_int8(w), got)
            ops.linear_glu_int8(a, ops.pack_int8(w, gated=True), got_gated)
            assert torch.equal(got, want) and torch.equal(got_gated, gated)


def test_tensors_of_another_device_than_the_current_one_are_refused(ops, monkeypatch):
    from xeno_rt_amd.ops import hip
    q, w, x = ops.int8_rows(4, 100, DEV), ops.pack_int8(rand(20, 100)), rand(4, 100)
    monkeypatch.setattr(hip, "_current_device", lambda: 1)
    for call in (lambda: ops.quantize_int8(x, q), lambda: ops.rmsnorm_int8(x, rand(100), EPS, q), lambda: ops.dequantize_int8(q, x), lambda: ops.pack_int8(x),
                 lambda: ops.linear_int8(q, w, rand(4, 20))):
        with pytest.raises(hip.KernelError, match="current device"):
            call()


def test_a_norm_whose_addend_is_the_stream_itself(ops):
    for k in (300, 40007):
        x = rand(3, k, seed=4)
        want, out, plain = x + x, ops.int8_rows(3, k, DEV), ops.int8_rows(3, k, DEV)
        ops.rmsnorm_int8(x, torch.ones(k, device=DEV), EPS, out, delta=x)
        ops.rmsnorm_int8(want.clone(), torch.ones(k, device=DEV), EPS, plain)
        assert torch.equal(x, want) and torch.equal(out.values, plain.values) and torch.equal(out.scales, plain.scales)


def test_no_rows(ops):
    w, gated = ops.pack_int8(rand(20, 100)), ops.pack_int8(rand(20, 100), gated=True)
    a = ops.int8_rows(0, 100, DEV)
    ops.quantize_int8(rand(0, 100), a)
    ops.rmsnorm_int8(rand(0, 100), rand(100), EPS, a, delta=rand(0, 100))
    ops.rmsnorm_int8(rand(5, 100), rand(100), EPS, a, rows=torch.empty(0, dtype=torch.int32, device=DEV))
    ops.dequantize_int8(a, rand(0, 100))
    ops.linear_int8(a, w, rand(0, 20))
    ops.linear_glu_int8(a, gated, rand(0, 10))


# ---- together, as a layer uses them -----------------------------------------------------------------------------------------------------------------------------

class Layer:
    """The feed-forward of a layer in 8 bits: x += what came before; x += down(to 8 bits(gate/up(norm(x))))."""

    def __init__(self, ops, rows, hidden, inner):
        self.ops, self.gain = ops, rand(hidden, seed=1, scale=0.1) + 1.0
        self.gate_up, self.down = rand(2 * inner, hidden, seed=2, scale=hidden ** -0.5), rand(hidden, inner, seed=3, scale=inner ** -0.5)
        self.packed = ops.pack_int8(self.gate_up, gated=True), ops.pack_int8(self.down)
        self.h, self.q = ops.int8_rows(rows, hidden, DEV), ops.int8_rows(rows, inner, DEV)
        self.act = torch.empty(rows, inner, dtype=torch.bfloat16, device=DEV)

    def forward(self, x, delta):
        self.ops.rmsnorm_int8(x, self.gain, EPS, self.h, delta=delta)
        self.ops.linear_glu_int8(self.h, self.packed[0], self.act)
        self.ops.quantize_int8(self.act, self.q)
        self.ops.linear_int8(self.q, self.packed[1], x, accumulate=True)

    def in_floats(self, x, delta):
        x = x.double() + delta.double()
        both = exact_norm(x, self.gain) @ self.gate_up.double().t()
        gate, up = both.chunk(2, dim=1)
        return x, (gate * torch.sigmoid(gate) * up) @ self.down.double().t()


@pytest.mark.parametrize("rows", [1, 8, 40, 333])
def test_a_feed_forward_in_8_bits(ops, rows):
    """Against the same layer in 64 bits without 8 bits: normal values of n columns stand within scale / sqrt(12), max / (127 sqrt(12)), of themselves, 1 % of
    their deviation for a maximum of 4.5 deviations; gate and up share two such errors, the last product has two more, and the gated values' maximum is some
    20 deviations (5 %): together below 8 % of what the layer adds, in the 2-norm."""
    layer = Layer(ops, rows, 1024, 2720)
    x, delta = rand(rows, 1024, seed=7, scale=2.0), rand(rows, 1024, seed=8, dtype=torch.bfloat16)
    added, change = layer.in_floats(x, delta)
    layer.forward(x, delta)
    assert float((x.double() - added - change).norm() / change.norm()) < 0.08


@pytest.mark.parametrize("rows", [3, 40, 333])
def test_captured_replayed_and_on_another_stream(ops, rows):
    layer = Layer(ops, rows, 512, 1400)
    x0, delta = rand(rows, 512, seed=7), rand(rows, 512, seed=8)
    want = x0.clone()
    layer.forward(want, delta)
    torch.cuda.synchronize()
    x = x0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward(x, delta)
    side.synchronize()
    assert torch.equal(x, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x, delta)
    for turn in range(4):
        x.copy_(x0)
        torch.cuda.synchronize()
        graph.replay()
        eager = x0.clone()
        Layer(ops, rows, 512, 1400).forward(eager, delta)      # the program's own work between the replays
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(eager, want)


def test_two_captured_graphs_and_two_streams_at_once(ops):
    """Products that are cut along k use a workspace of their own call: two that overlap do not disturb each other."""
    made = []
    for seed in (1, 2):
        a, w = whole_numbers(40, 9000, seed=seed), ops.pack_int8(whole_numbers(300, 9000, seed=seed + 10))
        out = torch.zeros(40, 300, device=DEV)
        want = torch.zeros(40, 300, device=DEV)
        ops.linear_int8(a, w, want)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            ops.linear_int8(a, w, out)
        made.append((graph, stream, out, want, a, w))          # (a graph reads its operands where they lay: they stay alive)
    for turn in range(5):
        for graph, stream, out, *_ in made:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, _, out, want, *_ in made)


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------------------------------

def test_refusals(ops):
    from xeno_rt_amd.ops.hip import INT8_MOST_K, Int8Matrix, Int8Rows, KernelError
    q, w, gated = ops.int8_rows(4, 100, DEV), ops.pack_int8(rand(20, 100)), ops.pack_int8(rand(20, 100), gated=True)
    x, gain = rand(4, 100), rand(100)
    refused = [
        lambda: ops.int8_rows(-1, 100, DEV), lambda: ops.int8_rows(1, 0, DEV), lambda: ops.int8_rows(1, INT8_MOST_K + 1, DEV),
        lambda: ops.quantize_int8(rand(4, 99), q), lambda: ops.quantize_int8(rand(3, 100), q), lambda: ops.quantize_int8(x.half(), q),
        lambda: ops.quantize_int8(rand(100, 4).t(), q), lambda: ops.quantize_int8(x.cpu(), q), lambda: ops.quantize_int8(x, x),
        lambda: ops.quantize_int8(rand(1, 100).expand(4, 100), q), lambda: ops.quantize_int8(x[0], q),
        lambda: ops.rmsnorm_int8(x.bfloat16(), gain, EPS, q), lambda: ops.rmsnorm_int8(x, rand(99), EPS, q), lambda: ops.rmsnorm_int8(x[:3], gain, EPS, q),
        lambda: ops.rmsnorm_int8(x, gain, EPS, q, delta=rand(4, 99)), lambda: ops.rmsnorm_int8(x, gain.half(), EPS, q),
        lambda: ops.rmsnorm_int8(x, gain, EPS, q, delta=x.half()), lambda: ops.rmsnorm_int8(rand(4, 200)[:, :100], gain, EPS, q),
        lambda: ops.rmsnorm_int8(x, gain, EPS, q, delta=x.clone(), rows=torch.zeros(4, dtype=torch.int32, device=DEV)),
        lambda: ops.rmsnorm_int8(x, gain, EPS, q, rows=torch.zeros(4, dtype=torch.int64, device=DEV)), lambda: ops.rmsnorm_int8(x, gain, EPS, q, rows=[0, 1, 2, 3]),
        lambda: ops.dequantize_int8(q, rand(4, 101)), lambda: ops.dequantize_int8(q, x.half()),
        lambda: ops.pack_int8(rand(21, 100), gated=True), lambda: ops.pack_int8(rand(0, 100)), lambda: ops.pack_int8(rand(100)), lambda: ops.pack_int8(rand(4, 100).cpu()),
        lambda: ops.linear_int8(x, w, rand(4, 20)), lambda: ops.linear_int8(q, rand(20, 100), rand(4, 20)), lambda: ops.linear_int8(q, gated, rand(4, 20)),
        lambda: ops.linear_int8(q, w, rand(4, 21)), lambda: ops.linear_int8(q, w, rand(3, 20)), lambda: ops.linear_int8(ops.int8_rows(4, 99, DEV), w, rand(4, 20)),
        lambda: ops.linear_int8(q, w, rand(4, 20).bfloat16(), accumulate=True), lambda: ops.linear_int8(q, w, rand(4, 20).half()),
        lambda: ops.linear_int8(q, w, rand(4, 40)[:, ::2]), lambda: Int8Rows(q.values[:, :100], q.scales, 100), lambda: Int8Rows(q.values.cpu(), q.scales, 100), lambda: Int8Rows(q.values[0], q.scales, 100), lambda: Int8Rows(q.values, q.scales, 129),
        lambda: Int8Rows(q.values.view(-1)[:-1].clone(), q.scales, 100), lambda: Int8Rows(torch.empty(4 * 128 + 8, dtype=torch.int8, device=DEV)[8:].view(4, 128), q.scales, 100),
        lambda: Int8Rows([1, 2], q.scales, 100), lambda: Int8Rows(q.values, q.scales[:3], 100), lambda: Int8Rows(q.values, q.scales.cpu(), 100), lambda: Int8Rows(q.values, q.scales, 0),
        lambda: Int8Matrix(w.data, w.scales, 20, 129, False), lambda: Int8Matrix(w.data, w.scales, 33, 100, False), lambda: Int8Matrix(w.data, w.scales[:8], 20, 100, False),
        lambda: Int8Matrix(w.data.view(torch.uint8), w.scales, 20, 100, False), lambda: Int8Matrix(gated.data, gated.scales, 21, 100, True),
        lambda: ops.rmsnorm_int8(x, gain, EPS, x), lambda: ops.linear_int8(Int8Rows(q.values, q.scales, 101), w, rand(4, 20)),
        lambda: ops.linear_glu_int8(q, w, rand(4, 10)), lambda: ops.linear_glu_int8(q, gated, rand(4, 20)), lambda: ops.linear_glu_int8(q, gated, rand(4, 10), activation="relu"),
    ]
    for index, call in enumerate(refused):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {index} was not refused")


def test_the_library_refuses_what_its_kernels_do_not_take(ops):
    at, s = ctypes.c_void_p(q_address(ops)), ops._stream(rand(1))
    bad = [
        lambda: ops.lib.xrt_quantize_int8(at, 2, ctypes.c_long(100), at, at, 1, 100, s), lambda: ops.lib.xrt_quantize_int8(at, 0, ctypes.c_long(99), at, at, 1, 100, s),
        lambda: ops.lib.xrt_quantize_int8(None, 0, ctypes.c_long(100), at, at, 1, 100, s), lambda: ops.lib.xrt_quantize_int8(at, 0, ctypes.c_long(1 << 20), at, at, 1, 131072, s),
        lambda: ops.lib.xrt_linear_int8(at, at, at, at, at, 1, 1, 1, 1, 1, None, ctypes.c_long(0), s), lambda: ops.lib.xrt_linear_int8(at, at, at, at, at, 0, 1, 1, 1, 3, None, ctypes.c_long(0), s),
        lambda: ops.lib.xrt_linear_int8(at, at, at, at, at, 0, 1, 1, 131072, 0, None, ctypes.c_long(0), s), lambda: ops.lib.xrt_linear_int8(at, at, at, at, at, 0, -1, 1, 1, 0, None, ctypes.c_long(0), s),
        lambda: ops.lib.xrt_linear_int8(at, at, at, at, at, 0, 1, 1, 1, 2 | 1 << 8, None, ctypes.c_long(0), s),
        lambda: ops.lib.xrt_pack_int8(at, at, at, at, 0, 1, 0, s), lambda: ops.lib.xrt_dequantize_int8(at, at, at, 5, 1, 1, s),
    ]
    for index, call in enumerate(bad):
        assert call() != 0, index
        assert ops.lib.xrt_last_error()


KEPT = []


def q_address(ops):
    KEPT.append(torch.zeros(1 << 12, device=DEV))
    return KEPT[-1].data_ptr()
