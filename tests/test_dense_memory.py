"""The memory of a dense decoder's layers launched by one call, asked of the library without a GPU: a step's buffers, which lie one behind another, fit the memory
that the call says it needs, also where they pass 2^31 bytes."""
import ctypes

import pytest

from xeno_rt_amd.ops import hip

BF16, F32 = 1, 0
# (hidden, query heads, key heads, head size, feed-forward width): the Llama-3-8B, Qwen3-32B and Llama-3.2-1B sizes and a tiny model's
SHAPES = [(4096, 32, 8, 128, 14336), (5120, 64, 8, 128, 25600), (2048, 32, 8, 64, 8192), (64, 4, 2, 16, 176)]


@pytest.fixture(scope="module")
def plan():
    from xeno_rt_amd.ops import build
    lib = ctypes.CDLL(build.find_library() or build.build())
    lib.xrt_dense_blocks.restype = ctypes.c_long
    lib.xrt_last_error.restype = ctypes.c_char_p

    def memory(shape, tokens, sequences, dtype=BF16, layers=3, wanted=None, context=None):
        hidden, heads, kv_heads, head_dim, width = shape
        at = 1 << 20                                            # (without memory the call follows no pointer)
        made = (hip.DenseLayer * layers)()
        for layer in made:
            for name in ("mixer_gain", "ff_gain", "rope_theta", "k_cache", "v_cache", "block_table"):
                setattr(layer, name, at)
            layer.qkv.data = layer.o.data = layer.gate_up.data = layer.down.data = at
            layer.mixer_eps = layer.ff_eps = 1e-5
            layer.n_heads, layer.n_kv_heads, layer.head_dim, layer.intermediate, layer.rope_dim = heads, kv_heads, head_dim, width, head_dim
            layer.rope_scale = layer.scale = 1.0
            layer.table_stride, layer.n_blocks, layer.writable = 1 << 16, 1 << 16, 1
        count = -(-tokens // sequences)
        step = hip._DenseStep(at, at, at, at, at, at, None, dtype, tokens, hidden, sequences, count, context or count, 1)
        rows = None if wanted is None else ctypes.byref(hip._DenseWanted(at if wanted else None, at if wanted else None, wanted))
        need = lib.xrt_dense_blocks(made, layers, ctypes.byref(step), rows, None, ctypes.c_long(0))
        assert need >= 0, lib.xrt_last_error().decode()
        return need

    return memory


def least(shape, tokens, dtype):
    """The buffers of a layer that are in use together: two hand-overs to the next layer, q/k/v, the attention's output, the rows between and the gated rows."""
    hidden, heads, kv_heads, head_dim, width = shape
    size = 2 if dtype == BF16 else 4
    return tokens * size * (3 * hidden + (heads + 2 * kv_heads) * head_dim + heads * head_dim + width)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_steps_buffers_fit_its_memory(plan, shape, dtype):
    for tokens, sequences in ((1, 1), (8, 8), (64, 64), (333, 1), (2048, 4), (8192, 16), (16384, 32), (26000, 64), (32768, 64), (65536, 64), (140000, 64), (250000, 64), (624000, 160)):
        for wanted in (None, 0, sequences):
            need = plan(shape, tokens, sequences, dtype, wanted=wanted)
            assert need >= least(shape, tokens, dtype), (tokens, sequences, wanted)
            assert need <= 2 * least(shape, tokens, dtype) + (1 << 29), (tokens, sequences, wanted)      # (and is what they take, not some other number)


def test_the_memory_grows_with_the_step(plan):
    for shape in SHAPES[:2]:
        sizes = [plan(shape, tokens, 64, wanted=0) for tokens in range(8192, 131072 + 1, 8192)]
        assert all(a < b for a, b in zip(sizes, sizes[1:]))
