"""An engine whose layers' matrices are kept in 8 bits, on the CPU with the stand-in for the kernels, and what parts say and hand on."""
import pytest
import torch

from conftest import TINY, make_folder
from helpers import errors, run_batched, run_tail_decoded, run_whole, token_ids
from int8_models import LIMITS, PlainInt8Model
from ops_emulation import EmulatedOps


def near(got, want):
    worst, rms = errors(got, want)
    return worst <= LIMITS["max"] and rms <= LIMITS["rms"]


@pytest.fixture(scope="module", params=["llama", "qwen3"])
def model(request, tmp_path_factory):
    folder = make_folder(TINY[request.param], tmp_path_factory.mktemp(request.param), seed=71, std=0.2)
    return folder, PlainInt8Model(folder).prepare(torch.float32)


def engine_of(folder, **options):
    from xeno_rt_amd.engine import Engine
    return Engine.load(folder, dtype="float32", device="cpu", ops=EmulatedOps(), max_tokens=64 * 6, max_slots=3, **options)


def test_the_engine_is_the_plain_model_in_8_bits(model):
    folder, plain = model
    engine = engine_of(folder, int8_weights=True)
    requests = [token_ids(plain.config.vocab_size, length, seed=length) for length in (1, 9, 30)]
    for ids in requests:
        want = plain.logits(ids)
        assert near(run_whole(engine, ids), want)
        assert near(run_tail_decoded(engine, ids, tail=5), want)
    for got, ids in zip(run_batched(engine, requests, [1, 4, 20]), requests):
        assert near(got, plain.logits(ids))


def test_8_bits_change_the_logits_and_little(model):
    """Against the engine as it is: each product's operands stand within 1/254 of their row's largest value, some percent of the result together."""
    folder, plain = model
    ids = token_ids(plain.config.vocab_size, 30, seed=4)
    worst, rms = errors(run_whole(engine_of(folder, int8_weights=True), ids), run_whole(engine_of(folder), ids))
    assert 1e-4 < rms < 0.05


def test_which_matrices_are_kept_in_8_bits(model):
    folder, _ = model
    engine = engine_of(folder, int8_weights=True)
    spec = engine.model.spec
    for block in spec.layers:
        assert isinstance(block.mixer.w_qkv, EmulatedOps.Int8Matrix) and isinstance(block.mixer.w_o, EmulatedOps.Int8Matrix)
        assert isinstance(block.feed_forward.w_gate_up, EmulatedOps.Int8Matrix) and block.feed_forward.w_gate_up.gated
        assert isinstance(block.feed_forward.w_down, EmulatedOps.Int8Matrix)
        assert block.first_norm() is None and not block.one_call
    assert isinstance(spec.head.weight, torch.Tensor) and isinstance(spec.embedding.table, torch.Tensor)
    plain = engine_of(folder).model.spec.layers[0]
    assert isinstance(plain.mixer.w_qkv, torch.Tensor) and not plain.mixer.reads_int8 and plain.first_norm() is plain.mixer_norm


def test_the_norms_before_such_products_make_the_rows(model):
    """No product of a layer brings the normed rows to 8 bits a second time, and none is left to do a norm."""
    folder, _ = model
    engine = engine_of(folder, int8_weights=True)
    made, whole = [], engine.ops.quantize_int8
    engine.ops.quantize_int8 = lambda x, out: (made.append(tuple(out.shape)), whole(x, out))[1]
    run_whole(engine, [1, 2, 3])
    c = engine.config
    per_layer = [(3, c.hidden_size), (3, c.num_attention_heads * c.head_dim), (3, c.hidden_size), (3, c.intermediate_size)]
    assert made == per_layer * c.num_hidden_layers              # the two norms, the attention's output, the gated pair
