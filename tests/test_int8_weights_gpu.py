"""An engine whose layers' matrices are kept in 8 bits, on the GPU: against the plain model in 8 bits, cut and batched, as a graph and kernel by kernel."""
import pytest
import torch

from conftest import TINY, make_folder
from helpers import errors, run_batched, run_tail_decoded, run_whole, token_ids
from int8_models import LIMITS, PlainInt8Model

pytestmark = pytest.mark.gpu
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
LENGTHS = [1, 5, 17, 64, 65, 120]


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {name: make_folder(TINY[name], tmp_path_factory.mktemp(name), seed=71, std=0.2) for name in TINY}


def engine_of(folder, dtype, **options):
    from xeno_rt_amd.engine import Engine
    return Engine.load(folder, dtype=dtype, max_tokens=64 * 8, max_slots=3, int8_weights=True, **options)


def near(got, want):
    worst, rms = errors(got, want)
    assert worst <= LIMITS["max"] and rms <= LIMITS["rms"], (worst, rms)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("name", list(TINY))
def test_requests_whole_cut_and_batched(folders, name, dtype):
    plain, engine = PlainInt8Model(folders[name]).prepare(DTYPES[dtype]), engine_of(folders[name], dtype)
    requests = [token_ids(plain.config.vocab_size, length, seed=length) for length in LENGTHS]
    for ids in requests:
        want, whole, cut = plain.logits(ids), run_whole(engine, ids), run_tail_decoded(engine, ids, tail=8)
        near(whole, want)
        near(cut, want)
        if dtype == "float32":                                  # sums of whole numbers and a row's own scale do not depend on the step's shape
            assert torch.equal(whole, cut)
    for got, ids in zip(run_batched(engine, requests[1:4], [2, 9, 30]), requests[1:4]):
        near(got, plain.logits(ids))
    engine.cache.check()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_replayed_steps_have_the_bits_of_launched_ones(folders, dtype):
    ids = token_ids(TINY["qwen3"]["vocab_size"], 40, seed=3)
    graph, direct = (run_tail_decoded(engine_of(folders["qwen3"], dtype, graphs=graphs), ids, tail=20) for graphs in (True, False))
    assert torch.equal(graph, direct)


def test_kernels_and_stand_in_agree_on_the_gpu(folders):
    from ops_emulation import EmulatedOps
    ids = token_ids(TINY["llama"]["vocab_size"], 50, seed=5)
    near(run_whole(engine_of(folders["llama"], "float32"), ids), run_whole(engine_of(folders["llama"], "float32", ops=EmulatedOps(), graphs=False), ids))


def test_generation_and_the_command_line(folders, capsys):
    from xeno_rt_amd.cli import main
    tokens = engine_of(folders["llama"], "float32").generate([[3, 4, 5]], max_tokens=12, stop_ids=[])[0]
    assert len(tokens) == 12
    assert main(["generate", "--model", folders["llama"], "--prompt-ids", "3,4,5", "--max-tokens", "12", "--temperature", "0", "--repetition-penalty", "1",
                 "--stop-ids", "", "--dtype", "float32", "--int8-weights"]) == 0
    assert capsys.readouterr().out.split() == [str(token) for token in tokens]


def test_a_norm_that_a_product_has_begun_does_not_reach_8_bit_weights():
    """Rows whose RMSNorm's division is left to the product after it are refused: a product in 8 bits cannot do it."""
    from xeno_rt_amd.ops import load_ops
    from xeno_rt_amd.ops.hip import KernelError, Prescaled
    ops = load_ops()
    w = ops.pack_int8(torch.randn(16, 64, device="cuda:0"))
    rows = Prescaled(torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda:0"), torch.zeros(4, 64, device="cuda:0"), 1e-5)
    for call in (lambda: ops.linear(rows, w, torch.zeros(4, 16, device="cuda:0")), lambda: ops.linear(None, w, torch.zeros(4, 16, device="cuda:0"))):
        with pytest.raises(KernelError):
            call()
