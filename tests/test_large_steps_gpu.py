"""Steps whose buffers pass 2^31 bytes, against the same sequences in small steps."""
import pytest
import torch

from helpers import TOLERANCE, errors, token_ids

pytestmark = pytest.mark.gpu

# two layers whose feed-forward is wide: 45 KB of buffers a token
WIDE = {"architectures": ["LlamaForCausalLM"], "vocab_size": 512, "hidden_size": 1024, "intermediate_size": 16384, "num_hidden_layers": 2,
        "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 128, "rms_norm_eps": 1e-5, "rope_theta": 10000.0,
        "max_position_embeddings": 1024, "tie_word_embeddings": False, "hidden_act": "silu", "eos_token_id": 1, "bos_token_id": 0}
SEQUENCES, TOKENS = 64, 900


def test_a_step_with_more_than_2_gigabytes_of_buffers():
    """Every prompt's last logits, and those of a decode step behind prompts of which nothing was wanted: 64 prompts in one step and eight at a time. Either is
    within the tolerance of the exact logits, so the two are within twice that of one another."""
    from xeno_rt_amd.config import parse_config
    from xeno_rt_amd.engine import Engine
    engine = Engine.random(parse_config(WIDE), seed=3, max_tokens=SEQUENCES * 1024, max_slots=SEQUENCES, max_context=1024)
    prompts = [token_ids(512, TOKENS, seed) for seed in range(SEQUENCES)]

    def run(at_once, wanted):
        slots = [engine.alloc_slot() for _ in prompts]
        rows = []
        for first in range(0, SEQUENCES, at_once):
            rows.append(engine.step([(slot, ids, wanted) for slot, ids in list(zip(slots, prompts))[first:first + at_once]]))
        assert all(row.shape == (min(at_once, SEQUENCES) * len(wanted), 512) for row in rows)
        decoded = engine.step([(slot, [7], [0]) for slot in slots])
        for slot in slots:
            engine.free_slot(slot)
        return torch.cat(rows + [decoded])

    limit = TOLERANCE["bfloat16"]
    for wanted in ([], [TOKENS - 1]):
        want = run(8, wanted)
        for _ in range(2):                                      # (the second time the step's memory is one piece, made as long as the first needed)
            print("step of", SEQUENCES * TOKENS, "tokens, wanted", wanted, flush=True)
            got = run(SEQUENCES, wanted)
            assert torch.isfinite(got).all()
            worst, rms = errors(got, want)
            assert worst <= 2 * limit["max"] and rms <= 2 * limit["rms"], (wanted, worst, rms)
    assert engine.runtime.arena.wanted > 2 ** 31
