"""Frequencies of rotary positions on the host, and what the operators around drafted tokens refuse without a GPU."""

import math

import pytest
import torch

from turboquant_vllm.rotary import rotary_inv_freq


def test_plain_and_linear():
    freq, factor = rotary_inv_freq(64, 500000.0)
    assert freq.dtype == torch.float64 and factor == 1.0
    assert torch.allclose(freq, torch.tensor([500000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-15)
    half, _ = rotary_inv_freq(64, 500000.0, {"rope_type": "linear", "factor": 2.0})
    assert torch.equal(half, freq / 2)
    theta, _ = rotary_inv_freq(64, scaling={"rope_type": "default", "rope_theta": 500000.0})
    assert torch.equal(theta, freq)


SCALINGS = {
    "linear": {"factor": 4.0},
    "dynamic": {"factor": 2.0, "original_max_position_embeddings": 2048},
    "yarn": {"factor": 16.0, "original_max_position_embeddings": 4096},
    "llama3": {"factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    "longrope": {"short_factor": [1.0 + i / 64 for i in range(64)], "long_factor": [2.0 + i for i in range(64)], "factor": 32.0,
                 "original_max_position_embeddings": 4096},
}


@pytest.mark.parametrize("kind", sorted(SCALINGS))
@pytest.mark.parametrize("seq_len", [None, 100, 20000])
def test_scaled_as_transformers_has_them(kind, seq_len):
    """The frequencies that a HuggingFace model of the same configuration computes (in fp32)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    scaling = {"rope_type": kind, "rope_theta": 10000.0, **SCALINGS[kind]}
    original = scaling.get("original_max_position_embeddings", 4096)
    config = LlamaConfig(hidden_size=1024, num_attention_heads=8, head_dim=128, rope_theta=10000.0, max_position_embeddings=original,
                         rope_parameters=scaling)
    config.original_max_position_embeddings = original
    want, want_factor = ROPE_INIT_FUNCTIONS[kind](config, torch.device("cpu"), seq_len=seq_len)
    got, factor = rotary_inv_freq(128, 10000.0, scaling, seq_len=seq_len)
    # (theirs: a power, a division and, for the ramps, a blend in fp32: some 2^-24 each, the power's exponent up to ln 10^4 times that)
    assert torch.allclose(got.float(), want.float(), rtol=16 * 2 ** -24, atol=0)
    assert math.isclose(factor, want_factor, rel_tol=1e-12)


def test_refusals():
    for dim in (0, -2, 7):
        with pytest.raises(ValueError, match="even"):
            rotary_inv_freq(dim)
    with pytest.raises(ValueError, match="unknown"):
        rotary_inv_freq(64, scaling={"rope_type": "spiral"})
    with pytest.raises(ValueError, match="original_max"):
        rotary_inv_freq(64, scaling={"rope_type": "dynamic", "factor": 2.0})
    with pytest.raises(ValueError, match="factors"):
        rotary_inv_freq(64, scaling={"rope_type": "longrope", "short_factor": [1.0], "original_max_position_embeddings": 10})


def test_cpu_tensors_are_refused(cuda_lib):
    from turboquant_vllm.kernels import ops

    q, ints = torch.zeros(2, 1, 64), torch.zeros(2, dtype=torch.int32)
    cache, table = torch.zeros(1, 16, 72, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32)
    calls = [
        lambda: ops.tq4_rotary(q, None, ints, torch.ones(32)),
        lambda: ops.tq4_tree_mask(ints, ints, 2),
        lambda: ops.paged_tq4_tree_attention(q, cache, table, ints[:1], ints, table, q[0, 0], q[0, 0], q, 1, 16),
        lambda: ops.tq4_copy_blocks(cache, table, 1, 64),
        lambda: ops.tq4_compact_rows([cache], table, ints[:1], table, ints[:1], 1, 64),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError):
        ops.tq4_rotary([1.0], None, ints, torch.ones(32))
    with pytest.raises(ValueError, match="unsupported attention shape"):
        ops.tree_attention_workspace_bytes(8, 8, 3, 128)


def test_status_of_the_c_entry_points_without_a_launch(cuda_lib):
    """Arguments that are refused, and calls with nothing to do, before anything touches a GPU."""
    lib = cuda_lib
    ok, invalid, unsupported, workspace = 0, 1, 2, 4
    assert lib.tq4_rotary(None, None, 2, 0, 8, 2, 128, None, None, None, 1, None, 1, 128, 0, 1.0, 0, None, None, None, None, None) == ok
    assert lib.tq4_rotary(None, None, 2, 4, 8, 2, 128, None, None, None, 1, None, 1, 128, 0, 1.0, 0, None, None, None, None, None) == invalid
    assert lib.tq4_rotary(None, None, 2, 4, 8, 2, 128, None, None, None, 1, None, 1, 127, 0, 1.0, 0, None, None, None, None, None) == invalid
    assert lib.tq4_rotary(None, None, 3, 4, 8, 2, 128, None, None, None, 1, None, 1, 128, 0, 1.0, 0, None, None, None, None, None) == unsupported
    assert lib.tq4_tree_mask(None, None, 0, 1, 1, None, None, None, None) == ok
    assert lib.tq4_tree_mask(None, None, 4, 1, 0, None, None, None, None) == invalid
    assert lib.tq4_tree_mask(None, None, 4, 1, 1, None, None, None, None) == invalid
    import ctypes

    at = (ctypes.c_void_p * 1)(256)  # (an address that nothing reads)
    assert lib.tq4_copy_blocks(at, 1, 8, 16, 16 * 272, 272, 2, 128, None, 1, 0, None, 0, None, None) == ok
    assert lib.tq4_copy_blocks(at, 1, 8, 16, 16 * 272, 272, 2, 128, None, 1, 3, None, 0, None, None) == invalid
    assert lib.tq4_copy_blocks(at, 1, 8, 16, 16 * 272, 271, 2, 128, at, 1, 3, None, 0, None, None) == invalid
    assert lib.tq4_copy_blocks(at, 1, 8, 16, 16 * 272, 272, 2, 100, at, 1, 3, None, 0, None, None) == unsupported
    assert lib.tq4_copy_blocks_workspace_bytes(384, 50) == 0 and lib.tq4_copy_blocks_workspace_bytes(385, 50) == 200
    assert lib.tq4_copy_blocks(at, 1, 8, 16, 16 * 272, 272, 2, 128, at, 1, 1025, None, 0, None, None) == workspace
    assert lib.tq4_compact_rows_workspace_bytes(3, 2, 64, 2, 128) == 0
    need = lib.tq4_compact_rows_workspace_bytes(3, 2, 65, 2, 128)
    assert need >= 4 * (1 + 2 + 3 * 2 * 2)
    assert lib.tq4_compact_rows(at, 1, 8, 16, 16 * 272, 272, 2, 128, at, 4, 4, 0, at, at, 5, 5, at, None, None, 0, None, None) == ok
    assert lib.tq4_compact_rows(at, 1, 8, 16, 16 * 272, 272, 2, 128, at, 4, 4, 2, at, at, 65, 65, at, None, None, 0, None, None) == workspace
    assert lib.tq4_compact_rows(at, 1, 8, 16, 16 * 272, 272, 2, 128, at, 4, 4, 2, None, at, 5, 5, at, None, None, 0, None, None) == invalid
    assert lib.tq4_tree_attention_workspace_bytes(0, 8, 2, 128) == 0 and lib.tq4_tree_attention_workspace_bytes(5, 8, 2, 100) == 0


@pytest.mark.parametrize("longest,extra", [(131072, {}), (131072, {"factor": 8.0}), (131072, {"attention_factor": 1.3}), (4096, {}), (2048, {})])
@pytest.mark.parametrize("seq_len", [None, 100, 20000])
def test_longrope_takes_its_factor_from_the_longest_context(longest, extra, seq_len):
    """A configuration as Phi-3 models carry it: lists of factors and the original context, no ``factor``."""
    from transformers import Phi3Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    scaling = {"rope_type": "longrope", "rope_theta": 10000.0, "short_factor": [1.0 + i / 64 for i in range(48)],
               "long_factor": [2.0 + i for i in range(48)], **extra}
    config = Phi3Config(hidden_size=96 * 4, num_attention_heads=4, num_key_value_heads=4, max_position_embeddings=longest,
                        original_max_position_embeddings=4096, rope_parameters=scaling, pad_token_id=0)
    assert config.rope_parameters["original_max_position_embeddings"] == 4096 and ("factor" in config.rope_parameters) == ("factor" in extra)
    want, want_factor = ROPE_INIT_FUNCTIONS["longrope"](config, torch.device("cpu"), seq_len=seq_len)
    got, factor = rotary_inv_freq(96, 10000.0, config.rope_parameters, seq_len=seq_len, max_position_embeddings=longest)
    assert torch.allclose(got.float(), want.float(), rtol=16 * 2 ** -24, atol=0)
    assert math.isclose(factor, want_factor, rel_tol=1e-12)


def test_longrope_without_anything_that_gives_its_factor_is_refused():
    scaling = {"rope_type": "longrope", "short_factor": [1.0] * 48, "long_factor": [2.0] * 48, "original_max_position_embeddings": 4096}
    with pytest.raises(ValueError, match="max_position_embeddings"):
        rotary_inv_freq(96, scaling=scaling)
    assert rotary_inv_freq(96, scaling={**scaling, "attention_factor": 1.0})[1] == 1.0


NEEDED = {
    "linear": ["factor"],
    "dynamic": ["factor", "original_max_position_embeddings"],
    "yarn": ["factor", "original_max_position_embeddings"],
    "llama3": ["factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"],
    "longrope": ["original_max_position_embeddings", "short_factor", "long_factor"],
}


@pytest.mark.parametrize("kind,key", [(kind, key) for kind, keys in NEEDED.items() for key in keys])
@pytest.mark.parametrize("absent", [False, True])
def test_a_dictionary_without_a_key_that_its_type_needs_is_refused_by_name(kind, key, absent):
    scaling = {"rope_type": kind, "low_freq_factor": 1.0, "high_freq_factor": 4.0, **SCALINGS[kind], key: None}
    if absent:
        del scaling[key]
    with pytest.raises(ValueError, match=f"{kind}.*{key}"):
        rotary_inv_freq(128, scaling=scaling, seq_len=None if key == "short_factor" else 20000)


def test_dynamic_scaling_of_a_single_pair_is_refused():
    """The exponent of its base is rotary_dim / (rotary_dim - 2)."""
    with pytest.raises(ValueError, match="dynamic.*rotary_dim"):
        rotary_inv_freq(2, scaling={"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048})
    assert rotary_inv_freq(4, scaling={"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048})[0].shape == (2,)


def test_modes_of_tree_attention_at_the_c_entry_point(cuda_lib):
    """0 and 3, and 4 for bf16 queries: others are refused before anything is looked at; no rows, nothing to do."""
    ok, invalid, unsupported = 0, 1, 2

    def call(mode, q_dtype=2, rows=0):
        return cuda_lib.tq4_tree_attention(
            None, q_dtype, rows, 1, 8, 2, 128, 1024, 128, None, 16 * 272, 272, 8, 16, None, 4, 4, None, None, 0, None, 1, 1, None, 16, None, 16, None,
            0.1, 0, None, 2, 1024, 128, None, 0, None, 0, mode, None, None)

    assert [call(mode) for mode in (0, 3, 4)] == [ok] * 3
    assert [call(mode) for mode in (1, 2, 5, -1)] == [invalid] * 4
    assert call(4, q_dtype=1) == call(4, q_dtype=0) == unsupported
    assert call(0, rows=3) == call(4, rows=3) == invalid
