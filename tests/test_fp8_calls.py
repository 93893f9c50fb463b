"""How rows and products in 8 bits are called and accounted for, without a GPU."""
import pytest
import torch

from llm_rs_b200 import ops


def test_engine_fields_keep_their_places():
    """Callers may name the engine's fields by place: what came later stands last."""
    from llm_rs_b200.engine import EngineConfig
    c = EngineConfig("folder", 1024, 16, "bfloat16", "cuda:0", 7, 300, 200, False, False)
    assert (c.max_requests, c.max_tokens_per_step, c.prefill_chunk, c.cuda_graphs, c.async_steps, c.products) == (7, 300, 200, False, False, "stored")
    assert EngineConfig("folder", products="fp8").products == "fp8"
