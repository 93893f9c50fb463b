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


def _meta(*shape, dtype):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("many", [0x7ffffe01, 2 ** 31, 2 ** 32, 2 ** 32 + 8])
def test_sizes_past_32_bits_are_refused(many):
    """They would reach the kernels cut to 32 bits: 2^32 rows as none, 2^32 + 8 as eight."""
    E4, E8, I32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int32

    def refused(f, *a, **k):
        with pytest.raises(ops.KernelError, match="at most 2147483136 rows"):
            f(*a, **k)
    narrow, wide, index = _meta(many, 2, dtype=torch.bfloat16), _meta(2, many, dtype=torch.bfloat16), _meta(many, dtype=I32)
    for x in (narrow, wide):
        refused(ops.quantize_fp8, x)
        refused(ops.silu_mul_fp8, x)
        refused(ops.add_rmsnorm_fp8, x.float(), None, _meta(x.size(1), dtype=torch.float32), 1e-6)
    refused(ops.quantize_fp8, _meta(4, 64, dtype=torch.float32), index)
    refused(ops.add_rmsnorm_fp8, _meta(4, 64, dtype=torch.float32), None, _meta(64, dtype=torch.float32), 1e-6, rows=index)
    few = (_meta(4, 16, dtype=E4), _meta(1, 4, 4, dtype=E8))
    tall, long = (_meta(many, 16, dtype=E4), _meta(1, many, 4, dtype=E8)), (_meta(4, many, dtype=E4), _meta((many + 511) // 512, 4, 4, dtype=E8))
    for x, w in ((tall, few), (few, tall), (long, long)):
        refused(ops.gemm_fp8, *x, *w)
    tiles, n = _meta(3, 3, dtype=I32), _meta(1, dtype=I32)
    grouped = lambda x, w, g, tiles: ops.gemm_fp8_grouped(*x, w[0].unflatten(0, (g, -1)), w[1], _meta(x[0].size(0), w[0].size(0) // g,
                                                          dtype=torch.float32), tiles, n, 64)
    refused(grouped, tall, few, 2, tiles)
    refused(grouped, few, tall, many, tiles)
    refused(grouped, few, few, 2, _meta(many, 3, dtype=I32))


def test_bytes_that_the_profiler_counts():
    """What each operator has to read and to write, whatever it is called with."""
    from llm_rs_b200.profiling import WRAPPED
    E4, E8, I32, BF, F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int32, torch.bfloat16, torch.float32
    cost = lambda name, *a, **k: WRAPPED[name](*a, **k)[1]
    eight = lambda rows, K: rows * K + rows * ((K + 511) // 512) * 4
    x, src = _meta(10, 1000, dtype=BF), _meta(35, dtype=I32)
    assert cost("quantize_fp8", x) == 10 * 1000 * 2 + eight(10, 1000)
    assert cost("quantize_fp8", x.float()) == 10 * 1000 * 4 + eight(10, 1000)
    assert cost("quantize_fp8", x, src) == 10 * 1000 * 2 + 35 * 4 + eight(35, 1000)
    assert cost("quantize_fp8", x, src[:3]) == 3 * 1000 * 2 + 3 * 4 + eight(3, 1000)
    assert cost("silu_mul_fp8", x, block=100, unit=(7.0, 1.0, 0.0)) == 10 * 1000 * 2 + eight(10, 500)
    h, w = _meta(10, 1000, dtype=F32), _meta(1000, dtype=F32)
    assert cost("add_rmsnorm_fp8", h, None, w, 1e-6) == 10 * 1000 * 4 + 4000 + eight(10, 1000)
    assert cost("add_rmsnorm_fp8", h, x, w, 1e-6) == 10 * 1000 * (4 + 2 + 4) + 4000 + eight(10, 1000)
    assert cost("add_rmsnorm_fp8", h, x, w, 1e-6, rows=src[:4]) == 4 * 1000 * (4 + 2) + 4 * 4 + 4000 + eight(4, 1000)
    q, s = _meta(10, 1000, dtype=E4), _meta(2, 10, 4, dtype=E8)
    v, t = _meta(300, 1000, dtype=E4), _meta(2, 300, 4, dtype=E8)
    assert cost("gemm_fp8", q, s, v, t) == eight(10, 1000) + eight(300, 1000) + 10 * 300 * 2
    assert cost("gemm_fp8", q, s, v, t, out=_meta(10, 300, dtype=F32), epilogue="residual") == eight(10, 1000) + eight(300, 1000) + 10 * 300 * 8
    # Three groups and ten rows dealt evenly: 3 (1 - (2/3)^10) groups have one.
    got = cost("gemm_fp8_grouped", q, s, v.unflatten(0, (3, 100)), t, _meta(10, 100, dtype=BF), _meta(5, 3, dtype=I32), _meta(1, dtype=I32), 64)
    assert abs(got - (3 * (1 - (2 / 3) ** 10) * eight(100, 1000) + eight(10, 1000) + 10 * 100 * 2)) <= 2


def test_products_in_8_bits_are_reported_against_their_own_rate(monkeypatch):
    from llm_rs_b200.profiling import Profiler

    class Event:
        def __init__(self, ms):
            self.ms = ms

        def elapsed_time(self, other):
            return other.ms - self.ms
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    p = Profiler(hbm_gbs=1000.0, tflops=1.0)
    # A millisecond each: 1e9 operations are the bfloat16 rate, half of the 8-bit rate; 3e8 bytes are 0.3 of the memory's.
    for name in ("gemm_bf16[8x8]", "gemm_fp8[8x8]", "gemm_fp8_grouped[2x8x8]"):
        p._calls.append((name, 3e8, 1e9, Event(0.0), Event(1.0)))
    got = {r["class"].split("[")[0]: (r["frac"], r["bound"]) for r in p.classes()}
    assert got == {"gemm_bf16": (1.0, "tensor"), "gemm_fp8": (0.5, "tensor"), "gemm_fp8_grouped": (0.5, "tensor")}
