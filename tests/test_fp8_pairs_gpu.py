"""Products in 8 bits on pairs of SMs (csrc/gemm_fp8.cu) where a pair walks several tiles: the rings of copies and of words of scales run
on from tile to tile, the sums of neighbouring tiles lie at the two ends of tensor memory or one after the other. The way is named, not
left to the estimate. Whole results against float64.

A product of two e4m3 numbers is exact in float32, and so are the powers of two: an output errs by at most K + 1 half ulps of the sum of
the products' magnitudes, and by half a step of its own type (bfloat16: 2^-8 of itself)."""
import random

import pytest
import torch

from test_fp8_gpu import _rows, _tiles, _values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _product(ops, x, xs, w, ws, out, nt, splits=0, epilogue=0, groups=1, tiles=None, n_tiles=None, tile_rows=0):
    """The product by the way of `nt` tokens a tile (256: pairs) and `splits` parts of k."""
    code = ops.F32 if out.dtype == torch.float32 else ops.BF16
    ops._check(ops._fp8_product()(
        x.data_ptr(), x.stride(0), xs.data_ptr(), x.size(0), x.size(0), w.data_ptr(), w.stride(0), ws.data_ptr(), w.size(0), out.data_ptr(),
        out.stride(0), code, epilogue, w.size(0) // groups, x.size(1), groups, None if tiles is None else tiles.data_ptr(),
        None if n_tiles is None else n_tiles.data_ptr(), 0 if tiles is None else tiles.size(0), tile_rows, nt, splits,
        ops.tc_error_flag(x.device).data_ptr(), ops._fp8_stream(x)), "gemm_fp8")
    return out


def _within(y, x, w, before=None):
    """y = x @ w.T (+ before) for the float64 rows x and w."""
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    bound = mag * (x.size(1) + 1) * 2.0 ** -24 + 1e-30
    if y.dtype == torch.bfloat16:
        bound = bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    if before is not None:
        want = want + before
        bound = bound + y.double().abs() * 2.0 ** -23      # half an ulp of the sum
    return bool(((y.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("out", ["bf16", "f32", "residual"])
@pytest.mark.parametrize("K", [640, 896, 1664, 200])                  # 5, 7, 13 and 2 blocks of k; the rings have 6 stages, 4 words
@pytest.mark.parametrize("tokens", [600, 700, 768, 530])              # tiles of 208 (two fit tensor memory), 240, 256, 192 tokens
def test_dense_tiles_that_follow_one_another(tokens, K, out):
    from llm_rs_b200 import ops
    features = 25600 + 72                                             # 303 tiles over 74 pairs
    x, xs = ops.quantize_fp8(_rows(tokens, K, seed=tokens))
    w, ws = ops.quantize_fp8(_rows(features, K, seed=K))
    y = torch.full((tokens, features), 7.0, dtype=torch.bfloat16 if out == "bf16" else torch.float32, device=DEV)
    before = None
    if out == "residual":
        y = _rows(tokens, features, seed=3)
        before = y.double()
    _product(ops, x, xs, w, ws, y, 256, epilogue=out == "residual")
    ops.check_tc_error(DEV)
    assert _within(y, _values(x, xs), _values(w, ws), before)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [640, 1000, 1664])
@pytest.mark.parametrize("seed", [0, 1])
def test_ragged_tiles_that_follow_one_another(seed, K, out_dtype):
    """Short and whole tiles in turn, groups without rows between them."""
    from llm_rs_b200 import ops
    rng = random.Random(seed)
    counts = [rng.choice([1, 17, 256, 256, 233, 130, 5, 0, 300]) for _ in range(41)]
    G, N, rows = len(counts), 2050, sum(counts)                       # nine tiles of features a group
    x, xs = ops.quantize_fp8(_rows(rows, K, seed=seed))
    w, ws = ops.quantize_fp8(_rows(G * N, K, seed=seed + 1))
    tiles, n_tiles, starts = _tiles(counts, 256)
    y = _product(ops, x, xs, w, ws, torch.full((rows, N), 7.0, dtype=out_dtype, device=DEV), 256, groups=G, tiles=tiles, n_tiles=n_tiles,
                 tile_rows=256)
    ops.check_tc_error(DEV)
    xv, wv = _values(x, xs), _values(w, ws).unflatten(0, (G, N))
    for g, (s, n) in enumerate(zip(starts, counts)):
        assert _within(y[s: s + n], xv[s: s + n], wv[g]), g


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,features,K,nt,splits", [(1, 6144, 4096, 16, 5), (60, 1000, 4096, 64, 1), (33, 520, 4096, 32, 3),
                                                         (300, 1000, 2500, 128, 1), (140, 520, 4096, 128, 8), (300, 520, 4096, 256, 1)])
def test_a_result_is_rounded_once(tokens, features, K, nt, splits, out_dtype):
    """Every epilogue (staged, by numbers, from shared sums, from pairs): half a step of the type over the float32 sums' error."""
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(tokens, K, seed=tokens, spread=False))
    w, ws = ops.quantize_fp8(_rows(features, K, seed=features + 1, spread=False))
    y = _product(ops, x, xs, w, ws, torch.empty((tokens, features), dtype=out_dtype, device=DEV), nt, splits)
    ops.check_tc_error(DEV)
    assert _within(y, _values(x, xs), _values(w, ws))


@pytest.mark.parametrize("tokens,features", [(300, 300), (600, 25600)])
def test_a_wait_of_a_pair_that_runs_out_is_reported(tokens, features):
    """A copy that never comes, on pairs with a tile and with several: both blocks give up, say so, and the next product is right."""
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(tokens, 1024))
    w, ws = ops.quantize_fp8(_rows(features, 1024, seed=1))
    y = torch.empty((tokens, features), device=DEV)
    want = _product(ops, x, xs, w, ws, y, 256).clone()
    ops.check_tc_error(DEV)
    ops.set_tc_wait_limit(2000)
    ops.test_skip_copy(gemm_k_block=1)
    try:
        _product(ops, x, xs, w, ws, y, 256)
        torch.cuda.synchronize()
    finally:
        ops.test_skip_copy()
        ops.set_tc_wait_limit()
    with pytest.raises(ops.KernelError, match="gave up"):
        ops.check_tc_error(DEV)
    assert bool((_product(ops, x, xs, w, ws, y, 256) == want).all())
    ops.check_tc_error(DEV)


def test_pairs_and_few_tokens_on_two_streams_at_once():
    """Both kernels in flight together: each as it is alone."""
    from llm_rs_b200 import ops
    sets = []
    for i, (T, N, K, nt, splits) in enumerate(((700, 9000, 2048, 256, 1), (5, 6000, 4096, 16, 4), (90, 4000, 4096, 128, 2))):
        x, w = ops.quantize_fp8(_rows(T, K, seed=i, spread=False)), ops.quantize_fp8(_rows(N, K, seed=i + 5, spread=False))
        sets.append((x, w, T, N, nt, splits))
    alone = [_product(ops, *x, *w, torch.empty((T, N), device=DEV), nt, splits) for x, w, T, N, nt, splits in sets]
    got = [[torch.empty_like(y) for _ in range(20)] for y in alone]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for i in range(20):
        for (x, w, T, N, nt, splits), stream, ys in zip(sets, streams, got):
            with torch.cuda.stream(stream):
                _product(ops, *x, *w, ys[i], nt, splits)
    torch.cuda.synchronize()
    for ys, y in zip(got, alone):
        assert all(bool((z == y).all()) for z in ys)
    ops.check_tc_error(DEV)


def test_a_first_product_that_is_captured_reports_too():
    """Operands made, then the process's first product captured: the word that a wait which runs out is reported in is not the
    graph's own, to be emptied by its replays. Without any call before it, the product is refused."""
    import os
    import subprocess
    import sys
    code = """
import torch
from llm_rs_b200 import ops
a, b = (torch.zeros((n, 256), dtype=torch.float8_e4m3fn, device="cuda:0") for n in (9, 200))
s, t = (torch.zeros((1, n, 4), dtype=torch.float8_e8m0fnu, device="cuda:0") for n in (9, 200))
torch.cuda.synchronize()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        ops.gemm_fp8(a, s, b, t)
except ops.KernelError as e:
    print("refused" if "must not be captured" in str(e) else e)
x, w = (ops.quantize_fp8(torch.randn(n, 256, device="cuda:0")) for n in (9, 200))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.gemm_fp8(*x, *w)
ops.check_tc_error("cuda:0")
ops.tc_error_flag("cuda:0").fill_(1)
g.replay()
torch.cuda.synchronize()
try:
    ops.check_tc_error("cuda:0")
    print("lost")
except ops.KernelError:
    print("reported", bool((y == ops.gemm_fp8(*x, *w)).all()))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.split() == ["refused", "reported", "True"], run.stdout + run.stderr[-2000:]
