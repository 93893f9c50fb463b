"""Rows and products in 8 bits (csrc/fp8_rows.cu, csrc/gemm_fp8.cu) against float64.

Quantised rows are compared bit for bit with a float64 statement of the format, where their input is exact. Where it is computed in
float32 first (the unit, the norm), the computed number errs by some ulps, so a quantised number is one of the two neighbours
of the exact one: it errs by a whole step where the exact one errs by half of one.
A product of two e4m3 numbers is exact in float32, and so are the powers of two: an output errs by at most K + 1 half ulps of the
sum of the products' magnitudes, and half an ulp of its own type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _exact(x):
    """float64 rows -> (what q stands for before its scale, E per block [rows, blocks])."""
    rows, K = x.shape
    nb = -(-K // 128)
    blocks = torch.nn.functional.pad(x, (0, nb * 128 - K)).reshape(rows, nb, 128)
    top = blocks.abs().amax(dim=2)
    e = torch.full_like(top, -127.0)
    for k in range(-126, 121):
        e = torch.where(top > 448.0 * 2.0 ** (k - 1), float(k), e)
    y = blocks / torch.exp2(e)[..., None]
    b = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30)))
    b = torch.where(torch.exp2(b) > y.abs(), b - 1, torch.where(torch.exp2(b + 1) <= y.abs(), b + 1, b)).clamp(min=-6)
    q = torch.round(y * torch.exp2(3 - b)) * torch.exp2(b - 3)
    return q.reshape(rows, nb * 128)[:, :K], e


def _scales(scales, K):
    """E per block [rows, blocks] as float64, and whether the places past the last block hold the least scale."""
    e = scales.view(torch.uint8).transpose(0, 1).reshape(scales.size(1), -1).double() - 127
    nb = -(-K // 128)
    return e[:, :nb], bool((e[:, nb:] == -127).all())


def _values(q, scales):
    rows, K = q.shape
    e, _ = _scales(scales, K)
    return q.double() * torch.exp2(e).repeat_interleave(128, dim=1)[:, :K]


def _rows(*shape, seed=0, spread=True):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn(*shape, generator=g, device=DEV)
    return x * torch.exp2(torch.randint(-20, 20, shape[:-1] + (1,), generator=g, device=DEV).float()) if spread else x


# -- rows -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 16), (3, 127), (9, 128), (2, 129), (17, 512), (5, 513), (64, 2200), (8, 4096), (700, 5005),
                                    (2, 16400)])
def test_quantize_is_the_nearest_number(rows, K, dtype):
    from llm_rs_b200 import ops
    x = _rows(rows, K, seed=rows + K).to(dtype)
    x[0, : min(K, 40)] = 0.0                      # (with K <= 40 an empty block)
    x[-1, K // 2] = 448.0 * 2.0 ** 30             # exactly the largest number, and rows far below it
    q, scales = ops.quantize_fp8(x)
    want, e = _exact(x.double())
    got_e, filled = _scales(scales, K)
    assert filled and bool((got_e == e).all())
    assert bool((q.double() == want).all())
    assert q.stride(0) % 16 == 0 and scales.shape == (-(-K // 512), rows, 4)


@pytest.mark.parametrize("top", [2.0 ** -149, 2.0 ** -130, 448 * 2.0 ** -127, 449 * 2.0 ** -127, 1.0, 447.0, 448.0, 449.0, 896.0, 3.4e38])
def test_quantize_at_the_borders_of_the_scales(top):
    from llm_rs_b200 import ops
    x = torch.tensor([[top, -top, top / 3, top / 7, 0.0, -0.0] * 30], device=DEV)
    q, scales = ops.quantize_fp8(x)
    want, e = _exact(x.double())
    assert bool((_scales(scales, 180)[0] == e).all()) and bool((q.double() == want).all())


def test_quantize_ties_go_to_even():
    from llm_rs_b200 import ops
    x = torch.tensor([[448.0, 17.0, 19.0, 17.0 + 2.0 ** -15, 0.0009765625, 0.0029296875, -17.0, -19.0]], device=DEV)
    q, _ = ops.quantize_fp8(x)
    assert q.double().tolist() == [[448.0, 16.0, 20.0, 18.0, 0.0, 0.00390625, -16.0, -20.0]]


@pytest.mark.parametrize("K", [512, 515])
def test_quantize_what_is_no_number(K):
    """NaN and infinities become NaN; their blocks' finite numbers stay finite, other blocks are as without them."""
    from llm_rs_b200 import ops
    x = _rows(4, K, spread=False)
    clean, clean_s = ops.quantize_fp8(x)
    x[0, 5], x[1, 130], x[2, 300], x[3, 0:128] = float("nan"), float("inf"), float("-inf"), float("nan")
    q, s = ops.quantize_fp8(x)
    bad = ~torch.isfinite(x)
    assert bool(q.float()[bad].isnan().all()) and bool(q.float()[~bad].isfinite().all())
    touched = torch.zeros_like(bad)
    for r, b in ((0, 0), (1, 1), (2, 2), (3, 0)):
        touched[r, 128 * b: 128 * (b + 1)] = True
    assert bool((q.float() == clean.float())[~touched].all())
    assert bool((q.float() == clean.float())[0][~bad[0]].all())      # a NaN does not enter the scale
    y = ops.gemm_fp8(q, s, *ops.quantize_fp8(_rows(70, K, seed=1, spread=False)), out_dtype=torch.float32)
    assert bool(y.isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [256, 250])
def test_quantize_rows_that_are_picked_and_strided(K, dtype):
    from llm_rs_b200 import ops
    wide = _rows(40, K + 70, seed=3).to(dtype)
    x = wide[3:33, 32: 32 + K]
    q, s = ops.quantize_fp8(x)
    want, e = _exact(x.double())
    assert bool((q.double() == want).all()) and bool((_scales(s, K)[0] == e).all())
    src = torch.tensor([0, 29, 29, 7, -1, 30, 3, 0, 0], dtype=torch.int32, device=DEV)
    q2, s2 = ops.quantize_fp8(x, src)
    for i, r in enumerate(src.tolist()):
        if 0 <= r < 30:
            assert bool((q2[i].float() == q[r].float()).all()) and bool((s2[:, i].view(torch.uint8) == s[:, r].view(torch.uint8)).all())
        else:
            assert not bool(q2[i].view(torch.uint8).any()) and not bool(s2[:, i].view(torch.uint8).any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_picks_from_no_rows(dtype):
    """Sources that name nothing, of a matrix without rows that starts in the middle of an aligned pair: zeros, and nothing is read."""
    from llm_rs_b200 import ops
    x = _rows(5, 1501, spread=False).to(dtype)
    src = torch.tensor([0, 4, -1], dtype=torch.int32, device=DEV)
    for part in (x[3:3], x[5:], x[:0]):
        q, s = ops.quantize_fp8(part, src)
        assert not bool(q.view(torch.uint8).any()) and not bool(s.view(torch.uint8).any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [511, 512, 514, 516, 528, 1501])
@pytest.mark.parametrize("off", [0, 1, 2, 4, 7])
def test_quantize_from_any_address(K, off, dtype):
    """Rows and pitches of every alignment, with numbers on both sides that must not matter."""
    from llm_rs_b200 import ops
    for pitch in (K + off, K + 8 + off):
        wide = torch.full((6 * pitch + off,), float("inf"), device=DEV, dtype=dtype)
        x = wide[off:].view(6, pitch)[:, :K]
        x.copy_(_rows(6, K, seed=K))
        q, s = ops.quantize_fp8(x)
        want, e = _exact(x.double())
        assert bool((q.double() == want).all()) and bool((_scales(s, K)[0] == e).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter,block", [(511, 0), (514, 0), (516, 0), (1040, 0), (640, 16), (516, 4), (515, 5), (512, 2), (1040, 80)])
def test_unit_from_any_address(inter, block, dtype):
    """Columns of every alignment and order: as the same columns are from dense rows."""
    from llm_rs_b200 import ops
    for off in (0, 1, 4, 6):
        wide = torch.full((5, 2 * inter + off + 3), float("inf"), device=DEV, dtype=dtype)
        gu = wide[:, off: off + 2 * inter]
        gu.copy_(_rows(5, 2 * inter, seed=inter, spread=False))
        both = gu.double().reshape(5, -1, 2, block or inter)
        gate, up = both[:, :, 0].reshape(5, inter), both[:, :, 1].reshape(5, inter)
        assert _neighbour(*ops.silu_mul_fp8(gu, block), gate * torch.sigmoid(gate) * up, inter)


def _neighbour(q, scales, x, K):
    """Whether (q, scales) stand for a neighbour of the float64 rows x: a whole step of e4m3 (2^-3 of a number in [1, 2)), or of its
    subnormal numbers. A block whose maximum lies at a border may have the scale above it: its step is twice that."""
    got = _values(q, scales)
    e, _ = _scales(scales, K)
    _, want_e = _exact(x)
    assert bool(((e - want_e).abs() <= 1).all()) and float((e != want_e).double().mean()) < 1e-3
    step = torch.maximum(x.abs() * 2.0 ** -3, torch.exp2(e).repeat_interleave(128, dim=1)[:, :K] * 2.0 ** -9)
    return bool(((got - x).abs() <= step).all()) and float((got - x).norm() / x.norm()) < 2.0 ** -4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,inter,block", [(1, 64, 64), (3, 640, 64), (33, 12288, 64), (5, 640, 0), (2, 333, 0), (7, 520, 8), (1, 1, 0),
                                              (600, 1000, 0)])
def test_unit(rows, inter, block, dtype):
    from llm_rs_b200 import ops
    gu = (2 * _rows(rows, 2 * inter, seed=inter, spread=False)).to(dtype)
    both = gu.double().reshape(rows, -1, 2, block or inter)
    gate, up = both[:, :, 0].reshape(rows, inter), both[:, :, 1].reshape(rows, inter)
    assert _neighbour(*ops.silu_mul_fp8(gu, block), gate * torch.sigmoid(gate) * up, inter)
    g, u = gate.clamp(max=1.5), up.clamp(-1.5, 1.5)
    assert _neighbour(*ops.silu_mul_fp8(gu, block, unit=(1.5, 1.702, 1.0)), g * torch.sigmoid(1.702 * g) * (u + 1), inter)


@pytest.mark.parametrize("dtype", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K", [(1, 16), (3, 64), (9, 333), (8, 4096), (700, 5120), (2, 16384), (2, 16400), (3, 20001), (1, 1)])
def test_norm(rows, K, dtype):
    from llm_rs_b200 import ops
    h = 3 * _rows(rows, K, seed=K, spread=False)
    w = 1 + 0.1 * _rows(1, K, seed=1, spread=False)[0]
    d = None if dtype is None else _rows(rows, K, seed=2, spread=False).to(dtype)
    before = h.clone()
    pick = torch.tensor([rows - 1, 0, 0, -1, rows], dtype=torch.int32, device=DEV)
    picked = ops.add_rmsnorm_fp8(h, d, w, 1e-6, rows=pick)
    assert bool((h == before).all())
    q, s = ops.add_rmsnorm_fp8(h, d, w, 1e-6)
    want_h = before if d is None else before + d.float()
    assert bool((h == want_h).all())
    x = want_h.double()
    assert _neighbour(q, s, x / torch.sqrt(x.square().mean(dim=1, keepdim=True) + 1e-6) * w.double(), K)
    for i, r in enumerate(pick.tolist()):
        if 0 <= r < rows:
            assert bool((picked[0][i].float() == q[r].float()).all())
        else:
            assert not bool(picked[0][i].view(torch.uint8).any()) and not bool(picked[1][:, i].view(torch.uint8).any())


@pytest.mark.parametrize("K", [512, 515, 17000])
def test_norm_of_rows_out_of_range(K):
    """Squares past float32, an infinity, a NaN: that row is NaN, its neighbours are as they are without it."""
    from llm_rs_b200 import ops
    h = _rows(6, K, spread=False)
    w = torch.ones(K, device=DEV)
    q, s = ops.add_rmsnorm_fp8(h.clone(), None, w, 1e-6)
    h[0] *= 1e25
    h[2, K - 1], h[4, 0], h[5] = float("inf"), float("nan"), 0.0
    q2, s2 = ops.add_rmsnorm_fp8(h, None, w, 1e-6)
    assert all(bool(q2[r].float().isnan().all()) for r in (0, 4)) and bool(q2[2, K - 1].float().isnan())
    assert not bool(q2[5].view(torch.uint8).any())
    for r in (1, 3):
        assert bool((q2[r].float() == q[r].float()).all()) and bool((s2[:, r].view(torch.uint8) == s[:, r].view(torch.uint8)).all())


# -- products ---------------------------------------------------------------------------------------------------------
def _bound(x, w, out_dtype, K):
    mag = x.abs() @ w.abs().t()
    return mag * (K + 1) * 2.0 ** -24 + (mag * 2.0 ** -8 if out_dtype == torch.bfloat16 else 0.0) + 1e-30


SHAPES = [(1, 64, 64), (1, 6144, 4096), (2, 100, 128), (15, 1000, 1000), (16, 128, 512), (17, 130, 640), (31, 24576, 512), (33, 257, 129),
          (64, 4096, 4096), (65, 127, 300), (100, 4096, 1024), (129, 300, 2048), (255, 640, 33), (256, 256, 256), (257, 1000, 777),
          (333, 2200, 5005), (600, 24576, 256), (2048, 1024, 4096), (1, 1, 1), (5, 33, 16384)]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,features,K", SHAPES)
def test_product(tokens, features, K, out_dtype):
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(tokens, K, seed=tokens))
    w, ws = ops.quantize_fp8(_rows(features, K, seed=features + 1))
    y = ops.gemm_fp8(x, xs, w, ws, out_dtype=out_dtype)
    ops.check_tc_error(DEV)
    xv, wv = _values(x, xs), _values(w, ws)
    want, bound = xv @ wv.t(), _bound(xv, wv, out_dtype, K)
    assert y.dtype == out_dtype and bool(((y.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens,features,K", [(1, 100, 300), (40, 4096, 4096), (129, 300, 513), (2048, 512, 256)])
def test_product_into_the_stream_and_strided(tokens, features, K):
    from llm_rs_b200 import ops
    big, bigs = ops.quantize_fp8(_rows(tokens + 9, K, seed=5, spread=False))
    x, xs = big[4: 4 + tokens], bigs[:, 4: 4 + tokens]
    wide, wides = ops.quantize_fp8(_rows(features + 50, K, seed=6, spread=False))
    w, ws = wide[50:], wides[:, 50:]
    xv, wv = _values(x, xs), _values(w, ws)
    want, bound = xv @ wv.t(), _bound(xv, wv, torch.float32, K)
    h = _rows(tokens, features + 3, seed=7, spread=False)
    before = h.clone()
    assert ops.gemm_fp8(x, xs, w, ws, out=h[:, 1: 1 + features], epilogue="residual") .data_ptr() == h[:, 1:].data_ptr()
    got = h[:, 1: 1 + features].double()
    # Half an ulp of the sum on top.
    assert bool(((got - (before[:, 1: 1 + features].double() + want)).abs() <= bound + got.abs() * 2.0 ** -23).all())
    assert bool((h[:, 0] == before[:, 0]).all()) and bool((h[:, 1 + features:] == before[:, 1 + features:]).all())
    out = torch.full((tokens + 2, features + 5), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.gemm_fp8(x, xs, w, ws, out=out[1: 1 + tokens, 2: 2 + features])
    assert bool(((out[1: 1 + tokens, 2: 2 + features].double() - want).abs() <= _bound(xv, wv, torch.bfloat16, K)).all())
    out[1: 1 + tokens, 2: 2 + features] = 7.0
    assert bool((out == 7.0).all())
    ops.check_tc_error(DEV)


def test_product_of_no_rows():
    from llm_rs_b200 import ops
    w, ws = ops.quantize_fp8(_rows(64, 256))
    x, xs = ops.quantize_fp8(torch.empty((0, 256), device=DEV))
    assert ops.gemm_fp8(x, xs, w, ws).shape == (0, 64)


def test_product_does_not_depend_on_the_other_rows():
    """A token's numbers in a step of 40 are those in a step of 33 of the same kernel, bit for bit, and the same twice."""
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(40, 2048, seed=1))
    w, ws = ops.quantize_fp8(_rows(1000, 2048, seed=2))
    y = ops.gemm_fp8(x, xs, w, ws, out_dtype=torch.float32)
    assert bool((ops.gemm_fp8(x, xs, w, ws, out_dtype=torch.float32) == y).all())
    assert bool((ops.gemm_fp8(x[7:], xs[:, 7:], w, ws, out_dtype=torch.float32) == y[7:]).all())


def _tiles(counts, tile_rows, spare=3):
    starts = [sum(counts[:g]) for g in range(len(counts))]
    tiles = [(g, s + a, min(tile_rows, n - a)) for g, (s, n) in enumerate(zip(starts, counts)) for a in range(0, n, tile_rows)]
    return (torch.tensor(tiles + [(0, 0, 0)] * spare, dtype=torch.int32, device=DEV),
            torch.tensor([len(tiles)], dtype=torch.int32, device=DEV), starts)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tile_rows", [8, 16, 32, 64, 128, 200, 256])
@pytest.mark.parametrize("N,K,counts", [(256, 64, [129, 0, 1, 128, 300]), (200, 72, [500, 20]), (1000, 136, [7, 257, 130]),
                                        (64, 2048, [384]), (33, 200, [128, 128, 5]), (1, 515, [1, 1, 0, 2]),
                                        (2048, 2048, [3, 0, 9, 1, 0, 40, 2])])
def test_grouped(N, K, counts, tile_rows, out_dtype):
    from llm_rs_b200 import ops
    G, rows = len(counts), sum(counts)
    x, xs = ops.quantize_fp8(_rows(rows, K, seed=K))
    w, ws = ops.quantize_fp8(_rows(G * N, K, seed=N))
    tiles, n_tiles, starts = _tiles(counts, tile_rows)
    out = torch.full((rows, N), 7.0, device=DEV, dtype=out_dtype)
    ops.gemm_fp8_grouped(x, xs, w.unflatten(0, (G, N)), ws, out, tiles, n_tiles, tile_rows)
    ops.check_tc_error(DEV)
    xv, wv = _values(x, xs), _values(w, ws).unflatten(0, (G, N))
    for g, (s, n) in enumerate(zip(starts, counts)):
        want, bound = xv[s: s + n] @ wv[g].t(), _bound(xv[s: s + n], wv[g], out_dtype, K)
        assert bool(((out[s: s + n].double() - want).abs() <= bound).all()), g


def test_grouped_tiles_that_name_nothing():
    """Entries past n_tiles, groups and rows that are not there, tiles of no rows, tiles that end past the rows: nothing but the
    rows that a tile names is written."""
    from llm_rs_b200 import ops
    G, N, K, rows = 3, 200, 256, 50
    x, xs = ops.quantize_fp8(_rows(rows, K))
    w, ws = ops.quantize_fp8(_rows(G * N, K, seed=1))
    tiles = torch.tensor([(0, 0, 10), (3, 10, 10), (-1, 20, 10), (1, 50, 4), (1, -5, 9), (2, 45, 32), (1, 30, 0), (1, 30, -4), (0, 20, 10)],
                         dtype=torch.int32, device=DEV)
    out = torch.full((rows, N), 7.0, device=DEV)
    ops.gemm_fp8_grouped(x, xs, w.unflatten(0, (G, N)), ws, out, tiles, torch.tensor([8], dtype=torch.int32, device=DEV), 32)
    ops.check_tc_error(DEV)
    xv, wv = _values(x, xs), _values(w, ws).unflatten(0, (G, N))
    for rs, g in ((slice(0, 10), 0), (slice(45, 50), 2)):
        assert bool(((out[rs].double() - xv[rs] @ wv[g].t()).abs() <= _bound(xv[rs], wv[g], torch.float32, K)).all())
    assert bool((out[10:45] == 7.0).all())
    # More tiles announced than the list holds, and none.
    out.fill_(7.0)
    ops.gemm_fp8_grouped(x, xs, w.unflatten(0, (G, N)), ws, out, tiles[:1], torch.tensor([100], dtype=torch.int32, device=DEV), 32)
    assert bool((out[10:] == 7.0).all()) and not bool((out[:10] == 7.0).any())
    out.fill_(7.0)
    ops.gemm_fp8_grouped(x, xs, w.unflatten(0, (G, N)), ws, out, tiles[:0], torch.tensor([0], dtype=torch.int32, device=DEV), 32)
    ops.gemm_fp8_grouped(x, xs, w.unflatten(0, (G, N)), ws, out, tiles, torch.tensor([0], dtype=torch.int32, device=DEV), 32)
    assert bool((out == 7.0).all())


# -- together, and how they are used ------------------------------------------------------------------------------------
def _layer(ops, h, d, norm_w, w_gu, w_down):
    x = ops.add_rmsnorm_fp8(h, d, norm_w, 1e-6)
    act = ops.silu_mul_fp8(ops.gemm_fp8(*x, *w_gu), block=64)
    return ops.gemm_fp8(*act, *w_down, out=h, epilogue="residual")


@pytest.mark.parametrize("tokens", [1, 30, 300])
def test_a_feed_forward_of_them_on_a_stream_and_captured(tokens):
    """norm -> gate|up -> unit -> down into the stream: on a stream of its own, and captured into two graphs whose replays read new
    inputs, the same bits as the plain calls."""
    from llm_rs_b200 import ops
    H, I = 512, 640
    w_gu, w_down = ops.quantize_fp8(0.05 * _rows(2 * I, H, seed=1, spread=False)), ops.quantize_fp8(0.05 * _rows(H, I, seed=2, spread=False))
    norm_w = 1 + 0.1 * _rows(1, H, seed=3, spread=False)[0]
    inputs = [(_rows(tokens, H, seed=10 + i, spread=False), _rows(tokens, H, seed=20 + i, spread=False).bfloat16()) for i in range(3)]
    want = [_layer(ops, h.clone(), d, norm_w, w_gu, w_down) for h, d in inputs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for (h, d), y in zip(inputs, want):
            assert bool((_layer(ops, h.clone(), d, norm_w, w_gu, w_down) == y).all())
    side.synchronize()
    graphs = []
    for _ in range(2):
        h, d = inputs[0][0].clone(), inputs[0][1].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _layer(ops, h, d, norm_w, w_gu, w_down)
        graphs.append((g, h, d))
    for i in (1, 2, 0):
        for g, h, d in graphs:
            h.copy_(inputs[i][0])
            d.copy_(inputs[i][1])
        for g, h, d in graphs:
            g.replay()
        for g, h, d in graphs:
            assert bool((h == want[i]).all())
    # Against float64 of the same formula without 8 bits: every quantised number errs by 2^-4 of itself at most, three in a row.
    h, d = inputs[0]
    s = h.double() + d.double()
    x = s / torch.sqrt(s.square().mean(dim=1, keepdim=True) + 1e-6) * norm_w.double()
    gu = (x @ (0.05 * _rows(2 * I, H, seed=1, spread=False).double()).t()).reshape(tokens, -1, 2, 64)
    act = (gu[:, :, 0] * torch.sigmoid(gu[:, :, 0]) * gu[:, :, 1]).reshape(tokens, I)
    y = s + act @ (0.05 * _rows(H, I, seed=2, spread=False).double()).t()
    assert float((want[0].double() - y).norm() / (y - s).norm()) < 5 * 2.0 ** -4


def test_quantised_just_before_the_product():
    """Weights made by the kernel before the product on the same stream are whole when it reads them."""
    from llm_rs_b200 import ops
    for seed in range(20):
        x, xs = ops.quantize_fp8(_rows(3, 4096, seed=seed, spread=False))
        wr = _rows(2048, 4096, seed=seed + 50, spread=False)
        y = ops.gemm_fp8(x, xs, *ops.quantize_fp8(wr), out_dtype=torch.float32)
        torch.cuda.synchronize()
        w, ws = ops.quantize_fp8(wr)
        torch.cuda.synchronize()
        assert bool((ops.gemm_fp8(x, xs, w, ws, out_dtype=torch.float32) == y).all())


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_wait_that_runs_out_is_reported(tokens):
    """A copy that never comes: the block gives up, says so, and the next product is right again."""
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(tokens, 1024))
    w, ws = ops.quantize_fp8(_rows(300, 1024, seed=1))
    want = ops.gemm_fp8(x, xs, w, ws, out_dtype=torch.float32)
    ops.check_tc_error(DEV)
    ops.set_tc_wait_limit(2000)
    ops.test_skip_copy(gemm_k_block=1)
    try:
        ops.gemm_fp8(x, xs, w, ws)
        torch.cuda.synchronize()
    finally:
        ops.test_skip_copy()
        ops.set_tc_wait_limit()
    with pytest.raises(ops.KernelError, match="gave up"):
        ops.check_tc_error(DEV)
    assert bool((ops.gemm_fp8(x, xs, w, ws, out_dtype=torch.float32) == want).all())
    ops.check_tc_error(DEV)


@pytest.mark.parametrize("seed", range(30))
def test_products_of_any_sizes(seed):
    """Sizes that nobody chose, dense and grouped (with tiles of any height): the ways that the estimate picks among."""
    import random
    from llm_rs_b200 import ops
    rng = random.Random(seed)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
    T, N, K = log(1, 5000), log(1, 9000), log(1, 9000)
    while T * N * K > 2e10:
        T, N, K = (T + 1) // 2, (N + 2) // 3 if N > 3000 else N, (K + 1) // 2
    x, xs = ops.quantize_fp8(_rows(T, K, seed=seed))
    w, ws = ops.quantize_fp8(_rows(N, K, seed=seed + 1))
    xv, wv = _values(x, xs), _values(w, ws)
    y = ops.gemm_fp8(x, xs, w, ws, out_dtype=torch.float32)
    assert bool(((y.double() - xv @ wv.t()).abs() <= _bound(xv, wv, torch.float32, K)).all()), (T, N, K)
    G = min(rng.choice([1, 2, 7, 30]), N)
    N //= G
    cuts = sorted(rng.randint(0, T) for _ in range(G - 1))
    counts = [b - a for a, b in zip([0] + cuts, cuts + [T])]
    tile_rows = rng.randint(1, 256)
    tiles, n_tiles, starts = _tiles(counts, tile_rows)
    out = torch.full((T, N), 7.0, device=DEV)
    ops.gemm_fp8_grouped(x, xs, w[: G * N].unflatten(0, (G, N)), ws[:, : G * N], out, tiles, n_tiles, tile_rows)
    for g, (s, n) in enumerate(zip(starts, counts)):
        wg = wv[g * N: (g + 1) * N]
        assert bool(((out[s: s + n].double() - xv[s: s + n] @ wg.t()).abs() <= _bound(xv[s: s + n], wg, torch.float32, K)).all()), (T, N, K, G)
    ops.check_tc_error(DEV)


def test_places_past_two_to_the_thirty_one():
    """Rows, results and streams whose places do not fit 32 bits; the last rows are right."""
    from llm_rs_b200 import ops
    K, rows = 4096, 530_000
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _rows(3, K, spread=False).bfloat16()
    q, s = ops.quantize_fp8(x)
    del x
    tail, tail_s = ops.quantize_fp8(_rows(3, K, spread=False).bfloat16())
    assert bool((q[-3:].float() == tail.float()).all()) and bool((s[:, -3:].view(torch.uint8) == tail_s.view(torch.uint8)).all())
    w, ws = ops.quantize_fp8(_rows(100, K, seed=1, spread=False))
    y = ops.gemm_fp8(q, s, w, ws, out_dtype=torch.float32)
    assert not bool(y[:-3].any())
    xv, wv = _values(tail, tail_s), _values(w, ws)
    assert bool(((y[-3:].double() - xv @ wv.t()).abs() <= _bound(xv, wv, torch.float32, K)).all())
    del q, s, y
    x, xs = ops.quantize_fp8(_rows(300_000, 64, seed=2, spread=False))
    w, ws = ops.quantize_fp8(_rows(8192, 64, seed=3, spread=False))
    y = ops.gemm_fp8(x, xs, w, ws)
    for at in (slice(0, 2), slice(262_140, 262_150), slice(299_990, 300_000)):
        xv, wv = _values(x[at], xs[:, at]), _values(w, ws)
        assert bool(((y[at].double() - xv @ wv.t()).abs() <= _bound(xv, wv, torch.bfloat16, 64)).all())
    ops.check_tc_error(DEV)


def test_two_streams_at_once():
    """Products of both kernels, quantised rows between them, in flight on two streams: each as it is alone."""
    from llm_rs_b200 import ops
    sets = []
    for i, (T, N, K) in enumerate(((700, 3000, 2048), (5, 6000, 4096))):
        sets.append((_rows(T, K, seed=i, spread=False), ops.quantize_fp8(_rows(N, K, seed=i + 5, spread=False))))
    alone = [ops.gemm_fp8(*ops.quantize_fp8(x), *w, out_dtype=torch.float32) for x, w in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(30):
        for i, ((x, w), stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(ops.gemm_fp8(*ops.quantize_fp8(x), *w, out_dtype=torch.float32))
    torch.cuda.synchronize()
    for ys, y in zip(got, alone):
        assert all(bool((z == y).all()) for z in ys)
    ops.check_tc_error(DEV)


@pytest.mark.parametrize("nt,splits", [(16, 1), (16, 3), (16, 8), (32, 2), (32, 7), (64, 1), (64, 5), (128, 1), (128, 2), (128, 8), (256, 1)])
@pytest.mark.parametrize("tokens,features,K", [(1, 130, 1100), (27, 300, 4000), (140, 520, 1024), (300, 1000, 2500)])
def test_every_way_of_a_product(tokens, features, K, nt, splits):
    """Tokens a tile and blocks that share a tile's k, whatever the estimate would take for these sizes."""
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(tokens, K, seed=tokens))
    w, ws = ops.quantize_fp8(_rows(features, K, seed=features + 1))
    y = torch.empty((tokens, features), device=DEV)
    ops._check(ops._fp8_product()(
        x.data_ptr(), x.stride(0), xs.data_ptr(), tokens, tokens, w.data_ptr(), w.stride(0), ws.data_ptr(), features, y.data_ptr(),
        features, ops.F32, 0, features, K, 1, None, None, 0, 0, nt, splits, ops.tc_error_flag(DEV).data_ptr(), ops._fp8_stream(x)), "gemm_fp8")
    ops.check_tc_error(DEV)
    xv, wv = _values(x, xs), _values(w, ws)
    assert bool(((y.double() - xv @ wv.t()).abs() <= _bound(xv, wv, torch.float32, K)).all())


@pytest.mark.parametrize("rows,N,K,tile_rows", [(5, 256, 2048, 16), (5, 130, 4096, 32), (300, 512, 1024, 128), (300, 512, 2048, 256)])
def test_lists_with_room_for_many_more_tiles(rows, N, K, tile_rows):
    """No tile, one, or a number below zero, of a list with room for fifty: blocks without a tile leave, shared ranges of k or not."""
    from llm_rs_b200 import ops
    x, xs = ops.quantize_fp8(_rows(rows, K, seed=1))
    w, ws = ops.quantize_fp8(_rows(2 * N, K, seed=2))
    xv, wv = _values(x, xs), _values(w, ws)
    tiles = torch.tensor([(1, rows - 3, 3)] + [(0, 0, min(rows, tile_rows))] * 49, dtype=torch.int32, device=DEV)
    for n in (0, 1, -4, 0):
        out = torch.full((rows, N), 7.0, device=DEV)
        ops.gemm_fp8_grouped(x, xs, w.unflatten(0, (2, N)), ws, out, tiles, torch.tensor([n], dtype=torch.int32, device=DEV), tile_rows)
        assert bool((out[: rows - 3 if n == 1 else rows] == 7.0).all())
        if n == 1:
            assert bool(((out[-3:].double() - xv[-3:] @ wv[N:].t()).abs() <= _bound(xv[-3:], wv[N:], torch.float32, K)).all())
    ops.check_tc_error(DEV)
