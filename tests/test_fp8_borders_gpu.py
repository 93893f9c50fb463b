"""Rows in 8 bits that are computed on the way (the norm, the gated unit), held to the nearest number.

What a kernel computes before its one rounding to e4m3 errs by a share `slack` of itself, which follows from its operations. So the
quantised number errs from the exact one by half a step of e4m3 (2^-4 of the number's power of two, 2^-10 * 2^E where it is subnormal)
and by the slack, and a block's scale is the exact one unless its largest magnitude lies within the slack of a border. A kernel that cut
numbers off instead of rounding them would be off by up to a step."""
import pytest
import torch

from test_fp8_gpu import _exact, _rows, _scales, _values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")


def _nearest(q, scales, x, slack):
    """Whether (q, scales) are the float64 rows x rounded once, where x may be off by `slack` (a number, or one for every number of x)."""
    K = x.size(1)
    e, filled = _scales(scales, K)
    _, lower = _exact(x.abs() * (1 - slack))
    _, upper = _exact(x.abs() * (1 + slack))
    assert filled and bool((e >= lower).all()) and bool((e <= upper).all())
    power = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -1000))))
    step = torch.maximum(power * 2.0 ** -3, torch.exp2(e).repeat_interleave(128, dim=1)[:, :K] * 2.0 ** -9)
    off = (_values(q, scales) - x).abs()
    return bool((off <= step / 2 + 2 * slack * x.abs()).all())      # (twice: x may lie just below a power of two, where the step doubles)


def _norm(h, w, eps=1e-6):
    return h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + torch.tensor(eps, dtype=torch.float32).double().item()) * w


# The sums are made in double, the result is carried in two float32 numbers and rounded to float32 once: half an ulp, 2^-24 of itself, and
# some 2^-40 for all the rest.
NORM_SLACK = 2.0 ** -24 * 1.001


@pytest.mark.parametrize("rows,K", [(1, 1), (3, 64), (9, 333), (8, 4096), (700, 5120), (2, 16384), (2, 16400), (3, 20001)])
def test_norm_is_the_nearest_number(rows, K):
    from llm_rs_b200 import ops
    h = 3 * _rows(rows, K, seed=K, spread=False)
    w = 1 + 0.1 * _rows(1, K, seed=1, spread=False)[0]
    d = _rows(rows, K, seed=2, spread=False).bfloat16()
    q, s = ops.add_rmsnorm_fp8(h, d, w, 1e-6)
    assert _nearest(q, s, _norm(h.double(), w.double()), NORM_SLACK)


@pytest.mark.parametrize("K", [2048, 8192, 16384, 1_000_003])
@pytest.mark.parametrize("c", [1.1, 30000.7])
def test_norm_next_to_the_borders(K, c):
    """Rows of one number: the norm is its weights but for eps, and the weights lie an ulp of float32 below, at and above what e4m3 rounds
    up or down at. Sums of squares in float32 would all err to the same side."""
    from llm_rs_b200 import ops
    h = torch.full((2, K), c, device=DEV)
    border = torch.tensor([17.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0], device=DEV)
    near = torch.stack([border * (1 + k * 2.0 ** -22) for k in (-2, -1, 1, 2)]).flatten()
    w = near.repeat(-(-K // 32))[:K].clone()
    w[::128] = 448.0 * 0.75                           # the blocks' largest numbers: the scale is 1
    q, s = ops.add_rmsnorm_fp8(h.clone(), None, w, 0.0)
    exact, _ = _exact(w.double()[None])               # eps 0: exactly the weights
    assert bool((_values(q, s) == exact * torch.exp2(_exact(w.double()[None])[1]).repeat_interleave(128, dim=1)[:, :K]).all())


@pytest.mark.parametrize("K", [512, 515, 4096, 17000])
def test_norm_of_large_rows(K):
    """Squares that pass float32 where their mean does not, wherever in the row they lie."""
    from llm_rs_b200 import ops
    w = 1 + 0.1 * _rows(1, K, seed=1, spread=False)[0]
    h = _rows(4, K, seed=2, spread=False)
    h[0, 3] = 3e19                                    # one square of 9e38
    h[1, :16] = 1.2e19                                # 1.4e38 each, neighbours
    h[2] = 1.5e19 * torch.sign(h[2])                  # 2.2e38 everywhere
    h[3, ::7] *= 5e18
    before = h.clone()
    for eps in (0.0, 1e-6):
        q, s = ops.add_rmsnorm_fp8(h, None, w, eps)
        assert bool((h == before).all())
        assert _nearest(q, s, _norm(h.double(), w.double(), eps), NORM_SLACK)


@pytest.mark.parametrize("K", [512, 515, 4096, 17000])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-42])
def test_norm_of_small_rows(K, eps):
    """Squares, and their mean, below what float32 holds; without an eps such rows are normed as any others, and empty rows are 0 / 0."""
    from llm_rs_b200 import ops
    w = 1 + 0.1 * _rows(1, K, seed=1, spread=False)[0]
    h = _rows(6, K, seed=2, spread=False) * torch.tensor([1e-15, 1e-19, 1e-22, 1e-25, 1e-31, 1e-36], device=DEV)[:, None]
    q, s = ops.add_rmsnorm_fp8(h, None, w, eps)
    assert _nearest(q, s, _norm(h.double(), w.double(), eps), NORM_SLACK)
    q, s = ops.add_rmsnorm_fp8(torch.zeros((2, K), device=DEV), None, w, eps)
    assert bool(q.float().isnan().all()) if eps == 0 else not bool(q.view(torch.uint8).any())


@pytest.mark.parametrize("K", [512, 515, 17000])
def test_norm_of_rows_whose_mean_passes_float32(K):
    """The mean of the squares is what decides, not how they are dealt to threads: just below the largest float32 a row is normed, just
    above it every number is NaN."""
    from llm_rs_b200 import ops
    w = torch.ones(K, device=DEV)
    h = torch.full((3, K), 1.0, device=DEV)
    h[0], h[1] = 1.8446743e19, 1.8447e19              # squares of 3.4028234e38 and 3.403e38; float32 ends at 3.40282347e38
    h[2] = 0.0
    h[2, 5] = 1.8446e19 * K ** 0.5                    # one number, mean 3.4025e38
    q, s = ops.add_rmsnorm_fp8(h, None, w, 1e-6)
    good = h[0::2]
    assert _nearest(q[0::2], s[:, 0::2], _norm(good.double(), w.double()), NORM_SLACK)
    assert bool(q[1].float().isnan().all())


# -- the gated unit ---------------------------------------------------------------------------------------------------
def _unit(gate, up, unit=(INF, 1.0, 0.0)):
    limit, alpha, shift = unit
    g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
    t = alpha * g
    a = torch.exp(-t.abs() / 2)                       # exp(t) = a * a for t < 0: no factor leaves float64
    return torch.where(t < 0, g * a / (1 + a * a) * (u + shift) * a, g / (1 + a * a) * (u + shift)), t


def _unit_slack(t):
    # Approximate power (2^-22.5 of itself; its square where the gate is far below zero: twice that), reciprocal (2^-23) and up to five
    # roundings of 2^-24; the power's argument errs by three roundings of itself: |t| 3 * 2^-24 of the power.
    return 2.0 ** -19.5 + 3 * t.abs() * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,inter,block", [(3, 640, 64), (33, 12288, 64), (2, 333, 0), (7, 520, 8), (5, 515, 5), (600, 1000, 0)])
def test_unit_is_the_nearest_number(rows, inter, block, dtype):
    from llm_rs_b200 import ops
    gu = (2 * _rows(rows, 2 * inter, seed=inter, spread=False)).to(dtype)
    both = gu.double().reshape(rows, -1, 2, block or inter)
    gate, up = both[:, :, 0].reshape(rows, inter), both[:, :, 1].reshape(rows, inter)
    for unit in ((INF, 1.0, 0.0), (1.5, 1.702, 1.0)):
        x, t = _unit(gate, up, unit)
        assert _nearest(*ops.silu_mul_fp8(gu, block, unit=unit), x, _unit_slack(t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter,block", [(512, 64), (516, 0), (515, 0), (515, 5), (1040, 16)])
@pytest.mark.parametrize("low,high", [(-87.0, -84.0), (-92.0, -86.0), (-130.0, -88.0), (-170.0, -100.0), (-95.0, 3.0)])
def test_unit_of_gates_far_below_zero(low, high, inter, block, dtype):
    """Blocks whose gates all are far below zero, beside ups that bring the result back into range: e^gate is below what float32 holds."""
    from llm_rs_b200 import ops
    g = torch.Generator(device=DEV)
    g.manual_seed(int(-low) + inter)
    gate = torch.rand((5, inter), generator=g, device=DEV) * (high - low) + low
    up = torch.randn((5, inter), generator=g, device=DEV) * 1e30
    b = block or inter
    gu = torch.stack([gate.reshape(5, -1, b), up.reshape(5, -1, b)], dim=2).reshape(5, 2 * inter).to(dtype)
    both = gu.double().reshape(5, -1, 2, b)
    gate, up = both[:, :, 0].reshape(5, inter), both[:, :, 1].reshape(5, inter)
    for unit in ((INF, 1.0, 0.0), (1e38, 1.0, 0.0), (1e38, 1.25, 0.0)):
        x, t = _unit(gate, up, unit)
        assert _nearest(*ops.silu_mul_fp8(gu, block, unit=unit), x, _unit_slack(t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter", [512, 516, 515])
@pytest.mark.parametrize("unit", [(INF, 1.0, 0.0), (7.0, 1.702, 1.0), (INF, 1.702, 0.0)])
def test_unit_of_what_is_no_number(unit, inter, dtype):
    """A NaN in the gate or the up becomes a NaN, whatever the unit's limit is; an infinity that no limit holds does too. Their neighbours
    are as without them."""
    from llm_rs_b200 import ops
    gu = _rows(4, 2 * inter, seed=inter, spread=False).to(dtype)
    gu[:, 5], gu[:, 200], gu[:, inter + 300] = 4.0, 4.0, 4.0      # (their blocks' largest results are elsewhere)
    gu[:, [100, 130, 300, 350, 400]], gu[:, [inter + c for c in (100, 130, 300, 350, 400)]] = 5.0, 5.0
    clean, _ = ops.silu_mul_fp8(gu, unit=unit)
    gu[0, 5], gu[1, inter + 300], gu[2, 200], gu[3, inter + 300] = NAN, NAN, INF, -INF
    q, _ = ops.silu_mul_fp8(gu, unit=unit)
    bad = torch.zeros((4, inter), dtype=torch.bool, device=DEV)
    bad[0, 5] = bad[1, 300] = True
    if unit[0] == INF:
        bad[2, 200] = bad[3, 300] = True
    assert bool(q.float()[bad].isnan().all()) and bool(q.float()[~bad].isfinite().all())
    assert bool((q.float() == clean.float())[0][~bad[0]].all()) and bool((q.float() == clean.float())[1][~bad[1]].all())
