"""Every call of an operator in 8 bits that a step of an engine makes, held to float64 where it is made, in every design; and that the
weights are the stored ones, quantised.

The errors are those of test_fp8_borders_gpu.py (rows: one rounding to e4m3 of a number that errs by a few ulps of float32) and of
test_fp8_pairs_gpu.py (products: K + 1 half ulps of the products' magnitudes, and half a step of the result's type)."""
import numpy as np
import pytest
import torch

from test_fp8_borders_gpu import NORM_SLACK, _nearest, _norm, _unit, _unit_slack
from test_fp8_engine_gpu import MODELS, _eight, _near, _runtime
from test_fp8_gpu import _exact, _rows, _scales, _values
from test_fp8_pairs_gpu import _within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Checked:
    """The operators' entry points, each call compared with float64."""

    def __init__(self, ops):
        self.calls, self.weights = {}, set()
        self.made = None      # rows that the last grouped product made: those of experts that run none hold anything
        self.real = {n: getattr(ops, n) for n in ("quantize_fp8", "silu_mul_fp8", "add_rmsnorm_fp8", "gemm_fp8", "gemm_fp8_grouped")}

    def _count(self, name):
        self.calls[name] = self.calls.get(name, 0) + 1

    def quantize_fp8(self, x, src=None):
        self._count("quantize_fp8")
        q, s = self.real["quantize_fp8"](x, src)
        rows = x if src is None else torch.where((src >= 0)[:, None] & (src < x.size(0))[:, None], x[src.long().clamp(0, x.size(0) - 1)], 0)
        want, e = _exact(rows.double())
        assert bool((q.double() == want).all()) and bool((_scales(s, x.size(1))[0] == e).all())
        return q, s

    def silu_mul_fp8(self, gate_up, block=0, unit=(float("inf"), 1.0, 0.0)):
        self._count("silu_mul_fp8")
        q, s = self.real["silu_mul_fp8"](gate_up, block, unit)
        n, inter = gate_up.size(0), gate_up.size(1) // 2
        both = gate_up.double().reshape(n, -1, 2, block or inter)
        x, t = _unit(both[:, :, 0].reshape(n, inter), both[:, :, 1].reshape(n, inter), unit)
        made = self.made if self.made is not None and len(self.made) == n else torch.ones(n, dtype=torch.bool, device=x.device)
        self.made = None
        assert _nearest(q[made], s[:, made], x[made], _unit_slack(t[made]))
        return q, s

    def add_rmsnorm_fp8(self, h, delta, weight, eps, rows=None):
        self._count("add_rmsnorm_fp8")
        want_h = h.clone() if delta is None else h + delta.float()
        q, s = self.real["add_rmsnorm_fp8"](h, delta, weight, eps, rows)
        assert rows is None and bool((h == want_h).all())
        assert _nearest(q, s, _norm(want_h.double(), weight.double(), eps), NORM_SLACK)
        return q, s

    def gemm_fp8(self, x, x_scales, w, w_scales, out=None, epilogue="store", out_dtype=torch.bfloat16):
        self._count("gemm_fp8 " + epilogue)
        self.weights.add((w.data_ptr(), w.size(0)))
        before = out.double() if epilogue == "residual" else None
        y = self.real["gemm_fp8"](x, x_scales, w, w_scales, out=out, epilogue=epilogue, out_dtype=out_dtype)
        assert _within(y, _values(x, x_scales), _values(w, w_scales), before)
        return y

    def gemm_fp8_grouped(self, x, x_scales, w, w_scales, out, tiles, n_tiles, tile_rows):
        self._count("gemm_fp8_grouped")
        self.real["gemm_fp8_grouped"](x, x_scales, w, w_scales, out, tiles, n_tiles, tile_rows)
        xv, wv = _values(x, x_scales), _values(w.flatten(0, 1), w_scales).unflatten(0, w.shape[:2])
        self.made = torch.zeros(out.size(0), dtype=torch.bool, device=out.device)
        for g, first, rows in tiles[: int(n_tiles)].tolist():
            self.made[first: first + rows] = True
            assert rows <= tile_rows and _within(out[first: first + rows], xv[first: first + rows], wv[g])
        return out


def _products(stored, eight, found, seen):
    """Pairs (stored product, the same part's product in 8 bits, its name) of everything that two bound models hold."""
    from llm_rs_b200.parts.base import Part
    from llm_rs_b200.parts.linear import Fp8Linear
    if id(eight) in seen:
        return
    seen.add(id(eight))
    if getattr(eight, "fp8", None) is not None:
        _experts(stored, eight)
    for name, b in vars(eight).items():
        a = vars(stored).get(name)
        if isinstance(b, Fp8Linear):
            found.append((a, b, f"{type(eight).__name__}.{name}"))
        elif isinstance(b, Part):
            _products(a, b, found, seen)
        elif isinstance(b, (list, tuple)):
            for i, y in enumerate(b):
                if isinstance(y, Part):
                    _products(a[i], y, found, seen)


def _experts(stored, eight):
    """The experts' weights: every expert's gate and up rows alternating by the part's runs, then its down rows."""
    q, scales, q_down, down_scales = eight.fp8
    E, F, H = stored.w_gate.shape
    both = _values(q.flatten(0, 1), scales).reshape(E, -1, 2, eight.block, H)
    for i, w in enumerate((stored.w_gate, stored.w_up)):
        assert bool((both[:, :, i].reshape(E * F, H) == _eight(w.flatten(0, 1))).all())
    assert bool((_values(q_down.flatten(0, 1), down_scales) == _eight(stored.w_down.flatten(0, 1))).all())


@pytest.mark.parametrize("name", list(MODELS))
def test_every_call_of_a_step(tmp_path, monkeypatch, name):
    from llm_rs_b200 import ops
    from llm_rs_b200.engine import ModelRunner, StepEntry
    write, which, page = MODELS[name]
    path = write(which, str(tmp_path))
    stored, eight = (ModelRunner.from_model_dir(path, max_tokens=512, page_size=page, max_requests=4, products=p) for p in ("stored", "fp8"))
    eight.use_graphs = False
    found, seen = [], set()
    for a, b in zip(stored.model.blocks, eight.model.blocks):
        _products(a, b, found, seen)
    for a, b, where in found:
        q, s = ops.quantize_fp8(a.weight)
        assert b.weight.shape == a.weight.shape, where
        assert bool((b.weight.view(torch.uint8) == q.view(torch.uint8)).all()) and bool((b.scales.view(torch.uint8) == s.view(torch.uint8)).all()), where
    checked = Checked(ops)
    for n in checked.real:
        monkeypatch.setattr(ops, n, getattr(checked, n))
    vocab = eight.spec.vocab_size
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, vocab, 70).tolist()
    eight.step([StepEntry("a", prompt, list(range(64, 70)))])
    eight.step([StepEntry("a", [3], [0]), StepEntry("b", prompt[:5], [4])])      # a decoded token beside a prompt
    eight.step([StepEntry("a", [4], [0]), StepEntry("b", [5], [0])])
    ops.check_tc_error(DEV)
    # Every product ran, but the query rows alone of layers that keep a cache of their own.
    for _, b, where in found:
        assert (b.weight.data_ptr(), b.weight.size(0)) in checked.weights or where.endswith(".q_proj"), where
    assert sum(v for k, v in checked.calls.items() if k.startswith("gemm")) > 0, checked.calls
    if name.startswith("qwen3"):
        assert checked.calls.get("silu_mul_fp8") and checked.calls.get("gemm_fp8 store") and checked.calls.get("gemm_fp8 residual"), checked.calls
        assert checked.calls.get("add_rmsnorm_fp8"), checked.calls


@pytest.mark.parametrize("tokens", [1, 45, 300])
@pytest.mark.parametrize("H,I", [(256, 640), (200, 333)])
def test_feed_forward_without_a_gate(tokens, H, I):
    from llm_rs_b200.parts.linear import Fp8Linear
    from llm_rs_b200.parts.mlp import DenseFF
    part = DenseFF(H, I)
    w = {n: (_rows(*s, seed=i, spread=False) * 0.08).bfloat16() for i, (n, s) in enumerate((("up", (I, H)), ("down", (H, I))))}
    part.bind(w, _runtime())
    assert isinstance(part.up, Fp8Linear) and isinstance(part.down, Fp8Linear) and part.takes_rows8
    x = _rows(tokens, H, seed=9, spread=False).bfloat16()
    z = (_eight(x) @ _eight(w["up"]).t()).bfloat16().double()
    want = _eight(z.clamp(min=0).square().bfloat16()) @ _eight(w["down"]).t()
    _near(part.forward(x, None), want)
    h = _rows(tokens, H, seed=10, spread=False)
    before = h.clone()
    assert part.forward(x, None, residual=h) is None
    _near(h - before, want)
