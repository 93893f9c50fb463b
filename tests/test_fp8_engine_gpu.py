"""Parts and whole models with products in 8 bits (``products="fp8"``).

A part is compared with float64 over the same quantised numbers: what its kernels quantise on the way (a unit's results) is one of
two neighbours where its float32 and the float64 number lie on two sides of a border, a step of 2^-3 at most; fewer than one in a
hundred do (a bfloat16 rounding in between, 2^-9 of a number, against steps of 2^-3 to 2^-4: one in 32 to 64 of the bfloat16
roundings that fall differently, which are few themselves), so that the 2-norm is off by less than 2^-3 / 10, and by 2^-9 for the
result's own rounding."""
import numpy as np
import pytest
import torch

from fekolorn_configs import write_fekolorn_model
from kopatar_configs import write_kopatar_model
from pozelix_configs import write_pozelix_model
from pusazen_configs import write_pusazen_model
from rusadra_configs import write_rusadra_model
from sumuvik_configs import write_sumuvik_model
from test_fp8_gpu import _rows, _values
from tiny_configs import TINY, write_tiny_model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _runtime():
    from llm_rs_b200.parts import Runtime
    return Runtime(torch.device(DEV), torch.bfloat16, 512, "fp8")


def _near(got, want):
    assert bool(got.isfinite().all())
    assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -3 / 10 + 2.0 ** -9


def _eight(x):
    from llm_rs_b200 import ops
    return _values(*ops.quantize_fp8(x))


def _unit(gate, up, unit=(float("inf"), 1.0, 0.0)):
    limit, alpha, shift = unit
    g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
    return g * torch.sigmoid(alpha * g) * (u + shift)


@pytest.mark.parametrize("tokens", [1, 45, 300])
@pytest.mark.parametrize("H,I", [(256, 640), (200, 333)])
def test_feed_forward(tokens, H, I):
    from llm_rs_b200.parts.linear import Fp8Linear
    from llm_rs_b200.parts.mlp import SwiGLU
    part = SwiGLU(H, I)
    w = {n: (_rows(I if n != "down" else H, H if n != "down" else I, seed=i, spread=False) * 0.08).bfloat16()
         for i, n in enumerate(("gate", "up", "down"))}
    part.bind({f"{n}.weight": t for n, t in w.items()}, _runtime())
    assert isinstance(part.gate_up, Fp8Linear) and isinstance(part.down, Fp8Linear) and part.takes_rows8
    x = _rows(tokens, H, seed=9, spread=False).bfloat16()
    gate, up = (_eight(x) @ _eight(w[n]).t() for n in ("gate", "up"))
    act = _unit(gate.bfloat16().double(), up.bfloat16().double())
    want = _eight(act.float()) @ _eight(w["down"]).t()
    _near(part.forward(x, None), want)
    h = _rows(tokens, H, seed=10, spread=False)
    before = h.clone()
    assert part.forward(x, None, residual=h) is None
    _near(h - before, want)


@pytest.mark.parametrize("tokens", [1, 20, 200])
@pytest.mark.parametrize("form", ["table", "identity", "groups"])
def test_experts(tokens, form):
    from llm_rs_b200.parts.moe import MixtureOfExperts
    H, F, E, top = 256, 192, 6, 2
    kw = {"table": dict(router="table", vocab_size=50, limit=2.0), "identity": dict(router="softmax_bias", n_identity=2, limit=None, alpha=1.0, up_shift=0.0),
          "groups": dict(router="sigmoid_groups", groups=(3, 2), route_scale=1.5, shared_size=128, limit=None, alpha=1.0, up_shift=0.0)}[form]
    part = MixtureOfExperts(H, F, E, top, **kw)
    g = torch.Generator().manual_seed(3)
    tensors = {}
    for s in part.weight_specs():
        if s.role == "expert_table":
            tensors[s.name] = torch.stack([torch.randperm(E, generator=g)[:top] for _ in range(s.shape[0])]).to(torch.int32).to(DEV)
        else:
            tensors[s.name] = (torch.randn(s.shape, generator=g) * (0.1 if len(s.shape) == 2 else 0.01)).bfloat16().to(DEV)
    part.bind(tensors, _runtime())
    assert part.fp8 is not None
    x = _rows(tokens, H, seed=4, spread=False).bfloat16()
    ctx = type("Ctx", (), {})()
    ctx.token_ids = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32).to(DEV)
    got = part.forward(x, ctx)
    unit = (part.limit, part.alpha, part.up_shift)
    x8 = _eight(x)

    def expert(prefix, x8, unit):
        gate, up = (x8 @ _eight(tensors[prefix + n]).t() for n in ("gate", "up"))
        return _eight(_unit(gate.bfloat16().double(), up.bfloat16().double(), unit).float()) @ _eight(tensors[prefix + "down"]).t()
    each = [expert(f"e{e}.", x8, unit) for e in range(E)] + [x.double()] * part.n_identity
    want = torch.zeros(tokens, H, dtype=torch.float64, device=DEV)
    if form == "table":
        for k in range(top):
            for e in range(E):
                want += torch.where((tensors["table"][ctx.token_ids.long(), k] == e)[:, None], each[e] / top, 0.0)
    else:
        logits = x.double() @ tensors["router"].double().t()
        s = logits.softmax(1) if form == "identity" else logits.sigmoid()
        choice = s + tensors["correction"].double()
        if form == "groups":
            best = choice.reshape(tokens, 3, 2).topk(2, dim=2).values.sum(2).topk(2, dim=1).indices
            keep = torch.zeros(tokens, 3, dtype=torch.bool, device=DEV).scatter_(1, best, True)
            choice = torch.where(keep.repeat_interleave(2, dim=1), choice, -1.0)
        chosen = choice.topk(top, dim=1).indices
        weight = s.gather(1, chosen)
        weight = weight if form == "identity" else 1.5 * weight / weight.sum(1, keepdim=True)
        for k in range(top):
            for e in range(len(each)):
                want += torch.where((chosen[:, k] == e)[:, None], each[e] * weight[:, k: k + 1], 0.0)
        if form == "groups":
            want += expert("shared.", x8, (float("inf"), 1.0, 0.0))
    _near(got, want)


MODELS = {"qwen3 " + n: (write_tiny_model, n, TINY[n][3]) for n in ("B", "C", "D")}
MODELS |= {"rusadra A": (write_rusadra_model, "A", 16), "pusazen A": (write_pusazen_model, "A", 16), "pozelix A": (write_pozelix_model, "A", 16),
           "fekolorn A": (write_fekolorn_model, "A", 16), "kopatar A": (write_kopatar_model, "A", 16), "sumuvik A": (write_sumuvik_model, "A", 16)}


@pytest.mark.parametrize("name", list(MODELS))
def test_engine(tmp_path, name):
    """Every design generates with its products in 8 bits, the same tokens from captured steps and from plain ones and the same
    twice; its logits are those of the stored weights up to errors of 8 bits: a product's rows err by some 4 % (two operands, an
    e4m3 rounding is uniform over at most 2^-4 of a number to each side: 2^-4 / sqrt(3) each at worst), and a handful of them in a
    row by less than half of their size."""
    from llm_rs_b200.engine import Engine, EngineConfig, ModelRunner, StepEntry
    from llm_rs_b200.parts.linear import Fp8Linear
    from llm_rs_b200.sampling import SamplingParams
    write, which, page = MODELS[name]
    path = write(which, str(tmp_path))
    runners = {p: ModelRunner.from_model_dir(path, max_tokens=512, page_size=page, max_requests=4, products=p) for p in ("stored", "fp8")}
    vocab = runners["fp8"].spec.vocab_size
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, vocab, 70).tolist()
    logits = {p: r.step([StepEntry("a", prompt, list(range(40, 70)))]) for p, r in runners.items()}
    assert bool(logits["fp8"].isfinite().all())
    off = logits["fp8"].double() - logits["stored"].double()
    assert 0 < float(off.norm() / logits["stored"].double().norm()) < 0.5
    if name.startswith("qwen3"):
        assert any(isinstance(p, Fp8Linear) for b in runners["fp8"].model.blocks for p in b.chain())
    prompts = [rng.integers(0, vocab, n).tolist() for n in (3, 40, 17, 70)]
    out = []
    for graphs in (False, True, True):
        e = Engine(EngineConfig(model_path=path, block_pool_size=64, page_size=page, max_requests=4, max_tokens_per_step=48,
                                prefill_chunk=32, cuda_graphs=graphs, products="fp8"))
        out.append(e.generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=12, ignore_eos=True)))
        e.check_kernels()
        assert not e.runner.manager.requests
    assert out[0] == out[1] == out[2] and [len(t) for t in out[0]] == [12] * 4


def test_products_that_are_refused(tmp_path):
    from llm_rs_b200.engine import Engine, EngineConfig
    path = write_tiny_model("A", str(tmp_path))
    with pytest.raises(ValueError, match="bfloat16 activations"):
        Engine(EngineConfig(model_path=path, dtype="float32", products="fp8"))
    with pytest.raises(ValueError, match="'stored' or 'fp8'"):
        Engine(EngineConfig(model_path=path, products="int8"))
