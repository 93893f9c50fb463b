"""Products in 8-bit floating point with a scale for each block of 128, and what makes their operands: the operators as cases
that can be timed and compared, with plain forms of them.

Rows of numbers are held as float8_e4m3fn ``q`` [rows, K] (rows start at multiples of 16 bytes) and float8_e8m0fnu ``scales``
[ceil(K / 512), rows, 4]: element [g, r, j] is the power of two that multiplies numbers 128 * (4 g + j) and following of row r,
the least one, not below 2^-127, with which the block's largest magnitude is at most 448. Places past the last block hold 2^-127.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
TOP = 448.0


# -- the cases --------------------------------------------------------------------------------------------------
def listed():
    return [
        # The rows of one decoded token of the 8B model before a product, and a ragged prompt's rows after attention.
        dict(name="rows_token", op="rows", rows=1, width=4096, dtype="bf16"),
        dict(name="rows_prompt", op="rows", rows=7211, width=4096, dtype="bf16"),
        # The gated unit between the two products of the 8B model's feed-forward: a decode step of 32 requests (gate and up
        # interleaved by 64 columns, as the framework lays them out), a prompt.
        dict(name="unit_decode", op="unit", rows=32, width=12288, block=64, dtype="bf16"),
        dict(name="unit_prompt", op="unit", rows=2048, width=12288, block=64, dtype="bf16"),
        # The residual sum and norm in front of a product: a decode step of eight requests, a prompt of the 14B model's width.
        dict(name="norm_decode", op="norm", rows=8, width=4096, dtype="bf16"),
        dict(name="norm_prompt", op="norm", rows=4001, width=5120, dtype="bf16"),
        # q|k|v of the 8B model for one token: the weights' stream is everything.
        dict(name="product_token", op="product", tokens=1, features=6144, k=4096, out="bf16"),
        # gate|up of the 8B model in a decode step of 32 requests.
        dict(name="product_decode", op="product", tokens=32, features=24576, k=4096, out="bf16"),
        # gate|up of the 8B model over a prompt portion: the tensor cores' rate is everything.
        dict(name="product_prompt", op="product", tokens=2048, features=24576, k=4096, out="bf16"),
        # An odd-sized product into the residual stream (down projection of an odd model, ragged prompt).
        dict(name="product_odd", op="product", tokens=333, features=2200, k=5005, out="residual"),
        # gate|up of 32 experts of 1,024 with two projections each: a decode step of 32 requests with four experts a token, and
        # a prompt of 2,048 tokens; rows are spread unevenly, some experts get none.
        dict(name="experts_decode", op="experts", rows=128, experts=32, features=2048, k=2048, out="bf16"),
        dict(name="experts_prompt", op="experts", rows=8192, experts=32, features=2048, k=2048, out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "unit", "norm", "product", "product", "experts"])
    if op in ("rows", "unit", "norm"):
        c = dict(op=op, rows=_log(rng, 1, 8192), width=_log(rng, 32, 16384), dtype=rng.choice(["bf16", "bf16", "f32"]))
        while c["rows"] * c["width"] > 2048 * 12288:
            c["rows"] = max(1, c["rows"] // 2)
        if op == "unit":
            c["block"] = rng.choice([0, 64])
            if c["block"]:
                c["width"] = max(64, c["width"] // 64 * 64)
        return c
    if op == "product":
        c = dict(op=op, tokens=_log(rng, 1, 4096), features=_log(rng, 64, 25600), k=_log(rng, 64, 12288),
                 out=rng.choice(["bf16", "bf16", "f32", "residual"]))
        while c["tokens"] * c["features"] * c["k"] > 2048 * 24576 * 4096:
            c["tokens"] = max(1, c["tokens"] // 2)
        return c
    c = dict(op=op, rows=_log(rng, 4, 16384), experts=rng.choice([4, 8, 16, 32, 60, 64]), features=_log(rng, 128, 4096),
             k=_log(rng, 128, 4096), out=rng.choice(["bf16", "f32"]))
    while c["rows"] * c["features"] * c["k"] > 2048 * 24576 * 4096:
        c["rows"] = c["rows"] // 2
    return c


# -- rows in 8 bits, plainly --------------------------------------------------------------------------------------
def _rows_of(n, width):
    """An uninitialised float8_e4m3fn [n, width] whose rows start at multiples of 16 bytes."""
    return torch.empty((n, -(-width // 16) * 16), dtype=torch.float8_e4m3fn, device=DEV)[:, :width]


def _quantize(x):
    """float32 [rows, K] -> (q, scales)."""
    rows, K = x.shape
    words = -(-K // 512)
    blocks = torch.nn.functional.pad(x, (0, words * 512 - K)).reshape(rows, words * 4, 128)
    top = blocks.abs().amax(dim=2)
    mant, exp = torch.frexp(top)                      # top = mant * 2^exp, mant in [1/2, 1); 448 = 7/8 * 2^9
    e = torch.where(top > 0, exp - 9 + (mant > 0.875).to(exp.dtype), torch.full_like(exp, -127)).clamp(min=-127)
    y = torch.ldexp(blocks, -e[..., None])            # a power of two: exact
    q = _rows_of(rows, K)
    q.copy_(y.reshape(rows, words * 512)[:, :K].to(torch.float8_e4m3fn))
    scales = (e + 127).to(torch.uint8).reshape(rows, words, 4).transpose(0, 1).contiguous()
    return q, scales.view(torch.float8_e8m0fnu)


def _values(q, scales, dtype=torch.float32):
    """What (q, scales) stand for: [rows, K]."""
    rows, K = q.shape
    s = scales.to(dtype).transpose(0, 1).reshape(rows, -1)
    return q.to(dtype) * s.repeat_interleave(128, dim=1)[:, :K]


def _gate_up(gu, block):
    """The gate and the up columns of the layout that alternates ``block`` columns of each (0: all gate, then all up)."""
    n, two = gu.shape
    block = block or two // 2
    both = gu.reshape(n, two // (2 * block), 2, block)
    return both[:, :, 0].reshape(n, two // 2), both[:, :, 1].reshape(n, two // 2)


# -- inputs -------------------------------------------------------------------------------------------------------
def _numbers(gen, *shape):
    """Activations: normal numbers, a few channels much larger than the others, as a trained model's are."""
    x = torch.randn(shape, generator=gen, device=DEV)
    loud = torch.rand(shape[-1], generator=gen, device=DEV) < 0.01
    return x * torch.where(loud, 30.0, 1.0)


def _sizes(case, seed):
    """Rows of each expert: uneven, some none."""
    r = np.random.RandomState(seed % (1 << 31))
    p = r.gamma(0.8, size=case["experts"]) + 1e-3
    p[r.randint(case["experts"])] = 0.0
    return r.multinomial(case["rows"], p / p.sum())


def tile_rows(rows, groups):
    """The most rows a tile of a group has: few where groups have few rows, so that more of the weights' stream is under way."""
    return 32 if rows <= 8 * groups else 128 if rows <= 64 * groups else 256


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = dict(case)
    op = case["op"]
    if op == "rows":
        s["x"] = _numbers(g, case["rows"], case["width"]).to(DTYPES[case["dtype"]])
    elif op == "unit":
        s["gate_up"] = _numbers(g, case["rows"], 2 * case["width"]).to(DTYPES[case["dtype"]])
    elif op == "norm":
        s["h"] = 3 * _numbers(g, case["rows"], case["width"])
        s["delta"] = _numbers(g, case["rows"], case["width"]).to(DTYPES[case["dtype"]])
        s["weight"] = 1 + 0.1 * torch.randn(case["width"], generator=g, device=DEV)
    elif op == "product":
        s["x"], s["x_scales"] = _quantize(_numbers(g, case["tokens"], case["k"]))
        s["w"], s["w_scales"] = _quantize(0.02 * torch.randn(case["features"], case["k"], generator=g, device=DEV))
        if case["out"] == "residual":
            s["h"] = _numbers(g, case["tokens"], case["features"])
    else:
        n, E, N, K = case["rows"], case["experts"], case["features"], case["k"]
        sizes = _sizes(case, seed)
        s["x"], s["x_scales"] = _quantize(_numbers(g, n, K))
        w, s["w_scales"] = _quantize(0.02 * torch.randn(E * N, K, generator=g, device=DEV))
        s["w"] = w.unflatten(0, (E, N))
        # The plan of the step: tiles of at most `tile_rows` rows of one expert, and their number; how many rows each expert has.
        s["tile_rows"] = tile_rows(n, E)
        tiles, at = [], 0
        for e, c in enumerate(sizes):
            tiles += [(e, at + i, min(s["tile_rows"], c - i)) for i in range(0, c, s["tile_rows"])]
            at += c
        most = -(-n // s["tile_rows"]) + E
        s["n_tiles"] = torch.tensor([len(tiles)], dtype=torch.int32, device=DEV)
        s["tiles"] = torch.tensor(tiles + [(0, 0, 0)] * (most - len(tiles)), dtype=torch.int32, device=DEV)
        s["expert_of"] = torch.from_numpy(np.repeat(np.arange(E), sizes)).to(DEV)
        s["place_of"] = torch.from_numpy(np.concatenate([np.arange(c) for c in sizes])).to(DEV)
        s["most_rows"] = int(sizes.max())
    return s


# -- one pass -----------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from llm_rs_b200 import ops
    op = s["op"]
    if op == "rows":
        return ops.quantize_fp8(s["x"])
    if op == "unit":
        return ops.silu_mul_fp8(s["gate_up"], block=s["block"])
    if op == "norm":
        return (*ops.add_rmsnorm_fp8(s["h"], s["delta"], s["weight"], EPS), s["h"])
    if op == "product":
        if s["out"] == "residual":
            return ops.gemm_fp8(s["x"], s["x_scales"], s["w"], s["w_scales"], out=s["h"], epilogue="residual")
        return ops.gemm_fp8(s["x"], s["x_scales"], s["w"], s["w_scales"], out_dtype=DTYPES[s["out"]])
    out = torch.empty((s["rows"], s["features"]), dtype=DTYPES[s["out"]], device=DEV)
    return ops.gemm_fp8_grouped(s["x"], s["x_scales"], s["w"], s["w_scales"], out, s["tiles"], s["n_tiles"],
                                tile_rows=s["tile_rows"])


def _run_plain(s):
    op = s["op"]
    if op == "rows":
        return _quantize(s["x"].float())
    if op == "unit":
        gate, up = _gate_up(s["gate_up"].float(), s["block"])
        return _quantize(gate / (1 + torch.exp(-gate)) * up)
    if op == "norm":
        h = s["h"].add_(s["delta"].float())
        rms = torch.sqrt(h.square().mean(dim=1, keepdim=True) + EPS)
        return (*_quantize(h / rms * s["weight"]), h)
    if op == "product":
        y = _values(s["x"], s["x_scales"]) @ _values(s["w"], s["w_scales"]).T
        return s["h"].add_(y) if s["out"] == "residual" else y.to(DTYPES[s["out"]])
    E, N, K = s["w"].shape
    w = _values(s["w"].flatten(0, 1), s["w_scales"]).unflatten(0, (E, N))
    x = torch.zeros((E, s["most_rows"], K), device=DEV)      # each expert's rows, filled up to the most that one has
    x[s["expert_of"], s["place_of"]] = _values(s["x"], s["x_scales"])
    return torch.bmm(x, w.transpose(1, 2))[s["expert_of"], s["place_of"]].to(DTYPES[s["out"]])


def work(case):
    op = case["op"]
    if op in ("rows", "unit", "norm"):
        n = case["rows"] * case["width"]
        size = 2 if case["dtype"] == "bf16" else 4
        read = {"rows": size * n, "unit": 2 * size * n, "norm": (4 + size) * n + 4 * case["width"]}[op]
        return {"bytes": read + n + n / 128 + (4 * n if op == "norm" else 0), "flops": {"rows": 2, "unit": 8, "norm": 6}[op] * n}
    size = {"bf16": 2, "f32": 4, "residual": 8}[case["out"]]
    N, K = case["features"], case["k"]
    if op == "product":
        T = case["tokens"]
        return {"bytes": (T + N) * (K + K / 128) + size * T * N, "flops": 2 * T * N * K}
    T = case["rows"]
    used = int((_sizes(case, 1) > 0).sum())      # experts without rows read nothing; another seed's number is much the same
    return {"bytes": (T + used * N) * (K + K / 128) + size * T * N, "flops": 2 * T * N * K}


# -- the same in 64 bits, from the definition -----------------------------------------------------------------------
def _round_e4m3(y):
    """float64 -> the nearest number that e4m3 has (ties to even), up to 448."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -40)))
    e = torch.where(torch.exp2(e) > y.abs(), e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= y.abs(), e + 1, e)
    step = torch.exp2(e.clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-TOP, TOP)


def _quantize_exact(x):
    rows, K = x.shape
    words = -(-K // 512)
    top = torch.zeros((rows, words * 4), dtype=torch.float64, device=x.device)
    for b in range(-(-K // 128)):
        top[:, b] = x[:, 128 * b: 128 * (b + 1)].abs().amax(dim=1)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / TOP)).clamp(min=-127)
    e = torch.where((e > -127) & (TOP * torch.exp2(e - 1) >= top), e - 1, e)      # log2 near a whole number
    e = torch.where(TOP * torch.exp2(e) < top, e + 1, e)
    s = torch.exp2(e)
    q = _round_e4m3(x / s.repeat_interleave(128, dim=1)[:, :K])
    return q, s.reshape(rows, words, 4).transpose(0, 1).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rows":
        return _quantize_exact(s["x"].double())
    if op == "unit":
        gu = s["gate_up"].double()
        n, two = gu.shape
        b = case["block"] or two // 2
        col = torch.arange(two // 2, device=DEV)
        gate, up = gu[:, col // b * 2 * b + col % b], gu[:, col // b * 2 * b + b + col % b]
        return _quantize_exact(up * gate * torch.sigmoid(gate))
    if op == "norm":
        h = s["h"].double() + s["delta"].double()
        x = h * torch.rsqrt((h * h).sum(dim=1, keepdim=True) / case["width"] + EPS) * s["weight"].double()
        return (*_quantize_exact(x), h)

    def wide(q, scales):
        rows, K = q.shape
        k = torch.arange(K, device=DEV)
        return q.double() * scales.double()[k // 512, :, k // 128 % 4].T

    x = wide(s["x"], s["x_scales"])
    if op == "product":
        y = x @ wide(s["w"], s["w_scales"]).T
        return s["h"].double() + y if case["out"] == "residual" else y
    E, N, K = s["w"].shape
    w = wide(s["w"].flatten(0, 1), s["w_scales"]).unflatten(0, (E, N))
    return torch.cat([x[s["expert_of"] == e] @ w[e].T for e in range(E)])
