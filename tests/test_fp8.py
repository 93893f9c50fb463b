"""What the operators of rows and products in 8 bits refuse, before anything is launched."""
import pytest
import torch

from llm_rs_b200 import ops

E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _q(rows, K, pitch=None):
    pitch = pitch or -(-K // 16) * 16
    return torch.zeros((rows, pitch), dtype=E4)[:, :K], torch.zeros((-(-K // 512), rows, 4), dtype=E8)


def _refused(match, f, *a, **kw):
    with pytest.raises(ops.KernelError, match=match):
        f(*a, **kw)


def test_rows_refuse():
    x = torch.zeros(4, 64)
    _refused("CUDA device", ops.quantize_fp8, x)
    _refused("float32 or bfloat16", ops.quantize_fp8, x.half())
    _refused("rows, numbers", ops.quantize_fp8, x[0])
    _refused("rows, numbers", ops.quantize_fp8, torch.zeros(4, 0))
    _refused("dense rows", ops.quantize_fp8, torch.zeros(64, 4).t())
    _refused("int32", ops.quantize_fp8, x, torch.zeros(4, dtype=torch.int64))
    _refused("int32", ops.quantize_fp8, x, torch.zeros(4, 1, dtype=torch.int32))
    _refused("CUDA device", ops.silu_mul_fp8, x)
    _refused("runs of", ops.silu_mul_fp8, torch.zeros(4, 63))
    _refused("runs of", ops.silu_mul_fp8, x, 24)
    _refused("runs of", ops.silu_mul_fp8, x, -1)
    w = torch.ones(64)
    _refused("CUDA device", ops.add_rmsnorm_fp8, x, None, w, 1e-6)
    _refused("h must be", ops.add_rmsnorm_fp8, x.bfloat16(), None, w, 1e-6)
    _refused("h must be", ops.add_rmsnorm_fp8, torch.zeros(4, 128)[:, :64], None, w, 1e-6)
    _refused("weight has", ops.add_rmsnorm_fp8, x, None, torch.ones(65), 1e-6)
    _refused("weight must be", ops.add_rmsnorm_fp8, x, None, w.bfloat16(), 1e-6)
    _refused("delta", ops.add_rmsnorm_fp8, x, x[:3], w, 1e-6)
    _refused("delta", ops.add_rmsnorm_fp8, x, x.half(), w, 1e-6)
    _refused("rows must be", ops.add_rmsnorm_fp8, x, None, w, 1e-6, rows=torch.zeros(2))


def test_products_refuse():
    x, xs = _q(4, 640)
    w, ws = _q(32, 640)
    f = ops.gemm_fp8
    _refused("CUDA device", f, x, xs, w, ws)
    _refused("must be torch.float8_e4m3fn", f, x.float(), xs, w, ws)
    _refused("scales of torch.float8_e8m0fnu", f, x, xs.float(), w, ws)
    _refused("its scales must be", f, x, xs[:1], w, ws)
    _refused("its scales must be", f, x[:3], xs, w, ws)
    _refused("columns", f, x, xs, *_q(32, 512))
    _refused("multiples of 16 bytes", f, _q(4, 640, 648)[0], xs, w, ws)
    _refused("multiples of 16 bytes", f, torch.zeros(4, 656, dtype=E4)[:, 8:648], xs, w, ws)
    _refused("multiples of 16 bytes", f, torch.zeros(640, 4, dtype=E4).t(), xs, w, ws)
    _refused("adjacent", f, x, torch.zeros(2, 4, 8, dtype=E8)[:, :, :4], w, ws)
    _refused("adjacent", f, x, torch.zeros(2, 8, 4, dtype=E8)[:, ::2], w, ws)
    _refused("no rows", f, x, xs, w[:0], ws[:, :0])
    _refused("unknown epilogue", f, x, xs, w, ws, epilogue="silu_mul")
    _refused("needs the stream", f, x, xs, w, ws, epilogue="residual")
    _refused("out is", f, x, xs, w, ws, out=torch.zeros(4, 32, dtype=torch.bfloat16), epilogue="residual")
    _refused("out is", f, x, xs, w, ws, out=torch.zeros(4, 32))
    _refused("out is", f, x, xs, w, ws, out=torch.zeros(5, 32, dtype=torch.bfloat16))
    _refused("dense rows", f, x, xs, w, ws, out=torch.zeros(32, 4, dtype=torch.bfloat16).t())
    _refused("float32 or bfloat16", f, x, xs, w, ws, out_dtype=torch.float16)


def test_grouped_products_refuse():
    x, xs = _q(4, 640)
    w, ws = _q(32, 640)
    w = w.unflatten(0, (2, 16))
    out, tiles, n = torch.zeros(4, 16), torch.zeros(3, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    f = ops.gemm_fp8_grouped
    _refused("CUDA device", f, x, xs, w, ws, out, tiles, n, 64)
    _refused("groups, features, K", f, x, xs, w[0], ws, out, tiles, n, 64)
    _refused("under one another", f, x, xs, w[:, :8], ws, out, tiles, n, 64)
    _refused("its scales must be", f, x, xs, w, ws[:, :16], out, tiles, n, 64)
    _refused("columns", f, *_q(4, 512), w, ws, out, tiles, n, 64)
    _refused("out is", f, x, xs, w, ws, out[:3], tiles, n, 64)
    _refused("out is", f, x, xs, w, ws, out.half(), tiles, n, 64)
    _refused("1 to 256 rows", f, x, xs, w, ws, out, tiles, n, 0)
    _refused("1 to 256 rows", f, x, xs, w, ws, out, tiles, n, 257)
    _refused("tiles must be", f, x, xs, w, ws, out, tiles.long(), n, 64)
    _refused("tiles must be", f, x, xs, w, ws, out, tiles[:, :2], n, 64)
    _refused("n_tiles must be", f, x, xs, w, ws, out, tiles, n.long(), 64)
