"""Adapters whose scale A x is small and whose B is large, without the shared projection to hide them
(W = 0): what the header says is lost of scale A x, and no more.

Tolerance, with u = scale A x (rank R, I columns):
  - u itself, a sum in fp32 (bf16 and fp16 products are exact): (I + 32) 2^-24 6 |scale| |A||x| (2-norms);
  - its parts: bf16 2^-16 |u| (two values, each rounded by 2^-8 of what is left), 2^-24 |u| (three);
    fp16 2^-22 |u|, or half its least step, 2^-25, where that is more;
  - the products' sum: (16 parts + 32) 2^-24 6 times its 2-norm;
  - the output's rounding, half a step; of fp16 below 2^-14 half the least one.
"""
import numpy as np
import pytest

from tests.test_adapter_head_gpu import dtype_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 90, 200])
@pytest.mark.parametrize("size", [1e-1, 1e-3, 1e-4, 1e-6])
@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_small_products(dtype, out, size, rows):
    import torch
    from neuraval_b200.adapter_head import CudaAdapterHead
    t, inner, cols, rank, scale = dtype_of(dtype), 64, 301, 8, 0.25
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, inner, device="cuda", generator=g).to(t)
    a = (torch.randn(rank, inner, device="cuda", generator=g) * (size / scale / inner ** 0.5)).to(t)
    b = (torch.randn(cols, rank, device="cuda", generator=g) * 1e3).to(t)
    y = torch.full((rows, cols), float("nan"), device="cuda", dtype=dtype_of(out))
    ids = torch.from_numpy((np.arange(rows) % 3 != 1).astype(np.int32) - 1).cuda()  # some without
    with CudaAdapterHead(torch.zeros(cols, inner, device="cuda", dtype=t), rows, 1, rank) as h:
        h.set_adapter(0, a, b, scale)
        h.project_device(x, ids, y)
        torch.cuda.synchronize()
    A, B, X = a.double(), b.double(), x.double()
    u = scale * (X @ A.T)
    u[ids < 0] = 0.0
    want = u @ B.T
    du = (inner + 32) * 2.0 ** -24 * 6 * scale * ((X ** 2) @ (A ** 2).T).sqrt()
    lost = u.abs() * 2.0 ** -22 if dtype == "f16" else u.abs() * 2.0 ** (-24 if out == "f32" else -16)
    if dtype == "f16":
        lost = lost.clamp(min=2.0 ** -25)
    tol = (du + lost) @ B.abs().T + (16 * 3 + 32) * 2.0 ** -24 * 6 * ((u ** 2) @ (B ** 2).T).sqrt()
    f = torch.finfo(y.dtype)
    tol += (f.eps / 2 * (want.abs() + tol)).clamp(min=f.tiny * f.eps / 2)
    tol[ids < 0] = 0.0
    err = (y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())
