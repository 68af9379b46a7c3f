"""Sampling with options per row and the head with adapters at the ends of their ranges: offsets past
32 bits, many rows, many tiles, all slots in use, rows whose counters are full, captured calls."""
import numpy as np
import pytest

from tests.test_adapter_head_gpu import Case
from tests.test_sample_min_p_gpu import compare, dtype_of, options, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_further_apart_than_32_bits(dtype):
    import torch
    rng = np.random.default_rng(1)
    t, ld, V = dtype_of(dtype), 2 ** 31 + 9, 5001
    flat = torch.empty(2 * ld + V, device="cuda", dtype=t)
    x = flat.as_strided((3, V), (ld, 1))
    x.copy_(torch.from_numpy(rng.standard_normal((3, V)) * 3).to(t))
    compare(x, *options(rng, 3, V))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_more_rows_than_16_bits(dtype):
    import torch
    rng = np.random.default_rng(2)
    rows, V = 70001, 37
    x = torch.from_numpy(rng.standard_normal((rows, V)) * 2).cuda().to(dtype_of(dtype))
    compare(x, *options(rng, rows, V))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("V", [32760, 32761, 32768, 32769, 65520, 65528, 65529, 131040, 131041, 131057, 262105, 524272, 524281])
def test_counters_that_are_full(V, dtype):
    """Rows of one value, of two, and of ordinary ones, at lengths where a CTA more has to count."""
    import torch
    rng = np.random.default_rng(V)
    x = np.full((4, V), 1.5)
    x[1] = np.where(rng.random(V) < 0.5, 1.5, -2.0)
    x[2:] = rng.standard_normal((2, V))
    x = torch.from_numpy(x).cuda().to(dtype_of(dtype))
    u = [0.0, 0.6, 0.999, 0.3]
    compare(x, np.full(4, 0.9), [0, V - 5, 0, 700], [1.0, 0.7, 0.95, 0.9], None, u)
    compare(x, np.full(4, 0.9), [V // 2, 0, 40, V], [0.5, 1.0, 1.0, 0.99], [0.0, 0.01, 0.1, 0.0], u)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_captured_calls(dtype):
    """Every kind of path of a type in one graph, replayed on other values."""
    import torch
    from neuraval_b200.sampler import sample_rows_min_p_device
    rng = np.random.default_rng(5)
    rows, V = 30, 20011
    xs = [torch.from_numpy(rng.standard_normal((rows, V)) * s).cuda().to(dtype_of(dtype)) for s in (0.4, 3.0)]
    T, k, p, m, u = options(rng, rows, V)
    alone = [run(x, T, k, p, m, u) for x in xs]
    dev = [torch.from_numpy(np.asarray(a, t)).cuda() for a, t in
           ((u, np.float32), (T, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    x, tokens, lp = xs[0].clone(), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sample_rows_min_p_device(x, dev[0], tokens, *dev[1:], logprobs=lp, stream=torch.cuda.current_stream())
    for i in (1, 0, 1):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(tokens.cpu().numpy(), alone[i]["tokens"])
        assert np.array_equal(lp.cpu().numpy(), alone[i]["logprobs"])


@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows", [1025, 2305, 4111])
def test_many_tiles(rows, dtype, out):
    """More tiles of rows than are worked on at the same time."""
    ids = np.random.default_rng(rows).integers(-1, 6, rows)
    c = Case(rows, 72, 515, [16, 3, 17, 40, 8, 1], ids, dtype, rows, whole=True)
    y, _ = c.want()
    with c.head() as h:
        got = c.run(h, out)
        assert (got == y.float().to(got.dtype)).all()
        bare = (c.x.double() @ c.w.double().T).float().to(got.dtype)
        assert (c.run(h, out, ids=False) == bare).all()


@pytest.mark.parametrize("rows", [90, 500])
def test_every_slot_in_use(rows):
    slots = 1024
    ids = np.random.default_rng(rows).permutation(slots)[:rows]
    ids[-3:] = [slots - 1, 0, slots]
    c = Case(rows, 64, 130, [1 + i % 20 for i in range(slots)], ids, "bf16", rows, whole=True)
    with c.head() as h:
        assert (c.run(h) == c.want()[0].float()).all()


def test_outputs_and_inputs_past_32_bits():
    """Row strides whose last rows lie past 2^32 values, and a weight of more than 2^31."""
    import torch
    from neuraval_b200.adapter_head import CudaAdapterHead
    c = Case(9, 64, 300, [8], [0, -1, 0] * 3, "bf16", 3, whole=True)
    want, ld = c.want()[0].float(), 2 ** 29 + 3
    flat = torch.empty(8 * ld + 300, device="cuda")
    y = flat.as_strided((9, 300), (ld, 1))
    big = torch.empty(8 * ld + 64, device="cuda", dtype=torch.bfloat16).as_strided((9, 64), (ld, 1))
    big.copy_(c.x)
    ids = torch.from_numpy(c.ids.astype(np.int32)).cuda()
    with c.head() as h:
        h.project_device(big, ids, y)
        torch.cuda.synchronize()
    assert (y == want).all()
    del flat, y, big
    out, inner = 600011, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-1, 2, (out, inner), device="cuda", generator=g, dtype=torch.int8).to(torch.bfloat16)
    x = torch.randint(-2, 3, (5, inner), device="cuda", generator=g).to(torch.bfloat16)
    a, b = x[:2].clone(), w[:, :2].contiguous()
    y = torch.empty(5, out, device="cuda")
    with CudaAdapterHead(w, 5, 1, 2) as h:
        h.set_adapter(0, a, b, 0.0625)
        h.project_device(x, torch.tensor([0, -1, 0, 0, -1], dtype=torch.int32, device="cuda"), y)
        torch.cuda.synchronize()
    u = 0.0625 * (x.double() @ a.double().T)
    u[[1, 4]] = 0
    for lo in range(0, out, 50000):
        part = x.double() @ w[lo:lo + 50000].double().T + u @ b[lo:lo + 50000].double().T
        assert (y[:, lo:lo + 50000] == part.float()).all(), lo
