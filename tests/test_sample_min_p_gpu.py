"""Sampling with options per row on the GPU against the definition in 64 bits
(tests/min_p_ref.py): tokens and counts equal, the log-probability within the
rounding of its type.

Tolerance: the kernel's and the definition's 64-bit sums agree to about 1e-13
relative (2^18 terms rounded at 2^-53 each), so a log-probability is off by its
own rounding to fp32, at most 2^-24 relative, and 1e-11 more.
"""
import numpy as np
import pytest

from neuraval_b200 import native
from tests.min_p_ref import sample_rows

pytestmark = pytest.mark.gpu

BAD = native.FLAG_NONFINITE | native.FLAG_BAD_OPTIONS


def run(x, T=None, k=None, p=None, m=None, u=None, stream=None):
    """x: a CUDA tensor; the options: numpy arrays or None."""
    import torch
    from neuraval_b200.sampler import sample_rows_min_p_device
    rows = x.shape[0]
    dev = lambda a, t: None if a is None else torch.from_numpy(np.asarray(a, t)).cuda()  # noqa: E731
    out = dict(tokens=torch.full((rows,), -7, dtype=torch.int32, device="cuda"),
               logprobs=torch.full((rows,), 5.0, device="cuda"),
               kept=torch.full((rows,), -7, dtype=torch.int32, device="cuda"),
               flags=torch.full((rows,), -1, dtype=torch.int32, device="cuda"))
    sample_rows_min_p_device(x, dev(u, np.float32), out["tokens"], dev(T, np.float32),
                             dev(k, np.int32), dev(p, np.float32), dev(m, np.float32),
                             out["logprobs"], out["kept"], out["flags"], stream)
    torch.cuda.synchronize()
    return {n: t.cpu().numpy() for n, t in out.items()}


def compare(x, T=None, k=None, p=None, m=None, u=None):
    rows = x.shape[0]
    got = run(x, T, k, p, m, u)
    f = lambda a, t, d: np.full(rows, d, t) if a is None else np.asarray(a, t)  # noqa: E731
    tok, kept, lp = sample_rows(x.double().cpu().numpy(), f(T, np.float32, 1), f(k, np.int32, 0),
                                f(p, np.float32, 1), f(m, np.float32, 0), f(u, np.float32, 0))
    assert not got["flags"].any()
    bad = np.flatnonzero((got["tokens"] != tok) | (got["kept"] != kept))
    assert bad.size == 0, [(r, got["tokens"][r], tok[r], got["kept"][r], kept[r]) for r in bad[:5]]
    assert np.all(np.abs(got["logprobs"] - lp) <= 2.0 ** -24 * np.abs(lp) + 1e-11)
    return got


def dtype_of(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def options(rng, rows, V):
    """Every kind of option, on and off, in one batch."""
    T = rng.uniform(0.3, 1.5, rows)
    T[rng.random(rows) < 0.1] = 0.0
    k = np.where(rng.random(rows) < 0.5, 0, rng.choice([1, 2, 5, 50, 200, 3000, V, V + 7], rows))
    p = np.where(rng.random(rows) < 0.4, 1.0, rng.uniform(0.05, 0.999, rows))
    m = np.where(rng.random(rows) < 0.5, 0.0, rng.uniform(0.001, 0.6, rows))
    u = np.minimum(rng.random(rows).astype(np.float32), np.float32(1 - 2.0 ** -24))
    return T, k, p, m, u


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [(1, 1), (5, 2), (7, 3), (9, 31), (3, 33), (64, 100), (40, 1000),
                                    (33, 4097), (12, 32000), (300, 9000), (6, 50257), (4, 151936)])
def test_mixed_options(rows, V, dtype):
    import torch
    rng = np.random.default_rng(rows * 1000003 + V)
    x = rng.standard_normal((rows, V)) * rng.choice([0.5, 2.0, 5.0], rows)[:, None]
    compare(torch.from_numpy(x).cuda().to(dtype_of(dtype)), *options(rng, rows, V))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("law", ["flat", "equal", "two", "coarse", "zipf"])
def test_value_laws(law, dtype):
    """Rows from flat to peaked, full of ties, at a size where the wanted values fill no list."""
    import torch
    rng = np.random.default_rng(5)
    rows, V = 24, 40003
    x = rng.standard_normal((rows, V))
    if law == "flat":
        x *= 0.3
    elif law == "equal":
        x[:] = -3.25
    elif law == "two":
        x = np.where(x > 1.0, 2.0, 1.0)
    elif law == "coarse":
        x = np.round(x * 2) / 2
    else:
        x = x * 2 - 1.2 * np.log1p(rng.integers(0, V, (rows, V)))
    T, k, p, m, u = options(rng, rows, V)
    compare(torch.from_numpy(x).cuda().to(dtype_of(dtype)), np.where(T == 0, 1.0, T), k, p, m, u)


@pytest.mark.parametrize("dtype,V", [("f32", 400003), ("bf16", 800001), ("f16", 600011)])
def test_rows_too_long_for_shared_memory(dtype, V):
    import torch
    rng = np.random.default_rng(V)
    x = rng.standard_normal((3, V)) * np.array([0.4, 1.5, 4.0])[:, None]
    compare(torch.from_numpy(x).cuda().to(dtype_of(dtype)), [1.0, 0.8, 1.1], [0, 0, 40],
            [0.97, 0.9, 1.0], [0.0, 0.01, 0.0], [0.93, 0.999, 0.5])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_banned_and_lowest_values(dtype):
    """-inf is never kept; the type's lowest value is an ordinary value without mass; rows with one
    finite value, with lowest values only, and with only their first or last value finite."""
    import torch
    rng = np.random.default_rng(9)
    t = dtype_of(dtype)
    rows, V = 16, 5003
    x = torch.from_numpy(rng.standard_normal((rows, V)) * 3).cuda().to(t)
    low = torch.finfo(t).min
    x[0:6, 64:4900] = -float("inf")
    x[6:9, 64:4900] = low
    x[9] = low
    x[10] = -float("inf")
    x[10, 0] = 1.0
    x[11] = -float("inf")
    x[11, V - 1] = -2.0
    x[12] = -float("inf")
    x[12, 17:19] = low
    x[13, :] = torch.finfo(t).max
    x[14, 5] = torch.finfo(t).max
    _, k, p, m, u = options(rng, rows, V)
    # a banned value is not a value: k beyond the finite ones keeps them all
    k[2], p[2], m[2] = 4000, 1.0, 0.0
    k[7], p[7], m[7] = 3000, 1.0, 0.0   # the k-th value is a lowest one
    k[8], p[8], m[8] = 0, 1.0, 0.0
    got = compare(x, np.full(rows, 0.9), k, p, m, u)
    assert got["kept"][2] == V - 4836 and got["kept"][7] == 3000 and got["kept"][8] == V


def test_zeros_of_both_signs_are_equal():
    import torch
    x = torch.zeros(4, 3001, device="cuda")
    x[:, ::2] = -0.0
    x[2:, 1000] = -1e-40
    got = compare(x, None, [5, 0, 3000, 0], [1, 0.5, 1, 0.999], None, [0.99, 0.9, 0.9999, 0.9995])
    assert got["tokens"][0] == 4
    # many zeros, many values on either side that differ from them in the last bits only
    rng = np.random.default_rng(3)
    y = rng.choice(np.array([0.0, -0.0, 1e-45, -1e-45, 3e-39, -3e-39]), (6, 60000))
    y[:, 7] = -80.0
    compare(torch.from_numpy(y).float().cuda(), None, [0, 0, 0, 30000, 10000, 50000],
            [1, .7, .3, 1, .5, .9], None, rng.random(6))


@pytest.mark.parametrize("spread", [1, 64, 5000])
def test_one_bin_holds_nearly_all(spread):
    """Values that differ in their last bits, with one far below them: the bins of values hold more
    than a list, and are divided by their bits."""
    import torch
    rng = np.random.default_rng(spread)
    rows, V = 10, 70001
    x = (1.0 + rng.integers(0, spread, (rows, V)) * 2.0 ** -23).astype(np.float32)
    x[:, 3] = -40.0
    x[5:, 100:200] = 1.5
    compare(torch.from_numpy(x).cuda(), np.full(rows, 1.0), [0, 0, 5000, 60000, 70001, 0, 0, 3000, 150, 0],
            [1, .9, 1, .5, 1, .99, .3, .8, .9, 1], np.full(rows, 0.0),
            [.5, .999, .01, .7, .9999, 0, .25, .6, .5, .99999])


def test_mass_in_clumps():
    """Guessed crossings miss: half the values sit at one edge of their bin, so the masses that
    counts suggest are off by up to a bin."""
    import torch
    rng = np.random.default_rng(31)
    rows, V = 12, 120000
    steps = rng.integers(0, 40, (rows, V))
    x = (-steps * 0.5 - rng.choice([0.0, 0.2399, 0.24], (rows, V))).astype(np.float32)
    x[:, 11] = 0.0
    x[:, 12] = -60.0
    compare(torch.from_numpy(x).cuda(), rng.uniform(0.7, 9.0, rows), None, rng.uniform(0.5, 0.999, rows),
            None, rng.random(rows))


@pytest.mark.parametrize("T", [1e-38, 1e-6, 1e6, 3e38])
def test_extreme_temperatures(T):
    import torch
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((6, 20011)) * 4).float().cuda()
    compare(x, np.full(6, T), [0, 0, 7, 0, 3000, 0], [1, .9, 1, .5, .8, .99], [0, 0, 0, .5, 1.0, .01],
            [.1, .5, .9, .99, .3, .7])


def test_extreme_values():
    import torch
    x = torch.zeros(5, 777, device="cuda")
    x[0] = 3e38
    x[0, 5:] = -3e38
    x[1] = torch.from_numpy(np.linspace(-3e38, 3e38, 777))  # torch.linspace's own step overflows here
    x[2] = 1e-45
    x[2, 9] = 3e-45
    x[3] = -3.4e38
    x[4] = torch.linspace(100.0, 100.001, 777)
    compare(x, [1, 3e37, 1e-45, 1, 1e-4], [0, 0, 700, 4, 0], [.9, .9, 1, 1, .6], [0, 0.01, 0, 0, .3],
            [.3, .8, .5, .99, .77])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_bad_rows_are_flagged_and_leave_the_others_alone(dtype):
    import torch
    rng = np.random.default_rng(4)
    rows, V = 14, 10007
    x = torch.from_numpy(rng.standard_normal((rows, V)) * 2).cuda().to(dtype_of(dtype))
    x[1, V - 1] = float("nan")
    x[2, 0] = float("inf")
    x[3] = -float("inf")
    T = np.full(rows, 0.8, np.float32)
    p, m, u = np.full(rows, 0.9, np.float32), np.full(rows, 0.02, np.float32), rng.random(rows).astype(np.float32)
    T[4], T[5], T[6] = -1.0, np.nan, np.inf
    p[7], p[8] = 0.0, np.nan
    m[9], m[10] = 1.5, -0.1
    u[11], u[12] = 1.0, np.nan
    got = run(x, T, None, p, m, u)
    assert list(got["flags"][1:4]) == [native.FLAG_NONFINITE] * 3
    assert list(got["flags"][4:13]) == [native.FLAG_BAD_OPTIONS] * 9
    assert (got["tokens"][1:13] == -1).all() and (got["kept"][1:13] == 0).all()
    assert np.isnan(got["logprobs"][1:13]).all()
    for r in (0, 13):
        assert got["flags"][r] == 0
        tok, kept, _ = sample_rows(x[r:r + 1].double().cpu().numpy(), T[r:], [0], p[r:], m[r:], u[r:])
        assert got["tokens"][r] == tok[0] and got["kept"][r] == kept[0]
    # greedy rows read none of the other options
    z = run(x[:1], [0.0], None, [np.nan], [-3.0], [np.nan])
    assert z["flags"][0] == 0 and z["tokens"][0] == int(x[0].float().argmax())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides_and_alignments(dtype):
    """Rows at every alignment, between values that must not be read as theirs."""
    import torch
    rng = np.random.default_rng(8)
    t = dtype_of(dtype)
    for V, ld, shift in [(1000, 1003, 1), (997, 2001, 3), (5, 9, 5), (8, 8, 7), (33001, 33009, 1)]:
        rows = 9
        flat = torch.full((rows * ld + shift + 16,), float("nan"), device="cuda", dtype=t)
        x = flat[shift:shift + rows * ld].view(rows, ld)[:, :V]
        x.copy_(torch.from_numpy(rng.standard_normal((rows, V)) * 2).cuda())
        compare(x, *options(rng, rows, V))


def test_options_left_out():
    import torch
    rng = np.random.default_rng(12)
    x = torch.from_numpy(rng.standard_normal((20, 3000)) * 3).float().cuda()
    u = rng.random(20)
    compare(x, u=u)
    compare(x, T=np.full(20, 0.7), m=np.full(20, 0.1), u=u)
    # only the tokens asked for
    from neuraval_b200.sampler import sample_rows_min_p_device
    tokens = torch.zeros(20, dtype=torch.int32, device="cuda")
    sample_rows_min_p_device(x, torch.from_numpy(u.astype(np.float32)).cuda(), tokens)
    torch.cuda.synchronize()
    assert np.array_equal(tokens.cpu().numpy(), run(x, u=u)["tokens"])


def test_same_call_same_bits_and_streams_and_graphs():
    """Two streams at once, and a captured call replayed with other inputs: the bits of a call alone."""
    import torch
    from neuraval_b200.sampler import sample_rows_min_p_device
    rng = np.random.default_rng(21)
    rows, V = 40, 30011
    xs = [torch.from_numpy(rng.standard_normal((rows, V)) * s).cuda().to(torch.bfloat16) for s in (0.5, 3.0)]
    T, k, p, m, u = options(rng, rows, V)
    alone = [run(x, T, k, p, m, u) for x in xs]
    dev = [torch.from_numpy(np.asarray(a, t)).cuda() for a, t in
           ((u, np.float32), (T, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]

    def outputs():
        return (torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda"),
                torch.zeros(rows, dtype=torch.int32, device="cuda"))

    def call(x, o, stream):
        sample_rows_min_p_device(x, dev[0], o[0], dev[1], dev[2], dev[3], dev[4], o[1], o[2], stream=stream)

    streams = [torch.cuda.Stream() for _ in xs]
    outs = [[outputs() for _ in range(4)] for _ in xs]
    torch.cuda.synchronize()
    for j in range(4):
        for i, x in enumerate(xs):
            call(x, outs[i][j], streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            for got, want in zip(o, (alone[i]["tokens"], alone[i]["logprobs"], alone[i]["kept"])):
                assert np.array_equal(got.cpu().numpy(), want)
    x, o = xs[0].clone(), outputs()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(x, o, torch.cuda.current_stream())
    for i in (1, 0):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(o[0].cpu().numpy(), alone[i]["tokens"])
        assert np.array_equal(o[1].cpu().numpy(), alone[i]["logprobs"])


def test_draws_follow_the_distribution_in_order():
    """Uniforms over a grid visit every kept token, in the order of falling values, as often as its
    probability says (the grid's own spacing either way)."""
    import torch
    n = 2000
    w = np.array([0.05, 0.4, 0.1, 0.25, 0.2])
    x = torch.log(torch.from_numpy(w)).float().cuda().expand(n, 5)
    u = (np.arange(n) + 0.5) / n
    got = run(x.contiguous(), None, np.full(n, 4), None, None, u)["tokens"]
    order = [1, 3, 4, 2]
    assert [t for i, t in enumerate(got) if i == 0 or got[i - 1] != t] == order
    for t in order:
        assert abs((got == t).mean() - w[t] / w[order].sum()) <= 1.0 / n
