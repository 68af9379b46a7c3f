"""The LM head with adapters on the GPU against its definition in 64 bits.

Two kinds of inputs. Small whole numbers, whose sums fp32 holds exactly: every
output bit has to be right (a misplaced, missing or doubled product shows). And
random values, within a tolerance derived from the arithmetic:
  - sums of n products in fp32: each addition is off by at most 2^-24 of the
    running sum (2^-23 where the hardware truncates, but then for 16 products at
    once); the running sum of products with random signs stays below 6 times
    their 2-norm q, so (K + R + 32) 2^-24 6 q covers them;
  - A_s x_n carried as the sum of two 16-bit values: off by 2^-16 relative
    (bf16: two roundings of 2^-9 and more; fp16: more exact, down to its least
    step, 2^-24), so 2^-16 |B_s| |u| + 2^-24 |B_s| 1;
  - the output's own rounding, half a step of its type.
"""
import numpy as np
import pytest

from neuraval_b200 import native

pytestmark = pytest.mark.gpu

DT = {"bf16": "bfloat16", "f16": "float16", "f32": "float32"}


def dtype_of(name):
    import torch
    return getattr(torch, DT[name])


class Case:
    """Inputs on the GPU and the definition's result."""

    def __init__(self, rows, inner, out, ranks, ids, dtype, seed, whole=False):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = dtype_of(dtype)

        def make(*s, scale=1.0, top=2):
            if whole:
                return torch.randint(-top, top + 1, s, device="cuda", generator=g).to(t)
            return (torch.randn(*s, device="cuda", generator=g) * scale).to(t)

        self.rows, self.inner, self.out, self.ranks = rows, inner, out, ranks
        self.x, self.w = make(rows, inner), make(out, inner, scale=inner ** -0.5)
        self.a = [make(r, inner, scale=inner ** -0.5, top=1) for r in ranks]
        self.b = [make(out, r, scale=0.5 * max(r, 1) ** -0.5) for r in ranks]
        self.scales = [2.0 ** (i % 3 - 1) if whole else 0.5 + 0.37 * i % 1.9 for i in range(len(ranks))]
        self.ids = np.asarray(ids, np.int64)
        if whole and ranks:  # u = scale A x must be whole for the scale of 1/2
            self.a = [a * 2 for a in self.a]

    def want(self):
        """(y, tolerance without the output's rounding)."""
        import torch
        x, w = self.x.double(), self.w.double()
        y, q = x @ w.T, (x ** 2) @ (w ** 2).T
        tol = torch.zeros_like(y)
        R = max(self.ranks, default=0)
        for n, i in enumerate(self.ids):
            if 0 <= i < len(self.ranks) and self.ranks[i]:
                a, b = self.a[i].double(), self.b[i].double()
                u = self.scales[i] * (a @ x[n])
                y[n] += b @ u
                q[n] += (b ** 2) @ (u ** 2)
                # u itself, a sum in fp32
                du = (self.inner + 32) * 2.0 ** -24 * 6 * self.scales[i] * ((a ** 2) @ (x[n] ** 2)).sqrt()
                tol[n] += b.abs() @ (2.0 ** -16 * u.abs() + 2.0 ** -24 + du)
        return y, tol + (self.inner + R + 32) * 2.0 ** -24 * 6 * q.sqrt()

    def head(self, max_rows=None, max_adapters=None, max_rank=None):
        from neuraval_b200.adapter_head import CudaAdapterHead
        h = CudaAdapterHead(self.w, max_rows or self.rows,
                            len(self.ranks) if max_adapters is None else max_adapters,
                            max(self.ranks, default=0) if max_rank is None else max_rank)
        for i, r in enumerate(self.ranks):
            if r:
                h.set_adapter(i, self.a[i], self.b[i], self.scales[i])
        return h

    def run(self, h, out="f32", ids=True):
        import torch
        y = torch.full((self.rows, self.out), float("nan"), device="cuda", dtype=dtype_of(out))
        t = torch.from_numpy(np.clip(self.ids, -2 ** 31, 2 ** 31 - 1).astype(np.int32)).cuda() if ids else None
        h.project_device(self.x, t, y)
        torch.cuda.synchronize()
        return y


def check(y, want, tol):
    import torch
    half = torch.finfo(y.dtype).eps / 2
    err = (y.double() - want).abs()
    bound = tol + half * want.abs() * (1 + 2.0 ** -10) + torch.finfo(y.dtype).tiny
    bad = ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), [int(i) for i in bad.nonzero()[0]],
                           float((err / bound).nan_to_num(nan=1e9).max()))


SHAPES = [(1, 1, 1), (1, 8, 3), (2, 16, 128), (3, 17, 129), (5, 64, 1000), (16, 100, 257),
          (17, 192, 300), (33, 256, 4096), (64, 1000, 515), (100, 72, 3001), (255, 320, 130),
          (256, 512, 2049), (257, 520, 1030), (300, 136, 640), (600, 64, 200), (1, 2048, 32000)]


def some_ids(rng, rows, n):
    return rng.choice(np.arange(-1, n), rows)


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_whole_numbers_are_exact(shape, dtype, out):
    rows, inner, cols = shape
    rng = np.random.default_rng(rows + inner)
    c = Case(rows, inner, cols, [1, 7, 16, 17], some_ids(rng, rows, 4), dtype, rows * 31 + cols, whole=True)
    y, _ = c.want()
    with c.head() as h:
        got = c.run(h, "f32" if out == "f32" else dtype)
    assert y.abs().max() < 2 ** 24
    assert (got == (y.float() if out == "f32" else y.float().to(got.dtype))).all()


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_random_values(shape, dtype, out):
    rows, inner, cols = shape
    rng = np.random.default_rng(rows + cols)
    c = Case(rows, inner, cols, [16, 8, 13, 32, 1], some_ids(rng, rows, 5), dtype, rows * 37 + inner)
    with c.head() as h:
        check(c.run(h, "f32" if out == "f32" else dtype), *c.want())


@pytest.mark.parametrize("ranks,rows", [([128], 40), ([64, 3], 20), ([16] * 40, 40), ([5] * 300, 300),
                                        ([1, 128, 2, 127, 15, 16, 17], 64)],
                         ids=["128", "64_3", "16x40", "5x300", "mixed"])
def test_ranks_and_many_adapters(ranks, rows):
    """One adapter for all rows, an adapter for each row, ranks on both sides of 16."""
    rng = np.random.default_rng(len(ranks))
    ids = rng.permutation(rows) % len(ranks)
    c = Case(rows, 264, 777, ranks, ids, "bf16", 11, whole=True)
    with c.head() as h:
        assert (c.run(h) == c.want()[0].float()).all()
    c = Case(rows, 264, 777, ranks, ids, "f16", 12)
    with c.head() as h:
        check(c.run(h), *c.want())


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("rows", [63, 65, 80, 81, 96, 97, 128, 129, 192, 194])
def test_sizes_where_the_tiles_change(rows, out):
    """Row counts on both sides of each change of tile, with many adapters and mixed ranks."""
    ranks = [16, 1, 17, 48] * 9 + [128]
    ids = np.random.default_rng(rows).integers(-1, len(ranks), rows)
    c = Case(rows, 264, 777, ranks, ids, "bf16", rows, whole=True)
    with c.head() as h:
        got, want = c.run(h, "f32" if out == "f32" else "bf16"), c.want()[0].float()
        assert (got == want.to(got.dtype)).all()
    c = Case(rows, 264, 777, ranks, ids, "bf16", rows + 1)
    with c.head() as h:
        check(c.run(h, "f32" if out == "f32" else "bf16"), *c.want())


def test_ids_without_an_adapter():
    """-1, ids outside the slots, empty and cleared slots: the shared projection alone."""
    ids = [-1, 0, 5, -2 ** 31, 2 ** 31 - 1, 2, 1, 3, 4, 0]
    c = Case(10, 128, 300, [8, 8, 8, 0, 8], ids, "bf16", 3, whole=True)
    with c.head() as h:
        assert (c.run(h) == c.want()[0].float()).all()
        c.ranks[2] = 0
        h.clear_adapter(2)
        assert (c.run(h) == c.want()[0].float()).all()
        bare = c.x.double() @ c.w.double().T
        assert (c.run(h, ids=False) == bare.float()).all()
    with c.head(max_adapters=5, max_rank=8) as h:
        for i in range(5):
            h.clear_adapter(i)
        assert (c.run(h) == bare.float()).all()
    c.ranks = []
    with c.head(max_adapters=0, max_rank=0) as h:
        assert (c.run(h) == bare.float()).all()


def test_slots_are_replaced():
    """A slot loaded again, with another rank and scale, takes effect in stream order."""
    c = Case(12, 96, 515, [16, 9], [0, 1] * 6, "bf16", 5, whole=True)
    d = Case(12, 96, 515, [3, 12], [0, 1] * 6, "bf16", 6, whole=True)
    with c.head() as h:
        assert (c.run(h) == c.want()[0].float()).all()
        for i in range(2):
            h.set_adapter(i, d.a[i], d.b[i], d.scales[i])
        c.ranks, c.a, c.b, c.scales = d.ranks, d.a, d.b, d.scales
        assert (c.run(h) == c.want()[0].float()).all()


def test_fewer_rows_than_the_head_holds():
    c = Case(5, 200, 900, [16, 4], [1, 0, -1, 1, 1], "f16", 7, whole=True)
    with c.head(max_rows=700, max_adapters=9, max_rank=40) as h:
        assert (c.run(h) == c.want()[0].float()).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_strides_alignments_and_guards(pad, dtype):
    """Every input with padded rows that hold NaN between them and a base off the 16-byte grid; the
    output's padding stays as it was."""
    import torch
    rows, inner, cols = 37, 130, 301
    c = Case(rows, inner, cols, [12, 5], np.arange(rows) % 3 - 1, dtype, 9, whole=True)
    y = c.want()[0].float()

    def padded(m):
        flat = torch.full((m.shape[0] * (m.shape[1] + pad) + pad,), float("nan"), device="cuda", dtype=m.dtype)
        v = flat[pad:].view(m.shape[0], m.shape[1] + pad)[:, :m.shape[1]]
        v.copy_(m)
        return v

    c.x, c.w = padded(c.x), padded(c.w)
    c.a, c.b = [padded(m) for m in c.a], [padded(m) for m in c.b]
    with c.head() as h:
        for out in (torch.float32, c.x.dtype):
            flat = torch.full((rows, cols + pad), 77.0, device="cuda", dtype=out)
            h.project_device(c.x, torch.from_numpy(c.ids.astype(np.int32)).cuda(), flat[:, :cols])
            torch.cuda.synchronize()
            assert (flat[:, :cols] == y.to(out)).all() and (flat[:, cols:] == 77.0).all()


def test_weight_set_again():
    import torch
    for pad in (0, 1):  # read in place, and copied
        c = Case(9, 64, 300, [4], [0] * 9, "bf16", 13, whole=True)
        flat = torch.zeros(300, 64 + pad, device="cuda", dtype=torch.bfloat16)
        flat[:, :64] = c.w
        c.w = flat[:, :64]
        with c.head() as h:
            assert (c.run(h) == c.want()[0].float()).all()
            c.w.mul_(-2)
            h.set_weight(c.w)
            assert (c.run(h) == c.want()[0].float()).all()


def test_non_finite_rows_stay_alone():
    """A row of x with NaN, an adapter with NaN in A or an infinity in B: the rows that use it show
    it, the other rows are as they were."""
    c = Case(20, 128, 260, [16, 16], np.arange(20) % 2, "bf16", 15, whole=True)
    want = c.want()[0].float()
    c.x[3, 5] = float("nan")
    with c.head() as h:
        got = c.run(h)
    assert got[3].isnan().all()
    keep = [i for i in range(20) if i != 3]
    assert (got[keep] == want[keep]).all()
    for spoil in (lambda: c.a[1].view(-1)[70:71].fill_(float("nan")), lambda: c.b[1].view(-1)[999:1000].fill_(float("inf"))):
        c = Case(20, 128, 260, [16, 16], np.arange(20) % 2, "bf16", 15, whole=True)
        spoil()
        with c.head() as h:
            got = c.run(h)
            assert not got[1::2].isfinite().all() and (got[::2] == want[::2]).all()
            h.set_adapter(1, c.a[0], c.b[0], 1.0)  # a sound one in its place
            assert c.run(h).isfinite().all()


def test_overflowing_adapter_product_stays_in_its_row():
    """fp16: scale A x beyond the type's range gives NaN in its row, and only there."""
    import torch
    c = Case(90, 64, 300, [8, 8], np.arange(90) % 2, "f16", 17, whole=True)
    want = c.want()[0].float()
    c.x[3] = 1000.0
    c.a[1][:] = 10.0
    with c.head() as h:
        got = c.run(h)
    assert got[3].isnan().all() and (got[::2] == want[::2]).all()
    assert got[1::2][torch.arange(45) != 1].isfinite().all()


def test_refusals_with_a_head():
    import torch
    from neuraval_b200.adapter_head import CudaAdapterHead
    lib = native.load()
    w = torch.zeros(100, 64, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros(8, 100, device="cuda")
    ids = torch.zeros(8, device="cuda", dtype=torch.int32)
    a, b = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(100, 4, device="cuda", dtype=torch.bfloat16)
    with CudaAdapterHead(w, 8, 2, 4) as h:
        P = lambda t: t.data_ptr()  # noqa: E731
        inv, cap = native.NCB_ERROR_INVALID_ARGUMENT, native.NCB_ERROR_CAPACITY
        for args, st in [((P(x), 63, 8, P(ids), P(y), 0, 100), inv), ((P(x), 64, 8, P(ids), P(y), 0, 99), inv),
                         ((P(x), 64, -1, P(ids), P(y), 0, 100), inv), ((P(x), 64, 9, P(ids), P(y), 0, 100), cap),
                         ((None, 64, 8, P(ids), P(y), 0, 100), inv), ((P(x), 64, 8, P(ids), None, 0, 100), inv),
                         ((P(x), 64, 8, P(ids), P(y), 1, 100), inv), ((P(x) + 1, 64, 8, P(ids), P(y), 0, 100), inv),
                         ((P(x), 64, 8, P(ids) + 2, P(y), 0, 100), inv), ((P(x), 64, 8, P(ids), P(y) + 2, 0, 100), inv),
                         ((None, 0, 0, None, None, 0, 0), native.NCB_OK)]:
            assert lib.ncb_adapter_head_project_device(h._h, *args, None) == st, args
        for args, st in [((2, P(a), 64, P(b), 4, 4, 1.0), inv), ((-1, P(a), 64, P(b), 4, 4, 1.0), inv),
                         ((0, P(a), 64, P(b), 5, 5, 1.0), cap), ((0, P(a), 64, P(b), 4, 0, 1.0), inv),
                         ((0, P(a), 63, P(b), 4, 4, 1.0), inv), ((0, P(a), 64, P(b), 3, 4, 1.0), inv),
                         ((0, P(a), 64, P(b), 4, 4, float("nan")), inv), ((0, None, 64, P(b), 4, 4, 1.0), inv)]:
            assert lib.ncb_adapter_head_set_adapter_device(h._h, *args, None) == st, args
        for bad in (lambda: h.project_device(x.float(), ids, y), lambda: h.project_device(x, ids.long(), y),
                    lambda: h.project_device(x, ids[:7], y), lambda: h.project_device(x, ids, y[:7]),
                    lambda: h.project_device(x, ids, y.half()), lambda: h.project_device(x.T, ids, y),
                    lambda: h.set_adapter(0, a, b[:, :3]), lambda: h.set_adapter(0, a[:, :63], b),
                    lambda: h.set_weight(w[:99]), lambda: h.project_device(x.cpu(), ids, y)):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(native.NcbError):
            h.set_adapter(0, torch.zeros(5, 64, device="cuda", dtype=w.dtype), torch.zeros(100, 5, device="cuda", dtype=w.dtype))


def test_graph_replay_and_two_heads_on_two_streams():
    """A captured call sees inputs, ids and adapters that change under it; two handles run at once."""
    import torch
    cs = [Case(24, 256, 2000, [16, 8, 4], np.arange(24) % 4 - 1, "bf16", s, whole=True) for s in (20, 21)]
    heads = [c.head() for c in cs]
    want = [c.want()[0].float() for c in cs]
    ids = torch.from_numpy(cs[0].ids.astype(np.int32)).cuda()
    streams = [torch.cuda.Stream() for _ in cs]
    ys = [[torch.zeros(24, 2000, device="cuda") for _ in range(5)] for _ in cs]
    torch.cuda.synchronize()
    for j in range(5):
        for c, h, s, y in zip(cs, heads, streams, ys):
            h.project_device(c.x, ids, y[j], stream=s)
    torch.cuda.synchronize()
    for w, y in zip(want, ys):
        assert all((t == w).all() for t in y)
    c, h = cs[0], heads[0]
    y = torch.zeros(24, 2000, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h.project_device(c.x, ids, y, stream=torch.cuda.current_stream())
    g.replay()
    torch.cuda.synchronize()
    assert (y == want[0]).all()
    c.x.copy_(cs[1].x)
    c.ids = (c.ids + 2) % 4 - 1
    ids.copy_(torch.from_numpy(c.ids))
    h.set_adapter(1, cs[1].a[2], cs[1].b[2], 2.0)
    c.ranks[1], c.a[1], c.b[1], c.scales[1] = 4, cs[1].a[2], cs[1].b[2], 2.0
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert (y == c.want()[0].float()).all()
    for h in heads:
        h.close()


def test_head_then_sampler():
    """Hidden states -> logits with each request's adapter -> a token by each request's options, in
    one stream without a wait between, fp32 and 16-bit logits with padded rows."""
    import torch
    from neuraval_b200.sampler import CudaTokenSampler, sample_rows_min_p_device
    from tests.min_p_ref import sample_rows
    rng = np.random.default_rng(40)
    rows, cols = 48, 5003
    c = Case(rows, 256, cols, [16, 8, 12], rng.integers(-1, 3, rows), "bf16", 41)
    ids = torch.from_numpy(c.ids.astype(np.int32)).cuda()
    T, k = rng.uniform(0.5, 1.2, rows).astype(np.float32), rng.choice([0, 5, 50], rows).astype(np.int32)
    p, m = rng.uniform(0.5, 1.0, rows).astype(np.float32), rng.choice([0.0, 0.1], rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    dev = [torch.from_numpy(z).cuda() for z in (u, T, k, p, m)]
    with c.head() as h:
        for t in (torch.float32, torch.bfloat16):
            buf = torch.full((rows, cols + 5), float("nan"), device="cuda", dtype=t)
            logits, tokens = buf[:, :cols], torch.zeros(rows, dtype=torch.int32, device="cuda")
            h.project_device(c.x, ids, logits)
            sample_rows_min_p_device(logits, dev[0], tokens, *dev[1:])
            torch.cuda.synchronize()
            want, _, _ = sample_rows(logits.double().cpu().numpy(), T, k, p, m, u)
            assert np.array_equal(tokens.cpu().numpy(), want)
            check(logits, *c.want())
        # and the sampler with one set of options for the batch, from the same logits
        logits = torch.empty(rows, cols, device="cuda")
        h.project_device(c.x, ids, logits)
        with CudaTokenSampler(0, rows, cols, 16) as s:
            hist, offs = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
            tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
            s.sample_rows_device(logits, hist, offs, dev[0], native.make_params(greedy=True), tokens)
            torch.cuda.synchronize()
            assert (tokens == logits.argmax(1)).all()
