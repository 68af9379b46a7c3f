"""The LM head with adapters on tiles of every kind (single CTAs, sorted pairs of CTAs, several
tiles): rows with non-finite values stay alone and leave nothing behind, and a call repeats itself
bit by bit."""
import numpy as np
import pytest

from tests.test_adapter_head_gpu import Case

pytestmark = pytest.mark.gpu

# slots of uneven sizes, some over several blocks of 32 rows, some within one, and rows without
SHARES = [0.30, 0.02, 0.25, 0.05, 0.13, 0.15]
RANKS = [16, 5, 40, 16, 17]


def uneven(rows):
    """Slots by shares, shuffled; the last share has no adapter."""
    n = np.maximum(1, np.round(np.array(SHARES) * rows).astype(int))
    ids = np.repeat([0, 1, 2, 3, 4, -1], n)[:rows]
    ids = np.concatenate([ids, np.full(rows - len(ids), -1)])
    return np.random.default_rng(rows).permutation(ids)


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [20, 90, 130, 250, 300, 520])
@pytest.mark.parametrize("spoilt", ["x", "a_nan", "a_inf", "b_inf", "b_nan"])
def test_non_finite_values_stay_in_their_rows(spoilt, rows, dtype, out):
    """Every value of a row whose adapter (or x) holds one is NaN, all others are exact; so is the
    next call on the same head, whose scratch held the NaN, with the values mended."""
    c = Case(rows, 96, 270, RANKS, uneven(rows), dtype, rows + 3, whole=True)
    want = c.want()[0].float()
    out = "f32" if out == "f32" else dtype
    slot = 2  # over several blocks in the larger tiles
    mine = c.ids == slot
    assert mine.any()
    kept = {"x": c.x, "a": c.a[slot], "b": c.b[slot]}
    if spoilt == "x":
        mine = np.zeros(rows, bool)
        mine[[0, rows // 2, rows - 1]] = True
        kept["x"] = c.x.clone()
        c.x[np.flatnonzero(mine), 7] = float("nan")
    elif spoilt[0] == "a":
        c.a[slot] = c.a[slot].clone()
        c.a[slot][3, 50] = float(spoilt[2:])
    else:
        c.b[slot] = c.b[slot].clone()
        c.b[slot][200, 33] = float(spoilt[2:])
    with c.head() as h:
        got = c.run(h, out)
        assert got[mine].isnan().all()
        assert (got[~mine] == want.to(got.dtype)[~mine]).all()
        c.x, c.a[slot], c.b[slot] = kept["x"], kept["a"], kept["b"]
        h.set_adapter(slot, c.a[slot], c.b[slot], c.scales[slot])
        got = c.run(h, out)
        assert (got == want.to(got.dtype)).all()


@pytest.mark.parametrize("rows", [90, 250, 520])
def test_products_past_the_type_stay_in_their_rows(rows):
    """fp16: scale A x beyond 65504 gives NaN in its row, and only there."""
    c = Case(rows, 64, 300, RANKS, uneven(rows), "f16", rows, whole=True)
    want = c.want()[0].float()
    r = int(np.flatnonzero(c.ids == 0)[-1])
    c.x[r] = 1000.0
    c.a[0] = c.a[0].abs() + 10.0
    want_0 = c.want()[0].float()
    with c.head() as h:
        got = c.run(h)
    assert got[r].isnan().all()
    for i in range(rows):
        if i != r:
            assert (got[i] == (want_0 if c.ids[i] == 0 else want)[i]).all(), i


@pytest.mark.parametrize("dtype,out", [("bf16", "same"), ("bf16", "f32"), ("f16", "same"), ("f16", "f32")])
@pytest.mark.parametrize("rows", [7, 96, 256, 512])
def test_a_call_repeats_itself(rows, dtype, out):
    """The same bits from the same call, alone and with calls on other inputs between, on one head and
    on another one with the same contents."""
    import torch
    out = "f32" if out == "f32" else dtype
    ranks = [16, 8, 31, 32] * 4
    ids = np.random.default_rng(rows).integers(-1, len(ranks), rows)
    c = Case(rows, 1032, 5000, ranks, ids, dtype, 50 + rows)
    d = Case(rows, 1032, 5000, ranks, ids[::-1].copy(), dtype, 60 + rows)
    with c.head() as h, c.head() as other:
        first = c.run(h, out)
        assert first.isfinite().all()
        bits = lambda t: t.view(torch.int32 if out == "f32" else torch.int16)  # noqa: E731
        for turn in range(12):
            if turn % 3 == 1:
                d.run(h, out)
            assert torch.equal(bits(c.run(other if turn % 4 == 3 else h, out)), bits(first)), turn
