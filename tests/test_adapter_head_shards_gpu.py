"""A head split by vocabulary: each part's logits go to the vocabulary shards of the sampler as they
are, and the tokens are those of the whole head's logits."""
import numpy as np
import pytest

from neuraval_b200 import native, sharding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("greedy", [True, False])
def test_head_parts_to_shard_records(greedy):
    import torch
    from neuraval_b200.adapter_head import CudaAdapterHead
    from neuraval_b200.sampler import CudaTokenSampler
    rows, inner, V, rank, shards = 20, 128, 30011, 8, 2
    g = torch.Generator(device="cuda").manual_seed(2)
    make = lambda *n: torch.randn(*n, device="cuda", generator=g).bfloat16()  # noqa: E731
    w, x = make(V, inner), make(rows, inner)
    a, b = [make(rank, inner) for _ in range(2)], [make(V, rank) for _ in range(2)]
    ids = torch.arange(rows, device="cuda", dtype=torch.int32) % 3 - 1
    u = torch.rand(rows, device="cuda", generator=g)
    hist, offs = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    p = native.make_params(greedy=True) if greedy else native.make_params(temperature=20.0, top_p=0.95, top_k=40)

    def head(lo, hi):
        h = CudaAdapterHead(w[lo:hi], rows, 2, rank)
        for s in range(2):
            h.set_adapter(s, a[s], b[s][lo:hi], 0.5)
        return h

    whole = torch.empty(rows, V, device="cuda")
    with head(0, V) as h, CudaTokenSampler(0, rows, V, 16) as s:
        h.project_device(x, ids, whole)
        want = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s.sample_rows_device(whole, hist, offs, u, p, want)
        recs = torch.zeros((shards, rows, s.shard_record_bytes // 4), dtype=torch.int32, device="cuda")
        for i in range(shards):
            lo, hi = sharding.vocab_range(V, shards, i)
            with head(lo, hi) as part:
                logits = torch.full((rows, hi - lo + 5), float("nan"), device="cuda")[:, :hi - lo]
                part.project_device(x, ids, logits)
                assert torch.equal(logits, whole[:, lo:hi])  # a value's sums do not depend on the others'
                s.shard_candidates_device(logits, V, lo, hist, offs, p, recs[i])
        got, flags = torch.full_like(want, -7), torch.zeros_like(want)
        s.shard_merge_device(recs, shards, rows, V, u, p, got, flags)
        torch.cuda.synchronize()
        assert not (flags & native.FLAG_TIES_OVERFLOW).any()
        assert torch.equal(got, want)
        assert greedy or len(set(np.asarray(got.cpu()))) > 1
