"""The serving operators that are measured: sampling with per-request options,
and the LM head with low-rank adapters of many requests.

`run` computes a case in its plain form (elementary torch operations) or, where
`own` is true, by the framework's calls. Sampling:

  d_i = (x_i - max x) / T, w_i = exp(d_i), order: x descending, id ascending
  the first top_k of the order, total Z; its smallest prefix of mass >= top_p Z;
  of that the values with w_i >= min_p; the first of the order whose prefix mass
  exceeds u times the mass that is left

The plain form takes it in 64 bits: a token is decided by a comparison of long
sums. The head: out_n = W x_n + s_a B_a (A_a x_n), a the adapter of row n.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request alone on a 32000-token vocabulary: latency
        {"name": "sample_1x32000_f32", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "f32", "law": "peaked",
         "top_k": "on", "top_p": "on", "min_p": "on", "banned": 0.0},
        # a small batch of nucleus requests in fp16, no top-k
        {"name": "sample_32x32000_f16", "op": "sample", "rows": 32, "vocab": 32000, "dtype": "f16", "law": "normal",
         "top_k": "off", "top_p": "on", "min_p": "off", "banned": 0.0},
        # the batch that a bf16 LM head leaves, every request with options of its own
        {"name": "sample_256x128256_bf16", "op": "sample", "rows": 256, "vocab": 128256, "dtype": "bf16", "law": "zipf",
         "top_k": "mixed", "top_p": "mixed", "min_p": "mixed", "banned": 0.0},
        # the same in fp32 with the usual top-k, top-p and min-p together
        {"name": "sample_256x128256_f32", "op": "sample", "rows": 256, "vocab": 128256, "dtype": "f32", "law": "zipf",
         "top_k": "on", "top_p": "on", "min_p": "on", "banned": 0.0},
        # constrained decoding: nine tokens of ten banned, an odd vocabulary
        {"name": "sample_100x50257_bf16_banned", "op": "sample", "rows": 100, "vocab": 50257, "dtype": "bf16", "law": "zipf",
         "top_k": "off", "top_p": "on", "min_p": "mixed", "banned": 0.9},
        # high temperature, nearly flat rows: the nucleus holds most of the vocabulary
        {"name": "sample_1024x151936_f32_flat", "op": "sample", "rows": 1024, "vocab": 151936, "dtype": "f32", "law": "flat",
         "top_k": "off", "top_p": "on", "min_p": "mixed", "banned": 0.0},
        # one token of one request through a small head
        {"name": "head_1x2048x32000_bf16", "op": "head", "rows": 1, "inner": 2048, "vocab": 32000, "dtype": "bf16", "out": "f32",
         "adapters": 1, "rank": 16, "ranks": "same", "bare": 0.0},
        # odd sizes: a vocabulary and ranks that fill no tile, fp16
        {"name": "head_7x1000x50257_f16", "op": "head", "rows": 7, "inner": 1000, "vocab": 50257, "dtype": "f16", "out": "f16",
         "adapters": 5, "rank": 13, "ranks": "mixed", "bare": 0.2},
        # an ordinary decode batch, logits for the fp32 sampler
        {"name": "head_32x4096x128256_bf16", "op": "head", "rows": 32, "inner": 4096, "vocab": 128256, "dtype": "bf16", "out": "f32",
         "adapters": 8, "rank": 16, "ranks": "same", "bare": 0.25},
        # a full decode batch with many tenants
        {"name": "head_256x4096x128256_bf16", "op": "head", "rows": 256, "inner": 4096, "vocab": 128256, "dtype": "bf16", "out": "bf16",
         "adapters": 32, "rank": 16, "ranks": "mixed", "bare": 0.1},
        # the largest: two tiles of rows, the widest vocabulary of the two
        {"name": "head_512x4096x151936_bf16", "op": "head", "rows": 512, "inner": 4096, "vocab": 151936, "dtype": "bf16", "out": "bf16",
         "adapters": 16, "rank": 32, "ranks": "same", "bare": 0.1},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _spread(rng, 100, 262144)
        rows = min(_spread(rng, 1, 1024), max(1, 1024 * 151936 // (2 * vocab)))
        return {"op": "sample", "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "f16", "bf16"]),
                "law": rng.choice(["peaked", "normal", "zipf", "flat"]), "top_k": rng.choice(["on", "off", "mixed"]),
                "top_p": rng.choice(["on", "off", "mixed"]), "min_p": rng.choice(["on", "off", "mixed"]),
                "banned": rng.choice([0.0, 0.0, 0.5, 0.95])}
    inner, vocab, rows = _spread(rng, 64, 8192), _spread(rng, 200, 151936), _spread(rng, 1, 512)
    if rng.random() < 0.6:
        inner = max(64, inner // 64 * 64)
    while inner * vocab > 4096 * 151936:
        inner = max(64, inner // 2)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    return {"op": "head", "rows": rows, "inner": inner, "vocab": vocab, "dtype": dtype, "out": rng.choice(["f32", dtype]),
            "adapters": _spread(rng, 1, 32), "rank": _spread(rng, 1, 32), "ranks": rng.choice(["same", "mixed"]),
            "bare": rng.choice([0.0, 0.1, 0.5])}


def _options(case, seed):
    """Each row's T, top_k, top_p, min_p and uniform: the ranges that requests ask for."""
    r, n, V = np.random.RandomState(seed % (2 ** 31)), case["rows"], case["vocab"]

    def asked(mode, on, off):
        use = np.ones(n, bool) if mode == "on" else np.zeros(n, bool) if mode == "off" else r.rand(n) < 0.5
        return np.where(use, on, off)

    hot = case["law"] == "flat"
    T = r.uniform(1.0, 1.4, n) if hot else r.uniform(0.5, 1.2, n)
    if case["top_k"] == "mixed":  # some requests decode greedily
        T = np.where(r.rand(n) < 0.1, 0.0, T)
    k = asked(case["top_k"], np.minimum(r.choice([1, 20, 40, 50, 64, 200], n), V), 0)
    p = asked(case["top_p"], r.uniform(0.8, 0.99, n), 1.0)
    m = asked(case["min_p"], r.uniform(0.01, 0.2, n), 0.0)
    u = np.minimum(r.rand(n).astype(np.float32), np.float32(1 - 2.0 ** -24))
    return T.astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32), u


def _ids(case, seed):
    """Each row's adapter, all of them in use where there are rows enough, -1 for rows without one; each adapter's rank and scale."""
    r, n = np.random.RandomState(seed % (2 ** 31)), case["rows"]
    ids = np.where(r.rand(n) < case["bare"], -1, r.permutation(n) % case["adapters"]).astype(np.int32)
    ranks = np.full(case["adapters"], case["rank"]) if case["ranks"] == "same" else r.randint(1, case["rank"] + 1, case["adapters"])
    return ids, [int(x) for x in ranks], [float(x) for x in r.choice([0.5, 1.0, 2.0], case["adapters"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dtype, n, V = DTYPES[case["dtype"]], case["rows"], case["vocab"]
    if case["op"] == "sample":
        x = randn(n, V) * {"peaked": 3.0, "normal": 2.0, "zipf": 2.5, "flat": 0.5}[case["law"]]
        if case["law"] == "peaked":
            x[torch.arange(n, device="cuda")[:, None], torch.randint(V, (n, 8), device="cuda", generator=g)] += 8.0
        if case["law"] == "zipf":
            fall = -12.0 / math.log(V) * torch.log1p(torch.arange(V, device="cuda", dtype=torch.float32))
            x += fall[torch.randint(V, (n, V), device="cuda", generator=g)]
        if case["banned"]:
            ban = torch.rand(n, V, device="cuda", generator=g) < case["banned"]
            ban[:, 0] = False
            x.masked_fill_(ban, -math.inf)
        T, k, p, m, u = (torch.from_numpy(o).cuda() for o in _options(case, seed))
        state = {"op": "sample", "logits": x.to(dtype), "temperature": T, "top_k": k, "top_p": p, "min_p": m, "uniforms": u}
        if own:
            state |= {"tokens": torch.empty(n, dtype=torch.int32, device="cuda"), "kept": torch.empty(n, dtype=torch.int32, device="cuda"),
                      "logprobs": torch.empty(n, device="cuda")}
        return state
    K, R, A = case["inner"], case["rank"], case["adapters"]
    ids, ranks, scales = _ids(case, seed)
    state = {"op": "head", "x": randn(n, K).to(dtype), "weight": torch.empty(V, K, dtype=dtype, device="cuda").normal_(0, K ** -0.5, generator=g),
             "ids": torch.from_numpy(ids).cuda(), "scales": torch.tensor(scales, device="cuda"), "out_dtype": DTYPES[case["out"]]}
    live = (torch.arange(R, device="cuda")[None, :] < torch.tensor(ranks, device="cuda")[:, None]).to(dtype)
    state["a"] = (randn(A, R, K) * K ** -0.5).to(dtype) * live[:, :, None]  # past an adapter's rank: zeros
    state["b"] = (torch.empty(A, V, R, dtype=dtype, device="cuda").normal_(0, 0.5 * R ** -0.5, generator=g)) * live[:, None, :]
    if own:
        from neuraval_b200.adapter_head import CudaAdapterHead
        head = CudaAdapterHead(state["weight"], max_rows=n, max_adapters=A, max_rank=R)
        for i, r in enumerate(ranks):
            head.set_adapter(i, state["a"][i, :r], state["b"][i, :, :r], scales[i])
        state |= {"head": head, "out": torch.empty(n, V, dtype=state["out_dtype"], device="cuda")}
    return state


def _sample_plain(s):
    x, T = s["logits"].double(), s["temperature"].double()[:, None]
    greedy = T == 0
    d = (x - x.max(1, keepdim=True).values) / torch.where(greedy, 1.0, T)
    d, ids = torch.sort(d, dim=1, descending=True, stable=True)
    del x
    w = torch.exp(d)
    rank = torch.arange(d.shape[1], device=d.device)[None, :]
    k = torch.where((s["top_k"] <= 0), d.shape[1], s["top_k"])[:, None]
    k = torch.where(greedy, 1, k)
    keep = (rank < k) & (d > -math.inf)
    w = torch.where(keep, w, 0.0)
    mass = torch.cumsum(w, 1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (mass - w < p * mass[:, -1:])
    keep &= w >= s["min_p"].double()[:, None]
    n = keep.sum(1, keepdim=True)
    total = mass.gather(1, n - 1)
    at = torch.minimum((mass <= s["uniforms"].double()[:, None] * total).sum(1, keepdim=True), n - 1)
    return {"tokens": ids.gather(1, at)[:, 0].int(), "kept": n[:, 0].int(), "logprobs": (d.gather(1, at) - torch.log(total))[:, 0].float()}


def _head_plain(s):
    x, ids = s["x"].float(), s["ids"].long()
    y = x @ s["weight"].float().T
    at, scale = ids.clamp(min=0), s["scales"]
    u = torch.einsum("nk,ark->nar", x, s["a"].float())  # every row with every adapter, and then only its own
    mine = (ids[:, None] == torch.arange(scale.numel(), device=x.device)[None, :]).float() * scale[None, :]
    u = (u * mine[:, :, None]).reshape(x.shape[0], -1)
    y += u @ s["b"].permute(0, 2, 1).reshape(u.shape[1], -1).float()
    return {"logits": y.to(s["out_dtype"])}


def run(state):
    if state["op"] == "sample":
        if not own:
            return _sample_plain(state)
        from neuraval_b200.sampler import sample_rows_min_p_device
        sample_rows_min_p_device(
            state["logits"], state["uniforms"], state["tokens"], temperature=state["temperature"], top_k=state["top_k"],
            top_p=state["top_p"], min_p=state["min_p"], logprobs=state["logprobs"], kept=state["kept"])
        return {"tokens": state["tokens"], "kept": state["kept"], "logprobs": state["logprobs"]}
    if not own:
        return _head_plain(state)
    state["head"].project_device(state["x"], state["ids"], state["out"])
    return {"logits": state["out"]}


def work(case):
    n, V = case["rows"], case["vocab"]
    if case["op"] == "sample":
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
        # one difference, one exponential, one sum and one comparison for each value
        return {"bytes": n * V * size + n * 32, "flops": 4 * n * V}
    K, R, used = case["inner"], case["rank"], min(case["adapters"], n)
    R = R if case["ranks"] == "same" else (R + 1) / 2
    out = 4 if case["out"] == "f32" else 2
    return {"bytes": 2 * (V * K + n * K + used * R * (K + V)) + out * n * V + 4 * n,
            "flops": 2 * n * V * K + (1 - case["bare"]) * 2 * n * R * (K + V)}


def exact(case, seed):
    """The definitions in 64 bits, row by row on the host for sampling."""
    if case["op"] == "head":
        if case["rows"] * case["inner"] * case["vocab"] > 3e11:
            return None
        s = prepare(case, seed)
        x, y = s["x"].double(), torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device="cuda")
        for c in range(0, case["vocab"], 16384):
            y[:, c:c + 16384] = x @ s["weight"][c:c + 16384].double().T
        for n, a in enumerate(s["ids"].tolist()):
            if a >= 0:
                y[n] += float(s["scales"][a]) * (s["b"][a].double() @ (s["a"][a].double() @ x[n]))
        return {"logits": y}
    if case["rows"] * case["vocab"] > 5e7:
        return None
    s = prepare(case, seed)
    T, k, p, m, u = _options(case, seed)
    tokens, kept, logprobs = [], [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double().cpu().numpy()
        fit = np.flatnonzero(x > -np.inf)
        best = x[fit].max()
        if T[r] == 0:
            tokens.append(int(fit[np.argmax(x[fit])]))
            kept.append(1)
            logprobs.append(0.0)
            continue
        by = np.lexsort((fit, -x[fit]))[: k[r] if k[r] > 0 else None]
        fit = fit[by]
        e = (x[fit] - best) / np.float64(T[r])
        w = np.exp(e)
        S = np.cumsum(w)
        many = len(w)
        if p[r] < 1:
            many = min(many, int(np.searchsorted(S, np.float64(p[r]) * S[-1], side="left")) + 1)
        if m[r] > 0:
            many = min(many, int((w >= np.float64(m[r])).sum()))
        j = min(int(np.searchsorted(S[:many], np.float64(u[r]) * S[many - 1], side="right")), many - 1)
        tokens.append(int(fit[j]))
        kept.append(many)
        logprobs.append(float(e[j] - np.log(S[many - 1])))
    dev = torch.device("cuda")
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=dev), "kept": torch.tensor(kept, dtype=torch.int32, device=dev),
            "logprobs": torch.tensor(logprobs, dtype=torch.float64, device=dev)}
