"""Cases and plain forms of the mixture-of-experts operators: routing, and quantised products grouped by expert.

``listed()`` and ``draw()`` give cases, ``prepare()`` makes a case's inputs on the GPU, ``run()`` makes one pass (the
framework's calls where ``own`` is true, elementary torch operations in 32 bits otherwise), ``exact()`` computes the
same outputs in 64 bits and ``work()`` counts the bytes and operations a pass cannot do without.

A case's ``op`` is one of

* ``route``     logits [T, E] -> the k largest of each row, their weights, and the rows sorted by expert;
* ``rows``      x [R, K], rows already grouped by expert -> x[r] . W[e(r)] for every row;
* ``gated``     x [T, K] and a plan -> silu(x W_gate) * (x W_up) for each of the T k (token, expert) pairs, by expert;
* ``combined``  h [T k, K] sorted by expert and a plan -> sum over a token's k experts of weight * (h W).

``fmt`` is the experts' weight format: ``w4`` (4-bit codes, groups of ``gs``, scale and zero per group), ``fp8`` (e4m3
bytes with a scale per 128 x 128 block; activations quantised per row and 128 values) or ``h16`` (16-bit weights).
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_FP32 = {"fp32": torch.float32, **_DT}


def _case(name, op, fmt="", dtype="bf16", T=1, E=8, k=2, K=0, N=0, gs=0, masked=False):
    return {"name": name, "op": op, "fmt": fmt, "dtype": dtype, "T": T, "E": E, "k": k, "K": K, "N": N, "gs": gs, "masked": masked}


def listed():
    return [
        # the router of one decode step of a single request
        _case("route_one_token", "route", dtype="bf16", T=1, E=64, k=6),
        # the router of a long prompt, with experts masked out for some tokens
        _case("route_prompt", "route", dtype="fp32", T=8191, E=128, k=8, masked=True),
        # few large experts: one request decodes, two experts' weights are streamed
        _case("w4_gated_one_token", "gated", "w4", "bf16", T=1, E=8, k=2, K=4096, N=28672, gs=128),
        # many small experts: a decode batch that touches nearly all of them with a few rows each
        _case("w4_gated_batch", "gated", "w4", "fp16", T=61, E=64, k=6, K=2048, N=2816, gs=64),
        # a prompt through few large experts
        _case("w4_gated_prompt", "gated", "w4", "bf16", T=2048, E=8, k=2, K=4096, N=28672, gs=128),
        # the way back of a decode batch
        _case("w4_combined_batch", "combined", "w4", "bf16", T=16, E=8, k=2, K=14336, N=4096, gs=128),
        # the way back of one request: short rows, the latency of two launches
        _case("fp8_combined_one_token", "combined", "fp8", "bf16", T=1, E=128, k=8, K=768, N=2048),
        # a mid-size batch on many small experts
        _case("fp8_gated_batch", "gated", "fp8", "bf16", T=257, E=128, k=8, K=2048, N=1536),
        # prompts, both ways
        _case("fp8_gated_prompt", "gated", "fp8", "bf16", T=4096, E=32, k=4, K=4096, N=4096),
        _case("fp8_combined_prompt", "combined", "fp8", "fp16", T=4001, E=64, k=8, K=1408, N=2048),
        # experts left unquantised, rows grouped by the caller (an exchange between ranks has sorted them)
        _case("h16_rows_small", "rows", "h16", "fp16", T=129, E=16, k=1, K=2048, N=1000),
        _case("h16_rows_prompt", "rows", "h16", "bf16", T=8200, E=16, k=1, K=4096, N=4096),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "rows", "gated", "gated", "combined", "combined"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "route":
        E = rng.choice([8, 16, 60, 64, 100, 128, 160, 256])
        return {"op": op, "fmt": "", "dtype": rng.choice(["bf16", "fp16", "fp32"]), "T": _spread(rng, 1, 8000), "E": E,
                "k": rng.randint(1, 8), "K": 0, "N": 0, "gs": 0, "masked": rng.random() < 0.5}
    fmt = rng.choice(["w4", "fp8", "h16"])
    E = rng.choice([4, 8, 16, 24, 32, 60, 64, 128])
    k = 1 if op == "rows" else rng.randint(1, min(8, E // 2))
    K = 128 * _spread(rng, 4, 56)
    N = 16 * _spread(rng, 32, 448)
    weights = {"w4": 400e6, "fp8": 300e6, "h16": 200e6}[fmt]      # values in all experts together
    while E * K * N > weights and N > 512:
        N = max(512, N // 32 * 16)
    while E * K * N > weights and K > 512:
        K = max(512, K // 256 * 128)
    T = _spread(rng, 1, 8000)
    while T * k * K * N > 2.5e11 and T > 1:                       # no more products than the largest listed case
        T //= 2
    return {"op": op, "fmt": fmt, "dtype": dtype, "T": T, "E": E, "k": k, "K": K, "N": N,
            "gs": rng.choice([32, 64, 128]) if fmt == "w4" else 0, "masked": op != "rows" and rng.random() < 0.3}


def _ids(g, T, E, k, masked):
    """Top-k expert ids of random logits with some experts more popular than others; -1: no expert (a masked slot)."""
    dev = "cuda"
    logits = torch.randn((T, E), generator=g, device=dev) + 0.7 * torch.randn((1, E), generator=g, device=dev)
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
    if masked:
        ids = torch.where(torch.rand((T, k), generator=g, device=dev) < 0.1, torch.full_like(ids, -1), ids)
    return ids


def _plan(ids, E):
    """Rows sorted by expert (slots without one at the end): offsets [E + 1], order [T k], places [T, k]."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, torch.full_like(flat, E), flat)
    order = torch.sort(key, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel(), device=order.device)
    counts = (key[:, None] == torch.arange(E, device=key.device)[None, :]).sum(0)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=key.device), torch.cumsum(counts, 0)])
    return offsets.to(torch.int32), order.to(torch.int32), places.view(ids.shape).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")      # noqa: E731
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")    # noqa: E731
    T, E, k, K, N = (case[n] for n in ("T", "E", "k", "K", "N"))
    if case["op"] == "route":
        logits = (2 * randn(T, E)).to(_FP32[case["dtype"]])
        if case["masked"]:
            logits = torch.where(rand(T, E) < 0.2, torch.full_like(logits, float("-inf")), logits)
        return {"case": case, "logits": logits}
    dt = _DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rows":
        share = rand(E) * (rand(E) > 0.15)                           # some experts get no rows
        expert = torch.sort(torch.multinomial(share + 1e-6, T, replacement=True, generator=g)).values
        s["offsets"] = torch.searchsorted(expert, torch.arange(E + 1, device="cuda")).to(torch.int32)
    else:
        s["ids"] = _ids(g, T, E, k, case["masked"])
        s["offsets"], s["order"], s["places"] = _plan(s["ids"], E)
        w = rand(T, k) + 0.1
        s["weights"] = w / w.sum(1, keepdim=True)
    s["x"] = randn(T * k if case["op"] == "combined" else T, K).to(dt)
    # most rows an expert has: what a program that lays rows out per expert keeps beside its plan
    s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    code = {"fp16": 1, "bf16": 2}[case["dtype"]]
    if case["fmt"] == "w4":
        gs = case["gs"]
        W = torch.randint(-2 ** 31, 2 ** 31, (E, K // 8, N), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        sc = (0.5 + rand(E, K // gs, N)) / (4.6 * math.sqrt(K))
        s["tensors"] = [W, sc.to(dt), (-sc * (6 + 3 * rand(E, K // gs, N))).to(dt)]
        s["meta"] = [0, 4, gs, 15, 8, code, code, 0, code, 0, 4, 1]
    elif case["fmt"] == "fp8":
        W = torch.empty((E, N, K), dtype=torch.float8_e4m3fn, device="cuda")
        W.copy_(randn(E, N, K) * 64)
        sc = (0.5 + rand(E, K // 128, (N + 127) // 128)) / (64 * math.sqrt(K))
        s["tensors"] = [W.transpose(1, 2), sc, none]
        s["meta"] = [1, 8, K, 255, 1, 3, code, 0, 0, 5, 0, 0]
    else:
        W = (randn(E, N, K) / math.sqrt(K)).to(dt)
        s["tensors"] = [W.transpose(1, 2), none, none]
        s["meta"] = [0, 16, 1, 65535, 1, code, code, 0, 6, 0, 0, 0]
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_route(logits, k):
    x = logits.float()
    E = x.shape[1]
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    none = best == float("-inf")
    e = torch.where(none, torch.zeros_like(best), torch.exp(best - best[:, :1]))
    total = e.sum(1, keepdim=True)
    weights = torch.where(none, torch.zeros_like(e), e / torch.where(total > 0, total, torch.ones_like(total)))
    ids = torch.where(none, torch.full_like(ids, -1), ids).to(torch.int32)
    offsets, order, places = _plan(ids, E)
    return weights, ids, offsets, order, places


def _plain_weights(case, tensors, pick=None):
    """The experts' weights [E or picked, K, N] in 32 bits (fp8: without the block scales, which come with them)."""
    W, sc, z = (t if pick is None or t.numel() == 0 else t[pick] for t in tensors)
    if case["fmt"] == "w4":
        shift = torch.arange(0, 32, 4, device=W.device, dtype=torch.int32)
        q = (W[:, :, None, :] >> shift[None, None, :, None]) & 15
        q = q.view(W.shape[0], sc.shape[1], -1, W.shape[2]).float()
        return (q * sc.float()[:, :, None, :] + z.float()[:, :, None, :]).view(W.shape[0], -1, W.shape[2])
    w = W.float()
    if case["fmt"] == "fp8":
        s = sc.repeat_interleave(128, dim=1).repeat_interleave(128, dim=2)[:, : w.shape[1], : w.shape[2]]
        w = w * s
    return w


def _plain_rows(case, s, x):
    """Product of each row of ``x`` (sorted by expert) with its expert's weights, in 32 bits."""
    R, E = x.shape[0], case["E"]
    x = x.float()
    if case["fmt"] == "fp8":
        b = x.view(R, -1, 128)
        sx = (b.abs().amax(2, keepdim=True) / 448.0).clamp_min(1e-6)
        x = ((b * (1.0 / sx)).clamp(-448, 448).to(torch.float8_e4m3fn).float() * sx).view(R, -1)
    off = s["offsets"].long()
    row = torch.arange(R, device=x.device)
    expert = torch.searchsorted(off, row, right=True) - 1            # E: no expert
    here = (expert < E)[:, None]
    expert = expert.clamp(max=E - 1)
    if R <= E:
        y = torch.bmm(x[:, None, :], _plain_weights(case, s["tensors"], expert))[:, 0]
    else:
        place = row - off[expert]
        place = torch.where(here[:, 0], place, torch.full_like(place, s["most"]))
        laid = torch.zeros((E, s["most"] + 1, x.shape[1]), device=x.device)
        laid[expert, place] = x
        y = torch.bmm(laid, _plain_weights(case, s["tensors"]))[expert, place]
    return torch.where(here, y, torch.zeros_like(y))


def _plain(s):
    case = s["case"]
    if case["op"] == "route":
        return _plain_route(s["logits"], case["k"])
    dt = s["x"].dtype
    if case["op"] == "rows":
        return _plain_rows(case, s, s["x"]).to(dt)
    if case["op"] == "gated":
        y = _plain_rows(case, s, s["x"][(s["order"] // case["k"]).long()])
        gate, up = y[:, : case["N"] // 2], y[:, case["N"] // 2:]
        return (gate / (1 + torch.exp(-gate)) * up).to(dt)
    y = _plain_rows(case, s, s["x"])[s["places"].reshape(-1).long()].view(case["T"], case["k"], case["N"])
    return (y * s["weights"][:, :, None]).sum(1).to(dt)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _calls(s):
    import gemlite_amd

    case = s["case"]
    if case["op"] == "route":
        return tuple(gemlite_amd.route_experts(s["logits"], case["k"]))
    if case["op"] == "rows":
        return gemlite_amd.experts_functional(s["x"], None, s["tensors"], s["meta"], s["offsets"])
    plan = gemlite_amd.ExpertPlan(s["weights"], s["ids"], s["offsets"], s["order"], s["places"])
    if case["op"] == "gated":
        return gemlite_amd.experts_gated_functional(s["x"], None, s["tensors"], s["meta"], plan)
    return gemlite_amd.experts_combined_functional(s["x"], None, s["tensors"], s["meta"], plan)


def run(state):
    return _calls(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without; 64-bit results
# ---------------------------------------------------------------------------
def work(case):
    T, E, k, K, N = (case[n] for n in ("T", "E", "k", "K", "N"))
    R = T * k
    if case["op"] == "route":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * E * size + R * 16 + (E + 1) * 4, "flops": T * E * (k + 4)}
    rows = 0.9 * R if case["masked"] else R
    active = E * (1 - (1 - 1 / E) ** rows)                           # experts that have a row, for even routing
    per = {"w4": 0.5 + (4 / case["gs"] if case["gs"] else 0), "fp8": 1 + 4 / 16384, "h16": 2}[case["fmt"]]
    size = {"rows": R * (K + N), "gated": T * K + R * N // 2, "combined": R * K + T * N}[case["op"]]
    return {"bytes": int(active * K * N * per + 2 * size + 12 * R), "flops": int(2 * rows * K * N)}


def exact(case, seed):
    s = prepare(case, seed)
    E, k = case["E"], case["k"]
    if case["op"] == "route":
        x = s["logits"].double()
        ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
        top = torch.gather(x, 1, ids)
        off = torch.isinf(top)
        p = torch.softmax(top, 1)
        p = torch.where(off, torch.zeros_like(p), p)
        ids = ids.masked_fill(off, -1)
        lists = [torch.nonzero(ids.reshape(-1) == e).reshape(-1) for e in list(range(E)) + [-1]]
        order = torch.cat(lists)
        offsets = torch.tensor([0] + [int(v.numel()) for v in lists[:E]], device=x.device).cumsum(0)
        places = torch.argsort(order).view(ids.shape)
        return p, ids.to(torch.int32), offsets.to(torch.int32), order.to(torch.int32), places.to(torch.int32)
    x = s["x"].double()
    if case["fmt"] == "fp8":
        # which code a value gets is defined by 32-bit steps (scale = max(amax / 448, 1e-6), code = e4m3(x * (1 / scale))):
        # 16-bit values over their block's maximum meet the borders between codes exactly, so 64 bits would choose others
        b = s["x"].float().reshape(x.shape[0], -1, 128)
        sx = torch.clamp(b.abs().max(dim=2, keepdim=True).values / 448, min=1e-6)
        code = (b * sx.reciprocal()).clamp(min=-448, max=448).to(torch.float8_e4m3fn)
        x = (code.double() * sx.double()).reshape(x.shape)
    W, sc, z = s["tensors"]
    R = case["T"] * k
    source = torch.arange(R, device=x.device)
    if case["op"] == "gated":
        source = s["order"].long() // k
    ends = s["offsets"].tolist()
    cols = case["N"] // 2 if case["op"] == "gated" else case["N"]
    out = torch.zeros((R, cols), dtype=torch.float64, device=x.device)
    for e in range(E):
        lo, hi = ends[e], ends[e + 1]
        if hi == lo:
            continue
        if case["fmt"] == "w4":
            w = torch.stack([(W[e] >> (4 * i)) & 15 for i in range(8)], 1).reshape(-1, case["N"]).double()
            group = torch.arange(w.shape[0], device=x.device) // case["gs"]
            w = w * sc[e].double()[group] + z[e].double()[group]
        else:
            w = W[e].double()
            if case["fmt"] == "fp8":
                i = torch.arange(w.shape[0], device=x.device) // 128
                j = torch.arange(w.shape[1], device=x.device) // 128
                w = w * sc[e].double()[i][:, j]
        y = x[source[lo:hi]] @ w
        if case["op"] == "gated":
            y = torch.nn.functional.silu(y[:, :cols]) * y[:, cols:]
        out[lo:hi] = y
    if case["op"] != "combined":
        return out
    return torch.stack([out[s["places"][:, j].long()] * s["weights"][:, j:j + 1].double() for j in range(k)]).sum(0)
