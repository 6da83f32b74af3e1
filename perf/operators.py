"""The steps of a decoder layer around the MoE block, for timing and comparing: the
residual addition with its RMS norm (in the activations' type or in 8 bits), and the
projections that read the normalised rows, with the low-rank adapters of many requests.

A case's ``op`` is

- norm: ``add_rms_norm``: h = x + residual and its norm;
- norm_q8: ``add_rms_norm_q8``: the norm in int8 with one scale per row;
- linear: a projection of bf16 rows (``rows`` = bf16) or 8-bit rows (q8) by weights in bf16,
  int8 with one scale per output channel (w8c) or int8 with one scale (w8t);
- lora: the same beside adapters: ``L`` adapters of rank ``R`` are loaded; the ``T`` tokens are
  those of ``requests`` requests side by side, of which some use none (a decode batch has one
  token per request);
- layer: the norm followed by the projection with adapters, on bf16 or 8-bit rows.

With ``own`` the operators are the framework's; without it they are elementary torch
operations in 32 bits, rounded once where an array of fewer bits is the result.

Widths are those of this repository's presets: the hidden sizes 1024, 2048, 2560 and 4096,
the query, key and value heads side by side (4096, 5120, 6144, 9216) and the attention's
output (4096 -> 2048); drawn cases have others too.
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
MOST_NORM = 16384 * 4096  # elements of the largest norm
MOST_FLOPS = 2 * 2048 * 4096 * 9216  # of the largest projection


def _norm(op, T, D, act="bf16"):
    return {"op": op, "T": T, "D": D, "act": act}


def _linear(T, D, N, weights="w8c", rows="bf16"):
    return {"op": "linear", "T": T, "D": D, "N": N, "weights": weights, "rows": rows}


def _lora(op, T, D, N, L, R, requests, weights="w8c", rows="bf16"):
    return {"op": op, "T": T, "D": D, "N": N, "L": L, "R": R, "requests": requests, "weights": weights, "rows": rows}


def listed():
    cases = {
        # one sequence being generated: the residual stream of one token
        "norm_1": _norm("norm", 1, 2048),
        # a batch of long prompts of the large model
        "norm_16384": _norm("norm", 16384, 4096),
        # a parity run in 32 bits, of odd length
        "norm_777_f32": _norm("norm", 777, 2560, "f32"),
        # a decode batch whose projections run in 8 bits
        "norm_q8_33": _norm("norm_q8", 33, 2048),
        # a prefill chunk whose projections run in 8 bits
        "norm_q8_8192": _norm("norm_q8", 8192, 4096),
        # one sequence being generated: query, key and value heads
        "linear_1": _linear(1, 2048, 5120),
        # a prefill chunk of the large model in 8 bits
        "linear_2048_q8": _linear(2048, 4096, 9216, rows="q8"),
        # a full decode batch, every request with its own choice of 32 adapters
        "lora_64": _lora("lora", 64, 2048, 5120, 32, 16, 64),
        # a short prompt batch of odd length on the reference's per-tensor weights
        "lora_333": _lora("lora", 333, 2560, 6144, 4, 8, 3, "w8t"),
        # a long prefill chunk of the unquantised checkpoint
        "lora_4096_bf16": _lora("lora", 4096, 2048, 5120, 8, 16, 6, "bf16"),
        # a decode step of the large model in 8 bits, from the residual to the heads
        "layer_24_q8": _lora("layer", 24, 4096, 9216, 16, 64, 24, rows="q8"),
        # a prefill chunk from the residual to the heads
        "layer_1500": _lora("layer", 1500, 2048, 5120, 8, 32, 5),
    }
    return [{"name": n, **c} for n, c in cases.items()]


def _spread(rng, top):
    """1 .. top, even over the logarithm."""
    return min(top, int(round(math.exp(rng.uniform(0.0, math.log(top))))))


def draw(rng):
    op = rng.choice(("norm", "norm_q8", "linear", "linear", "lora", "lora", "lora", "layer"))
    if op in ("norm", "norm_q8"):
        D = rng.choice((1024, 2048, 2560, 4096, rng.randint(16, 4096)))
        return _norm(op, _spread(rng, min(65536, MOST_NORM // D)), D, rng.choice(("bf16", "bf16", "f32")))
    D = rng.choice((1024, 2048, 2048, 2560, 4096, rng.randint(64, 4096)))
    N = rng.choice((512, 2048, 4096, 5120, 6144, 9216, rng.randint(64, 6144)))
    T = _spread(rng, min(4096, MOST_FLOPS // (2 * D * N)))
    rows = rng.choice(("bf16", "bf16", "q8"))
    weights = rng.choice(("w8c", "w8c", "w8t")) if rows == "q8" else rng.choice(("w8c", "w8c", "w8t", "bf16", "bf16"))
    if op == "linear":
        return _linear(T, D, N, weights, rows)
    requests = T if T <= 64 and rng.random() < 0.7 else min(T, rng.randint(1, 12))
    return _lora(op, T, D, N, rng.randint(1, 32), rng.choice((4, 8, 16, 16, 24, 32, 64)), requests, weights, rows)


# --- inputs ------------------------------------------------------------------


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _stream(g, T, D, dtype):
    """Rows of a residual stream: a few channels are much larger than the others."""
    gain = torch.ones(D, device=DEV)
    gain[torch.randperm(D, generator=g, device=DEV)[: max(1, D // 256)]] = 12.0
    return (torch.randn(T, D, generator=g, device=DEV) * gain).to(dtype)


def _weights(case, g):
    """[D, N] in bf16, or int8 values and their scale as the quantisers give them."""
    w = _randn(g, case["D"], case["N"], std=0.02)
    if case["weights"] == "bf16":
        return w, None
    wf = w.float()
    s = (wf.abs().amax(dim=0, keepdim=True) if case["weights"] == "w8c" else wf.abs().amax()) / 127.0
    q = torch.clamp(torch.round(wf / s), -128, 127).to(torch.int8)
    return q, s if case["weights"] == "w8c" else s.to(torch.bfloat16)


def _adapters(case, g):
    """A [L, D, R], B [L, R, N], the adapters' factors [L] and each token's adapter [T] (-1: none)."""
    T, L, R = case["T"], case["L"], case["R"]
    a = _randn(g, L, case["D"], R, std=case["D"] ** -0.5)
    b = _randn(g, L, R, case["N"], std=0.02)
    factor = torch.rand(L, generator=g, device=DEV) * 1.5 + 0.5
    # about one request in eight uses no adapter
    n = case["requests"]
    of = torch.randint(0, L, (n,), generator=g, device=DEV)
    of = torch.where(torch.rand(n, generator=g, device=DEV) < 0.125, torch.full_like(of, -1), of)
    # lengths of the requests: the cuts between them at random places
    cuts = torch.randperm(T - 1, generator=g, device=DEV)[: n - 1] + 1 if T > 1 else of.new_empty(0)
    request = torch.zeros(T, dtype=torch.int64, device=DEV)
    request[cuts] = 1
    return a, b, factor, of[torch.cumsum(request, 0)].to(torch.int32)


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    T, D = case["T"], case["D"]
    got = {}
    if case["op"] in ("norm", "norm_q8", "layer"):
        dtype = torch.float32 if case.get("act") == "f32" else torch.bfloat16
        got["x"] = _randn(g, T, D, std=0.5, dtype=dtype)
        got["residual"] = _stream(g, T, D, dtype)
        got["norm"] = (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    elif case["rows"] == "q8":
        # rows as the 8-bit norm gives them: the largest value of a row at 127
        v = _stream(g, T, D, torch.float32)
        got["x_scale"] = v.abs().amax(dim=1, keepdim=True) / 127.0
        got["x"] = torch.clamp(torch.round(v / got["x_scale"]), -127, 127).to(torch.int8)
    else:
        got["x"] = _randn(g, T, D)
    if case["op"] in ("linear", "lora", "layer"):
        got["w"], got["w_scale"] = _weights(case, g)
    if case["op"] in ("lora", "layer"):
        got["a"], got["b"], got["factor"], got["adapter"] = _adapters(case, g)
    return got


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"], s["rows"] = case["op"], case.get("rows")
    if own and "w" in s:
        # what a program has done when its weights and adapters were loaded, and once for
        # the step whose projections all follow
        from kappa_amd.qwen3 import Q8Weight, lora_batch, prepack_linear, prepack_lora

        s["packed"] = prepack_linear(s["w"] if s["w_scale"] is None else Q8Weight(s["w"], s["w_scale"]))
        if "a" in s:
            s["lora"] = prepack_lora(s["a"], s["b"], s["factor"])
            s["batch"] = lora_batch(s["adapter"], case["L"])
    return s


# --- the plain forms ----------------------------------------------------------


def _plain_norm(s):
    x = s["x"]
    h = (x.float() + s["residual"].float()).to(x.dtype)
    hf = h.float()
    r = torch.rsqrt(hf.square().mean(dim=-1, keepdim=True) + EPS)
    return hf * r * s["norm"].float(), h


def _plain_q8(v):
    scale = v.abs().amax(dim=-1, keepdim=True) / 127.0
    return torch.clamp(torch.round(v / scale), -127.0, 127.0), scale


def _plain_linear(s, x):
    w = s["w"].float() if s["w_scale"] is None else s["w"].float() * s["w_scale"].float()
    y = x @ w
    if "a" in s:
        L, D, R = s["a"].shape
        # every adapter's inner values, then those of each token's own
        u = (x @ s["a"].float().permute(1, 0, 2).reshape(D, L * R)).reshape(-1, L, R)
        mine = s["adapter"].unsqueeze(1) == torch.arange(L, device=x.device)
        u = torch.where(mine.unsqueeze(2), u * s["factor"].reshape(L, 1), u.new_zeros(()))
        y = y + u.reshape(-1, L * R) @ s["b"].float().reshape(L * R, -1)
    return y.to(torch.bfloat16)


def _plain(s):
    op = s["op"]
    if op == "norm":
        v, h = _plain_norm(s)
        return {"normed": v.to(h.dtype), "h": h}
    if op == "norm_q8":
        v, h = _plain_norm(s)
        q, scale = _plain_q8(v)
        return {"values": (q * scale).to(torch.bfloat16), "scale": scale, "h": h}
    if op == "layer":
        v, h = _plain_norm(s)
        if s["rows"] == "q8":
            q, scale = _plain_q8(v)
            return {"y": _plain_linear(s, q * scale), "h": h}
        return {"y": _plain_linear(s, v.to(h.dtype).float()), "h": h}
    x = s["x"].float()
    return {"y": _plain_linear(s, x * s["x_scale"] if s["rows"] == "q8" else x)}


def run(state):
    s = state
    if not own:
        return _plain(s)
    from kappa_amd.qwen3 import Q8Rows, add_rms_norm, add_rms_norm_q8, linear

    op = s["op"]
    if op == "norm":
        normed, h = add_rms_norm(s["x"], s["residual"], s["norm"], epsilon=EPS)
        return {"normed": normed, "h": h}
    if op == "norm_q8":
        q, h = add_rms_norm_q8(s["x"], s["residual"], s["norm"], epsilon=EPS)
        # the values that the 8 bits stand for
        values = torch.empty(q.values.shape, dtype=torch.bfloat16, device=h.device)
        return {"values": torch.mul(q.values, q.scale, out=values), "scale": q.scale, "h": h}
    if op == "layer":
        norm = add_rms_norm_q8 if s["rows"] == "q8" else add_rms_norm
        n, h = norm(s["x"], s["residual"], s["norm"], epsilon=EPS)
        return {"y": linear(n, s["packed"], lora=s["lora"], batch=s["batch"]), "h": h}
    x = Q8Rows(s["x"], s["x_scale"]) if s["rows"] == "q8" else s["x"]
    return {"y": linear(x, s["packed"], lora=s.get("lora"), batch=s.get("batch"))}


def work(case):
    T, D = case["T"], case["D"]
    act = 4 if case.get("act") == "f32" else 2
    n_bytes = flops = 0
    if case["op"] in ("norm", "norm_q8", "layer"):
        # both inputs and the sum; the normalised rows too where they are the result
        n_bytes += 3 * act * T * D + act * D
        n_bytes += {"norm": act * T * D, "norm_q8": T * D + 4 * T, "layer": 0}[case["op"]]
        flops += 6 * T * D
    if case["op"] in ("linear", "lora", "layer"):
        N = case["N"]
        if case["op"] != "layer":
            n_bytes += T * D + 4 * T if case["rows"] == "q8" else 2 * T * D
        n_bytes += {"bf16": 2 * D * N, "w8c": D * N + 4 * N, "w8t": D * N}[case["weights"]] + 2 * T * N
        flops += 2 * T * D * N
    if case["op"] in ("lora", "layer"):
        L, R = case["L"], case["R"]
        used = L * (1.0 - (1.0 - 0.875 / L) ** case["requests"])  # adapters that the requests choose
        n_bytes += 2 * used * R * (D + case["N"]) + 4 * T
        flops += 0.875 * 2 * T * R * (D + case["N"])
    return {"bytes": n_bytes, "flops": flops}


# --- the same in 64 bits -------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    out = {}
    x = s["x"].double()
    if "residual" in s:
        # the stream is an array of the activations' type
        h = (x + s["residual"].double()).to(s["x"].dtype)
        out["h"] = h.double()
        x = h.double()
        x = x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / case["D"] + EPS) * s["norm"].double()
        if case["op"] == "norm":
            return {"normed": x, **out}
        if case["op"] == "norm_q8" or case["rows"] == "q8":
            scale = x.abs().max(dim=1, keepdim=True).values / 127.0
            x = torch.round(x / scale) * scale
            if case["op"] == "norm_q8":
                return {"values": x, "scale": scale, **out}
        else:
            x = x.to(h.dtype).double()
    elif case["rows"] == "q8":
        x = x * s["x_scale"].double()
    w = s["w"].double()
    if s["w_scale"] is not None:
        w = w * s["w_scale"].double()
    y = x @ w
    if "a" in s:
        for i in range(case["L"]):
            rows = torch.nonzero(s["adapter"] == i).squeeze(1)
            if len(rows):
                y[rows] += (x[rows] @ s["a"][i].double()) @ s["b"][i].double() * s["factor"][i].double()
    out["y"] = y
    return out
