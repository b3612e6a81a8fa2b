"""The 8-bit-integer linear and mixture-of-experts operators as measured cases.

Five operators, as one quantised mixture-of-experts layer uses them:

* ``gemm``     y = (a_s8 . w_s8^T) * a_scale[token] * w_scale[channel] + bias
* ``grouped``  the same product for each expert on its rows of a token batch sorted by expert
* ``quant``    per-token s8 quantisation with the expert's activation in the same pass
* ``route``    scores, top-k experts, weights, and the batch sorted by expert
* ``combine``  the weighted sum of each token's expert outputs

``run`` computes the plain form in elementary torch operations, or, when ``own`` is true, makes
the framework's calls.
"""
import math

import numpy as np
import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one token through a gate|up-sized layer: weights streamed once, the latency of a decode step
        dict(name="gemm_decode", op="gemm", M=1, K=5120, N=17408, out="bf16", bias=False),
        # a chunk of a prompt through the down projection: long K, few output tiles
        dict(name="gemm_chunk", op="gemm", M=200, K=17408, N=5120, out="f16", bias=True),
        # a full prompt batch through the gate|up-sized layer: bound by the tensor cores
        dict(name="gemm_prefill", op="gemm", M=8192, K=5120, N=17408, out="bf16", bias=False),
        # four decoding sequences: a row or two for each active expert, token rows gathered
        dict(name="grouped_decode", op="grouped", T=4, k=6, E=64, K=2688, N=3712, out="bf16", gather=True, bias=False),
        # a mixed serving batch through the experts' down projection, ragged counts, some experts empty
        dict(name="grouped_mixed", op="grouped", T=192, k=8, E=128, K=1856, N=2688, out="f16", gather=False, bias=True),
        # a prompt batch through the experts' gate|up projection, token rows gathered
        dict(name="grouped_prefill", op="grouped", T=4096, k=6, E=64, K=2688, N=3712, out="bf16", gather=True, bias=False),
        # the SwiGLU of a decode batch on its way into the down projection
        dict(name="quant_decode", op="quant", M=16, K=17408, act="silu_mul", dtype="bf16"),
        # the SwiGLU of every routed row of a prompt batch
        dict(name="quant_prefill", op="quant", M=24576, K=1856, act="silu_mul", dtype="bf16"),
        # the router of a decode step: softmax scores
        dict(name="route_decode", op="route", T=8, E=64, k=6, score="softmax", bias=False, n_group=1, topk_group=1,
             group_score="max", renorm=True, dtype="bf16", padded=False),
        # the router of a prompt batch: sigmoid scores with a balance bias, experts limited to half of the groups
        dict(name="route_prefill", op="route", T=8192, E=256, k=8, score="sigmoid", bias=True, n_group=8, topk_group=4,
             group_score="top2", renorm=True, dtype="f32", padded=True),
        # the end of a decode step's layer
        dict(name="combine_decode", op="combine", T=8, k=6, H=2688, dtype="bf16", add=True),
        # the end of a prompt batch's layer
        dict(name="combine_prefill", op="combine", T=8192, k=8, H=4096, dtype="bf16", add=False),
    ]


def _logint(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "grouped", "grouped", "quant", "route", "combine"])
    if op == "gemm":
        # decode, chunk and prefill batches; K a multiple of 16, any N
        M, K, N = _logint(rng, 1, 8192), _logint(rng, 256, 17408, 16), _logint(rng, 64, 17408)
        while M * K * N > 8192 * 5120 * 17408:
            M = max(1, M // 2)
        return dict(op=op, M=M, K=K, N=N, out=rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.5)
    if op == "grouped":
        E = _logint(rng, 8, 256)
        k = rng.randint(1, min(8, E))
        T, K, N = _logint(rng, 1, 4096), _logint(rng, 256, 2688, 16), _logint(rng, 128, 3712)
        return dict(op=op, T=T, k=k, E=E, K=K, N=N, out=rng.choice(["bf16", "f16", "f32"]),
                    gather=rng.random() < 0.5, bias=rng.random() < 0.3)
    if op == "quant":
        K = _logint(rng, 256, 17408, 16)
        M = _logint(rng, 1, max(1, 24576 * 1856 // K))
        return dict(op=op, M=M, K=K, act=rng.choice(["none", "silu_mul", "relu2"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "route":
        grouped = rng.random() < 0.5
        n_group = rng.choice([2, 4, 8]) if grouped else 1
        E = n_group * _logint(rng, 8, 384 // n_group)
        topk_group = rng.randint(1, n_group)
        k = rng.randint(1, min(8, topk_group * (E // n_group)))
        return dict(op=op, T=_logint(rng, 1, 8192), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, n_group=n_group, topk_group=topk_group,
                    group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7,
                    dtype=rng.choice(["bf16", "f16", "f32"]), padded=rng.random() < 0.3)
    k = rng.randint(1, 8)
    return dict(op=op, T=_logint(rng, 1, 8192), k=k, H=_logint(rng, 128, 4096, 8),
                dtype=rng.choice(["bf16", "f16", "f32"]), add=rng.random() < 0.5)


# ------------------------------------------------------------------------------------- inputs
def _tokens_s8(rows, K, g):
    """Token rows as a per-token quantiser leaves them: bell-shaped codes up to +-127, scales of a few
    hundredths (hidden states with a spread of sizes from token to token)."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    amax = x.abs().amax(1, keepdim=True)
    q = torch.round(x * (127.0 / amax)).to(torch.int8)
    size = torch.exp(0.3 * torch.randn(rows, generator=g, device="cuda"))
    return q, (amax[:, 0] / 127.0 * size).contiguous()


def _weights_s8(shape, g):
    """Weights [..., N, K] quantised with a scale for each output channel, stored as int8."""
    w = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = w.view(-1, shape[-1])
    step = max(1, (1 << 27) // shape[-1])
    for i in range(0, flat.shape[0], step):
        part = torch.randn(min(step, flat.shape[0] - i), shape[-1], generator=g, device="cuda")
        flat[i:i + step] = torch.round(part * 28.0).clamp_(-127, 127).to(torch.int8)
    scale = (0.7 + 0.6 * torch.rand(shape[:-1], generator=g, device="cuda")) / (28.0 * math.sqrt(shape[-1]))
    return w, scale


def _routing(T, k, E, g):
    """Distinct experts for each token, some experts preferred: offsets [E+1], token of each sorted row."""
    pull = 0.7 * torch.randn(E, generator=g, device="cuda")
    gumbel = -torch.log(-torch.log(torch.rand(T, E, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)))
    ids = torch.topk(gumbel + pull, k, dim=1).indices.reshape(-1)
    order = torch.sort(ids, stable=True).indices
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(torch.bincount(ids, minlength=E), 0).to(torch.int32)
    return offsets, (order // k).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    s = dict(case)
    if case["op"] == "gemm":
        s["a"], s["a_scale"] = _tokens_s8(case["M"], case["K"], g)
        s["w"], s["w_scale"] = _weights_s8((case["N"], case["K"]), g)
        s["b"] = torch.randn(case["N"], generator=g, device="cuda") if case["bias"] else None
    elif case["op"] == "grouped":
        T, k, E = case["T"], case["k"], case["E"]
        s["offsets"], s["rows"] = _routing(T, k, E, g)
        s["a"], s["a_scale"] = _tokens_s8(T if case["gather"] else T * k, case["K"], g)
        s["w"], s["w_scale"] = _weights_s8((E, case["N"], case["K"]), g)
        s["b"] = torch.randn(E, case["N"], generator=g, device="cuda") if case["bias"] else None
    elif case["op"] == "quant":
        cols = case["K"] * (2 if case["act"] == "silu_mul" else 1)
        s["x"] = (1.5 * torch.randn(case["M"], cols, generator=g, device="cuda")).to(DT[case["dtype"]])
    elif case["op"] == "route":
        T, E = case["T"], case["E"]
        x = 1.3 * torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")
        if case["padded"]:  # rows of a padded batch route nowhere; one expert is switched off
            x[T - T // 8:] = -math.inf
            x[:, E // 2] = -math.inf
        s["logits"] = x.to(DT[case["dtype"]])
        s["b"] = 0.1 * torch.randn(E, generator=g, device="cuda") if case["bias"] else None
    else:
        T, k, H = case["T"], case["k"], case["H"]
        s["y"] = torch.randn(T * k, H, generator=g, device="cuda").to(DT[case["dtype"]])
        s["slots"] = torch.randperm(T * k, generator=g, device="cuda").view(T, k).to(torch.int32)
        w = torch.rand(T, k, generator=g, device="cuda")
        s["weights"] = w / w.sum(1, keepdim=True)
        s["add"] = torch.randn(T, H, generator=g, device="cuda").to(DT[case["dtype"]]) if case["add"] else None
    return s


# ------------------------------------------------------------------------------------- plain forms
def _gemm(s):
    acc = s["a"].float() @ s["w"].float().t()
    y = acc * s["a_scale"][:, None] * s["w_scale"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DT[s["out"]])


def _grouped(s):
    """Every expert's rows padded to the longest expert's, one batched product."""
    E, off = s["E"], s["offsets"].long()
    R = s["T"] * s["k"]
    rows = torch.arange(R, device="cuda")
    expert = torch.searchsorted(off[1:].contiguous(), rows, right=True)
    at = rows - off[expert]
    src = s["rows"].long() if s["gather"] else rows
    cap = int((off[1:] - off[:-1]).max())
    a = torch.zeros(E, cap, s["K"], device="cuda")
    a[expert, at] = s["a"][src].float()
    acc = torch.bmm(a, s["w"].float().transpose(1, 2))[expert, at]
    y = acc * s["a_scale"][src][:, None] * s["w_scale"][expert]
    if s["b"] is not None:
        y = y + s["b"][expert]
    return y.to(DT[s["out"]])


def _quant(s):
    x, K = s["x"].float(), s["K"]
    if s["act"] == "silu_mul":
        gate, up = x[:, :K], x[:, K:]
        y = gate / (1 + torch.exp(-gate)) * up
    elif s["act"] == "relu2":
        y = x.clamp(min=0).square()
    else:
        y = x
    amax = y.abs().amax(1)
    scale = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    q = torch.round(y / scale[:, None]).clamp(-127, 127)
    return {"values": (q * scale[:, None]).to(torch.bfloat16), "scale": scale}


def _route(s):
    """In 64 bits: the k-th and the next score can lie closer than 32 bits tell apart."""
    T, E, k = s["T"], s["E"], s["k"]
    low = -math.inf
    x = s["logits"].double()
    if s["score"] == "softmax":
        top = x.amax(1, keepdim=True)
        e = torch.exp(x - torch.where(top == low, 0.0, top))
        score = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        score = 1 / (1 + torch.exp(-x))
    off = x == low
    key = score + s["b"].double() if s["b"] is not None else x
    key = torch.where(off, low, key)
    G = s["n_group"]
    if G > 1:
        inside = (score if s["group_score"] == "top2" and s["b"] is None else key).masked_fill(off, low)
        best = torch.sort(inside.view(T, G, E // G), dim=2, descending=True).values
        group = best[:, :, 0]
        if s["group_score"] == "top2":
            group = group + torch.where(best[:, :, 1] == low, 0.0, best[:, :, 1])
        order = torch.sort(group, dim=1, descending=True, stable=True).indices
        taken = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, order[:, :s["topk_group"]], True)
        key = torch.where(taken[:, :, None].expand(T, G, E // G).reshape(T, E), key, low)
    key, ids = torch.sort(key, dim=1, descending=True, stable=True)
    key, ids = key[:, :k], ids[:, :k]
    none = key == low
    w = torch.where(none, 0.0, score.gather(1, ids))
    if s["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    ids = torch.where(none, -1, ids)
    flat = torch.where(none, E, ids).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=E + 1)[:E]
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)])
    slots = torch.empty_like(order).scatter_(0, order, torch.arange(T * k, device="cuda"))
    slots = torch.where(none.reshape(-1), -1, slots).view(T, k)
    rows = torch.where(flat[order] == E, -1, order // k)
    i32 = torch.int32
    return {"ids": ids.to(i32), "weights": w.float(), "offsets": offsets.to(i32), "rows": rows.to(i32),
            "slots": slots.to(i32)}


def _combine(s):
    y = s["y"].float()[s["slots"].long()]
    out = (y * s["weights"][:, :, None]).sum(1)
    if s["add"] is not None:
        out = out + s["add"].float()
    return out.to(DT[s["dtype"]])


# ------------------------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return {"gemm": _gemm, "grouped": _grouped, "quant": _quant, "route": _route, "combine": _combine}[s["op"]](s)
    from xe2x2_b200 import ops
    if s["op"] == "gemm":
        return ops.s8_gemm(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["b"], out_dtype=DT[s["out"]])
    if s["op"] == "grouped":
        return ops.s8_gemm_grouped(s["a"], s["a_scale"], s["w"], s["w_scale"], s["offsets"],
                                   rows=s["rows"] if s["gather"] else None, bias=s["b"], out_dtype=DT[s["out"]])
    if s["op"] == "quant":
        q, scale = ops.quant_s8(s["x"], act=s["act"])
        values = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        return {"values": torch.mul(q, scale[:, None], out=values), "scale": scale}
    if s["op"] == "route":
        r = ops.moe_route(s["logits"], s["k"], bias=s["b"], score=s["score"], renormalize=s["renorm"],
                          n_group=s["n_group"], topk_group=s["topk_group"], group_score=s["group_score"])
        return {"ids": r.ids, "weights": r.weights, "offsets": r.offsets, "rows": r.rows, "slots": r.slots}
    return ops.moe_combine(s["y"], s["slots"], s["weights"], add=s["add"])


def work(case):
    if case["op"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        by = M * K + N * K + 4 * (M + N) + (4 * N if case["bias"] else 0) + M * N * ES[case["out"]]
        return {"bytes": by, "flops": 2 * M * N * K}
    if case["op"] == "grouped":
        T, k, E, K, N = (case[v] for v in ("T", "k", "E", "K", "N"))
        active = E * (1 - (1 - k / E) ** T)  # experts that some token takes, were all alike
        by = active * N * (K + 4 + (4 if case["bias"] else 0)) + (T if case["gather"] else T * k) * (K + 4)
        return {"bytes": by + T * k * N * ES[case["out"]] + 4 * (E + 1) + (4 * T * k if case["gather"] else 0),
                "flops": 2 * T * k * N * K}
    if case["op"] == "quant":
        M, K = case["M"], case["K"]
        n = 2 if case["act"] == "silu_mul" else 1
        return {"bytes": M * K * (n * ES[case["dtype"]] + 1) + 4 * M, "flops": 6 * M * K}
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": T * E * ES[case["dtype"]] + 16 * T * k + 4 * (E + 1), "flops": 8 * T * E}
    T, k, H, es = case["T"], case["k"], case["H"], ES[case["dtype"]]
    return {"bytes": T * H * es * (k + 1 + (1 if case["add"] else 0)) + 8 * T * k, "flops": 2 * T * k * H}


# ------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        y = torch.matmul(s["a"].double(), s["w"].double().T)
        y.mul_(s["a_scale"].double().unsqueeze(1)).mul_(s["w_scale"].double())
        return y if s["b"] is None else y.add_(s["b"].double())
    if case["op"] == "grouped":
        off = s["offsets"].tolist()
        a, sc = s["a"], s["a_scale"]
        if case["gather"]:
            a, sc = a.index_select(0, s["rows"]), sc.index_select(0, s["rows"])
        out = torch.empty(off[-1], case["N"], dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            i, j = off[e], off[e + 1]
            if i < j:
                out[i:j] = a[i:j].double() @ s["w"][e].double().T
                out[i:j] *= sc[i:j].double().outer(s["w_scale"][e].double())
                if s["b"] is not None:
                    out[i:j] += s["b"][e].double()
        return out
    if case["op"] == "quant":
        x = s["x"].double()
        if case["act"] == "silu_mul":
            x = torch.sigmoid(x[:, :case["K"]]) * x[:, :case["K"]] * x[:, case["K"]:]
        elif case["act"] == "relu2":
            x = torch.where(x > 0, x * x, 0.0)
        top = x.abs().max(dim=1, keepdim=True).values
        step = torch.where(top == 0, 1.0, top / 127)
        return {"values": torch.round(x / step) * step, "scale": step[:, 0]}
    if case["op"] == "route":
        return _route_exact(case, s)
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    for j in range(case["k"]):
        out += s["weights"][:, j:j + 1].double() * s["y"].index_select(0, s["slots"][:, j]).double()
    return out if s["add"] is None else out + s["add"].double()


def _route_exact(case, s):
    """The definition token by token, on the host."""
    x = s["logits"].double().cpu().numpy()
    b = None if s["b"] is None else s["b"].double().cpu().numpy()
    T, E, k, G = case["T"], case["E"], case["k"], case["n_group"]
    ids, weights = np.full((T, k), -1), np.zeros((T, k))
    for t in range(T):
        live = np.flatnonzero(x[t] > -np.inf)
        if not live.size:
            continue
        if case["score"] == "softmax":
            p = np.exp(x[t] - x[t, live].max())
            p /= p.sum()
        else:
            with np.errstate(over="ignore"):
                p = 1 / (1 + np.exp(-x[t]))
        key = x[t] if b is None else p + b
        if G > 1:
            size = E // G
            base = p if b is None and case["group_score"] == "top2" else key
            total = np.full(G, -np.inf)
            for gr in range(G):
                mine = np.sort(base[live[live // size == gr]])[::-1][:2 if case["group_score"] == "top2" else 1]
                if mine.size:
                    total[gr] = mine.sum()
            kept = np.argsort(-total, kind="stable")[:case["topk_group"]]
            live = live[np.isin(live // size, kept)]
        chosen = live[np.argsort(-key[live], kind="stable")][:k]
        w = p[chosen]
        if case["renorm"] and w.sum() > 0:
            w = w / w.sum()
        ids[t, :len(chosen)], weights[t, :len(chosen)] = chosen, w
    taken = [(e, t, j) for t in range(T) for j, e in enumerate(ids[t]) if e >= 0]
    taken.sort()
    rows, slots = np.full(T * k, -1), np.full((T, k), -1)
    for r, (_, t, j) in enumerate(taken):
        rows[r], slots[t, j] = t, r
    offsets = np.concatenate([[0], np.cumsum(np.bincount(ids[ids >= 0], minlength=E))])
    return {"ids": ids, "weights": weights, "offsets": offsets, "rows": rows, "slots": slots}
