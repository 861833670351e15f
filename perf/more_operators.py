"""The workloads that the speed of 8-bit floating point projections with block scales, and of a mixture-of-experts layer on
weights of that form, is judged on.

  op "quant"    one call of fp8.quantize_act: activation rows to e4m3 codes with one scale per 128 inputs
  op "gemm"     one call of fp8.gemm: such rows times e4m3 weights that have one scale per block of 128 x 128
  op "route"    one call of moe.route: a router's logits to each token's experts and their weights
  op "experts"  one call of moe.experts: a token's experts, gate, up, SwiGLU, down and the weighted sum, for a few tokens

"rows" is the number of rows the buffers hold (a token bucket), "live" the rows really there; rows behind them stay as they
are.  Weights are laid out once, in `prepare`, as a program does at load.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_MIN = 1e-10


def _quant(name, rows, k, x="bf16", live=None):
    return dict(name=name, op="quant", rows=rows, live=rows if live is None else live, k=k, x=x)


def _gemm(name, rows, n, k, live=None):
    return dict(name=name, op="gemm", rows=rows, live=rows if live is None else live, n=n, k=k)


def _route(name, rows, experts, top, score, logits="f32", live=None):
    return dict(name=name, op="route", rows=rows, live=rows if live is None else live, experts=experts, top=top, score=score,
                logits=logits)


def _experts(name, rows, experts, top, hidden, inter, live=None):
    return dict(name=name, op="experts", rows=rows, live=rows if live is None else live, experts=experts, top=top,
                hidden=hidden, inter=inter)


def listed():
    return [
        # one token's activations in front of a projection: latency
        _quant("quant_1", 1, 5120),
        # a long prompt's, in front of the down projection
        _quant("quant_8191", 8191, 17408),
        # one token of one user: a weight stream, latency
        _gemm("gemm_1", 1, 5120, 5120),
        # a full decode batch of 16 through the down projection
        _gemm("gemm_16", 16, 5120, 17408),
        # 37 users in a bucket of 48
        _gemm("gemm_37_of_48", 48, 13824, 5120, live=37),
        # a short prompt of an odd length: too few tiles for the card
        _gemm("gemm_333", 333, 5120, 17408),
        # a long prompt through the widest projection
        _gemm("gemm_8191", 8191, 27648, 5120),
        # one token's experts: latency
        _route("route_1", 1, 128, 8, "softmax"),
        # a long prompt's, scored one by one with a bias that balances the experts, logits as a projection leaves them
        _route("route_8191", 8191, 256, 8, "sigmoid", "bf16"),
        # one token of one user through a layer of many small experts: latency
        _experts("experts_1", 1, 128, 8, 2048, 768),
        # 11 users in a bucket of 16, wide experts of which each token takes two
        _experts("experts_11_of_16", 16, 16, 2, 5120, 1408, live=11),
        # a decode batch that reaches every expert
        _experts("experts_64", 64, 128, 8, 2048, 768),
    ]


def _log(rng, lo, hi):
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))), lo), hi)


def _live(rng, rows):
    return max(1, rows - rng.choice((0, rng.randint(0, rows // 4))))


def draw(rng):
    op = rng.choice(("quant", "gemm", "gemm", "gemm", "route", "experts", "experts"))
    most = [work(d) for d in listed() if d["op"] == op]
    while True:
        if op == "quant":
            rows = _log(rng, 1, 8191)
            c = _quant("", rows, rng.choice((128 * rng.randint(1, 136), _log(rng, 1, 17408))), rng.choice(("bf16", "f32")),
                       _live(rng, rows))
        elif op == "gemm":
            rows = _log(rng, 1, 8191)
            c = _gemm("", rows, rng.choice((128 * rng.randint(1, 216), _log(rng, 1, 27648))),
                      rng.choice((128 * rng.randint(1, 136), _log(rng, 16, 17408))), _live(rng, rows))
        elif op == "route":
            rows, experts = _log(rng, 1, 8191), _log(rng, 4, 512)
            c = _route("", rows, experts, rng.randint(1, min(experts, 12)), rng.choice(("softmax", "sigmoid")),
                       rng.choice(("f32", "bf16")), _live(rng, rows))
        else:
            rows, experts = _log(rng, 1, 128), rng.choice((8, 16, 40, 64, 128, 256))
            c = _experts("", rows, experts, rng.randint(1, 8), 16 * _log(rng, 32, 448), 16 * _log(rng, 8, 128),
                         _live(rng, rows))
        w = work(c)
        fits = op != "experts" or 3 * c["experts"] * c["hidden"] * c["inter"] <= 700 << 20
        if fits and all(w[x] <= max(m[x] for m in most) for x in w):
            del c["name"]
            return c


def _blocks(k):
    return -(-k // BLOCK)


def work(case):
    c, t = case, case["live"]
    if c["op"] == "quant":
        return {"bytes": t * (c["k"] * (2 if c["x"] == "bf16" else 4) + _blocks(c["k"]) * (BLOCK + 4)), "flops": t * c["k"]}
    if c["op"] == "gemm":
        n, k = c["n"], c["k"]
        return {"bytes": n * k + _blocks(n) * _blocks(k) * 4 + t * (k + _blocks(k) * 4) + t * n * 2, "flops": 2 * t * n * k}
    if c["op"] == "route":
        return {"bytes": t * (c["experts"] * (2 if c["logits"] == "bf16" else 4) + c["top"] * 8),
                "flops": t * c["experts"] * 8}
    e, h, i, top = c["experts"], c["hidden"], c["inter"], c["top"]
    reached = e * (1 - (1 - top / e) ** t)                             # distinct experts, expected of random choices
    return {"bytes": int(reached * (3 * h * i + 3 * _blocks(h) * _blocks(i) * 4)) + t * (4 * h + top * 8),
            "flops": 6 * t * top * h * i}


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, *shape):
    """e4m3 weights as a quantizer leaves them: normal values whose blocks' largest reach 448."""
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat, step = out.view(-1), 1 << 26
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_((100 * _normal(g, part.numel())).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn))
    return out


def _weight_scales(g, k, *shape):
    """Scales that give outputs near 1, blocks a factor of four apart."""
    return (0.5 + 1.5 * torch.rand(*shape, generator=g, device="cuda")) / (100 * math.sqrt(k))


def _rows(c, g, k):
    """Activation rows e4m3 [rows, whole blocks of k] and their scales, as the quantizer leaves them."""
    x = torch.zeros(c["rows"], _blocks(k) * BLOCK, device="cuda")
    x[:, :k] = _activations(g, c["rows"], k)
    x = x.unflatten(1, (-1, BLOCK))
    s = x.abs().amax(2).clamp(min=AMAX_MIN) / E4M3_MAX
    return (x / s[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).flatten(1), s


def _activations(g, rows, k):
    """Normal values, a few channels twenty times larger, as hidden rows have them."""
    x = _normal(g, rows, k)
    return torch.where(torch.rand(k, generator=g, device="cuda") < 0.004, 20 * x, x)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c, "n": torch.tensor([c["live"]], dtype=torch.int32, device="cuda")}
    if own:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "startlux-prism_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        from prism_amd import fp8, moe
        s["fp8"], s["moe"] = fp8, moe
    if c["op"] == "quant":
        s["x"] = _activations(g, c["rows"], c["k"]).to(torch.bfloat16 if c["x"] == "bf16" else torch.float32)
        s["q"] = torch.zeros(c["rows"], _blocks(c["k"]) * BLOCK, device="cuda").to(torch.float8_e4m3fn)
        s["s"] = torch.zeros(c["rows"], _blocks(c["k"]), device="cuda")
    elif c["op"] == "gemm":
        n, k = c["n"], c["k"]
        s["a"], s["as"] = _rows(c, g, k)
        s["w"], s["ws"] = _codes(g, n, k), _weight_scales(g, k, _blocks(n), _blocks(k))
        s["out"] = torch.zeros(c["rows"], n, dtype=torch.bfloat16, device="cuda")
        if own:
            s["weight"] = fp8.from_rows(s["w"], s["ws"])
    elif c["op"] == "route":
        x = 2 * _normal(g, c["rows"], c["experts"])
        s["x"] = x.to(torch.bfloat16) if c["logits"] == "bf16" else x
        s["bias"] = 0.1 * _normal(g, c["experts"]) if c["score"] == "sigmoid" else None
        s["ids"] = torch.full((c["rows"], c["top"]), -1, dtype=torch.int32, device="cuda")
        s["w"] = torch.zeros(c["rows"], c["top"], device="cuda")
    else:
        e, h, i = c["experts"], c["hidden"], c["inter"]
        s["x"] = _activations(g, c["rows"], h).to(torch.bfloat16)
        p, s["ids"] = torch.softmax(_normal(g, c["rows"], e), 1).topk(c["top"], 1)
        s["ids"], s["w"] = s["ids"].to(torch.int32), p / p.sum(1, keepdim=True)
        for name, n, k in (("gate", i, h), ("up", i, h), ("down", h, i)):
            s[name], s[name + "_s"] = _codes(g, e, n, k), _weight_scales(g, k, e, _blocks(n), _blocks(k))
            if own:
                s[name + "_weight"] = fp8.from_rows(s[name], s[name + "_s"])
        s["out"] = torch.zeros(c["rows"], h, dtype=torch.bfloat16, device="cuda")
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _spread(s, n, k):
    """A scale per 128 x 128 block -> one per weight [n, k]."""
    return s.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_quant(s):
    c, t = s["case"], s["case"]["live"]
    x = torch.zeros(t, s["q"].shape[1], device="cuda")
    x[:, :c["k"]] = s["x"][:t].float()
    x = x.unflatten(1, (-1, BLOCK))
    scale = x.abs().amax(2).clamp(min=AMAX_MIN) / E4M3_MAX
    s["q"][:t] = (x / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).flatten(1)
    s["s"][:t] = scale
    return s["q"], s["s"]


def _plain_gemm(s):
    c, t = s["case"], s["case"]["live"]
    a = (s["a"][:t].float().unflatten(1, (-1, BLOCK)) * s["as"][:t, :, None]).flatten(1)[:, :c["k"]]
    w = s["w"].float() * _spread(s["ws"], c["n"], c["k"])
    s["out"][:t] = (a @ w.T).to(torch.bfloat16)
    return s["out"]


def _plain_route(s):
    c, t = s["case"], s["case"]["live"]
    x = s["x"][:t].float()
    if c["score"] == "softmax":
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :c["top"]]
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x.double()))                            # 64 bits: neighbours decide the choice
        ids = torch.sort(p + s["bias"].double(), dim=1, descending=True, stable=True)[1][:, :c["top"]]
    w = torch.gather(p, 1, ids)
    s["ids"][:t] = ids.to(torch.int32)
    s["w"][:t] = (w / w.sum(1, keepdim=True)).float()
    return s["ids"], s["w"]


def _plain_experts(s):
    """Each pair's experts gathered where there are fewer pairs than experts, else every expert in turn."""
    c, t = s["case"], s["case"]["live"]
    x, ids = s["x"][:t].float(), s["ids"][:t].long()

    def silu(a):
        return a / (1 + torch.exp(-a))
    if ids.numel() < c["experts"]:
        of = ids.flatten()

        def product(name, v):
            w, sc = s[name][of].float(), s[name + "_s"][of]
            sc = sc.repeat_interleave(BLOCK, 1)[:, :w.shape[1]].repeat_interleave(BLOCK, 2)[:, :, :w.shape[2]]
            return torch.bmm(w * sc, v[:, :, None])[:, :, 0]
        v = x.repeat_interleave(c["top"], 0)
        y = product("down", silu(product("gate", v)) * product("up", v)) * s["w"][:t].flatten()[:, None]
        y = y.unflatten(0, (t, c["top"])).sum(1)
    else:
        y = torch.zeros(t, c["hidden"], device="cuda")
        share = torch.zeros(t, c["experts"], device="cuda").scatter_add_(1, ids, s["w"][:t])
        for e in range(c["experts"]):
            gate, up, down = (s[k][e].float() * _spread(s[k + "_s"][e], *s[k][e].shape) for k in ("gate", "up", "down"))
            y += ((silu(x @ gate.T) * (x @ up.T)) @ down.T) * share[:, e:e + 1]
    s["out"][:t] = y.to(torch.bfloat16)
    return s["out"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"quant": _plain_quant, "gemm": _plain_gemm, "route": _plain_route, "experts": _plain_experts}[c["op"]](s)
    if c["op"] == "quant":
        s["fp8"].quantize_act(s["x"], s["q"], s["s"], s["n"], c["rows"])
        return s["q"], s["s"]
    if c["op"] == "gemm":
        s["fp8"].gemm(s["a"], s["as"], s["weight"], s["out"], s["n"], c["rows"])
        return s["out"]
    if c["op"] == "route":
        s["moe"].route(s["x"], s["ids"], s["w"], s["n"], c["rows"], score=c["score"], bias=s["bias"])
        return s["ids"], s["w"]
    s["moe"].experts(s["x"], s["ids"], s["w"], s["gate_weight"], s["up_weight"], s["down_weight"], s["out"], s["n"],
                     c["rows"])
    return s["out"]


# ------------------------------------------------------------------------------------------------ 64 bits, by definition
def exact(case, seed):
    c, s, t = case, prepare(case, seed), case["live"]
    f64 = torch.float64
    if c["op"] == "quant":
        q, scale = s["q"].to(f64), s["s"].to(f64)
        for b in range(_blocks(c["k"])):
            x = s["x"][:t, BLOCK * b:BLOCK * (b + 1)].to(f64)
            x = x[:, :c["k"] - BLOCK * b]
            scale[:t, b] = torch.clamp(torch.maximum(x.amax(1), -x.amin(1)), min=AMAX_MIN) / E4M3_MAX
            q[:t, BLOCK * b:BLOCK * b + x.shape[1]] = x / scale[:t, b:b + 1]
        return q, scale
    if c["op"] == "gemm":
        out = s["out"].to(f64)
        for b in range(_blocks(c["k"])):
            lo, hi = BLOCK * b, min(BLOCK * (b + 1), c["k"])
            of = torch.arange(c["n"], device="cuda") // BLOCK
            out[:t] += (s["a"][:t, lo:hi].to(f64) * s["as"][:t, b:b + 1].to(f64)) @ (
                s["w"][:, lo:hi].to(f64) * s["ws"][of, b].to(f64)[:, None]).T
        return out
    if c["op"] == "route":
        x, ids, w = s["x"][:t].to(f64).cpu(), s["ids"].cpu(), s["w"].to(f64).cpu()
        p = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
        key = x.clone() if c["score"] == "softmax" else p + s["bias"].to(f64).cpu()
        for j in range(c["top"]):
            best = (key == key.max(1, keepdim=True).values).to(torch.int8).argmax(1)
            ids[:t, j] = best.to(torch.int32)
            w[:t, j] = p[torch.arange(t), best]
            key[torch.arange(t), best] = -math.inf
        w[:t] /= w[:t].sum(1, keepdim=True)
        return ids.cuda(), w.cuda()
    out = s["out"].to(f64)

    def wide(name, e):
        w, sc = s[name][e].to(f64), s[name + "_s"][e].to(f64)
        i, j = (torch.arange(d, device="cuda") // BLOCK for d in w.shape)
        return w * sc[i][:, j]
    for e in sorted(set(s["ids"][:t].flatten().tolist())):
        at, j = (s["ids"][:t] == e).nonzero(as_tuple=True)
        x = s["x"][at].to(f64)
        y = (torch.nn.functional.silu(x @ wide("gate", e).T) * (x @ wide("up", e).T)) @ wide("down", e).T
        out.index_add_(0, at, y * s["w"][at, j].to(f64)[:, None])
    return out
