"""Operators around and inside an expert layer: routing with groups of experts, products with 8-bit floating-point
weights that carry one scale per block of 128 x 128, and the norms before and after a block with its gate and residual
scale. Each case is one call of one operator, over the range of sizes that serving and prefill meet.

  route    rows -> expert ids and weights (`moe.RouterPlan.forward`: the router product, then the selection)
  select   logits -> expert ids and weights (`moe.RouterPlan.select`)
  dense    a projection or a gated feed-forward (`dense.DensePlan` with `synth.FMT_F8_E4M3`)
  experts  routed tokens through their experts onto the residual (`moe.F8ExpertPlan.forward`)
  norm     residual update with post-norm, gate and scales, then the next block's norm (`moe.block_norm`)

Where `own` is false the operators run in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
BLOCK = 128
TINY_SUM = 2.0 ** -14      # the divisor of renormalised weights is at least this


def listed():
    def route(name, rows, hidden, experts, active, score, groups=1, top_groups=1, best=1, bias=False, normalize=True, scale=1.0):
        return dict(name=name, op="route", rows=rows, hidden=hidden, experts=experts, active=active, score=score, groups=groups,
                    top_groups=top_groups, best=best, bias=bias, normalize=normalize, scale=scale)

    def dense(name, rows, kind, hidden, ffn):
        return dict(name=name, op="dense", rows=rows, kind=kind, hidden=hidden, ffn=ffn)

    def experts(name, rows, hidden, ffn, experts, active, absent=0.0):
        return dict(name=name, op="experts", rows=rows, hidden=hidden, ffn=ffn, experts=experts, active=active, absent=absent)

    def norm(name, rows, hidden, kind, post, gate, act, wide, residual_scale=1.0, block_scale=1.0, offset=0.0):
        return dict(name=name, op="norm", rows=rows, hidden=hidden, kind=kind, post=post, gate=gate, act=act, wide=wide,
                    residual_scale=residual_scale, block_scale=block_scale, offset=offset)

    return [
        # one token of a decode loop: softmax over all experts, the winners renormalised
        route("route-token", 1, 2048, 128, 8, "softmax"),
        # the ragged last chunk of a prompt, sigmoid scores, five groups of 32 experts
        route("route-chunk-333", 333, 2688, 160, 6, "sigmoid", 5, 2, 2, True, True, 2.5),
        # a prefill batch: 256 experts in eight groups, half of the groups kept
        route("route-prefill-8192", 8192, 4096, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5),
        # logits that another product made, many tokens
        dict(route("select-32768", 32768, 0, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5), op="select"),
        # one token through a projection: the weights are read once
        dense("f8-projection-token", 1, "projection", 4096, 6144),
        # a decode batch through a gated feed-forward
        dense("f8-ffn-48", 48, "silu_gate", 2048, 6144),
        # a prefill batch through a projection
        dense("f8-projection-8192", 8192, "projection", 4096, 8192),
        # one token through its eight experts
        experts("f8-experts-token", 1, 2048, 768, 128, 8),
        # a decode batch: most experts are touched by a few tokens each, some rows are padding
        experts("f8-experts-64", 64, 2048, 768, 128, 8, 0.06),
        # a prefill batch over wide experts
        experts("f8-experts-4096", 4096, 4096, 2048, 64, 6),
        # one token between two blocks
        norm("norm-token", 1, 2880, "rms", True, "none", "none", False),
        # a batch of rows with a gate value for each element and scaled branches
        norm("norm-8192", 8192, 4096, "rms", True, "row", "sigmoid", False, 1.0, 0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, lo, hi, step):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, _log(rng, lo, hi) // step * step))


def draw(rng):
    op = rng.choice(["route", "route", "select", "dense", "dense", "experts", "experts", "norm", "norm"])
    if op in ("route", "select"):
        groups = rng.choice([1, 1, 2, 4, 5, 8, 16])
        size = max(2, _log(rng, 8, 512) // groups)
        experts = min(size, 512 // groups) * groups
        top_groups = rng.randint(1, groups)
        active = rng.randint(1, max(1, min(16, top_groups * (experts // groups))))
        hidden = 0 if op == "select" else _mult(rng, 256, 8192, 32)
        most = 65536 if op == "select" else min(8192, max(1, 8192 * 4096 * 256 // (hidden * experts)))
        rows = _log(rng, 1, most if op == "route" else max(1, most * 128 // max(128, experts)))
        return dict(op=op, rows=rows, hidden=hidden, experts=experts, active=active, score=rng.choice(["sigmoid", "softmax"]),
                    groups=groups, top_groups=top_groups, best=rng.choice([1, 2]), bias=rng.random() < 0.6,
                    normalize=rng.random() < 0.7, scale=rng.choice([1.0, 1.0, 2.5]))
    if op == "dense":
        kind = rng.choice(["projection", "silu_gate"])
        hidden, ffn = _mult(rng, 256, 8192, 32), _mult(rng, 256, 8192, 32)
        most = 8192 * 4096 * 8192 // (hidden * ffn * (3 if kind == "silu_gate" else 1))
        return dict(op=op, rows=_log(rng, 1, max(1, min(8192, most))), kind=kind, hidden=hidden, ffn=ffn)
    if op == "experts":
        hidden, ffn = _mult(rng, 256, 4096, 32), _mult(rng, 128, 2048, 32)
        experts = max(4, min(_log(rng, 4, 256), 64 * 4096 * 2048 // (hidden * ffn)))
        active = rng.randint(1, min(8, experts))
        most = 4096 * 6 * 4096 * 2048 // (hidden * ffn * active)
        return dict(op=op, rows=_log(rng, 1, max(1, min(4096, most))), hidden=hidden, ffn=ffn, experts=experts, active=active,
                    absent=rng.choice([0.0, 0.0, 0.1, 0.5]))
    hidden = _mult(rng, 64, 16384, 8)
    rows = _log(rng, 1, max(1, min(16384, 8192 * 2048 // hidden)))
    return dict(op=op, rows=rows, hidden=hidden, kind=rng.choice(["rms", "rms", "layer"]), post=rng.random() < 0.6,
                gate=rng.choice(["none", "channel", "row"]), act=rng.choice(["none", "sigmoid", "tanh"]), wide=rng.random() < 0.3,
                residual_scale=rng.choice([1.0, 1.0, 0.7]), block_scale=rng.choice([1.0, 0.22]), offset=rng.choice([0.0, 1.0]))


# ---- inputs ----------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, scale=1.0, mean=0.0):
    return torch.randn(shape, device="cuda", generator=g) * scale + mean


def _f8_weights(g, lead, n, k):
    """Codes [*lead, n, k] and one positive scale per block of 128 x 128, as a checkpoint holds them: the largest code of
    a block is near the format's largest value."""
    codes = (torch.randn((*lead, n, k), device="cuda", generator=g, dtype=torch.bfloat16) * 105.0).clamp_(-F8_MAX, F8_MAX).to(F8)
    blocks = (*lead, -(-n // BLOCK), -(-k // BLOCK))
    scales = (torch.rand(blocks, device="cuda", generator=g) + 0.5) * (0.02 / 105.0)
    return codes, scales


def _inputs(case, seed):
    g = _gen(seed)
    s = dict(case)
    rows, op = case["rows"], case["op"]
    if op in ("route", "select"):
        E, H = case["experts"], case["hidden"]
        s["bias"] = _normal(g, (E,), 0.1) if case["bias"] else None
        if op == "route":
            s["w"] = _normal(g, (E, H), 0.02)
            s["x"] = _normal(g, (rows, H)).to(torch.bfloat16)
        else:
            s["logits"] = _normal(g, (rows, E), 1.3)
    elif op == "dense":
        H, F = case["hidden"], case["ffn"]
        s["x"] = _normal(g, (rows, H)).to(torch.bfloat16)
        s["up"], s["up_s"] = _f8_weights(g, (), F, H)
        if case["kind"] == "silu_gate":
            s["gate"], s["gate_s"] = _f8_weights(g, (), F, H)
            s["down"], s["down_s"] = _f8_weights(g, (), H, F)
    elif op == "experts":
        H, F, E, k = case["hidden"], case["ffn"], case["experts"], case["active"]
        s["x"] = _normal(g, (rows, H)).to(torch.bfloat16)
        s["residual"] = _normal(g, (rows, H)).to(torch.bfloat16)
        s["ids"] = torch.topk(torch.rand((rows, E), device="cuda", generator=g), k, dim=1).indices.to(torch.int32)
        gone = torch.rand((rows, k), device="cuda", generator=g) < case["absent"]
        s["ids"] = torch.where(gone, torch.full_like(s["ids"], -1), s["ids"])     # routes of padding or of another shard
        p = torch.rand((rows, k), device="cuda", generator=g) + 0.05
        s["probs"] = p / p.sum(1, keepdim=True)
        for name, n, kk in (("gate", F, H), ("up", F, H), ("down", H, F)):
            s[name], s[name + "_s"] = _f8_weights(g, (E,), n, kk)
    else:
        H = case["hidden"]
        t = torch.float32 if case["wide"] else torch.bfloat16
        s["hidden_rows"] = _normal(g, (rows, H), 2.0).to(t)
        s["block"] = _normal(g, (rows, H), 0.7, 0.05).to(torch.bfloat16)
        s["pre_w"] = _normal(g, (H,), 0.1, 1.0 - case["offset"])
        s["pre_b"] = _normal(g, (H,), 0.1) if case["kind"] == "layer" else None
        s["post_w"] = _normal(g, (H,), 0.1, 1.0 - case["offset"]) if case["post"] else None
        s["post_b"] = _normal(g, (H,), 0.1) if case["post"] and case["kind"] == "layer" else None
        s["gate_v"] = None
        if case["gate"] == "channel":
            s["gate_v"] = _normal(g, (H,), 0.5, 0.5)
        elif case["gate"] == "row":
            s["gate_v"] = _normal(g, (rows, H)).to(torch.bfloat16)
        s["eps"] = 1e-5
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    rows, op = case["rows"], case["op"]
    new = lambda shape, t: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
    if own:
        from oco_b200 import dense, moe, synth
        s["moe"] = moe
    if op in ("route", "select"):
        k = case["active"]
        s["ids"], s["probs"] = new((rows, k), torch.int32), new((rows, k), torch.float32)
        if op == "route":
            s["logits"] = new((rows, case["experts"]), torch.float32)
        if own:
            s["plan"] = moe.RouterPlan.new(case["hidden"], case["experts"], k, score=case["score"], groups=case["groups"],
                                           top_groups=case["top_groups"], group_best=case["best"], normalize=case["normalize"],
                                           scale=case["scale"])
            s["plan"].reserve(rows)
            s["plan"].bind(s.get("w"), s["bias"])
    elif op == "dense":
        s["y"] = new((rows, case["ffn"] if case["kind"] == "projection" else case["hidden"]), torch.bfloat16)
        if own:
            kind = dense.PROJECTION if case["kind"] == "projection" else dense.FFN_SILU_GATE
            s["plan"] = dense.DensePlan(kind, synth.FMT_F8_E4M3, case["hidden"], case["ffn"])
            s["plan"].reserve(rows)
            s["plan"].bind(s["up"], s.get("gate"), s.get("down"), up_scale=s["up_s"], gate_scale=s.get("gate_s"),
                           down_scale=s.get("down_s"))
    elif op == "experts":
        s["out"] = new((rows, case["hidden"]), torch.bfloat16)
        if own:
            s["plan"] = moe.F8ExpertPlan.new(case["hidden"], case["ffn"], case["experts"], case["active"])
            s["plan"].reserve(rows)
            s["plan"].bind(moe.F8Experts(gate_w=s["gate"], gate_s=s["gate_s"], up_w=s["up"], up_s=s["up_s"], down_w=s["down"],
                                         down_s=s["down_s"]))
    else:
        s["hidden_out"] = torch.empty_like(s["hidden_rows"])
        s["norm_out"] = new((rows, case["hidden"]), torch.bfloat16)
    torch.cuda.synchronize()
    return s


# ---- the operators in their plain form ----------------------------------------------------------------------
def _choose(logits, bias, s):
    """Ids and weights of the winners; everything in 64 bits, since neighbouring scores decide which experts run."""
    T, E = logits.shape
    if s["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    else:
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    rank = score if bias is None else score + bias.double()
    G = s["groups"]
    if s["top_groups"] < G:
        best = torch.sort(rank.reshape(T, G, E // G), dim=2, descending=True).values[:, :, :s["best"]].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        open_ = torch.zeros((T, G), dtype=torch.bool, device=rank.device).scatter_(1, kept, True)
        rank = rank.masked_fill(~open_.repeat_interleave(E // G, dim=1), -math.inf)
    ids = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :s["active"]]
    p = torch.gather(score, 1, ids)
    if s["normalize"]:
        p = p / p.sum(1, keepdim=True).clamp_min(TINY_SUM)
    return ids.to(torch.int32), (p * s["scale"]).float()


def _quantized(x):
    """Rows in 32 bits, each block of 128 elements rounded to 8-bit floating point under its own scale (largest / 448).
    b * 448 / largest with one rounding: b * (7 / 8) is exact for bf16 rows, so that an element halfway between two codes
    is seen as such (b / (largest / 448) lands beside the middle)."""
    T, K = x.shape
    pad = -K % BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).reshape(T, -1, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    q = (b * 0.875 / torch.where(top > 0, top, torch.ones_like(top)) * 512.0).to(F8).float()
    return (q * (top / F8_MAX)).reshape(T, -1)[:, :K]


def _weights(codes, scales):
    n, k = codes.shape[-2:]
    wide = scales.repeat_interleave(BLOCK, dim=-2)[..., :n, :].repeat_interleave(BLOCK, dim=-1)[..., :k]
    return codes.float() * wide


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _plain_dense(s):
    x = _quantized(s["x"].float())
    up = x @ _weights(s["up"], s["up_s"]).t()
    if s["kind"] == "projection":
        return up.to(torch.bfloat16)
    act = _silu(x @ _weights(s["gate"], s["gate_s"]).t()) * up
    return (_quantized(act) @ _weights(s["down"], s["down_s"]).t()).to(torch.bfloat16)


def _plain_experts(s):
    """Routes sorted by expert, each expert's padded to whole tiles of rows, one batched product over the tiles."""
    T, k, E, H, F = s["rows"], s["active"], s["experts"], s["hidden"], s["ffn"]
    R = T * k
    t = 256 if R >= 8192 else 64 if R >= 1024 else 16
    tiles = R // t + min(E, R)
    at = s["x"].device
    ids = s["ids"].reshape(-1).long()
    key = torch.where((ids >= 0) & (ids < E), ids, torch.full_like(ids, E))
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.long, device=at).scatter_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(counts, 0) - counts
    end_tile = torch.cumsum((counts[:E] + t - 1) // t, 0)
    begin_tile = torch.cat([end_tile - (counts[:E] + t - 1) // t, torch.full((1,), tiles, dtype=torch.long, device=at)])
    of = key[order]
    slot = begin_tile[of] * t + torch.where(of < E, torch.arange(R, device=at) - first[of], torch.zeros_like(of))
    expert = torch.searchsorted(end_tile, torch.arange(tiles, device=at), right=True).clamp_max(E - 1)
    rows = torch.zeros((tiles * t + 1, H), device=at)      # the last row takes the routes that no expert here serves
    rows[slot] = _quantized(s["x"].float())[order // k]
    rows = rows[:-1].reshape(tiles, t, H)
    pick = lambda name: _weights(s[name].view(torch.uint8)[expert].view(F8), s[name + "_s"][expert])  # noqa: E731
    g = torch.bmm(rows, pick("gate").transpose(1, 2))
    act = _silu(g) * torch.bmm(rows, pick("up").transpose(1, 2))
    act = _quantized(act.reshape(tiles * t, F)).reshape(tiles, t, F)
    y = torch.bmm(act, pick("down").transpose(1, 2)).reshape(tiles * t, H)
    y = torch.cat([y, torch.zeros((1, H), device=at)])
    back = torch.empty((R, H), device=at)
    back[order] = y[slot]
    total = (back.reshape(T, k, H) * s["probs"].unsqueeze(2)).sum(1)
    return (s["residual"].float() + total).to(torch.bfloat16)


def _norm(v, kind, weight, bias, offset, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * (weight + offset)
    return v if bias is None else v + bias


def _plain_norm(s):
    b = s["block"].float()
    if s["post"]:
        b = _norm(b, s["kind"], s["post_w"], s["post_b"], s["offset"], s["eps"])
    if s["gate_v"] is not None:
        g = s["gate_v"].float()
        g = 1.0 / (1.0 + torch.exp(-g)) if s["act"] == "sigmoid" else torch.tanh(g) if s["act"] == "tanh" else g
        b = g * b
    h = s["residual_scale"] * s["hidden_rows"].float() + s["block_scale"] * b
    x = _norm(h, s["kind"], s["pre_w"], s["pre_b"], s["offset"], s["eps"])
    return h.to(s["hidden_rows"].dtype), x.to(torch.bfloat16)


def run(s):
    op = s["op"]
    if own:
        if op == "route":
            s["plan"].forward(s["x"], s["ids"], s["probs"], s["rows"], logits=s["logits"])
            return s["ids"], s["probs"], s["logits"]
        if op == "select":
            s["plan"].select(s["logits"], s["ids"], s["probs"], s["rows"])
            return s["ids"], s["probs"]
        if op == "dense":
            s["plan"].forward(s["x"], s["y"], s["rows"])
            return s["y"]
        if op == "experts":
            s["plan"].forward(s["x"], s["ids"], s["probs"], s["residual"], s["rows"], out=s["out"])
            return s["out"]
        s["moe"].block_norm(s["hidden_rows"], s["block"], hidden_out=s["hidden_out"], norm_out=s["norm_out"], pre_weight=s["pre_w"],
                            pre_bias=s["pre_b"], post_weight=s["post_w"], post_bias=s["post_b"], gate=s["gate_v"], gate_act=s["act"],
                            kind=s["kind"], weight_offset=s["offset"], residual_scale=s["residual_scale"],
                            block_scale=s["block_scale"], epsilon=s["eps"])
        return s["hidden_out"], s["norm_out"]
    if op == "route":
        logits = s["x"].double() @ s["w"].double().t()
        ids, probs = _choose(logits, s["bias"], s)
        return ids, probs, logits.float()
    if op == "select":
        return _choose(s["logits"].double(), s["bias"], s)
    if op == "dense":
        return _plain_dense(s)
    if op == "experts":
        return _plain_experts(s)
    return _plain_norm(s)


# ---- what a pass cannot do without -------------------------------------------------------------------------
def work(case):
    rows, op = case["rows"], case["op"]
    if op in ("route", "select"):
        E, H, k = case["experts"], case["hidden"], case["active"]
        moved = rows * 8 * k + 4 * rows * E + (4 * E if case["bias"] else 0)
        if op == "select":
            return dict(bytes=moved, flops=0.0)
        return dict(bytes=moved + 4 * E * H + 2 * rows * H, flops=2.0 * rows * E * H)
    if op == "dense":
        H, F = case["hidden"], case["ffn"]
        mats, out = (1, F) if case["kind"] == "projection" else (3, H)
        return dict(bytes=mats * (H * F + 4 * -(-H // BLOCK) * -(-F // BLOCK)) + 2 * rows * (H + out), flops=2.0 * rows * mats * H * F)
    if op == "experts":
        H, F, E, k = case["hidden"], case["ffn"], case["experts"], case["active"]
        live = k * (1.0 - case["absent"])
        touched = E * (1.0 - (1.0 - live / E) ** rows)       # experts that some token of the batch chooses
        moved = touched * 3 * (H * F + 4 * -(-H // BLOCK) * -(-F // BLOCK)) + rows * (6 * H + 8 * k)
        return dict(bytes=moved, flops=6.0 * rows * live * H * F)
    H = case["hidden"]
    moved = rows * H * (2 * (4 if case["wide"] else 2) + 4) + 4 * H * (1 + case["post"]) * (2 if case["kind"] == "layer" else 1)
    moved += 2 * rows * H if case["gate"] == "row" else 4 * H if case["gate"] == "channel" else 0
    return dict(bytes=moved, flops=20.0 * rows * H)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def _exact_choice(logits, bias, c):
    v = logits.cpu().numpy()
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + np.exp(-v))
    else:
        score = np.exp(v - v.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    rank = score.copy() if bias is None else score + bias.cpu().numpy().astype(np.float64)
    T, E = rank.shape
    G = c["groups"]
    if c["top_groups"] < G:
        parts = np.partition(rank.reshape(T, G, E // G), E // G - c["best"], axis=2) if c["best"] < E // G else rank.reshape(T, G, E // G)
        worth = parts[:, :, E // G - c["best"]:].sum(2) if c["best"] < E // G else parts.sum(2)
        place = np.argsort(np.argsort(-worth, axis=1, kind="stable"), axis=1, kind="stable")
        rank[np.repeat(place >= c["top_groups"], E // G, axis=1)] = -np.inf
    ids = np.argsort(-rank, axis=1, kind="stable")[:, :c["active"]]
    p = np.take_along_axis(score, ids, 1)
    if c["normalize"]:
        p = p / np.maximum(p.sum(1, keepdims=True), TINY_SUM)
    return ids.astype(np.int32), p * c["scale"]


def _exact_rounded(x):
    T, K = x.shape
    out = torch.empty_like(x)
    for a in range(0, K, BLOCK):
        b = x[:, a:a + BLOCK]
        top = b.abs().max(1, keepdim=True).values
        out[:, a:a + BLOCK] = torch.where(top > 0, (b * F8_MAX / top.clamp_min(1e-300)).to(F8).double() * (top / F8_MAX), torch.zeros_like(b))
    return out


def _exact_product(x, codes, scales):
    """x [rows, k] times the transpose of codes [n, k], block of k by block of k."""
    y = torch.zeros((x.shape[0], codes.shape[0]), dtype=torch.float64, device=x.device)
    rows = torch.arange(codes.shape[0], device=x.device) // BLOCK
    for i, a in enumerate(range(0, codes.shape[1], BLOCK)):
        y += x[:, a:a + BLOCK] @ codes[:, a:a + BLOCK].double().t() * scales[rows, i].double()
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("route", "select"):
        logits = s["x"].double() @ s["w"].double().t() if op == "route" else s["logits"].double()
        ids, p = _exact_choice(logits, s["bias"], case)
        return (ids, p, logits.cpu().numpy()) if op == "route" else (ids, p)
    if op == "dense":
        x = _exact_rounded(s["x"].double())
        up = _exact_product(x, s["up"], s["up_s"])
        if case["kind"] == "projection":
            return up
        g = _exact_product(x, s["gate"], s["gate_s"])
        return _exact_product(_exact_rounded(g * torch.sigmoid(g) * up), s["down"], s["down_s"])
    if op == "experts":
        x = _exact_rounded(s["x"].double())
        out = s["residual"].double()
        for e in range(case["experts"]):
            token, place = torch.nonzero(s["ids"] == e, as_tuple=True)
            if token.numel():
                g = _exact_product(x[token], s["gate"][e], s["gate_s"][e])
                a = _exact_rounded(g * torch.sigmoid(g) * _exact_product(x[token], s["up"][e], s["up_s"][e]))
                out.index_add_(0, token, _exact_product(a, s["down"][e], s["down_s"][e]) * s["probs"][token, place].double().unsqueeze(1))
        return out
    def normed(v, w, b):
        if case["kind"] == "layer":
            z = (v - v.mean(1, keepdim=True)) * torch.rsqrt(v.var(1, unbiased=False, keepdim=True) + s["eps"])
        else:
            z = v * torch.rsqrt(v.square().mean(1, keepdim=True) + s["eps"])
        z = z * (w.double() + case["offset"])
        return z if b is None else z + b.double()

    b = s["block"].double()
    if case["post"]:
        b = normed(b, s["post_w"], s["post_b"])
    if s["gate_v"] is not None:
        g = s["gate_v"].double()
        b = b * (torch.sigmoid(g) if case["act"] == "sigmoid" else torch.tanh(g) if case["act"] == "tanh" else g)
    h = case["residual_scale"] * s["hidden_rows"].double() + case["block_scale"] * b
    return h, normed(h, s["pre_w"], s["pre_b"])
