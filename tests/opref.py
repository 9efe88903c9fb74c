"""Plain 64-bit forms of grouped routing, 8-bit float products and the norms around a block, for the tests."""
import numpy as np
import torch

TINY_SUM = 2.0 ** -14


def route(logits, bias, experts, active, score, groups, top_groups, best, normalize, scale):
    """numpy f64 logits [T, E] -> ids, weights; token by token, straight from the definition."""
    T, E = logits.shape
    ids, probs = np.zeros((T, active), np.int64), np.zeros((T, active))
    size = E // groups
    for t in range(T):
        l = logits[t]
        s = 1.0 / (1.0 + np.exp(-l)) if score == "sigmoid" else np.exp(l - l.max()) / np.exp(l - l.max()).sum()
        r = s if bias is None else s + bias
        worth = [sum(sorted(r[g * size:(g + 1) * size], reverse=True)[:best]) for g in range(groups)]
        kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:top_groups]
        pool = sorted((e for g in kept for e in range(g * size, (g + 1) * size)), key=lambda e: (-r[e], e))
        ids[t] = pool[:active]
        p = s[ids[t]]
        probs[t] = p / max(p.sum(), TINY_SUM) * scale if normalize else p * scale
    return ids, probs


def quantize(x):
    """Rows f64 [T, K] -> (codes as f64, scales [T, blocks]); blocks of 128, the last one may be short."""
    T, K = x.shape
    codes, scales = torch.zeros_like(x), []
    for a in range(0, K, 128):
        b = x[:, a:a + 128]
        top = b.abs().amax(1, keepdim=True)
        q = torch.where(top > 0, b * 448.0 / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(b))
        codes[:, a:a + 128] = q.to(torch.float8_e4m3fn).double()
        scales.append(top / 448.0)
    return codes, torch.cat(scales, 1)


def product(codes, scales, w, ws):
    """codes [T, K], scales [T, kb]; w e4m3 [n, K], ws [nb, kb] -> (y, sum of the absolute terms), f64."""
    n, K = w.shape
    wide = ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :K] * w.double()
    x = codes * scales.repeat_interleave(128, 1)[:, :K]
    return x @ wide.t(), x.abs() @ wide.abs().t()


def ffn(x, gate, gate_s, up, up_s, down, down_s):
    c, s = quantize(x)
    g, _ = product(c, s, gate, gate_s)
    u, _ = product(c, s, up, up_s)
    ac, as_ = quantize(g * torch.sigmoid(g) * u)
    return product(ac, as_, down, down_s)[0]


def weights(gen, lead, n, k, device="cuda"):
    """e4m3 codes that reach the format's largest value and scales of one binade."""
    codes = (torch.randn((*lead, n, k), device=device, generator=gen) * 105.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = (torch.rand((*lead, -(-n // 128), -(-k // 128)), device=device, generator=gen) + 0.5) * 2e-4
    return codes, scales


def norm(v, kind, w, b, offset, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + eps)
    if w is not None:
        v = v * (w.double() + offset)
    return v if b is None else v + b.double()


def block_norm(hidden, block, pre_w=None, pre_b=None, post_w=None, post_b=None, gate=None, act="none", kind="rms", offset=0.0,
               residual_scale=1.0, block_scale=1.0, eps=1e-6):
    h = residual_scale * hidden.double()
    if block is not None:
        b = block.double()
        if post_w is not None:
            b = norm(b, kind, post_w, post_b, offset, eps)
        if gate is not None:
            g = gate.double()
            b = b * (torch.sigmoid(g) if act == "sigmoid" else torch.tanh(g) if act == "tanh" else g)
        h = h + block_scale * b
    return h, norm(h, kind, pre_w, pre_b, offset, eps)
