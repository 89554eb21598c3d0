"""Plain 64-bit definitions of the per-request operators (numpy), and the error bounds their tests use."""

import numpy as np
import torch

HALF_STEP_BF16 = 2.0 ** -8   # half a rounding step of bf16 relative to the value: torch.finfo(bfloat16).eps / 2
HALF_STEP_F32 = 2.0 ** -24


def f64(t):
    """A tensor's values in float64 (exact for bf16 and fp32)."""
    return t.detach().to(torch.float64).cpu().numpy()


def dequantize(w, scales, biases, group, bits):
    """The format's weights, bf16(fp32(s q + b)): s q is exact in fp32, so the fp64 sum rounded to fp32 is the
    format's fp32 value."""
    words = w.cpu().numpy().view(np.uint32)
    n, kw = words.shape
    shift = np.arange(32 // bits, dtype=np.uint32) * bits
    q = ((words[:, :, None] >> shift) & np.uint32(2**bits - 1)).reshape(n, -1, group).astype(np.float64)
    v = (f64(scales)[:, :, None] * q + f64(biases)[:, :, None]).astype(np.float32).reshape(n, -1)
    return f64(torch.from_numpy(v).to(torch.bfloat16))


def lora(x, wd, lora_a, lora_b, lora_scale, adapters):
    """(y, base, mag): the exact result, the projection alone, and the sum of the magnitudes of all terms."""
    x, lora_a, lora_b, lora_scale = (f64(t) for t in (x, lora_a, lora_b, lora_scale))
    ids = adapters.cpu().numpy()
    base = x @ wd.T
    y, mag = base.copy(), np.abs(x) @ np.abs(wd).T
    for a in range(lora_a.shape[0]):
        rows = ids == a
        y[rows] += lora_scale[a] * ((x[rows] @ lora_a[a].T) @ lora_b[a].T)
        mag[rows] += abs(lora_scale[a]) * ((np.abs(x[rows]) @ np.abs(lora_a[a]).T) @ np.abs(lora_b[a]).T)
    return y, base, mag


def rope(x, weight, eps, positions, inv_freq, interleaved):
    """(o, mag): heads x [M, H, D] normed and rotated, and the magnitude of each value's terms."""
    x, weight, freq = f64(x), f64(weight), f64(inv_freq)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    p = len(freq)
    i = np.arange(p)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + p)
    angle = positions.cpu().numpy().astype(np.float64)[:, None, None] * freq
    a, b = n[..., first], n[..., second]
    o, mag = n.copy(), np.abs(n)
    o[..., first], o[..., second] = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    mag[..., first] = mag[..., second] = np.abs(a) + np.abs(b)
    return o, mag


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability) of one row of float64 logits."""
    l = np.where(np.isnan(logits), -np.inf, logits)
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if len(order) == 0:
        return -1, -np.inf
    if not temperature > 0:
        return int(order[0]), 0.0
    v = l[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / temperature))
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        before = np.cumsum(w) - w
        w = w[:max(1, int((before < top_p * w.sum()).sum()))]
    if min_p > 0:
        w = w[:max(1, int((w >= min_p).sum()))]
    cum = np.cumsum(w)
    at = min(int((cum <= u * cum[-1]).sum()), int((w > 0).sum()) - 1)
    return int(order[at]), float(np.log(w[at] / cum[-1]))


def sample(logits, uniform, **settings):
    logits, uniform = f64(logits), f64(uniform)
    rows = [{k: (v[i].item() if isinstance(v, torch.Tensor) else float(np.float32(v)) if k != "top_k" else v)
             for k, v in settings.items()} for i in range(len(logits))]
    out = [sample_row(l, u, **r) for l, u, r in zip(logits, uniform, rows)]
    return np.array([t for t, _ in out], np.int64), np.array([p for _, p in out])
