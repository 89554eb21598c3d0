"""Inputs and the bound of the adapters' GPU tests at sizes whose 64-bit reference is computed on the GPU, some columns
at a time. The weights' exact values come from `dequantize`, whose bits have tests of their own."""

import torch

from mlx_tree_spec_amd import dequantize

DEV = "cuda:0"
HALF_STEP_BF16 = 2.0 ** -8
HALF_STEP_F32 = 2.0 ** -24


def inputs(m, k, n, rank, count, seed, ids=None):
    """x, w, scales, biases, lora_a, lora_b, lora_scale, adapters of a 4-bit projection in groups of 64."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    w = torch.randint(-2**31, 2**31, (n, k // 8), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    s = (randn(n, k // 64).abs() * 0.004 + 1e-4).bfloat16()
    b = (-8 * s.float() + randn(n, k // 64) * 1e-3).bfloat16()
    if ids is None:
        ids = torch.randint(-1, count, (m,), generator=g, device=DEV)
    return [randn(m, k).bfloat16(), w, s, b, (randn(count, rank, k) / k ** 0.5).bfloat16(),
            (randn(count, n, rank) * 0.3).bfloat16(), torch.rand(count, generator=g, device=DEV) * 3 - 1.5,
            torch.as_tensor(ids).to(device=DEV, dtype=torch.int32)]


def check(args, y):
    """The bound of test_gpu_lora.py: the result rounded to bf16 (half a step, and a hundredth for the value that is
    rounded being off already), t = x A^T kept to 2^-18, and fp32 sums of K + R + 4 terms, each off by at most half a
    step of the magnitudes' sum."""
    x, w, s, b, la, lb, scale, ids = args
    m, k, n, rank = x.shape[0], x.shape[1], w.shape[0], la.shape[1]
    assert y.shape == (m, n) and y.dtype == torch.bfloat16
    xd = x.double()
    used = [a for a in ids.unique().tolist() if 0 <= a < la.shape[0]]
    rows = {a: ids == a for a in used}
    t, tm = {}, {}
    for a in used:
        at = la[a].double().T.contiguous()
        t[a], tm[a] = scale[a].double() * (xd[rows[a]] @ at), scale[a].double().abs() * (xd[rows[a]].abs() @ at.abs())
    step = 1 << 14
    for c in range(0, n, step):
        wd = dequantize(w[c:c + step], s[c:c + step], b[c:c + step]).double().T.contiguous()
        ref, mag = xd @ wd, xd.abs() @ wd.abs()
        for a in used:
            bt = lb[a, c:c + step].double().T.contiguous()
            ref[rows[a]] += t[a] @ bt
            mag[rows[a]] += tm[a] @ bt.abs()
        bound = HALF_STEP_BF16 * ref.abs() * 1.01 + ((k + rank + 4) * HALF_STEP_F32 + 2.0 ** -18) * mag
        over = (y[:, c:c + step].double() - ref).abs() - bound
        assert not over.isnan().any()
        at = int(over.argmax())
        assert over.max().item() <= 0, (over.max().item(), at // over.shape[1], c + at % over.shape[1])
