"""Oracle of the 8-bit paged KV cache (PyTorch).  TEST INFRASTRUCTURE ONLY.

No reference counterpart.  Tokens are given as a whole history; what the cache
stands for after ``n`` of them is: complete blocks of 64 quantised per (block,
head), the rest as they came.  The quantiser is restated in float32 in the
kernel's order (bit-exact); attention is float64.  Follows its inputs' device.
"""
from __future__ import annotations

import torch

BLOCK = 64
TOP = {"e4m3": 448.0, "int8": 127.0}


def quantize_blocks(x, codes):
    """x [..., 64, D] float16 / bfloat16 -> (codes as float32 [..., 64, D], scales float32 [...])."""
    x = x.float()
    amax = x.abs().amax((-2, -1))
    bad = ~torch.isfinite(x).all(-1).all(-1)
    # (torch divides by a Python number by multiplying with its reciprocal)
    scale = torch.clamp_min(amax / torch.full_like(amax, TOP[codes]), 2.0 ** -126)
    y = (x * (1.0 / scale)[..., None, None]).clamp(-TOP[codes], TOP[codes])
    c = y.to(torch.float8_e4m3fn).float() if codes == "e4m3" else torch.round(y)
    c = torch.where(bad[..., None, None], torch.zeros_like(c), c)
    return c, torch.where(bad, torch.full_like(scale, float("nan")), scale)


def held(x, n, codes):
    """What a cache holds of the first n tokens of x [Hkv, >= n, D], in float64."""
    full = n // BLOCK * BLOCK
    h, _, d = x.shape
    tail = x[:, full:n].double()
    tail = torch.where(torch.isfinite(tail), tail, torch.full_like(tail, float("nan")))
    if not full:
        return tail
    c, s = quantize_blocks(x[:, :full].reshape(h, full // BLOCK, BLOCK, d), codes)
    return torch.cat([(c.double() * s.double()[..., None, None]).reshape(h, full, d), tail], 1)


def seen(n, cnt, i, window=None, sink=4, device="cpu"):
    """Mask [n] of the positions that query row i of cnt sees in a sequence of n tokens."""
    limit = n - cnt + i + 1
    pos = torch.arange(n, device=device)
    m = pos < limit
    if window is not None:
        m &= (pos < sink) | (pos >= limit - window)
    return m


def attend(q, k, v, cnt, scale, window=None, sink=4):
    """One sequence: q [H, T, D], k / v [Hkv, n, D] float64 -> (o, spread, reach), all float64:
    o [H, T, D]; spread = softmax . |v| [H, T, D] and reach = max over seen tokens of sum |q||k| * scale
    [H, T, 1], from which error bounds are made.  Rows that see nothing, and rows i >= cnt, are 0."""
    hh, t, d = q.shape
    hkv, n, _ = k.shape
    q = q.double()
    o, spread = torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(hh, t, 1, dtype=torch.float64, device=q.device)
    for i in range(min(t, cnt)):
        m = seen(n, cnt, i, window, sink, q.device)
        if not bool(m.any()):
            continue
        qi = q[:, i].reshape(hkv, hh // hkv, d)
        ks, vs = k[:, m], v[:, m]
        p = torch.softmax(torch.einsum("gqd,gnd->gqn", qi, ks) * scale, -1)
        o[:, i] = torch.einsum("gqn,gnd->gqd", p, vs).reshape(hh, d)
        spread[:, i] = torch.einsum("gqn,gnd->gqd", p, vs.abs()).reshape(hh, d)
        reach[:, i] = (torch.einsum("gqd,gnd->gqn", qi.abs(), ks.abs()).amax(-1) * abs(scale)).reshape(hh, 1)
    return o, spread, reach


def bound(o, spread, reach, dtype, d):
    """How far a correct kernel may be from o, element by element.
    * the output's rounding: half a step, eps / 2 of its type;
    * a score is a sum of d products with float32 rounding (2^-24 each, some more for its scaling and exponential
      argument): d + 16 roundings of at most `reach`; softmax weights then move by at most twice that, relatively;
    * the exponential itself and the sums: 2^-20;
    * P in two fp16 parts (2^-22, or 2^-40 of the largest of the 32 weights that it is taken with: not in the bound, for
      scores that differ by less than 10), in two bfloat16 ones (2^-18) beside 16-bit tokens of bfloat16;
    * an element below the type's smallest normal number: its absolute step."""
    fi = torch.finfo(dtype)
    p_err = 2.0 ** -18 if dtype == torch.bfloat16 else 2.0 ** -22
    rel = 2 * (d + 16) * 2.0 ** -24 * reach + 2.0 ** -20 + p_err
    return fi.eps / 2 * o.abs() * (1 + 1e-3) + rel * spread * (1 + fi.eps) + fi.smallest_normal * fi.eps
