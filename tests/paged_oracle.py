"""Paged attention, appends and rotary positions in 64 bits on the CPU, with bounds on what the kernels'
roundings may change (test infrastructure only)."""

from __future__ import annotations

import math

import torch


def attention(q, k_pages, v_pages, table, new, keys, *, window=(-1, -1), causal=True, scale=None):
    """(out, bound) in float64 of q [T, Hq, D]; only allowed keys are touched, row by row.

    The bound, per element, with w the weights and A = sum_j w_j |v_j|:
    - probabilities are rounded to bf16 (half a step: 2^-8 relative) in numerator and normaliser alike, so
      out' = sum w_j (1 + e_j) v_j / sum w_j (1 + e_j), |out' - out| <= 2 * 2^-8 * A / (1 - 2^-8);
    - a score is an fp32 sum of D products, times the scale, in base 2, then an exponential of 1 ulp: off by
      at most 2^-24 * (D + 4) * scale * sum |q_i k_i|, which moves w_j by that factor: twice it, times A;
    - fp32 sums over n keys, pairwise or in order: 2^-24 * 2 n A;
    - the output's rounding: 2^-8 |out|."""
    T, hq, d = q.shape
    n_pages, page, hkv, _ = k_pages.shape
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    left, right = window
    if causal:
        right = 0
    first = 0
    for s, (n, lk) in enumerate(zip(new, keys)):
        pages = table[s].tolist()
        for r in range(n):
            at = lk - n + r
            lo = max(0, at - left) if left >= 0 else 0
            hi = min(lk, at + right + 1) if right >= 0 else lk
            places = [(pages[j // page], j % page) for j in range(lo, hi) if 0 <= pages[j // page] < n_pages]
            if not places:
                continue
            pg, slot = (torch.tensor(x) for x in zip(*places))
            k = k_pages[pg, slot].double().repeat_interleave(group, 1)  # [keys, hq, d]
            v = v_pages[pg, slot].double().repeat_interleave(group, 1)
            qr = q[first + r].double()
            scores = (k * qr).sum(-1) * scale  # [keys, hq]
            w = torch.softmax(scores, 0)
            o = (w[..., None] * v).sum(0)
            a = (w[..., None] * v.abs()).sum(0)
            score_error = 2.0 ** -24 * (d + 4) * scale * (k * qr).abs().sum(-1).amax(0)
            out[first + r] = o
            bound[first + r] = a * (2.0 ** -7 / (1 - 2.0 ** -8) + 2 * score_error[:, None]
                                    + 2.0 ** -23 * len(places)) + 2.0 ** -8 * o.abs() + 1e-30
        first += n
    return out, bound


def rotate(x, positions, inv_freq, *, interleaved=False, scale=1.0, inverse=False):
    """(out, bound) in float64 of x [T, H, D]: each pair as a complex number times scale * exp(i angle).

    The bound, per element, of a pair (a, b): the reduced angle is off by at most 2.4e-8 (quarter turns in
    fp32) + 3e-8 (its product with pi / 2), the series by 3e-9 and its fp32 steps by 4e-8, the product with
    the scale by 2^-24: below 1.8e-7 on sine and cosine together with their rounding; the products and the
    sum round twice more (2^-24 each). 4e-7 * scale * (|a| + |b|) covers them; the output rounds by half a
    step."""
    r = inv_freq.numel()
    xd = x.double()
    angle = positions.double().view(-1, 1, 1) * inv_freq.double()
    if inverse:
        angle = -angle
    if interleaved:
        a, b = xd[..., 0:2 * r:2], xd[..., 1:2 * r:2]
    else:
        a, b = xd[..., :r], xd[..., r:2 * r]
    z = torch.complex(a, b) * torch.polar(torch.full_like(angle, float(scale)), angle)
    size = (a.abs() + b.abs()) * (4e-7 * abs(scale))
    out, slack = xd.clone(), torch.zeros_like(xd)
    if interleaved:
        out[..., 0:2 * r:2], out[..., 1:2 * r:2] = z.real, z.imag
        slack[..., 0:2 * r:2] = slack[..., 1:2 * r:2] = size
    else:
        out[..., :r], out[..., r:2 * r] = z.real, z.imag
        slack[..., :r] = slack[..., r:2 * r] = size
    half_step = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # subnormal results round absolutely
    return out, slack + half_step * out.abs() * (1 + 1e-6) + half_step * slack + tiny


def assert_within(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    over = (got - want).abs() - bound
    worst = int(over.argmax())
    assert over.max() <= 0, (f"{what}: {float(got.flatten()[worst])} for {float(want.flatten()[worst])}, bound "
                             f"{float(bound.flatten()[worst])} at {worst}, {int((over > 0).sum())} values")


def layout(keys, page, gen, spare=3, columns=None):
    """A random page table [n_seq, columns] for sequences of `keys` tokens and its number of pages."""
    used = [math.ceil(k / page) for k in keys]
    n_pages = sum(used) + spare
    order = torch.randperm(n_pages, generator=gen).tolist()
    columns = max([1, *used]) if columns is None else columns
    table = torch.full((len(keys), columns), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, n_pages


def bounds(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32)
