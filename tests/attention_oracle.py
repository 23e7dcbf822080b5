"""The paged-attention operators' definitions in double precision, and the error bounds of the kernels' arithmetic.

Bounds, derived from the formats and the order of operations (u: the largest relative error of rounding to the output
type, 2^-8 for bf16's 8 and 2^-11 for f16's 11 significant bits, with half the smallest subnormal, 2^-25 for f16, as a
floor; e = 2^-24 the same for f32; n: keys of a row; tests/test_attention_oracle.py checks u against the formats):
  * scores: head_dim products and sums in f32, a scaling, and for capped scores a tanh evaluated to about 2^-21:
    dx = (head_dim + 4) e * max_j sum_d |q_d k_jd| * scale + 2^-21 * (1 + max_j |x_j| + softcap); a weight is off by a
    factor of 1 + 2 dx at most (its own score and the maximum's), plus 2^-21 for the exponential;
  * the sum of weights and the weighted values: n + 8 f32 additions each;
  * weights rounded for the second product: prefill u relative, decode (two parts) u^2 * 4; f16 has in addition an
    absolute floor of 2^-25 per weight (subnormals) against a sum of weights of at least 1 (prefill: reference up to
    2^8 below the maximum, so the floor only shrinks);
  * the output's own rounding: u |y|.
  |y - y*| <= u |y*| + (w + 4 dx + 2^-20 + 2 (n + 8) e) * sum_j p_j |v_j| + [f16] n 2^-25 max |v|
  |lse - lse*| <= 2 dx + 2^-20 + (n + 8) e + 4 e |lse*|
"""
import math

import numpy as np
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
E = 2.0 ** -24


def rounding(y, dtype):
    """The largest error of rounding each y to dtype."""
    return U[dtype] * y.abs() + FLOOR[dtype]


def gathered(pool, pages, n):
    """[heads, n, D] f64 of the first n tokens of a sequence's pages."""
    page, D = pool.shape[2], pool.shape[3]
    ids = pages[:-(-n // page)].long().cpu()
    return pool[ids.to(pool.device)].double().cpu().transpose(0, 1).reshape(pool.shape[1], -1, D)[:, :n]


def attention(q, k, v, first, scale, softcap, window, weight_error):
    """q [rows, heads, D] at positions first.., k and v [kv_heads, n, D] (f64): y, its bound, lse, its bound."""
    rows, heads, D = q.shape
    n, group = k.shape[1], heads // k.shape[0]
    y, yb = torch.zeros_like(q), torch.zeros_like(q)
    lse, lb = torch.full((rows, heads), -math.inf, dtype=torch.float64), torch.zeros((rows, heads), dtype=torch.float64)
    pos = first + torch.arange(rows)[:, None]
    key = torch.arange(n)[None]
    seen = key <= pos
    if window:
        seen = seen & (key > pos - window)
    for h in range(heads):
        kk, vv = k[h // group], v[h // group]
        x = (q[:, h] @ kk.t()) * scale
        mag = (q[:, h].abs() @ kk.abs().t()) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        x = x.masked_fill(~seen, -math.inf)
        any_ = seen.any(1)
        m = torch.where(any_, x.amax(1), torch.zeros(rows, dtype=torch.float64))
        p = torch.exp(x - m[:, None])
        s = p.sum(1)
        safe = torch.where(any_, s, torch.ones_like(s))
        w = p / safe[:, None]
        y[:, h] = w @ vv
        lse[:, h] = torch.where(any_, m + torch.log(safe), torch.full_like(m, -math.inf))
        top = (mag * seen).amax(1) if n else torch.zeros(rows, dtype=torch.float64)
        big = torch.where(seen, x.abs(), torch.zeros_like(x)).amax(1)
        dx = (D + 4) * E * top + 2.0 ** -21 * (1 + big + softcap)
        cnt = seen.sum(1).double()
        yb[:, h] = (weight_error + 4 * dx + 2.0 ** -20 + 2 * (cnt + 8) * E)[:, None] * (w @ vv.abs())
        lb[:, h] = 2 * dx + 2.0 ** -20 + (cnt + 8) * E + 4 * E * torch.where(any_, lse[:, h].abs(), torch.zeros_like(m))
    return y, yb, lse, lb


def run(q, k_pool, v_pool, table, lens, cu, scale, softcap, window, weight_error):
    """Every sequence: the rows cu[b]..cu[b + 1] - 1 of q at its last positions."""
    qd = q.double().cpu()
    y, yb = torch.zeros_like(qd), torch.zeros_like(qd)
    lse = torch.full(qd.shape[:2], -math.inf, dtype=torch.float64)
    lb = torch.zeros(qd.shape[:2], dtype=torch.float64)
    for b, n in enumerate(lens):
        a, z = cu[b], cu[b + 1]
        if n <= 0 or z <= a:
            continue
        k, v = gathered(k_pool, table[b], n), gathered(v_pool, table[b], n)
        y[a:z], yb[a:z], lse[a:z], lb[a:z] = attention(qd[a:z], k, v, n - (z - a), scale, softcap, window, weight_error)
        if q.dtype == torch.float16:
            yb[a:z] += n * 2.0 ** -25 * v.abs().max()
    return y, yb + rounding(y, q.dtype), lse, lb


def assert_within(got, want, bound, what):
    got, want, bound = got.double().cpu().numpy(), want.numpy(), bound.numpy()
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite], want[~finite]), f"{what}: -inf rows differ"
    err = np.abs(got[finite] - want[finite])
    assert np.isfinite(got[finite]).all(), f"{what}: not finite"
    over = err > bound[finite]
    assert not over.any(), f"{what}: {over.sum()} of {over.size} off by up to {np.max(err / np.maximum(bound[finite], 1e-300)):.2f} bounds"


def append(x, norm, eps, table, positions, sections, rope_dim, adjacent):
    """One of q / k: [T, heads, D] values after norm and rotation, and the bound of their f32 evaluation."""
    x = x.double().cpu().clone()
    T, heads, D = x.shape
    e = torch.zeros_like(x)
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double().cpu()
        e = (D + 8) * E * x.abs()
    if rope_dim:
        half = rope_dim // 2
        axis = torch.tensor(sum(([a] * n for a, n in enumerate(sections)), []))
        cs = table.double().cpu()[positions.cpu().long()[axis].t(), torch.arange(half)]
        c, s = cs[..., 0][:, None], cs[..., 1][:, None]
        i = torch.arange(half)
        ia, ib = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        a, b = x[..., ia].clone(), x[..., ib].clone()
        ea, eb = e[..., ia].clone(), e[..., ib].clone()
        mag = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
        x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
        e[..., ia] = ea * c.abs() + eb * s.abs() + 4 * E * mag[0]
        e[..., ib] = eb * c.abs() + ea * s.abs() + 4 * E * mag[1]
    return x, e
