"""The oracle of the paged-attention tests, checked on the CPU: its rounding bounds against the formats, its attention
against torch's in double precision, its rotation against complex multiplication."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as AO  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rounding_bound_holds_and_is_tight(dtype):
    g = torch.Generator().manual_seed(0)
    y = torch.randn(1 << 18, generator=g, dtype=torch.float64) * torch.logspace(-8, 2, 1 << 18, dtype=torch.float64)
    err = (y.to(dtype).double() - y).abs()
    ratio = err / AO.rounding(y, dtype)
    assert ratio.max() <= 1.0 and ratio.max() > 0.95


def test_attention_matches_torch_in_double():
    g = torch.Generator().manual_seed(1)
    n, rows, kv, group, D = 37, 9, 2, 3, 64
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((rows, kv * group, D), (kv, n, D), (kv, n, D)))
    y, bound, lse, _ = AO.attention(q, k, v, n - rows, 0.2, 0.0, 0, 0.0)
    mask = torch.ones(rows, n, dtype=torch.bool).tril(n - rows)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), k.repeat_interleave(group, 0),
                                                            v.repeat_interleave(group, 0), attn_mask=mask, scale=0.2)
    assert torch.allclose(y, want.transpose(0, 1), atol=1e-12)
    assert (bound > 0).all() and torch.isfinite(lse).all()


def test_attention_window_cap_and_rows_before_the_cache():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((4, 1, 8), (1, 2, 8), (1, 2, 8)))
    y, _, lse, _ = AO.attention(q, k, v, -2, 1.0, 0.5, 1, 0.0)  # rows at positions -2 .. 1, each seeing one key at most
    assert not y[:2].any() and torch.isneginf(lse[:2]).all()
    assert torch.allclose(y[2:, 0], v[0])
    x = torch.stack([q[2 + i, 0] @ k[0, i] for i in range(2)])
    assert torch.allclose(lse[2:, 0], 0.5 * torch.tanh(x / 0.5))


@pytest.mark.parametrize("adjacent", [False, True])
def test_rotation_is_complex_multiplication(adjacent):
    g = torch.Generator().manual_seed(3)
    T, D, r = 5, 32, 16
    x = torch.randn((T, 2, D), generator=g, dtype=torch.float64)
    angle = torch.rand((9, r // 2), generator=g, dtype=torch.float64) * 6
    table = torch.stack([angle.cos(), angle.sin()], -1)
    pos = torch.randint(0, 9, (3, T), generator=g)
    y, _ = AO.append(x, None, 0.0, table, pos, (2, 3, 3), r, adjacent)
    turn = torch.cat([angle[pos[0]][:, :2], angle[pos[1]][:, 2:5], angle[pos[2]][:, 5:]], 1)
    pairs = x[..., :r].reshape(T, 2, r // 2, 2) if adjacent else x[..., :r].reshape(T, 2, 2, r // 2).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(turn), turn)[:, None]
    back = torch.view_as_real(z)
    back = back.reshape(T, 2, r) if adjacent else back.transpose(-1, -2).reshape(T, 2, r)
    assert torch.allclose(y[..., :r], back) and torch.equal(y[..., r:], x[..., r:])


def test_norm_is_unit_rms():
    g = torch.Generator().manual_seed(4)
    x = torch.randn((3, 2, 64), generator=g, dtype=torch.float64)
    y, e = AO.append(x, torch.ones(64, dtype=torch.float64), 0.0, None, None, (), 0, False)
    assert torch.allclose((y * y).mean(-1), torch.ones(3, 2, dtype=torch.float64)) and (e >= 0).all()
    assert math.isclose(float(e.max() / y.abs().max()), (64 + 8) * AO.E)
