"""Edges of the paged-attention operators on the GPU: tails of small weights, infinities, padding rows, plans that do not fit."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.fixture(scope="module")
def M():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import moe_b200
    return moe_b200


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def one_sequence(n, kv_heads, D, page, dtype):
    """Pools of zeros that hold one sequence in order, and its page table."""
    pages = -(-n // page)
    pools = [torch.zeros((pages, kv_heads, page, D), dtype=dtype, device="cuda") for _ in range(2)]
    return pools[0], pools[1], torch.arange(pages, dtype=torch.int32, device="cuda")[None]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_a_long_flat_tail_behind_a_score_without_a_value(M, dtype, D, op):
    """The first key scores 17.5 above all others and has the value 0 (a first token that collects attention), the others 1: the
    output is the tail's share of the weights, t / (1 + t) with t = (n - 1) e^-17.5, 1% (decode) or 0.3%, each weight below f16's
    smallest value. Many sequences, so that one stream of keys meets the first and much of the tail.
    Bound, relative: the output's rounding; the weights' rounding (bf16: u; f16 in two parts 2^-20, in one, scaled by 2^11 to
    5.1e-5 or more, 2^-25 / 5.1e-5); n / 16 additions of equal values, and as many to the sum, 2^-24 each."""
    B, n, kv = (40, 400000, 8) if op == "decode" else (300, 131071, 1)
    k, v, table = one_sequence(n, kv, D, 128, dtype)
    k[0, :, 0, 0] = 1.0
    v.fill_(1.0)
    v[0, :, 0] = 0.0
    q = torch.zeros((B, kv, D), dtype=dtype, device="cuda")
    q[..., 0] = 17.5
    att = M.PagedAttention(M.AttentionConfig(kv, kv, D, scale=1.0), k, v, max_seqs=B)
    lens, table = i32([n] * B), table.expand(B, -1).contiguous()
    if op == "decode":
        y, lse = att.decode(q, lens, table, return_lse=True)
    else:
        y, lse = att.prefill(q, i32(list(range(B + 1))), lens, table, return_lse=True)
    att.check()
    t = (n - 1) * math.exp(-17.5)
    weights = U[dtype] if dtype == BF16 else 2.0 ** -20 if op == "decode" else 2.0 ** -25 / 5.1e-5
    adds = n / 16 * 2.0 ** -24
    off = (y.double() * (1 + t) / t - 1).abs().max()
    assert off <= U[dtype] + weights + 2 * adds, off
    assert (lse.double() - (17.5 + math.log1p(t))).abs().max() <= adds + 2.0 ** -18
