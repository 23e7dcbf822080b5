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


# ---- rows that no sequence holds ----------------------------------------------------------------------


def prompt(M, lens, heads=4, kv=2, D=64, dtype=BF16, page=16):
    """A handle over random pools, the query rows and the arguments of a prefill of whole prompts."""
    g = torch.Generator(device="cuda").manual_seed(5)
    pages = [-(-n // page) for n in lens]
    shape = (sum(pages) + 1, kv, page, D)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    table = torch.zeros((len(lens), max(pages, default=1) or 1), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    q = torch.randn((sum(lens), heads, D), generator=g, device="cuda").to(dtype)
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return M.PagedAttention(M.AttentionConfig(heads, kv, D), k, v, max_seqs=8), q, cu, table.cuda()


def refused(M, att):
    with pytest.raises(M.MoeError) as e:
        att.check()
    assert e.value.status == 5, e.value


def filled(q, rows):
    """Outputs of `rows` rows that hold something else before the call."""
    return (torch.full((rows,) + q.shape[1:], 7.0, dtype=q.dtype, device="cuda"),
            torch.full((rows, q.shape[1]), 7.0, device="cuda"))


@pytest.mark.parametrize("D,pad", [(64, 1), (128, 37), (64, 700)])
def test_prefill_padding_rows_are_zero(M, D, pad):
    lens = [5, 0, 70, 129]
    att, q, cu, table = prompt(M, lens, D=D)
    want, wl = att.prefill(q, i32(cu), i32(lens), table, return_lse=True)
    wide = torch.cat([q, torch.full((pad,) + q.shape[1:], float("nan"), dtype=q.dtype, device="cuda")])
    y, lse = filled(q, len(wide))
    att.prefill(wide, i32(cu), i32(lens), table, out=y, lse=lse)
    att.check()
    n = len(q)
    assert torch.equal(y[:n], want) and torch.equal(lse[:n], wl)
    assert not y[n:].any() and torch.isneginf(lse[n:]).all()


def test_prefill_graph_of_the_largest_batch_serves_smaller_ones(M):
    lens = [40, 90, 17]
    att, q, cu, table = prompt(M, lens)
    want = att.prefill(q, i32(cu), i32(lens), table)
    c, n = i32(cu), i32(lens)
    y, lse = filled(q, len(q))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.prefill(q, c, n, table, out=y, lse=lse)
    for live in (3, 1, 0, 2):
        y.fill_(7.0), lse.fill_(7.0)
        c.copy_(i32([cu[min(i, live)] for i in range(4)])), n.copy_(i32(lens[:live] + [0] * (3 - live)))
        graph.replay()
        att.check()
        rows = cu[live]
        assert torch.equal(y[:rows], want[:rows]) and not y[rows:].any()
        assert torch.isfinite(lse[:rows]).all() and torch.isneginf(lse[rows:]).all()


def test_prefill_without_a_sequence(M):
    att, q, _, table = prompt(M, [33])
    y, lse = filled(q, len(q))
    att.prefill(q, i32([0]), i32([]), table[:0], out=y, lse=lse)
    att.check()
    assert not y.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("cu", [[2, 5, 20], [0, 25, 20], [0, 8, 21], [-1, 8, 20], [0, 30, 20]])
def test_prefill_reports_row_offsets_that_do_not_fit(M, cu):
    att, q, _, table = prompt(M, [12, 8])
    y, lse = filled(q, len(q))
    att.prefill(q, i32(cu), i32([64, 64]), table.repeat(1, 4), out=y, lse=lse)
    refused(M, att)
    first = max(cu[0], 0)
    assert not y[:first].any() and torch.isneginf(lse[:first]).all() and torch.isfinite(lse[first:]).all()
    att.check()


# ---- waits that run out -------------------------------------------------------------------------------


@pytest.mark.parametrize("lens,heads,kv,D", [([700, 300], 8, 2, 128), ([3, 1500], 4, 4, 64), ([4000], 2, 2, 128)])
def test_prefill_waits_that_run_out_are_reported(M, lens, heads, kv, D):
    """Limits from one clock (the first wait gives up) to about a call's length (some role in the middle of its work does): the
    call ends, says so, leaves the handle usable, and the next call gives the bits that it always gives."""
    from moe_b200 import _lib

    att, q, cu, table = prompt(M, lens, heads=heads, kv=kv, D=D)
    c, n = i32(cu), i32(lens)
    want = att.prefill(q, c, n, table)
    gave_up = []
    for limit in (1, 300, 1000, 2000, 4000, 6000, 8000, 10000, 14000, 20000, 40000):
        att.set_wait_limit(limit)
        y = att.prefill(q, c, n, table)
        still, _ = filled(q, len(q))
        att.prefill(q, c, n, table, out=still)  # behind a wait that ran out: nothing
        try:
            att.check()
        except M.MoeError as e:
            assert e.status == _lib.MOE_ERR_TIMEOUT
            gave_up.append(limit)
        else:
            assert torch.equal(y, want) and torch.equal(still, want)
        att.set_wait_limit(400_000_000)
        assert torch.equal(att.prefill(q, c, n, table), want)
        att.check()
    assert 1 in gave_up


def test_prefill_does_nothing_between_a_wait_that_ran_out_and_the_check(M):
    from moe_b200 import _lib

    att, q, cu, table = prompt(M, [200, 90])
    c, n = i32(cu), i32([200, 90])
    want = att.prefill(q, c, n, table)
    att.set_wait_limit(1)
    att.prefill(q, c, n, table)
    att.set_wait_limit(400_000_000)
    for _ in range(3):
        y, _ = filled(q, len(q))
        att.prefill(q, c, n, table, out=y)
        assert (y == 7.0).all()
    with pytest.raises(M.MoeError) as e:
        att.check()
    assert e.value.status == _lib.MOE_ERR_TIMEOUT
    assert torch.equal(att.prefill(q, c, n, table), want)
    att.check()


# ---- infinities and NaN among the values ---------------------------------------------------------------


def plain_row(q, k, v, scale):
    """One query row of one head over the keys it sees, in 64 bits."""
    p = torch.softmax((k.double() @ q.double()) * scale, 0)
    return p @ v.double()


def same_kind(got, want, bound):
    """NaN where the definition gives NaN, the same infinities, and finite values within the bound."""
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (got, want)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.isfinite(got[~inf & ~torch.isnan(want)]).all()
    ok = torch.isfinite(want)
    assert ((got - want)[ok].abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,D,n", [(2, 64, 1), (8, 128, 37), (24, 64, 300), (3, 128, 5000)])
def test_decode_infinite_and_nan_values_reach_what_sees_them(M, dtype, heads, D, n):
    """An infinite value gives an infinite output in its column and no other, a NaN value a NaN there; a NaN key makes the whole row NaN;
    values outside the window or past the length reach nothing. Scores within +-2, so every weight counts. Bound: u of
    the largest value and twice u of the weights (the definition's own scale), with |v| below 8."""
    inf, nan = math.inf, math.nan
    window = 200
    g = torch.Generator(device="cuda").manual_seed(2)
    for what in ("inf", "-inf", "both", "nan value", "nan key", "nan row", "outside"):
        k, v, table = one_sequence(n + 30, 1, D, 16, dtype)
        k.copy_(torch.randn(k.shape, generator=g, device="cuda") * 0.1), v.copy_(torch.randn(v.shape, generator=g, device="cuda"))
        v.clamp_(-7, 7)
        q = torch.randn((1, heads, D), generator=g, device="cuda").clamp_(-3, 3).to(dtype)
        at = n - 1 - min(n, window) // 3
        if what in ("inf", "both"):
            v[at // 16, 0, at % 16, 3] = inf
        if what == "-inf":
            v[at // 16, 0, at % 16, 3] = -inf
        if what == "both" and n > 1:
            v[(n - 1) // 16, 0, (n - 1) % 16, 3] = -inf
        if what == "nan value":
            v[at // 16, 0, at % 16, 5] = nan
        if what == "nan key":
            k[at // 16, 0, at % 16, 5] = nan
        if what == "nan row":
            q[0, 1, 7] = nan
        for past in range(n, n + 30):
            k[past // 16, 0, past % 16], v[past // 16, 0, past % 16] = (nan, inf) if past % 2 else (inf, nan)
        if what == "outside" and n > window:
            v[0, 0, 0], k[0, 0, 0] = nan, nan
        att = M.PagedAttention(M.AttentionConfig(heads, 1, D, window=window), k, v, max_seqs=1)
        y = att.decode(q, i32([n]), table)
        att.check()
        rows = slice(max(0, n - window), n)
        ks, vs = (p.transpose(1, 2).reshape(-1, D)[rows] for p in (k, v))
        for h in range(heads):
            same_kind(y[0, h], plain_row(q[0, h], ks, vs, D ** -0.5), 8 * 3 * U[dtype])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_infinite_and_nan_values_reach_the_rows_that_see_them(M, dtype):
    """Rows from the value's position on: as decode. Other columns, other heads' values and other sequences: untouched."""
    lens, D = [150, 90], 128
    att, q, cu, table = prompt(M, lens, heads=4, kv=2, D=D, dtype=dtype)
    c, n = i32(cu), i32(lens)
    clean = att.prefill(q, c, n, table)
    k, v = att._keep[0], att._keep[1]
    at, page = 70, int(table[0, 70 // 16])
    for bad in (math.inf, -math.inf, math.nan):
        keep = v[page, 1, at % 16, 9].clone()
        v[page, 1, at % 16, 9] = bad
        y = att.prefill(q, c, n, table)
        att.check()
        v[page, 1, at % 16, 9] = keep
        seen = y[at:150, 2:, 9].float()  # the heads of key/value head 1
        assert torch.isnan(seen).all() if math.isnan(bad) else (seen == bad).all()
        y[:150, 2:, 9] = clean[:150, 2:, 9]
        assert torch.equal(y, clean)
    keep = k[page, 1, at % 16, 9].clone()
    k[page, 1, at % 16, 9] = math.nan
    y = att.prefill(q, c, n, table)
    k[page, 1, at % 16, 9] = keep
    assert torch.isnan(y[at:150, 2:]).all()
    y[at:150, 2:] = clean[at:150, 2:]
    assert torch.equal(y, clean)
    att.check()


# ---- large caps ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("softcap", [60.0, 70.0, 1000.0, 1e5, 1e30, 3e38])
@pytest.mark.parametrize("size", [1.5, 60.0])
def test_large_caps(M, dtype, softcap, size):
    """A cap far above the scores leaves them as they are, and one near them bends them exactly, however large it is: the bound
    is that of uncapped scores (tests/attention_oracle.py), plus the formula's 2^-21 of the cap up to 64 and 2^-21 of the score
    above, twice per weight."""
    import attention_oracle as AO

    lens, heads, kv, D = [130, 77], 4, 2, 64
    att, q, cu, table = prompt(M, lens, heads=heads, kv=kv, D=D, dtype=dtype)
    k, v = att._keep[0], att._keep[1]
    q = (q * size).to(dtype)
    att = M.PagedAttention(M.AttentionConfig(heads, kv, D, softcap=softcap), k, v, max_seqs=2)
    y, lse = att.prefill(q, i32(cu), i32(lens), table, return_lse=True)
    last = torch.tensor([c - 1 for c in cu[1:]], device="cuda")
    z, zl = att.decode(q[last].contiguous(), i32(lens), table, return_lse=True)
    att.check()
    # a cap whose f64 tanh is its argument to the last bit: the oracle's softcap * tanh(x / softcap) is exact enough at 1e30
    want = AO.run(q, k, v, table, lens, cu, 1 / math.sqrt(D), softcap, 0, AO.U[dtype])
    loose = AO.run(q, k, v, table, lens, cu, 1 / math.sqrt(D), 0.0, 0, AO.U[dtype])
    extra = 2.0 ** -21 * min(softcap, 64.0) if softcap <= 64 else 0.0
    vmax = v.double().abs().max().item()
    yb, lb = loose[1] + 4 * extra * vmax + 2 * AO.U[dtype] * vmax, loose[3] + 2 * extra
    AO.assert_within(y, want[0], yb, "prefill")
    AO.assert_within(lse, want[2], lb, "prefill lse")
    AO.assert_within(z, want[0][last.cpu()], yb[last.cpu()], "decode")
    AO.assert_within(zl, want[2][last.cpu()], lb[last.cpu()], "decode lse")


# ---- pages behind the window ----------------------------------------------------------------------------


@pytest.mark.parametrize("D,page,window", [(64, 16, 40), (128, 16, 1), (128, 32, 200), (64, 64, 130), (128, 128, 300)])
@pytest.mark.parametrize("entry", ["none", "reused"])
def test_pages_behind_the_window_are_not_read(M, D, page, window, entry):
    """A cache that frees pages behind the window: their table entries name nothing, or pages that hold something else (NaN and
    infinities here). The rows' outputs are those of the full cache, bit for bit."""
    heads, kv, rows, lens = 4, 2, [70, 3, 200], [900, 513, 640]
    g = torch.Generator(device="cuda").manual_seed(8)
    need = [-(-n // page) for n in lens]
    shape = (sum(need) + 1, kv, page, D)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(BF16) for _ in range(2))
    k[-1], v[-1] = math.inf, math.nan
    table = torch.zeros((3, max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    cut = table.clone()
    for b in range(3):
        first = max(0, lens[b] - rows[b] - window + 1)  # of the chunk's first row
        cut[b, :first // page] = -1 if entry == "none" else shape[0] - 1
    cu = [0, 70, 73, 273]
    q = torch.randn((273, heads, D), generator=g, device="cuda").to(BF16)
    att = M.PagedAttention(M.AttentionConfig(heads, kv, D, window=window), k, v, max_seqs=3)
    want = att.prefill(q, i32(cu), i32(lens), table.cuda(), return_lse=True)
    got = att.prefill(q, i32(cu), i32(lens), cut.cuda(), return_lse=True)
    att.check()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    last = q[torch.tensor([69, 72, 272], device="cuda")].contiguous()
    assert torch.equal(att.decode(last, i32(lens), cut.cuda()), att.decode(last, i32(lens), table.cuda()))
    att.check()


# ---- the smallest table, the largest window --------------------------------------------------------------


def test_an_empty_page_table_serves_empty_sequences(M):
    """No sequence has a page yet: zeros and -inf, as for a sequence of length 0 in a larger table; a length that the table does
    not hold is reported."""
    att, q, _, table = prompt(M, [5])
    none = table.new_empty((3, 0))
    y, lse = filled(q, 3)
    att.decode(q[:3], i32([0, 0, 0]), none, out=y, lse=lse)
    att.check()
    assert not y.any() and torch.isneginf(lse).all()
    y, lse = filled(q, len(q))
    att.prefill(q, i32([0, 0, 0, 0]), i32([0, 0, 0]), none, out=y, lse=lse)
    att.check()
    assert not y.any() and torch.isneginf(lse).all()
    y, _ = filled(q, 3)
    att.decode(q[:3], i32([0, 1, 0]), none, out=y)
    refused(M, att)
    assert not y.any()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 200, 2 ** 30])
def test_a_window_longer_than_any_sequence_is_none(M, window):
    """Bit for bit: few long items are cut along their keys, and the cut follows from the window."""
    lens = [4000, 129]
    att, q, cu, table = prompt(M, lens, D=128)
    other = M.PagedAttention(M.AttentionConfig(4, 2, 128, window=window), att._keep[0], att._keep[1], max_seqs=2)
    args = (i32(cu), i32(lens), table)
    assert torch.equal(other.prefill(q, *args), att.prefill(q, *args))
    last = q[[c - 1 for c in cu[1:]]].contiguous()
    assert torch.equal(other.decode(last, *args[1:]), att.decode(last, *args[1:]))
    other.check()


# ---- further forms against the definition ----------------------------------------------------------------


@pytest.mark.parametrize("scale", [0.02, 0.5])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (20.0, 77)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_with_a_scale_of_its_own(M, scale, softcap, window, dtype):
    import attention_oracle as AO

    lens, D = [150, 301], 64
    att, q, cu, table = prompt(M, lens, heads=6, kv=2, D=D, dtype=dtype)
    k, v = att._keep[0], att._keep[1]
    att = M.PagedAttention(M.AttentionConfig(6, 2, D, scale=scale, softcap=softcap, window=window), k, v, max_seqs=2)
    y, lse = att.prefill(q, i32(cu), i32(lens), table, return_lse=True)
    att.check()
    want = AO.run(q, k, v, table, lens, cu, scale, softcap, window, AO.U[dtype])
    AO.assert_within(y, want[0], want[1], "y")
    AO.assert_within(lse, want[2], want[3], "lse")


@pytest.mark.parametrize("T,heads,kv,D,rope_dim,sections", [(31, 6, 2, 128, 64, (8, 12, 12)), (5, 3, 3, 64, 32, (1, 0, 15)),
                                                          (17, 5, 1, 128, 16, (3, 3, 2)), (9, 9, 3, 64, 48, ())])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_adjacent_pairs_of_part_of_a_head(M, T, heads, kv, D, rope_dim, sections, dtype):
    import test_paged_attention as A

    A.test_append_matches_definition(M, T, heads, kv, D, 16, dtype, rope_dim, "adjacent", sections, True)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_and_attention_each_within_its_bound(M, dtype):
    """A prompt in two chunks and a token: what append stores and returns against the definition, and the attention of those
    stored values (no rounding in between) against the definition."""
    import attention_oracle as AO

    heads, kv, D, page, n = 8, 2, 128, 16, 75
    g = torch.Generator(device="cuda").manual_seed(4)
    k_pool, v_pool = M.kv_pools(8, kv, page, D, dtype=dtype)
    k_pool.fill_(math.nan), v_pool.fill_(math.nan)
    table = i32([[6, 1, 3, 0, 7]])
    rope = M.rope_table(D, 100)
    norm = (1 + torch.randn(D, generator=g, device="cuda") * 0.1).to(dtype)
    att = M.PagedAttention(M.AttentionConfig(heads, kv, D, rope_dim=D), k_pool, v_pool, rope_table=rope, q_norm=norm, k_norm=norm)
    q, k, v = (torch.randn((n, h, D), generator=g, device="cuda").to(dtype) for h in (heads, kv, kv))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = M.page_slots(table, torch.zeros_like(pos), pos, page)
    outs, turned = [], []
    for a, z in ((0, 50), (50, 74), (74, 75)):
        turned.append(att.append(q[a:z], k[a:z], v[a:z], pos[a:z], slots[a:z]))
        outs.append(att.prefill(turned[-1], i32([0, z - a]), i32([z]), table) if z - a > 1 else
                    att.decode(turned[-1], i32([z]), table))
    att.check()
    turned = torch.cat(turned)
    for got, x in ((turned, q), (k_pool[slots // page, :, slots % page], k)):
        want, bound = AO.append(x, norm, 1e-6, rope, pos[None], (D // 2,), D, False)
        AO.assert_within(got, want, bound + AO.rounding(want, dtype), "append")
    want = AO.run(turned, k_pool.nan_to_num(0.0), v_pool.nan_to_num(0.0), table, [n], [0, n], 1 / math.sqrt(D), 0.0, 0, AO.U[dtype])
    AO.assert_within(torch.cat(outs), want[0], want[1], "attention")
