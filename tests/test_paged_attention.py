"""The paged-attention operators (moe_attn_*) on the GPU against their definitions in double precision
(tests/attention_oracle.py, which derives the bounds), and their refusals."""
import math

import pytest

import attention_oracle as AO

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def M():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import moe_b200
    return moe_b200


def randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def cache(seed, lens, kv_heads, D, page, dtype, junk=float("nan"), interleaved=False):
    """Pools whose pages lie anywhere and hold `junk` wherever no token lies, and the page table (-1 past a sequence)."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    shape = (total, kv_heads, page, D)
    if interleaved:
        both = torch.full((total, 2, kv_heads, page, D), junk, dtype=dtype, device="cuda")
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.full(shape, junk, dtype=dtype, device="cuda") for _ in range(2))
    kd, vd = randn(seed + 1, shape, dtype), randn(seed + 2, shape, dtype)
    at = 0
    for b, n in enumerate(lens):
        for i in range(need[b]):
            pg, rows = order[at], min(page, n - i * page)
            table[b, i] = pg
            k[pg, :, :rows], v[pg, :, :rows] = kd[pg, :, :rows], vd[pg, :, :rows]
            at += 1
    return k, v, table.cuda()


def handle(M, heads, kv_heads, D, k, v, max_seqs=8, **kw):
    return M.PagedAttention(M.AttentionConfig(num_heads=heads, num_kv_heads=kv_heads, head_dim=D, **kw), k, v,
                            max_seqs=max_seqs)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def clean(pool):
    return torch.nan_to_num(pool, nan=0.0)


# ---- decode ------------------------------------------------------------------------------------------

DECODE = [
    # lens, kv_heads, group, D, page, dtype, softcap, window
    ([1], 1, 1, 64, 16, BF16, 0.0, 0),
    ([0], 2, 4, 128, 16, BF16, 0.0, 0),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33], 4, 8, 128, 16, BF16, 0.0, 0),
    ([63, 64, 65, 0, 127, 128, 129], 2, 5, 64, 32, F16, 0.0, 0),
    ([700, 3, 1500], 4, 7, 128, 64, BF16, 25.0, 0),
    ([700, 3, 1500], 3, 3, 128, 128, F16, 25.0, 100),
    ([40, 41, 56, 57, 1, 0], 2, 8, 128, 16, BF16, 0.0, 1),
    ([40, 41, 56, 57, 1, 0], 2, 12, 64, 16, BF16, 0.0, 16),
    ([400, 41, 2000, 57, 1, 0], 1, 16, 128, 32, F16, 0.0, 17),
    ([333, 90], 2, 9, 128, 16, BF16, 0.0, 0),
    ([333, 90], 1, 20, 64, 16, F16, 0.0, 0),
    ([333, 90], 2, 33, 128, 16, BF16, 30.0, 77),
    ([30011], 1, 8, 128, 64, BF16, 0.0, 0),
    ([20001], 1, 1, 64, 128, F16, 0.0, 0),
    ([5, 9000, 1, 0, 4000], 2, 4, 64, 32, BF16, 0.0, 0),
]


@pytest.mark.parametrize("lens,kv_heads,group,D,page,dtype,softcap,window", DECODE)
@pytest.mark.parametrize("scale", [0.0, 0.3])
def test_decode_matches_definition(M, lens, kv_heads, group, D, page, dtype, softcap, window, scale):
    heads = kv_heads * group
    k, v, table = cache(len(lens) + D, lens, kv_heads, D, page, dtype)
    q = randn(5, (len(lens), heads, D), dtype, 1.5)
    att = handle(M, heads, kv_heads, D, k, v, max_seqs=len(lens), softcap=softcap, window=window, scale=scale)
    y, lse = att.decode(q, i32(lens), table, return_lse=True)
    again = att.decode(q, i32(lens), table)
    att.check()
    want = AO.run(q, clean(k), clean(v), table, lens, list(range(len(lens) + 1)), scale or 1 / math.sqrt(D), softcap, window,
                  4 * AO.U[dtype] ** 2)
    AO.assert_within(y, want[0], want[1], "y")
    AO.assert_within(lse, want[2], want[3], "lse")
    assert torch.equal(y, again), "two calls on the same inputs differ"


def test_decode_large_batch_and_back_to_back_calls(M):
    """More sequences than a CTA has threads, calls of other shapes between them, nothing waited for."""
    lens = [(i * 37) % 291 for i in range(300)]
    k, v, table = cache(3, lens, 2, 64, 16, BF16)
    q = randn(6, (300, 8, 64), BF16, 1.5)
    att = handle(M, 8, 2, 64, k, v, max_seqs=300)
    want = AO.run(q, clean(k), clean(v), table, lens, list(range(301)), 1 / 8, 0.0, 0, 4 * AO.U[BF16] ** 2)
    outs = []
    for _ in range(5):
        outs.append(att.decode(q, i32(lens), table))
        outs.append(att.decode(q[:7].contiguous(), i32(lens[:7]), table[:7].contiguous()))
    att.check()
    for i, y in enumerate(outs):
        n = y.shape[0]
        AO.assert_within(y, want[0][:n], want[1][:n], f"call {i}")


@pytest.mark.parametrize("lens,kv_heads,group,D,dtype,window", [
    ([100003, 60001, 1, 90000], 8, 4, 64, BF16, 0),
    ([140001], 8, 9, 128, F16, 0),
    ([70000, 0, 65000, 5, 33333, 64000], 8, 1, 64, F16, 60001),
])
def test_decode_long_streams_repeat_to_the_bit(M, lens, kv_heads, group, D, dtype, window):
    heads = kv_heads * group
    k, v, table = cache(11, lens, kv_heads, D, 128, dtype)
    q = randn(5, (len(lens), heads, D), dtype, 1.5)
    att = handle(M, heads, kv_heads, D, k, v, max_seqs=len(lens), window=window)
    outs = [att.decode(q, i32(lens), table, return_lse=True) for _ in range(4)]
    att.check()
    want = AO.run(q, clean(k), clean(v), table, lens, list(range(len(lens) + 1)), 1 / math.sqrt(D), 0.0, window,
                  4 * AO.U[dtype] ** 2)
    for y, lse in outs:
        AO.assert_within(y, want[0], want[1], "y")
        AO.assert_within(lse, want[2], want[3], "lse")
        assert torch.equal(y, outs[0][0]) and torch.equal(lse, outs[0][1]), "calls on the same inputs differ"


def test_decode_strided_rows_interleaved_pools_side_stream_and_graph(M):
    lens = [100, 513, 0, 77]
    k, v, table = cache(9, lens, 2, 128, 32, BF16, interleaved=True)
    wide = randn(7, (4, 30, 128), BF16, 1.5)
    q = wide[:, 3:19].transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost in memory
    att = handle(M, 16, 2, 128, k, v)
    want = AO.run(q, clean(k), clean(v), table, lens, list(range(5)), 1 / math.sqrt(128), 0.0, 0, 4 * AO.U[BF16] ** 2)
    n = i32(lens)
    y0 = att.decode(wide[:, 3:19], n, table)
    y1 = att.decode(q, n, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y2 = att.decode(q, n, table, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    out = torch.empty_like(y1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.decode(q, n, table, out=out)
    for _ in range(3):
        graph.replay()
    att.check()
    for y in (y0, y1, y2, out):
        AO.assert_within(y, want[0], want[1], "y")


def test_decode_and_prefill_past_32_bit_offsets(M):
    """A pool of more than 2^32 values: its last pages are read at their own addresses."""
    page, heads, D = 64, 8, 128
    pages = (2 ** 32) // (page * heads * D) + 8
    k = torch.empty((pages, heads, page, D), dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    n = 3 * page - 5
    ids = [pages - 1, 0, pages - 3]
    for j, pg in enumerate(ids):
        k[pg], v[pg] = randn(20 + j, (heads, page, D), BF16), randn(30 + j, (heads, page, D), BF16)
    table = i32([ids])
    q = randn(8, (n, heads, D), BF16, 1.5)
    att = handle(M, heads, heads, D, k, v)
    y = att.decode(q[-1:], i32([n]), table)
    z = att.prefill(q, i32([0, n]), i32([n]), table)
    att.check()
    want = AO.run(q[-1:], k, v, table, [n], [0, 1], 1 / math.sqrt(D), 0.0, 0, 4 * AO.U[BF16] ** 2)
    AO.assert_within(y, want[0], want[1], "decode")
    want = AO.run(q, k, v, table, [n], [0, n], 1 / math.sqrt(D), 0.0, 0, AO.U[BF16])
    AO.assert_within(z, want[0], want[1], "prefill")


# ---- prefill -----------------------------------------------------------------------------------------

PREFILL = [
    # (rows, cached before them) of each sequence, kv_heads, group, D, page, dtype, softcap, window
    ([(1, 0)], 1, 1, 64, 16, BF16, 0.0, 0),
    ([(1, 0), (0, 0), (2, 0), (1, 16)], 2, 8, 128, 16, BF16, 0.0, 0),
    ([(129, 0)], 1, 1, 128, 16, BF16, 0.0, 0),
    ([(257, 0), (300, 0)], 1, 2, 64, 32, F16, 0.0, 0),
    ([(33, 95), (64, 64), (100, 1)], 2, 4, 128, 64, BF16, 0.0, 0),
    ([(40, 500), (0, 0), (7, 1000), (90, 3)], 2, 5, 64, 128, F16, 20.0, 0),
    ([(200, 300)], 2, 3, 128, 16, BF16, 0.0, 1),
    ([(200, 300), (5, 128)], 2, 7, 128, 32, BF16, 0.0, 130),
    ([(150, 77)], 1, 16, 64, 16, F16, 0.0, 40),
    ([(50, 77)], 1, 48, 128, 16, BF16, 0.0, 0),
    ([(600, 0)], 2, 8, 128, 64, BF16, 30.0, 0),
    ([(3, 4096), (17, 2047)], 4, 8, 128, 64, BF16, 0.0, 0),
    ([(1024, 0)], 1, 4, 128, 64, F16, 0.0, 0),
]


@pytest.mark.parametrize("seqs,kv_heads,group,D,page,dtype,softcap,window", PREFILL)
def test_prefill_matches_definition(M, seqs, kv_heads, group, D, page, dtype, softcap, window):
    heads = kv_heads * group
    lens = [r + c for r, c in seqs]
    cu = [0]
    for r, _ in seqs:
        cu.append(cu[-1] + r)
    k, v, table = cache(len(lens) + D, lens, kv_heads, D, page, dtype)
    q = randn(5, (cu[-1], heads, D), dtype, 1.5)
    att = handle(M, heads, kv_heads, D, k, v, softcap=softcap, window=window)
    y, lse = att.prefill(q, i32(cu), i32(lens), table, return_lse=True)
    again = att.prefill(q, i32(cu), i32(lens), table)
    att.check()
    want = AO.run(q, clean(k), clean(v), table, lens, cu, 1 / math.sqrt(D), softcap, window, AO.U[dtype])
    AO.assert_within(y, want[0], want[1], "y")
    AO.assert_within(lse, want[2], want[3], "lse")
    assert torch.equal(y, again), "two calls on the same inputs differ"


def test_prefill_scores_that_grow_along_the_row(M):
    """Every tile raises the maximum by far more than the rescale threshold, and the values before it vanish."""
    n, D = 520, 128
    k, v, table = cache(2, [n], 1, D, 64, BF16)
    q = torch.zeros((n, 2, D), device="cuda")
    q[..., 0] = 8.0
    q = q.to(BF16)
    ramp = torch.arange(table.shape[1] * 64, device="cuda").float().div(4)
    for i, pg in enumerate(table[0].tolist()):
        k[pg, 0, :, 0] = ramp[i * 64:(i + 1) * 64].to(BF16)
    att = handle(M, 2, 1, D, k, v)
    y, lse = att.prefill(q, i32([0, n]), i32([n]), table, return_lse=True)
    att.check()
    want = AO.run(q, clean(k), clean(v), table, [n], [0, n], 1 / math.sqrt(D), 0.0, 0, AO.U[BF16])
    AO.assert_within(y, want[0], want[1], "y")
    AO.assert_within(lse, want[2], want[3], "lse")


def test_prefill_agrees_with_decode_row_by_row(M):
    n, heads, kv, D = 150, 8, 2, 128
    k, v, table = cache(4, [n], kv, D, 16, BF16)
    q = randn(5, (n, heads, D), BF16, 1.5)
    att = handle(M, heads, kv, D, k, v, max_seqs=n)
    y = att.prefill(q, i32([0, n]), i32([n]), table)
    z = att.decode(q, i32(list(range(1, n + 1))), table.expand(n, -1))
    att.check()
    want = AO.run(q, clean(k), clean(v), table, [n], [0, n], 1 / math.sqrt(D), 0.0, 0, AO.U[BF16])
    AO.assert_within(y, want[0], want[1], "prefill")
    AO.assert_within(z, want[0], want[1], "decode")


def test_prefill_strided_rows_side_stream_and_graph(M):
    lens, cu = [90, 200], [0, 50, 250]
    k, v, table = cache(9, lens, 2, 128, 32, BF16, interleaved=True)
    wide = randn(7, (250, 24, 128), BF16, 1.5)
    q = wide[:, 4:12]
    att = handle(M, 8, 2, 128, k, v)
    want = AO.run(q, clean(k), clean(v), table, lens, cu, 1 / math.sqrt(128), 0.0, 0, AO.U[BF16])
    n, c = i32(lens), i32(cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y0 = att.prefill(q, c, n, table, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    out = torch.empty_like(y0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.prefill(q, c, n, table, out=out)
    for _ in range(3):
        graph.replay()
    att.check()
    for y in (y0, out):
        AO.assert_within(y, want[0], want[1], "y")


# ---- append ------------------------------------------------------------------------------------------

APPEND = [
    # T, heads, kv_heads, D, page, dtype, rope_dim, pairs, sections, norms
    (1, 1, 1, 64, 16, BF16, 64, "halves", (), True),
    (7, 32, 4, 128, 16, BF16, 128, "halves", (), True),
    (33, 5, 1, 128, 32, F16, 64, "adjacent", (), True),
    (64, 12, 3, 64, 64, BF16, 32, "halves", (4, 6, 6), False),
    (129, 14, 2, 64, 128, F16, 64, "adjacent", (8, 12, 12), True),
    (300, 8, 8, 128, 16, BF16, 96, "halves", (0, 24, 24), False),
    (50, 3, 1, 128, 16, BF16, 16, "halves", (), False),
    (20, 6, 2, 64, 16, F16, 0, "halves", (), True),
    (20, 6, 2, 128, 16, BF16, 0, "halves", (), False),
]


@pytest.mark.parametrize("T,heads,kv_heads,D,page,dtype,rope_dim,pairs,sections,norms", APPEND)
def test_append_matches_definition(M, T, heads, kv_heads, D, page, dtype, rope_dim, pairs, sections, norms):
    pages, P = -(-T // page) + 3, 500
    g = torch.Generator().manual_seed(T)
    k0, v0 = randn(1, (pages, kv_heads, page, D), dtype), randn(2, (pages, kv_heads, page, D), dtype)
    k_pool, v_pool = k0.clone(), v0.clone()
    qkv = randn(3, (T, heads + 2 * kv_heads, D), dtype, 2.0)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 3:
        slots[2] = -1
    axes = max(1, len(sections))
    pos = torch.randint(0, P, (axes, T), generator=g).to(torch.int32).cuda()
    table = M.rope_table(rope_dim, P) if rope_dim else None
    qn = (1 + randn(4, (D,), torch.float32, 0.1)).to(dtype) if norms else None
    kn = (1 + randn(5, (D,), torch.float32, 0.1)).to(dtype) if norms else None
    att = M.PagedAttention(M.AttentionConfig(heads, kv_heads, D, rope_dim=rope_dim, rope_pairs=pairs,
                                             rope_sections=sections, norm_eps=1e-5), k_pool, v_pool, rope_table=table,
                           q_norm=qn, k_norm=kn)
    out = att.append(q, k, v, pos if axes > 1 else pos[0], slots.cuda())
    inplace = qkv.clone()
    same = att.append(inplace[:, :heads], k, v, pos, slots.cuda(), out=inplace[:, :heads])
    att.check()
    assert torch.equal(same, out) and torch.equal(inplace[:, heads:], qkv[:, heads:])
    adj = pairs == "adjacent"
    sec = sections or (rope_dim // 2,)
    wq, bq = AO.append(q, qn, 1e-5, table, pos, sec, rope_dim, adj)
    wk, bk = AO.append(k, kn, 1e-5, table, pos, sec, rope_dim, adj)
    keep = slots >= 0
    wq[~keep], bq[~keep] = 0, 0
    AO.assert_within(out, wq, bq + AO.rounding(wq, dtype), "q")
    ek, ev = k0.clone(), v0.clone()  # where each token's slot is, compare; everywhere else the pools are untouched
    at = slots[keep].cuda()
    got_k, got_v = k_pool[at // page, :, at % page], v_pool[at // page, :, at % page]
    AO.assert_within(got_k, wk[keep], bk[keep] + AO.rounding(wk[keep], dtype), "k")
    assert torch.equal(got_v, v[keep.cuda()])
    ek[at // page, :, at % page], ev[at // page, :, at % page] = got_k, got_v
    assert torch.equal(ek, k_pool) and torch.equal(ev, v_pool)


def test_append_then_attend_is_the_layer(M):
    """append, prefill a prompt in two chunks, decode a token: the whole against one pass of the definition."""
    heads, kv, D, page, n = 8, 2, 128, 16, 75
    k_pool, v_pool = M.kv_pools(8, kv, page, D)
    k_pool.fill_(float("nan")), v_pool.fill_(float("nan"))
    table = i32([[6, 1, 3, 0, 7]])
    rope = M.rope_table(D, 100)
    att = M.PagedAttention(M.AttentionConfig(heads, kv, D, rope_dim=D), k_pool, v_pool, rope_table=rope)
    q, k, v = (randn(s, (n, h, D), BF16) for s, h in ((1, heads), (2, kv), (3, kv)))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = M.page_slots(table, torch.zeros_like(pos), pos, page)
    outs = []
    for a, z in ((0, 50), (50, 74), (74, 75)):
        qr = att.append(q[a:z], k[a:z], v[a:z], pos[a:z], slots[a:z])
        if z - a > 1:
            outs.append(att.prefill(qr, i32([0, z - a]), i32([z]), table))
        else:
            outs.append(att.decode(qr, i32([z]), table))
    att.check()
    y = torch.cat(outs)
    qr = AO.append(q, None, 0, rope, pos[None], (D // 2,), D, False)[0].to(BF16)  # rounded once, as stored
    kr = AO.append(k, None, 0, rope, pos[None], (D // 2,), D, False)[0].to(BF16)
    want = AO.attention(qr.double(), kr.double().transpose(0, 1), v.double().cpu().transpose(0, 1), 0, 1 / math.sqrt(D), 0.0,
                        0, AO.U[BF16])
    # q or k may round to the other neighbour: 2 u of a score's terms on top of the kernel's bound
    mag = (qr.double().abs().amax() * kr.double().abs().sum(-1).amax()) / math.sqrt(D)
    assert (y.double().cpu() - want[0]).abs().max() < 0.05 and float(mag) > 0
    err = (y.double().cpu() - want[0]).norm() / want[0].norm()
    assert err < 4 * AO.U[BF16], err


# ---- refusals ----------------------------------------------------------------------------------------


def refused(M, fn, status=1):
    with pytest.raises(M.MoeError) as e:
        fn()
    assert e.value.status == status, e.value


def test_refusals(M):
    k, v, table = cache(1, [20], 2, 64, 16, BF16)
    A, C = M.PagedAttention, M.AttentionConfig
    refused(M, lambda: A(C(5, 2, 64), k, v))
    refused(M, lambda: A(C(4, 2, 128), k, v))
    refused(M, lambda: A(C(4, 2, 64), k, v.to(F16)))
    refused(M, lambda: A(C(4, 2, 64), k.float(), v.float()))
    refused(M, lambda: A(C(4, 2, 64, softcap=-1.0), k, v))
    refused(M, lambda: A(C(4, 2, 64, window=-1), k, v))
    refused(M, lambda: A(C(4, 2, 64, rope_dim=24), k, v, rope_table=torch.zeros((4, 12, 2), device="cuda")))
    refused(M, lambda: A(C(4, 2, 64, rope_dim=64), k, v))
    refused(M, lambda: A(C(4, 2, 64, rope_dim=64, rope_sections=(1, 2, 3)), k, v, rope_table=M.rope_table(64, 10)))
    refused(M, lambda: A(C(4, 2, 64), k[:, :, :8], v[:, :, :8]))
    refused(M, lambda: A(C(4, 2, 64), k, v, max_seqs=0))
    wide = torch.zeros((3, 1, 16, 96), dtype=BF16, device="cuda")
    refused(M, lambda: A(C(1, 1, 96), wide, wide), status=6)
    att = A(C(4, 2, 64), k, v, max_seqs=1)
    q = randn(1, (1, 4, 64), BF16)
    refused(M, lambda: att.decode(q.to(F16), i32([20]), table))
    refused(M, lambda: att.decode(q[:, :3], i32([20]), table))
    refused(M, lambda: att.decode(torch.cat([q, q]), i32([20, 20]), torch.cat([table, table])))
    refused(M, lambda: att.decode(q, torch.tensor([20], device="cuda"), table))
    refused(M, lambda: att.decode(q, i32([20]), table[0]))
    refused(M, lambda: att.decode(q.cpu(), i32([20]), table))
    refused(M, lambda: att.prefill(q, i32([0]), i32([20]), table))
    refused(M, lambda: att.append(q, q, q, None, torch.zeros(1, dtype=torch.int64, device="cuda")))
    kv1 = randn(1, (1, 2, 64), BF16)
    refused(M, lambda: att.append(q, kv1, kv1, None, torch.zeros(1, dtype=torch.int32, device="cuda")))
    assert att.decode(q[:0], i32([]), table[:0]).shape == (0, 4, 64)
    att.check()


def test_device_side_errors_are_latched_and_nothing_is_written(M):
    k, v, table = cache(1, [20], 2, 64, 16, BF16, junk=0.0)
    rope = M.rope_table(64, 10)
    att = M.PagedAttention(M.AttentionConfig(4, 2, 64, rope_dim=64), k, v, rope_table=rope, max_seqs=1)
    q, kv1 = randn(1, (3, 4, 64), BF16), randn(2, (3, 2, 64), BF16)
    k0, v0 = k.clone(), v.clone()
    for slots, pos in (([-1, k.shape[0] * 16, -1], [0, 0, 0]), ([-2, -1, -1], [0, 0, 0]), ([0, -1, -1], [10, 0, 0]),
                       ([0, -1, -1], [-1, 0, 0])):
        out = att.append(q, kv1, kv1, i32(pos), torch.tensor(slots, device="cuda"))
        refused(M, att.check, status=5)
        assert torch.equal(k, k0) and torch.equal(v, v0) and not out.any()
    att.check()
    for bad, n in (([[k.shape[0], 0]], 20), ([[-1, 0]], 20), ([[0, 1]], 33)):
        att.decode(q[:1], i32([n]), i32(bad))
        refused(M, att.check, status=5)
        att.prefill(q, i32([0, 3]), i32([n]), i32(bad))
        refused(M, att.check, status=5)
    y, lse = att.prefill(q, i32([0, 3]), i32([2]), table, return_lse=True)  # more rows than cached positions
    refused(M, att.check, status=5)
    assert not y[0].any() and torch.isneginf(lse[0]).all() and y[1].any() and torch.isfinite(lse[1:]).all()
    att.check()
