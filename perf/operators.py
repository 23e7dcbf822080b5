"""The paged-attention operators as a serving program calls them: real sizes, plain forms, 64-bit values.

Three operators of a decoder layer's attention, which runs next to the routed experts:

  append   one pass of new tokens into a paged key/value cache: per-head RMS norm of q and k, rotary
           position rotation (one position axis, or three for time / height / width), k and v stored
           into the cache's pages, rotated q returned;
  decode   attention of one new token per sequence over its pages;
  prefill  causal attention of a ragged batch of prompt chunks over their pages.

Sizes: 32 query and 4 key/value heads of 128 (the layer of the 48-layer stack workload: 32 sequences,
prompts of 128 to 2048 tokens, 256 decode steps; the 4096-token prompt in 512-token chunks), and generic
ones. `run` takes torch tensors; with `own` it calls moe_b200.PagedAttention.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- the cases ---------------------------------------------------------------------------------------


def _append(name, tokens, q_heads=32, kv_heads=4, head_dim=128, dtype="bf16", page=16, rope=128, axes=1,
            pairs="halves", norm=True, padding=0):
    return {"name": name, "op": "append", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "page": page, "rope": rope, "axes": axes, "pairs": pairs,
            "norm": norm, "padding": padding}


def _decode(name, seqs, lo, hi, empty=0, q_heads=32, kv_heads=4, head_dim=128, dtype="bf16", page=16, softcap=0.0,
            window=0, lse=False):
    return {"name": name, "op": "decode", "seqs": seqs, "lo": lo, "hi": hi, "empty": empty, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "softcap": softcap,
            "window": window, "lse": lse}


def _prefill(name, seqs, lo, hi, past=0, empty=0, q_heads=32, kv_heads=4, head_dim=128, dtype="bf16", page=16,
             softcap=0.0, window=0, lse=False):
    return {"name": name, "op": "prefill", "seqs": seqs, "lo": lo, "hi": hi, "past": past, "empty": empty,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page,
            "softcap": softcap, "window": window, "lse": lse}


def listed():
    return [
        # one decode step of 32 sequences: a launch-bound call, made once per layer and token
        _append("append-step32", 32),
        # a 4096-token prompt written in one pass: the bandwidth-bound end
        _append("append-prompt4096", 4096, page=64),
        # an image prompt: three position axes, half-rotated heads of 64 without norm, odd token count, padding tokens
        _append("append-axes1531", 1531, q_heads=14, kv_heads=2, head_dim=64, dtype="f16", page=32, rope=64, axes=3,
                norm=False, padding=27),
        # one user at the start of an answer: nothing but latency
        _decode("decode-one129", 1, 129, 129),
        # the stack workload's step: 32 sequences between their shortest prompt and longest answer
        _decode("decode-step32", 32, 128, 2304),
        # a large batch of long contexts: cache bandwidth
        _decode("decode-batch128", 128, 1, 8191, page=64),
        # one long context: the length has to be split over the GPU
        _decode("decode-long131071", 1, 131071, 131071, page=64, lse=True),
        # capped scores in a sliding window, odd head group, finished sequences left in the batch
        _decode("decode-window61", 61, 1, 6001, empty=3, q_heads=20, kv_heads=4, head_dim=64, dtype="f16", page=32,
                softcap=30.0, window=1000),
        # the 4096-token prompt at once: tensor-core bound
        _prefill("prefill-prompt4096", 1, 4096, 4096, page=64),
        # a 512-token chunk of a prompt whose first 12288 tokens are in the cache
        _prefill("prefill-chunk512", 1, 512, 512, past=12288, page=64),
        # prompts of 128 to 2048 tokens batched raggedly
        _prefill("prefill-batch8", 8, 128, 2047, lse=True),
        # short chunks of one to a hundred tokens on odd contexts: capped scores, window, heads of 64, an empty one
        _prefill("prefill-odd9", 9, 1, 101, past=1777, empty=1, q_heads=12, kv_heads=2, head_dim=64, dtype="f16",
                 page=32, softcap=50.0, window=700),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    while kv_heads * group > 48:
        kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    head_dim, dtype, page = rng.choice([64, 128]), rng.choice(["bf16", "f16"]), rng.choice([16, 32, 64, 128])
    heads = {"q_heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page}
    if op == "append":
        tokens = _log(rng, 1, 4096)
        c = _append("", tokens, rope=rng.choice([head_dim, head_dim // 2]), axes=rng.choice([1, 1, 3]),
                    pairs=rng.choice(["halves", "adjacent"]), norm=rng.random() < 0.5,
                    padding=min(tokens - 1, rng.choice([0, 0, 1, 5])), **heads)
    else:
        softcap, window = rng.choice([0.0, 0.0, 20.0, 50.0]), rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        lse = rng.random() < 0.3
        if op == "decode":
            seqs = _log(rng, 1, 256)
            hi = _log(rng, 1, max(2, min(131071, 2 * 128 * 4096 * 4 * 128 // (seqs * kv_heads * head_dim * 2))))
            c = _decode("", seqs, max(1, int(hi * rng.random())), hi, empty=rng.choice([0, 0, min(2, seqs - 1)]),
                        softcap=softcap, window=window, lse=lse, **heads)
        else:
            while True:  # no more score entries than the 4096-token prompt's
                seqs, hi, past = _log(rng, 1, 16), _log(rng, 1, 4096), rng.choice([0, 0, _log(rng, 1, 16384)])
                if seqs * heads["q_heads"] * hi * (hi + past) <= 32 * 4096 * 4096:
                    break
            c = _prefill("", seqs, max(1, int(hi * rng.random())), hi, past=past,
                         empty=rng.choice([0, 0, min(1, seqs - 1)]), softcap=softcap, window=window, lse=lse, **heads)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------


def _spread(case):
    """The batch's lengths: evenly from lo to hi, the first `empty` of them zero (a seed only orders them)."""
    n = case["seqs"]
    v = [case["hi"] if n == 1 else case["lo"] + (case["hi"] - case["lo"]) * i // (n - 1) for i in range(n)]
    return [0] * case["empty"] + v[case["empty"]:]


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _table(rng, lens, page, spare):
    """A page table of randomly placed pages ([seqs, widest] int32, -1 past a sequence's pages) and their count."""
    need = _pages(lens, page)
    total = sum(need) + spare
    order = list(range(total))
    rng.shuffle(order)
    width, rows, at = max(1, max(need)), [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), total


def _rope_table(rope, positions, base=10000.0):
    inv = base ** (-torch.arange(0, rope, 2, dtype=torch.float64) / rope)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv[None]
    return torch.stack([angle.cos(), angle.sin()], -1).float().cuda()  # [positions, rope / 2, 2]


def _sections(case):
    """Rotary pairs of each position axis: a quarter for time, the rest between height and width."""
    n = case["rope"] // 2
    if case["axes"] == 1:
        return [n]
    t = n // 4
    return [t, (n - t) // 2, n - t - (n - t) // 2]


def _handle(case, s):
    if not own:
        return None
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "naiwa-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import moe_b200 as M

    cfg = M.AttentionConfig(num_heads=case["q_heads"], num_kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                            softcap=case.get("softcap", 0.0), window=case.get("window", 0),
                            rope_dim=case.get("rope", 0), rope_pairs=case.get("pairs", "halves"),
                            rope_sections=tuple(_sections(case)) if case["op"] == "append" else (),
                            norm_eps=1e-6)
    return M.PagedAttention(cfg, s["k_pool"], s["v_pool"], rope_table=s.get("rope_table"), q_norm=s.get("q_norm"),
                            k_norm=s.get("k_norm"), max_seqs=case.get("seqs", 1))


def prepare(case, seed):
    rng, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    dt, D, Hq, Hk, page = DTYPES[case["dtype"]], case["head_dim"], case["q_heads"], case["kv_heads"], case["page"]
    s = {"case": case}
    if case["op"] == "append":
        T, context = case["tokens"], 2304
        live = T - case["padding"]
        if T <= 256:  # a decode step: every token in a sequence, and a page, of its own
            slots = [p * page + rng.randrange(page) for p in rng.sample(range(2 * T), live)]
            first = [rng.randrange(context) for _ in range(live)]
            pages = 2 * T
        else:  # a prompt: consecutive slots of pages that lie anywhere
            pages = _pages([live], page)[0] + 8
            order = rng.sample(range(pages), pages - 8)
            slots = [order[i // page] * page + i % page for i in range(live)]
            start = rng.randrange(context)
            first = [start + i for i in range(live)]
            context += T
        slots += [-1] * case["padding"]
        first += [0] * case["padding"]
        where = [first]
        if case["axes"] == 3:  # rows of a picture 41 wide, after the text before it
            where = [[p - p % 41 for p in first], [p // 41 for p in first], [p % 41 for p in first]]
        # q, k and v are views of one projection's output rows
        qkv = _randn(g, (T, (Hq + 2 * Hk) * D), dt)
        s["q"] = qkv[:, :Hq * D].view(T, Hq, D)
        s["k"] = qkv[:, Hq * D:(Hq + Hk) * D].view(T, Hk, D)
        s["v"] = qkv[:, (Hq + Hk) * D:].view(T, Hk, D)
        s["positions"] = torch.tensor(where, dtype=torch.int32, device="cuda")
        s["slots"] = torch.tensor(slots, dtype=torch.int64, device="cuda")
        s["rope_table"] = _rope_table(case["rope"], context)
        if case["norm"]:
            s["q_norm"] = (1 + _randn(g, (D,), torch.float32, 0.1)).to(dt)
            s["k_norm"] = (1 + _randn(g, (D,), torch.float32, 0.1)).to(dt)
    else:
        lens = _spread(case)
        rng.shuffle(lens)
        if case["op"] == "decode":
            news, tokens = None, case["seqs"]
        else:
            news, tokens = lens, sum(lens)
            lens = [n + case["past"] if n else 0 for n in lens]
            ends = [sum(news[:i]) for i in range(len(news) + 1)]
            s["cu_q"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
            s["most"] = max(news)
        s["table"], pages = _table(rng, lens, page, 4)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        # query rows a little larger than the keys, so that a row's weights spread over decades
        s["q"] = _randn(g, (tokens, Hq, D), dt, 1.5)
    s["k_pool"] = _randn(g, (pages, Hk, page, D), dt)
    s["v_pool"] = _randn(g, (pages, Hk, page, D), dt)
    s["handle"] = _handle(case, s)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------


def _norm(x, w, eps=1e-6):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()


def _axis_of_pair(case, device):
    n = _sections(case)
    return torch.tensor([0] * n[0] + ([1] * n[1] + [2] * n[2] if len(n) == 3 else []), device=device)


def _rotate(x, case, table, positions):
    """x [T, heads, D] f32: the first `rope` values of each head rotated pair by pair."""
    r = case["rope"]
    axis = _axis_of_pair(case, x.device)
    cs = table[positions.long()[axis].t(), torch.arange(r // 2, device=x.device)]  # [T, r / 2, 2]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if case["pairs"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., r:]], -1)


def _plain_append(s):
    case, dt = s["case"], s["q"].dtype
    q, k = s["q"].float(), s["k"].float()
    if case["norm"]:
        q, k = _norm(q, s["q_norm"]), _norm(k, s["k_norm"])
    q = _rotate(q, case, s["rope_table"], s["positions"])
    k = _rotate(k, case, s["rope_table"], s["positions"])
    live = s["slots"] >= 0
    q = torch.where(live[:, None, None], q, torch.zeros((), device=q.device))
    n = case["tokens"] - case["padding"]  # padding tokens come last
    at = s["slots"][:n]
    s["k_pool"][at // case["page"], :, at % case["page"]] = k[:n].to(dt)
    s["v_pool"][at // case["page"], :, at % case["page"]] = s["v"][:n]
    return {"q": q.to(dt), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _gathered(s, pool):
    """[seqs, kv_heads, widest length, D] f32 of every sequence's pages."""
    page = s["case"]["page"]
    tok = torch.arange(s["table"].shape[1] * page, device=pool.device)
    return pool[s["table"].long().clamp(min=0)[:, tok // page], :, tok % page].permute(0, 2, 1, 3).float()


def _softmax_rows(s, q, k, v, mask):
    """q [B, Hk, rows, D], k and v [B, Hk, L, D] f32, mask broadcast to the scores: outputs and log-sum-exp."""
    case = s["case"]
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(case["head_dim"]))
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    x = x.masked_fill(~mask, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    y = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return y, (m + torch.log(total)).squeeze(-1)


def _plain_decode(s):
    case = s["case"]
    B, Hq, D = s["q"].shape
    Hk = case["kv_heads"]
    k, v = _gathered(s, s["k_pool"]), _gathered(s, s["v_pool"])
    at, n = torch.arange(k.shape[2], device=k.device)[None], s["seq_lens"][:, None]
    mask = at < n
    if case["window"]:
        mask = mask & (at >= n - case["window"])
    y, lse = _softmax_rows(s, s["q"].float().view(B, Hk, Hq // Hk, D), k, v, mask[:, None, None])
    y = y.reshape(B, Hq, D).to(s["q"].dtype)
    return {"y": y, "lse": lse.reshape(B, Hq)} if case["lse"] else {"y": y}


def _plain_prefill(s):
    case, most = s["case"], s["most"]
    T, Hq, D = s["q"].shape
    Hk, B = case["kv_heads"], case["seqs"]
    group = Hq // Hk
    start, news = s["cu_q"][:-1, None], (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
    i = torch.arange(most, device=s["q"].device)[None]
    rows = i < news
    q = s["q"].float()[(start + i).clamp(max=T - 1)]  # [B, most, Hq, D]
    q = q.view(B, most, Hk, group, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, most * group, D)
    k, v = _gathered(s, s["k_pool"]), _gathered(s, s["v_pool"])
    at = torch.arange(k.shape[2], device=k.device)[None, None]
    here = (s["seq_lens"][:, None] - news + i)[..., None]  # each row's own position in the cache
    mask = (at <= here) & rows[..., None]
    if case["window"]:
        mask = mask & (at > here - case["window"])
    mask = mask[:, None].repeat_interleave(group, 2)
    y, lse = _softmax_rows(s, q, k, v, mask)
    y = y.view(B, Hk, most, group, D).permute(0, 2, 1, 3, 4).reshape(B, most, Hq, D)[rows].to(s["q"].dtype)
    if not case["lse"]:
        return {"y": y}
    return {"y": y, "lse": lse.view(B, Hk, most, group).permute(0, 2, 1, 3).reshape(B, most, Hq)[rows]}


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[case["op"]](state)
    att = state["handle"]
    if case["op"] == "append":
        q = att.append(state["q"], state["k"], state["v"], state["positions"], state["slots"])
        return {"q": q, "k_pool": state["k_pool"], "v_pool": state["v_pool"]}
    if case["op"] == "decode":
        r = att.decode(state["q"], state["seq_lens"], state["table"], return_lse=case["lse"])
    else:
        r = att.prefill(state["q"], state["cu_q"], state["seq_lens"], state["table"], return_lse=case["lse"])
    return {"y": r[0], "lse": r[1]} if case["lse"] else {"y": r}


# ---- floors ------------------------------------------------------------------------------------------


def work(case):
    D, Hq, Hk = case["head_dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        T = case["tokens"] - case["padding"]
        row = (Hq + 2 * Hk) * D * 2
        table = min(T, 2304 + case["tokens"]) * case["rope"] * 4
        return {"bytes": 2 * T * row + T * (4 * case["axes"] + 8) + table,
                "flops": T * (Hq + Hk) * (3 * case["rope"] + (4 * D if case["norm"] else 0))}
    w, byte, pairs = case["window"], 0, 0
    for n in _spread(case):
        if not n:
            continue
        if case["op"] == "decode":
            seen = min(n, w) if w else n
            byte += 2 * seen * Hk * D * 2 + 2 * Hq * D * 2 + 4 * -(-seen // case["page"]) + (4 * Hq if case["lse"] else 0)
            pairs += seen
        else:
            total = n + case["past"]
            read = min(total, n + w - 1) if w else total
            byte += 2 * read * Hk * D * 2 + 2 * n * Hq * D * 2 + (4 * n * Hq if case["lse"] else 0)
            # row i sees past + i + 1 keys, at most w
            first = case["past"] + 1
            if not w or total <= w:
                pairs += n * (first + total) // 2
            elif first >= w:
                pairs += n * w
            else:
                full = w - first  # rows that see fewer than w
                pairs += full * (first + w - 1) // 2 + (n - full) * w
    return {"bytes": byte, "flops": 4 * D * Hq * pairs}


# ---- values in 64 bits -------------------------------------------------------------------------------


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)


def _exact_append(case, s):
    """Token by token from complex numbers: pair (a, b) at angle t becomes (a + ib) e^{it}."""
    T, r, n = case["tokens"], case["rope"], case["rope"] // 2
    sections = _sections(case)
    pos = s["positions"].long().cpu()
    turn = torch.empty((T, n), dtype=torch.complex128)
    table = torch.view_as_complex(s["rope_table"].double().cpu())
    at = 0
    for a, width in enumerate(sections):
        turn[:, at:at + width] = table[pos[a], at:at + width]
        at += width

    def through(x, w):
        x = x.double().cpu()
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double().cpu()
        head, tail = x[..., :r], x[..., r:]
        if case["pairs"] == "halves":
            z = torch.complex(head[..., :n].contiguous(), head[..., n:].contiguous()) * turn[:, None]
            head = torch.cat((z.real, z.imag), -1)
        else:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], n, 2).contiguous()) * turn[:, None]
            head = torch.view_as_real(z).reshape(*head.shape)
        return torch.cat((head, tail), -1)

    q, k, v = through(s["q"], s.get("q_norm")), through(s["k"], s.get("k_norm")), s["v"].double().cpu()
    kp, vp = s["k_pool"].double().cpu(), s["v_pool"].double().cpu()
    for t, slot in enumerate(s["slots"].tolist()):
        if slot < 0:
            q[t] = 0
            continue
        kp[slot // case["page"], :, slot % case["page"]] = k[t]
        vp[slot // case["page"], :, slot % case["page"]] = v[t]
    return {"q": q, "k_pool": kp, "v_pool": vp}


def _exact_attention(case, s):
    """Sequence by sequence and head by head, the definition in double precision."""
    Hq, Hk, D, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    lens = s["seq_lens"].tolist()
    cu = s["cu_q"].tolist() if case["op"] == "prefill" else list(range(len(lens) + 1))
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        rows = cu[b + 1] - cu[b]
        if not n or not rows:
            continue
        ids = s["table"][b, :-(-n // page)].long()
        k = s["k_pool"][ids].transpose(0, 1).reshape(Hk, -1, D)[:, :n].double()
        v = s["v_pool"][ids].transpose(0, 1).reshape(Hk, -1, D)[:, :n].double()
        here = torch.arange(n - rows, n, device="cuda")[:, None]
        keys = torch.arange(n, device="cuda")[None]
        seen = keys <= here
        if case["window"]:
            seen &= here - keys < case["window"]
        for h in range(Hq):
            x = s["q"][cu[b]:cu[b + 1], h].double() @ k[h // (Hq // Hk)].t() / math.sqrt(D)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            x[~seen] = -math.inf
            y[cu[b]:cu[b + 1], h] = torch.softmax(x, -1) @ v[h // (Hq // Hk)]
            lse[cu[b]:cu[b + 1], h] = torch.logsumexp(x, -1)
    return {"y": y, "lse": lse} if case["lse"] else {"y": y}
