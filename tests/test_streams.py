"""Calls given a stream make their copies and allocations on that stream: on the CPU with stand-ins for the streams and the
library, on the GPU behind a long kernel of the current stream."""
import contextlib

import pytest

torch = pytest.importorskip("torch")
from torch.utils._python_dispatch import TorchDispatchMode  # noqa: E402


class FakeStream:
    device_index = -1  # a CPU tensor's get_device()
    cuda_stream = 7


@pytest.fixture
def ops(monkeypatch):
    """Collects (operation, the stream current at that time); None stands for the caller's stream."""
    active, seen = [None], []

    @contextlib.contextmanager
    def stream(s):
        active.append(s)
        try:
            yield
        finally:
            active.pop()

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append((func.overloadpacket.__name__, active[-1]))
            return func(*args, **(kwargs or {}))

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: active[-1])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: active[-1].cuda_stream if active[-1] else 0,
                        raising=False)
    with Record():
        yield seen


def stand_in(calls):
    """A PagedAttention over CPU tensors whose entry points only note their arguments."""
    import moe_b200 as M

    att = object.__new__(M.PagedAttention)
    att.config, att._h, att.axes, att.max_seqs = M.AttentionConfig(num_heads=4, num_kv_heads=2, head_dim=64), None, 1, 8
    att._torch, att._int32, att._dtype, att._dim, att._index = torch, torch.int32, torch.bfloat16, 64, -1
    att.device, att._raw_stream = torch.device("cpu"), torch._C._cuda_getCurrentRawStream

    def entry(*args):
        calls.append(args)
        return 0

    att._append = att._decode = att._prefill = entry
    return att


def misaligned(rows, heads):
    """Rows that the kernels do not take as they are: every value's neighbours lie two apart."""
    return torch.zeros((rows, heads, 128), dtype=torch.bfloat16)[..., ::2]


def spread(values, dtype):
    return torch.tensor(values, dtype=dtype).repeat_interleave(2, -1)[..., ::2]


@pytest.mark.parametrize("name", ["append", "decode", "prefill"])
def test_attention_copies_and_allocates_on_the_given_stream(ops, name):
    calls = []
    att, side = stand_in(calls), FakeStream()
    q, kv = misaligned(2, 4), misaligned(2, 2)
    lens, table = spread([3, 4], torch.int32), spread([[0, 1], [2, 3]], torch.int32)
    slots, cu_q = spread([0, 1], torch.int64), spread([0, 1, 2], torch.int32)
    del ops[:]
    if name == "append":
        att.append(q, kv, kv, None, slots, stream=side)
    elif name == "decode":
        att.decode(q, lens, table, return_lse=True, stream=side)
    else:
        att.prefill(q, cu_q, lens, table, return_lse=True, stream=side)
    assert calls[0][-1] == side.cuda_stream
    made = [op for op, _ in ops if op in ("clone", "empty_like", "new_empty", "empty", "_to_copy", "copy_")]
    assert made.count("clone") >= 2 and made, ops
    assert all(s is side for _, s in ops), ops


def test_a_stream_of_another_device_is_refused(ops):
    import moe_b200 as M

    att, side = stand_in([]), FakeStream()
    side.device_index = 1
    with pytest.raises(M.MoeError):
        att.decode(misaligned(1, 4), torch.tensor([1], dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32), stream=side)


class FakeLibrary:
    def __init__(self):
        self.streams = []

    def __getattr__(self, name):
        def entry(*args):
            if name.endswith("_bytes"):
                return 64
            self.streams += [a.value for a in args[-2:] if hasattr(a, "value")][:1]
            return 0
        return entry


@pytest.mark.parametrize("name", ["plan_pairs", "route_tokens", "Router", "ep_dispatch", "ep_pack_rows", "ep_combine",
                                  "PagedMoE.forward", "PagedMoE.prefill"])
def test_older_calls_copy_and_allocate_on_the_given_stream(ops, monkeypatch, name):
    import moe_b200 as M
    from moe_b200 import ep, layer, paged

    fake = FakeLibrary()
    for module in (layer, ep, paged):
        monkeypatch.setattr(module, "lib", lambda: fake)
    side = FakeStream()
    x = torch.zeros((4, 64), dtype=torch.bfloat16)[:, ::2]
    ids, w = torch.zeros((4, 2), dtype=torch.int64), torch.zeros((4, 4))[:, ::2]
    gate = torch.zeros((8, 64), dtype=torch.bfloat16)[:, ::2]
    rows = torch.zeros((4, 1), dtype=torch.int32)
    router = M.Router(gate, 2, 0, max_tokens=4)
    moe = object.__new__(paged.PagedMoE)
    moe._h = None
    calls = {
        "plan_pairs": lambda: layer.plan_pairs(ids, 8, stream=side),
        "route_tokens": lambda: layer.route_tokens(x, gate, 2, 0, stream=side),
        "Router": lambda: router.route(x, stream=side),
        "ep_dispatch": lambda: ep.ep_dispatch(ids, w, 4, 2, stream=side),
        "ep_pack_rows": lambda: ep.ep_pack_rows(x, rows, rows, 4, stream=side),
        "ep_combine": lambda: ep.ep_combine(x, rows, 4, stream=side),
        "PagedMoE.forward": lambda: moe.forward(x, w, ids, stream=side),
        "PagedMoE.prefill": lambda: moe.prefill(x, w, ids, stream=side),
    }
    del ops[:]
    calls[name]()
    assert fake.streams == [side.cuda_stream] and ops and all(s is side for _, s in ops), (fake.streams, ops)


# ---- on the GPU ---------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_attention_rows_that_need_a_copy_on_a_side_stream():
    """The inputs are ready before the call; the current stream is busy with something else during it, and the memory that a
    copy on it would take holds other values."""
    import moe_b200 as M

    bf = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(1)
    heads, kv, D, page, n = 8, 2, 128, 16, 40

    def rows(h):
        return torch.randn((n, h, 2 * D), generator=g, device="cuda").to(bf)[..., ::2]

    q, k, v = rows(heads), rows(kv), rows(kv)
    slots = torch.randperm(4 * page, device="cuda")[:n].repeat_interleave(2)[::2]
    lens = torch.arange(1, n + 1, dtype=torch.int32, device="cuda").repeat_interleave(2)[::2]
    table = torch.tensor([[2, 0, 1, 3]], dtype=torch.int32, device="cuda").expand(n, 4)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda").repeat_interleave(2)[::2]
    seq = torch.tensor([n], dtype=torch.int32, device="cuda")

    def handle():
        pools = [torch.zeros((4, kv, page, D), dtype=bf, device="cuda") for _ in range(2)]
        return M.PagedAttention(M.AttentionConfig(heads, kv, D), *pools, max_seqs=n), pools

    def run(att, **kw):
        a = att.append(q, k, v, None, slots, **kw)
        return [a, att.decode(q, lens, table, **kw), att.prefill(q, cu, seq, table[:1], **kw)]

    att, pools = handle()
    want = [t.clone() for t in run(att)]
    want += [t.clone() for t in pools]
    att, pools = handle()
    side = torch.cuda.Stream()
    busy = torch.randn((8192, 8192), device="cuda").to(bf)
    torch.cuda.synchronize()
    for _ in range(20):
        busy = (busy @ busy).mul_(1e-3)
    got = run(att, stream=side)
    side.synchronize()
    got = [t.clone() for t in got] + pools
    torch.cuda.synchronize()
    att.check()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_expert_inputs_that_need_a_copy_on_a_side_stream():
    import numpy as np

    import moe_b200 as M
    from oracle import oracle as O

    rng = np.random.default_rng(3)
    E, k, H, I, T = 16, 4, 256, 128, 6
    stacks = [O.quantize(O.DT_Q8_0, rng.normal(0, 0.02, s).astype(np.float32))[0] for s in ((E, I, H), (E, I, H), (E, H, I))]
    cfg = M.MoeConfig(num_experts=E, num_experts_per_tok=k, hidden_size=H, moe_intermediate_size=I)
    layer = M.RoutedExpertsProvider().build(M.ExpertLoadContext(
        layer=0, device=0, config=cfg, wdtype=O.DT_Q8_0, gate=stacks[0], up=stacks[1], down=stacks[2], max_tokens=T))
    x = torch.randn((T, 2 * H), device="cuda").to(torch.bfloat16)[:, ::2]
    ids = torch.from_numpy(np.stack([rng.permutation(E)[:k] for _ in range(T)])).cuda()  # int64
    w = torch.rand((T, 2 * k), device="cuda")[:, ::2]
    want = layer.forward(x, w, ids)
    side = torch.cuda.Stream()
    busy = torch.randn((8192, 8192), device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    for _ in range(20):
        busy = (busy @ busy).mul_(1e-3)
    got = layer.forward(x, w, ids, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    layer.check()
