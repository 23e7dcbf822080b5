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
