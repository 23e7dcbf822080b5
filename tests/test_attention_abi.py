"""The paged-attention entry points without a GPU: the descriptor's layout and every refusal that comes before a launch."""
import ctypes
import os
import re

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "moe_b200.h")


def test_attn_desc_matches_header():
    from moe_b200._lib import AttnDesc

    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    end = text.index("} moe_attn_desc;")
    body = text[text.rindex("typedef struct {", 0, end) + len("typedef struct {"):end]
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"((?:const\s+)?\w+\s*\**)\s*(.*)", decl).groups()
        kind = "void*" if "*" in kind else kind.strip()
        for name in names.split(","):
            count = re.search(r"\[(\d+)\]", name)
            fields.append((re.sub(r"[\[\]\d\s*]+$", "", name).strip(" *"), kind, int(count.group(1)) if count else 1))
    ctype = {"int": ctypes.c_int, "float": ctypes.c_float, "int64_t": ctypes.c_int64, "void*": ctypes.c_void_p}
    want = [(n, ctype[k] * c if c > 1 else ctype[k]) for n, k, c in fields]
    assert [n for n, _ in AttnDesc._fields_] == [n for n, _ in want]
    for (_, a), (_, b) in zip(AttnDesc._fields_, want):
        assert a is b or (ctypes.sizeof(a) == ctypes.sizeof(b) and a._type_ is b._type_)


def desc(**kw):
    from moe_b200._lib import AttnDesc

    good = dict(dtype=0, num_heads=8, num_kv_heads=2, head_dim=128, k_pool=4096, v_pool=8192, num_pages=4, page_size=16,
                max_seqs=4)
    good.update(kw)
    sections = good.pop("rope_sections", None)
    d = AttnDesc(**good)
    if sections:
        d.rope_sections = (ctypes.c_int * 3)(*sections)
    return d


INVALID, UNSUPPORTED = 1, 6


@pytest.mark.parametrize("kw,status,word", [
    (dict(dtype=2), UNSUPPORTED, "dtype"),
    (dict(head_dim=96), UNSUPPORTED, "head_dim"),
    (dict(num_heads=7), INVALID, "num_heads"),
    (dict(num_heads=0), INVALID, "num_heads"),
    (dict(num_kv_heads=0), INVALID, "num_heads"),
    (dict(num_heads=258, num_kv_heads=2), INVALID, "num_heads"),
    (dict(page_size=8), INVALID, "page_size"),
    (dict(page_size=48), INVALID, "page_size"),
    (dict(num_pages=0), INVALID, "num_pages"),
    (dict(num_pages=1 << 27), INVALID, "num_pages"),
    (dict(page_stride=8), INVALID, "page_stride"),
    (dict(page_stride=2 * 16 * 128 + 4), INVALID, "page_stride"),
    (dict(k_pool=0), INVALID, "pools"),
    (dict(v_pool=8200), INVALID, "pools"),
    (dict(scale=-1.0), INVALID, "scale"),
    (dict(scale=float("nan")), INVALID, "scale"),
    (dict(softcap=float("inf")), INVALID, "softcap"),
    (dict(window=-1), INVALID, "window"),
    (dict(rope_dim=24, rope_table=4096, rope_positions=4, rope_axes=1), INVALID, "rope_dim"),
    (dict(rope_dim=144, rope_table=4096, rope_positions=4, rope_axes=1), INVALID, "rope_dim"),
    (dict(rope_dim=64), INVALID, "rope_table"),
    (dict(rope_dim=64, rope_table=4096, rope_positions=0, rope_axes=1), INVALID, "rope_table"),
    (dict(rope_dim=64, rope_table=4096, rope_positions=4, rope_axes=2), INVALID, "rope_axes"),
    (dict(rope_dim=64, rope_table=4096, rope_positions=4, rope_axes=1, rope_pairs=2), INVALID, "rope_pairs"),
    (dict(rope_dim=64, rope_table=4096, rope_positions=4, rope_axes=3, rope_sections=(8, 8, 8)), INVALID, "sections"),
    (dict(rope_dim=64, rope_table=4096, rope_positions=4, rope_axes=3, rope_sections=(-8, 20, 20)), INVALID, "section"),
    (dict(q_norm=4100), INVALID, "norm"),
    (dict(q_norm=4096, norm_eps=-1.0), INVALID, "norm_eps"),
    (dict(max_seqs=0), INVALID, "max_seqs"),
    (dict(max_seqs=1 << 27), INVALID, "max_seqs"),
])
def test_create_refuses(kw, status, word):
    from moe_b200 import _lib

    out = ctypes.c_void_p(1)
    assert _lib.lib().moe_attn_create(ctypes.byref(desc(**kw)), ctypes.byref(out)) == status
    assert word in _lib.last_error() and not out.value


def test_null_arguments_are_refused():
    from moe_b200 import _lib

    L = _lib.lib()
    out = ctypes.c_void_p()
    assert L.moe_attn_create(None, ctypes.byref(out)) == INVALID
    assert L.moe_attn_create(ctypes.byref(desc()), None) == INVALID
    assert L.moe_attn_append(None, *[None, 0, 0] * 3, 1, None, None, None, 0, 0, None) == INVALID
    assert L.moe_attn_decode(None, None, 0, 0, None, None, 1, 1, None, None, None) == INVALID
    assert L.moe_attn_prefill(None, None, 0, 0, None, None, None, 1, 1, 1, None, None, None) == INVALID
    assert L.moe_attn_check(None, None) == INVALID
    assert L.moe_attn_device_bytes(None) == 0
    L.moe_attn_destroy(None)


def test_rope_table_and_page_slots_on_the_cpu():
    torch = pytest.importorskip("torch")
    import moe_b200 as M

    t = M.rope_table(16, 5, base=100.0, device="cpu")
    assert t.shape == (5, 8, 2) and t.dtype == torch.float32
    angle = torch.tensor(3 * 100.0 ** -0.25, dtype=torch.float64)
    assert torch.allclose(t[3, 2].double(), torch.stack([angle.cos(), angle.sin()]), atol=1e-7)
    scaled = M.rope_table(16, 5, inv_freq=[0.5] * 8, device="cpu")
    assert torch.allclose(scaled[2, 7], torch.stack([torch.cos(torch.tensor(1.0)), torch.sin(torch.tensor(1.0))]))
    table = torch.tensor([[5, 2], [7, 1]], dtype=torch.int32)
    slots = M.page_slots(table, torch.tensor([0, 0, 1]), torch.tensor([3, 17, 16]), 16)
    assert slots.tolist() == [5 * 16 + 3, 2 * 16 + 1, 1 * 16] and slots.dtype == torch.int64
