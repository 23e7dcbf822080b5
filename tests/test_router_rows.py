"""Router.route takes rows as they come: strided ones are copied, others than the gate's kind are refused (on the CPU, with a
stand-in for the library)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def router(monkeypatch):
    import moe_b200 as M
    from moe_b200 import layer

    class Library:
        seen = []

        def moe_route_workspace_bytes(self, T, E):
            return 64

        def moe_route_tokens(self, x, w, bias, T, H, *rest):
            self.seen.append(bytes(ctypes.string_at(x, T * H * 2)))
            return 0

    fake = Library()
    monkeypatch.setattr(layer, "lib", lambda: fake)
    monkeypatch.setattr(layer, "_stream", lambda stream=None: 0)
    return M.Router(torch.zeros((8, 32), dtype=torch.bfloat16), 2, 0, max_tokens=4), fake


def test_strided_rows_reach_the_kernel_as_rows(router):
    r, fake = router
    wide = torch.arange(3 * 64, dtype=torch.float32).view(3, 64).to(torch.bfloat16)
    for x in (wide[:, :32], wide[:, ::2], wide.t()[:32, :3].t()):
        del fake.seen[:]
        r.route(x)
        assert fake.seen == [x.contiguous().view(torch.int16).numpy().tobytes()]


@pytest.mark.parametrize("x", [torch.zeros((3, 16), dtype=torch.bfloat16), torch.zeros((3, 32)),
                               torch.zeros((1, 3, 32), dtype=torch.bfloat16), torch.zeros((5, 32), dtype=torch.bfloat16)])
def test_rows_of_another_kind_are_refused(router, x):
    import moe_b200 as M

    r, fake = router
    with pytest.raises(M.MoeError):
        r.route(x)
    assert not fake.seen
