"""Overlapped chains on the GPU: calls without a live expert between calls that have some, nothing waited for in between."""
import numpy as np
import pytest

from oracle import oracle as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [O.DT_Q8_0, O.DT_BF16])
def test_calls_without_a_live_expert_between_others(dtype):
    """A call whose ids are all empty has no CTA with work in its expert kernels, and the call behind it overwrites the plan.
    Every call gives the bits that it gives alone, and zeros where nothing is routed."""
    import moe_b200 as M

    rng = np.random.default_rng(9)
    E, k, H, I, T = 16, 4, 256, 128, 5
    q = [O.quantize(dtype, rng.normal(0, 0.02, s).astype(np.float32))[0] for s in ((E, I, H), (E, I, H), (E, H, I))]
    cfg = M.MoeConfig(num_experts=E, num_experts_per_tok=k, hidden_size=H, moe_intermediate_size=I)
    layer = M.RoutedExpertsProvider().build(M.ExpertLoadContext(
        layer=0, device=0, config=cfg, wdtype=dtype, gate=q[0], up=q[1], down=q[2], max_tokens=T))
    x = torch.from_numpy(rng.normal(0, 1, (T, H)).astype(np.float32)).cuda().to(torch.bfloat16)
    w = torch.from_numpy(rng.dirichlet(np.ones(k), T).astype(np.float32)).cuda()
    none = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    routed = [torch.from_numpy(np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)).cuda() for _ in range(6)]
    alone = []
    for ids in routed:
        alone.append(layer.forward(x, w, ids))
        torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for ids in routed:
            outs.append((layer.forward(x, w, none), layer.forward(x, w, none), layer.forward(x, w, ids)))
    torch.cuda.synchronize()
    layer.check()
    for i, (a, b, y) in enumerate(outs):
        assert not a.any() and not b.any() and torch.equal(y, alone[i % len(routed)]), i
