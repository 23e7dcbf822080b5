"""A decoder stack served from the library: paged attention next to the routed experts.

Each layer is  x += attention(norm(x));  x += experts(norm(x))  with
  * q, k, v and output projections (plain matrix products, torch),
  * PagedAttention.append / prefill / decode over the layer's page pools,
  * RoutedExperts.route / forward for the MoE block.
Weights are random; the point is the calls and their order. A ragged batch of prompts is prefilled in one pass, then
decoded token by token with continuous lengths; the decode step is captured in a CUDA graph and replayed.

  python examples/decoder_layer.py                         # small: two layers, seconds
  python examples/decoder_layer.py --hidden 2048 --heads 32 --kv-heads 4 --experts 128 --inter 768 --layers 4 \\
      --seqs 32 --lo 128 --hi 2048 --steps 64
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "naiwa-rs_b200"))

import torch  # noqa: E402

import moe_b200 as M  # noqa: E402
from moe_b200 import synth  # noqa: E402

PAGE = 16


def norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Layer:
    def __init__(self, a, index, pages, rope, device="cuda"):
        g = torch.Generator(device=device).manual_seed(index)
        D, H = a.head_dim, a.hidden

        def weight(rows, cols):
            return (torch.randn((rows, cols), generator=g, device=device) * cols ** -0.5).to(torch.bfloat16)

        self.qkv, self.out = weight((a.heads + 2 * a.kv_heads) * D, H), weight(H, a.heads * D)
        self.heads, self.kv_heads, self.dim = a.heads, a.kv_heads, D
        pools = M.kv_pools(pages, a.kv_heads, PAGE, D)
        ones = torch.ones(D, dtype=torch.bfloat16, device=device)
        self.attention = M.PagedAttention(
            M.AttentionConfig(num_heads=a.heads, num_kv_heads=a.kv_heads, head_dim=D, rope_dim=D), *pools,
            rope_table=rope, q_norm=ones, k_norm=ones, max_seqs=a.seqs)
        cfg = M.MoeConfig(num_experts=a.experts, num_experts_per_tok=a.top_k, hidden_size=H,
                          moe_intermediate_size=a.inter)
        gate, up, down = synth.expert_stacks(a.experts, H, a.inter, M.DTYPE_Q8_0, 0.02, seed=100 + index, device=device)
        router = synth.router_weight(a.experts, H, 0.02, seed=200 + index, device=device)
        self.experts = M.RoutedExpertsProvider().build(M.ExpertLoadContext(
            layer=index, device=0, config=cfg, wdtype=M.DTYPE_Q8_0, gate=gate, up=up, down=down, router_weight=router,
            max_tokens=a.seqs * a.hi))

    def __call__(self, x, batch):
        qkv = (norm(x) @ self.qkv.t()).view(x.shape[0], -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = self.attention.append(q, k, v, batch["positions"], batch["slots"])
        if "cu_q" in batch:
            y = self.attention.prefill(q, batch["cu_q"], batch["lens"], batch["table"])
        else:
            y = self.attention.decode(q, batch["lens"], batch["table"])
        x = x + y.flatten(1) @ self.out.t()
        h = norm(x)
        ids, w = self.experts.route(h)
        return x + self.experts.forward(h, w, ids)

    def check(self):
        self.attention.check()
        self.experts.check()


class Stack:
    def __init__(self, a):
        g = torch.Generator().manual_seed(a.seed)
        self.prompts = torch.randint(a.lo, a.hi + 1, (a.seqs,), generator=g).tolist()
        width = -(-(max(self.prompts) + a.steps) // PAGE)
        # pages in any order: a real server hands them out as sequences grow
        self.table = torch.randperm(a.seqs * width, generator=g).to(torch.int32).view(a.seqs, width).cuda()
        rope = M.rope_table(a.head_dim, a.hi + a.steps, base=1e6)
        self.layers = [Layer(a, i, a.seqs * width, rope) for i in range(a.layers)]

    def run(self, x, batch):
        for layer in self.layers:
            x = layer(x, batch)
        return x

    def batch(self, first, rows):
        """The rows that follow `first` cached tokens of each sequence (lists, per sequence)."""
        seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
        pos = torch.cat([torch.arange(f, f + r) for f, r in zip(first, rows)]).to(torch.int32).cuda()
        return {"positions": pos, "slots": M.page_slots(self.table, seq.cuda(), pos, PAGE), "table": self.table,
                "lens": torch.tensor([f + r for f, r in zip(first, rows)], dtype=torch.int32, device="cuda")}

    def prefill(self, x, first, rows):
        batch = self.batch(first, rows)
        ends = torch.tensor([0] + rows).cumsum(0)
        batch["cu_q"] = ends.to(torch.int32).cuda()
        return self.run(x, batch)

    def decoder(self, seqs, hidden):
        """A captured decode step: fill .x, .positions, .slots and .lens, replay, read .y."""
        step = argparse.Namespace(
            x=torch.zeros((seqs, hidden), dtype=torch.bfloat16, device="cuda"),
            batch={"positions": torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                   "slots": torch.full((seqs,), -1, dtype=torch.int64, device="cuda"),
                   "lens": torch.zeros(seqs, dtype=torch.int32, device="cuda"), "table": self.table})
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.run(step.x, step.batch)  # warm-up; slot -1 and length 0: padding, nothing is stored
        torch.cuda.current_stream().wait_stream(side)
        step.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(step.graph):
            step.y = self.run(step.x, step.batch)
        return step

    def decode(self, step, x, lens):
        """One token per sequence behind lens[b] cached ones."""
        batch = self.batch(lens, [1] * len(lens))
        step.x.copy_(x)
        for name in ("positions", "slots", "lens"):
            step.batch[name].copy_(batch[name])
        step.graph.replay()
        return step.y.clone()


def arguments(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 2), ("hidden", 512), ("heads", 8), ("kv-heads", 2), ("head-dim", 128), ("experts", 16),
                        ("top-k", 4), ("inter", 256), ("seqs", 5), ("lo", 3), ("hi", 70), ("steps", 8), ("seed", 0)):
        p.add_argument("--" + name, type=int, default=value)
    return p.parse_args(argv)


def main(argv=None):
    a = arguments(argv)
    stack = Stack(a)
    total = sum(stack.prompts)
    g = torch.Generator(device="cuda").manual_seed(a.seed)
    x = torch.randn((total, a.hidden), generator=g, device="cuda").to(torch.bfloat16)  # the prompts' embeddings
    y = stack.prefill(x, [0] * a.seqs, stack.prompts)
    last = torch.tensor(stack.prompts).cumsum(0).cuda() - 1
    step = stack.decoder(a.seqs, a.hidden)
    lens, h = list(stack.prompts), norm(y[last])
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(a.steps):  # the last hidden state stands in for the next token's embedding
        h = norm(stack.decode(step, h, lens))
        lens = [n + 1 for n in lens]
    end.record()
    torch.cuda.synchronize()
    for layer in stack.layers:
        layer.check()
    print(f"{a.layers} layers, {a.seqs} sequences, {total} prompt tokens prefilled, {a.steps} decode steps of "
          f"{start.elapsed_time(end) / a.steps:.3f} ms (host bookkeeping included)")
    return h


if __name__ == "__main__":
    main()
