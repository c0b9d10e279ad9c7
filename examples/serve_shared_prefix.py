"""Serving from a paged key/value cache: conversations that share a system prompt.

One attention layer with random weights (BF16, rotated queries and keys, grouped heads), run the way a
server runs it: the system prompt is cached once, in chunks; every conversation's own prompt goes into
pages of its own behind it; then all conversations generate together, one token a step, as one captured
CUDA graph that is replayed with growing lengths.

    python examples/serve_shared_prefix.py [--conversations 16] [--prefix 1000] [--steps 24] [--check]

--check recomputes every conversation with the contiguous attention of the library and compares.
"""
import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "flash-attention-v4-rocm_b200"))
from fav4_bshd import ops, paged  # noqa: E402

D, PAGE = 128, 16


class Layer:
    """hidden -> attention -> hidden, without the rest of a transformer block."""

    def __init__(self, heads, kv_heads, width, gen):
        def init(*shape):
            return (torch.randn(*shape, generator=gen, device="cuda") / shape[0] ** 0.5).bfloat16()

        self.heads, self.kv_heads = heads, kv_heads
        self.qkv, self.out = init(width, (heads + 2 * kv_heads) * D), init(heads * D, width)

    def project(self, x):
        rows = (x @ self.qkv).view(-1, self.heads + 2 * self.kv_heads, D)
        return rows.split((self.heads, self.kv_heads, self.kv_heads), dim=1)

    def finish(self, o):
        return o.reshape(o.shape[0], -1) @ self.out


class Pages:
    """Hands out pages of one cache."""

    def __init__(self, count, kv_heads):
        self.k, self.v = (torch.empty(count, PAGE, kv_heads, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.free = list(range(count))

    def take(self, keys):
        return [self.free.pop() for _ in range(-(-keys // PAGE))]


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def rotation(positions):
    angle = torch.outer(torch.arange(positions, dtype=torch.float64), 10000.0 ** (-torch.arange(64) / 64.0))
    return angle.cos().float().cuda(), angle.sin().float().cuda()


@torch.no_grad()
def serve(layer, pages, cos, sin, prefix, prompts, steps, chunk):
    """Hidden states of the generated tokens [conversations, steps, width]; the next token's hidden state is the
    layer's output for the last one."""
    n, total = len(prompts), prefix.shape[0]
    # the system prompt, a chunk at a time
    prefix_pages = i32(pages.take(total))
    for a in range(0, total, chunk):
        rows = prefix[a:a + chunk]
        cu, lens = i32([0, rows.shape[0]]), i32([a + rows.shape[0]])
        paged.append(*layer.project(rows), pages.k, pages.v, prefix_pages[None], lens, cu, cos, sin)
    # the conversations' own prompts, packed, behind it
    own = [p.shape[0] for p in prompts]
    table = i32([pages.take(max(own) + steps) for _ in prompts])
    lens, cu, prefix_len = i32(own), i32([0] + own).cumsum(0).to(torch.int32), i32([total])
    shift = prefix_len.expand(n).contiguous()  # rotation positions go on from the prefix
    q = paged.append(*(layer.project(torch.cat(prompts))), pages.k, pages.v, table, lens, cu, cos, sin, offsets=shift)
    o = paged.shared_prefix_attention(q, pages.k, pages.v, prefix_pages, prefix_len, table, lens, cu, max(own))
    x = layer.finish(o)[cu[1:].long() - 1].clone()
    # one token a step, all conversations together
    ones = torch.arange(n + 1, dtype=torch.int32, device="cuda")

    def step():
        lens.add_(1)
        q = paged.append(*layer.project(x), pages.k, pages.v, table, lens, ones, cos, sin, offsets=shift)
        o = paged.shared_prefix_attention(q, pages.k, pages.v, prefix_pages, prefix_len, table, lens, ones, 1)
        x.copy_(layer.finish(o))

    start, begin = lens.clone(), x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the first call sets the kernels up, outside the capture
        step()
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(start), x.copy_(begin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    made = []
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(steps):
        made.append(x.clone())
        graph.replay()
    torch.cuda.synchronize()
    return torch.stack(made, dim=1), (time.perf_counter() - t) / steps


@torch.no_grad()
def recompute(layer, cos, sin, prefix, prompt, made):
    """The same states from one contiguous causal attention over everything that the conversation saw."""
    x = torch.cat((prefix, prompt, made))
    q, k, v = layer.project(x)
    c, s = cos[:x.shape[0], None], sin[:x.shape[0], None]

    def turn(z):
        a, b = z.float().chunk(2, dim=-1)
        return torch.cat((a * c - b * s, b * c + a * s), dim=-1).bfloat16()

    o = ops.attention(turn(q)[None], turn(k)[None], v.contiguous()[None], causal=True)[0]
    at = prefix.shape[0] + prompt.shape[0]
    return layer.finish(o)[at - 1:at - 1 + made.shape[0]]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--conversations", type=int, default=16)
    ap.add_argument("--prefix", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--kv-heads", type=int, default=2)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--chunk", type=int, default=256)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    gen = torch.Generator(device="cuda").manual_seed(0)
    layer = Layer(a.heads, a.kv_heads, a.width, gen)
    prefix = torch.randn(a.prefix, a.width, generator=gen, device="cuda").bfloat16()
    prompts = [torch.randn(3 + 17 * i % 150, a.width, generator=gen, device="cuda").bfloat16()
               for i in range(a.conversations)]
    longest = max(p.shape[0] for p in prompts) + a.steps
    pages = Pages(-(-a.prefix // PAGE) + a.conversations * (-(-longest // PAGE)) + 1, a.kv_heads)
    cos, sin = rotation(a.prefix + longest)
    made, seconds = serve(layer, pages, cos, sin, prefix, prompts, a.steps, a.chunk)
    print(f"{a.conversations} conversations behind {a.prefix} keys: {seconds * 1e6:.1f} us a step, "
          f"{a.conversations / seconds:.0f} tokens/s")
    if a.check:
        worst = 0.0
        for i, prompt in enumerate(prompts):
            want = recompute(layer, cos, sin, prefix, prompt, made[i])
            worst = max(worst, ((made[i].float() - want.float()).norm() / want.float().norm()).item())
        print(f"largest relative difference from the contiguous attention: {worst:.2e}")
        # two BF16 computations of the same states: each rounds P, O and the product, 2^-8 each
        if not worst < 2 ** -6:
            raise SystemExit("the results differ")


if __name__ == "__main__":
    main()
