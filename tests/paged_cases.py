"""A paged cache for the tests, and the operators on it in 64 bits, written from their definitions."""
import math

import torch

D = 128
U = 2 ** -8  # unit roundoff of BF16 (8 significant bits): the largest relative error of one rounding


class Batch:
    """Sequences of `sq` new tokens whose caches hold `keys` keys, these tokens included, in shuffled pages.

    Pages that no sequence owns, the slots past each sequence's end and the unused table entries hold NaN
    (entries: -1), so anything that reads them shows."""

    def __init__(self, sq, keys, h, hk, page, seed, prefix=0, heads_outside=False, gap=0, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        self.sq, self.keys, self.h, self.hk, self.page, self.prefix = list(sq), list(keys), h, hk, page, prefix
        b = len(self.sq)
        need = [-(-n // page) for n in self.keys]
        n_pre = -(-prefix // page)
        pages = sum(need) + n_pre + 3
        order = torch.randperm(pages, generator=gen)
        width = max(max(need), 1) + gap
        self.table = torch.full((b, width), -1, dtype=torch.int32)
        at = n_pre
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.prefix_pages = order[:max(n_pre, 1)].to(torch.int32)
        nan = float("nan")
        shape = (pages, hk, page, D) if heads_outside else (pages, page, hk, D)
        self.k_cache, self.v_cache = (torch.full(shape, nan, dtype=torch.bfloat16) for _ in range(2))
        if heads_outside:
            self.k_cache, self.v_cache = self.k_cache.transpose(1, 2), self.v_cache.transpose(1, 2)
        # dense keys and values of each sequence (the prefix first), in 64 bits, as the cache holds them
        self.k, self.v = [], []
        pre = [torch.randn(prefix, hk, D, generator=gen).bfloat16() for _ in range(2)]
        for s in range(prefix):
            p, slot = int(self.prefix_pages[s // page]), s % page
            self.k_cache[p, slot], self.v_cache[p, slot] = pre[0][s], pre[1][s]
        for i, n in enumerate(self.keys):
            k, v = (torch.randn(n, hk, D, generator=gen).bfloat16() for _ in range(2))
            idx = torch.arange(n)
            rows = self.table[i].long()[idx // page]
            self.k_cache[rows, idx % page], self.v_cache[rows, idx % page] = k, v
            self.k.append(torch.cat((pre[0], k)).double())
            self.v.append(torch.cat((pre[1], v)).double())
        self.q = torch.randn(sum(self.sq), h, D, generator=gen).bfloat16()
        self.cu = torch.tensor([0] + self.sq).cumsum(0).to(torch.int32)
        self.lens = torch.tensor(self.keys, dtype=torch.int32)
        self.prefix_len = torch.tensor([prefix], dtype=torch.int32)
        self.max_sq = max(self.sq)
        for name in ("q", "cu", "lens", "table", "k_cache", "v_cache", "prefix_pages", "prefix_len"):
            x = getattr(self, name)
            setattr(self, name, x.to(device, memory_format=torch.preserve_format) if x.dim() == 4 else x.to(device))

    def reference(self, causal=True, scale=None):
        """O, LSE and the bound's weights P |V| in 64 bits."""
        scale = 1 / math.sqrt(D) if scale is None else scale
        o = torch.zeros(sum(self.sq), self.h, D, dtype=torch.float64)
        w = torch.zeros_like(o)
        lse = torch.full((self.h, sum(self.sq)), -math.inf, dtype=torch.float64)
        q = self.q.cpu().double()
        t = 0
        for i, (s, n) in enumerate(zip(self.sq, self.keys)):
            n += self.prefix
            if s and n:
                group = self.h // self.hk
                k = self.k[i].repeat_interleave(group, dim=1)
                v = self.v[i].repeat_interleave(group, dim=1)
                x = torch.einsum("shd,lhd->hsl", q[t:t + s], k) * scale
                if causal:
                    last = torch.arange(s)[:, None] + (n - s)
                    x = x.masked_fill((torch.arange(n) > last), -math.inf)
                m = x.amax(-1, keepdim=True)
                e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
                total = e.sum(-1, keepdim=True)
                e = e / torch.where(total == 0, 1.0, total)
                o[t:t + s] = torch.einsum("hsl,lhd->shd", e, v)
                w[t:t + s] = torch.einsum("hsl,lhd->shd", e, v.abs())
                lse[:, t:t + s] = (torch.where(m == -math.inf, 0.0, m) + total.log()).squeeze(-1)
            t += s
        return o, lse, w


def check_attention(o, lse, ref):
    """O: every probability is rounded to BF16 once and O once, each by at most U of itself; scores are FP32 sums of
    128 exact products, at most 128 * 2^-23 * sum |q k| * scale (about 10 for unit normals) off, 2^-12. LSE: that score
    error."""
    want_o, want_lse, w = ref
    o, lse = o.double().cpu(), lse.double().cpu()
    assert torch.isfinite(o).all()
    assert ((o - want_o).abs() <= (2 * U + 2 ** -12) * w).all(), ((o - want_o).abs() / w).max()
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (lse - want_lse)[~empty].abs().le(2 ** -12).all()


def tables(positions, rotary, device="cuda"):
    half = rotary // 2
    angle = torch.outer(torch.arange(positions, dtype=torch.float64),
                        10000.0 ** (-torch.arange(half, dtype=torch.float64) / half))
    return angle.cos().float().to(device), angle.sin().float().to(device)


def rotate64(x, cos, sin, interleaved):
    """R x in 64 bits for rows x [T, H, D] with cos / sin rows [T, rotary/2], and |x cos| + |y sin| of each element."""
    x, cos, sin = x.double().cpu(), cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    rotary = 2 * cos.shape[-1]
    out, size = x.clone(), torch.zeros_like(x)
    first, second = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else \
        (slice(0, rotary // 2), slice(rotary // 2, rotary))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first], size[..., second] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    return out, size


def check_rotated(got, want, size):
    """The BF16 value nearest to `want`, or to what three FP32 roundings (2^-21 of the terms) make of it."""
    got, slack = got.cpu(), 2 ** -21 * size
    assert (got >= (want - slack).bfloat16()).all() and (got <= (want + slack).bfloat16()).all()
