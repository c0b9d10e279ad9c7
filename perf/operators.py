"""Serving from a paged key/value cache, measured operator by operator: the rotated append of new keys
and values, attention over the pages, and attention of a batch whose sequences share a long prefix.

Each case runs one operator. ``own = False`` computes it with elementary torch operations in 32 bits,
``own = True`` through this repository's ``fav4_bshd.paged``. Head dim 128, BF16, caches
``[pages, page_size, kv_heads, 128]``; sequence ``b`` has the query rows ``[cu[b], cu[b + 1])`` and
``seq_lens[b]`` keys (this step's included) at the pages ``table[b]``.

Fields of a case: ``op`` (append / attend / shared), ``batch``, ``heads``, ``kv_heads``, ``page``;
``sq_lo``..``sq_hi`` new tokens per sequence; ``ctx_lo``..``ctx_hi`` keys that were there before them;
``causal``; append: ``rotary`` (rotated elements per head) and ``interleaved`` (pairs (2i, 2i+1) rather
than (i, i + rotary/2)); shared: ``prefix`` keys that every sequence sees.
"""
import math
import sys
from pathlib import Path

import torch

own = False

D = 128
_HEADS = ((8, 8), (8, 2), (8, 1), (6, 3), (5, 5), (4, 4))
_PAGES = (16, 32, 48, 64, 128)


def _case(name, op, batch, heads, kv_heads, page, sq, ctx, causal=True, rotary=128, interleaved=False, prefix=0):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "page": page,
            "sq_lo": sq[0], "sq_hi": sq[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "causal": causal, "rotary": rotary,
            "interleaved": interleaved, "prefix": prefix}


def listed():
    return [
        # one decode step of a full batch: a few hundred kilobytes, all latency
        _case("append decode b128", "append", 128, 8, 2, 16, (1, 1), (100, 8192)),
        # packed prompt chunks of odd lengths, half of each head rotated, pairs interleaved
        _case("append ragged b7", "append", 7, 6, 3, 48, (129, 1537), (0, 1000), rotary=64, interleaved=True),
        # the prompts of a whole batch at once
        _case("append prompt b32", "append", 32, 8, 8, 64, (4096, 4096), (0, 0)),
        # the next token of one conversation: latency
        _case("decode b1", "attend", 1, 8, 8, 16, (1, 1), (8191, 8191)),
        # a serving batch of very unlike lengths with grouped heads
        _case("decode ragged b32", "attend", 32, 8, 2, 16, (1, 1), (1, 32767)),
        # a full batch of long conversations, every head its own keys: bandwidth
        _case("decode b64", "attend", 64, 8, 8, 64, (1, 1), (8192, 24576)),
        # drafted tokens verified together, one key head for all query heads
        _case("verify b16", "attend", 16, 8, 1, 32, (3, 7), (1000, 16384)),
        # prompt chunks of odd lengths behind odd contexts
        _case("chunk ragged b3", "attend", 3, 6, 3, 48, (700, 1000), (0, 1537)),
        # a long prompt's last chunk: matrix products
        _case("chunk 4096 of 32768", "attend", 1, 8, 2, 64, (4096, 4096), (28672, 28672)),
        # a few questions on one short document
        _case("shared b8", "shared", 8, 8, 8, 16, (1, 1), (0, 100), prefix=1000),
        # a batch behind a long system prompt, one token each
        _case("shared b64", "shared", 64, 8, 2, 16, (1, 1), (16, 2048), prefix=32768),
        # a wide batch on one very long document, short chunks
        _case("shared b128 long", "shared", 128, 8, 1, 64, (1, 4), (0, 1000), prefix=131072),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "shared"))
    heads, kv_heads = rng.choice(_HEADS)
    c = _case("", op, 1, heads, kv_heads, rng.choice(_PAGES), (1, 1), (0, 0))
    del c["name"]
    if op == "append":
        c["batch"] = _spread(rng, 1, 128)
        c["sq_hi"] = _spread(rng, 1, min(4096, 131072 // c["batch"]))
        c["ctx_hi"] = _spread(rng, 1, 4096)
        c["rotary"], c["interleaved"] = rng.choice((128, 128, 96, 64, 32)), rng.random() < 0.3
    elif op == "attend" and rng.random() < 0.6:  # next tokens
        c["batch"] = _spread(rng, 1, 64)
        c["sq_hi"] = rng.choice((1, 1, 1, 2, 5, 8))
        c["ctx_hi"] = _spread(rng, 16, 32768)
    elif op == "attend":  # prompt chunks
        c["batch"] = _spread(rng, 1, 8)
        c["sq_hi"] = _spread(rng, 17, 4096 // c["batch"])
        c["ctx_hi"] = _spread(rng, 1, 28672)
        c["causal"] = rng.random() < 0.8
    else:
        c["batch"] = _spread(rng, 2, 128)
        c["sq_hi"] = rng.choice((1, 1, 1, 3, 8))
        c["ctx_hi"] = _spread(rng, 1, 2048)
        c["prefix"] = _spread(rng, 100, min(131072, 131072 * 8 * 4 // (heads * c["sq_hi"])))
    c["sq_lo"] = rng.choice((c["sq_hi"], (c["sq_hi"] + 1) // 2, 1))
    c["ctx_lo"] = rng.choice((c["ctx_hi"], c["ctx_hi"] // 2, 0))
    return c


def _lengths(case):
    """New tokens and keys of each sequence: evenly spread over their ranges, in a mixed order."""
    b = case["batch"]

    def over(lo, hi, ratio):
        order = sorted(range(b), key=lambda i: (i * ratio) % 1.0)
        return [lo + i * (hi - lo) // max(1, b - 1) for i in order]

    sq = over(case["sq_lo"], case["sq_hi"], 0.6180339887498949)
    ctx = over(case["ctx_lo"], case["ctx_hi"], 0.4142135623730951)
    return sq, [s + c for s, c in zip(sq, ctx)]


def work(case):
    sq, keys = _lengths(case)
    tokens, h, hk = sum(sq), case["heads"], case["kv_heads"]
    row = 2 * D
    index = 4 * (2 * case["batch"] + 1 + sum(-(-n // case["page"]) for n in keys))
    if case["op"] == "append":
        # q, k, v in and out; a cos and a sin row for each position; one multiplication and one
        # multiplication-addition per rotated element
        seen = set()
        for s, n in zip(sq, keys):
            seen.update(range(n - s, n))
        table = 4 * case["rotary"] * len(seen)
        return {"bytes": 2 * tokens * (h + 2 * hk) * row + table + index,
                "flops": 3 * tokens * (h + hk) * case["rotary"]}
    if case["causal"]:
        pairs = sum(s * n - s * (s - 1) // 2 for s, n in zip(sq, keys))
    else:
        pairs = sum(s * n for s, n in zip(sq, keys))
    pairs += tokens * case["prefix"]
    read = (sum(keys) + case["prefix"]) * hk * 2 * row
    return {"bytes": read + 2 * tokens * h * row + 4 * tokens * h + index, "flops": 4 * D * h * pairs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    sq, keys = _lengths(case)
    tokens, h, hk, page, b = sum(sq), case["heads"], case["kv_heads"], case["page"], case["batch"]
    per_seq = [-(-n // page) for n in keys]
    shared = -(-case["prefix"] // page)
    pages = sum(per_seq) + shared + 8
    order = torch.randperm(pages, generator=host).to(torch.int32)
    table = torch.full((b, max(max(per_seq), 1)), -1, dtype=torch.int32)
    at = shared
    for i, n in enumerate(per_seq):
        table[i, :n] = order[at:at + n]
        at += n

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    state = {"case": case, "max_sq": max(sq), "max_keys": max(keys), "table": table.cuda(),
             "cu": torch.tensor([0] + sq).cumsum(0).to(torch.int32).cuda(),
             "lens": torch.tensor(keys, dtype=torch.int32).cuda(),
             "k_cache": randn(pages, page, hk, D), "v_cache": randn(pages, page, hk, D)}
    if case["op"] == "append":
        # one row per token out of the projection: its query heads, then its key and value heads
        state["qkv"] = randn(tokens, h + 2 * hk, D)
        half = case["rotary"] // 2
        angle = torch.outer(torch.arange(max(keys), dtype=torch.float64),
                            10000.0 ** (-torch.arange(half, dtype=torch.float64) / half))
        state["cos"], state["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    else:
        state["q"] = randn(tokens, h, D)
    if case["op"] == "shared":
        state["prefix_pages"] = order[:shared].cuda()
        state["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32).cuda()
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    paged = _package()
    case = state["case"]
    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        q, k, v = state["qkv"].split((h, hk, hk), dim=1)
        out = paged.append(q, k, v, state["k_cache"], state["v_cache"], state["table"], state["lens"], state["cu"],
                           state["cos"], state["sin"], interleaved=case["interleaved"])
        return out, state["k_cache"], state["v_cache"]
    if case["op"] == "attend":
        return paged.attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lens"],
                               state["cu"], state["max_sq"], causal=case["causal"], return_lse=True)
    return paged.shared_prefix_attention(state["q"], state["k_cache"], state["v_cache"], state["prefix_pages"],
                                         state["prefix_len"], state["table"], state["lens"], state["cu"],
                                         state["max_sq"], causal=case["causal"], return_lse=True)


def _package():
    if "fav4_bshd.paged" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "flash-attention-v4-rocm_b200"))
        import fav4_bshd.paged  # noqa: F401
    return sys.modules["fav4_bshd.paged"]


def _rows(cu, tokens):
    """Sequence of each packed row, and the row's place in it."""
    t = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu[1:], t.to(cu.dtype), right=True)
    return seq, t - cu[seq]


def _run_plain(state):
    return _append_plain(state) if state["case"]["op"] == "append" else _attend_plain(state)


def _append_plain(state):
    case, cu = state["case"], state["cu"].long()
    h, hk, page, rotary = case["heads"], case["kv_heads"], case["page"], case["rotary"]
    q, k, v = state["qkv"].split((h, hk, hk), dim=1)
    seq, i = _rows(cu, q.shape[0])
    pos = state["lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + i
    cos, sin = state["cos"][pos, None], state["sin"][pos, None]

    def rotate(x):
        x = x.float()
        r, rest = x[..., :rotary], x[..., rotary:]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = r[..., :rotary // 2], r[..., rotary // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((r, rest), dim=-1).to(torch.bfloat16)

    where = (state["table"].long()[seq, pos // page], pos % page)
    state["k_cache"][where] = rotate(k)
    state["v_cache"][where] = v
    return rotate(q), state["k_cache"], state["v_cache"]


def _attend_plain(state):
    case, cu, lens = state["case"], state["cu"].long(), state["lens"].long()
    h, hk, page, b, s = case["heads"], case["kv_heads"], case["page"], case["batch"], state["max_sq"]
    tokens, n, dev = state["q"].shape[0], state["max_keys"], cu.device
    seq, i = _rows(cu, tokens)
    q = torch.zeros(b, s, hk, h // hk, D, device=dev)
    q[seq, i] = state["q"].float().view(tokens, hk, h // hk, D)
    q *= 1 / math.sqrt(D)
    table = state["table"].long()[:, :-(-n // page)].clamp(min=0)
    k = state["k_cache"][table].flatten(1, 2)[:, :n].float()
    scores = torch.einsum("bshgd,blhd->bhgsl", q, k)
    del k
    key = torch.arange(n, device=dev)
    seen = (key < lens[:, None])[:, None, :]
    if case["causal"]:
        pos = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(s, device=dev)
        seen = seen & (key <= pos[:, :, None])
    scores.masked_fill_(~seen[:, None, None].expand(b, 1, 1, s, n), -math.inf)
    m = scores.amax(-1, keepdim=True)
    if case["op"] == "shared":
        before = state["k_cache"][state["prefix_pages"].long()].flatten(0, 1)[:case["prefix"]].float()
        scores_before = torch.einsum("bshgd,lhd->bhgsl", q, before)
        m = torch.maximum(m, scores_before.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)
    p = scores.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgsl,blhd->bhgsd", p, state["v_cache"][table].flatten(1, 2)[:, :n].float())
    if case["op"] == "shared":
        p = scores_before.sub_(m).exp_()
        total = total + p.sum(-1, keepdim=True)
        before = state["v_cache"][state["prefix_pages"].long()].flatten(0, 1)[:case["prefix"]].float()
        o = o + torch.einsum("bhgsl,lhd->bhgsd", p, before)
    o = o / torch.where(total > 0, total, 1.0)
    lse = (m + total.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, s, h, D)[seq, i].to(torch.bfloat16)
    lse = lse.permute(0, 3, 1, 2).reshape(b, s, h)[seq, i].t().contiguous()
    return o, lse


def exact(case, seed):
    """What run() returns, from the definitions, sequence by sequence in 64 bits."""
    st = prepare(case, seed)
    sq, keys = _lengths(case)
    h, hk, page = case["heads"], case["kv_heads"], case["page"]
    f64 = torch.float64
    k_pool, v_pool = st["k_cache"], st["v_cache"]
    if case["op"] == "append":
        rotary = case["rotary"]
        k_new, v_new = k_pool.to(f64), v_pool.to(f64)
        q_new = st["qkv"][:, :h].to(f64)
        first, second = (slice(0, rotary, 2), slice(1, rotary, 2)) if case["interleaved"] else \
            (slice(0, rotary // 2), slice(rotary // 2, rotary))
        t = 0
        for i, (s, n) in enumerate(zip(sq, keys)):
            at = torch.arange(n - s, n, device="cuda")
            turn = torch.complex(st["cos"][at].to(f64), st["sin"][at].to(f64))[:, None]
            block = st["qkv"][t:t + s].to(f64)
            z = turn * torch.complex(block[:, :h + hk, first].contiguous(), block[:, :h + hk, second].contiguous())
            block[:, :h + hk, first], block[:, :h + hk, second] = z.real, z.imag
            rows = st["table"][i].long()[torch.div(at, page, rounding_mode="floor")]
            q_new[t:t + s] = block[:, :h]
            k_new[rows, at % page] = block[:, h:h + hk]
            v_new[rows, at % page] = block[:, h + hk:]
            t += s
        return q_new, k_new, v_new
    o = torch.empty(sum(sq), h, D, dtype=f64, device="cuda")
    lse = torch.empty(h, sum(sq), dtype=f64, device="cuda")
    head = torch.arange(h, device="cuda") // (h // hk)
    pre = case["prefix"]
    t = 0
    for i, (s, n) in enumerate(zip(sq, keys)):
        at = torch.arange(n, device="cuda")
        rows = st["table"][i].long()[torch.div(at, page, rounding_mode="floor")]
        k, v = k_pool[rows, at % page], v_pool[rows, at % page]
        if pre:
            at = torch.arange(pre, device="cuda")
            rows = st["prefix_pages"].long()[torch.div(at, page, rounding_mode="floor")]
            k, v = torch.cat((k_pool[rows, at % page], k)), torch.cat((v_pool[rows, at % page], v))
        k, v = k.to(f64).permute(1, 2, 0), v.to(f64).transpose(0, 1)
        step = max(1, 2 ** 27 // (h * (pre + n)))
        for a in range(0, s, step):
            z = min(s, a + step)
            x = st["q"][t + a:t + z].to(f64).transpose(0, 1) @ k[head] / math.sqrt(D)
            if case["causal"]:
                last = torch.arange(a, z, device="cuda")[:, None] + (pre + n - s)
                x = x.where(torch.arange(pre + n, device="cuda") <= last, -math.inf)
            lse[:, t + a:t + z] = x.logsumexp(-1)
            o[t + a:t + z] = (x.softmax(-1) @ v[head]).transpose(0, 1)
        t += s
    return o, lse
