"""GPU tests of the paged cache: append with rotation, attention over pages and behind a shared prefix,
against their definitions in 64 bits (tests/paged_cases.py)."""
import ctypes as C
import math

import pytest
import torch

import fav4_bshd as F
from fav4_bshd import paged
from paged_cases import D, U, Batch, check_attention, check_rotated, rotate64, tables

pytestmark = pytest.mark.gpu


def attend(x, causal=True, **kw):
    return paged.attention(x.q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, x.max_sq, causal=causal, return_lse=True,
                           **kw)


def attend_shared(x, causal=True, **kw):
    return paged.shared_prefix_attention(x.q, x.k_cache, x.v_cache, x.prefix_pages, x.prefix_len, x.table, x.lens,
                                         x.cu, x.max_sq, causal=causal, return_lse=True, **kw)


# new tokens, keys (new ones included), heads, K/V heads, page size
SHAPES = [
    ([1], [1], 8, 8, 16),
    ([1], [8192], 8, 8, 16),
    ([1, 1, 1], [15, 16, 17], 8, 2, 16),
    ([1, 1, 1, 1], [63, 64, 65, 1000], 6, 3, 48),
    ([1] * 33, [1 + 37 * i for i in range(33)], 8, 1, 32),
    ([2, 5, 1], [130, 5, 700], 8, 1, 64),            # 8 to 40 rows per K/V head
    ([0, 3, 0, 1], [40, 3, 0, 77], 8, 2, 16),        # sequences without new tokens
    ([1, 2, 4], [0, 1, 2], 4, 4, 16),                # no keys, and more tokens than keys: empty rows
    ([17, 128, 129], [17, 300, 1000], 6, 3, 48),
    ([300], [1537], 5, 5, 128),
    ([1000, 1, 33], [1000, 2049, 500], 8, 2, 64),
    ([257, 64], [257, 129], 12, 4, 16),              # a group of 3
    ([40, 1], [600, 64], 7, 1, 16),                  # a group of 7
    ([5, 70], [300, 333], 160, 1, 32),               # more query heads per K/V head than a tile has rows
    ([512], [4000], 8, 8, 256),
    # chunks among sequences of a key or none, whose units of one step lie at the blocks' boundaries
    ([1, 0, 121, 14, 1, 77, 383, 2, 1, 1, 0, 2, 1, 2, 348, 0, 2, 209, 1, 1, 473, 2, 1, 461, 1, 369, 2, 2, 1, 0, 1, 0, 1],
     [786, 10, 846, 324, 497, 354, 815, 453, 0, 706, 540, 277, 933, 525, 650, 834, 759, 385, 626, 987, 1149, 2, 956, 655,
      892, 1304, 970, 143, 452, 246, 698, 406, 979], 3, 3, 32),
    # two tiles per block
    ([700, 1000, 850], [700, 2387, 1500], 6, 3, 48),
    ([2100, 1], [2100, 900], 8, 8, 64),
    ([513, 30], [1700, 30], 8, 2, 16),
    ([700, 5, 90], [690, 3, 1000], 12, 4, 32),       # a group of 3, rows before the first key
    ([129, 600], [0, 777], 40, 2, 16),               # a group of 20; a sequence without keys
]


@pytest.mark.parametrize("sq,keys,h,hk,page", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention(cuda, sq, keys, h, hk, page, causal):
    x = Batch(sq, keys, h, hk, page, seed=sum(keys) + h)
    o, lse = attend(x, causal)
    check_attention(o, lse, x.reference(causal))


@pytest.mark.parametrize("sq,keys,h,hk,page", [SHAPES[3], SHAPES[5], SHAPES[8], SHAPES[10]])
def test_heads_outside_pages_and_wide_tables(cuda, sq, keys, h, hk, page):
    # [pages][heads][slots][128] storage, tables with unused columns, and O the same bits as the other layout's
    x = Batch(sq, keys, h, hk, page, seed=3, heads_outside=True, gap=5)
    assert x.k_cache.stride(2) > x.k_cache.stride(1)
    o, lse = attend(x)
    check_attention(o, lse, x.reference())
    x.k_cache, x.v_cache = x.k_cache.contiguous(), x.v_cache.contiguous()
    again, lse_again = attend(x)
    assert torch.equal(o, again) and torch.equal(lse, lse_again)


PREFIXED = [
    ([1] * 8, [1, 2, 17, 40, 64, 65, 99, 100], 8, 8, 16, 1000),
    ([1] * 40, [1 + 13 * i for i in range(40)], 8, 2, 16, 4097),
    ([1, 4, 2, 0], [5, 300, 2, 9], 8, 1, 64, 131),
    ([30, 1, 70], [30, 90, 100], 6, 3, 48, 15),
    ([1, 1], [0, 3], 4, 4, 32, 64),                   # a sequence without keys of its own
    ([3, 2], [1, 0], 4, 2, 16, 0),                    # no prefix keys: empty rows stay empty
    ([200, 100], [200, 150], 8, 2, 64, 777),
    ([9], [20], 160, 1, 16, 333),
    ([300, 260], [300, 700], 8, 2, 64, 1500),        # two tiles per block for the prefix
    ([9] * 30, [9 + 7 * i for i in range(30)], 8, 1, 16, 2500),
]


@pytest.mark.parametrize("sq,keys,h,hk,page,prefix", PREFIXED)
@pytest.mark.parametrize("causal", [True, False])
def test_shared_prefix(cuda, sq, keys, h, hk, page, prefix, causal):
    x = Batch(sq, keys, h, hk, page, seed=prefix + h, prefix=prefix)
    if causal and prefix:  # rows past the own keys' mask still see the whole prefix: the definition of the call
        keys_cover = all(n >= s for s, n in zip(sq, keys))
        if not keys_cover:
            pytest.skip("the reference's mask counts from the end of all keys")
    o, lse = attend_shared(x, causal)
    check_attention(o, lse, x.reference(causal))


def test_shared_prefix_seen_by_rows_without_own_keys(cuda):
    # seq_lens < sq: the first rows see none of their own keys but all of the prefix, as a dense call over it
    x = Batch([4, 1], [2, 0], 8, 2, 16, seed=5, prefix=90)
    o, lse = attend_shared(x)
    dense = Batch([4, 1], [2, 0], 8, 2, 16, seed=5, prefix=90)
    dense.k, dense.v = [k[:90] for k in dense.k], [v[:90] for v in dense.v]
    dense.keys = [0, 0]
    want_o, want_lse, w = dense.reference(causal=False)
    rows = [0, 1, 4]
    check_attention(o[rows], lse[:, rows], (want_o[rows], want_lse[:, rows], w[rows]))


def test_table_rows_shared_by_sequences(cuda):
    # an expanded table (stride 0): every sequence reads the same pages
    x = Batch([1], [500], 8, 2, 16, seed=8)
    b = 5
    q = torch.randn(b, 8, D, device=cuda).bfloat16()
    o = paged.attention(q, x.k_cache, x.v_cache, x.table.expand(b, -1), x.lens.repeat(b),
                        torch.arange(b + 1, dtype=torch.int32, device=cuda), 1)
    for i in range(b):
        one = paged.attention(q[i:i + 1], x.k_cache, x.v_cache, x.table, x.lens, x.cu, 1)
        ref = Batch([1], [500], 8, 2, 16, seed=8)
        ref.q = q[i:i + 1]
        want, _, w = ref.reference()
        for got in (o[i:i + 1], one):
            assert ((got.double().cpu() - want).abs() <= (2 * U + 2 ** -12) * w).all()


@pytest.mark.parametrize("sq,keys", [([1] * 6, [9, 100, 1000, 64, 65, 3000]), ([40, 1, 300], [40, 900, 1100])])
def test_matches_contiguous_attention(cuda, runner, sq, keys):
    # the same problem through the packed entry: dense, so that the two mask conventions agree
    x = Batch(sq, keys, 8, 2, 16, seed=4)
    o, lse = attend(x, causal=False)
    k = torch.cat(x.k).bfloat16().cuda()
    v = torch.cat(x.v).bfloat16().cuda()
    cu_k = torch.tensor([0] + keys, device=cuda).cumsum(0).to(torch.int32)
    want, want_lse = torch.empty_like(x.q), torch.empty(8, sum(sq), device=cuda)
    runner.call_varlen(x.q, k, v, want, want_lse, x.cu, cu_k, max(sq), False)
    _, _, w = x.reference(False)
    assert ((o.double() - want.double()).abs().cpu() <= 2 * (2 * U + 2 ** -10) * w).all()
    assert (lse - want_lse).abs().max() <= 1e-3


def test_scale_and_large_scores(cuda):
    x = Batch([1, 3], [700, 50], 8, 2, 16, seed=6)
    o, lse = attend(x, scale=0.5)
    want_o, want_lse, w = x.reference(scale=0.5)
    # scores are 0.5 sqrt(128) = 5.7 times those of check_attention, and so is their error
    assert ((o.double().cpu() - want_o).abs() <= (2 * U + 6 * 2 ** -12) * w).all()
    assert (lse.double().cpu() - want_lse).abs().max() <= 6 * 2 ** -12


def test_rising_maximum(cuda):
    # keys whose scores grow along the sequence: the running maximum moves in every step
    x = Batch([1, 20], [900, 900], 4, 2, 16, seed=7)
    x.q = torch.ones_like(x.q)
    for i in range(2):
        for s in range(900):
            p, slot = int(x.table[i, s // 16]), s % 16
            value = torch.full((2, D), s / 64.0, dtype=torch.bfloat16)
            x.k_cache[p, slot] = value.cuda()
            x.k[i][s] = value.double()
    o, lse = attend(x)
    want_o, want_lse, w = x.reference()
    # scores up to 159; products and sums are exact, one FP32 rounding by scale log2 e: 160 * 2^-23
    assert ((o.double().cpu() - want_o).abs() <= (2 * U + 2 ** -12) * w).all()
    assert (lse.double().cpu() - want_lse).abs().max() <= 1e-4


def test_nan_of_a_visible_key_shows_and_stays_in_its_rows(cuda):
    x = Batch([1, 1], [100, 100], 4, 2, 16, seed=9)
    x.k_cache[int(x.table[1, 2]), 3, 0] = float("nan")
    o, lse = attend(x)
    ref_o, ref_lse, w = x.reference()
    assert torch.isnan(o[1, :2]).all() and torch.isnan(lse[:2, 1]).all()
    keep = torch.ones(2, 4, dtype=torch.bool)
    keep[1, :2] = False
    assert ((o.double().cpu() - ref_o).abs()[keep] <= ((2 * U + 2 ** -12) * w)[keep]).all()


def test_same_bits_every_time(cuda):
    for x in (Batch([1] * 17, [1 + 211 * i for i in range(17)], 8, 2, 16, seed=1), Batch([200], [5000], 8, 1, 64, seed=2)):
        first = attend(x)
        for _ in range(5):
            again = attend(x)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_two_streams(cuda):
    # each stream has a workspace of its own: calls in flight together do not disturb one another
    xs = [Batch([1] * 8, [3000 + 100 * i for i in range(8)], 8, 2, 16, seed=s) for s in (11, 12)]
    want = [attend(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for j, x in enumerate(xs):
            with torch.cuda.stream(streams[j]):
                got[j].append(attend(x))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, want[j][0]) and torch.equal(lse, want[j][1]) for o, lse in got[j])


def test_graph_replays_with_other_lengths(cuda):
    x = Batch([1, 1, 1], [400, 30, 999], 8, 2, 16, seed=13)
    out, lse = torch.empty_like(x.q), None
    attend(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = attend(x)
    for shorter in (0, 7, 29):
        x.lens.copy_(torch.tensor([400 - shorter, 30 - shorter, 999 - shorter], dtype=torch.int32))
        g.replay()
        eager = attend(x)
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


def test_malformed_tables_stay_inside(cuda):
    # page numbers outside the cache, lengths past the table, offsets out of order: no access outside, no hang
    x = Batch([3, 1, 40], [200, 90, 60], 8, 2, 16, seed=14)
    good = Batch([3, 1, 40], [200, 90, 60], 8, 2, 16, seed=14)
    x.k_cache.nan_to_num_(0), x.v_cache.nan_to_num_(0)
    x.table[0, :] = torch.tensor([-5, 2 ** 30] * x.table.shape[1], dtype=torch.int32)[:x.table.shape[1]]
    x.lens[1] = 2 ** 30
    x.lens[2] = -7
    out = attend(x)
    x.cu.copy_(torch.tensor([5, -3, 2 ** 30, 2], dtype=torch.int32))
    attend(x)
    cos, sin = tables(16, 128)
    k = torch.randn(44, 2, D, device=cuda).bfloat16()
    paged.append(x.q, k, k, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin)
    torch.cuda.synchronize()
    assert torch.isfinite(out[0]).all() and (out[1][:, 4:] == -math.inf).all()
    o, lse = attend(good)  # the workspace is none the worse for it
    check_attention(o, lse, good.reference())


# ------------------------------------------------------------------------------------------- append
APPENDS = [
    ([1], [1], 8, 8, 16, 128, False),
    ([1] * 40, [1 + 33 * i for i in range(40)], 8, 2, 16, 128, False),
    ([5, 0, 70, 1], [5, 9, 200, 17], 6, 3, 48, 64, True),
    ([33, 100], [500, 100], 5, 5, 64, 96, False),
    ([3, 2], [20, 2], 4, 1, 32, 16, True),
    ([3, 2], [20, 2], 4, 1, 32, 0, False),
    ([2, 1], [900, 40], 160, 1, 16, 128, True),
]


def do_append(x, rotary, interleaved, cuda, offsets=None, fused=True):
    cos, sin = tables(2048, rotary) if rotary else (None, None)
    gen = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(sum(x.sq), x.h + 2 * x.hk, D, generator=gen, device=cuda).bfloat16()
    q, k, v = qkv.split((x.h, x.hk, x.hk), dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    out = paged.append(q, k, v, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin, interleaved=interleaved,
                       offsets=offsets)
    return q, k, v, out, cos, sin


@pytest.mark.parametrize("sq,keys,h,hk,page,rotary,interleaved", APPENDS)
@pytest.mark.parametrize("heads_outside,shifted", [(False, False), (True, True)])
def test_append(cuda, sq, keys, h, hk, page, rotary, interleaved, heads_outside, shifted):
    x = Batch(sq, keys, h, hk, page, seed=21, heads_outside=heads_outside)
    before = x.k_cache.clone(), x.v_cache.clone()
    offsets = torch.arange(3, 3 + len(sq), dtype=torch.int32, device=cuda) if shifted else None
    q, k, v, out, cos, sin = do_append(x, rotary, interleaved, cuda, offsets, fused=not shifted)
    written = torch.zeros(x.k_cache.shape[:2], dtype=torch.bool, device=cuda)
    t = 0
    for i, (s, n) in enumerate(zip(sq, keys)):
        pos = torch.arange(n - s, n, device=cuda)
        page_of, slot = x.table[i].long()[pos // page], pos % page
        written[page_of, slot] = True
        new_k, new_v = x.k_cache[page_of, slot], x.v_cache[page_of, slot]
        assert torch.equal(new_v, v[t:t + s])
        if rotary:
            at = pos + (int(offsets[i]) if shifted else 0)
            check_rotated(out[t:t + s], *rotate64(q[t:t + s], cos[at], sin[at], interleaved))
            check_rotated(new_k, *rotate64(k[t:t + s], cos[at], sin[at], interleaved))
        else:
            assert torch.equal(out[t:t + s], q[t:t + s]) and torch.equal(new_k, k[t:t + s])
        t += s
    for now, then in zip((x.k_cache, x.v_cache), before):  # every other slot is as it was, NaN included
        assert torch.equal(now[~written].view(torch.int16), then[~written].view(torch.int16))


def test_append_in_place_of_q(cuda):
    x = Batch([7, 1], [30, 99], 8, 2, 16, seed=22)
    q, k, v, out, cos, sin = do_append(x, 128, False, cuda, fused=False)
    mine = q.clone()
    paged.append(mine, k, v, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin, out=mine)
    assert torch.equal(mine, out)


def test_append_without_a_slot_writes_nothing(cuda):
    # more tokens than keys (negative positions), no page (-1), positions past the table
    x = Batch([4, 2, 1], [2, 40, 33], 8, 2, 16, seed=23)
    x.table[1, 2] = -1           # keys 32..47 of sequence 1 have no page
    x.lens[2] = 16 * x.table.shape[1] + 1000
    before = x.k_cache.clone()
    cos, sin = tables(64, 128)
    k = torch.ones(7, 2, D, device=cuda).bfloat16()
    out = paged.append(x.q, k, k, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin)
    torch.cuda.synchronize()
    changed = (x.k_cache.view(torch.int16) != before.view(torch.int16)).any(-1).any(-1)
    want = torch.zeros_like(changed)
    want[int(x.table[0, 0]), 0] = want[int(x.table[0, 0]), 1] = True
    assert torch.equal(changed, want)
    assert torch.isfinite(out).all()


def test_append_then_attend_equals_contiguous(cuda, runner):
    # prompt in two chunks, then three single tokens, against one causal forward of the whole sequence
    h, hk, page, total = 8, 2, 16, 203
    gen = torch.Generator(device="cuda").manual_seed(31)
    qkv = torch.randn(total, h + 2 * hk, D, generator=gen, device=cuda).bfloat16()
    cos, sin = tables(total, 128)
    pages = -(-total // page)
    table = torch.randperm(pages + 2, generator=torch.Generator().manual_seed(1))[:pages].to(torch.int32).cuda()[None]
    kc, vc = (torch.full((pages + 2, page, hk, D), float("nan"), device=cuda, dtype=torch.bfloat16) for _ in range(2))
    outs, qs, t = [], [], 0
    for n in (150, 50, 1, 1, 1):
        q, k, v = qkv[t:t + n].split((h, hk, hk), dim=1)
        t += n
        lens = torch.tensor([t], dtype=torch.int32, device=cuda)
        cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        qr = paged.append(q, k, v, kc, vc, table, lens, cu, cos, sin)
        outs.append(paged.attention(qr, kc, vc, table, lens, cu, n))
        qs.append(qr)
    at = torch.arange(total)
    k_all, v_all = (c[table[0].long().cpu()[at // page], at % page][None].contiguous() for c in (kc, vc))
    q_all, got = torch.cat(qs)[None], torch.cat(outs)[None]
    want = torch.empty_like(q_all)
    runner.call_gqa(q_all, k_all, v_all, want, None, True)
    torch.cuda.synchronize()
    assert (got.float() - want.float()).abs().max() <= 3e-2  # two BF16 results of the same definition


# ------------------------------------------------------------------------------- operators and refusals
def test_torch_operators(cuda):
    from fav4_bshd import ops  # noqa: F401
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=41, prefix=33)
    cos, sin = tables(64, 128)
    k = torch.randn(3, 2, D, device=cuda).bfloat16()
    y = Batch([2, 1], [50, 40], 8, 2, 16, seed=41, prefix=33)
    q = torch.ops.fav4.paged_append(x.q, k, k, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin, False, None)
    want = paged.append(y.q, k, k, y.k_cache, y.v_cache, y.table, y.lens, y.cu, cos, sin)
    assert torch.equal(q, want)
    assert torch.equal(x.k_cache.view(torch.int16), y.k_cache.view(torch.int16))
    o, lse = torch.ops.fav4.paged_forward(q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2, True, -1.0)
    w = paged.attention(q, y.k_cache, y.v_cache, y.table, y.lens, y.cu, 2, return_lse=True)
    assert torch.equal(o, w[0]) and torch.equal(lse, w[1])
    o, lse = torch.ops.fav4.shared_prefix_forward(q, x.k_cache, x.v_cache, x.prefix_pages, x.prefix_len, x.table,
                                                  x.lens, x.cu, 2, True, -1.0)
    w = paged.shared_prefix_attention(q, y.k_cache, y.v_cache, y.prefix_pages, y.prefix_len, y.table, y.lens, y.cu, 2,
                                      return_lse=True)
    assert torch.equal(o, w[0]) and torch.equal(lse, w[1])
    torch.library.opcheck(torch.ops.fav4.paged_forward.default,
                          (q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2, True, -1.0),
                          test_utils=("test_schema", "test_faketensor"))


def test_nothing_to_do(cuda):
    x = Batch([0, 0], [5, 9], 4, 2, 16, seed=42)
    o, lse = attend(x)
    assert o.shape == (0, 4, D) and lse.shape == (4, 0)
    paged.append(x.q, x.q[:, :2], x.q[:, :2], x.k_cache, x.v_cache, x.table, x.lens, x.cu)


@pytest.mark.parametrize("break_it", [
    lambda x: setattr(x, "q", x.q.float()),
    lambda x: setattr(x, "q", x.q[..., :64]),
    lambda x: setattr(x, "q", x.q[:, :3]),                       # heads not a multiple of the K/V heads
    lambda x: setattr(x, "lens", x.lens.long()),
    lambda x: setattr(x, "lens", x.lens[:1]),
    lambda x: setattr(x, "table", x.table.cpu()),
    lambda x: setattr(x, "cu", x.cu[:2]),
    lambda x: setattr(x, "v_cache", x.v_cache[:-1]),
    lambda x: (setattr(x, "k_cache", x.k_cache[:, :8]), setattr(x, "v_cache", x.v_cache[:, :8])),
    lambda x: setattr(x, "k_cache", x.k_cache.transpose(1, 2).contiguous().transpose(1, 2)),
])
def test_refusals(cuda, break_it):
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=43)
    break_it(x)
    with pytest.raises(RuntimeError):
        attend(x)


def test_small_workspace_is_refused(cuda, lib):
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=44)
    o, ws = torch.full_like(x.q, 7.0), torch.zeros(1 << 20, dtype=torch.uint8, device=cuda)
    c = F.PagedCache(x.k_cache.data_ptr(), x.v_cache.data_ptr(), x.table.data_ptr(), x.lens.data_ptr(),
                     *x.k_cache.stride()[:3], x.table.stride(0), 2, 2, x.k_cache.shape[0], 16, x.table.shape[1])
    a = F.PagedArgs(c, x.q.data_ptr(), o.data_ptr(), None, x.cu.data_ptr(), None, None, *x.q.stride()[:2], 8, 2, 3, 0, 0.1)
    need = lib.fav4_bshd_paged_workspace_bytes(C.byref(a))
    assert need > ws.numel()
    assert lib.fav4_bshd_forward_paged(C.byref(a), 1, ws.data_ptr(), ws.numel(), None) == F.CUDA_ERROR_INVALID_VALUE
    ws = torch.zeros(need, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.fav4_bshd_forward_paged(C.byref(a), 1, ws.data_ptr(), need, stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(o, paged.attention(x.q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2, scale=0.1))
    assert (ws[:4096] == 0).all()  # the counters, as they were
    assert lib.fav4_bshd_pipeline_status(1) == 0


def test_inputs_that_want_a_gradient_are_refused(cuda):
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=45)
    q = x.q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        paged.attention(q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2)
    with torch.no_grad():
        paged.attention(q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2)


def test_two_graphs_and_eager_calls_do_not_share_a_workspace(cuda):
    # captured one after the other on one stream, replayed on two others, eager calls between
    xs = [Batch([1, 1], [3000, 900], 8, 2, 16, seed=s) for s in (51, 52)]
    want = [attend(x) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attend(x))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = attend(xs[0])
    torch.cuda.synchronize()
    for got, ref in (*zip(outs, want), (eager, want[0])):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("sq,keys", [([1, 1], [5000, 5000]), ([40, 40], [5000, 5000])])
def test_nan_query_shows_in_its_rows_only(cuda, sq, keys):
    # also where a row's keys are split over many blocks
    x = Batch(sq, keys, 4, 2, 16, seed=53)
    x.q[0, 1] = float("nan")
    o, lse = attend(x)
    assert torch.isnan(o[0, 1]).all() and torch.isnan(lse[1, 0])
    o[0, 1], lse[1, 0] = 0, 0
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()


def test_many_short_sequences(cuda):
    # more sequences than one scan step, and blocks whose stretch has more pieces than are listed at a time
    b = 4500
    keys = [1 + i % 3 for i in range(b)]
    x = Batch([1] * b, keys, 8, 8, 16, seed=54)
    o, lse = attend(x)
    check_attention(o, lse, x.reference())


@pytest.mark.parametrize("sq,keys,bound", [([3, 1, 6], [300, 40, 5], 2), ([90, 20, 300], [500, 20, 310], 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_past_the_bound_are_left_alone(cuda, sq, keys, bound, causal):
    # max_sq below a sequence's rows: the first rows are right, the others are not written
    x = Batch(sq, keys, 8, 2, 16, seed=55)
    out = torch.full_like(x.q, 7.0)
    o, lse = paged.attention(x.q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, bound, causal=causal, out=out,
                             return_lse=True)
    want_o, want_lse, w = x.reference(causal)
    rows = torch.cat([torch.arange(int(a), int(a) + min(n, bound)) for a, n in zip(x.cu.cpu(), sq)])
    check_attention(o[rows], lse[:, rows], (want_o[rows], want_lse[:, rows], w[rows]))
    left = torch.ones(sum(sq), dtype=torch.bool)
    left[rows] = False
    assert (o[left] == 7.0).all()


@pytest.mark.parametrize("sq", [1, 5, 40])
def test_offsets_past_32_bits(cuda, sq):
    # pages whose elements lie beyond 2^31 (and bytes beyond 2^32) of a cache
    h, hk, page, n = 8, 2, 64, 300
    pages = 2 ** 31 // (page * hk * D) + 40
    k_cache, v_cache = (torch.empty(pages, page, hk, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    small = Batch([sq], [n], h, hk, page, seed=56)
    last = small.k_cache.shape[0]
    k_cache[-last:], v_cache[-last:] = small.k_cache, small.v_cache
    table = (small.table + (pages - last)).to(torch.int32)
    o, lse = paged.attention(small.q, k_cache, v_cache, table, small.lens, small.cu, sq, return_lse=True)
    check_attention(o, lse, small.reference())
    k = torch.randn(sq, hk, D, device=cuda).bfloat16()
    paged.append(small.q, k, -k, k_cache, v_cache, table, small.lens, small.cu)
    at = torch.arange(n - sq, n, device=cuda)
    rows = table[0].long()[at // page]
    assert torch.equal(k_cache[rows, at % page], k) and torch.equal(v_cache[rows, at % page], -k)


def test_every_input_that_wants_a_gradient_is_refused(cuda):
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=61)
    q, k, v, _, cos, sin = do_append(x, 128, False, cuda, fused=False)
    wants = lambda t: t.clone().requires_grad_()
    appends = [q, k, v, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin]
    for i in (0, 1, 2, 3, 4, 8, 9):
        with pytest.raises(RuntimeError, match="no gradient"):
            paged.append(*[wants(t) if j == i else t for j, t in enumerate(appends)])
    attends = [x.q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2]
    for i in (0, 1, 2):
        with pytest.raises(RuntimeError, match="no gradient"):
            paged.attention(*[wants(t) if j == i else t for j, t in enumerate(attends)])
    with pytest.raises(RuntimeError, match="no gradient"):
        paged.attention(*attends, out=wants(x.q))


def test_results_that_overlap_an_input_are_refused(cuda):
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=62)
    q, k, v, _, cos, sin = do_append(x, 128, False, cuda, fused=False)
    cache = (x.k_cache, x.v_cache, x.table, x.lens, x.cu)
    both = torch.zeros(4, 8, D, dtype=torch.bfloat16, device=cuda)
    for out in (both[:3], both[1:]):
        with pytest.raises(RuntimeError, match="overlap"):
            paged.attention(both[:3], *cache, 2, out=out)
    with pytest.raises(RuntimeError, match="not a part"):
        paged.append(both[:3], k, v, *cache, cos, sin, out=both[1:])
    wide = torch.zeros(3, 12, D, dtype=torch.bfloat16, device=cuda)  # out over a projection's slices
    with pytest.raises(RuntimeError, match="not a part"):
        paged.append(wide[:, :8], wide[:, 8:10], wide[:, 10:], *cache, cos, sin, out=wide.view(-1)[:3 * 8 * D].view(3, 8, D))
    with pytest.raises(RuntimeError, match="overlap k or v"):
        paged.append(q, both.view(-1)[:3 * 2 * D].view(3, 2, D), v, *cache, cos, sin, out=both[:3])
    paged.attention(both[:3], *cache, 2, out=torch.empty_like(both[:3]))


# prefix and own keys on the 16-row kernel; the prefix on the tile kernel; both on it, with one tile and with two
NAN_BEHIND = [
    ([1] * 8, [0, 2, 17, 0, 64, 65, 99, 100], 8, 8, 16, 300),
    ([1] * 40, [0] + [13 * i for i in range(39)], 8, 2, 16, 1500),
    ([30, 1, 40], [2, 0, 50], 6, 3, 48, 777),
    ([30, 1, 70], [2, 0, 90], 6, 3, 48, 777),
    ([300, 260], [5, 0], 8, 2, 64, 1500),
]


@pytest.mark.parametrize("sq,keys,h,hk,page,prefix", NAN_BEHIND)
def test_nan_query_behind_a_prefix_shows_in_its_rows_only(cuda, sq, keys, h, hk, page, prefix):
    # rows that see no own key take the prefix's result as it is, NaN included
    x = Batch(sq, keys, h, hk, page, seed=71, prefix=prefix)
    first = [int(a) for a in x.cu[:-1]]
    for t in first:
        x.q[t, 1] = float("nan")
    o, lse = attend_shared(x)
    assert torch.isnan(o[first, 1]).all() and torch.isnan(lse[1, first]).all()
    o[first, 1], lse[1, first] = 0, 0
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("sq,keys,h,hk,page,prefix", NAN_BEHIND)
def test_nan_of_a_prefix_key_shows_in_every_row_of_its_heads(cuda, sq, keys, h, hk, page, prefix):
    x = Batch(sq, keys, h, hk, page, seed=72, prefix=prefix)
    s = prefix // 2
    x.k_cache[int(x.prefix_pages[s // page]), s % page, 0] = float("nan")
    o, lse = attend_shared(x)
    heads = h // hk
    assert torch.isnan(o[:, :heads]).all() and torch.isnan(lse[:heads]).all()
    assert torch.isfinite(o[:, heads:]).all() and torch.isfinite(lse[heads:]).all()


def test_written_tensors_tell_autograd(cuda):
    # a tensor that an expression saved for its backward is not overwritten unnoticed
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=73)
    q, k, v, _, cos, sin = do_append(x, 128, False, cuda, fused=False)
    cache = (x.k_cache, x.v_cache, x.table, x.lens, x.cu)
    one = torch.ones((), dtype=torch.bfloat16, device=cuda, requires_grad=True)

    def raises(saved, call):
        loss = (one * saved).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()

    for saved in (x.k_cache, x.v_cache, x.k_cache[1:]):
        raises(saved, lambda: paged.append(q, k, v, *cache, cos, sin))
    out = torch.zeros_like(q)
    raises(out, lambda: paged.append(q, k, v, *cache, cos, sin, out=out))
    raises(out, lambda: paged.attention(q, *cache, 2, out=out))
    versions = [t._version for t in (q, k, v, *cache)]
    paged.attention(q, *cache, 2)
    assert versions == [t._version for t in (q, k, v, *cache)]  # what is only read stays as it is
    with torch.inference_mode():  # tensors without a version
        a, b = x.k_cache.clone(), x.v_cache.clone()
        paged.append(q, k, v, a, b, *cache[2:], cos, sin, out=torch.empty_like(q))
        paged.append(q, k, v, *cache, cos, sin)
        assert torch.equal(a.view(torch.int16), x.k_cache.view(torch.int16))


def test_inputs_with_a_tangent_are_refused(cuda):
    # forward-mode derivatives, which torch.no_grad() does not turn off
    import torch.autograd.forward_ad as fwd
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=74)
    q, k, v, _, cos, sin = do_append(x, 128, False, cuda, fused=False)
    appends = [q, k, v, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin]
    attends = [x.q, x.k_cache, x.v_cache, x.table, x.lens, x.cu, 2]
    with fwd.dual_level():
        for call, args, places in ((paged.append, appends, (0, 1, 2, 3, 4, 8, 9)), (paged.attention, attends, (0, 1, 2))):
            for i in places:
                dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="no gradient"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                    call(*dual)
        paged.attention(*attends)
    paged.attention(*attends)


def test_results_that_overlap_the_caches_are_refused(cuda):
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=77)
    q, k, v, _, cos, sin = do_append(x, 128, False, cuda, fused=False)
    cache = (x.k_cache, x.v_cache, x.table, x.lens, x.cu)
    for c in (x.k_cache, x.v_cache):
        rows = c.view(-1)
        for out in (rows[:q.numel()].view_as(q), rows[-q.numel():].view_as(q)):
            with pytest.raises(RuntimeError, match="overlap the caches"):
                paged.attention(q, *cache, 2, out=out)
            with pytest.raises(RuntimeError, match="overlap the caches"):
                paged.shared_prefix_attention(q, *cache[:2], x.prefix_pages, x.prefix_len, *cache[2:], 2, out=out)
            with pytest.raises(RuntimeError, match="overlap the caches"):
                paged.append(q, k, v, *cache, cos, sin, out=out)
    pool = torch.zeros(2 * x.k_cache.numel() + q.numel(), dtype=torch.bfloat16, device=cuda)  # neighbours are no overlap
    n = x.k_cache.numel()
    k_cache, out, v_cache = (part.view(like.shape) for part, like in
                             zip(pool.split((n, q.numel(), n)), (x.k_cache, q, x.v_cache)))
    k_cache.copy_(x.k_cache), v_cache.copy_(x.v_cache)
    assert torch.equal(paged.attention(q, k_cache, v_cache, *cache[2:], 2, out=out), paged.attention(q, *cache, 2))


def test_the_stride_of_a_single_head_says_nothing(cuda):
    # one K/V head: storage with the heads inside and outside the pages is the same memory
    x = Batch([20, 1], [50, 40], 8, 1, 16, seed=78)
    want = attend(x)
    x.v_cache = x.v_cache.view(-1, 1, 16, D).transpose(1, 2)
    assert x.v_cache.stride() != x.k_cache.stride()
    got = attend(x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# a prefix of the 16-row kernel and own tables much wider than it, or wide for the lengths: the own keys of such a
# call share the SMs with the end of the prefix, each launch with counters and pieces of its own
WIDE_OWN = [
    ([1] * 8, [4000 - 531 * i for i in range(8)], 8, 8, 16, 300, 0),
    ([1] * 8, [0, 3, 1, 40, 64, 65, 99, 100], 8, 8, 16, 1000, 256),
    ([1, 1], [700, 9000], 4, 4, 32, 2500, 0),
]


@pytest.mark.parametrize("sq,keys,h,hk,page,prefix,gap", WIDE_OWN)
@pytest.mark.parametrize("causal", [True, False])
def test_shared_prefix_before_wide_tables(cuda, sq, keys, h, hk, page, prefix, gap, causal):
    x = Batch(sq, keys, h, hk, page, seed=75, prefix=prefix, gap=gap)
    ref = x.reference(causal=False)  # one token a sequence sees every key, with the mask or without
    first = attend_shared(x, causal)
    check_attention(*first, ref)
    for _ in range(10):
        again = attend_shared(x, causal)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_operators_that_write_and_share(cuda):
    from fav4_bshd import ops  # noqa: F401
    x = Batch([2, 1], [50, 40], 8, 2, 16, seed=76, prefix=33)
    x.k_cache.nan_to_num_(0), x.v_cache.nan_to_num_(0)  # the check compares what is not written
    cos, sin = tables(64, 128)
    qkv = torch.randn(3, 12, D, device=cuda).bfloat16()
    q, k, v = qkv.split((8, 2, 2), dim=1)
    utils = ("test_schema", "test_faketensor")
    for offsets in (None, torch.tensor([3, 5], dtype=torch.int32, device=cuda)):
        torch.library.opcheck(torch.ops.fav4.paged_append.default,
                              (q, k, v, x.k_cache, x.v_cache, x.table, x.lens, x.cu, cos, sin, False, offsets),
                              test_utils=utils)
    torch.library.opcheck(torch.ops.fav4.paged_append.default,
                          (q, k, v, x.k_cache, x.v_cache, x.table, x.lens, x.cu, None, None, False, None),
                          test_utils=utils)
    torch.library.opcheck(torch.ops.fav4.shared_prefix_forward.default,
                          (x.q, x.k_cache, x.v_cache, x.prefix_pages, x.prefix_len, x.table, x.lens, x.cu, 2, True, -1.0),
                          test_utils=utils)
