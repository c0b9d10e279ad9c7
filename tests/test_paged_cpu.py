"""CPU tests of the paged cache's entries: struct layouts, refusals of the C ABI (before any CUDA call),
and the PyTorch operators' schemas and fake implementations."""
import ctypes as C
import re
import subprocess
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fav4_bshd as F
from fav4_bshd import ops  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]
INVALID = F.CUDA_ERROR_INVALID_VALUE
A = 0x10000  # an aligned dummy address, never read: the checks fail first


def flat(struct, prefix=""):
    for name, kind in struct._fields_:
        at = getattr(struct, name).offset
        if issubclass(kind, C.Structure):
            yield from ((f"{name}.{n}", at + o) for n, o in flat(kind))
        else:
            yield name, at


@pytest.mark.parametrize("name,struct", [("Fav4PagedCache", F.PagedCache),
                                         ("Fav4PagedAppendArgs", F.PagedAppendArgs), ("Fav4PagedArgs", F.PagedArgs)])
def test_layout_matches_c_compiler(tmp_path, name, struct):
    fields = list(flat(struct))
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fav4_bshd.h"\nint main(void){\n'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {n}));\n' for n, _ in fields)
                   + f'printf("%zu\\n", sizeof({name}));return 0;}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)],
                   check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [o for _, o in fields] + [C.sizeof(struct)]


def cache(**kw):
    f = dict(k=A, v=A, page_table=A, seq_lens=A, page_stride=16 * 2 * 128, token_stride=2 * 128, head_stride=128,
             table_stride=8, batch=2, kv_heads=2, num_pages=20, page_size=16, max_pages=8)
    f.update(kw)
    return F.PagedCache(**f)


def paged_args(cache_kw=None, **kw):
    f = dict(q=A, o=A, lse=A, cu_seqlens_q=A, q_token_stride=8 * 128, q_head_stride=128, heads=8, max_sq=2, total_q=3,
             scale=0.1)
    f.update(kw)
    return F.PagedArgs(cache=cache(**(cache_kw or {})), **f)


def append_args(cache_kw=None, **kw):
    f = dict(q=A, k=A, v=A, q_out=A, cu_seqlens_q=A, cos_table=A, sin_table=A, q_token_stride=1536, q_head_stride=128,
             k_token_stride=1536, k_head_stride=128, v_token_stride=1536, v_head_stride=128, heads=8, total_q=3,
             rotary_dim=128, interleaved=0, table_rows=100)
    f.update(kw)
    return F.PagedAppendArgs(cache=cache(**(cache_kw or {})), **f)


CACHE_BAD = [dict(k=None), dict(v=None), dict(page_table=None), dict(seq_lens=None), dict(k=A + 8), dict(v=A + 2),
             dict(page_table=A + 2), dict(seq_lens=A + 1), dict(page_stride=-8), dict(token_stride=100),
             dict(head_stride=4), dict(table_stride=-1), dict(batch=0), dict(kv_heads=0), dict(num_pages=0),
             dict(page_size=0), dict(page_size=8), dict(page_size=40), dict(max_pages=0),
             dict(page_size=1024, max_pages=2 ** 21)]
PAGED_BAD = [dict(q=None), dict(o=None), dict(cu_seqlens_q=None), dict(q=A + 8), dict(o=A + 4), dict(lse=A + 2),
             dict(cu_seqlens_q=A + 3), dict(q_token_stride=12), dict(q_head_stride=-128), dict(heads=0), dict(heads=7),
             dict(heads=2 ** 24), dict(max_sq=0), dict(max_sq=4), dict(total_q=-1), dict(scale=0.0), dict(scale=-1.0),
             dict(scale=float("nan")), dict(scale=float("inf")), dict(prefix_pages=A), dict(prefix_len=A)]
PREFIX_BAD = [dict(max_prefix_pages=0), dict(prefix_pages=A + 2), dict(prefix_len=A + 1),
              dict(max_prefix_pages=2 ** 28)]
APPEND_BAD = [dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(q=A + 8), dict(k=A + 4), dict(v=A + 2),
              dict(q_out=A + 8), dict(cu_seqlens_q=None), dict(cu_seqlens_q=A + 2), dict(offsets=A + 2),
              dict(cos_table=None), dict(sin_table=None), dict(cos_table=A + 4), dict(sin_table=A + 8),
              dict(q_token_stride=4), dict(k_token_stride=-8), dict(v_head_stride=20), dict(heads=0), dict(total_q=-1),
              dict(rotary_dim=8), dict(rotary_dim=144), dict(rotary_dim=-16), dict(interleaved=2), dict(table_rows=0)]


@pytest.mark.parametrize("kw", CACHE_BAD, ids=str)
def test_bad_caches_are_refused(lib, kw):
    assert lib.fav4_bshd_forward_paged(C.byref(paged_args(kw)), 1, A, 1 << 30, None) == INVALID
    assert lib.fav4_bshd_paged_append(C.byref(append_args(kw)), None) == INVALID
    assert lib.fav4_bshd_paged_workspace_bytes(C.byref(paged_args(kw))) == 0


@pytest.mark.parametrize("kw", PAGED_BAD, ids=str)
def test_bad_attention_arguments_are_refused(lib, kw):
    a = paged_args(**kw)
    assert lib.fav4_bshd_forward_paged(C.byref(a), 1, A, 1 << 30, None) == INVALID
    assert lib.fav4_bshd_forward_shared_prefix(C.byref(a), 1, A, 1 << 30, None) == INVALID
    assert lib.fav4_bshd_paged_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("kw", PREFIX_BAD, ids=str)
def test_bad_prefixes_are_refused(lib, kw):
    a = paged_args(**{**dict(prefix_pages=A, prefix_len=A, max_prefix_pages=4), **kw})
    assert lib.fav4_bshd_forward_shared_prefix(C.byref(a), 0, A, 1 << 30, None) == INVALID


@pytest.mark.parametrize("kw", APPEND_BAD, ids=str)
def test_bad_append_arguments_are_refused(lib, kw):
    assert lib.fav4_bshd_paged_append(C.byref(append_args(**kw)), None) == INVALID


def test_modes_and_workspaces_are_checked(lib):
    a = paged_args()
    need = lib.fav4_bshd_paged_workspace_bytes(C.byref(a))
    assert need > 0
    with_prefix = paged_args(prefix_pages=A, prefix_len=A, max_prefix_pages=4)
    assert lib.fav4_bshd_paged_workspace_bytes(C.byref(with_prefix)) > need
    for causal, ws, size in ((2, A, need), (-1, A, need), (1, None, need), (1, A + 128, need), (1, A, need - 1)):
        assert lib.fav4_bshd_forward_paged(C.byref(a), causal, ws, size, None) == INVALID
    # each entry takes its own kind of call only
    assert lib.fav4_bshd_forward_paged(C.byref(with_prefix), 1, A, 1 << 30, None) == INVALID
    assert lib.fav4_bshd_forward_shared_prefix(C.byref(a), 1, A, 1 << 30, None) == INVALID
    for f in (lib.fav4_bshd_forward_paged, lib.fav4_bshd_forward_shared_prefix):
        assert f(None, 1, A, need, None) == INVALID
    assert lib.fav4_bshd_paged_append(None, None) == INVALID
    assert lib.fav4_bshd_paged_workspace_bytes(None) == 0
    # nothing to do is not an error
    none = paged_args(q=None, o=None, total_q=0, max_sq=0)
    assert lib.fav4_bshd_forward_paged(C.byref(none), 1, None, 0, None) == 0
    assert lib.fav4_bshd_paged_append(C.byref(append_args(q=None, k=None, v=None, q_out=None, total_q=0)), None) == 0


def fakes(t=5, h=8, hk=2, page=16, b=3):
    def new(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")
    i32 = torch.int32
    return dict(q=new(t, h, 128), kv=new(t, hk, 128), cache=new(20, page, hk, 128), table=new(b, 6, dtype=i32),
                lens=new(b, dtype=i32), cu=new(b + 1, dtype=i32), cos=new(100, 64, dtype=torch.float32),
                pages=new(4, dtype=i32), n=new(1, dtype=i32))


def test_fake_shapes():
    with FakeTensorMode():
        x = fakes()
        q = torch.ops.fav4.paged_append(x["q"], x["kv"], x["kv"], x["cache"], x["cache"].clone(), x["table"], x["lens"],
                                        x["cu"], x["cos"], x["cos"], False, None)
        assert q.shape == x["q"].shape and q.dtype == torch.bfloat16
        o, lse = torch.ops.fav4.paged_forward(q, x["cache"], x["cache"], x["table"], x["lens"], x["cu"], 2, True, -1.0)
        assert o.shape == q.shape and lse.shape == (8, 5) and lse.dtype == torch.float32
        o, lse = torch.ops.fav4.shared_prefix_forward(q, x["cache"], x["cache"], x["pages"], x["n"], x["table"],
                                                      x["lens"], x["cu"], 2, True, -1.0)
        assert o.shape == q.shape and lse.shape == (8, 5)


@pytest.mark.parametrize("change", [dict(page=24), dict(q="float"), dict(table="long"), dict(lens="short"),
                                    dict(cu="short"), dict(cache="dim")])
def test_fake_refusals(change):
    with FakeTensorMode():
        x = fakes(page=change.get("page", 16))
        if "q" in change:
            x["q"] = x["q"].float()
        if "table" in change:
            x["table"] = x["table"].long()
        if "lens" in change:
            x["lens"] = x["lens"][:1]
        if "cu" in change:
            x["cu"] = x["cu"][:2]
        if "cache" in change:
            x["cache"] = x["cache"][..., :64]
        with pytest.raises(RuntimeError):
            torch.ops.fav4.paged_forward(x["q"], x["cache"], x["cache"], x["table"], x["lens"], x["cu"], 2, True, -1.0)


def test_schema_says_what_is_written():
    schema = str(torch.ops.fav4.paged_append.default._schema)
    assert re.search(r"Tensor\(\w+!\) k_cache, Tensor\(\w+!\) v_cache", schema)


SIZES = [(8, 1, 1), (8, 4, 64), (8, 257, 2056), (16, 8, 8), (160, 1, 40), (7, 19, 300)]
TABLES = [dict(batch=b, kv_heads=hk, page_size=page, max_pages=n)
          for b in (1, 4, 64, 1000) for hk in (1, 2, 7, 8, 160) for page in (16, 128) for n in (1, 20, 512, 8192)]


@pytest.mark.parametrize("prefix", [False, True])
def test_workspace_depends_on_the_rows_alone(lib, prefix):
    # a server's batch and tables change from step to step: one workspace does for all of them
    def need(table, heads, max_sq, total_q, pages=4):
        more = dict(prefix_pages=A, prefix_len=A, max_prefix_pages=pages) if prefix else {}
        return lib.fav4_bshd_paged_workspace_bytes(C.byref(paged_args(table, heads=heads, max_sq=max_sq,
                                                                      total_q=total_q, **more)))

    for heads, max_sq, total_q in SIZES:
        sizes = {need(t, heads, max_sq, total_q, pages) for t in TABLES if heads % t["kv_heads"] == 0
                 for pages in (1, 4, 3000)}
        assert len(sizes) == 1 and min(sizes) > 0, (heads, max_sq, total_q, sizes)
        for more in ((2 * heads, max_sq, total_q), (heads, max_sq + 1, total_q + 1), (heads, max_sq, 3 * total_q)):
            assert need(dict(kv_heads=1), *more) >= max(sizes)


def test_kernels_do_not_read_through_the_non_coherent_path():
    # the kernels are resident while their predecessor writes what they read, so ld.global.nc is not theirs to use
    for path in (F.PKG_ROOT / "csrc").glob("paged*"):
        code = re.sub(r"//[^\n]*", "", path.read_text())
        assert not re.search(r"__ldg\b|\.nc\b|__restrict__", code), path.name


def test_the_stride_of_a_single_head_says_nothing():
    # one K/V head: storage with the heads inside and outside the pages is the same memory
    with FakeTensorMode():
        x = fakes(hk=1)
        outside = x["cache"].new_empty(20, 1, 16, 128).transpose(1, 2)
        assert outside.stride() != x["cache"].stride()
        o, lse = torch.ops.fav4.paged_forward(x["q"], x["cache"], outside, x["table"], x["lens"], x["cu"], 2, True, -1.0)
        assert o.shape == x["q"].shape
        two = fakes(hk=2)
        with pytest.raises(RuntimeError):
            torch.ops.fav4.paged_forward(two["q"], two["cache"], two["cache"].new_empty(20, 2, 16, 128).transpose(1, 2),
                                         two["table"], two["lens"], two["cu"], 2, True, -1.0)
