"""CPU: refusals of the 4-bit cache's and page planning's calls (Python and C ABI), rotary tables, and their oracle."""
import ctypes as C
import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from b200kernels import _lib
from b200kernels.page_plan import PageTables, StepPlan
from b200kernels.paged_int4 import (PagedKVInt4, paged_int4_append, paged_int4_attention, paged_int4_attention_workspace,
                                    paged_int4_read, rotary_tables)
from oracle.int4_ref import plan_ref, quantise_ref, values_ref

OK, ARG, SHAPE, DTYPE, ALIGN = 0, 1, 2, 3, 4
HALF, U8 = torch.float16, torch.uint8


def pool(pages=4, kvh=2, ps=16, D=64, dtype=HALF, **kw):
    return PagedKVInt4.empty(pages, kvh, ps, D, dtype, "cpu", **kw)


def refused(call, match, err=ValueError):
    with pytest.raises(err, match=match):
        call()


def test_pool_refusals():
    refused(lambda: pool(dtype=torch.float32), "fp16 or bf16", TypeError)
    for kw in (dict(D=96), dict(group_size=16), dict(group_size=128), dict(ps=8), dict(ps=24), dict(ps=1040), dict(ps=0)):
        refused(lambda: pool(**kw), "groups|multiple of 16")
    block = PagedKVInt4.page_bytes(16, 64)
    assert block == 16 * (32 + 4) * 2 == _lib.load().b2d_int4_page_bytes(16, 64, 64)
    assert _lib.load().b2d_int4_page_bytes(24, 64, 64) == 0
    make = lambda t: PagedKVInt4(t, 16, 64, HALF)  # noqa: E731
    refused(lambda: make(torch.zeros(4, 2, block, dtype=torch.int8)), "uint8", TypeError)
    refused(lambda: make(torch.zeros(4, 2, block + 16, dtype=U8)), r"\[num_pages")
    refused(lambda: make(torch.zeros(4, block, dtype=U8)), r"\[num_pages")
    refused(lambda: make(torch.zeros(4, block, 2, dtype=U8).transpose(1, 2)), "contiguous")
    refused(lambda: make(torch.zeros(4, 0, block, dtype=U8)), "no heads")
    one = torch.zeros(1, 1, block, dtype=U8)
    refused(lambda: make(one.expand(2 ** 31, 1, block)), "2\\^31")
    refused(lambda: make(one.expand(1, 2 ** 32 + 2, block)), "2\\^31")


def append_args(N=2, H=4, kvh=2, D=64, B=2):
    return dict(q=torch.zeros(N, H, D).half(), k=torch.zeros(N, kvh, D).half(), v=torch.zeros(N, kvh, D).half(),
                positions=torch.zeros(N, dtype=torch.int64), page_table=torch.zeros(B, 3, dtype=torch.int32),
                cos=torch.zeros(32, D // 2), sin=torch.zeros(32, D // 2))


@pytest.mark.parametrize("change,err", [
    (dict(q=torch.zeros(2, 4, 32).half()), ValueError),
    (dict(q=torch.zeros(3, 4, 64).half()), ValueError),
    (dict(q=torch.zeros(2, 3, 64).half()), ValueError),             # 3 heads over 2 KV heads
    (dict(k=torch.zeros(3, 2, 64).half()), ValueError),
    (dict(k=torch.zeros(2, 128).half()), ValueError),
    (dict(v=torch.zeros(2, 2, 64)), TypeError),
    (dict(q=torch.zeros(2, 4, 64).bfloat16()), TypeError),
    (dict(k=torch.zeros(2, 2, 64).bfloat16(), q=None), TypeError),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), ValueError),   # 2 tokens over 3 sequences
    (dict(seq_ids=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(cos=None), ValueError),
    (dict(cos=torch.zeros(32, 64), sin=torch.zeros(32, 64)), ValueError),  # R of 128 in heads of 64
    (dict(cos=torch.zeros(32, 12), sin=torch.zeros(32, 12)), ValueError),  # R of 24
    (dict(cos=torch.zeros(32, 0), sin=torch.zeros(32, 0)), ValueError),
    (dict(sin=torch.zeros(32, 64)[:, :32]), ValueError),                   # another layout
    (dict(cos=torch.zeros(32, 32).double(), sin=torch.zeros(32, 32).double()), TypeError),
    (dict(q_weight=torch.zeros(32).half()), ValueError),
    (dict(k_weight=torch.zeros(64)), ValueError),
    (dict(q_out=torch.zeros(2, 4, 64)), ValueError),
    (dict(q=None, q_out=torch.zeros(2, 4, 64).half()), ValueError),
    (dict(q_out=torch.zeros(1, 4, 64).half().expand(2, 4, 64)), ValueError),
    (dict(q=torch.zeros(2, 64, 4).half().transpose(1, 2)), ValueError),
    (dict(k=3), TypeError),
    (dict(), ValueError),                                           # sound, but not on a GPU
])
def test_append_refusals(change, err):
    with pytest.raises(err):
        paged_int4_append(pool(), **{**append_args(), **change})


def test_append_refuses_pools_that_overlap():
    block = PagedKVInt4.page_bytes(16, 64)
    memory = torch.zeros(64 * block, dtype=U8)
    for shape, strides in (((4, 2, block), (0, block, 1)), ((4, 2, block), (2 * block, 0, 1)), ((4, 2, block), (block, block, 1)),
                           ((4, 2, block), (2 * block - 16, block, 1))):
        kv = PagedKVInt4(memory.as_strided(shape, strides), 16, 64, HALF)
        refused(lambda: paged_int4_append(kv, **append_args()), "overlap")
        refused(lambda: paged_int4_read(kv, torch.zeros(2, dtype=torch.int64), append_args()["page_table"]), "CUDA")   # read only: fine
    for shape, strides in (((4, 2, block), (2 * block, block, 1)), ((4, 2, block), (block, 4 * block, 1))):
        kv = PagedKVInt4(memory.as_strided(shape, strides), 16, 64, HALF)
        refused(lambda: paged_int4_append(kv, **append_args()), "CUDA")


def test_read_refusals():
    pos, table = torch.zeros(4, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int32)
    out = torch.zeros(4, 2, 64).half()
    call = lambda *a, **kw: lambda: paged_int4_read(pool(), *a, **kw)  # noqa: E731
    refused(call(pos.int(), table), "positions")
    refused(call(pos.view(2, 2), table), "positions")
    refused(call(pos[:3], table), "seq_ids")
    refused(call(pos, table.long()), "page_table")
    refused(call(pos, table, seq_ids=torch.zeros(3, dtype=torch.int32)), "seq_ids")
    refused(call(pos, table, out_dtype=torch.bfloat16), "fp32 or in the cache", TypeError)
    refused(call(pos, table, out_dtype=torch.float64), "fp32 or in the cache", TypeError)
    refused(call(pos, table, k_out=out.float(), v_out=out), "dtype", TypeError)
    refused(call(pos, table, k_out=out, out_dtype=torch.float32), "dtype", TypeError)
    refused(call(pos, table, k_out=out[:3]), "k_out")
    refused(call(pos, table, v_out=out[:1].expand(4, 2, 64)), "overlaps itself")
    refused(call(pos, table, k_out=out, v_out=out), "one memory")
    refused(call(pos, table, k_out=torch.zeros(4, 64, 2).half().transpose(1, 2)), "contiguous")
    refused(call(pos, table, k_out=False), "CUDA")
    refused(call(pos, table, k_out=True), "tensor", TypeError)


def attn_args(B=2, T=1, H=4, D=64):
    return dict(q=torch.zeros(B, T, H, D).half(), page_table=torch.zeros(B, 3, dtype=torch.int32),
                seqlens=torch.ones(B, dtype=torch.int32))


def test_outputs_that_overlap_are_refused():
    pos, table = torch.zeros(4, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int32)
    memory = torch.zeros(3 * 4 * 2 * 64).half()
    first, shifted, behind = (memory[n:n + 512].view(4, 2, 64) for n in (0, 256, 512))
    refused(lambda: paged_int4_read(pool(), pos, table, k_out=first, v_out=shifted), "one memory")
    refused(lambda: paged_int4_read(pool(), pos, table, k_out=first, v_out=behind), "CUDA")
    both = memory[:1024].view(4, 4, 64)                       # rows of keys and values by turns
    refused(lambda: paged_int4_read(pool(), pos, table, k_out=both[:, :2], v_out=both[:, 2:]), "CUDA")
    q, shifted, behind = (memory[n:n + 512].view(2, 1, 4, 64) for n in (0, 8, 512))
    args = {**attn_args(), "q": q}
    refused(lambda: paged_int4_attention(pool(), **args, out=shifted), "overlaps q")
    refused(lambda: paged_int4_attention(pool(), **args, out=memory.view(torch.float32)[:512].view(2, 1, 4, 64)), "overlaps q")
    refused(lambda: paged_int4_attention(pool(), **args, out=behind, workspace=memory[1016:].view(U8)), "workspace")
    refused(lambda: paged_int4_attention(pool(), **args, out=q), "CUDA")
    refused(lambda: paged_int4_attention(pool(), **args, out=behind), "CUDA")


def test_append_outputs_that_overlap_inputs_are_refused():
    N, H, KVH, D = 4, 4, 2, 64
    args = append_args(N=N)
    row = (H + 2 * KVH) * D
    memory = torch.zeros(3 * N * row).half()
    call = lambda **kw: lambda: paged_int4_append(pool(), **{**args, **kw})  # noqa: E731

    def view(start, stride, heads=H):
        return memory[start:].as_strided((N, heads, D), (stride, D, 1))

    q = view(0, H * D)
    for out in (view(8, H * D), view(0, row), view(0, 2 * H * D), view(N * H * D - 8, H * D), view(H * D, H * D)):   # shifted, other rows, its end
        refused(call(q=q, q_out=out), "overlaps q and is not q")
    refused(call(q=q, q_out=memory[:N * H * D].view(H, N, D).transpose(0, 1)), "overlaps q and is not q")   # same memory, other strides
    refused(call(q=q, q_out=q), "CUDA")
    refused(call(q=q, q_out=view(0, H * D)), "CUDA")
    refused(call(q=q, q_out=view(N * H * D, H * D)), "CUDA")
    # a fused projection: q in place, and beside one another
    q, k, v = view(0, row), view(H * D, row, KVH), view((H + KVH) * D, row, KVH)
    refused(call(q=q, k=k, v=v, q_out=q), "CUDA")
    refused(call(q=args["q"], k=k, v=v, q_out=q), "CUDA")
    refused(call(q=q, k=k, v=v, q_out=view(KVH * D, row)), "overlaps q")
    refused(call(q=args["q"], k=k, v=v, q_out=view(KVH * D, row)), "q_out and k are one memory")
    refused(call(q=args["q"], k=k, v=v, q_out=view(2 * KVH * D, row)), "q_out and k are one memory")
    refused(call(q=args["q"], v=v, q_out=view((KVH + 2) * D, row)), "q_out and v are one memory")
    refused(call(q=args["q"], k=k, v=v, q_out=view(N * row, row)), "CUDA")
    weight = memory[70:134]
    refused(call(q_out=view(0, H * D), q_weight=weight), "q_out and q_weight")
    refused(call(q_out=view(0, H * D), k_weight=weight), "q_out and k_weight")
    ids = memory[:4 * N].view(torch.int64)
    refused(call(q_out=view(0, H * D), positions=ids), "q_out and positions")
    tables = memory[:32 * 32].view(32, 32)
    refused(call(q_out=view(0, H * D), cos=tables, sin=tables), "q_out and cos")


def test_attention_outputs_that_overlap_strided_inputs_are_refused():
    args = attn_args(B=2, T=2)
    memory = torch.zeros(4096).half()
    wide = memory[:2 * 2 * 8 * 64].view(2, 2, 8, 64)
    q, beside = wide[:, :, :4], wide[:, :, 4:]                  # parts of one projection
    call = lambda **kw: lambda: paged_int4_attention(pool(), **{**args, **kw})  # noqa: E731
    refused(call(q=q, out=q), "CUDA")
    refused(call(q=q, out=beside), "CUDA")
    refused(call(q=q, out=memory[:1024].view(2, 2, 4, 64)), "overlaps q")       # the same address, other strides
    refused(call(q=q, out=wide[:, :, 2:6]), "overlaps q")
    refused(call(q=q, out=wide.transpose(0, 1)[:, :, :4]), "overlaps q")
    refused(call(q=q, out=beside, workspace=memory.view(U8)[:2048]), "workspace and")
    refused(call(q=q, out=torch.zeros(2, 2, 4, 64).half(), workspace=memory.view(U8)[:2048]), "workspace and q")
    refused(call(seqlens=memory[:4].view(torch.int32), out=memory[:1024].view(2, 2, 4, 64)), "out and seqlens")
    refused(call(seqlens=memory[:4].view(torch.int32), workspace=memory[:512].view(U8)), "workspace and seqlens")
    refused(call(q=q, out=beside, workspace=memory[2048:].view(U8)), "CUDA")


def test_read_outputs_that_overlap_are_refused():
    pos, table = torch.zeros(4, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int32)
    memory = torch.zeros(4096).half()
    call = lambda k, v, **kw: lambda: paged_int4_read(pool(), pos, table, k_out=k, v_out=v, **kw)  # noqa: E731
    turns = memory[:4 * 2 * 2 * 64].view(4, 2, 2, 64)           # a head's key and value side by side
    refused(call(turns[:, :, 0], turns[:, :, 1]), "CUDA")
    rows = memory[:4 * 4 * 64].view(4, 4, 64)
    refused(call(rows[:, :2], rows[:, 1:3]), "one memory")
    refused(call(rows[:, :2], rows[:, 2:]), "CUDA")
    refused(call(rows[:, :2], rows[:, ::2]), "one memory")
    refused(call(rows[:, ::2], rows[:, 1::2]), "CUDA")
    refused(lambda: paged_int4_read(pool(), memory[:16].view(torch.int64), table, k_out=rows[:, :2]), "k_out and positions")


@pytest.mark.parametrize("change,err", [
    (dict(q=torch.zeros(2, 1, 4, 128).half()), ValueError),
    (dict(q=torch.zeros(2, 1, 5, 64).half()), ValueError),
    (dict(q=torch.zeros(3, 1, 4, 64).half()), ValueError),
    (dict(q=torch.zeros(2, 4, 64).half()), ValueError),
    (dict(q=torch.zeros(2, 1, 4, 64)), TypeError),
    (dict(seqlens=torch.ones(2, dtype=torch.int64)), ValueError),
    (dict(seqlens=torch.ones(3, dtype=torch.int32)), ValueError),
    (dict(max_len=2 ** 40), ValueError),
    (dict(out=torch.zeros(2, 1, 4, 32).half()), ValueError),
    (dict(out=torch.zeros(2, 1, 4, 64).half(), out_dtype=torch.float32), ValueError),
    (dict(out=torch.zeros(1, 1, 4, 64).half().expand(2, 1, 4, 64)), ValueError),
    (dict(workspace=torch.zeros(1, dtype=U8).expand(1 << 20)), ValueError),
    (dict(), ValueError),                                           # sound, but not on a GPU
])
def test_attention_refusals(change, err):
    with pytest.raises(err):
        paged_int4_attention(pool(), **{**attn_args(), **change})


@pytest.mark.parametrize("q,table,err", [
    (torch.zeros(2, 17, 4, 64).half(), torch.zeros(2, 3, dtype=torch.int32), _lib.B2DError),       # more than 16 tokens
    (torch.zeros(2, 1, 34, 64).half(), torch.zeros(2, 3, dtype=torch.int32), _lib.B2DError),       # 17 heads of a KV head
    (torch.zeros(2, 1, 4, 64).half(), torch.zeros(2, 1 << 27, dtype=torch.int32, device="meta"), _lib.B2DError),   # 2^31 positions
    (torch.zeros(2, 1, 5, 64).half(), torch.zeros(2, 3, dtype=torch.int32), ValueError),
    (torch.zeros(2, 1, 4, 128).half(), torch.zeros(2, 3, dtype=torch.int32), ValueError),
    (torch.zeros(2, 4, 64).half(), torch.zeros(2, 3, dtype=torch.int32), ValueError),
    (torch.zeros(2, 1, 4, 64), torch.zeros(2, 3, dtype=torch.int32), TypeError),
    (torch.zeros(2, 1, 4, 64).half(), torch.zeros(3, 3, dtype=torch.int32), ValueError),
    (torch.zeros(2, 1, 4, 64).half(), torch.zeros(2, 3, dtype=torch.int64), ValueError),
    (torch.zeros(2, 1, 4, 64).half(), torch.zeros(2, 3, dtype=torch.int32), ValueError)])          # sound, but not on a GPU
def test_workspace_refuses_what_the_attention_refuses(q, table, err):
    with pytest.raises(err):
        paged_int4_attention_workspace(pool(), q, table)
    if err is _lib.B2DError:
        refused(lambda: paged_int4_attention_workspace(pool(), q, table), "b2d_int4_attention", err)


def test_plan_refusals():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    tables = PageTables.empty(8, 16, 3, 4, "cpu")
    refused(lambda: PageTables.empty(8, 0, 3, 4, "cpu"), "1..1024")
    refused(lambda: PageTables.empty(8, 1025, 3, 4, "cpu"), "1..1024")
    refused(lambda: PageTables.empty(8, 16, 8193, 1, "cpu"), "8192")
    refused(lambda: PageTables(i32(4), i32(4), i32(8), i32(2), 16), "page_table")
    refused(lambda: tables.step(i32(3), i32(3)), "max_tokens")
    refused(lambda: tables.step(i32(3), i32(3), 5, out=StepPlan.empty(3, 4, "cpu")), "4 tokens")
    refused(lambda: tables.step(i32(3), i32(3), 5), "CUDA")
    refused(lambda: tables.step(i32(4), i32(3), 5), "cached")
    refused(lambda: tables.step(i32(3), i32(3).long(), 5), "new")
    refused(lambda: tables.step(i32(3), i32(6)[::2], 5), "new")
    refused(lambda: tables.step(i32(3), i32(3), out=StepPlan.empty(2, 5, "cpu")), "seqlens")
    good = StepPlan.empty(3, 5, "cpu")
    refused(lambda: tables.step(i32(3), i32(3), out=good._replace(slots=good.positions)), "one memory")
    refused(lambda: tables.step(i32(3), i32(3), out=good._replace(seq_ids=i32(4))), "seq_ids")
    new = i32(3)
    refused(lambda: tables.step(i32(3), new, out=good._replace(granted=new)), "one memory")
    run = torch.zeros(9, dtype=torch.int64)               # windows of one memory that share an element
    refused(lambda: tables.step(i32(3), i32(3), out=good._replace(positions=run[:5], slots=run[4:])), "one memory")
    refused(lambda: tables.step(i32(3), i32(3), out=good._replace(positions=run[:4], slots=run[4:8], seq_ids=i32(4))), "CUDA")
    refused(lambda: tables.step(tables.free[2:5], i32(3), out=good), "one memory")
    for field, bad in (("held", i32(4)), ("free", i32(2, 4)), ("ring", i32(3)), ("page_table", i32(1, 4).expand(3, 4)), ("page_table", i32(4, 3).t())):
        t = PageTables.empty(8, 16, 3, 4, "cpu")
        setattr(t, field, bad)
        refused(lambda: t.step(i32(3), i32(3), 5), field if field != "page_table" else "page_table")


# ---- C ABI: arguments are checked before the device is touched
BUF = C.create_string_buffer(4096)
P = (C.addressof(BUF) + 255) & ~255


def desc(**kw):
    f = dict(pages=P, sp_p=2304, sp_h=1152, num_pages=4, page_size=16, KVH=2, D=64, group=64, dtype=0)
    f.update(kw)
    return C.byref(_lib.Int4KvDesc(**f))


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), DTYPE), (dict(page_size=8), SHAPE), (dict(page_size=1040), SHAPE), (dict(page_size=40), SHAPE), (dict(KVH=0), SHAPE),
    (dict(KVH=65536), SHAPE), (dict(D=96), SHAPE), (dict(group=128), SHAPE), (dict(group=0), SHAPE), (dict(pages=P + 8), ALIGN),
    (dict(sp_h=1160), ALIGN), (dict(sp_p=8), ALIGN), (dict(pages=None), ARG), (dict(num_pages=-1), ARG), (dict(D=-8), ARG)])
def test_c_pool_checks(kw, status):
    lib = _lib.load()
    assert lib.b2d_int4_attention(desc(**kw), P, 256, 256, 64, P, 3, 3, P, 0, 1, 1, 4, 1.0, P, 256, 256, 64, 0, None, 0, 0, None) == status
    assert lib.b2d_int4_append(desc(**kw), P, 256, 64, P, 128, 64, P, 128, 64, P, None, P, 3, 3, 1, P, P, 32, 32, 2, 64, 0, None, None,
                               1e-6, P, 256, 64, 1, 4, 0, None) == status
    assert lib.b2d_int4_read(desc(**kw), P, None, P, 3, 3, 1, P, 128, 64, P, 128, 64, 0, 1, 0, None) == status
    assert lib.b2d_int4_attention_workspace_bytes(desc(**kw), 1, 1, 4, 3, 0) == 0
    assert lib.b2d_int4_attention(None, P, 256, 256, 64, P, 3, 3, P, 0, 1, 1, 4, 1.0, P, 256, 256, 64, 0, None, 0, 0, None) == ARG


def test_c_append_checks():
    lib = _lib.load()

    def call(d=None, q=P, sqn=256, k=P, ksn=128, pos=P, seq=None, B=1, cs=P, sn=P, ldcs=32, cdt=2, R=64, qw=None, qo=P, N=1, H=4, per=3, table=P):
        return lib.b2d_int4_append(d or desc(), q, sqn, 64, k, ksn, 64, P, 128, 64, pos, seq, table, 3, per, B, cs, sn, ldcs, 32, cdt, R, 0,
                                   qw, None, 1e-6, qo, 256, 64, N, H, 0, None)
    assert call(N=0) == OK
    assert call(H=5) == SHAPE and call(H=65536) == SHAPE and call(B=0) == SHAPE and call(N=3, B=2) == SHAPE and call(per=1 << 28) == SHAPE
    assert call(R=24) == SHAPE and call(R=0) == SHAPE and call(R=80) == SHAPE and call(cdt=1) == DTYPE
    assert call(N=-1) == ARG and call(k=None) == ARG and call(pos=None) == ARG and call(sn=None) == ARG and call(cs=None) == ARG
    assert call(qo=None) == ARG and call(table=None) == ARG and call(ldcs=-4) == ARG
    assert call(ksn=124) == ALIGN and call(sqn=252) == ALIGN and call(ldcs=34) == ALIGN and call(cdt=0, ldcs=36) == ALIGN
    assert call(qw=P + 4) == ALIGN and call(cs=P + 8) == ALIGN and call(pos=P + 4) == ALIGN


def test_c_read_and_attention_checks():
    lib = _lib.load()

    def read(k=P, v=P, sn=128, odt=0, N=1, B=1, pos=P, seq=None, per=3, table=P):
        return lib.b2d_int4_read(desc(), pos, seq, table, 3, per, B, k, sn, 64, v, 128, 64, odt, N, 0, None)
    assert read(N=0) == OK and read(k=None, v=None) == OK
    assert read(odt=1) == DTYPE and read(N=-1) == ARG and read(pos=None) == ARG and read(table=None) == ARG
    assert read(B=0) == SHAPE and read(N=3, B=2) == SHAPE and read(per=1 << 28) == SHAPE
    assert read(sn=124) == ALIGN and read(k=P + 8) == ALIGN and read(v=P + 2) == ALIGN

    def call(q=P, sq=(256, 256, 64), table=P, ld=3, per=3, lens=P, B=1, T=1, H=4, out=P, odt=0, most=0):
        return lib.b2d_int4_attention(desc(), q, *sq, table, ld, per, lens, most, B, T, H, 1.0, out, 256, 256, 64, odt, None, 0, 0, None)
    assert call(B=0) == OK and call(T=0) == OK and call(H=0) == OK
    assert call(T=17) == SHAPE and call(H=34) == SHAPE and call(H=5) == SHAPE and call(per=1 << 28) == SHAPE and call(ld=-1) == SHAPE
    assert call(odt=1) == DTYPE
    assert call(q=None) == ARG and call(lens=None) == ARG and call(out=None) == ARG and call(table=None) == ARG
    assert call(B=-1) == ARG and call(most=-1) == ARG
    assert call(q=P + 2) == ALIGN and call(sq=(256, 256, 60)) == ALIGN and call(out=P + 1) == ALIGN


def test_c_plan_checks():
    lib = _lib.load()

    def call(table=P, ld=3, per=3, held=P, free=P, pages=8, ring=P, cached=P, new=P, B=1, ps=16, N=4, pos=P, seq=P, slots=P, lens=P, starts=P, granted=P):
        return lib.b2d_page_plan(table, ld, per, held, free, pages, ring, cached, new, B, ps, N, pos, seq, slots, lens, starts, granted, 0, None)
    assert call(B=8193) == SHAPE and call(ps=0) == SHAPE and call(ps=1025) == SHAPE and call(per=1 << 28) == SHAPE and call(ld=-1) == SHAPE
    assert call(pages=2 ** 31 - 1) == SHAPE and call(N=2 ** 31 - 1) == SHAPE
    for kw in (dict(B=-1), dict(N=-1), dict(pages=-1), dict(per=-1), *({n: None} for n in (
            "table", "held", "free", "ring", "cached", "new", "pos", "seq", "slots", "lens", "starts", "granted"))):
        assert call(**kw) == ARG, kw
    assert call(pos=P + 4) == ALIGN and call(slots=P + 4) == ALIGN and call(held=P + 2) == ALIGN and call(table=P + 1) == ALIGN


# ---- the kernels' sources
def test_every_bounded_wait_is_looked_at():
    """A wait on an mbarrier that runs out has to reach the result (as NaN): each one's outcome goes into `landed`."""
    source = Path(__file__).resolve().parent.parent / "llm-decode-triton-6gb_b200" / "csrc" / "int4_attention.cu"
    waits = [line.split("//")[0] for line in source.read_text().splitlines() if "mbar_wait(" in line.split("//")[0]]
    assert len(waits) >= 2
    for line in waits:
        assert re.search(r"landed = (landed && )?mbar_wait\(", line), line


def test_nothing_that_kernels_write_takes_the_read_only_path():
    """With programmatic launches a kernel may be resident while earlier ones still write what it reads behind its wait: no
    load of these kernels may be one that promises data constant for the kernel's lifetime."""
    folder = Path(__file__).resolve().parent.parent / "llm-decode-triton-6gb_b200" / "csrc"
    for name in ("int4_append.cu", "int4_attention.cu", "int4_kv.cuh", "page_plan.cu"):
        code = "\n".join(line.split("//")[0] for line in (folder / name).read_text().splitlines())
        assert not re.search(r"__ldg\(|ldg_\w+\(|\.nc\b|__restrict__", code), name


# ---- rotary tables
def angles(cos, sin):
    return torch.atan2(sin.double(), cos.double())


def test_rotary_tables_plain_and_linear():
    cos, sin = rotary_tables(50, 16, 1e4)
    assert cos.shape == sin.shape == (50, 8) and cos.dtype == torch.float32
    want = np.arange(50)[:, None] * 1e4 ** (-np.arange(0, 16, 2) / 16)
    assert np.abs(cos.numpy() - np.cos(want)).max() <= 2 ** -24 and np.abs(sin.numpy() - np.sin(want)).max() <= 2 ** -24
    c2, _ = rotary_tables(50, 16, 1e4, scaling={"type": "linear", "factor": 2.0})
    assert torch.equal(c2[::2], cos[:25])
    far = rotary_tables(300001, 2, 1e4, dtype=torch.float16)[0]
    assert far[-1, 0] == torch.tensor(math.cos(300000)).half()
    refused(lambda: rotary_tables(8, 7), "even")
    refused(lambda: rotary_tables(8, 8, scaling={"rope_type": "spiral"}), "spiral")


@pytest.mark.parametrize("kind", ["llama3", "yarn"])
def test_rotary_tables_scaled(kind):
    """Against the scalings' definitions, pair by pair: the wavelengths that stay, that are stretched, and those between."""
    R, theta, factor, original = 128, 5e5, 8.0, 8192
    scaling = {"rope_type": kind, "factor": factor, "original_max_position_embeddings": original}
    scaling |= {"low_freq_factor": 1.0, "high_freq_factor": 4.0} if kind == "llama3" else {}
    cos, sin = rotary_tables(2, R, theta, scaling=scaling, dtype=torch.float64)
    gain = 0.1 * math.log(factor) + 1 if kind == "yarn" else 1.0
    seen = set()
    for i in range(R // 2):
        f = theta ** (-2 * i / R)
        if kind == "llama3":
            wave = 2 * math.pi / f
            if wave < original / 4.0:
                want, case = f, "stays"
            elif wave > original / 1.0:
                want, case = f / factor, "stretched"
            else:
                smooth = (original / wave - 1.0) / 3.0
                want, case = (1 - smooth) * f / factor + smooth * f, "between"
        else:
            pair = lambda turns: R * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), R - 1)
            ramp = min(max((i - low) / (high - low), 0.0), 1.0)
            want, case = f * (1 - ramp) + f / factor * ramp, "stays" if ramp == 0 else "stretched" if ramp == 1 else "between"
        seen.add(case)
        assert abs(float(cos[1, i]) - gain * math.cos(want)) < 1e-12 and abs(float(sin[1, i]) - gain * math.sin(want)) < 1e-12
    assert seen == {"stays", "stretched", "between"}
    if kind == "yarn":
        c2, _ = rotary_tables(1, R, theta, scaling={**scaling, "attention_factor": 1.5}, dtype=torch.float64)
        assert float(c2[0, 0]) == 1.5
        c3, _ = rotary_tables(1, R, theta, scaling={**scaling, "mscale": 0.707, "mscale_all_dim": 1.0}, dtype=torch.float64)
        assert abs(float(c3[0, 0]) - (0.0707 * math.log(8) + 1) / (0.1 * math.log(8) + 1)) < 1e-12


# ---- the oracle
def test_quantiser_keeps_the_ends_and_halves_a_step():
    g = np.random.default_rng(0)
    x = g.standard_normal((200, 2, 64)).astype(np.float16).astype(np.float32)
    codes, s, m = quantise_ref(x, 32, HALF)
    v = values_ref(codes, s, m, 64).reshape(200, 2, 2, 32)
    parts = x.reshape(200, 2, 2, 32)
    assert (v.min(-1) == parts.min(-1)).all() and codes.min() == 0 and codes.max() == 15
    # half a step, and at the upper end what the scale's rounding (2^-11 of 15 steps) takes
    assert (np.abs(v - parts) <= s[..., None] * (0.5 + 15 * 2.0 ** -11) * 1.0001).all()
    codes, s, m = quantise_ref(np.full((1, 64), 2.5, np.float32), 64, HALF)
    assert (codes == 0).all() and s[0, 0] == 0 and m[0, 0] == 2.5
    assert np.isnan(quantise_ref(np.array([[np.inf] + [0.0] * 63], np.float32), 64, HALF)[1]).all()


def test_plan_oracle_by_hand():
    r = plan_ref([[7, -1], [3, 4], [-1, -1]], [1, 2, 0], [0, 1, 2, 5, 6, 9, 9, 9], [1, 3], [16, 3, 0], [1, 2, 40], 16, 10)
    # sequence 0 takes page 1 for position 16; sequence 1 gives page 4 back; sequence 2's 40 tokens do not fit
    assert r["granted"].tolist() == [1, 2, -1] and r["starts"].tolist() == [0, 1, 3, 3] and r["seqlens"].tolist() == [17, 5, 0]
    assert r["page_table"].tolist() == [[7, 1], [3, -1], [-1, -1]] and r["held"].tolist() == [2, 1, 0]
    assert r["ring"].tolist() == [2, 3] and r["free"].tolist() == [0, 1, 2, 5, 4, 9, 9, 9]
    assert r["positions"].tolist() == [16, 3, 4] + [-1] * 7 and r["seq_ids"].tolist()[:4] == [0, 1, 1, -1]
    assert r["slots"].tolist()[:4] == [16, 51, 52, -1]
