"""CPU: refusals of the paged-cache and draft-verification calls (Python and C ABI), and their oracle."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from b200kernels import _lib
from b200kernels.paged import PagedKV, paged_attention, paged_rope_append
from b200kernels.speculative import verify_drafts
from oracle.paged_ref import verify_ref

OK, ARG, SHAPE, DTYPE, ALIGN = 0, 1, 2, 3, 4


def pool(pages=4, kvh=2, ps=16, D=64, dtype=torch.float16):
    return PagedKV(torch.zeros(pages, kvh, ps, D, dtype=dtype), torch.zeros(pages, kvh, ps, D, dtype=dtype))


@pytest.mark.parametrize("k,v,err", [
    (torch.zeros(4, 2, 16, 64).half(), torch.zeros(4, 2, 16, 32).half(), ValueError),
    (torch.zeros(4, 2, 16).half(), torch.zeros(4, 2, 16).half(), ValueError),
    (torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64), TypeError),
    (torch.zeros(4, 2, 16, 64).half(), torch.zeros(4, 2, 16, 64).bfloat16(), TypeError),
    (torch.zeros(4, 2, 64, 16).half().transpose(2, 3), torch.zeros(4, 2, 16, 64).half(), ValueError),
    (torch.zeros(4, 2, 2048, 64).half(), torch.zeros(4, 2, 2048, 64).half(), ValueError),
    (torch.zeros(4, 0, 16, 64).half(), torch.zeros(4, 0, 16, 64).half(), ValueError),
])
def test_pool_refusals(k, v, err):
    with pytest.raises(err):
        PagedKV(k, v)


def test_pool_of_too_many_pages_or_heads_is_refused():
    """The kernels count pages and heads in 32 bits; a number past them must not wrap."""
    one = torch.zeros(1, 1, 1, 16).half()
    for shape in ((2 ** 31, 1, 1, 16), (2 ** 32 + 4, 1, 1, 16), (4, 2 ** 32 + 2, 1, 16)):
        with pytest.raises(ValueError, match="too many"):
            PagedKV(one.expand(shape), one.expand(shape))


def append_args(N=2, H=4, kvh=2, D=64, B=2):
    return dict(q=torch.zeros(N, H, D).half(), k=torch.zeros(N, kvh, D).half(), v=torch.zeros(N, kvh, D).half(),
                positions=torch.zeros(N, dtype=torch.int64), page_table=torch.zeros(B, 3, dtype=torch.int32),
                cos=torch.zeros(32, D).half(), sin=torch.zeros(32, D).half())


@pytest.mark.parametrize("change,err", [
    (dict(q=torch.zeros(2, 4, 32).half()), ValueError),
    (dict(q=torch.zeros(2, 3, 64).half()), ValueError),             # 3 heads over 2 KV heads
    (dict(k=torch.zeros(3, 2, 64).half()), ValueError),
    (dict(v=torch.zeros(2, 2, 64)), TypeError),
    (dict(q=torch.zeros(2, 4, 64).bfloat16()), TypeError),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), ValueError),   # 2 tokens over 3 sequences
    (dict(seq_ids=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(cos=torch.zeros(32, 32).half()), ValueError),
    (dict(cos=torch.zeros(32, 64).double(), sin=torch.zeros(32, 64).double()), TypeError),
    (dict(q_weight=torch.zeros(32).half()), ValueError),
    (dict(k_weight=torch.zeros(64)), ValueError),
    (dict(q_out=torch.zeros(2, 4, 64)), ValueError),
    (dict(q=torch.zeros(2, 64, 4).half().transpose(1, 2)), ValueError),
    (dict(), ValueError),                                           # sound, but not on a GPU
])
def test_append_refusals(change, err):
    with pytest.raises(err):
        paged_rope_append(pool(), **{**append_args(), **change})


def attn_args(B=2, T=1, H=4, D=64):
    return dict(q=torch.zeros(B, T, H, D).half(), page_table=torch.zeros(B, 3, dtype=torch.int32),
                seqlens=torch.ones(B, dtype=torch.int32))


@pytest.mark.parametrize("change,err", [
    (dict(q=torch.zeros(2, 1, 4, 128).half()), ValueError),
    (dict(q=torch.zeros(2, 1, 5, 64).half()), ValueError),
    (dict(q=torch.zeros(3, 1, 4, 64).half()), ValueError),
    (dict(q=torch.zeros(2, 1, 4, 64)), TypeError),
    (dict(seqlens=torch.ones(2, dtype=torch.int64)), ValueError),
    (dict(seqlens=torch.ones(3, dtype=torch.int32)), ValueError),
    (dict(prefix_len=5), ValueError),
    (dict(prefix_len=33, prefix_table=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(prefix_len=-1, prefix_table=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(out=torch.zeros(2, 1, 4, 32).half()), ValueError),
    (dict(out=torch.zeros(2, 1, 4, 64).half(), out_dtype=torch.float32), ValueError),
    (dict(), ValueError),                                           # sound, but not on a GPU
])
def test_attention_refusals(change, err):
    with pytest.raises(err):
        paged_attention(pool(), **{**attn_args(), **change})


@pytest.mark.parametrize("change,err", [
    (dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int32)), ValueError),
    (dict(draft_tokens=torch.zeros(2, 32, dtype=torch.int64)), ValueError),
    (dict(target_probs=torch.zeros(2, 3, 10)), ValueError),
    (dict(target_probs=torch.zeros(2, 4, 0)), ValueError),
    (dict(target_probs=torch.zeros(2, 4, 10).double()), TypeError),
    (dict(draft_probs=torch.zeros(2, 4, 10)), ValueError),
    (dict(draft_probs=torch.zeros(2, 3, 10).half()), TypeError),
    (dict(uniforms=torch.zeros(2, 3)), ValueError),
    (dict(uniforms=torch.zeros(2, 4).double()), ValueError),
    (dict(draft_lens=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(tokens=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(accepted=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(target_probs=torch.zeros(2, 10, 4).transpose(1, 2)), ValueError),
    (dict(), ValueError),                                           # sound, but not on a GPU
])
def test_verify_refusals(change, err):
    args = dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int64), target_probs=torch.zeros(2, 4, 10),
                uniforms=torch.zeros(2, 4))
    with pytest.raises(err):
        verify_drafts(**{**args, **change})


# ---- C ABI: arguments are checked before the device is touched
BUF = C.create_string_buffer(4096)
P = (C.addressof(BUF) + 255) & ~255


def desc(**kw):
    f = dict(k=P, sk_p=2048, sk_h=1024, sk_s=64, v=P, sv_p=2048, sv_h=1024, sv_s=64, num_pages=4, page_size=16, KVH=2,
             D=64, dtype=0)
    f.update(kw)
    return C.byref(_lib.PagedKvDesc(**f))


def test_outputs_that_overlap_themselves_are_refused():
    with pytest.raises(ValueError, match="overlaps itself"):
        paged_rope_append(pool(), **{**append_args(), "q_out": torch.zeros(1, 4, 64).half().expand(2, 4, 64)})
    with pytest.raises(ValueError, match="overlaps itself"):
        paged_attention(pool(), **{**attn_args(), "out": torch.zeros(1, 1, 4, 64).half().expand(2, 1, 4, 64)})
    with pytest.raises(ValueError, match="overlaps itself"):
        verify_drafts(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4, 10), torch.zeros(2, 4),
                      tokens=torch.zeros(1, 4, dtype=torch.int64).expand(2, 4))


def test_outputs_whose_rows_run_into_each_other_are_refused():
    """Overlap without a zero stride: windows of one memory."""
    def windows(dtype, *shape_and_strides):
        return torch.zeros(4096, dtype=dtype).as_strided(*shape_and_strides)
    with pytest.raises(ValueError, match="overlaps itself"):
        paged_attention(pool(), **attn_args(), out=windows(torch.float16, (2, 1, 4, 64), (64, 64, 32, 1)))
    with pytest.raises(ValueError, match="overlaps itself"):
        paged_attention(pool(), **attn_args(), out=windows(torch.float16, (2, 1, 4, 64), (192, 64, 64, 1)))
    with pytest.raises(ValueError, match="overlaps itself"):
        paged_rope_append(pool(), **append_args(), q_out=windows(torch.float16, (2, 4, 64), (64, 64, 1)))
    with pytest.raises(ValueError, match="overlaps itself"):
        verify_drafts(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4, 10), torch.zeros(2, 4),
                      tokens=windows(torch.int64, (2, 4), (3, 1)))
    # views of larger tensors are fine: the call goes on to ask for a GPU
    for out in (torch.zeros(1, 2, 6, 64).half().transpose(0, 1)[:, :, 1:5], torch.zeros(4, 2, 1, 64).half().permute(1, 2, 0, 3)):
        with pytest.raises(ValueError, match="CUDA"):
            paged_attention(pool(), **attn_args(), out=out)
    with pytest.raises(ValueError, match="CUDA"):
        paged_rope_append(pool(), **append_args(), q_out=torch.zeros(2, 8, 64).half()[:, ::2])


def test_append_refuses_pools_that_overlap():
    one = torch.zeros(1, 2, 16, 64).half()
    both = torch.zeros(4, 2, 2, 16, 64).half()
    for k, v in ((one.expand(4, 2, 16, 64), both[:, 0]), (both[:, 1], one.expand(4, 2, 16, 64)),
                 (torch.zeros(9000).half().as_strided((4, 2, 16, 64), (1024, 1024, 64, 1)), both[:, 0]),
                 (both[:, 0], both[:, 0])):
        with pytest.raises(ValueError, match="overlap"):
            paged_rope_append(PagedKV(k, v), **append_args())
        with pytest.raises(ValueError, match="CUDA"):      # read only: fine
            paged_attention(PagedKV(k, v), **attn_args())
    nhd = torch.zeros(4, 2, 16, 2, 64).half().transpose(2, 3)   # [pages, K or V, head, slot, D]
    for k, v in ((both[:, 0], both[:, 1]), (nhd[:, 0], nhd[:, 1]), (one, one.clone())):
        with pytest.raises(ValueError, match="CUDA"):
            paged_rope_append(PagedKV(k, v), **append_args())


def test_workspace_without_its_own_memory_is_refused():
    """A workspace whose elements are one memory (expanded) or lie apart has fewer bytes than its size says."""
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 21, dtype=torch.uint8)[::2],
               torch.zeros(1, 64, dtype=torch.uint8).expand(1 << 14, 64)):
        with pytest.raises(ValueError, match="workspace"):
            paged_attention(pool(), **attn_args(), workspace=ws)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), DTYPE), (dict(page_size=0), SHAPE), (dict(page_size=1025), SHAPE), (dict(KVH=0), SHAPE),
    (dict(k=P + 2), ALIGN), (dict(sv_s=60), ALIGN), (dict(k=None), ARG), (dict(num_pages=-1), ARG), (dict(D=-8), ARG),
])
def test_c_pool_checks(kw, status):
    lib = _lib.load()
    assert lib.b2d_paged_attention(desc(**kw), P, 256, 256, 64, P, 3, 3, P, None, 0, 0, 1, 1, 4, 1.0, P, 256, 256, 64, 0,
                                   None, 0, 0, None) == status
    assert lib.b2d_paged_rope_append(desc(**kw), P, 256, 64, P, 128, 64, P, 128, 64, P, None, P, 3, 3, 1, P, P, 64, 32, 0,
                                     None, None, 1e-6, P, 256, 64, 1, 4, 0, None) == status


def test_c_attention_checks():
    lib = _lib.load()

    def call(d=None, q=P, sq=(256, 256, 64), table=P, ld=3, per=3, lens=P, pt=None, pl=0, B=1, T=1, H=4, out=P, odt=0):
        return lib.b2d_paged_attention(d or desc(), q, *sq, table, ld, per, lens, pt, pl, 0, B, T, H, 1.0, out, 256, 256,
                                       64, odt, None, 0, 0, None)
    assert call(B=0) == OK and call(T=0) == OK
    assert call(d=desc(D=96)) == SHAPE and call(T=17) == SHAPE and call(H=34) == SHAPE and call(H=5) == SHAPE
    assert call(odt=1) == DTYPE
    assert call(q=None) == ARG and call(lens=None) == ARG and call(out=None) == ARG and call(table=None) == ARG
    assert call(pl=4) == ARG and call(pl=-1) == ARG and call(B=-1) == ARG
    assert call(q=P + 2) == ALIGN and call(sq=(256, 256, 60)) == ALIGN
    assert call(d=desc(page_size=1024), per=1 << 21) == SHAPE and call(pl=2 ** 31 - 1, pt=P) == SHAPE


def test_c_append_checks():
    lib = _lib.load()

    def call(d=None, q=P, ksn=128, pos=P, seq=None, B=1, cs=P, ldcs=64, cdt=0, qw=None, N=1, H=4):
        return lib.b2d_paged_rope_append(d or desc(), q, 256, 64, P, ksn, 64, P, 128, 64, pos, seq, P, 3, 3, B, cs, P, ldcs,
                                         32, cdt, qw, None, 1e-6, P, 256, 64, N, H, 0, None)
    assert call(N=0) == OK
    assert call(d=desc(D=40)) == SHAPE and call(d=desc(D=272)) == SHAPE and call(H=5) == SHAPE
    assert call(B=0) == SHAPE and call(N=3, B=2) == SHAPE and call(H=65536) == SHAPE
    assert call(cdt=1) == DTYPE and call(N=-1) == ARG and call(q=None) == ARG and call(pos=None) == ARG
    assert call(ksn=124) == ALIGN and call(ldcs=60) == ALIGN and call(qw=P + 4) == ALIGN and call(cs=P + 8) == ALIGN


def test_c_verify_checks():
    lib = _lib.load()

    def call(draft=P, tp=P, dt=2, u=P, out=P, ldo=5, B=1, K=4, V=10):
        return lib.b2d_verify_drafts(draft, 4, None, tp, 50, 10, None, 0, 0, dt, u, 5, out, ldo, None, B, K, V, 0, None)
    assert call(B=0) == OK
    assert call(K=32, ldo=33) == SHAPE and call(V=0) == SHAPE and call(V=2 ** 30 + 1) == SHAPE and call(ldo=4) == SHAPE and call(dt=5) == DTYPE
    assert call(draft=None) == ARG and call(tp=None) == ARG and call(u=None) == ARG and call(out=None) == ARG
    assert call(B=-1) == ARG and call(draft=P + 4) == ALIGN and call(tp=P + 2) == ALIGN


# ---- the kernels' sources
def test_nothing_that_kernels_write_takes_the_read_only_path():
    """With programmatic launches a kernel may be resident while earlier ones still write what it reads: no load of these kernels may
    be one that promises data constant for the kernel's lifetime, and lengths, read ahead of a wait, come from L2. (Rotary tables and
    weights, which no kernel writes, may take it.)"""
    folder = Path(__file__).resolve().parent.parent / "llm-decode-triton-6gb_b200" / "csrc"
    for name in ("paged_append.cu", "paged_attention.cu", "paged_prefix.cu", "paged.cuh", "pipeline.cuh", "verify_drafts.cu"):
        code = "\n".join(line.split("//")[0] for line in (folder / name).read_text().splitlines())
        code = re.sub(r"void load8\(const C\* p,.*?\n}\n", "", code, flags=re.S)
        assert not re.search(r"__ldg\(|ldg_\w+\(|\.nc\b|__restrict__|\bseqlens\[", code), name


def test_every_bounded_wait_of_the_paged_kernels_is_looked_at():
    """A wait on an mbarrier that runs out has to reach the result (as NaN): each one's outcome goes into a flag, or
    into the number of tries that the next waits have."""
    csrc = Path(__file__).resolve().parent.parent / "llm-decode-triton-6gb_b200" / "csrc"
    found = 0
    for name in ("paged_attention.cu", "paged_prefix.cu"):
        for line in (csrc / name).read_text().splitlines():
            code = line.split("//")[0]
            if re.search(r"mbar_wait(_tries)?\(", code):
                found += 1
                assert re.search(r"\b(ok|landed) (=|&&) .*mbar_wait\(|\btries = mbar_wait_tries\(.*, tries\);", code), f"{name}: {line.strip()}"
    assert found >= 15


# ---- the oracle draws from the target's own distribution
def test_oracle_draws_as_the_target():
    """Averaging over the drafts' distribution and over a fine grid of the random numbers, the first token
    is distributed as p[0] exactly (up to the grid's step)."""
    rng = np.random.default_rng(0)
    V, n = 5, 400
    p = rng.dirichlet(np.ones(V), 2)[None]
    q = rng.dirichlet(np.ones(V), 1)[None]
    got = np.zeros(V)
    grid = (np.arange(n) + 0.5) / n
    for x in range(V):
        for u in grid:
            accept = u * q[0, 0, x] < p[0, 0, x]
            if accept:
                got[x] += q[0, 0, x] / n
            else:   # the accepting number only decides; the drawing one spans the grid
                us = np.stack([np.full(n, u), grid], 1)
                tok, acc = verify_ref(np.full((n, 1), x), np.repeat(p, n, 0), us, np.repeat(q, n, 0))
                assert not acc.any()
                got += np.bincount(tok[:, 0], minlength=V) * q[0, 0, x] / n / n
    # each of the grid's two averages is off by at most a step per token
    assert np.abs(got - p[0, 0]).max() <= 2.0 * V / n


def test_oracle_edges():
    p = np.array([[[0.5, 0.0, 0.5], [0.0, 1.0, 0.0]]])
    same = p[:, :1]
    # u q = p exactly is a refusal; with p == q nothing is left over, so the draw is from p
    tok, acc = verify_ref(np.array([[0]]), p, np.array([[1.0, 0.6]]), same)
    assert acc[0] == 0 and tok.tolist() == [[2, -1]]
    tok, acc = verify_ref(np.array([[2]]), p, np.array([[0.9, 0.0]]), same)
    assert acc[0] == 1 and tok.tolist() == [[2, 1]]
    tok, acc = verify_ref(np.array([[1]]), p, np.array([[0.0, 0.999]]))   # p = 0 is never accepted
    assert acc[0] == 0 and tok.tolist() == [[2, -1]]
