"""GPU: the 4-bit paged cache (append, read, attention) and page planning against their definitions (``oracle/int4_ref.py``).

Bounds, element by element, h = half a step of a dtype (2^-8 bf16, 2^-11 fp16):

* codes, scales and bases follow IEEE fp32 steps: the values read back are equal;
* q_out: fp32 between load and store, under 2^-19 of the terms' size (as in ``test_paged_gpu.py``), and one rounding;
* page planning: whole numbers, equal;
* attention: a value's weight p s is rounded to fp16 (2^-11) or, below 2^-21 of the largest s, by 2^-25 steps of a unit of
  2^(E - 7) <= 2^-5 s_max, times a code up to 15 <= 2^4: 2^-26 s_max per key against a sum of weights of at least 1. Scores:
  the sums over D elements of q c s and q m in fp32, 2 D 2^-23 reach with reach = max scale sum |q_d| (|m| + s c), twice since
  the normalising sum has it too, and doubled for the running maximum; the sums over n keys n 2^-23. All times mass = sum p_j (|m| + s c)_j,
  then the output's own rounding.
"""
import numpy as np
import pytest
import torch

from b200kernels import _lib
from b200kernels.page_plan import PageTables, StepPlan
from b200kernels.paged import PagedKV, paged_attention, paged_rope_append
from b200kernels.paged_int4 import (PagedKVInt4, paged_int4_append, paged_int4_attention, paged_int4_attention_workspace,
                                    paged_int4_read, rotary_tables)
from b200kernels.speculative import verify_drafts
from oracle.int4_ref import plan_ref, quantise_ref, size_ref, turn_ref, values_ref
from oracle.paged_ref import paged_attention_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def empty_pool(pages, KVH, ps, D, dtype, group=64):
    """A pool whose every byte is 0xFF: scales and bases that are NaN."""
    kv = PagedKVInt4.empty(pages, KVH, ps, D, dtype, DEV, group_size=group)
    kv.pages.fill_(255)
    return kv


# ------------------------------------------------------------------ append and read
def append_case(N, B, H, KVH, D, dtype, seed=0, S=512, ps=16, magnitude=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (magnitude * torch.randn(N, h, D, generator=g) for h in (H, KVH, KVH))
    k *= torch.exp(0.5 * torch.randn(KVH, D, generator=g))
    v += torch.randn(KVH, D, generator=g)
    per = -(-S // ps)
    table = torch.randperm(B * per, generator=g).view(B, per).int()
    pos = torch.randint(0, S - N // B - 1, (B,), generator=g)[:, None] + torch.arange(N // B)
    return q.to(dtype), k.to(dtype), v.to(dtype), pos.reshape(-1), table


def check_values(got, x32, group, dtype):
    """`got` [N, KVH, D] fp32 of the cache against x32, what was quantised."""
    codes, s, m = quantise_ref(x32, group, dtype)
    want = values_ref(codes, s, m, x32.shape[-1])
    got = got.cpu().numpy()
    assert (np.isnan(got) == np.isnan(want)).all()
    assert (got == want)[~np.isnan(want)].all(), np.abs(np.nan_to_num(got - want)).max()


@pytest.mark.parametrize("D,group", [(128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,B", [(1, 1), (15, 3), (64, 64), (700, 2)])
def test_append_without_rotation_is_exact(D, group, dtype, N, B):
    """Keys and values as they are, codes equal to the definition's, through any page order."""
    q, k, v, pos, table = append_case(N, B, 4, 3, D, dtype, seed=N + D)
    kv = empty_pool(table.numel(), 3, 16, D, dtype, group)
    assert paged_int4_append(kv, None, k.to(DEV), v.to(DEV), pos.to(DEV), table.to(DEV)) is None
    gk, gv = paged_int4_read(kv, pos.to(DEV), table.to(DEV), out_dtype=F32)
    check_values(gk, k.float().numpy(), group, dtype)
    check_values(gv, v.float().numpy(), group, dtype)
    hk, hv = paged_int4_read(kv, pos.to(DEV), table.to(DEV))
    assert torch.equal(hk, gk.to(dtype)) and torch.equal(hv, gv.to(dtype))


@pytest.mark.parametrize("dtype,D,group", [(BF16, 128, 64), (BF16, 64, 32), (F16, 128, 64)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_agrees_with_torch_bit_for_bit(dtype, D, group, norm):
    """A prompt's keys and values against the same steps in elementary torch operations on the GPU: a scale that falls on the other side
    of a 16-bit step moves codes of its run by a whole step, half the spread of the values."""
    N, KVH, ps = 8168, 8, 64
    for seed in range(3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        k, v = (torch.randn(N, KVH, D, generator=g, device=DEV) for _ in range(2))
        k = (k * torch.exp(0.3 * torch.randn(KVH, D, generator=g, device=DEV))).to(dtype)
        v = v.to(dtype)
        w = (1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
        cos, sin = (t.to(DEV) for t in rotary_tables(N, D, 1e6))
        kv = empty_pool(-(-N // ps), KVH, ps, D, dtype, group)
        table, pos = torch.arange(kv.num_pages, dtype=torch.int32, device=DEV)[None], torch.arange(N, device=DEV)
        paged_int4_append(kv, None, k, v, pos, table, cos, sin, k_weight=w, eps=1e-5)
        got = paged_int4_read(kv, pos, table, out_dtype=F32)
        x = k.float()
        if norm:
            x = x * (x.double().square().mean(-1, keepdim=True) + float(np.float32(1e-5))).rsqrt().float() * w.float()
        a, b = x[..., :D // 2], x[..., D // 2:]
        c, s = cos[:, None], sin[:, None]
        for out, x in zip(got, (torch.cat((a * c - b * s, b * c + a * s), -1), v.float())):
            x = x.unflatten(-1, (-1, group))
            base = x.amin(-1, keepdim=True).to(dtype).float()
            scale = ((x.amax(-1, keepdim=True) - base) / 15).clamp(min=0).to(dtype).float()
            code = torch.where(scale > 0, ((x - base) / scale).round().clamp(0, 15), 0.0)
            want = (base.double() + scale.double() * code.double()).float().flatten(-2)
            assert torch.equal(out, want), int((out != want).sum())


def test_append_touches_its_own_slots_only():
    """Every byte of the pool that is not the new entries' stays as it was, and an entry does not depend on its neighbours."""
    D, KVH, ps = 128, 2, 48
    g = torch.Generator().manual_seed(1)
    kv = empty_pool(5, KVH, ps, D, F16)
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=DEV)
    every = torch.arange(96, device=DEV)
    k, v = (torch.randn(96, KVH, D, generator=g).half().to(DEV) for _ in range(2))
    other = torch.tensor([x for x in (0, 2, 4)], device=DEV)
    for at in (0, 5, 9, 15, 16, 47, 48, 95):
        before_k, before_v = paged_int4_read(kv, every, table, out_dtype=F32)
        paged_int4_append(kv, None, k[at:at + 1], v[at:at + 1], every[at:at + 1], table)
        after_k, after_v = paged_int4_read(kv, every, table, out_dtype=F32)
        keep = every != at
        assert torch.equal(before_k[keep].nan_to_num(7), after_k[keep].nan_to_num(7))
        assert torch.equal(before_v[keep].nan_to_num(7), after_v[keep].nan_to_num(7))
        check_values(after_k[at:at + 1], k[at:at + 1].float().cpu().numpy(), 64, F16)
        check_values(after_v[at:at + 1], v[at:at + 1].float().cpu().numpy(), 64, F16)
        assert (kv.pages[other] == 255).all()


@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (128, 32), (128, 96), (128, 16), (64, 64), (64, 48), (64, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype,table_dtype", [(F16, F32), (BF16, F32), (BF16, BF16)])
def test_append_rotations(D, R, interleaved, norm, dtype, table_dtype):
    N, B, H, KVH, group = 36, 3, 6, 3, 32 if R == 96 else 64
    q, k, v, pos, table = append_case(N, B, H, KVH, D, dtype, seed=D + R)
    cos, sin = rotary_tables(512, R, 1e4, dtype=table_dtype)
    g = torch.Generator().manual_seed(5)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)) if norm else (None, None)
    kv = empty_pool(table.numel(), KVH, 16, D, dtype, group)
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    out = paged_int4_append(kv, on(q), on(k), on(v), on(pos), on(table), on(cos), on(sin), interleaved=interleaved,
                            q_weight=on(qw), k_weight=on(kw), eps=1e-5)
    gk, gv = paged_int4_read(kv, on(pos), on(table), out_dtype=F32)
    c, s = f64(cos)[pos.numpy()], f64(sin)[pos.numpy()]
    w = lambda t: None if t is None else f64(t)  # noqa: E731
    check_values(gk, turn_ref(k.float().numpy(), c, s, interleaved, w(kw), 1e-5, exact32=True), group, dtype)
    check_values(gv, v.float().numpy(), group, dtype)
    ref = turn_ref(f64(q), c, s, interleaved, w(qw), 1e-5)
    normed = turn_ref(f64(q), None, None, interleaved, w(qw), 1e-5)
    size = np.abs(turn_ref(np.abs(normed), np.abs(c), -np.abs(s), interleaved)) + np.abs(turn_ref(np.abs(normed), np.abs(c), np.abs(s), interleaved))
    err = np.abs(f64(out) - ref)
    assert (err <= half_step(dtype) * np.abs(ref) + 2.0 ** -19 * size + 2.0 ** -25).all(), err.max()


@pytest.mark.parametrize("D,R", [(128, 128), (128, 96), (64, 32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_rotations_with_fp16_tables(D, R, interleaved):
    test_append_rotations(D, R, interleaved, True, F16, F16)


def test_append_weights_alone_of_either():
    """A norm of the keys and none of the queries, and the other way round; tables of none."""
    q, k, v, pos, table = append_case(8, 2, 4, 2, 64, F16, seed=3)
    w = (1 + 0.2 * torch.randn(64, generator=torch.Generator().manual_seed(2))).half()
    for qw, kw in ((w, None), (None, w)):
        kv = empty_pool(table.numel(), 2, 16, 64, F16)
        out = paged_int4_append(kv, q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), table.to(DEV), eps=1e-5,
                                q_weight=None if qw is None else qw.to(DEV), k_weight=None if kw is None else kw.to(DEV))
        ref = turn_ref(f64(q), None, None, False, None if qw is None else f64(qw), 1e-5)
        assert (np.abs(f64(out) - ref) <= (half_step(F16) + 2.0 ** -19) * np.abs(ref) + 2.0 ** -25).all()
        gk, _ = paged_int4_read(kv, pos.to(DEV), table.to(DEV), out_dtype=F32)
        check_values(gk, turn_ref(k.float().numpy(), None, None, False, None if kw is None else f64(kw), 1e-5, exact32=True), 64, F16)


@pytest.mark.parametrize("D,R,interleaved", [(128, 128, False), (128, 64, True), (64, 64, False), (64, 16, True)])
@pytest.mark.parametrize("size", [1e38, 1e30, 1e19, 2.0 ** 60, 1e-13, 1e-25, 1e-37])
def test_append_norms_of_any_size(D, R, interleaved, size):
    """Heads whose squares leave fp32's range, next to ordinary ones (whose bits stay) and one of zeros; queries and keys alike."""
    N, B, H, KVH = 24, 3, 10, 5
    q, k, v, pos, table = append_case(N, B, H, KVH, D, BF16, seed=D)
    cos, sin = rotary_tables(512, R, 1e4)
    w = (1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(6))).bfloat16()
    kv = empty_pool(table.numel(), KVH, 16, D, BF16)

    def run(q, k):
        return paged_int4_append(kv, q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), table.to(DEV), cos.to(DEV), sin.to(DEV),
                                 interleaved=interleaved, q_weight=w.to(DEV), k_weight=w.to(DEV), eps=0.0)

    usual = run(q, k)
    q, k = q.clamp(-3, 3), k.clamp(-3, 3)
    q[:, 1::3], k[:, 1::3] = (q[:, 1::3].float() * size).bfloat16(), (k[:, 1::3].float() * size).bfloat16()
    q[:, 5] = 0
    out = run(q, k)
    gk, _ = paged_int4_read(kv, pos.to(DEV), table.to(DEV), out_dtype=F32)
    c, s = f64(cos)[pos.numpy()], f64(sin)[pos.numpy()]
    check_values(gk, turn_ref(k.float().numpy(), c, s, interleaved, f64(w), 0.0, exact32=True), 64, BF16)
    keep = [0, 2, 3, 6, 8, 9]
    same = (q[:, keep].abs() < 3).all(-1)
    assert torch.equal(out.cpu()[:, keep][same], usual.cpu()[:, keep][same]) and same.any()
    live = [h for h in range(H) if h != 5]
    ref = turn_ref(f64(q)[:, live], c, s, interleaved, f64(w), 0.0)
    normed = turn_ref(f64(q)[:, live], None, None, interleaved, f64(w), 0.0)
    bound = np.abs(turn_ref(np.abs(normed), np.abs(c), -np.abs(s), interleaved)) + np.abs(turn_ref(np.abs(normed), np.abs(c), np.abs(s), interleaved))
    err = np.abs(f64(out)[:, live] - ref)
    assert (err <= half_step(BF16) * np.abs(ref) + 2.0 ** -19 * bound + 2.0 ** -25).all(), err.max()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_odd_values(dtype):
    """Equal elements, tiny and huge ranges, ties of the rounding, signed zeros, infinities and NaN."""
    D, rows = 128, []
    g = torch.Generator().manual_seed(7)
    big = torch.finfo(dtype).max
    rows += [torch.zeros(D), torch.full((D,), 3.7), torch.full((D,), -0.0), torch.arange(D) / 2.0 - 20, torch.arange(D).float()]
    rows += [torch.where(torch.arange(D) % 2 == 0, 0.0, 7.5), (torch.arange(D) % 31) * 0.5]           # ties at s = 1 and s = 0.5
    rows += [torch.randn(D, generator=g) * 1e-7, torch.randn(D, generator=g) * 3e4, torch.full((D,), float(big))]
    rows += [torch.where(torch.arange(D) % 2 == 0, float(big), -float(big)), torch.randn(D, generator=g) * torch.finfo(dtype).tiny]
    for bad in (INF, -INF, NAN):
        x = torch.randn(D, generator=g)
        x[70] = bad                           # the second run of 64 only
        rows.append(x)
    x = torch.stack(rows).to(dtype)
    k = x[:, None].contiguous()
    kv = empty_pool(2, 1, 16, D, dtype)
    pos = torch.arange(len(rows), device=DEV)
    table = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    paged_int4_append(kv, None, k.to(DEV), k.to(DEV), pos, table)
    gk, gv = paged_int4_read(kv, pos, table, out_dtype=F32)
    check_values(gk, k.float().numpy(), 64, dtype)
    check_values(gv, k.float().numpy(), 64, dtype)
    assert torch.isfinite(gk[-1, 0, :64]).all() and torch.isnan(gk[-1, 0, 64:]).all()


def test_append_padding_bad_pages_and_read_of_them():
    N, H, KVH, D, ps, S = 9, 4, 2, 64, 16, 40
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(N, h, D, generator=g).half().to(DEV) for h in (H, KVH, KVH))
    kv = empty_pool(6, KVH, ps, D, F16)
    clean = kv.pages.clone()
    cos, sin = (t.to(DEV) for t in rotary_tables(S, D))
    table = torch.tensor([[0, 1], [2, 99], [-1, 3]], dtype=torch.int32, device=DEV)
    #                 fine  padding: sequence -1, 3; position -1, S; page 99, -1, outside the table; far out
    seq = torch.tensor([0, -1, 3, 0, 1, 1, 2, 0, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([17, 3, 3, -1, S, 20, 2, 39, 2 ** 40], dtype=torch.int64, device=DEV)
    q_out = torch.full((N, H, D), 9.0, dtype=F16, device=DEV)
    paged_int4_append(kv, q, k, v, pos, table, cos, sin, q_out=q_out, seq_ids=seq)
    assert (q_out[1:5] == 9).all() and (q_out[8] == 9).all() and not (q_out[5:8] == 9).all(-1).any() and not (q_out[0] == 9).any()
    at = torch.tensor([1, 17], device=DEV)
    gk, gv = paged_int4_read(kv, at, table[:1], out_dtype=F32)
    assert torch.isnan(gk[0]).all() and torch.isfinite(gk[1]).all()
    check_values(gv[1:], v[:1].float().cpu().numpy(), 64, F16)
    changed = (kv.pages != clean).flatten(1).any(1)
    assert changed.tolist() == [False, True, False, False, False, False]
    # reads: padding keeps its rows, bad pages give zeros
    ko, vo = (torch.full((N, KVH, D), 5.0, dtype=F16, device=DEV) for _ in range(2))
    r = paged_int4_read(kv, pos, table, seq_ids=seq, k_out=ko, v_out=vo)
    assert r[0] is ko and r[1] is vo
    for t in (ko, vo):
        assert (t[[1, 2, 3, 4, 7, 8]] == 5).all() and (t[[5, 6]] == 0).all() and torch.isfinite(t[0]).all()


def test_append_in_place_strides_and_views():
    """q_out aliasing q, parts of a fused projection, pools with the heads outside the pages, reads into slices."""
    N, H, KVH, D, ps = 10, 8, 2, 128, 32
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(N, (H + 2 * KVH) * D + 64, generator=g).bfloat16().to(DEV)
    q, k, v = fused[:, :H * D].view(N, H, D), fused[:, H * D:(H + KVH) * D].view(N, KVH, D), fused[:, (H + KVH) * D:-64].view(N, KVH, D)
    cos, sin = (t.to(DEV) for t in rotary_tables(64, 64, dtype=F32))
    wide = torch.zeros(64, 96, device=DEV)
    wide[:, :32], wide[:, 32:64] = cos, sin
    w = torch.rand(D, generator=g).bfloat16().to(DEV)
    pos = torch.tensor([0, 15, 16, 40, 63, 1, 2, 3, 4, 5], device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    a = empty_pool(4, KVH, ps, D, BF16)
    want = paged_int4_append(a, q, k, v, pos, table, cos, sin, q_weight=w, k_weight=w)
    block = a.pages.shape[2]
    memory = torch.full((KVH, 4, block + 32), 255, dtype=torch.uint8, device=DEV)
    b = PagedKVInt4(memory.transpose(0, 1)[:, :, :block], ps, D, BF16)
    q2 = q.clone()
    got = paged_int4_append(b, q2, k, v, pos, table, wide[:, :32], wide[:, 32:64], q_weight=w, k_weight=w, q_out=q2)
    assert got is q2 and torch.equal(q2, want) and torch.equal(a.pages, b.pages) and (memory[:, :, block:] == 255).all()
    ko = torch.full((N, KVH + 1, D + 8), 7.0, device=DEV)
    rk, rv = paged_int4_read(b, pos, table, k_out=ko[:, :KVH, :D], v_out=False)
    assert rv is None and torch.equal(rk, paged_int4_read(a, pos, table, out_dtype=F32)[0])
    assert (ko[:, KVH] == 7).all() and (ko[:, :, D:] == 7).all()


@pytest.mark.parametrize("D,KVH", [(128, 8), (128, 9), (64, 17), (64, 8), (128, 1)])
@pytest.mark.parametrize("out", ["both", "keys", "values"])
def test_read_of_whole_tiles_and_their_borders(D, KVH, out):
    """Whole sequences of odd lengths, whose tiles lie anywhere in the call, among tokens in another order, padding and pages
    outside the pool: each row as it is read alone."""
    g = torch.Generator().manual_seed(D + KVH)
    lens, ps = [3333, 16, 1, 47, 1600, 15, 640], 32
    per = -(-max(lens) // ps)
    table = torch.randperm(len(lens) * per, generator=g).int().view(len(lens), per)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).int()
    pos = torch.cat([torch.arange(n) for n in lens])
    N = pos.numel()
    k, v = (torch.randn(N, KVH, D, generator=g).half() for _ in range(2))
    kv = empty_pool(table.numel(), KVH, ps, D, F16)
    paged_int4_append(kv, None, k.to(DEV), v.to(DEV), pos.to(DEV), table.to(DEV), seq_ids=seq.to(DEV))
    table[0, 5], table[4, 3] = -1, 10 ** 6
    order = torch.cat([torch.arange(1000), 1000 + torch.randperm(500, generator=g), torch.arange(1500, N)])
    seq, pos, k, v = seq[order], pos[order], k[order], v[order]
    seq[2000:2003], pos[40] = -1, -7                     # padding inside of tiles
    keep = torch.ones(N, dtype=torch.bool)
    keep[2000:2003] = keep[40] = False
    gone = keep & (((seq == 0) & (pos // ps == 5)) | ((seq == 4) & (pos // ps == 3)))
    outs = [torch.full((N, KVH, D), 9.0, device=DEV) if out != skip else False for skip in ("values", "keys")]
    got = paged_int4_read(kv, pos.to(DEV), table.to(DEV), seq_ids=seq.to(DEV), k_out=outs[0], v_out=outs[1])
    for x, y in zip(got, (k, v)):
        if x is None:
            continue
        assert (x[~keep] == 9).all() and (x[gone] == 0).all()
        check_values(x.cpu()[keep & ~gone], y[keep & ~gone].float().numpy(), 64, F16)


# ------------------------------------------------------------------ attention
class Case:
    """Random sequences whose unused slots and pages hold NaN factors and whose unused table entries point nowhere."""

    def __init__(self, lens, H=8, KVH=2, D=128, T=1, ps=16, group=64, dtype=F16, seed=0, spare=3, magnitude=1.0, keys=None, values=None):
        g = torch.Generator().manual_seed(seed)
        B, self.ps, self.group, self.dtype = len(lens), ps, group, dtype
        need = [-(-n // ps) for n in lens]
        total = sum(need) + spare
        perm = torch.randperm(total, generator=g).int()
        self.table = torch.full((B, max(max(need), 1) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        N = sum(lens)
        seq = torch.repeat_interleave(torch.arange(B), self.lens.long()).int()
        pos = torch.cat([torch.arange(n) for n in lens]) if N else torch.zeros(0, dtype=torch.long)
        self.k = (magnitude * torch.randn(N, KVH, D, generator=g) * torch.exp(0.3 * torch.randn(KVH, D, generator=g))).to(dtype) if keys is None else keys(seq, pos).to(dtype)
        self.v = (magnitude * torch.randn(N, KVH, D, generator=g) + 0.5 * torch.randn(KVH, D, generator=g)).to(dtype) if values is None else values(seq, pos).to(dtype)
        self.q = (magnitude * torch.randn(B, T, H, D, generator=g)).to(dtype)
        self.seq, self.pos, self.scale = seq, pos, D ** -0.5
        self.kv = empty_pool(total, KVH, ps, D, dtype, group)
        if N:
            paged_int4_append(self.kv, None, self.k.to(DEV), self.v.to(DEV), pos.to(DEV), self.table.to(DEV), seq_ids=seq.to(DEV))

    def run(self, **kw):
        return paged_int4_attention(self.kv, self.q.to(DEV), self.table.to(DEV), self.lens.to(DEV), **kw)

    def pools(self, what):
        """The codes' values (or sizes) as [pages, KVH, ps, D] of float64, zeros elsewhere."""
        KVH, D = self.k.shape[1:]
        out = []
        for x in (self.k, self.v):
            parts = quantise_ref(x.float().numpy(), self.group, self.dtype)
            pool = np.zeros((self.kv.num_pages, KVH, self.ps, D))
            page = self.table[self.seq.long(), self.pos // self.ps].numpy()
            keep = (page >= 0) & (page < self.kv.num_pages)
            pool[page[keep], :, (self.pos % self.ps).numpy()[keep]] = what(*parts, D)[keep]
            out.append((pool, parts))
        return out

    def check(self, out):
        (k, _), (v, (_, vs, _)) = self.pools(values_ref)
        (ksize, _), (vsize, _) = self.pools(size_ref)
        B, T, H, D = self.q.shape
        args = (self.table.numpy(), self.lens.numpy(), self.scale)
        ref, _, _ = paged_attention_ref(f64(self.q), k, v, *args)
        mass, _, _ = paged_attention_ref(f64(self.q), k, vsize, *args)
        _, _, reach = paged_attention_ref(f64(self.q), ksize, v, *args)
        n = max(1, int(self.lens.max()))
        s_max = float(np.nanmax(vs)) if vs.size else 0.0
        bound = (2.0 ** -11 + 4 * 2 * D * 2.0 ** -23 * reach[..., None] + n * 2.0 ** -23) * mass + n * 2.0 ** -26 * s_max
        bound = bound + half_step(out.dtype) * (np.abs(ref) + bound) + 2.0 ** -25
        got = f64(out)
        assert np.isfinite(got).all()
        err = np.abs(got - ref)
        assert (err <= bound).all(), f"worst error / bound {(err / bound).max():.2f}, error {err.max():.3e}"
        for b, n_b in enumerate(self.lens.tolist()):   # queries that see nothing give zeros
            for t in range(T):
                if n_b - T + 1 + t <= 0:
                    assert (got[b, t] == 0).all()


@pytest.mark.parametrize("lens", [[1], [2], [15, 16, 17], [63], [64], [65], [128, 1, 0, 127], [300, 517, 16, 15, 17]])
@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_attention_lengths(lens, D, group):
    c = Case(lens, D=D, group=group, seed=len(lens) + D)
    c.check(c.run())


@pytest.mark.parametrize("ps", [16, 32, 48, 64, 112, 256, 1024])
def test_attention_page_sizes(ps):
    c = Case([1, 257, 100, 0, 64, 1100], ps=ps, T=2, dtype=BF16, seed=ps)
    c.check(c.run())


@pytest.mark.parametrize("H,KVH,T", [(1, 1, 1), (8, 8, 1), (14, 2, 1), (16, 1, 1), (8, 2, 2), (8, 2, 3), (7, 1, 5), (9, 3, 3),
                                     (32, 8, 5), (16, 1, 4), (15, 1, 4), (16, 1, 16), (6, 2, 16), (12, 1, 11)])
@pytest.mark.parametrize("dtype,group", [(F16, 64), (BF16, 32)])
def test_attention_heads_and_drafts(H, KVH, T, dtype, group):
    lens = [T + 130, 0, 1, T, max(0, T - 1), T + 63]   # shorter than the drafts, too: their first queries see nothing
    c = Case(lens, H=H, KVH=KVH, T=T, dtype=dtype, group=group, seed=H + T)
    c.check(c.run())
    c = Case(lens, H=H, KVH=KVH, T=T, D=64, dtype=dtype, group=group, seed=H + T)
    c.check(c.run(out_dtype=F32))


@pytest.mark.parametrize("lens,H,KVH,T,D,ps", [
    ([5000, 1, 2777, 4096, 0, 63, 64, 65, 129], 8, 2, 1, 128, 16), ([3001, 517, 2, 128, 1500], 12, 2, 3, 64, 64),
    ([700, 1300], 16, 1, 4, 128, 32), ([9001], 1, 1, 1, 128, 16), ([20011], 4, 1, 1, 64, 64), ([2050 + 37 * i for i in range(9)], 4, 4, 1, 64, 128),
    ([77 * i % 1009 for i in range(300)], 2, 1, 1, 64, 16)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_counts_every_key_once(lens, H, KVH, T, D, ps, dtype):
    """Queries of zeros weigh all keys alike, and values of 0 and 15 (s = 1, m = 0: exact) that mark a key's position modulo
    D / 2 and its run of 64 then give counts over the number of keys: a key that is lost or taken twice at a border of tiles,
    pages, shares or parts changes a count by a whole. Weights and their products with s are powers of two and all
    sums whole numbers below 2^24, so five roundings are left at most; 5 x 2^-24."""
    half = D // 2

    def marks(seq, pos):
        one = torch.nn.functional.one_hot
        return 15.0 * torch.cat([one(pos % half, half), one(pos // 64 % half, half)], -1)[:, None].expand(-1, KVH, -1).float()

    c = Case(lens, H=H, KVH=KVH, T=T, D=D, ps=ps, group=32, dtype=dtype, seed=D + ps, values=marks)
    c.q.zero_()
    got = f64(c.run(out_dtype=F32))
    top = torch.arange(max(max(lens), 1))
    running = np.cumsum(marks(None, top)[:, 0].double().numpy(), 0)
    for b, n_b in enumerate(lens):
        for t in range(T):
            n = n_b - T + 1 + t
            want = running[n - 1] / n if n > 0 else np.zeros(D)
            assert (np.abs(got[b, t] - want) <= 5 * 2.0 ** -24 * want).all(), (b, t, np.abs(got[b, t] - want).max() * max(n, 1))


def test_attention_long_ragged_and_hints():
    c = Case([5000, 1, 2777, 4096], seed=8)
    out = c.run()
    c.check(out)
    c.check(c.run(max_len=5000))
    for hint in (1, 200, 300, 2000, 4096):   # wrong hints cost time only: a CTA or a cluster a unit, however long
        c.check(c.run(max_len=hint))
    assert torch.equal(out, c.run())   # the same bits every run


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_large_scores_and_negative_scale(dtype):
    """Scores of several hundred: the running maximum matters, one key takes nearly all the weight."""
    c = Case([400, 129], T=2, magnitude=6.0, dtype=dtype, seed=4)
    c.check(c.run())
    c.scale = -c.scale
    c.check(c.run(scale=c.scale))


@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1e9, 1e15])
@pytest.mark.parametrize("T,H", [(1, 8), (4, 16)])
def test_attention_scores_of_any_size(size, T, H):
    """Scores up to 10^32, whose steps in fp32 are far above one: the key with the largest takes all the weight. (The oracle checks that no
    other comes near it: the fp32 sums are within D 2^-23 of a score's terms, twice for a difference, and 2^-30 of weight is 30 more.)"""
    c = Case([700, 90], H=H, KVH=2, T=T, D=64, dtype=BF16, seed=T, magnitude=1.0)
    c = Case([700, 90], H=H, KVH=2, T=T, D=64, dtype=BF16, seed=T,
             keys=lambda seq, pos: c.k.float() * size, values=lambda seq, pos: c.v.float())
    c.q = (c.q.float() * size).bfloat16()
    (k, _), (v, parts) = c.pools(values_ref)
    ksize, wide = c.pools(size_ref)[0][0], c.pools(lambda codes, s, m, D: size_ref(np.full_like(codes, 15), s, m, D))[1][0]
    got = f64(c.run(out_dtype=F32))
    sure = 0
    for b, n in enumerate(c.lens.tolist()):
        page = c.table[b, torch.arange(n) // c.ps].long().numpy()
        slot = np.arange(n) % c.ps
        for t in range(T):
            lim = n - T + 1 + t
            for h in range(H):
                kk, vv, ss, ww = (x[page, h * 2 // H, slot][:lim] for x in (k, v, ksize, wide))
                q = f64(c.q[b, t, h])
                score = kk @ q * c.scale
                order = np.argsort(score)
                reach = (ss @ np.abs(q)).max() * c.scale
                if score[order[-1]] - score[order[-2]] < 4 * 64 * 2.0 ** -23 * reach + 30:
                    continue
                sure += 1
                err = np.abs(got[b, t, h] - vv[order[-1]])
                assert (err <= (2.0 ** -11 + n * 2.0 ** -23) * ww[order[-1]] + 2.0 ** -29 * np.abs(ww).max()).all(), (b, t, h, err.max())
    assert np.isfinite(got).all() and sure > T * H


def test_attention_rising_scores():
    """Scores that grow along the sequence: the running maximum moves again and again."""
    direction = torch.randn(64, generator=torch.Generator().manual_seed(1)).sign()
    c = Case([1300, 700], H=8, KVH=2, T=2, D=64, dtype=BF16, seed=50,
             keys=lambda seq, pos: (0.2 * torch.randn(pos.numel(), 2, 64, generator=torch.Generator().manual_seed(3)) + direction * (0.02 * pos[:, None, None])))
    c.q = (c.q.float() * 0.2 + direction).bfloat16()
    c.check(c.run())


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e20])
def test_attention_sizes_of_queries_and_values(size):
    """Queries far from one, and keys that undo it; values of sizes that rise and fall by ten decades along a sequence."""
    g = torch.Generator().manual_seed(11)
    grow = lambda seq, pos: torch.randn(pos.numel(), 2, 64, generator=g) * 10.0 ** (5 * torch.sin(pos / 97.0))[:, None, None]  # noqa: E731
    c = Case([900, 33], D=64, T=3, dtype=BF16, seed=12, values=grow,
             keys=lambda seq, pos: torch.randn(pos.numel(), 2, 64, generator=g) / size)
    c.q = (c.q.float() * size).bfloat16()
    c.check(c.run())


def check_by_row(c, out):
    """Each row against what its own keys add to it. A weight p s keeps its 11 bits down to 2^-19 of the largest p s that the row
    has met and is rounded by 2^-30 of that below (2^-25 steps of a unit in which the largest was 2^5 or more), times a centred
    code up to 8: 2^-27 of it a key; its size is at most a fifteenth of the row's largest mass = sum p (|m| + 15 s). Scores and sums as
    in the bounds above, of this mass (codes are centred, so that sums are as large as the run's range)."""
    (k, _), (v, _) = c.pools(values_ref)
    (ksize, _), (wide, _) = c.pools(lambda codes, s, m, D: size_ref(np.full_like(codes, 15), s, m, D))
    ksize = c.pools(size_ref)[0][0]
    args = (c.table.numpy(), c.lens.numpy(), c.scale)
    ref, _, _ = paged_attention_ref(f64(c.q), k, v, *args)
    mass, _, _ = paged_attention_ref(f64(c.q), k, wide, *args)
    _, _, reach = paged_attention_ref(f64(c.q), ksize, v, *args)
    n, D = int(c.lens.max()), c.q.shape[-1]
    bound = (2.0 ** -11 + 8 * D * 2.0 ** -23 * reach[..., None] + n * 2.0 ** -23) * mass + n * 2.0 ** -27 / 15 * mass.max(-1, keepdims=True)
    bound = bound + half_step(out.dtype) * (np.abs(ref) + bound) + 2.0 ** -25 * (out.dtype == F16)
    err = np.abs(f64(out) - ref)
    assert (err <= bound).all(), f"worst error / bound {(err / bound).max():.2e}"


@pytest.mark.parametrize("H,T", [(8, 2), (16, 2), (16, 3), (16, 4)])   # 8 to 32 rows of a KV head
@pytest.mark.parametrize("D,group,dtype", [(64, 64, BF16), (128, 32, BF16), (128, 64, F16), (64, 32, F16)])
@pytest.mark.parametrize("where", ["hidden", "first", "middle", "last", "many"])
def test_attention_huge_values_of_little_weight(H, T, D, group, dtype, where):
    """Values 2^40 (fp16: 2^25) times the others' that a row does not see, or gives next to no weight, wherever they lie: the first keys
    that a warp meets, before a running maximum that rises by 60, or behind it."""
    g = torch.Generator().manual_seed(D + T)
    lens = [700, 300 + T]
    direction = torch.randn(D, generator=g).sign()
    small, huge = (1.0, 2.0 ** 40) if dtype == BF16 else (2.0 ** -10, 2.0 ** 15 - 2.0 ** 5)

    def chosen(seq, pos):
        n = torch.tensor(lens)[seq.long()]
        return {"hidden": pos == n - 1, "first": pos == 0, "middle": pos == 150, "last": pos == n - T - 1, "many": pos < 200}[where]

    def values(seq, pos):
        return torch.randn(pos.numel(), 2, D, generator=g).clamp(-2, 2) * torch.where(chosen(seq, pos), huge / 2, small)[:, None, None]

    def keys(seq, pos):   # little weight: scores of -60 log2 units against a few
        low = torch.where(chosen(seq, pos) & (where != "hidden"), -42.0 * D ** -0.5, 0.0)[:, None, None]
        return 0.3 * torch.randn(pos.numel(), 2, D, generator=g) + low * direction

    c = Case(lens, H=H, KVH=2, T=T, D=D, group=group, dtype=dtype, seed=H + T, keys=keys, values=values)
    c.q = (0.2 * torch.randn(c.q.shape, generator=g) + direction).to(dtype)
    check_by_row(c, c.run(out_dtype=F32))
    check_by_row(c, c.run(max_len=200, out_dtype=F32))    # a unit a block


def test_attention_rows_do_not_depend_on_one_another():
    """Bits of a row with and without others that move their own maximum or unit in the same tiles."""
    g = torch.Generator().manual_seed(4)
    grow = lambda seq, pos: torch.randn(pos.numel(), 1, 64, generator=torch.Generator().manual_seed(8)) * 2.0 ** (pos % 23)[:, None, None]  # noqa: E731
    c = Case([900], H=4, KVH=1, T=1, D=64, dtype=BF16, seed=3, values=grow)
    c.q = torch.randn(1, 1, 4, 64, generator=g).bfloat16()
    want = c.run()
    check_by_row(c, want)
    for row in range(4):
        other = c.q.clone()
        c.q = (torch.randn(1, 1, 4, 64, generator=g) * 20).bfloat16()
        c.q[:, :, row] = other[:, :, row]
        assert torch.equal(c.run()[:, :, row], want[:, :, row])
        c.q = other


def test_attention_layouts_and_strides():
    c = Case([100, 33, 257], dtype=BF16, T=2, seed=5)
    ref = c.run()
    c.check(ref)
    B, T, H, D = c.q.shape
    wide = torch.full((B, T, H + 4, D), NAN, dtype=BF16, device=DEV)     # q as part of a fused projection
    wide[:, :, :H] = c.q.to(DEV)
    table = torch.full((B, c.table.shape[1] + 5), 10 ** 9, dtype=torch.int32, device=DEV)
    table[:, :c.table.shape[1]] = c.table.to(DEV)
    outw = torch.full((T, B, H + 2, D), 7.0, dtype=BF16, device=DEV)
    out = outw.transpose(0, 1)[:, :, 1:H + 1]
    heads = torch.full((c.kv.kv_heads, c.kv.num_pages, c.kv.pages.shape[2] + 16), 9, dtype=torch.uint8, device=DEV)
    heads[:, :, :-16] = c.kv.pages.transpose(0, 1)
    kv = PagedKVInt4(heads.transpose(0, 1)[:, :, :-16], c.ps, D, BF16)
    got = paged_int4_attention(kv, wide[:, :, :H], table[:, :c.table.shape[1]], c.lens.to(DEV), out=out)
    assert got is out and torch.equal(out, ref)
    assert (outw[:, :, 0] == 7).all() and (outw[:, :, -1] == 7).all()
    odd = torch.empty(B * T * H * D + 1, dtype=BF16, device=DEV)[1:].view(B, T, H, D)   # rows that start on odd halves
    assert torch.equal(paged_int4_attention(c.kv, c.q.to(DEV), c.table.to(DEV), c.lens.to(DEV), out=odd), ref)


def test_attention_lengths_beyond_the_table_and_bad_pages():
    """seqlens past the table's reach are cut to it; a page id outside the pool is not followed (its keys and values count as
    zeros)."""
    c = Case([64, 48], ps=16, seed=6)
    c.table = c.table[:, :3].contiguous()
    c.lens = torch.tensor([64, 2 ** 31 - 1], dtype=torch.int32)
    keep = c.pos < 48
    out = c.run()
    c.lens = torch.tensor([48, 48], dtype=torch.int32)
    c.k, c.v, c.seq, c.pos = c.k[keep], c.v[keep], c.seq[keep], c.pos[keep]
    c.check(out)
    c.table[0, 1], c.table[1, 0] = 10 ** 6, -7
    c.check(c.run())
    c.lens = torch.tensor([-5, 0], dtype=torch.int32)
    assert (c.run() == 0).all()
    assert (paged_int4_attention(c.kv, c.q.to(DEV), torch.zeros(2, 0, dtype=torch.int32, device=DEV), c.lens.to(DEV) + 50) == 0).all()


@pytest.mark.parametrize("H,KVH,T,D,lens", [(8, 2, 4, 128, [130, 64, 7]), (16, 2, 4, 128, [193, 66, 4]),
                                            (16, 1, 4, 64, [129, 260, 5]), (4, 1, 3, 64, [128, 2, 300]), (16, 1, 16, 128, [70, 16, 5])])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_attention_masked_infinities_and_nans(H, KVH, T, D, lens, value):
    """A newest token with an infinite or NaN element (cached as a NaN run) reaches no query before it; the last query sees it."""
    c = Case(lens, H=H, KVH=KVH, T=T, D=D, dtype=BF16, seed=T + D)
    clean = c.run()
    last = torch.tensor([n - 1 for n in lens])
    k, v = (torch.randn(len(lens), KVH, D, generator=torch.Generator().manual_seed(1)) for _ in range(2))
    v[:, :, 5] = value
    paged_int4_append(c.kv, None, k.bfloat16().to(DEV), v.bfloat16().to(DEV), last.to(DEV), c.table.to(DEV))
    got = c.run()
    assert torch.equal(got[:, :-1], clean[:, :-1])
    assert torch.isnan(got[:, -1, :, :64]).all() and torch.isfinite(got[:, -1, :, 64:]).all()
    k[:, :, 5] = value
    paged_int4_append(c.kv, None, k.bfloat16().to(DEV), v.bfloat16().to(DEV), last.to(DEV), c.table.to(DEV))
    got = c.run()
    assert torch.equal(got[:, :-1], clean[:, :-1]) and torch.isnan(got[:, -1]).all()


def test_attention_nonfinite_queries_stay_alone():
    c = Case([200, 90], T=3, dtype=BF16, seed=9)
    clean = c.run()
    c.q[0, 1, 3, 7], c.q[1, 0, 0, 0] = NAN, INF
    got = c.run()
    assert torch.isnan(got[0, 1, 3]).all() and torch.isnan(got[1, 0, 0]).all()
    got[0, 1, 3], got[1, 0, 0] = clean[0, 1, 3], clean[1, 0, 0]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("lens,H,T", [([200, 90, 5], 8, 1), ([5000, 1700, 33], 8, 1), ([900, 4000], 16, 8), ([120, 30], 16, 8)])
def test_attention_in_place(lens, H, T):
    """The queries' memory as the output: units whole, cut over blocks, and of several row tiles."""
    c = Case(lens, H=H, KVH=2, T=T, dtype=BF16, seed=H + T)
    want = c.run()
    q = c.q.to(DEV)
    for max_len in (0, max(lens)):
        mine = q.clone()
        got = paged_int4_attention(c.kv, mine, c.table.to(DEV), c.lens.to(DEV), max_len=max_len, out=mine)
        clean = paged_int4_attention(c.kv, q, c.table.to(DEV), c.lens.to(DEV), max_len=max_len)
        assert got.data_ptr() == mine.data_ptr() and torch.equal(mine, clean)
    assert torch.isfinite(want).all()


def test_attention_workspaces_graphs_and_streams():
    """Two captured graphs and an eager call, each with scratch of its own, on several streams at once; the launch flag."""
    a, b = Case([9000, 1700, 900], seed=1), Case([800, 9500], T=4, H=16, seed=2)     # parts that meet in scratch
    want = [c.run() for c in (a, b)]
    args = [(c.kv, c.q.to(DEV), c.table.to(DEV), c.lens.to(DEV)) for c in (a, b)]
    outs, graphs = [torch.zeros_like(w) for w in want], []
    for x, out in zip(args, outs):
        ws = paged_int4_attention_workspace(*x[:3])
        ws.fill_(255)                   # no initial contents are needed
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_int4_attention(*x, out=out, workspace=ws)
        graphs.append((graph, ws))
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = paged_int4_attention(*args[0], flags=_lib.LAUNCH_PDL)
            eager = paged_int4_attention(*args[0], flags=_lib.LAUNCH_PDL)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
    short = paged_int4_attention_workspace(*args[0][:3])[:-4]
    assert short.numel() > 0
    with pytest.raises(_lib.B2DError, match="workspace"):
        paged_int4_attention(*args[0], workspace=short)


def test_attention_refused_for_its_workspace_writes_nothing():
    """300 sequences, two launches: the first runs its units whole, the second needs scratch. Without enough of it the call is refused
    before the first, with the queries as the output too."""
    lens = [300 + i % 200 for i in range(300)]
    c = Case(lens, H=4, KVH=2, D=64, ps=32, seed=13, dtype=BF16)
    table, lens = c.table.to(DEV)[:, :16].contiguous(), c.lens.to(DEV)
    q = c.q.to(DEV)
    need = paged_int4_attention_workspace(c.kv, q, table, max_len=512)
    assert need.numel() > 0 and paged_int4_attention_workspace(c.kv, q[:256], table[:256], max_len=512).numel() == 0
    for ws in (need[:0], need[:-16]):
        mine, apart = q.clone(), torch.full_like(q, 7.0)
        for out in (mine, apart):
            with pytest.raises(_lib.B2DError, match="workspace"):
                paged_int4_attention(c.kv, mine, table, lens, max_len=512, out=out, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(mine, q) and (apart == 7).all()
    got = paged_int4_attention(c.kv, mine, table, lens, max_len=512, out=mine, workspace=need)
    c.check(got)
    c.check(paged_int4_attention(c.kv, q, table, lens))


def test_programmatic_launches_see_what_the_kernel_before_wrote():
    """Chains of dependent launches: a read writes what an append takes, whose keys and queries an attention takes."""
    a = Case([700, 900, 333], H=8, KVH=2, dtype=BF16, seed=21)
    pos, seq, table, lens = a.pos.to(DEV), a.seq.to(DEV), a.table.to(DEV), a.lens.to(DEV)
    N, w = pos.numel(), torch.rand(128, device=DEV).bfloat16()
    cos, sin = (t.to(DEV) for t in rotary_tables(1000, 128))
    k, v, q = (torch.zeros(N, h, 128, dtype=BF16, device=DEV) for h in (2, 2, 8))
    last = (lens.cumsum(0) - 1).long()

    def chain(flags):
        kv = empty_pool(a.kv.num_pages, 2, a.ps, 128, BF16)
        out = []
        for _ in range(8):
            k.zero_(), v.zero_(), q.zero_()
            paged_int4_read(a.kv, pos, table, seq_ids=seq, k_out=k, v_out=v, flags=flags)
            q.copy_(k.repeat_interleave(4, 1))
            q_rot = paged_int4_append(kv, q, k, v, pos, table, cos, sin,
                                      q_weight=w, k_weight=w, seq_ids=seq, flags=flags)
            paged_int4_read(a.kv, pos, table, seq_ids=seq, k_out=k, v_out=v, flags=flags)
            paged_int4_append(kv, None, k, v, pos, table, cos, sin, seq_ids=seq, flags=flags)
            out.append(paged_int4_attention(kv, q_rot[last][:, None], table, lens, flags=flags))
        return out

    plain, early = chain(0), chain(_lib.LAUNCH_PDL)
    assert all(torch.equal(x, y) for x, y in zip(plain, early)) and torch.isfinite(plain[0]).all()


def test_programmatic_read_append_read_of_one_pool():
    """Each read sees the append before it, all of them dependent launches on the same positions: no kernel between them."""
    N, KVH, D, ps = 4096, 4, 128, 16
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(N // ps, generator=g).int().view(4, -1).to(DEV)
    pos = torch.arange(N // 4).repeat(4).to(DEV)
    rounds = [[torch.randn(N, KVH, D, generator=g).half().to(DEV) for _ in range(2)] for _ in range(6)]

    def chain(flags):
        kv = PagedKVInt4.empty(N // ps, KVH, ps, D, F16, DEV)
        outs = [[torch.empty(N, KVH, D, dtype=F16, device=DEV) for _ in range(2)] for _ in rounds]
        torch.cuda.synchronize()
        for (k, v), (ko, vo) in zip(rounds, outs):
            paged_int4_read(kv, pos, table, k_out=ko, v_out=vo, flags=flags)      # the round's before
            paged_int4_append(kv, None, k, v, pos, table, flags=flags)
            paged_int4_read(kv, pos, table, k_out=ko, v_out=vo, flags=flags)
        return outs

    for plain, early in zip(chain(0), chain(_lib.LAUNCH_PDL)):
        assert all(torch.equal(x, y) for x, y in zip(plain, early))
    for (k, _), (ko, _) in zip(rounds, chain(_lib.LAUNCH_PDL)):
        step = (k.unflatten(-1, (-1, 64)).float().amax(-1) - k.unflatten(-1, (-1, 64)).float().amin(-1)).max() / 15
        assert (ko.float() - k.float()).abs().max() <= 0.51 * step


@pytest.mark.parametrize("T,base", [(1, 900), (4, 300), (3, 2500)])
def test_programmatic_serving_steps(T, base):
    """Plan, append, attention, plan, ... as dependent launches with no other kernel among them: the attention's queries are the append's
    output as it lies, its lengths and tables the plan's, and the next plan takes and gives back pages that the attention has read."""
    B, H, KVH, D, ps, W = 24, 8, 2, 128, 16, 200
    g = torch.Generator().manual_seed(T)
    cos, sin = (t.to(DEV) for t in rotary_tables(W * ps, D))
    start = torch.randint(base // 2, base, (B,), generator=g).int()
    steps = []
    for i in range(8):   # grow by T, and by turns fall back by some pages
        cached = (start + T * i if i % 3 else (start * 0.7).int()).to(DEV)
        q, k, v = (torch.randn(B * T, h, D, generator=g).half().to(DEV) for h in (H, KVH, KVH))
        steps.append((cached, q, k, v))
    new = torch.full((B,), T, dtype=torch.int32, device=DEV)
    fill = [torch.randn(B * W * ps, KVH, D, generator=g).half().to(DEV) for _ in range(2)]

    def chain(flags):
        tables = PageTables.empty(B * W, ps, B, W, DEV)
        kv = PagedKVInt4.empty(B * W, KVH, ps, D, F16, DEV)
        every = torch.arange(B * W, dtype=torch.int32, device=DEV).view(B, W)
        paged_int4_append(kv, None, *fill, torch.arange(W * ps, device=DEV).repeat(B), every)   # (every page holds something)
        plans = [StepPlan.empty(B, B * T, DEV) for _ in steps]
        q_rots, outs = ([torch.empty(B * T, H, D, dtype=F16, device=DEV) for _ in steps] for _ in range(2))
        ws = paged_int4_attention_workspace(kv, outs[0].view(B, T, H, D), tables.page_table)
        torch.cuda.synchronize()
        for (cached, q, k, v), plan, q_rot, out in zip(steps, plans, q_rots, outs):
            tables.step(cached, new, out=plan, flags=flags)
            paged_int4_append(kv, q, k, v, plan.positions, tables.page_table, cos, sin, seq_ids=plan.seq_ids, q_out=q_rot, flags=flags)
            paged_int4_attention(kv, q_rot.view(B, T, H, D), tables.page_table, plan.seqlens, out=out.view(B, T, H, D),
                                 workspace=ws, flags=flags)
        return [*outs, *q_rots, *(t for p in plans for t in p), tables.page_table, tables.held, tables.free, tables.ring, kv.pages]

    plain, early = chain(0), chain(_lib.LAUNCH_PDL)
    assert all(torch.equal(x, y) for x, y in zip(plain, early)) and all(torch.isfinite(x).all() and x.any() for x in plain[:16])
    graph_pool = []   # and as one graph of dependent launches
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        kv = PagedKVInt4.empty(B * W, KVH, ps, D, F16, DEV)
        tables = PageTables(torch.full((B, W), -1, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV),
                            torch.arange(B * W, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), ps)
        tables.ring[1:].fill_(B * W)
        every = torch.arange(B * W, dtype=torch.int32, device=DEV).view(B, W)
        paged_int4_append(kv, None, *fill, torch.arange(W * ps, device=DEV).repeat(B), every)
        for cached, q, k, v in steps:
            plan = tables.step(cached, new, B * T, flags=_lib.LAUNCH_PDL)
            q_rot = paged_int4_append(kv, q, k, v, plan.positions, tables.page_table, cos, sin, seq_ids=plan.seq_ids, flags=_lib.LAUNCH_PDL)
            graph_pool.append(paged_int4_attention(kv, q_rot.view(B, T, H, D), tables.page_table, plan.seqlens, flags=_lib.LAUNCH_PDL).view(B * T, H, D))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(plain, graph_pool))


def test_pool_past_four_gigabytes():
    """Pages further apart than 32 bits of bytes."""
    D, ps, KVH = 128, 16, 2
    block = PagedKVInt4.page_bytes(ps, D)
    stride = 1_500_000_000 // 16 * 16
    memory = torch.empty(3 * stride + KVH * block, dtype=torch.uint8, device=DEV)
    far = PagedKVInt4(memory.as_strided((4, KVH, block), (stride, block, 1)), ps, D, F16)
    near = empty_pool(4, KVH, ps, D, F16)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(60, KVH, D, generator=g).half().to(DEV) for _ in range(2))
    q = torch.randn(1, 1, 8, D, generator=g).half().to(DEV)
    table = torch.tensor([[3, 1, 2, 0]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([60], dtype=torch.int32, device=DEV)
    out = []
    for kv in (far, near):
        paged_int4_append(kv, None, k, v, torch.arange(60, device=DEV), table)
        out.append((*paged_int4_read(kv, torch.arange(60, device=DEV), table), paged_int4_attention(kv, q, table, lens)))
    assert all(torch.equal(x, y) for x, y in zip(*out)) and torch.isfinite(out[0][2]).all()


@pytest.mark.parametrize("D,dtype,out_dtype", [(64, F16, F16), (128, BF16, BF16), (128, F16, F32), (64, BF16, F32)])
def test_read_into_rows_of_any_allowed_alignment(D, dtype, out_dtype):
    """Outputs that begin, or whose rows lie, at multiples of 16 bytes but not of 32, whole tiles and single tokens; what lies
    beside them stays."""
    c = Case([40, 21], KVH=3, H=3, D=D, dtype=dtype, seed=D)
    N, item = c.pos.numel(), 8                               # rows apart by multiples of 8 elements
    want = paged_int4_read(c.kv, c.pos.to(DEV), c.table.to(DEV), seq_ids=c.seq.to(DEV), out_dtype=out_dtype)
    shuffle = torch.randperm(N, generator=torch.Generator().manual_seed(1))
    for order in (torch.arange(N), shuffle):
        for start, pad in ((0, 0), (4 if out_dtype == F32 else 8, 0), (0, item), (item, item)):
            row = 3 * D + pad
            memory = torch.full((2, N * row + 64), 7.0, dtype=out_dtype, device=DEV)
            k, v = (m[start:start + N * row].view(N, row)[:, :3 * D].view(N, 3, D) for m in memory)
            paged_int4_read(c.kv, c.pos[order].to(DEV), c.table.to(DEV), seq_ids=c.seq[order].to(DEV), k_out=k, v_out=v)
            assert torch.equal(k, want[0][order.to(DEV)]) and torch.equal(v, want[1][order.to(DEV)])
            k.fill_(7), v.fill_(7)
            assert (memory == 7).all()


# ------------------------------------------------------------------ page planning
STATE = ("page_table", "held", "free", "ring")


def check_step(tables, cached, new, N, **kw):
    before = [getattr(tables, n).cpu().numpy() for n in STATE]
    want = plan_ref(*before, cached.tolist(), new.tolist(), tables.page_size, N)
    plan = tables.step(cached.to(DEV), new.to(DEV), N, **kw)
    for name in StepPlan._fields:
        assert np.array_equal(getattr(plan, name).cpu().numpy(), want[name]), name
    for name in STATE:
        assert np.array_equal(getattr(tables, name).cpu().numpy(), want[name]), name
    return plan


@pytest.mark.parametrize("B,W,ps,P,most", [(1, 1, 16, 1, 20), (1, 9, 16, 9, 200), (7, 5, 1, 30, 4), (40, 8, 16, 200, 60), (256, 33, 32, 2000, 300),
                                           (257, 6, 5, 900, 9), (1024, 20, 16, 9000, 90), (1500, 3, 64, 4000, 100), (8192, 4, 16, 20000, 9)])
def test_plan_over_many_steps(B, W, ps, P, most):
    """Requests that grow, shrink, end and are refused, over steps that turn the ring round."""
    g = torch.Generator().manual_seed(B + P)
    tables = PageTables.empty(P, ps, B, W, DEV)
    cached = torch.zeros(B, dtype=torch.int32)
    for step in range(8):
        new = torch.randint(0, most + 1, (B,), generator=g, dtype=torch.int32)
        new[torch.rand(B, generator=g) < 0.2] = 0
        N = [int(new.sum()), B * most, int(new.sum()) * 2 // 3, 1][step % 4]
        plan = check_step(tables, cached, new, N)
        granted = plan.granted.cpu()
        cached = cached + granted.clamp(min=0)
        back = torch.rand(B, generator=g)
        cached = torch.where(back < 0.3, (cached * 0.4).int(), cached)
        cached = torch.where(back > 0.85, 0, cached)
        table, held, free, ring = (getattr(tables, n).cpu() for n in STATE)
        pages = [p for b in range(B) for p in table[b, :held[b]].tolist()] + [int(free[(ring[0] + i) % P]) for i in range(int(ring[1]))]
        assert sorted(pages) == list(range(P))       # every page is held once or free


@pytest.mark.parametrize("B,tokens", [(256, 1024), (257, 1024), (512, 1024), (512, 1025), (513, 1024), (513, 1)])
def test_plan_on_both_sides_of_its_launch_rules(B, tokens):
    """One block or a cluster, 256 threads or 512, with pages that come and go for nearly every sequence."""
    g = torch.Generator().manual_seed(B)
    tables = PageTables.empty(3 * B, 4, B, 6, DEV)
    cached = torch.zeros(B, dtype=torch.int32)
    for _ in range(4):
        cached = (cached + check_step(tables, cached, torch.randint(0, 6, (B,), generator=g, dtype=torch.int32), tokens).granted.cpu().clamp(min=0))
        cached = torch.where(torch.rand(B, generator=g) < 0.4, cached // 3, cached)
        check_step(tables, cached, torch.zeros(B, dtype=torch.int32), 0)


def test_plan_edges():
    """Negative lengths, tables too narrow, a ring without pages, no tokens, no sequences, lengths whose sum passes 32 bits."""
    tables = PageTables.empty(10, 16, 6, 3, DEV)
    big = 2 ** 31 - 1
    check_step(tables, torch.tensor([-5, 0, 48, 49, big, 16], dtype=torch.int32), torch.tensor([3, -9, 0, 1, big, 0], dtype=torch.int32), 8)
    check_step(tables, torch.tensor([0, 0, 48, 0, 0, 16], dtype=torch.int32), torch.tensor([48, 48, 0, 48, 1, 1], dtype=torch.int32), 200)
    check_step(tables, torch.zeros(6, dtype=torch.int32), torch.zeros(6, dtype=torch.int32), 0)
    check_step(tables, torch.zeros(6, dtype=torch.int32), torch.full((6,), big, dtype=torch.int32), 5)
    none = PageTables.empty(0, 16, 3, 4, DEV)
    check_step(none, torch.zeros(3, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32), 4)
    nobody = PageTables.empty(4, 16, 0, 4, DEV)
    plan = nobody.step(torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), 3)
    assert plan.starts.tolist() == [0] and plan.positions.tolist() == [-1] * 3 and nobody.ring.tolist() == [0, 4]


def test_plan_state_that_counts_pages_twice_stays_inside():
    """A state that holds nonsense: ids anywhere, counts too large. Nothing outside the arrays is written."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    memory = torch.full((4, 8), 77, dtype=torch.int32, device=DEV)
    guard = torch.full((9,), 55, dtype=torch.int32, device=DEV)
    tables = PageTables(memory[:, :5], i32([99, -4, 3, 5]), guard[:5], i32([-7, 1000]), 16)
    for cached, new in (([0, 0, 0, 0], [0, 80, 1, 0]), ([300, 10, 5, 0], [0, 0, 0, 0]), ([0] * 4, [0] * 4), ([0] * 4, [80] * 4)):
        check_step(tables, torch.tensor(cached, dtype=torch.int32), torch.tensor(new, dtype=torch.int32), 90)
    assert (memory[:, 5:] == 77).all() and (guard[5:] == 55).all()


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("int4", [True, False])
def test_serving_step_in_one_graph(int4):
    """Plan, append, attention and draft verification as one captured graph: requests of different lengths with drafts, one
    that ends, one that cannot have its pages, over steps without the host -- each part against its definition. With
    the 16-bit cache the plan feeds the calls that were there before."""
    B, T, H, KVH, D, ps, V, W, P = 5, 4, 8, 2, 64, 16, 500, 8, 11   # 11 pages: not enough once the third request grows
    K, S = T - 1, 128
    g = torch.Generator().manual_seed(9)
    tables = PageTables.empty(P, ps, B, W, DEV)
    plan = StepPlan.empty(B, B * T, DEV)
    cos, sin = rotary_tables(S, D, 1e4)
    if int4:
        kv = empty_pool(P, KVH, ps, D, F16, 32)
    else:
        kv = PagedKV(*(torch.zeros(P, KVH, ps, D, dtype=F16, device=DEV) for _ in range(2)))
    cd, sd = (x.to(DEV) if int4 else torch.cat((x, x), -1).half().to(DEV) for x in (cos, sin))
    head = (torch.randn(H * D, V, generator=g) * 0.2).half().to(DEV)
    q, k, v = (torch.zeros(B * T, h, D, dtype=F16, device=DEV) for h in (H, KVH, KVH))
    cached, new = torch.zeros(B, dtype=torch.int32, device=DEV), torch.full((B,), T, dtype=torch.int32, device=DEV)
    ids, u = torch.zeros(B, K, dtype=torch.int64, device=DEV), torch.zeros(B, T, device=DEV)
    rows = torch.arange(T, device=DEV)

    def step():
        tables.step(cached, new, out=plan)
        if int4:
            q_rot = paged_int4_append(kv, q, k, v, plan.positions, tables.page_table, cd, sd, seq_ids=plan.seq_ids)
        else:
            q_rot = paged_rope_append(kv, q, k, v, plan.positions, tables.page_table, cd, sd, seq_ids=plan.seq_ids)
        # a sequence's rows as [B, T]: those of a sequence without tokens are anything
        own = (plan.starts[:-1, None] + rows).clamp(max=B * T - 1).long()
        lens = torch.where(plan.granted > 0, plan.seqlens, 0)
        qs = q_rot[own.view(-1)].view(B, T, H, D)
        out = (paged_int4_attention if int4 else paged_attention)(kv, qs, tables.page_table, lens)
        probs = torch.softmax((out.view(B, T, H * D) @ head).float(), -1)
        tok, acc = verify_drafts(ids, probs, u)
        return q_rot, qs, lens, out, probs, tok, acc

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    # back to the start: the warm-up's pages go home
    tables.step(torch.zeros_like(cached), torch.zeros_like(new), 0)
    seen_refusal = False
    held_k, held_v = {}, {}
    for i in range(7):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        ids.copy_(torch.randint(0, V, (B, K), generator=g))
        u.copy_(torch.rand(B, T, generator=g) * 0.01)
        new.fill_(T)
        if i == 0:
            cached.copy_(torch.tensor([0, 30, 60, 17, 5]))   # (nothing of these is cached: NaN or zero slots, set below)
        if i == 4:
            cached[2], new[2] = 0, 0                          # ends
        before = [getattr(tables, n).cpu().numpy() for n in STATE]
        c0, n0 = cached.cpu(), new.cpu()
        if i == 0:   # start from requests that are cached in earnest
            fill = StepPlan.empty(B, 200, DEV)
            tables.step(torch.zeros_like(cached), cached, out=fill)
            n = int(fill.starts[-1])
            fk, fv = (torch.randn(200, KVH, D, generator=g).half().to(DEV) for _ in range(2))
            if int4:
                paged_int4_append(kv, None, fk, fv, fill.positions, tables.page_table, seq_ids=fill.seq_ids)
            else:
                one, zero = torch.ones(S, D, device=DEV), torch.zeros(S, D, device=DEV)
                paged_rope_append(kv, torch.zeros(200, KVH, D, dtype=F16, device=DEV), fk, fv, fill.positions, tables.page_table, one, zero, seq_ids=fill.seq_ids)
            for j in range(n):
                held_k[int(fill.seq_ids[j]), int(fill.positions[j])] = fk[j].float().cpu().numpy()
                held_v[int(fill.seq_ids[j]), int(fill.positions[j])] = fv[j].float().cpu().numpy()
            before = [getattr(tables, n).cpu().numpy() for n in STATE]
        graph.replay()
        torch.cuda.synchronize()
        want = plan_ref(*before, c0.tolist(), n0.tolist(), ps, B * T)
        for name in StepPlan._fields:
            assert np.array_equal(getattr(plan, name).cpu().numpy(), want[name]), name
        for name in STATE:
            assert np.array_equal(getattr(tables, name).cpu().numpy(), want[name]), name
        q_rot, qs, lens, out, probs, tok, acc = got
        seq, pos, live = want["seq_ids"], want["positions"], int(want["starts"][-1])
        cc, ss = (f64(x)[np.maximum(pos, 0)] for x in ((cos, sin) if int4 else (cos.half(), sin.half())))
        kr = turn_ref(k.float().cpu().numpy(), cc, ss, False, exact32=True)
        for j in range(live):
            held_k[int(seq[j]), int(pos[j])] = kr[j]
            held_v[int(seq[j]), int(pos[j])] = v[j].float().cpu().numpy()
        # attention against the cache as the definition has it
        c = Case.__new__(Case)
        ln = lens.cpu()
        c.seq = torch.cat([torch.full((int(x),), b) for b, x in enumerate(ln)]).int()
        c.pos = torch.cat([torch.arange(int(x)) for x in ln])
        c.k = torch.from_numpy(np.stack([held_k[int(b), int(p)] for b, p in zip(c.seq, c.pos)]))
        c.v = torch.from_numpy(np.stack([held_v[int(b), int(p)] for b, p in zip(c.seq, c.pos)]))
        c.q, c.table, c.lens, c.scale, c.dtype, c.ps, c.group, c.kv = qs.cpu(), torch.from_numpy(want["page_table"]), ln, D ** -0.5, F16, ps, 32, kv
        if int4:
            c.check(out)
        else:   # four half steps: keys, weights, output, and the plain rounding of the queries' products
            kp, vp = (np.zeros((P, KVH, ps, D)) for _ in range(2))
            pages = c.table[c.seq.long(), c.pos // ps].numpy()
            kp[pages, :, (c.pos % ps).numpy()], vp[pages, :, (c.pos % ps).numpy()] = c.k.half().double().numpy(), c.v.double().numpy()
            ref, mass, reach = paged_attention_ref(f64(c.q), kp, vp, c.table.numpy(), ln.numpy(), c.scale)
            bound = half_step(F16) * (1 + 2 * reach[..., None]) * mass + 8 * D * 2.0 ** -23 * reach[..., None] * mass + half_step(F16) * np.abs(ref) + 2.0 ** -16
            assert (np.abs(f64(out) - ref) <= bound).all()
        seen_refusal |= bool((plan.granted == -1).any())
        # accepted drafts and the token behind them stay
        cached.copy_(torch.where(plan.granted > 0, c0.to(DEV) + acc + 1, cached))
    assert seen_refusal


def test_int4_is_near_the_16_bit_cache():
    """The same tokens through both caches: attention differs by what 4 bits lose, at most half a step s / 2 an element on the
    values and scale sum |q| s / 2 on a score."""
    g = torch.Generator().manual_seed(3)
    N, KVH, H, D, ps = 500, 2, 8, 128, 16
    k, v = (torch.randn(N, KVH, D, generator=g).half().to(DEV) for _ in range(2))
    q = torch.randn(1, 1, H, D, generator=g).half().to(DEV)
    table = torch.randperm(32, generator=g).int().view(1, -1).to(DEV)
    pos, lens = torch.arange(N, device=DEV), torch.tensor([N], dtype=torch.int32, device=DEV)
    full = PagedKV(*(torch.zeros(32, KVH, ps, D, dtype=F16, device=DEV) for _ in range(2)))
    one, zero = torch.ones(N, D, device=DEV), torch.zeros(N, D, device=DEV)
    paged_rope_append(full, torch.zeros(N, KVH, D, dtype=F16, device=DEV), k, v, pos, table, one, zero)
    kv = empty_pool(32, KVH, ps, D, F16, 32)
    paged_int4_append(kv, None, k, v, pos, table)
    a, b = paged_attention(full, q, table, lens, out_dtype=F32), paged_int4_attention(kv, q, table, lens, out_dtype=F32)
    ks, vs = (quantise_ref(x.float().cpu().numpy(), 32, F16)[1].max() for x in (k, v))
    ds = 0.51 * ks * float(q.float().abs().sum(-1).max()) * D ** -0.5      # 0.51: the scale's own rounding
    assert (a - b).abs().max().item() <= 0.51 * vs + (np.exp(2 * ds) - 1) * float(v.float().abs().max())
