"""GPU: paged append and paged attention against their float64 definitions (``oracle/paged_ref.py``).

Bounds (element by element, from the arithmetic; h = eps / 2 of a dtype is half a step, 2^-8 for bf16, 2^-11
for fp16):

* append: fp32 between load and store. The norm's mean, reciprocal root and two products, the rotation's two
  products and sum are each off by at most 2^-23 of the terms' size, under 2^-19 in all; then one rounding of the
  result, or half a step of the subnormals (2^-25, fp16).
* attention: a weight p_j is off by h (its rounding before the second product), and by 2 D 2^-23 reach
  (fp32 accumulation of D products, doubled for the running maximum), reach = max scale sum |q_d k_jd|, twice since
  the normalising sum has it too; the second product's accumulation over n keys by n 2^-23; fp16 weights below 2^-14
  by 2^-25 each, against a sum of at least 1. All of these times mass = sum p_j |v_j| (the last one times n max|v|),
  then the output's own rounding.
"""
import numpy as np
import pytest
import torch

from b200kernels import _lib
from b200kernels.decode_attention import decode_attention
from b200kernels.glue import rope_kv_append
from b200kernels.paged import PagedKV, paged_attention, paged_attention_workspace, paged_rope_append
from b200kernels.speculative import verify_drafts
from oracle.paged_ref import paged_attention_ref, rope_ref, verify_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------------ attention
class Case:
    """Random pools whose unused slots hold NaN and whose unused table entries point nowhere."""

    def __init__(self, lens, H=8, KVH=2, D=128, T=1, ps=16, prefix=0, dtype=F16, seed=0, layout="hnd", spare=3, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        B, self.prefix, self.ps = len(lens), prefix, ps
        per = max(1, -(-max(max(lens), 1) // ps) + 1)
        need = [-(-n // ps) for n in lens]
        npre = -(-prefix // ps)
        total = sum(need) + npre + spare
        perm = torch.randperm(total, generator=g).int()
        self.table = torch.full((B, per), -1, dtype=torch.int32)
        self.prefix_table = perm[:npre].clone() if prefix else None
        k = torch.full((total, KVH, ps, D), NAN)
        v = torch.full((total, KVH, ps, D), NAN)
        at = npre
        fill = lambda *s: magnitude * torch.randn(*s, generator=g)
        for i in range(npre):   # the prefix's pages, filled up to its end only
            n = min(ps, prefix - i * ps)
            k[perm[i], :, :n], v[perm[i], :, :n] = fill(KVH, n, D), fill(KVH, n, D)
        for b, n in enumerate(lens):
            for i in range(need[b]):
                if (i + 1) * ps <= prefix:
                    continue   # a page that only the prefix covers: not in the sequence's own row
                self.table[b, i] = perm[at]
                m = min(ps, n - i * ps)
                k[perm[at], :, :m], v[perm[at], :, :m] = fill(KVH, m, D), fill(KVH, m, D)
                if i * ps < prefix:   # the slots of the prefix in a page that it shares with the sequence
                    k[perm[at], :, :prefix - i * ps] = NAN
                    v[perm[at], :, :prefix - i * ps] = NAN
                at += 1
        self.k, self.v = k.to(dtype), v.to(dtype)
        self.q = magnitude * torch.randn(B, T, H, D, generator=g).to(dtype)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.scale, self.dtype = D ** -0.5, dtype
        if layout == "nhd":
            self.kd, self.vd = (x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for x in (self.k, self.v))
        else:
            self.kd, self.vd = self.k.to(DEV), self.v.to(DEV)
        self.cache = PagedKV(self.kd, self.vd)

    def run(self, **kw):
        if self.prefix:
            kw.update(prefix_table=self.prefix_table.to(DEV), prefix_len=self.prefix)
        return paged_attention(self.cache, self.q.to(DEV), self.table.to(DEV), self.lens.to(DEV), **kw)

    def check(self, out):
        D = self.q.shape[-1]
        k, v = np.nan_to_num(f64(self.k)), np.nan_to_num(f64(self.v))
        ref, mass, reach = paged_attention_ref(f64(self.q), k, v, self.table.numpy(), self.lens.numpy(), self.scale,
                                               None if self.prefix_table is None else self.prefix_table.numpy(), self.prefix)
        n = max(1, int(self.lens.max()))
        h = half_step(self.dtype)
        bound = (h + 4 * 2 * D * 2.0 ** -23 * reach[..., None] + n * 2.0 ** -23) * mass
        if self.dtype == F16:
            bound = bound + n * 2.0 ** -25 * np.abs(v).max()
        bound = bound + half_step(out.dtype) * (np.abs(ref) + bound) + 2.0 ** -25
        got = f64(out)
        assert np.isfinite(got).all()
        err = np.abs(got - ref)
        assert (err <= bound).all(), f"worst error / bound {(err / bound).max():.2f}, error {err.max():.3e}"
        for b, n_b in enumerate(self.lens.tolist()):   # queries that see nothing give zeros
            for t in range(self.q.shape[1]):
                if n_b - self.q.shape[1] + 1 + t <= 0:
                    assert (got[b, t] == 0).all()


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [128, 1, 0, 127], [300, 517, 16, 15, 17]])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_lengths(lens, D):
    c = Case(lens, D=D, seed=len(lens) + D)
    c.check(c.run())


@pytest.mark.parametrize("ps", [1, 5, 16, 48, 64, 256, 1000])
def test_attention_page_sizes(ps):
    c = Case([1, 257, 100, 0, 64], ps=ps, seed=ps)
    c.check(c.run())
    c = Case([400, 277, 320, 0, 301], ps=ps, prefix=261, T=2, seed=ps)
    c.check(c.run())


@pytest.mark.parametrize("H,KVH,T", [(1, 1, 1), (8, 8, 1), (14, 2, 1), (16, 1, 1), (8, 2, 2), (8, 2, 3), (7, 1, 5),
                                     (32, 8, 5), (16, 1, 4), (15, 1, 4), (16, 1, 16), (6, 2, 16), (12, 1, 11)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_heads_and_drafts(H, KVH, T, dtype):
    lens = [T + 130, 0, 1, T, max(0, T - 1), T + 63]   # shorter than the drafts, too: their first queries see nothing
    c = Case(lens, H=H, KVH=KVH, T=T, dtype=dtype, seed=H + T)
    c.check(c.run())


@pytest.mark.parametrize("B,T,H,KVH,prefix,ps", [
    (3, 1, 8, 2, 16, 16), (3, 1, 8, 2, 1, 16), (5, 1, 8, 2, 130, 16), (20, 1, 8, 2, 257, 16), (20, 4, 8, 2, 512, 64),
    (9, 8, 8, 1, 300, 32), (40, 1, 16, 1, 700, 128), (70, 1, 4, 2, 333, 16), (33, 2, 16, 2, 1024, 256)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_shared_prefix(B, T, H, KVH, prefix, ps, dtype):
    g = torch.Generator().manual_seed(B)
    lens = (prefix + torch.randint(T, 90, (B,), generator=g)).tolist()
    lens[0] = 0                        # a padded row of the batch
    lens[1] = prefix + T               # only the new tokens behind the prefix
    lens[2] = max(prefix - 3, 0)       # ends inside the prefix
    c = Case(lens, H=H, KVH=KVH, T=T, prefix=prefix, ps=ps, dtype=dtype, seed=prefix)
    c.check(c.run())
    c.check(c.run(out_dtype=F32))


@pytest.mark.parametrize("B,T,H,KVH,D,prefix,ps,extra", [
    (12, 1, 6, 2, 128, 64, 16, 40),      # 36 rows: one step of 64 keys would do, the streaming kernel takes it
    (12, 1, 6, 2, 128, 128, 8, 40), (12, 1, 6, 2, 128, 192, 64, 40), (30, 1, 8, 2, 64, 320, 32, 70),
    (16, 2, 8, 2, 128, 2048, 16, 33),    # 128 rows, several splits, a table of small pages
    (17, 2, 4, 1, 64, 1984, 16, 33),     # 136 rows: the second row tile almost empty
    (16, 4, 12, 2, 128, 960, 192, 90),   # 384 rows: a second pair of row tiles; pages of three boxes
    (65, 2, 4, 1, 128, 4160, 64, 20)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_prefix_on_tensor_cores(B, T, H, KVH, D, prefix, ps, extra, dtype):
    g = torch.Generator().manual_seed(B + prefix)
    lens = (prefix + torch.randint(T, extra, (B,), generator=g)).tolist()
    lens[2], lens[3] = 0, prefix // 2
    c = Case(lens, H=H, KVH=KVH, T=T, D=D, prefix=prefix, ps=ps, dtype=dtype, seed=B)
    c.check(c.run())
    c.scale = -c.scale                   # a negative scale
    c.check(c.run(scale=c.scale))


def test_attention_prefix_rising_scores():
    """Scores that grow along the prefix: the running maximum moves again and again."""
    c = Case([1300 + i for i in range(20)], H=8, KVH=2, T=2, D=64, prefix=1280, ps=64, dtype=BF16, seed=50)
    direction = torch.randn(64, generator=torch.Generator().manual_seed(1)).sign()
    c.q = (c.q.float() * 0.2 + direction).bfloat16()
    for i, page in enumerate(c.prefix_table.tolist()):
        c.k[page] = (c.k[page].float() * 0.2 + direction * (0.3 * i)).bfloat16()
    c.kd.copy_(c.k)
    c.check(c.run())


@pytest.mark.parametrize("hidden", [[0, 1, 2, 3, 8, 9, 10, 11], list(range(8)), list(range(16))])
@pytest.mark.parametrize("scale", [1.0, -1.0])
def test_attention_prefix_keys_without_weight_first(hidden, scale):
    """Pages of the prefix whose scores are all -infinity -- the first step of each warpgroup, a warpgroup's whole
    part, a split's -- ahead of keys with scores far below zero: as if they were not there."""
    c = Case([530 + 3 * i for i in range(12)], H=8, KVH=2, D=128, prefix=512, ps=16, dtype=BF16, seed=70)
    c.scale *= scale
    c.q = c.q.abs()
    c.k.copy_((0.2 * c.k.float() - 20 * scale).to(BF16))      # scores of about -180
    gone = c.prefix_table[hidden].long()
    c.k[gone, :, :, 0] = -float("inf") * scale
    c.kd.copy_(c.k)
    out = c.run(scale=c.scale)
    n = 16 * len(hidden)
    keep = [i for i in range(32) if i not in hidden]
    c.prefix_table, c.prefix, c.lens, c.table = c.prefix_table[keep], 512 - n, c.lens - n, c.table[:, len(hidden):]
    c.check(out)
    assert (out != 0).any(-1).all()


def test_attention_prefix_heads_of_64():
    c = Case([600 + 7 * i for i in range(24)], H=12, KVH=2, D=64, T=3, prefix=576, ps=32, dtype=BF16, seed=3)
    c.check(c.run())


def test_attention_long_ragged():
    c = Case([5000, 1, 2777, 4096], H=8, KVH=2, seed=8)
    c.check(c.run())
    c.check(c.run(max_len=5000))
    c.check(c.run(max_len=1))          # a wrong hint costs time only


@pytest.mark.parametrize("lens,H,KVH,T,D,prefix,ps", [
    ([5000, 1, 2777, 4096, 0, 63, 64, 65, 129], 8, 2, 1, 128, 0, 16),      # shares of a ragged batch
    ([3001, 517, 2, 128, 1500], 12, 2, 3, 64, 0, 64), ([700, 1300], 16, 1, 4, 128, 0, 32),
    ([9001], 1, 1, 1, 128, 0, 16), ([8200], 4, 1, 1, 64, 0, 64),           # a unit in many parts
    ([260, 77, 1001], 8, 2, 2, 128, 0, 5),                                 # pages that tensor copies do not fit
    ([1100, 1000, 1001, 400, 1530], 8, 2, 1, 128, 1000, 8),                # a prefix on the streaming kernel
    ([3000 + 37 * i for i in range(9)], 4, 4, 1, 64, 2944, 64),
    ([2100 + 19 * i for i in range(20)], 8, 2, 2, 128, 2048, 16),          # and on the tensor cores
    ([2000 + 7 * i for i in range(17)], 4, 1, 2, 64, 1984, 16), ([330 + i for i in range(40)], 8, 2, 4, 128, 320, 32)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_counts_every_key_once(lens, H, KVH, T, D, prefix, ps, dtype):
    """Queries of zeros weigh all keys alike, and values that mark a key's position modulo D / 2 and its run of 64 then
    give counts over the number of keys: a key that is lost or taken twice at a border of stages, shares or splits
    changes a count by a whole. Weights are 1 (2^0 is exact) and all sums whole numbers below 2^24, so five roundings are
    left at most: the reciprocal of the sum, the product with it, and the sum of four warps' quotients; 5 x 2^-24."""
    c = Case(lens, H=H, KVH=KVH, T=T, D=D, ps=ps, prefix=prefix, dtype=dtype, seed=D + ps)
    half = D // 2
    mark = lambda pos: torch.cat([torch.nn.functional.one_hot(pos % half, half), torch.nn.functional.one_hot(pos // 64 % half, half)], -1).to(dtype)
    top = -(-max(max(lens), prefix) // ps) * ps
    marks = mark(torch.arange(top)).view(-1, 1, ps, D)   # [page, 1, slot, D]
    if prefix:
        c.v[c.prefix_table.long()] = torch.where(c.v[c.prefix_table.long()].isnan(), NAN, marks[:c.prefix_table.numel()])
    for b in range(len(lens)):
        at = (c.table[b] >= 0).nonzero()[:, 0]
        pages = c.table[b, at].long()
        c.v[pages] = torch.where(c.v[pages].isnan(), NAN, marks[at])
    c.vd.copy_(c.v)
    c.q.zero_()
    got = f64(c.run(out_dtype=F32))
    running = np.cumsum(f64(mark(torch.arange(top))), 0)
    for b, n_b in enumerate(lens):
        for t in range(T):
            n = n_b - T + 1 + t
            want = running[n - 1] / n if n > 0 else np.zeros(D)
            assert (np.abs(got[b, t] - want) <= 5 * 2.0 ** -24 * want).all(), (b, t, np.abs(got[b, t] - want).max() * max(n, 1))


def test_attention_large_scores():
    """Scores of several hundred: the running maximum matters, one key takes nearly all the weight."""
    for dtype in (F16, BF16):
        c = Case([400, 129], T=2, prefix=64, magnitude=6.0, dtype=dtype, seed=4)
        c.check(c.run())


def test_attention_layouts_and_strides():
    c = Case([100, 33, 257], layout="nhd", dtype=BF16, T=2, seed=5)
    assert c.kd.stride(2) > c.kd.stride(1)
    ref = c.run()
    c.check(ref)
    B, T, H, D = c.q.shape
    wide = torch.full((B, T, H + 4, D), NAN, dtype=BF16, device=DEV)     # q as part of a fused projection
    wide[:, :, :H] = c.q.to(DEV)
    table = torch.full((B, c.table.shape[1] + 5), 10 ** 9, dtype=torch.int32, device=DEV)
    table[:, :c.table.shape[1]] = c.table.to(DEV)
    outw = torch.full((T, B, H + 2, D), 7.0, dtype=BF16, device=DEV)
    out = outw.transpose(0, 1)[:, :, 1:H + 1]
    got = paged_attention(c.cache, wide[:, :, :H], table[:, :c.table.shape[1]], c.lens.to(DEV), out=out)
    assert got is out and torch.equal(out, ref)
    assert (outw[:, :, 0] == 7).all() and (outw[:, :, -1] == 7).all()


def test_attention_lengths_beyond_the_table_and_bad_pages():
    """seqlens past the table's reach are cut to it; a page id outside the pool is not followed (its keys and
    values count as zeros)."""
    c = Case([64, 48], ps=16, seed=6)
    c.table = c.table[:, :3].contiguous()
    ref_lens = c.lens.clamp(max=48)
    c.lens = torch.tensor([64, 2 ** 31 - 1], dtype=torch.int32)
    out = c.run()
    c.lens = ref_lens
    c.check(out)
    c.table[0, 1], c.table[1, 0] = 10 ** 6, -7
    c.check(c.run())


@pytest.mark.parametrize("B,T,H,KVH,D,prefix,ps", [
    (1, 1, 8, 2, 64, 64, 16),            # one sequence: nothing is shared
    (5, 1, 8, 2, 128, 64, 16), (5, 3, 4, 2, 64, 200, 16), (5, 2, 8, 2, 128, 130, 5),     # prefix units, copies by cp.async last
    (20, 1, 8, 2, 128, 256, 16), (20, 3, 8, 2, 64, 448, 64), (5, 16, 8, 1, 128, 192, 32)])   # on the tensor cores
@pytest.mark.parametrize("width", [0, 1, 3])
def test_attention_page_table_narrower_than_the_prefix(B, T, H, KVH, D, prefix, ps, width):
    """A table whose entries end inside the prefix (they are not read there): lengths are cut to the prefix's end,
    never lengthened to it."""
    reach = max(width * ps, prefix)
    lens = [min(width * ps + 4, prefix - 1), prefix - 1, prefix, prefix + T + 40, 0, T, prefix // 2, 2 ** 31 - 1]
    lens = [20] if B == 1 else (lens + [prefix - 1 - i for i in range(B)])[:B]
    c = Case([min(n, reach) for n in lens], H=H, KVH=KVH, D=D, T=T, ps=ps, prefix=prefix, dtype=BF16, seed=B + width)
    cut, c.table = c.lens, c.table[:, :width].contiguous()
    for kw in ({}, {"max_len": prefix}):
        c.lens = torch.tensor(lens, dtype=torch.int32)
        out = c.run(**kw)
        c.lens = cut
        c.check(out)


@pytest.mark.parametrize("H,KVH,T,D,lens", [(8, 2, 4, 128, [130, 64, 7]), (16, 2, 4, 128, [193, 66, 4]),
                                            (16, 1, 4, 64, [129, 260, 5]), (4, 1, 3, 64, [128, 2, 300]),
                                            (16, 1, 16, 128, [70, 16, 5])])
@pytest.mark.parametrize("value", [float("inf"), NAN])
def test_attention_masked_infinities_and_nans(H, KVH, T, D, lens, value):
    """An infinite or NaN key and value of the newest token reaches no query before it, and every later query
    that sees it (a NaN key, an infinite value) is not finite."""
    c = Case(lens, H=H, KVH=KVH, T=T, D=D, dtype=BF16, seed=T + D)
    clean = c.run()
    for b, n in enumerate(lens):
        page = c.table[b, (n - 1) // 16].long().item()
        c.kd[page, :, (n - 1) % 16, ::3] = value
        c.vd[page, :, (n - 1) % 16, 1::2] = value
    got = c.run()
    assert torch.equal(got[:, :-1], clean[:, :-1])
    assert not torch.isfinite(got[:, -1, :, 1::2]).any()


def test_attention_infinite_value_alone():
    """An infinite value among the newest tokens: the queries that see it get it, in its elements only."""
    c = Case([70, 140], H=8, KVH=2, T=3, seed=40)
    clean = c.run()
    for b, n in enumerate([70, 140]):
        c.vd[c.table[b, (n - 2) // 16].long().item(), :, (n - 2) % 16, 5] = -float("inf")
    got = c.run()
    assert torch.equal(got[:, 0], clean[:, 0]) and (got[:, 1:, :, 5] == -float("inf")).all()
    got[:, 1:, :, 5] = clean[:, 1:, :, 5]
    assert torch.allclose(got.float(), clean.float(), rtol=2.0 ** -9, atol=2.0 ** -9)   # summed in another order


def test_attention_empty_calls():
    kv = PagedKV(torch.zeros(2, 2, 16, 64, dtype=F16, device=DEV), torch.zeros(2, 2, 16, 64, dtype=F16, device=DEV))
    t0 = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    assert paged_attention(kv, torch.zeros(0, 1, 4, 64, dtype=F16, device=DEV), t0,
                           torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 1, 4, 64)
    out = paged_attention(kv, torch.ones(2, 1, 4, 64, dtype=F16, device=DEV), torch.zeros(2, 0, dtype=torch.int32, device=DEV),
                          torch.tensor([0, 9], dtype=torch.int32, device=DEV))
    assert (out == 0).all()


def test_attention_offsets_beyond_32_bits():
    """Pages whose element offset passes 2^32 (one pool serves as keys and values)."""
    ps, KVH, D = 64, 8, 128
    pages = (2 ** 32) // (ps * KVH * D) + 3
    pool = torch.empty(pages, KVH, ps, D, dtype=F16, device=DEV)
    kv = PagedKV(pool, pool)
    ids = torch.tensor([pages - 1, 0, pages - 2], dtype=torch.int32, device=DEV)
    pool[ids.long()] = torch.randn(3, KVH, ps, D, device=DEV).half()
    small = PagedKV(pool[ids.long()].contiguous(), pool[ids.long()].contiguous())
    q = torch.randn(1, 2, 32, D, device=DEV).half()
    lens = torch.tensor([150], dtype=torch.int32, device=DEV)
    want = paged_attention(small, q, torch.arange(3, dtype=torch.int32, device=DEV)[None], lens)
    assert torch.equal(paged_attention(kv, q, ids[None], lens), want)
    q2 = torch.randn(1, 2, 32, D, device=DEV).half()
    both = [paged_attention(c, q2.expand(20, 2, 32, D), t[None].expand(20, 3), lens.expand(20).contiguous(), prefix_table=t,
                            prefix_len=128) for c, t in ((small, torch.arange(3, dtype=torch.int32, device=DEV)), (kv, ids))]
    assert torch.equal(both[0], both[1])
    del pool, kv
    torch.cuda.empty_cache()


def test_attention_agrees_with_contiguous_decode():
    """T = 1 over pages of the same keys as the contiguous kernel: both within their bounds of each other."""
    c = Case([512, 100, 2048, 1333], H=32, KVH=8, seed=11)
    S = 2048
    k, v = (torch.zeros(4, 8, S, 128, dtype=F16) for _ in range(2))
    for b, n in enumerate(c.lens.tolist()):
        for p in range(-(-n // 16)):
            m = min(16, n - 16 * p)
            k[b, :, 16 * p:16 * p + m], v[b, :, 16 * p:16 * p + m] = c.k[c.table[b, p], :, :m], c.v[c.table[b, p], :, :m]
    q = c.q.transpose(1, 2).contiguous().to(DEV)
    want = decode_attention(q, k.to(DEV), v.to(DEV), 128 ** -0.5, seqlens=c.lens.to(DEV), out_dtype=F32)
    c.check(want)
    c.check(c.run(out_dtype=F32))


def test_attention_repeats_bitwise_and_on_another_stream():
    c = Case([700 + i for i in range(20)], T=2, prefix=512, seed=12)
    want = c.run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [c.run() for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_attention_two_graphs_replayed_at_once():
    """Two captured graphs (each with the scratch of its own capture) replayed on two streams."""
    cs = [Case([900 + 13 * i + j for i in range(20)], T=2, prefix=512, seed=20 + j) for j in range(2)]
    graphs, outs, want = [], [], []
    for c in cs:
        want.append(c.run())
        q, table, lens, pt = c.q.to(DEV), c.table.to(DEV), c.lens.to(DEV), c.prefix_table.to(DEV)
        c.keep = (q, table, lens, pt)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(c.cache, q, table, lens, prefix_table=pt, prefix_len=512))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(20):
        for o in outs:
            o.fill_(NAN)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    # the graph follows the lengths on the device
    cs[0].keep[2].fill_(700)
    graphs[0].replay()
    torch.cuda.synchronize()
    cs[0].lens.fill_(700)
    cs[0].check(outs[0])


@pytest.mark.parametrize("B,T,prefix", [(300, 1, 0), (300, 1, 128), (261, 3, 192), (257, 1, 64)])
def test_attention_large_batches(B, T, prefix):
    """More sequences than one launch takes."""
    g = torch.Generator().manual_seed(B)
    lens = (prefix + torch.randint(0, 70, (B,), generator=g)).tolist()
    c = Case(lens, H=4, KVH=2, D=64, T=T, prefix=prefix, seed=B, dtype=BF16)
    c.check(c.run())


def test_attention_refused_for_its_workspace_writes_nothing():
    """288 sequences on a prefix, two launches of which the second needs more scratch: without it the call is refused before the first."""
    g = torch.Generator().manual_seed(2)
    c = Case((128 + torch.randint(0, 70, (288,), generator=g)).tolist(), H=1, KVH=1, D=64, prefix=128, ps=64, seed=2, dtype=BF16)
    q, table = c.q.to(DEV), c.table.to(DEV)
    need = paged_attention_workspace(c.cache, q, table, prefix_len=128)
    full = paged_attention_workspace(c.cache, q[:256], table[:256], prefix_len=128).numel()
    assert 0 < full < need.numel()
    out = torch.full_like(q, 7.0)
    for ws in (need[:0], need[:full], need[:-16]):
        with pytest.raises(_lib.B2DError, match="workspace"):
            c.run(workspace=ws, out=out)
        torch.cuda.synchronize()
        assert (out == 7).all()
    c.check(c.run(workspace=need, out=out))


def test_attention_programmatic_launches():
    """The calls as programmatic dependents of one another, in a captured chain, give the same bits."""
    for prefix, T in ((0, 1), (512, 3)):
        c = Case([600 + 31 * i for i in range(12)], H=8, KVH=2, T=T, prefix=prefix, seed=60)
        q, table, lens = c.q.to(DEV), c.table.to(DEV), c.lens.to(DEV)
        kw = dict(prefix_table=c.prefix_table.to(DEV), prefix_len=prefix) if prefix else {}
        N = 12 * T
        pos = (c.lens[:, None] - T + torch.arange(T)).reshape(-1).long().to(DEV)
        g = torch.Generator().manual_seed(6)
        k, v = (torch.randn(N, 2, 128, generator=g).half().to(DEV) for _ in range(2))
        cos, sin = (torch.rand(1024, 128, generator=g).to(DEV) for _ in range(2))

        def chain(flags):
            qr = paged_rope_append(c.cache, q.view(N, 8, 128), k, v, pos, table, cos, sin, flags=flags)
            out = paged_attention(c.cache, qr.view(12, T, 8, 128), table, lens, flags=flags, **kw)
            probs = torch.softmax(out.float().view(12, T, -1), -1).contiguous()
            return out, verify_drafts(torch.zeros(12, T - 1, dtype=torch.int64, device=DEV), probs,
                                      torch.full((12, T), 0.3, device=DEV), flags=flags)

        want = chain(0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [chain(_lib.LAUNCH_PDL) for _ in range(3)]
        for _ in range(5):
            graph.replay()
        torch.cuda.synchronize()
        for out, (tok, acc) in got:
            assert torch.equal(out, want[0]) and torch.equal(tok, want[1][0]) and torch.equal(acc, want[1][1])


def test_attention_caller_workspace():
    c = Case([900 + i for i in range(20)], T=2, prefix=512, seed=30)
    ws = paged_attention_workspace(c.cache, c.q.to(DEV), c.table.to(DEV), prefix_len=512)
    ws.fill_(0xFF)   # needs no initial contents
    assert torch.equal(c.run(workspace=ws), c.run())
    if ws.numel():
        with pytest.raises(_lib.B2DError):
            c.run(workspace=ws[:ws.numel() - 1])


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("N,B,H,KVH,D,ps", [(1, 1, 32, 8, 128, 16), (3, 3, 4, 4, 64, 16), (10, 2, 7, 1, 128, 5),
                                            (37, 37, 8, 2, 80, 64), (130, 1, 6, 3, 256, 32), (24, 8, 2, 1, 16, 1),
                                            (1030, 2, 32, 8, 128, 16), (4100, 4, 5, 5, 96, 128)])
@pytest.mark.parametrize("dtype,table_dtype", [(F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("norm", ["none", "both", "k"])
def test_append(N, B, H, KVH, D, ps, dtype, table_dtype, norm):
    g = torch.Generator().manual_seed(N + D)
    T, S = N // B, N // B + 9
    start = torch.randint(0, 9, (B,), generator=g)
    positions = (start[:, None] + torch.arange(T)).reshape(-1)
    per = -(-S // ps)
    table = torch.randperm(B * per + 2, generator=g)[:B * per].int().view(B, per)
    fused = torch.randn(N, (H + 2 * KVH) * D, generator=g).to(dtype)
    q, k, v = (fused[:, a * D:b * D].view(N, b - a, D) for a, b in ((0, H), (H, H + KVH), (H + KVH, H + 2 * KVH)))
    ang = torch.randn(S, D, generator=g) * 3
    cos, sin = ang.cos().to(table_dtype), ang.sin().to(table_dtype)
    qw = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm == "both" else None
    kw = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm != "none" else None
    kp = torch.full((B * per + 2, KVH, ps, D), 5.0, dtype=dtype, device=DEV)
    vp = torch.full((B * per + 2, KVH, ps, D), 6.0, dtype=dtype, device=DEV)
    dev = fused.to(DEV)
    qd, kd, vd = (dev[:, a * D:b * D].view(N, b - a, D) for a, b in ((0, H), (H, H + KVH), (H + KVH, H + 2 * KVH)))
    out = paged_rope_append(PagedKV(kp, vp), qd, kd, vd, positions.to(DEV), table.to(DEV), cos.to(DEV), sin.to(DEV),
                            q_weight=None if qw is None else qw.to(DEV), k_weight=None if kw is None else kw.to(DEV), eps=1e-5)
    c, s = f64(cos)[positions.numpy()], f64(sin)[positions.numpy()]

    def check(got, x, w):
        ref, size = rope_ref(f64(x), c, s, None if w is None else f64(w), 1e-5)
        err = np.abs(f64(got) - ref)
        assert (err <= half_step(dtype) * np.abs(ref) + 2.0 ** -19 * size + 2.0 ** -25).all(), err.max()

    check(out, q, qw)
    page = table[torch.arange(N) // T, positions // ps].long()
    slot = positions % ps
    check(kp.cpu()[page, :, slot], k, kw)
    assert torch.equal(vp.cpu()[page, :, slot], v)
    untouched = torch.ones(B * per + 2, ps, dtype=torch.bool)
    untouched[page, slot] = False
    assert (kp.cpu().transpose(1, 2)[untouched] == 5).all() and (vp.cpu().transpose(1, 2)[untouched] == 6).all()


@pytest.mark.parametrize("N,norm", [(3000, "q"), (3000, "both"), (300, "q"), (5, "q"), (5000, "none")])
def test_append_mixed_batch(N, norm):
    """Tokens of a mixed batch in any order (``seq_ids``), padding among them, through the staged and the direct kernel;
    a norm of the queries alone."""
    B, H, KVH, D, ps = 7, 32, 8, 128, 16
    g = torch.Generator().manual_seed(N)
    per = -(-N // ps) + 1
    table = torch.randperm(B * per + 3, generator=g)[:B * per].int().view(B, per)
    seq = torch.randint(-1, B + 1, (N,), generator=g).int()            # -1 and B: padding
    positions = torch.zeros(N, dtype=torch.int64)
    for b in range(-1, B + 1):
        at = (seq == b).nonzero()[:, 0]
        positions[at] = torch.arange(at.numel()) + (b + 1)
    order = torch.randperm(N, generator=g)
    seq, positions = seq[order], positions[order]
    S = int(positions.max()) + 1
    q, k, v = (torch.randn(N, h, D, generator=g).to(BF16) for h in (H, KVH, KVH))
    ang = torch.randn(S, D, generator=g) * 3
    cos, sin = ang.cos(), ang.sin()
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(BF16)
    qw, kw = w if norm != "none" else None, w if norm == "both" else None
    kp, vp = (torch.full((B * per + 3, KVH, ps, D), 5.0, dtype=BF16, device=DEV) for _ in range(2))
    q_out = torch.full((N, H, D), 9.0, dtype=BF16, device=DEV)
    paged_rope_append(PagedKV(kp, vp), q.to(DEV), k.to(DEV), v.to(DEV), positions.to(DEV), table.to(DEV), cos.to(DEV), sin.to(DEV),
                      q_out=q_out, seq_ids=seq.to(DEV), q_weight=None if qw is None else qw.to(DEV),
                      k_weight=None if kw is None else kw.to(DEV), eps=1e-5)
    live = (seq >= 0) & (seq < B)
    c, s = f64(cos)[positions.numpy()], f64(sin)[positions.numpy()]

    def check(got, x, weight):
        ref, size = rope_ref(f64(x), c, s, None if weight is None else f64(weight), 1e-5)
        err = np.abs(f64(got) - ref[live.numpy()])
        assert (err <= half_step(BF16) * np.abs(ref[live.numpy()]) + 2.0 ** -19 * size[live.numpy()] + 2.0 ** -25).all(), err.max()

    check(q_out.cpu()[live], q, qw)
    assert (q_out.cpu()[~live] == 9).all()
    page, slot = table[seq[live].long(), positions[live] // ps].long(), positions[live] % ps
    check(kp.cpu()[page, :, slot], k, kw)
    assert torch.equal(vp.cpu()[page, :, slot], v[live])
    untouched = torch.ones(B * per + 3, ps, dtype=torch.bool)
    untouched[page, slot] = False
    assert (kp.cpu().transpose(1, 2)[untouched] == 5).all() and (vp.cpu().transpose(1, 2)[untouched] == 5).all()


@pytest.mark.parametrize("N,H,KVH,D", [(6, 10, 5, 128), (6, 7, 7, 80), (4000, 32, 8, 128)])   # direct, with idle lanes, staged
@pytest.mark.parametrize("size", [1e38, 1e19, 2.0 ** 60, 1e-13, 1e-25, 1e-37])
def test_append_norms_of_any_size(N, H, KVH, D, size):
    """Heads whose squares leave fp32's range, next to ordinary ones whose bits stay."""
    g = torch.Generator().manual_seed(N + D)
    per = N // 2 // 16 + 1
    table = torch.randperm(2 * per, generator=g).int().view(2, per)
    positions = torch.arange(N // 2).repeat(2)
    q, k, v = (torch.randn(N, h, D, generator=g).clamp(-3, 3).to(BF16) for h in (H, KVH, KVH))
    ang = torch.randn(N, D, generator=g) * 3
    cos, sin = ang.cos(), ang.sin()
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(BF16)
    kp, vp = (torch.zeros(2 * per, KVH, 16, D, dtype=BF16, device=DEV) for _ in range(2))
    page, slot = table[torch.arange(N) // (N // 2), positions // 16].long(), positions % 16

    def run(q, k):
        out = paged_rope_append(PagedKV(kp, vp), q.to(DEV), k.to(DEV), v.to(DEV), positions.to(DEV), table.to(DEV), cos.to(DEV),
                                sin.to(DEV), q_weight=w.to(DEV), k_weight=w.to(DEV), eps=0.0)
        return out.cpu(), kp.cpu()[page, :, slot]

    usual = run(q, k)
    q[:, 1::3], k[:, 1::3] = (q[:, 1::3].float() * size).to(BF16), (k[:, 1::3].float() * size).to(BF16)
    for got, x, was in zip(run(q, k), (q, k), usual):
        keep = [h for h in range(x.shape[1]) if h % 3 != 1]
        assert torch.equal(got[:, keep], was[:, keep])
        ref, bound = rope_ref(f64(x), f64(cos)[positions.numpy()], f64(sin)[positions.numpy()], f64(w), 0.0)
        err = np.abs(f64(got) - ref)
        assert (err <= half_step(BF16) * np.abs(ref) + 2.0 ** -19 * bound + 2.0 ** -25).all(), err.max()


def test_append_padding_and_bad_pages_write_nothing():
    N, H, KVH, D, ps, S = 8, 4, 2, 64, 16, 40
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(N, h, D, generator=g).half().to(DEV) for h in (H, KVH, KVH))
    kp, vp = (torch.full((6, KVH, ps, D), 5.0, dtype=F16, device=DEV) for _ in range(2))
    cos, sin = torch.randn(S, D, generator=g).half().to(DEV), torch.randn(S, D, generator=g).half().to(DEV)
    table = torch.tensor([[0, 1], [2, 99], [-1, 3]], dtype=torch.int32, device=DEV)
    #                 fine  padding: sequence -1, 3; position -1, S; page 99, -1, outside the table
    seq = torch.tensor([0, -1, 3, 0, 1, 1, 2, 0], dtype=torch.int32, device=DEV)
    pos = torch.tensor([17, 3, 3, -1, S, 20, 2, 39], dtype=torch.int64, device=DEV)
    q_out = torch.full((N, H, D), 9.0, dtype=F16, device=DEV)
    paged_rope_append(PagedKV(kp, vp), q, k, v, pos, table, cos, sin, q_out=q_out, seq_ids=seq)
    assert (q_out[1:5] == 9).all() and not (q_out[5:] == 9).all(-1).any() and not (q_out[0] == 9).any()
    assert torch.equal(vp[1, :, 1], v[0])
    vp[1, :, 1] = 5
    kp[1, :, 1] = 5
    assert (kp == 5).all() and (vp == 5).all()


def test_append_in_place_and_strided_pool():
    """q_out aliasing q, and a [pages, page_size, KVH, D] pool."""
    N, H, KVH, D = 5, 8, 2, 128
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(N, h, D, generator=g).bfloat16().to(DEV) for h in (H, KVH, KVH))
    cos, sin = torch.randn(64, D, generator=g).to(DEV), torch.randn(64, D, generator=g).to(DEV)
    w = torch.rand(D, generator=g).bfloat16().to(DEV)
    pos = torch.tensor([0, 15, 16, 40, 63], device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4)
    pools = [torch.zeros(4, KVH, 16, D, dtype=BF16, device=DEV) for _ in range(2)]
    nhd = [torch.zeros(4, 16, KVH, D, dtype=BF16, device=DEV) for _ in range(2)]
    want = paged_rope_append(PagedKV(*pools), q, k, v, pos, table, cos, sin, q_weight=w, k_weight=w)
    q2 = q.clone()
    got = paged_rope_append(PagedKV(*[p.transpose(1, 2) for p in nhd]), q2, k, v, pos, table, cos, sin, q_weight=w, k_weight=w,
                            q_out=q2)
    assert got is q2 and torch.equal(q2, want)
    assert all(torch.equal(a, b.transpose(1, 2)) for a, b in zip(pools, nhd))


def test_append_agrees_with_contiguous_rope():
    """Same rotation as ``rope_kv_append`` up to that kernel's extra roundings (each product and the sum to
    fp16: three half steps of the terms' size, against one here)."""
    B, H, KVH, D, S = 4, 8, 2, 128, 64
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(B, h * D, generator=g).half().to(DEV) for h in (H, KVH, KVH))
    cos, sin = torch.rand(S, D, generator=g).half().to(DEV), torch.rand(S, D, generator=g).half().to(DEV)
    pos = torch.tensor([0, 5, 33, 63], device=DEV)
    kc, vc = (torch.zeros(B, KVH, S, D, dtype=F16, device=DEV) for _ in range(2))
    q_out = torch.empty(B, H, D, dtype=F16, device=DEV)
    rope_kv_append(q, k, v, pos, cos, sin, q_out, kc, vc)
    kp, vp = (torch.zeros(B, KVH, S, D, dtype=F16, device=DEV) for _ in range(2))   # a page per sequence
    table = torch.arange(B, dtype=torch.int32, device=DEV).view(B, 1)
    got = paged_rope_append(PagedKV(kp, vp), q.view(B, H, D), k.view(B, KVH, D), v.view(B, KVH, D), pos, table, cos, sin)
    for a, b, x in ((got, q_out, q.view(B, H, D)), (kp, kc, None)):
        size = 2 * 6.0 if x is None else 2 * x.abs().max().item()
        assert (a.float() - b.float()).abs().max().item() <= 4 * half_step(F16) * size
    assert torch.equal(vp, vc)


# ------------------------------------------------------------------ verification
def verify_case(B, K, V, dtype=F32, seed=0, lookup=False, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = sharp * torch.randn(B, K + 1, V, generator=g)
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :K] + 0.7 * torch.randn(B, K, V, generator=g), -1).to(dtype)
    ids = torch.multinomial(draft.float().reshape(-1, V), 1, generator=g).view(B, K) if K else torch.zeros(B, 0, dtype=torch.int64)
    return ids, target, torch.rand(B, K + 1, generator=g), None if lookup else draft


def run_verify(ids, target, u, draft=None, lens=None, **kw):
    tok, acc = verify_drafts(ids.to(DEV), target.to(DEV), u.to(DEV), draft_probs=None if draft is None else draft.to(DEV),
                             draft_lens=None if lens is None else lens.to(DEV), **kw)
    want = verify_ref(ids.numpy(), f64(target), f64(u), None if draft is None else f64(draft), None if lens is None else lens.numpy())
    assert np.array_equal(acc.cpu().numpy(), want[1])
    assert np.array_equal(tok.cpu().numpy(), want[0])
    return tok, acc


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 2), (3, 0, 50), (5, 4, 31), (4, 7, 33), (33, 5, 1000), (2, 31, 1025),
                                   (7, 3, 32000), (1, 4, 131071)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lookup", [False, True])
def test_verify(B, K, V, dtype, lookup):
    run_verify(*verify_case(B, K, V, dtype, seed=B + K + V, lookup=lookup))


def test_verify_draft_lengths():
    ids, target, u, draft = verify_case(6, 5, 300, seed=3, sharp=0.3)
    run_verify(ids, target, u, draft, lens=torch.tensor([0, 1, 5, 9, -2, 3], dtype=torch.int32))


def test_verify_all_and_none_accepted():
    ids, target, u, draft = verify_case(4, 6, 500, seed=4)
    u[:, :6] = 0.0                      # every draft with p > 0 is accepted
    _, acc = run_verify(ids, target, u, draft)
    assert (acc == 6).all()
    u[:, :6] = 1.0
    run_verify(ids, torch.roll(target, 1, -1), u, draft)


def test_verify_borders():
    """Random numbers exactly on a border of the running sum, at 0 and just below 1; equal probabilities."""
    V = 4096
    target = torch.full((6, 2, V), 1.0 / V)
    draft = torch.full((6, 1, V), 1.0 / V)
    ids = torch.zeros(6, 1, dtype=torch.int64)
    ids[:, 0] = torch.arange(6) * 700
    u = torch.tensor([[0.0, 0.0], [0.5, 0.25], [0.999, 1 - 2.0 ** -24], [0.3, 1 / V], [0.1, 0.5], [1.0, 0.75]])
    tok, acc = run_verify(ids, target, u, draft)
    assert acc.tolist() == [1, 1, 1, 1, 1, 0] and tok[1, 1].item() == V // 4 and tok[0, 1].item() == 0
    assert tok[5, 0].item() == 3 * V // 4          # nothing is left of p - q: drawn from p


def test_verify_invalid_ids_and_weights():
    ids, target, u, draft = verify_case(8, 3, 200, seed=6)
    ids[0, 0], ids[1, 0], ids[2, 1] = -1, 200, 2 ** 40
    target[3, :, 5:60] = NAN
    target[4, :, 100:] = -1.0
    target[5] = 0.0                                # no weight anywhere: -1
    tok, _ = run_verify(ids, target, u, draft)
    assert tok[5, 0].item() == -1
    run_verify(ids, target, u, None)
    u[6, 3], u[7, 3] = NAN, 1.5                    # no border is exceeded: the last token with a weight
    run_verify(ids, target, u, draft)


def test_verify_tiny_and_negative_weights():
    """Subnormal probabilities keep their values, zeros on either side too, and a negative draft probability
    counts as it stands."""
    g = torch.Generator().manual_seed(8)
    V = 3000
    target, draft = torch.rand(4, 2, V, generator=g), torch.rand(4, 1, V, generator=g)
    target[0] *= 1e-39                   # subnormal throughout, and the draft larger: drawn from the target
    target[1, :, ::2], draft[1, :, 1::3] = 0.0, 0.0
    target[2], draft[2] = target[2] * 2e-38, draft[2] * 1e-38   # around the smallest normal number
    draft[3, :, ::5] *= -1
    ids = torch.full((4, 1), 7, dtype=torch.int64)
    for u in (0.0, 0.37, 0.999):
        run_verify(ids, target, torch.tensor([[1.0, u]] * 4), draft)
        run_verify(ids, target, torch.tensor([[1.0, u]] * 4))


def test_verify_strides_and_buffers():
    ids, target, u, draft = verify_case(3, 4, 257, seed=7)
    wide = torch.zeros(5, 3, 300)                  # [K+1, B, V'] with a longer row
    wide[:, :, :257] = target.transpose(0, 1)
    td = wide.to(DEV).transpose(0, 1)[:, :, :257]
    tok = torch.full((3, 9), 77, dtype=torch.int64, device=DEV)
    acc = torch.empty(3, dtype=torch.int32, device=DEV)
    got = verify_drafts(ids.to(DEV), td, u.to(DEV), draft_probs=draft.to(DEV), tokens=tok[:, :5], accepted=acc)
    want = verify_ref(ids.numpy(), f64(target), f64(u), f64(draft))
    assert got[1] is acc and np.array_equal(tok[:, :5].cpu().numpy(), want[0]) and (tok[:, 5:] == 77).all()
    assert np.array_equal(acc.cpu().numpy(), want[1])


# ------------------------------------------------------------------ together
def test_speculative_step_over_pages():
    """Append the drafts of a batch with a shared prompt, attend, draw logits, verify -- captured as one graph and
    replayed over several steps -- against the float64 definitions of every part."""
    B, T, H, KVH, D, ps, V, prefix = 6, 4, 8, 2, 64, 16, 600, 40
    K = T - 1
    g = torch.Generator().manual_seed(9)
    steps, S = 3, 128
    kp, vp = (torch.zeros(64, KVH, ps, D, dtype=F16, device=DEV) for _ in range(2))
    table = torch.randperm(60, generator=g)[:B * 8].int().view(B, 8).to(DEV)
    ptab = torch.tensor([61, 62, 63], dtype=torch.int32, device=DEV)
    cache = PagedKV(kp, vp)
    ang = torch.arange(S).double()[:, None] * (1e4 ** (-torch.arange(0, D, 2).double() / D))
    cos, sin = (torch.cat((f, f), -1).half().to(DEV) for f in (ang.cos(), ang.sin()))
    pk, pv = (torch.randn(prefix, KVH, D, generator=g).half().to(DEV) for _ in range(2))
    paged_rope_append(cache, torch.zeros(prefix, KVH, D, dtype=F16, device=DEV), pk, pv, torch.arange(prefix, device=DEV),
                      ptab[None], cos, sin)
    head = (torch.randn(H * D, V, generator=g) * 0.2).half().to(DEV)
    q, k, v = (torch.zeros(B * T, h, D, dtype=F16, device=DEV) for h in (H, KVH, KVH))
    lens = torch.full((B,), prefix, dtype=torch.int32, device=DEV)
    ids = torch.zeros(B, K, dtype=torch.int64, device=DEV)
    draft = torch.zeros(B, K, V, device=DEV)
    u = torch.zeros(B, T, device=DEV)
    w = torch.ones(D, dtype=F16, device=DEV)

    def step():
        positions = (lens[:, None] + torch.arange(T, device=DEV)).reshape(-1).long()
        q_rot = paged_rope_append(cache, q, k, v, positions, table, cos, sin, q_weight=w, k_weight=w, eps=1e-5)
        out = paged_attention(cache, q_rot.view(B, T, H, D), table, lens + T, prefix_table=ptab, prefix_len=prefix)
        probs = torch.softmax((out.view(B, T, H * D) @ head).float(), -1)
        tok, acc = verify_drafts(ids, probs, u, draft_probs=draft)
        return q_rot, out, probs, tok, acc

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(steps):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        draft.copy_(torch.softmax(0.2 * torch.randn(B, K, V, generator=g), -1))
        ids.copy_(torch.multinomial(draft.cpu().view(-1, V), 1, generator=g).view(B, K))
        u.copy_(torch.rand(B, T, generator=g))
        before = lens.cpu()
        graph.replay()
        torch.cuda.synchronize()
        q_rot, out, probs, tok, acc = got
        c = Case.__new__(Case)
        c.q, c.k, c.v, c.table, c.lens = q_rot.cpu().view(B, T, H, D), kp.cpu(), vp.cpu(), table.cpu(), before + T
        c.prefix_table, c.prefix, c.scale, c.dtype = ptab.cpu(), prefix, D ** -0.5, F16
        c.check(out)
        pos = (before[:, None] + torch.arange(T)).reshape(-1).numpy()
        ref, size = rope_ref(f64(k), f64(cos)[pos], f64(sin)[pos], f64(w), 1e-5)
        at = table.cpu().numpy()[np.arange(B * T) // T, pos // ps]
        assert (np.abs(f64(kp)[at, :, pos % ps] - ref) <= half_step(F16) * np.abs(ref) + 2.0 ** -19 * size + 2.0 ** -25).all()
        want = verify_ref(ids.cpu().numpy(), f64(probs), f64(u), f64(draft))
        assert np.array_equal(tok.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])
        lens += acc + 1                 # refused drafts are overwritten by the next step
