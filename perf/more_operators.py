"""Cases of serving from a paged cache held in 4 bits, their plain forms and their definition in 64 bits.

* ``plan``: ``PageTables.step`` -- pages, positions and slots of a step's new tokens from the requests' lengths, then the
  same requests without their new tokens (drafts refused, requests put off): the pages go back;
* ``append``: ``paged_int4_append`` -- (norms,) rotary embedding, q out, k and v quantised into their pages, which
  ``paged_int4_read`` then gives back: 4-bit values are compared as the values they stand for;
* ``read``: ``paged_int4_read`` -- cached keys and values of whole sequences in 16 bits (a prompt's next chunk);
* ``attention``: ``paged_int4_attention`` -- T new tokens per sequence over the 4-bit pages.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
ROPE_THETA = 1e6


def listed():
    heads = {"H": 32, "KVH": 8, "D": 128, "group": 64}
    return [
        # the batch-8 decode of the benchmark: one token each
        {"name": "plan_8", "op": "plan", "B": 8, "new_lo": 1, "new_hi": 1, "base": 2000, "page": 16, "free": 64},
        # a large batch, prompts of up to 127 tokens among it, not enough free pages for all
        {"name": "plan_1024_prompts", "op": "plan", "B": 1024, "new_lo": 1, "new_hi": 127, "base": 4000, "page": 16,
         "free": 3900},
        # one sequence, one new token
        {"name": "append_1", "op": "append", "B": 1, "T": 1, **heads, "rotary": 128, "interleaved": False, "page": 16,
         "base": 700, "norm": False, "dtype": "fp16"},
        # 64 sequences, five drafted tokens each, half of every head rotated in neighbouring pairs
        {"name": "append_64x5_part", "op": "append", "B": 64, "T": 5, **heads, "rotary": 64, "interleaved": True,
         "page": 32, "base": 2048, "norm": True, "dtype": "bf16"},
        # the prompts of eight sequences, 1021 tokens each
        {"name": "append_prompt", "op": "append", "B": 8, "T": 1021, **heads, "rotary": 128, "interleaved": False,
         "page": 64, "base": 0, "norm": True, "dtype": "bf16"},
        # a short sequence's cache
        {"name": "read_1", "op": "read", "B": 1, "T": 300, "KVH": 8, "D": 128, "group": 64, "page": 16, "dtype": "fp16"},
        # eight sequences before the next chunk of their prompts
        {"name": "read_8_chunk", "op": "read", "B": 8, "T": 4001, "KVH": 8, "D": 128, "group": 32, "page": 64,
         "dtype": "bf16"},
        # one sequence early in its answer: latency
        {"name": "attn_1", "op": "attention", "B": 1, "T": 1, **heads, "page": 16, "lo": 300, "hi": 300,
         "padded": False, "dtype": "fp16"},
        # the batch-8 decode of the benchmark, lengths 512 to 2048
        {"name": "attn_8_ragged", "op": "attention", "B": 8, "T": 1, **heads, "page": 16, "lo": 512, "hi": 2048,
         "padded": False, "dtype": "fp16"},
        # drafts of five tokens verified at once, odd lengths, one row of the batch empty
        {"name": "attn_16x5_drafts", "op": "attention", "B": 16, "T": 5, **heads, "page": 32, "lo": 5, "hi": 4099,
         "padded": True, "dtype": "bf16"},
        # 64 conversations, finer groups
        {"name": "attn_64_group32", "op": "attention", "B": 64, "T": 1, "H": 32, "KVH": 8, "D": 128, "group": 32,
         "page": 16, "lo": 100, "hi": 4609, "padded": False, "dtype": "bf16"},
        # long contexts: what the 4 bits are for
        {"name": "attn_8_long", "op": "attention", "B": 8, "T": 1, **heads, "page": 64, "lo": 16001, "hi": 32768,
         "padded": False, "dtype": "fp16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "read", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        B, hi = _spread(rng, 1, 1024), _spread(rng, 1, 127)
        return {"op": op, "B": B, "new_lo": rng.choice([0, 1, hi]), "new_hi": hi, "base": rng.randint(0, 4000),
                "page": page, "free": _spread(rng, 1, 3900)}
    dtype, D, group = rng.choice(["fp16", "bf16"]), rng.choice([64, 128, 128]), rng.choice([32, 64])
    KVH = rng.choice([1, 2, 4, 8, 8])
    H = KVH * rng.choice([g for g in (1, 2, 3, 4, 4, 7, 8) if KVH * g <= 32])
    common = {"op": op, "KVH": KVH, "D": D, "group": group, "page": page, "dtype": dtype}
    B = _spread(rng, 1, 64)
    if op == "append":
        T = _spread(rng, 1, max(1, 8168 // B)) if rng.random() < 0.5 else rng.randint(1, 8)
        return {**common, "B": B, "T": T, "H": H, "rotary": rng.choice([D, D, D // 2, D // 4]),
                "interleaved": rng.random() < 0.4, "base": rng.randint(0, 4096), "norm": rng.random() < 0.5}
    if op == "read":
        return {**common, "B": B, "T": _spread(rng, 1, 32008 // B)}
    T = rng.choice([1, 1, 1, 2, 4, 5, 8])
    hi = _spread(rng, T, max(T, min(32768, 195000 // T // B)))
    return {**common, "B": B, "T": T, "H": H, "lo": rng.randint(T, hi), "hi": hi,
            "padded": B > 1 and rng.random() < 0.3}


def _lengths(case):
    """Keys of each sequence: evenly spread, the first none where the batch is padded."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    lens = [lo + (hi - lo) * i // max(1, B - 1) for i in range(B)]
    if case["padded"]:
        lens[0] = 0
    return lens


def _kernels():
    """The framework's package; a user has its folder on the path."""
    folder = os.path.join(os.getcwd(), "llm-decode-triton-6gb_b200")
    if folder not in sys.path:
        sys.path.insert(1, folder)
    from b200kernels import page_plan, paged_int4
    return page_plan, paged_int4


def _quantised(x, group, dtype):
    """[..., D] in 32 bits -> codes, scales and bases per group of elements, the latter two as they are stored."""
    x = x.unflatten(-1, (-1, group))
    base = x.amin(-1, keepdim=True).to(dtype).float()
    scale = ((x.amax(-1, keepdim=True) - base) / 15).clamp(min=0).to(dtype).float()
    code = torch.where(scale > 0, ((x - base) / scale).round().clamp(0, 15), 0.0)
    return code, scale, base


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "plan":
        return _prepare_plan(s, case, g)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)

    B, T, KVH, D, page, group = (case[k] for k in ("B", "T", "KVH", "D", "page", "group"))
    channel = torch.exp(0.3 * normal(KVH, D))   # keys have stronger and weaker channels
    if case["op"] == "append":
        H = case["H"]
        per_seq = -(-(case["base"] + 16 + T) // page)
        pages = B * (-(-T // page) + 1)
        # positions of sequence b: base + b % 16, ...; only the pages that this call touches exist
        start = case["base"] + torch.arange(B, device=DEV) % 16
        s["positions"] = (start[:, None] + torch.arange(T, device=DEV)).reshape(-1)
        perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(B, -1)
        table = torch.zeros(B, per_seq + 1, dtype=torch.int32, device=DEV)
        table.scatter_(1, ((start // page)[:, None] + torch.arange(perm.shape[1], device=DEV)).clamp(max=per_seq), perm)
        s["page_table"] = table
        qkv = normal(B * T, (H + 2 * KVH) * D)      # one projection's output, split without a copy
        qkv[:, H * D:(H + KVH) * D] *= channel.reshape(-1)
        qkv = qkv.to(dtype)
        s["q"] = qkv[:, :H * D].view(B * T, H, D)
        s["k"] = qkv[:, H * D:(H + KVH) * D].view(B * T, KVH, D)
        s["v"] = qkv[:, (H + KVH) * D:].view(B * T, KVH, D)
        R = case["rotary"]
        inv = ROPE_THETA ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
        ang = torch.arange(case["base"] + 16 + T, dtype=torch.float64, device=DEV)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["q_weight"] = (1 + 0.2 * normal(D)).to(dtype) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * normal(D)).to(dtype) if case["norm"] else None
        s["q_out"] = torch.empty(B * T, H, D, dtype=dtype, device=DEV)
        s["k_out"], s["v_out"] = (torch.empty(B * T, KVH, D, dtype=dtype, device=DEV) for _ in range(2))
        if own:
            s["cache"] = _kernels()[1].PagedKVInt4.empty(pages, KVH, page, D, dtype, DEV, group_size=group)
        else:   # the pages in plain form: a code an element, a scale and a base a group
            for x in ("k", "v"):
                s[x + "_codes"] = torch.zeros(pages, page, KVH, D, dtype=torch.uint8, device=DEV)
                s[x + "_scales"], s[x + "_bases"] = (torch.zeros(pages, page, KVH, D // group, dtype=dtype, device=DEV)
                                                     for _ in range(2))
        return s

    lens = [T] * B if case["op"] == "read" else _lengths(case)
    n_pages = torch.tensor([-(-n // page) for n in lens], device=DEV)
    total, width = int(n_pages.sum()), max(1, int(n_pages.max()))
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    at = torch.arange(width, device=DEV)
    first = n_pages.cumsum(0) - n_pages
    table = torch.where(at < n_pages[:, None], perm[(first[:, None] + at).clamp(max=total - 1)], 0)
    if case["op"] == "attention":
        order = torch.randperm(B, generator=g, device=DEV)
        s["seqlens"] = torch.tensor(lens, device=DEV)[order].to(torch.int32)
        table = table[order]
        s["q"] = normal(B, T, case["H"], D).to(dtype)
        s["out"] = torch.empty(B, T, case["H"], D, dtype=dtype, device=DEV)
    else:
        s["positions"] = torch.arange(T, device=DEV).repeat(B)
        s["k_out"], s["v_out"] = (torch.empty(B * T, KVH, D, dtype=dtype, device=DEV) for _ in range(2))
    s["page_table"] = table.contiguous()
    # the cache's contents, page by page (keys as they come out of the rotation)
    k, v = (normal(total, page, KVH, D) * channel).to(dtype), normal(total, page, KVH, D).to(dtype)
    if own:
        cache = s["cache"] = _kernels()[1].PagedKVInt4.empty(total, KVH, page, D, dtype, DEV, group_size=group)
        slot = torch.arange(page, device=DEV).repeat(total)
        every = torch.arange(total, dtype=torch.int32, device=DEV)[:, None]
        _kernels()[1].paged_int4_append(cache, None, k.view(-1, KVH, D), v.view(-1, KVH, D), slot, every)
        if case["op"] == "attention":
            s["workspace"] = _kernels()[1].paged_int4_attention_workspace(cache, s["q"], s["page_table"])
    else:
        for x, t in (("k", k), ("v", v)):
            code, scale, base = _quantised(t.float(), group, dtype)
            s[x + "_codes"] = code.flatten(-2).to(torch.uint8)
            s[x + "_scales"], s[x + "_bases"] = scale[..., 0].to(dtype), base[..., 0].to(dtype)
    return s


def _prepare_plan(s, case, g):
    B, page = case["B"], case["page"]

    def whole(lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)

    s["cached"] = whole(0, case["base"], B)
    s["new"] = whole(case["new_lo"], case["new_hi"], B)
    s["none"] = torch.zeros_like(s["new"])
    s["held"] = (s["cached"] + page - 1) // page
    width = -(-(case["base"] + case["new_hi"]) // page)
    pages = B * -(-case["base"] // page) + case["free"]   # some of them are neither held nor free: other users'
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = torch.arange(width, device=DEV)
    first = s["held"].cumsum(0) - s["held"]
    s["page_table"] = torch.where(at < s["held"][:, None], perm[(first[:, None] + at).clamp(max=pages - 1)], -1)
    # a ring in the middle of its life: the free pages begin somewhere and run over its end
    begin = int(torch.randint(0, pages, (1,), generator=g, device=DEV))
    s["free"] = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    s["free"][(begin + torch.arange(case["free"], device=DEV)) % pages] = perm[pages - case["free"]:]
    s["ring"] = torch.tensor([begin, case["free"]], dtype=torch.int32, device=DEV)
    s["tokens"] = B * case["new_hi"]
    if own:
        s["tables"] = _kernels()[0].PageTables(s["page_table"], s["held"], s["free"], s["ring"], page)
        s["step"] = _kernels()[0].StepPlan.empty(B, s["tokens"], DEV)
        s["back"] = _kernels()[0].StepPlan.empty(B, 0, DEV)
    return s


def run(s):
    return {"plan": _plan, "append": _append, "read": _read, "attention": _attention}[s["case"]["op"]](s)


def _plan(s):
    if own:
        step = s["tables"].step(s["cached"], s["new"], out=s["step"])
        s["tables"].step(s["cached"], s["none"], out=s["back"])
    else:
        step = _step(s, s["new"], s["tokens"])
        _step(s, s["none"], 0)
    return {**{k: getattr(step, k) if own else step[k] for k in ("positions", "seq_ids", "slots", "seqlens", "starts", "granted")},
            "page_table": s["page_table"], "held": s["held"], "free": s["free"], "ring": s["ring"]}


def _step(s, new, tokens):
    page, table, free = s["case"]["page"], s["page_table"], s["free"]
    (B, W), P = table.shape, free.numel()
    cached, new = s["cached"].long().clamp(min=0), new.long().clamp(min=0)
    held, begin, count = s["held"].long(), s["ring"][0].long(), s["ring"][1].long()
    want = cached + new
    target = (want + page - 1) // page
    fits = target <= W
    need = torch.where(fits, (target - held).clamp(min=0), 0)
    asked = torch.where(fits, new, 0)
    ok = fits & ((need == 0) | (need.cumsum(0) <= count)) & ((asked == 0) | (asked.cumsum(0) <= tokens))
    need, asked = torch.where(ok, need, 0), torch.where(ok, new, 0)
    give = torch.where(ok, (held - target).clamp(min=0), 0)
    # pages taken from the ring's front, pages put behind its end
    col = torch.arange(W, device=DEV)
    taken = ok[:, None] & (col >= held[:, None]) & (col < target[:, None])
    given = ok[:, None] & (col >= target[:, None]) & (col < held[:, None])
    source = (begin + (need.cumsum(0) - need)[:, None] + col - held[:, None]) % P
    place = count + (give.cumsum(0) - give)[:, None] + col - target[:, None]
    before = table.clone()
    table.copy_(torch.where(taken, free[source.clamp(0, P - 1)], torch.where(given, -1, table)))
    ring = torch.cat((free, free[:1]))               # one more place, for entries that do not move
    ring[torch.where(given & (place < P), (begin + place) % P, P)] = torch.where(given, before, -1)
    free.copy_(ring[:P])
    s["held"].copy_(torch.where(ok, target, held))
    s["ring"].copy_(torch.stack(((begin + need.sum()) % P, (count - need.sum() + give.sum()).clamp(max=P))))
    starts = torch.cat((torch.zeros_like(asked[:1]), asked.cumsum(0)))
    n = torch.arange(tokens, device=DEV)
    real = n < starts[-1]
    seq = torch.searchsorted(starts[1:], n, right=True).clamp(max=B - 1)
    pos = cached[seq] + n - starts[seq]
    entry = table[seq, (pos // page).clamp(max=W - 1)].long()
    inside = real & (entry >= 0) & (entry < P)
    return {"positions": torch.where(real, pos, -1), "seq_ids": torch.where(real, seq, -1).int(),
            "slots": torch.where(inside, entry * page + pos % page, -1),
            "seqlens": torch.where(ok, want, cached).int(), "starts": starts.int(),
            "granted": torch.where(ok, asked, -1).int()}


def _append(s):
    c = s["case"]
    if own:
        _kernels()[1].paged_int4_append(s["cache"], s["q"], s["k"], s["v"], s["positions"], s["page_table"], s["cos"],
                                        s["sin"], interleaved=c["interleaved"], q_weight=s["q_weight"],
                                        k_weight=s["k_weight"], eps=EPS, q_out=s["q_out"])
        return s["q_out"], *_read(s)
    pos, T, page, R, group, dtype = s["positions"], c["T"], c["page"], c["rotary"], c["group"], DTYPES[c["dtype"]]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(x, weight):
        x = x.float()
        if weight is not None:   # the mean in 64 bits: a key's code may hang on the last bit
            r = (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
            x = x * r * weight.float()
        y, rest = x[..., :R], x[..., R:]
        a, b = (y[..., 0::2], y[..., 1::2]) if c["interleaved"] else (y[..., :R // 2], y[..., R // 2:])
        a, b = a * cos - b * sin, b * cos + a * sin
        y = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((y, rest), -1)

    s["q_out"].copy_(turned(s["q"], s["q_weight"]))
    at = s["page_table"][torch.arange(pos.numel(), device=DEV) // T, pos // page].long(), pos % page
    _store(s, "k", at, turned(s["k"], s["k_weight"]), group, dtype)
    _store(s, "v", at, s["v"].float(), group, dtype)
    return s["q_out"], *_read(s)


def _store(s, x, at, values, group, dtype):
    code, scale, base = _quantised(values, group, dtype)
    s[x + "_codes"][at] = code.flatten(-2).to(torch.uint8)
    s[x + "_scales"][at], s[x + "_bases"][at] = scale[..., 0].to(dtype), base[..., 0].to(dtype)


def _values(s, x, at):
    """What the plain pages stand for at `at`, in 32 bits."""
    code, scale, base = (s[x + n][at].float() for n in ("_codes", "_scales", "_bases"))
    return (base[..., None] + scale[..., None] * code.unflatten(-1, (-1, s["case"]["group"]))).flatten(-2)


def _read(s):
    if own:
        _kernels()[1].paged_int4_read(s["cache"], s["positions"], s["page_table"], k_out=s["k_out"], v_out=s["v_out"])
        return s["k_out"], s["v_out"]
    pos, T, page = s["positions"], s["case"]["T"], s["case"]["page"]
    at = s["page_table"][torch.arange(pos.numel(), device=DEV) // T, pos // page].long(), pos % page
    return s["k_out"].copy_(_values(s, "k", at)), s["v_out"].copy_(_values(s, "v", at))


def _attention(s):
    if own:
        return _kernels()[1].paged_int4_attention(s["cache"], s["q"], s["page_table"], s["seqlens"], out=s["out"],
                                                  workspace=s["workspace"])
    c = s["case"]
    B, T, H, KVH, D = (c[k] for k in ("B", "T", "H", "KVH", "D"))
    q = s["q"].float().view(B, T, KVH, H // KVH, D)
    table = s["page_table"].long()
    k = _values(s, "k", table).flatten(1, 2)        # [B, keys, KVH, D]
    scores = torch.einsum("btkgd,bskd->btkgs", q, k) * D ** -0.5
    del k
    limit = s["seqlens"][:, None] - T + 1 + torch.arange(T, device=DEV)
    hidden = torch.arange(scores.shape[-1], device=DEV) >= limit[..., None]
    scores.masked_fill_(hidden[:, :, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores.sub_(torch.where(top.isinf(), 0.0, top)))
    total = weights.sum(-1, keepdim=True)
    o = torch.einsum("btkgs,bskd->btkgd", weights, _values(s, "v", table).flatten(1, 2))
    return s["out"].copy_((o / torch.where(total > 0, total, 1.0)).reshape(B, T, H, D))


def _entry(case):
    """Bytes of a key or a value of one head in 4 bits."""
    return case["D"] // 2 + 4 * (case["D"] // case["group"])


def work(case):
    B = case["B"]
    if case["op"] == "plan":
        new = (case["new_lo"] + case["new_hi"]) / 2
        # lengths in and out, tokens out, and the pages that come and go, about one for `page` new tokens
        pages = min(case["free"], B * new / case["page"])
        return {"bytes": 2 * B * 24 + 20 * B * case["new_hi"] + 2 * 8 * pages, "flops": 0}
    T, KVH, D = (case[k] for k in ("T", "KVH", "D"))
    N = B * T
    if case["op"] == "read":
        return {"bytes": N * KVH * (2 * _entry(case) + 4 * D) + 12 * N, "flops": 4 * N * KVH * D}
    H = case["H"]
    if case["op"] == "append":
        # in and out, and the new entries read back
        moved = N * (2 * (H + 2 * KVH) * D + 2 * H * D + 2 * KVH * _entry(case)) + N * KVH * (2 * _entry(case) + 4 * D)
        positions = min(N, T + min(B, 16) - 1)   # the tables' rows that are needed, once each
        return {"bytes": moved + 4 * positions * case["rotary"] + 12 * N,
                "flops": N * (H + KVH) * D * (7 if case["norm"] else 3) + 2 * N * KVH * D * 5}
    keys = sum(_lengths(case))
    return {"bytes": 2 * keys * KVH * _entry(case) + 4 * N * H * D + 4 * keys // case["page"] + 4 * B,
            "flops": 4 * T * H * D * keys}


def _quantised64(x, group, dtype):
    """The values that 4 bits leave of x, in 64 bits; the scale and the base are rounded to 16 bits by definition."""
    parts = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    low = parts.min(-1, keepdim=True).values.to(dtype).double()
    step = ((parts.max(-1, keepdim=True).values - low) / 15).clamp_min(0).to(dtype).double()
    code = torch.round((parts - low) / torch.where(step > 0, step, 1.0)).clamp(0, 15)
    return (low + step * code).reshape(x.shape)


def exact(case, seed):
    global own
    if case["op"] == "plan":
        return None   # whole numbers only
    was, own = own, False
    s = prepare(case, seed)
    own = was
    dtype, B, T, KVH, D, page, group = (DTYPES[case["dtype"]] if k == "dtype" else case[k]
                                        for k in ("dtype", "B", "T", "KVH", "D", "page", "group"))
    if case["op"] == "append":
        R = case["rotary"]
        i = torch.arange(D, device=DEV)
        if case["interleaved"]:
            partner, column, sign = i ^ 1, i // 2, torch.where(i % 2 == 0, -1.0, 1.0)
        else:
            partner, column, sign = (i + R // 2) % R, i % (R // 2), torch.where(i < R // 2, -1.0, 1.0)
        turns = i < R
        partner, column = torch.where(turns, partner, i), torch.where(turns, column, 0)

        def one(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            co = s["cos"].double()[s["positions"]][:, column][:, None]
            si = s["sin"].double()[s["positions"]][:, column][:, None]
            return torch.where(turns, co * x + sign.double() * si * x.index_select(-1, partner), x)

        return (one(s["q"], s["q_weight"]), _quantised64(one(s["k"], s["k_weight"]), group, dtype),
                _quantised64(s["v"].double(), group, dtype))

    def pages_of(x, ids):   # [keys, KVH, D] of one sequence's pages
        code = s[x + "_codes"].index_select(0, ids).double().reshape(-1, KVH, D // group, group)
        low, step = (s[x + n].index_select(0, ids).double().reshape(-1, KVH, D // group, 1) for n in ("_bases", "_scales"))
        return (low + step * code).reshape(-1, KVH, D)

    if case["op"] == "read":
        return tuple(torch.cat([pages_of(x, s["page_table"][b].long())[:T] for b in range(B)]) for x in ("k", "v"))
    H = case["H"]
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    lens = s["seqlens"].tolist()
    for b in range(B):
        if not lens[b]:
            continue
        ids = s["page_table"][b, :-(-lens[b] // page)].long()
        k, v = (pages_of(x, ids).transpose(0, 1) for x in ("k", "v"))
        for t in range(T):
            n = lens[b] - T + 1 + t
            if n > 0:
                q = s["q"][b, t].double().view(KVH, H // KVH, D)
                weight = torch.softmax(torch.matmul(q, k[:, :n].transpose(1, 2)) / math.sqrt(D), -1)
                out[b, t] = torch.matmul(weight, v[:, :n]).view(H, D)
    return out
