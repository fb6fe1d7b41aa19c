"""Cases of the paged-cache and speculative-decoding operators, their plain forms and their definition in 64 bits.

* ``append``: ``paged_rope_append`` -- (norms of the q and k heads,) rotary embedding, q out, k and v into their pages;
* ``attention``: ``paged_attention`` -- T new tokens per sequence over a paged cache, with a prefix shared by the batch;
* ``verify``: ``verify_drafts`` -- accept drafted tokens against the target's probabilities and draw the next token.
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
    heads = {"H": 32, "KVH": 8, "D": 128}
    return [
        # one sequence, one new token: the smallest call of a decode step
        {"name": "append_1", "op": "append", "B": 1, "T": 1, **heads, "page": 16, "base": 700, "norm": False,
         "dtype": "fp16", "table": "same"},
        # 64 sequences, five drafted tokens each, heads normalised before the rotation
        {"name": "append_64x5_norm", "op": "append", "B": 64, "T": 5, **heads, "page": 16, "base": 2048, "norm": True,
         "dtype": "bf16", "table": "fp32"},
        # the prompts of eight sequences, 1021 tokens each
        {"name": "append_prompt", "op": "append", "B": 8, "T": 1021, **heads, "page": 64, "base": 0, "norm": True,
         "dtype": "bf16", "table": "same"},
        # one sequence early in its answer: latency
        {"name": "attn_1", "op": "attention", "B": 1, "T": 1, **heads, "page": 16, "prefix": 0, "lo": 300, "hi": 300,
         "padded": False, "dtype": "fp16"},
        # the batch-8 decode of the benchmark, lengths 512 to 2048, through pages
        {"name": "attn_8_ragged", "op": "attention", "B": 8, "T": 1, **heads, "page": 16, "prefix": 0, "lo": 512,
         "hi": 2048, "padded": False, "dtype": "fp16"},
        # drafts of five tokens verified at once, odd lengths, one row of the batch empty
        {"name": "attn_16x5_drafts", "op": "attention", "B": 16, "T": 5, **heads, "page": 32, "prefix": 0, "lo": 5,
         "hi": 4099, "padded": True, "dtype": "bf16"},
        # 64 conversations on one system prompt
        {"name": "attn_64_prefix", "op": "attention", "B": 64, "T": 1, **heads, "page": 16, "prefix": 4096, "lo": 1,
         "hi": 513, "padded": False, "dtype": "bf16"},
        # many drafts against one long shared document: tensor-core work
        {"name": "attn_32x4_long_prefix", "op": "attention", "B": 32, "T": 4, **heads, "page": 64, "prefix": 16384,
         "lo": 4, "hi": 1000, "padded": False, "dtype": "bf16"},
        # long context without sharing, heads of 64
        {"name": "attn_8_long", "op": "attention", "B": 8, "T": 1, "H": 32, "KVH": 8, "D": 64, "page": 64, "prefix": 0,
         "lo": 16001, "hi": 32768, "padded": False, "dtype": "fp16"},
        # one sequence, four drafts, the benchmark's vocabulary
        {"name": "verify_1", "op": "verify", "B": 1, "K": 4, "V": 32000, "draft": True, "dtype": "fp32"},
        # a batch whose drafts come without probabilities (looked up in the prompt)
        {"name": "verify_64_lookup", "op": "verify", "B": 64, "K": 5, "V": 32768, "draft": False, "dtype": "fp32"},
        # a large batch over a large vocabulary
        {"name": "verify_128_large", "op": "verify", "B": 128, "K": 7, "V": 131071, "draft": True, "dtype": "fp32"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "verify"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "verify":
        B, V = _spread(rng, 1, 128), _spread(rng, 32000, 131071)
        return {"op": op, "B": B, "K": rng.randint(1, 7), "V": V, "draft": rng.random() < 0.7,
                "dtype": rng.choice(["fp32", "fp32", dtype])}
    D = rng.choice([64, 128, 128])
    KVH = rng.choice([1, 2, 4, 8, 8])
    H = KVH * rng.choice([1, 2, 3, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64])
    if op == "append":
        B = _spread(rng, 1, 64)
        T = _spread(rng, 1, max(1, 8168 // B)) if rng.random() < 0.5 else rng.randint(1, 8)
        return {"op": op, "B": B, "T": T, "H": min(H, 32), "KVH": KVH if min(H, 32) % KVH == 0 else 1, "D": D,
                "page": page, "base": rng.randint(0, 4096), "norm": rng.random() < 0.5, "dtype": dtype,
                "table": rng.choice(["same", "fp32"])}
    H = min(H, 32)
    KVH = KVH if H % KVH == 0 else 1
    B, T = _spread(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 5, 8])
    shared = rng.random() < 0.5
    prefix = _spread(rng, 1, 16384 // page) * page if shared else 0
    prefix = min(prefix, 16384 * 128 // (B * T) // page * page)
    most = min(16384 if shared else 524288 // T, 95000 * 1024 // (KVH * D))   # keys of the whole batch
    hi = _spread(rng, T, max(T, min(32768, most // B)))
    return {"op": op, "B": B, "T": T, "H": H, "KVH": KVH, "D": D, "page": page, "prefix": prefix,
            "lo": rng.randint(T, hi), "hi": hi, "padded": B > 1 and rng.random() < 0.3, "dtype": dtype}


def _lengths(case):
    """Keys of each sequence behind the shared prefix: evenly spread, the first none where the batch is padded."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    own_len = [lo + (hi - lo) * i // max(1, B - 1) for i in range(B)]
    if case["padded"]:
        own_len[0] = 0
    return own_len


def _tables(max_pos, D, dtype):
    inv = ROPE_THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    ang = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * inv
    ang = torch.cat((ang, ang), -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _kernels():
    """The framework's package; a user has its folder on the path."""
    folder = os.path.join(os.getcwd(), "llm-decode-triton-6gb_b200")
    if folder not in sys.path:
        sys.path.insert(1, folder)
    from b200kernels import paged, speculative
    return paged, speculative


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)

    s = {"case": case}
    if case["op"] == "verify":
        B, K, V = case["B"], case["K"], case["V"]
        logits = 2.5 * normal(B, K + 1, V)
        s["target"] = torch.softmax(logits, -1).to(dtype)
        # the drafting model is a noisier copy of the target; without one, the likeliest token is drafted
        if case["draft"]:
            draft = torch.softmax(logits[:, :K] + 0.5 * normal(B, K, V), -1).to(dtype)
            s["tokens"] = torch.multinomial(draft.view(B * K, V).float(), 1, generator=g).view(B, K)
            s["draft"] = draft
        else:
            s["tokens"] = logits[:, :K].argmax(-1)
            s["target"] = torch.softmax(4 * logits, -1).to(dtype)
            s["draft"] = None
        del logits
        s["uniforms"] = torch.rand((B, K + 1), generator=g, device=DEV)
        s["out_tokens"] = torch.empty(B, K + 1, dtype=torch.int64, device=DEV)
        s["accepted"] = torch.empty(B, dtype=torch.int32, device=DEV)
        return s

    B, T, H, KVH, D, page = (case[k] for k in ("B", "T", "H", "KVH", "D", "page"))
    if case["op"] == "append":
        per_seq = -(-(case["base"] + 16 + T) // page)
        pages = B * (-(-T // page) + 1)
        # positions of sequence b: base + b % 16, ...; only the pages that this call touches exist
        start = case["base"] + torch.arange(B, device=DEV) % 16
        s["positions"] = (start[:, None] + torch.arange(T, device=DEV)).reshape(-1)
        perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(B, -1)
        table = torch.zeros(B, per_seq + 1, dtype=torch.int32, device=DEV)
        slot = (start // page)[:, None] + torch.arange(perm.shape[1], device=DEV)
        table.scatter_(1, slot.clamp(max=per_seq), perm)
        s["page_table"] = table
        qkv = normal(B * T, (H + 2 * KVH) * D).to(dtype)   # one projection's output, split without a copy
        s["q"] = qkv[:, :H * D].view(B * T, H, D)
        s["k"] = qkv[:, H * D:(H + KVH) * D].view(B * T, KVH, D)
        s["v"] = qkv[:, (H + KVH) * D:].view(B * T, KVH, D)
        s["cos"], s["sin"] = _tables(case["base"] + 16 + T, D, dtype if case["table"] == "same" else torch.float32)
        s["q_weight"] = (1 + 0.2 * normal(D)).to(dtype) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * normal(D)).to(dtype) if case["norm"] else None
        s["q_out"] = torch.empty(B * T, H, D, dtype=dtype, device=DEV)
        s["k_pages"] = torch.zeros(pages, KVH, page, D, dtype=dtype, device=DEV)
        s["v_pages"] = torch.zeros(pages, KVH, page, D, dtype=dtype, device=DEV)
    else:
        prefix, lens = case["prefix"], _lengths(case)
        order = torch.randperm(B, generator=g, device=DEV)
        own_len = torch.tensor(lens, device=DEV)[order]
        n_pre, n_own = prefix // page, -(-own_len // page)
        s["seqlens"] = torch.where(own_len > 0, own_len + prefix, 0).to(torch.int32)
        total = n_pre + sum(-(-n // page) for n in lens)
        perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        s["prefix_table"] = perm[:n_pre].contiguous() if prefix else None
        width = n_pre + -(-max(lens) // page)
        table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
        table[:, :n_pre] = perm[:n_pre]
        at = torch.arange(width - n_pre, device=DEV)
        first = n_pre + n_own.cumsum(0) - n_own
        live = at < n_own[:, None]
        table[:, n_pre:] = torch.where(live, perm[(first[:, None] + at).clamp(max=total - 1)], 0)
        s["page_table"] = table
        s["q"] = normal(B, T, H, D).to(dtype)
        s["k_pages"] = normal(total, KVH, page, D).to(dtype)
        s["v_pages"] = normal(total, KVH, page, D).to(dtype)
        s["out"] = torch.empty(B, T, H, D, dtype=dtype, device=DEV)
    if own:
        s["cache"] = _kernels()[0].PagedKV(s["k_pages"], s["v_pages"])
    return s


def run(s):
    return {"append": _append, "attention": _attention, "verify": _verify}[s["case"]["op"]](s)


def _append(s):
    if own:
        _kernels()[0].paged_rope_append(s["cache"], s["q"], s["k"], s["v"], s["positions"], s["page_table"], s["cos"],
                                        s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                                        q_out=s["q_out"])
        return s["q_out"], s["k_pages"], s["v_pages"]
    pos, T, page = s["positions"], s["case"]["T"], s["case"]["page"]
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        half = x.shape[-1] // 2
        return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin

    s["q_out"].copy_(turned(s["q"], s["q_weight"]))
    seq = torch.arange(pos.numel(), device=pos.device) // T
    at = s["page_table"][seq, pos // page].long(), slice(None), pos % page
    s["k_pages"][at] = turned(s["k"], s["k_weight"]).to(s["k_pages"].dtype)
    s["v_pages"][at] = s["v"]
    return s["q_out"], s["k_pages"], s["v_pages"]


def _attention(s):
    if own:
        return _kernels()[0].paged_attention(s["cache"], s["q"], s["page_table"], s["seqlens"],
                                             prefix_table=s["prefix_table"], prefix_len=s["case"]["prefix"],
                                             out=s["out"])
    c = s["case"]
    B, T, H, KVH, D, page, prefix = (c[k] for k in ("B", "T", "H", "KVH", "D", "page", "prefix"))
    first = prefix // page
    q = s["q"].float().view(B, T, KVH, H // KVH, D)
    table = s["page_table"][:, first:].long()

    def of_sequences(pages):   # [B, KVH, keys, D]
        return pages[table].float().transpose(1, 2).reshape(B, KVH, -1, D)

    def of_prefix(pages):      # [KVH, keys, D], once for the batch
        return pages[s["prefix_table"].long()].float().transpose(0, 1).reshape(KVH, -1, D)

    scores = torch.einsum("btkgd,bksd->btkgs", q, of_sequences(s["k_pages"]))
    if prefix:
        scores = torch.cat((torch.einsum("btkgd,kpd->btkgp", q, of_prefix(s["k_pages"])), scores), -1)
    scores *= D ** -0.5
    limit = s["seqlens"][:, None] - T + 1 + torch.arange(T, device=q.device)
    hidden = torch.arange(scores.shape[-1], device=q.device) >= limit[..., None]
    scores.masked_fill_(hidden[:, :, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores.sub_(torch.where(top.isinf(), 0.0, top)))
    total = weights.sum(-1, keepdim=True)
    o = torch.einsum("btkgs,bksd->btkgd", weights[..., prefix:], of_sequences(s["v_pages"]))
    if prefix:
        o += torch.einsum("btkgp,kpd->btkgd", weights[..., :prefix], of_prefix(s["v_pages"]))
    return s["out"].copy_((o / torch.where(total > 0, total, 1.0)).reshape(B, T, H, D))


def _verify(s):
    if own:
        return _kernels()[1].verify_drafts(s["tokens"], s["target"], s["uniforms"], draft_probs=s["draft"],
                                           tokens=s["out_tokens"], accepted=s["accepted"])
    tokens, target, u = s["tokens"], s["target"], s["uniforms"].double()
    B, K = tokens.shape
    V = target.shape[-1]
    p_x = target[:, :K].gather(-1, tokens[..., None])[..., 0].double()
    q_x = s["draft"].gather(-1, tokens[..., None])[..., 0].double() if s["draft"] is not None else torch.ones_like(p_x)
    accepted = (u[:, :K] * q_x < p_x).long().cumprod(1).sum(1)
    rows = torch.arange(B, device=tokens.device)
    p = target[rows, accepted].double()
    at = accepted.clamp(max=K - 1)
    if s["draft"] is not None:
        q = s["draft"][rows, at].double()
    else:
        q = torch.zeros_like(p).scatter_(1, tokens[rows, at][:, None], float("inf"))
    rest = (p - q).clamp(min=0)
    rest = torch.where((accepted == K)[:, None] | (rest.sum(1, keepdim=True) <= 0), p, rest)
    running = rest.cumsum(1)
    above = running > u[:, K:] * running[:, -1:]
    index = torch.arange(V, device=tokens.device)
    last = torch.where(rest > 0, index, 0).amax(1)
    drawn = torch.where(above.any(1), above.int().argmax(1), last)
    place = torch.arange(K + 1, device=tokens.device)
    s["out_tokens"].fill_(-1)
    s["out_tokens"][:, :K].copy_(torch.where(place[:K] < accepted[:, None], tokens, -1))
    s["out_tokens"][rows, accepted] = drawn
    s["accepted"].copy_(accepted)
    return s["out_tokens"], s["accepted"]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B = case["B"]
    if case["op"] == "verify":
        # one row of the target's (and of the draft's) probabilities a sequence, and the drafted tokens' own
        rows = B * case["V"] * (2 if case["draft"] else 1)
        K = case["K"]
        return {"bytes": rows * size + B * K * (8 + 4 + 2 * size) + B * (4 + 8 * (K + 1) + 4), "flops": 3 * rows}
    T, H, KVH, D = (case[k] for k in ("T", "H", "KVH", "D"))
    if case["op"] == "append":
        N = B * T
        moved = 2 * N * (H + 2 * KVH) * D * size
        positions = min(N, T + min(B, 16) - 1)   # the tables' rows that are needed, once each
        table = 2 * positions * D * (size if case["table"] == "same" else 4)
        return {"bytes": moved + table + 12 * N, "flops": N * (H + KVH) * D * (7 if case["norm"] else 3)}
    keys = sum(_lengths(case))
    live = sum(n > 0 for n in _lengths(case))
    seen = live * case["prefix"] + keys
    cache = 2 * (case["prefix"] + keys) * KVH * D * size
    return {"bytes": cache + 2 * B * T * H * D * size + 4 * (keys + case["prefix"]) // case["page"] + 4 * B,
            "flops": 4 * T * H * D * seen}


def exact(case, seed):
    if case["op"] == "verify":
        return None   # whole numbers only
    s = prepare(case, seed)
    D = case["D"]
    if case["op"] == "append":
        half = D // 2
        cos, sin = s["cos"].double(), s["sin"].double()
        i = torch.arange(D, device=DEV)
        partner = (i + half) % D
        sign = torch.where(i < half, -1.0, 1.0).double()

        def one(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            c, n = cos.index_select(0, s["positions"]), sin.index_select(0, s["positions"])
            return c.unsqueeze(1) * x + sign * n.unsqueeze(1) * x.index_select(-1, partner)

        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        keys, page, T = one(s["k"], s["k_weight"]), case["page"], case["T"]
        flat_k = k_pages.transpose(1, 2).reshape(-1, case["KVH"], D)   # [pages * page, KVH, D]
        flat_v = v_pages.transpose(1, 2).reshape(-1, case["KVH"], D)
        n = torch.arange(s["positions"].numel(), device=DEV)
        row = s["page_table"].long()[n // T].gather(1, (s["positions"] // page)[:, None])[:, 0] * page
        row = row + s["positions"] % page
        flat_k.index_copy_(0, row, keys)
        flat_v.index_copy_(0, row, s["v"].double())
        shape = (-1, page, case["KVH"], D)
        return (one(s["q"], s["q_weight"]), flat_k.view(shape).transpose(1, 2).contiguous(),
                flat_v.view(shape).transpose(1, 2).contiguous())
    B, T, H, KVH, page, prefix = (case[k] for k in ("B", "T", "H", "KVH", "page", "prefix"))
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    lens = s["seqlens"].tolist()

    def keys_of(table, pages):
        return pages[table.long()].double().permute(1, 0, 2, 3).reshape(KVH, -1, D)

    for b in range(B):
        need = -(-lens[b] // page)
        table = s["page_table"][b, :need].clone()
        if prefix:
            table[:prefix // page] = s["prefix_table"][:need]
        if not lens[b]:
            continue
        k, v = keys_of(table, s["k_pages"]), keys_of(table, s["v_pages"])
        for t in range(T):
            n = lens[b] - T + 1 + t
            if n > 0:
                q = s["q"][b, t].double().view(KVH, H // KVH, D)
                weight = torch.softmax(torch.matmul(q, k[:, :n].transpose(1, 2)) / math.sqrt(D), -1)
                out[b, t] = torch.matmul(weight, v[:, :n]).view(H, D)
    return out
