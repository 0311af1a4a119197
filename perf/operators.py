"""The speculative-decoding operators as measured cases: inputs, plain forms, the library's calls, and 64-bit results.

Four operators: per-head norm of queries and keys with the position rotation ("rope"), entmax attention of a tree of
drafted tokens over the cache ("tree"), block tables and slot maps from request lengths ("plan"), and rows written
into the paged cache with their page statistics ("extend").  Lengths are functions of the case; values, tree shapes
and permutations of the seed.
"""

import math

import torch

#: true: ``run`` calls the library; false: elementary torch operations
own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------

def _rope(name, batch, tokens, q_heads, kv_heads, dim, dtype, far, rotary=0, interleaved=False):
    return dict(name=name, op="rope", batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, far=far, rotary=rotary or dim, interleaved=interleaved)


def _tree(name, batch, context, tokens, q_heads, kv_heads, dim, dtype, alpha, layout, ragged, short):
    return dict(name=name, op="tree", batch=batch, context=context, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads,
                dim=dim, dtype=dtype, alpha=alpha, layout=layout, ragged=ragged, short=short)


def _plan(name, batch, context, page, new, chunk, every, spare):
    return dict(name=name, op="plan", batch=batch, context=context, page=page, new=new, chunk=chunk, every=every,
                spare=spare)


def _extend(name, batch, context, tokens, kv_heads, dim, page, dtype, path):
    return dict(name=name, op="extend", batch=batch, context=context, tokens=tokens, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype, path=path)


def listed():
    return [
        # one request's next token, between the projection and the attention of a layer: latency counts
        _rope("rope_one_token", 1, 1, 32, 8, 128, "bf16", 32768),
        # 32 requests with 16 drafted tokens each, deep in a long context
        _rope("rope_drafts", 32, 16, 64, 8, 128, "fp16", 1048576),
        # prompts of odd length: only half of each head is rotated, neighbouring elements are the pairs
        _rope("rope_prompt", 5, 4099, 32, 32, 64, "bf16", 8192, rotary=32, interleaved=True),
        # a short conversation with a handful of drafts: latency counts
        _tree("tree_chat", 1, 4096, 8, 32, 8, 128, "bf16", 1.5, "dense", False, False),
        # a batch of requests of different lengths over a pool of blocks, trees of different sizes
        _tree("tree_batch", 8, 32768, 16, 32, 8, 128, "bf16", 1.5, "blocks", True, True),
        # every query head its own keys, small heads, sparsemax
        _tree("tree_mha", 3, 16001, 5, 16, 16, 64, "fp16", 2.0, "dense", True, False),
        # one long document and a wide tree, groups of eight
        _tree("tree_long", 1, 131072, 64, 64, 8, 128, "bf16", 1.5, "dense", False, False),
        # a decode step of a serving loop: one new token per request
        _plan("plan_decode", 64, 4096, 16, 1, 0, 0, 1.0),
        # many requests, every seventh with a prompt chunk; the pool runs dry near the end
        _plan("plan_prompts", 1500, 2048, 16, 3, 1021, 7, 0.97),
        # the accepted path of each request's tree goes into its cache
        _extend("extend_path", 32, 2048, 16, 8, 128, 16, "bf16", True),
        # chunks of prompts behind what the cache holds
        _extend("extend_chunk", 8, 4001, 4096, 8, 128, 16, "bf16", False),
        # full precision, a page size that divides nothing
        _extend("extend_fp32", 3, 1000, 333, 4, 64, 24, "fp32", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "tree", "tree", "plan", "extend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 128, 128])
    if op == "rope":
        q_heads, kv_heads = rng.choice([(32, 8), (64, 8), (32, 32), (8, 2), (6, 3), (1, 1)])
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, min(8192, 160000 // (batch * (q_heads + kv_heads)) * 128 // dim * 8)))
        case = _rope("", batch, tokens, q_heads, kv_heads, dim, dtype, _log(rng, 1000, 1048576),
                     rng.choice([dim, dim, dim // 2]), rng.random() < 0.4)
    elif op == "tree":
        q_heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (8, 2), (12, 4), (4, 4)])
        batch, tokens = _log(rng, 1, 16), _log(rng, 1, 64)
        # full precision has no tensor-core products, so its share of the range is smaller
        room = (1 << 29) // (16 if dtype == "fp32" else 1)
        most = min(131072, (1 << 21) // (batch * kv_heads), room // (batch * q_heads * tokens))
        case = _tree("", batch, _log(rng, 100, max(101, most)), tokens, q_heads, kv_heads, dim, dtype,
                     rng.choice([1.5, 1.5, 2.0]), rng.choice(["dense", "blocks"]), rng.random() < 0.5,
                     rng.random() < 0.5)
    elif op == "plan":
        batch = _log(rng, 1, 2048)
        case = _plan("", batch, _log(rng, 10, 4096), rng.choice([1, 8, 16, 24, 64]), rng.choice([0, 1, 1, 5]),
                     _log(rng, 1, 1024), rng.choice([0, 1, 7, 30]) if batch < 300 else rng.choice([0, 7, 30]),
                     rng.choice([1.0, 1.0, 0.9]))
    else:
        batch, kv_heads = _log(rng, 1, 32), rng.choice([1, 2, 8, 16])
        tokens = _log(rng, 1, max(1, min(4096, 262144 // (batch * kv_heads))))
        case = _extend("", batch, _log(rng, 1, min(8192, 524288 // (batch * kv_heads))), tokens, kv_heads, dim,
                       rng.choice([8, 16, 16, 24]), dtype, tokens <= 64 and rng.random() < 0.5)
    case.pop("name")
    return case


def _context_lens(case):
    """Tokens that each sequence holds before the call."""
    b, s = case["batch"], case["context"]
    if case["op"] == "tree":
        return [max(1, s - (i * 7919) % (s // 2 + 1)) if case["ragged"] else s for i in range(b)]
    if case["op"] == "plan":
        return [(s - (i * 7919) % (s + 1)) for i in range(b)]
    return [max(1, s - (i * 211) % (s // 2 + 1)) for i in range(b)]


def _new_lens(case):
    """Tokens that each sequence gets."""
    b = case["batch"]
    if case["op"] == "plan":
        return [case["chunk"] - i % 5 * (case["chunk"] // 9) if case["every"] and i % case["every"] == 0 else case["new"]
                for i in range(b)]
    t = case["tokens"]
    if case["path"]:
        return [min(t, i * 5 % 7) for i in range(b)]
    return [t - (i * 37) % (t // 4 + 1) for i in range(b)]


def _draft_lens(case):
    t = case["tokens"]
    return [1 + (i * 5 + t // 2) % t if case["short"] else t for i in range(case["batch"])]


# ---- inputs -----------------------------------------------------------------------------------------------------

def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _prepare_rope(case, gen):
    b, t, d, dtype = case["batch"], case["tokens"], case["dim"], DTYPES[case["dtype"]]
    hq, hk = case["q_heads"], case["kv_heads"]
    # queries and keys are slices of the fused projection's output
    qkv = _normal((b, t, hq + 2 * hk, d), gen, dtype) * 1.5
    first = torch.randint(0, max(1, case["far"] - t), (b, 1), generator=gen, device="cuda")
    half = case["rotary"] // 2
    return dict(q=qkv[:, :, :hq].transpose(1, 2), k=qkv[:, :, hq:hq + hk].transpose(1, 2),
                positions=(first + torch.arange(t, device="cuda")).to(torch.int32),
                inv_freq=(500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).to(torch.float32),
                q_weight=(1 + 0.2 * _normal((d,), gen, torch.float32)).to(dtype),
                k_weight=(1 + 0.2 * _normal((d,), gen, torch.float32)).to(dtype))


def _prepare_tree(case, gen, seed):
    b, s, t, d, dtype = case["batch"], case["context"], case["tokens"], case["dim"], DTYPES[case["dtype"]]
    hq, hk, page = case["q_heads"], case["kv_heads"], 16
    k, v = _normal((b, hk, s, d), gen, dtype), _normal((b, hk, s, d), gen, dtype)
    # drafted tokens of one request ask for similar things; one page in a hundred answers them, the first one always
    base = torch.randn((b, hq, 1, d), generator=gen, device="cuda")
    q = (0.8 * base + 0.6 * torch.randn((b, hq, t, d), generator=gen, device="cuda")).to(dtype)
    lead = base[:, ::hq // hk]
    shift = 0.5 * math.sqrt(d) * lead / lead.norm(dim=-1, keepdim=True)
    pages = torch.rand(s // page + 1, generator=gen, device="cuda") < 0.01
    pages[0] = True
    hit = pages.repeat_interleave(page)[:s].view(1, 1, s, 1)
    k = torch.where(hit, (k.float() + shift).to(dtype), k)
    host = torch.Generator().manual_seed(seed + 17)
    mask = torch.zeros(b, t, t, dtype=torch.bool)
    for i in range(t):          # every drafted token sees itself and what its parent sees
        parent = (torch.rand(b, generator=host) * (i + 1)).long() - 1
        if i:
            mask[:, i] = torch.where((parent >= 0)[:, None], mask[torch.arange(b), parent.clamp(min=0)], mask[:, i])
        mask[:, i, i] = True
    state = dict(q=q, k_draft=_normal((b, hk, t, d), gen, dtype), v_draft=_normal((b, hk, t, d), gen, dtype),
                 mask=mask.cuda(), draft_lens=_ints(_draft_lens(case)) if case["short"] else None,
                 out=torch.zeros(b, hq, t, d, dtype=dtype, device="cuda"),
                 taus=torch.zeros(b, hq, t, dtype=torch.float32, device="cuda"))
    lens = _context_lens(case)
    if own:
        from entmaxkv_b200 import PagedKVCache
        if case["layout"] == "blocks":
            state["cache"] = PagedKVCache(page, block_table=True, num_blocks=sum(-(-n // page) for n in lens) + 8)
        else:
            state["cache"] = PagedKVCache(page)
        state["cache"].initialize(k, v, seq_lens=lens)
        return state
    if case["layout"] == "blocks":
        n = -(-s // page)
        table = torch.randperm(b * n, generator=gen, device="cuda")
        pad = torch.zeros(b, hk, n * page - s, d, dtype=dtype, device="cuda")
        for name, x in (("k", k), ("v", v)):
            rows = torch.cat([x, pad], dim=2).view(b, hk, n, page, d).transpose(1, 2).reshape(b * n, hk, page, d)
            state[name] = torch.empty_like(rows).index_copy_(0, table, rows)
        state["table"] = table.view(b, n)
    else:
        state["k"], state["v"], state["table"] = k, v, None
    state["lens"] = _ints(lens)
    return state


def _prepare_plan(case, gen):
    b, page, lens, new = case["batch"], case["page"], _context_lens(case), _new_lens(case)
    held = [-(-n // page) for n in lens]
    need = [-(-(n + m) // page) for n, m in zip(lens, new)]
    width = max(max(need), 1)
    blocks = max(sum(held) + int((sum(need) - sum(held)) * case["spare"]), 1)
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(width, device="cuda") < _ints(held)[:, None]
    table[mine] = order[:sum(held)]
    tokens = max(sum(new) + 13, 1)          # a fixed token budget, a little more than is used
    return dict(seq_lens=_ints(lens), new_lens=_ints(new), table=table, free=order, page=page,
                slots=torch.empty(tokens, dtype=torch.int64, device="cuda"),
                positions=torch.empty(tokens, dtype=torch.int32, device="cuda"),
                row_starts=torch.empty(b + 1, dtype=torch.int32, device="cuda"))


def _prepare_extend(case, gen, seed):
    b, s, t, d, dtype, page = (case["batch"], case["context"], case["tokens"], case["dim"], DTYPES[case["dtype"]],
                               case["page"])
    lens, new = _context_lens(case), _new_lens(case)
    rows = -(-(s + t) // page) * page
    k, v = _normal((b, case["kv_heads"], rows, d), gen, dtype), _normal((b, case["kv_heads"], rows, d), gen, dtype)
    # keys and values come as slices of the fused projection's output
    kv = _normal((b, t, 2 * case["kv_heads"], d), gen, dtype)
    index = None
    if case["path"]:            # the accepted path: ascending places of the tree
        index = torch.rand(b, t, generator=gen, device="cuda").argsort(1)[:, :min(t, 7)].sort(1).values.to(torch.int32)
        index = torch.cat([index, index.new_zeros(b, t - index.shape[1])], dim=1)
    state = dict(k_new=kv[:, :, :case["kv_heads"]].transpose(1, 2), v_new=kv[:, :, case["kv_heads"]:].transpose(1, 2),
                 counts=_ints(new), index=index, start=_ints(lens), most=s + t, page=page)
    if own:
        from entmaxkv_b200 import PagedKVCache
        state["cache"] = PagedKVCache(page)
        state["cache"].initialize(k, v, seq_lens=lens, capacity=rows)
        return state
    state.update(k=k, v=v, lens=_ints(lens))
    pages = rows // page + 1        # the plain form looks at one page more than it may need
    at = torch.arange(pages, device="cuda").expand(b, pages)
    stats = _page_statistics(k, at, state["start"], page)
    mine = (at * page < state["start"][:, None])[:, None, :, None]
    state["stats"] = [torch.where(mine, x, 0).to(dtype) for x in stats]
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rope":
        state = _prepare_rope(case, gen)
    elif case["op"] == "tree":
        state = _prepare_tree(case, gen, seed)
    elif case["op"] == "plan":
        state = _prepare_plan(case, gen)
    else:
        state = _prepare_extend(case, gen, seed)
    state["case"] = case
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------

def _plain_norm_rope(x, weight, cos, sin, half, interleaved):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    turned, rest = y[..., :2 * half], y[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(x.dtype)


def _run_rope(s):
    case = s["case"]
    if own:
        from entmaxkv_b200 import qk_norm_rope
        return qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], 1e-6,
                            interleaved=case["interleaved"])
    # far positions leave 32 bits too few digits of the angle
    angle = s["positions"].double()[:, None, :, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    half = s["inv_freq"].numel()
    return (_plain_norm_rope(s["q"], s["q_weight"], cos, sin, half, case["interleaved"]),
            _plain_norm_rope(s["k"], s["k_weight"], cos, sin, half, case["interleaved"]))


def _plain_threshold(z, alpha):
    """tau with sum (z - tau)_+^(1/(alpha-1)) = 1 along the last axis, alpha 1.5 or 2, from the sorted scores: the
    first k of them are the support when the k-th lies above the threshold that they give."""
    top = z.amax(-1, keepdim=True)
    # 64 bits: long sums.  What lies more than 1 under the largest score is never in the support
    x = (z - top).clamp_(min=-1.0).sort(-1, descending=True).values.double()
    n = torch.arange(1, z.shape[-1] + 1, device=z.device)
    total = x.cumsum(-1)
    if alpha == 2.0:
        tau = (total - 1) / n
    else:
        mean = total / n
        tau = mean - ((1 / n - (x.square().cumsum(-1) / n - mean.square())).clamp(min=0)).sqrt()
    size = (x > tau).sum(-1, keepdim=True)
    return tau.gather(-1, size - 1) + top.double()


def _run_tree(s):
    case = s["case"]
    if own:
        from entmaxkv_b200 import tree_attention_decode
        tree_attention_decode(s["q"], s["cache"], s["k_draft"], s["v_draft"], s["mask"], s["out"],
                              draft_lens=s["draft_lens"], alpha=case["alpha"], taus_out=s["taus"])
        return s["out"], s["taus"]
    q, alpha = s["q"], case["alpha"]
    b, hq, t, d = q.shape
    hk = s["k_draft"].shape[1]
    k, v = s["k"], s["v"]
    if s["table"] is not None:
        k, v = (x[s["table"]].transpose(1, 2).reshape(b, hk, -1, d)[:, :, :case["context"]] for x in (k, v))
    rows = q.view(b, hk, hq // hk * t, d).float() * ((alpha - 1) / math.sqrt(d))
    z = torch.cat([rows @ k.float().transpose(-1, -2), rows @ s["k_draft"].float().transpose(-1, -2)], dim=-1)
    n = k.shape[2]
    seen = torch.cat([(torch.arange(n, device="cuda") < s["lens"][:, None])[:, None].expand(b, t, n), s["mask"]], -1)
    z = z.view(b, hk, hq // hk, t, n + t).masked_fill_(~seen[:, None, None], -math.inf).view(b, hk, -1, n + t)
    tau = _plain_threshold(z, alpha)
    p = (z - tau).clamp_(min=0).float()
    if alpha == 1.5:
        p = p.square_()
    out = (p[..., :n] @ v.float() + p[..., n:] @ s["v_draft"].float()).view(b, hq, t, d)
    tau = tau.float().view(b, hq, t)
    if s["draft_lens"] is not None:         # rows behind a short tree stay as they were
        live = (torch.arange(t, device="cuda") < s["draft_lens"][:, None])[:, None]
        out = torch.where(live[..., None], out, s["out"].float())
        tau = torch.where(live, tau, s["taus"])
    s["out"].copy_(out)
    s["taus"].copy_(tau)
    return s["out"], s["taus"]


def _run_plan(s):
    if own:
        from entmaxkv_b200 import plan_block_tables
        plan_block_tables(s["seq_lens"], s["new_lens"], s["table"], s["free"], s["page"], slots=s["slots"],
                          positions=s["positions"], row_starts=s["row_starts"])
        return s["table"], s["slots"], s["positions"], s["row_starts"]
    seq, new, table, page = s["seq_lens"].long(), s["new_lens"].long(), s["table"], s["page"]
    held, need = (seq + page - 1) // page, (seq + new + page - 1) // page
    grown = need - held
    at = torch.arange(table.shape[1], device="cuda")
    place = held.sum() + (grown.cumsum(0) - grown)[:, None] + at - held[:, None]
    block = torch.where(place < s["free"].numel(), s["free"][place.clamp(0, s["free"].numel() - 1)], -1)
    fresh = (at >= held[:, None]) & (at < need[:, None])
    table.copy_(torch.where(fresh, block, table))
    ends = new.cumsum(0)
    r = torch.arange(s["slots"].numel(), device="cuda")
    row = torch.searchsorted(ends, r, right=True)
    live, row = row < len(seq), row.clamp(max=len(seq) - 1)
    pos = seq[row] + r - (ends - new)[row]
    block = table[row, (pos // page).clamp(0, table.shape[1] - 1)].long()
    s["slots"].copy_(torch.where(live & (block >= 0), block * page + pos % page, -1))
    s["positions"].copy_(torch.where(live, pos, -1))
    s["row_starts"][0] = 0
    s["row_starts"][1:] = ends
    return table, s["slots"], s["positions"], s["row_starts"]


def _page_statistics(k, pages, lens, page):
    """min, max, mean, standard deviation in 32 bits of the pages `pages` [B, n] of k [B, H, S, D], up to `lens`."""
    b, h, rows, d = k.shape
    at = pages[:, :, None] * page + torch.arange(page, device=k.device)
    seen = (at < lens[:, None, None])[:, None, :, :, None]
    x = k.gather(2, at.clamp(max=rows - 1).view(b, 1, -1, 1).expand(b, h, -1, d)).view(b, h, -1, page, d).float()
    n = seen.sum(3).clamp(min=1)
    mean = torch.where(seen, x, 0).sum(3) / n
    std = (torch.where(seen, x - mean[:, :, :, None], 0).square().sum(3) / n).sqrt().clamp(min=1e-6)
    return torch.where(seen, x, math.inf).amin(3), torch.where(seen, x, -math.inf).amax(3), mean, std


def _run_extend(s):
    case, page = s["case"], s["page"]
    if own:
        cache = s["cache"]
        cache.extend(s["k_new"], s["v_new"], counts=s["counts"], index=s["index"], start=s["start"],
                     max_seq_len=s["most"])
        return dict(k=cache.k_cache, v=cache.v_cache, k_min=cache.k_min, k_max=cache.k_max, k_mean=cache.k_mean,
                    k_std=cache.k_std, lens=cache.seq_lens)
    k, v, start, counts = s["k"], s["v"], s["start"].long(), s["counts"].long()
    b, h, rows, d = k.shape
    t = s["k_new"].shape[2]
    i = torch.arange(t, device="cuda")
    live = i < counts[:, None]
    # rows that are not taken are written back as they are
    to = (start[:, None] + i).clamp(max=rows - 1)
    spot = to[:, None, :, None].expand(b, h, t, d)
    take = (i.expand(b, t) if s["index"] is None else s["index"].long())[:, None, :, None].expand(b, h, t, d)
    for x, fresh in ((k, s["k_new"]), (v, s["v_new"])):
        rows_in = torch.where(live[:, None, :, None], fresh.gather(2, take), x.gather(2, spot))
        x.scatter_(2, spot, rows_in)
    lens = start + counts
    pages = start[:, None] // page + torch.arange((t - 1) // page + 2, device="cuda")
    touched = ((pages * page < lens[:, None]) & (counts > 0)[:, None])[:, None, :, None]
    spot = pages[:, None, :, None].expand(b, h, -1, d)
    for x, fresh in zip(s["stats"], _page_statistics(k, pages, lens, page)):
        x.scatter_(2, spot, torch.where(touched, fresh.to(x.dtype), x.gather(2, spot)))
    s["lens"].copy_(lens)
    used = -(-s["most"] // page)
    stats = [x[:, :, :used] for x in s["stats"]]
    return dict(k=k[:, :, :s["most"]], v=v[:, :, :s["most"]], k_min=stats[0], k_max=stats[1], k_mean=stats[2],
                k_std=stats[3], lens=s["lens"])


def run(state):
    op = state["case"]["op"]
    if op == "rope":
        return _run_rope(state)
    if op == "tree":
        return _run_tree(state)
    if op == "plan":
        return _run_plan(state)
    return _run_extend(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    size = DTYPES[case["dtype"]].itemsize if "dtype" in case else 0
    if case["op"] == "rope":
        n = case["batch"] * case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        small = case["batch"] * case["tokens"] * 4 + case["rotary"] * 2 + 2 * case["dim"] * size
        return {"bytes": 2 * n * size + small, "flops": 8 * n}
    if case["op"] == "tree":
        b, t, d, hq, hk = case["batch"], case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
        lens, live = _context_lens(case), _draft_lens(case)
        # every key of the cache; of the values only rows with a weight are needed, and those depend on the data
        moved = sum(lens) * hk * d * size + sum(live) * (2 * hq + 2 * hk) * d * size + 4 * sum(live) * hq + b * t * t
        return {"bytes": moved, "flops": sum(2 * hq * m * (n + m) * d for n, m in zip(lens, live))}
    if case["op"] == "plan":
        page, lens, new = case["page"], _context_lens(case), _new_lens(case)
        fresh = sum(-(-(n + m) // page) - -(-n // page) for n, m in zip(lens, new))
        return {"bytes": 12 * case["batch"] + 8 * fresh + 12 * (sum(new) + 13), "flops": sum(new)}
    page, lens, new = case["page"], _context_lens(case), _new_lens(case)
    row = case["kv_heads"] * case["dim"] * size
    touched = sum(-(-(n + m) // page) - n // page for n, m in zip(lens, new) if m)
    before = sum(n % page for n, m in zip(lens, new) if m)
    return {"bytes": row * (4 * sum(new) + 4 * touched + before), "flops": 6 * row // size * sum(new)}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------

def _exact_rope(case, s):
    half = s["inv_freq"].numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, :, None] * s["inv_freq"].double())[:, None]
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.double()
        x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        if case["interleaved"]:
            pairs = x[..., :2 * half].unflatten(-1, (half, 2))
        else:
            pairs = x[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
        outs.append(torch.cat([pairs.flatten(-2), x[..., 2 * half:]], dim=-1))
    return tuple(outs)


def _exact_tree(case, s):
    """One (sequence, query head) at a time: scores, the root of the constraint by bisection, the weighted sum."""
    b, hq, t, d = s["q"].shape
    group, alpha = hq // s["k_draft"].shape[1], case["alpha"]
    out, taus = s["out"].double(), s["taus"].double()
    lens, live = _context_lens(case), _draft_lens(case)
    for i in range(b):
        for h in range(hq):
            g, n, m = h // group, lens[i], live[i]
            if s["table"] is None:
                k, v = s["k"][i, g, :n], s["v"][i, g, :n]
            else:
                blocks = s["table"][i]
                k, v = (x[blocks, g].reshape(-1, d)[:n] for x in (s["k"], s["v"]))
            k = torch.cat([k, s["k_draft"][i, g, :m]]).double()
            v = torch.cat([v, s["v_draft"][i, g, :m]]).double()
            z = (alpha - 1) * (s["q"][i, h, :m].double() @ k.T) / math.sqrt(d)
            z[:, n:].masked_fill_(~s["mask"][i, :m, :m], -math.inf)
            hi = z.amax(-1, keepdim=True)
            lo = hi - 1
            for _ in range(56):
                mid = (lo + hi) / 2
                over = (z - mid).clamp(min=0).pow(1 / (alpha - 1)).sum(-1, keepdim=True) > 1
                lo, hi = torch.where(over, mid, lo), torch.where(over, hi, mid)
            tau = (lo + hi) / 2
            out[i, h, :m] = (z - tau).clamp(min=0).pow(1 / (alpha - 1)) @ v
            taus[i, h, :m] = tau[:, 0]
    return out, taus


def _exact_extend(case, s):
    """One sequence at a time."""
    page, lens, new = case["page"], _context_lens(case), _new_lens(case)
    k, v, stats = s["k"].double(), s["v"].double(), [x.double() for x in s["stats"]]
    for b, (n, m) in enumerate(zip(lens, new)):
        if m == 0:
            continue
        rows = slice(0, m) if s["index"] is None else s["index"][b, :m].long()
        k[b, :, n:n + m], v[b, :, n:n + m] = s["k_new"][b, :, rows].double(), s["v_new"][b, :, rows].double()
        first, full = n // page, (n + m) // page
        spans = [(first, full)] if full > first else []
        if (n + m) % page:
            spans.append((full, full + 1))
        for p0, p1 in spans:
            x = k[b, :, p0 * page:min(p1 * page, n + m)].unflatten(1, (p1 - p0, -1))
            for to, y in zip(stats, (x.amin(2), x.amax(2), x.mean(2), x.std(2, unbiased=False).clamp(min=1e-6))):
                to[b, :, p0:p1] = y
    most = case["context"] + case["tokens"]
    used = -(-most // page)
    stats = [x[:, :, :used] for x in stats]
    return dict(k=k[:, :, :most], v=v[:, :, :most], k_min=stats[0], k_max=stats[1], k_mean=stats[2], k_std=stats[3],
                lens=None)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rope":
        return _exact_rope(case, s)
    return _exact_tree(case, s) if case["op"] == "tree" else _exact_extend(case, s)
