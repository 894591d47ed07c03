"""The quantised KV cache and the attention that reads it: what is measured.

Four operators over one paged cache whose rows are grouped-affine codes (4 or 8 bits along head_dim, one bf16 scale and
one bf16 bias per group):

  append   new K / V rows are quantised into the pages and read back as the values that they now stand for
  read     the last rows of each sequence, read back
  attend   causal attention of the newest tokens of each sequence over its pages
  prefix   the same for a batch whose sequences share one long prefix

A sequence's tokens are addressed in one way throughout: of `lens[b]` cached tokens the last `cu[b+1] - cu[b]` are the
call's own, in rows cu[b] .. cu[b+1] of its packed tensors; token t of a sequence lies in row t % page of page
table[b, t // page].
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------

def _case(name, op, batch, length, new, kv_heads, per_kv, head_dim, bits, group, page, dtype, prefix=0, ragged=True):
    c = {"op": op, "batch": batch, "length": length, "new": new, "kv_heads": kv_heads, "per_kv": per_kv,
         "head_dim": head_dim, "bits": bits, "group": group, "page": page, "dtype": dtype, "prefix": prefix, "ragged": ragged}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one new token for each of 64 running sequences: the call between the qkv linear and the attention of every layer
        _case("append_tokens", "append", 64, 2000, 1, 8, 4, 128, 8, 64, 64, "bf16"),
        # prompts of eight requests at once, 4-bit cache
        _case("append_prompts", "append", 8, 4100, 4100, 8, 4, 128, 4, 64, 64, "bf16"),
        # the last tokens of a few sequences, exact in 32 bits (what a debugger or a cache migration looks at)
        _case("read_few", "read", 3, 700, 37, 2, 4, 64, 4, 32, 16, "f32"),
        # whole sequences back to bf16, as a dense attention or a transfer of the cache wants them
        _case("read_sequences", "read", 16, 6000, 6000, 8, 4, 128, 8, 64, 64, "bf16"),
        # one user, a short conversation: latency of the smallest call
        _case("attend_single", "attend", 1, 531, 1, 8, 4, 128, 8, 64, 64, "bf16"),
        # ordinary serving batch, 32 query heads on 8 cached heads
        _case("attend_batch", "attend", 64, 4096, 1, 8, 4, 128, 8, 64, 64, "bf16"),
        # long contexts in 4 bits, 64 query heads on 8 cached heads
        _case("attend_long_4bit", "attend", 12, 32771, 1, 8, 8, 128, 4, 64, 64, "bf16"),
        # drafted tokens checked in one call, small pages, 32-code groups, heads of 64
        _case("attend_drafts", "attend", 24, 3001, 5, 8, 4, 64, 8, 32, 16, "bf16"),
        # 32-bit activations, as a host that keeps its residual stream in f32 calls it
        _case("attend_f32", "attend", 16, 2500, 1, 8, 4, 128, 8, 64, 32, "f32"),
        # a chunk of two prompts over what is cached already
        _case("attend_chunk", "attend", 2, 5000, 1024, 8, 4, 128, 8, 64, 64, "bf16"),
        # a system prompt shared by 96 conversations
        _case("prefix_batch", "prefix", 96, 420, 1, 8, 8, 128, 8, 64, 64, "bf16", prefix=16384),
        # a few answers sampled from one short prompt, 4-bit cache
        _case("prefix_few", "prefix", 5, 77, 1, 4, 3, 128, 4, 32, 16, "bf16", prefix=1111),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "prefix", "prefix"])
    head_dim = rng.choice([64, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= head_dim])
    kv_heads = rng.choice([1, 2, 4, 8])
    per_kv = rng.choice([1, 2, 3, 4, 5, 7, 8])
    bits, page, dtype = rng.choice([4, 8]), rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "bf16", "f32"])
    batch = _log(rng, 1, 96)
    most = 96 * 1024 // batch                          # cached tokens of all sequences
    prefix = 0
    if op in ("append", "read"):
        length = _log(rng, 1, max(2, min(8192, most)))
        new = 1 if op == "append" and rng.random() < 0.5 else rng.randint(1, length)
    elif op == "attend":
        length = _log(rng, 1, max(2, min(32768, most)))
        new = min(length, rng.choice([1, 1, 1, 2, 5, _log(rng, 2, 700)]), max(1, 2 ** 28 // (batch * length * kv_heads * per_kv)))
    else:
        length = _log(rng, 1, max(2, min(1000, most)))
        new = min(length, rng.choice([1, 1, 1, 3]))
        prefix = _log(rng, 16, 12000)
    return _case("", op, batch, length, new, kv_heads, per_kv, head_dim, bits, group, page, dtype, prefix, rng.random() < 0.8)


def _lengths(case):
    """Cached and new tokens of each sequence: the longest first, the others spread below it."""
    most, new = case["length"], case["new"]
    if not case["ragged"]:
        return [most] * case["batch"], [new] * case["batch"]
    lens = [most - (i * 7919) % max(1, most // 2 + 1) for i in range(case["batch"])]
    news = [max(1, min(n, new - (i * 31) % max(1, new // 4 + 1))) for i, n in enumerate(lens)]
    if case["op"] == "append" and new == most:         # prompts: everything is new
        news = list(lens)
    return lens, news


# ---- the operators' plain forms ---------------------------------------------------------------------------------------

def _quantise(x, bits, group):
    """Codes (uint8, one each), scales and biases (bf16) of the last axis' groups."""
    most = float(2 ** bits - 1)
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    b = lo.to(torch.bfloat16)
    s = ((hi * 0.5 - lo * 0.5) / (most * 0.5)).to(torch.bfloat16)
    s = torch.where(s.float() < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    half = (s.float() * 0.5).unsqueeze(-1)
    q = ((g * 0.5 - b.float().unsqueeze(-1) * 0.5) / half).round().clamp(0.0, most)
    q = torch.where(half > 0, q, torch.zeros_like(q))
    return q.flatten(-2).to(torch.uint8), s, b


def _pack(q, bits):
    if bits == 4:
        q = q[..., 0::2] | (q[..., 1::2] << 4)
    return q.contiguous().view(torch.int32)


def _unpack(packed, bits):
    q = packed.contiguous().view(torch.uint8)
    return torch.stack((q & 15, q >> 4), -1).flatten(-2) if bits == 4 else q


def _places(table, lens, cu, total, page):
    """Sequence, page and row of each of the call's own tokens."""
    t = torch.arange(total, device=lens.device)
    b = torch.searchsorted(cu.long(), t, right=True) - 1
    at = lens.long()[b] - (cu.long()[b + 1] - t)
    return b, table.long()[b, at // page], at % page


def _rows(s, which, pages, rows):
    """Values in 32 bits of K (0) or V (1) rows: [..., kv_heads, head_dim] at (page, row)."""
    q = _unpack(s["packed"][pages, which, :, rows], s["bits"]).float()
    scale, bias = (s[n][pages, which, :, rows].float().repeat_interleave(s["group"], -1) for n in ("scales", "biases"))
    return q * scale + bias


def _all_rows(s, which, table):
    """Values in 32 bits of whole block tables: [..., kv_heads, tokens, head_dim]."""
    t = table.long().clamp(min=0)
    q = _unpack(s["packed"][:, which][t], s["bits"]).float()
    scale, bias = (s[n][:, which][t].float().repeat_interleave(s["group"], -1) for n in ("scales", "biases"))
    return (q * scale + bias).transpose(-4, -3).flatten(-3, -2)


def _plain_attention(s):
    q, cu, lens, page = s["q"], s["cu"].long(), s["lens"].long(), s["page"]
    batch, kv_heads, per_kv, dim = lens.numel(), s["kv_heads"], s["per_kv"], q.shape[-1]
    most = s["max_new"]
    i = torch.arange(most, device=q.device)
    news = cu[1:] - cu[:-1]
    own_rows = i < news[:, None]                                              # [batch, most]
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q.float()[at].view(batch, most, kv_heads, per_kv, dim).permute(0, 2, 3, 1, 4) / math.sqrt(dim)
    rows = rows.reshape(batch, kv_heads, per_kv * most, dim)
    keys, values = _all_rows(s, 0, s["table"]), _all_rows(s, 1, s["table"])   # [batch, kv_heads, tokens, dim]
    j = torch.arange(keys.shape[2], device=q.device)
    live = (j < lens[:, None])[:, None, :, None]
    keys, values = torch.where(live, keys, 0.0), torch.where(live, values, 0.0)
    seen = (j <= (lens - news)[:, None, None] + i[:, None]) & own_rows[:, :, None]   # [batch, most, tokens]
    seen = seen[:, None, None].expand(-1, -1, per_kv, -1, -1).reshape(batch, 1, per_kv * most, -1)
    score = (rows @ keys.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["prefix"]:
        n = s["prefix"]
        pk, pv = _all_rows(s, 0, s["prefix_table"])[:, :n], _all_rows(s, 1, s["prefix_table"])[:, :n]
        every = rows.transpose(0, 1).flatten(1, 2)                            # [kv_heads, batch * per_kv * most, dim]
        pscore = every @ pk.transpose(-1, -2)
        top = torch.maximum(top, pscore.amax(-1).unflatten(1, (batch, -1)).transpose(0, 1).unsqueeze(-1))
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total, out = p.sum(-1, keepdim=True), p @ values
    if s["prefix"]:
        pp = torch.exp(pscore - top.squeeze(-1).transpose(0, 1).flatten(1, 2).unsqueeze(-1))
        total = total + pp.sum(-1).unflatten(1, (batch, -1)).transpose(0, 1).unsqueeze(-1)
        out = out + (pp @ pv).unflatten(1, (batch, -1)).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.view(batch, kv_heads, per_kv, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, -1, dim)
    b, _, _ = _places(s["table"], lens, cu, q.shape[0], page)
    return out[b, torch.arange(q.shape[0], device=q.device) - cu[b]].to(q.dtype)


def _plain(s):
    if s["op"] in ("attend", "prefix"):
        return _plain_attention(s)
    _, pages, rows = _places(s["table"], s["lens"], s["cu"], s["total"], s["page"])
    if s["op"] == "append":
        x = torch.stack((s["k"], s["v"]), 1)                                  # [total, 2, kv_heads, head_dim]
        q, scale, bias = _quantise(x, s["bits"], s["group"])
        for name, v in (("packed", _pack(q, s["bits"])), ("scales", scale), ("biases", bias)):
            s[name][pages, :, :, rows] = v
    return {"k": _rows(s, 0, pages, rows).to(s["dtype"]), "v": _rows(s, 1, pages, rows).to(s["dtype"])}


# ---- state and one pass -----------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens, news = _lengths(case)
    page, kv_heads, dim, group, bits = (case[k] for k in ("page", "kv_heads", "head_dim", "group", "bits"))
    heads, batch, prefix, dtype = kv_heads * case["per_kv"], case["batch"], case["prefix"], DTYPES[case["dtype"]]
    wide = max(-(-n // page) for n in lens)
    need = [-(-n // page) for n in lens]
    prefix_pages = -(-prefix // page)
    pages = sum(need) + prefix_pages
    order = torch.randperm(pages, generator=gen, device=dev).int()            # a running server's pages lie in no order
    take = torch.tensor(need, device=dev)
    col = torch.arange(wide, device=dev)
    first = torch.cumsum(take, 0) - take
    table = torch.where(col < take[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).int()

    # K rows have a few strong channels, as keys after rotation have; V rows are even
    packed = torch.empty(pages, 2, kv_heads, page, dim * bits // 32, dtype=torch.int32, device=dev)
    scales = torch.empty(pages, 2, kv_heads, page, dim // group, dtype=torch.bfloat16, device=dev)
    biases = torch.empty_like(scales)
    strong = torch.exp(torch.randn(kv_heads, 1, dim, generator=gen, device=dev) * 0.5)
    for at in range(0, pages, 1024):
        n = min(1024, pages - at)
        x = torch.randn(n, 2, kv_heads, page, dim, generator=gen, device=dev)
        x[:, 0] *= strong
        q, s, b = _quantise(x.to(torch.bfloat16), bits, group)
        packed[at:at + n], scales[at:at + n], biases[at:at + n] = _pack(q, bits), s, b
    total = sum(news)
    qkv = torch.randn(total, (heads + 2 * kv_heads) * dim, generator=gen, device=dev).to(dtype)   # the qkv linear's output
    cu = torch.zeros(batch + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(news), 0)
    state = {
        "op": case["op"], "bits": bits, "group": group, "page": page, "kv_heads": kv_heads, "per_kv": case["per_kv"],
        "prefix": prefix, "dtype": dtype, "total": total, "max_new": max(news), "packed": packed, "scales": scales, "biases": biases,
        "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "cu": cu.to(dev),
        "prefix_table": order[pages - prefix_pages:].contiguous(),
        "q": qkv[:, :heads * dim].unflatten(1, (heads, dim)),
        "k": qkv[:, heads * dim:(heads + kv_heads) * dim].unflatten(1, (kv_heads, dim)),
        "v": qkv[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim)),
    }
    if own:
        import talu_b200 as gaf
        ctx = gaf.Context(0)
        state["ctx"], state["cache"] = ctx, gaf.KvCache.wrap_device(ctx, packed, scales, biases, group, bits)
    return state


def run(s):
    if not own:
        return _plain(s)
    import talu_b200 as gaf
    ctx, cache, at = s["ctx"], s["cache"], (s["table"], s["lens"])
    if s["op"] == "attend":
        return gaf.attention(ctx, cache, s["q"], *at, cu=s["cu"], max_new=s["max_new"])
    if s["op"] == "prefix":
        return gaf.attention_shared_prefix(ctx, cache, s["q"], s["prefix_table"], s["prefix"], *at, cu=s["cu"], max_new=s["max_new"])
    if s["op"] == "append":
        gaf.kv_append(ctx, cache, s["k"], s["v"], *at, cu=s["cu"])
    k, v = gaf.kv_read(ctx, cache, *at, cu=s["cu"], total=s["total"], dtype=s["dtype"])
    return {"k": k, "v": v}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    lens, news = _lengths(case)
    dim, kv_heads, per_kv = case["head_dim"], case["kv_heads"], case["per_kv"]
    elt = 2 if case["dtype"] == "bf16" else 4
    stored = kv_heads * 2 * (dim * case["bits"] / 8 + dim / case["group"] * 4)     # bytes of one token's K and V
    if case["op"] in ("append", "read"):
        plain = kv_heads * 2 * dim * elt
        times = 2 if case["op"] == "append" else 1                                # written, then read back
        return {"bytes": sum(news) * times * (stored + plain), "flops": sum(news) * kv_heads * 2 * dim * (8 * (times - 1) + 2)}
    # causal: query i of n new ones sees all but the n - 1 - i tokens behind it
    pairs = sum(n * m - n * (n - 1) // 2 for m, n in zip(lens, news)) + sum(news) * case["prefix"]
    return {"bytes": (sum(lens) + case["prefix"]) * stored + sum(news) * kv_heads * per_kv * dim * 2 * elt,
            "flops": 4 * dim * kv_heads * per_kv * pairs}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def _exact_rows(packed, scales, biases, bits, group):
    """Stored rows [n, ...words] as 64-bit values: value j of a word at bits j * bits."""
    shift = torch.arange(0, 32, bits, device=packed.device)
    q = ((packed.long().unsqueeze(-1) >> shift) & (2 ** bits - 1)).flatten(-2).double()
    q = q.view(*q.shape[:-1], -1, group)
    return (q * scales.double().unsqueeze(-1) + biases.double().unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    lens, news = _lengths(case)
    page, bits, group, dim = s["page"], s["bits"], s["group"], case["head_dim"]
    pairs = work(case)["flops"] / (4 * dim)
    if case["op"] in ("attend", "prefix") and pairs > 1.5e9:
        return None
    out_q, out_k, out_v, begin = [], [], [], 0
    most = 2.0 ** bits - 1

    def seq(table, n, which):
        """[kv_heads, n, dim] of the first n tokens of one block table."""
        pages = table[:-(-n // page)].long()
        x = _exact_rows(s["packed"][pages, which], s["scales"][pages, which], s["biases"][pages, which], bits, group)
        return x.transpose(0, 1).reshape(case["kv_heads"], -1, dim)[:, :n]

    if case["op"] == "prefix":
        prefix_k, prefix_v = seq(s["prefix_table"], case["prefix"], 0), seq(s["prefix_table"], case["prefix"], 1)
    for b, (n, m) in enumerate(zip(lens, news)):
        mine = slice(begin, begin + m)
        begin += m
        if case["op"] == "append":
            for x, to in ((s["k"], out_k), (s["v"], out_v)):
                g = x[mine].double().unflatten(-1, (-1, group))
                low = g.amin(-1, keepdim=True)
                step = ((g.amax(-1, keepdim=True) - low) / most).to(torch.bfloat16).double()
                low = low.to(torch.bfloat16).double()
                code = torch.where(step > 0, (g - low) / torch.where(step > 0, step, 1.0), 0.0).round().clamp(0.0, most)
                to.append((code * step + low).flatten(-2))
        elif case["op"] == "read":
            out_k.append(seq(s["table"][b], n, 0)[:, n - m:].transpose(0, 1))
            out_v.append(seq(s["table"][b], n, 1)[:, n - m:].transpose(0, 1))
        else:
            k, v = seq(s["table"][b], n, 0), seq(s["table"][b], n, 1)
            hidden = torch.ones(m, n, dtype=torch.bool, device=k.device).triu(n - m + 1)
            if case["op"] == "prefix":
                k, v = torch.cat((prefix_k, k), 1), torch.cat((prefix_v, v), 1)
                hidden = torch.cat((hidden.new_zeros(m, case["prefix"]), hidden), 1)
            q = s["q"][mine].double().unflatten(1, (case["kv_heads"], -1)).permute(1, 2, 0, 3)    # [kv_heads, per_kv, m, dim]
            w = torch.einsum("hgmd,hnd->hgmn", q, k) / dim ** 0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out_q.append(torch.einsum("hgmn,hnd->mhgd", w, v).flatten(1, 2))
    if out_q:
        return torch.cat(out_q)
    return {"k": torch.cat(out_k), "v": torch.cat(out_v)}
