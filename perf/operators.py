"""What the operators next to the recurrent state are measured on: the 8-bit key/value cache of a hybrid
model's full-attention layers (append and attention) and the norm at the entry of every layer, with its
8-bit output.

A case is a dict of plain values with a ``kind``:

* ``attend``  queries over the paged cache: one token a request (decode), a few (speculation), a whole chunk
  of a prompt.  Codes are e4m3 with one scale for each block of tokens and head;
* ``append``  new tokens' keys and values into the cache;
* ``norm``    residual addition, root-mean-square norm, e4m3 codes with a scale per token or per 128 columns.

``prepare`` makes the inputs on the GPU from the seed, ``run`` is one pass (plain torch, or with ``own`` the
framework's calls), ``exact`` the same in 64 bits, ``work`` the bytes and operations that it cannot do without.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
TINY_EXP, BIG_EXP = -100, 119          # the cache's scales are powers of two from 2^-100 to 2^119
NORM_EPS, AMAX_FLOOR, GROUP = 1e-6, 1e-12, 128


def _attend(name, requests, tokens, context, heads=32, kv_heads=8, dim=128, act="bf16", page=64, block=32,
            ragged_context=False, ragged_tokens=False):
    """``context``: cached tokens of a request with the new ones among them (the longest one, where ragged)."""
    return dict(name=name, kind="attend", requests=requests, tokens=tokens, context=context, heads=heads,
                kv_heads=kv_heads, dim=dim, act=act, page=page, block=block, ragged_context=ragged_context,
                ragged_tokens=ragged_tokens)


def _append(name, requests, tokens, context, kv_heads=8, dim=128, act="bf16", page=64, block=32,
            ragged_context=False, ragged_tokens=False):
    return dict(name=name, kind="append", requests=requests, tokens=tokens, context=context, kv_heads=kv_heads,
                dim=dim, act=act, page=page, block=block, ragged_context=ragged_context, ragged_tokens=ragged_tokens)


def _norm(name, rows, width, act="bf16", grouped=False):
    return dict(name=name, kind="norm", rows=rows, width=width, act=act, grouped=grouped)


def listed():
    return [
        # one interactive user's decode step: a single query token over a short context, small pages
        _attend("attend_decode_1", 1, 1, 1500, page=16, block=16),
        # the serving batch: 64 requests at every stage of their contexts
        _attend("attend_decode_64", 64, 1, 8192, ragged_context=True),
        # the largest batch: 128 requests deep into their contexts; the keys pass 2^30 bytes
        _attend("attend_decode_128", 128, 1, 8192, page=128, block=64),
        # two very long documents, few key/value heads: the work is in the length alone
        _attend("attend_decode_long", 2, 1, 131071, heads=16, kv_heads=2),
        # four speculated tokens of every request checked at once, narrow heads, fp16
        _attend("attend_verify_4", 32, 4, 4096, heads=16, kv_heads=8, dim=64, act="fp16", block=16, ragged_context=True),
        # a chunk of 2048 tokens of a long prompt, over what is cached of it
        _attend("attend_chunk_2048", 1, 2048, 16384, block=64),
        # whole prompts of six requests, of all lengths, in one call
        _attend("attend_prompts_6", 6, 2000, 2000, heads=16, kv_heads=16, ragged_tokens=True),
        # one new token of each of 64 requests into the cache
        _append("append_64", 64, 1, 2048, ragged_context=True),
        # a prompt chunk of four requests into the cache
        _append("append_8192", 4, 2048, 4100),
        # the entry of a layer: one token, a decode batch, a prompt
        _norm("norm_1", 1, 4096),
        _norm("norm_256", 256, 5120),
        _norm("norm_16384", 16384, 4096, grouped=True),
    ]


# ---------------------------------------------------------------------------
# lengths: a function of the case alone, so that work() knows them
# ---------------------------------------------------------------------------

def _spread(n, top):
    """``n`` whole numbers spread evenly over 1..top in an order of no pattern; the last one is ``top``."""
    part = [math.modf((i + 1) * 0.6180339887498949)[0] for i in range(n)]
    return [1 + int((top - 1) * p) for p in part[:-1]] + [top]


def _lengths(c):
    """New tokens and cached tokens (new ones among them) of every request."""
    B = c["requests"]
    new = _spread(B, c["tokens"]) if c["ragged_tokens"] else [c["tokens"]] * B
    old = c["context"] - c["tokens"]
    old = [x - 1 for x in _spread(B, old + 1)] if c["ragged_context"] else [old] * B
    return new, [n + o for n, o in zip(new, old)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(["decode", "decode", "verify", "chunk", "append", "append1", "norm", "norm"])
    act = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        return _norm("", _log_int(rng, 1, 16384), _log_int(rng, 64, 16384), act, rng.random() < 0.5)
    page = rng.choice([16, 32, 64, 128])
    more = dict(act=act, page=page, block=rng.choice([b for b in (16, 32, 64, 128) if b <= page]),
                dim=rng.choice([64, 128]), kv_heads=rng.choice([1, 2, 4, 8, 16]))
    if kind in ("append", "append1"):
        tokens = 1 if kind == "append1" else _log_int(rng, 2, 4096)
        return _append("", _log_int(rng, 1, 256 if tokens == 1 else 16), tokens, tokens + _log_int(rng, 1, 4096) - 1,
                       ragged_context=rng.random() < 0.5, ragged_tokens=tokens > 1 and rng.random() < 0.5, **more)
    more["heads"] = more["kv_heads"] * rng.choice([1, 2, 3, 4, 8])
    if kind == "decode":
        requests, tokens, context = _log_int(rng, 1, 128), 1, _log_int(rng, 1, 65536)
    elif kind == "verify":
        requests, tokens, context = _log_int(rng, 1, 64), rng.randrange(2, 9), _log_int(rng, 16, 16384)
    else:
        requests, tokens = _log_int(rng, 1, 8), _log_int(rng, 9, 2048)
        context = tokens + _log_int(rng, 1, 8192) - 1
    return _attend("", requests, tokens, context, ragged_context=rng.random() < 0.5,
                   ragged_tokens=tokens > 8 and rng.random() < 0.5, **more)


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _draw_once(rng)
        w = work(c)
        dense = 0
        if c["kind"] == "attend":                       # what the plain form holds: every score, padded keys
            dense = 4 * c["requests"] * c["context"] * (c["heads"] * c["tokens"] + 4 * c["kv_heads"] * c["dim"])
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and dense <= 24e9:
            del c["name"]
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(shape, g, sigma=1.0):
    return torch.empty(shape, device=DEV).normal_(0.0, sigma, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cache(c, pages, g):
    """Codes of keys or values whose blocks fill the upper half of the e4m3 range, and their scales: values of
    about 1."""
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    codes = torch.empty(shape, dtype=F8, device=DEV)
    for part in codes.split(max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))):      # bounds the fp32 scratch
        part.copy_(_normal(part.shape, g, 100.0).clamp_(-F8_MAX, F8_MAX))
    power = torch.randint(-7, -5, (*shape[:2], c["page"] // c["block"]), device=DEV, generator=g)
    return codes, torch.ldexp(torch.ones(power.shape, device=DEV), power)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    st, dt = {"case": c}, DTYPES[c["act"]]
    if c["kind"] == "norm":
        N, W = c["rows"], c["width"]
        # a residual stream grows over the layers, and some of its columns are far larger than the others
        st["x"] = _normal((N, W), g).to(dt)
        st["residual"] = (_normal((N, W), g, 3.0) * torch.exp(_normal((W,), g))).to(dt)
        st["weight"] = (1.0 + _normal((W,), g, 0.1)).to(dt)
        st["residual_out"] = torch.zeros((N, W), dtype=dt, device=DEV)
        st["codes"] = torch.zeros((N, W), dtype=F8, device=DEV)
        st["scale"] = torch.zeros((N, -(-W // GROUP)) if c["grouped"] else (N,), device=DEV)
        return st
    B, page = c["requests"], c["page"]
    new, lengths = _lengths(c)
    need = [-(-n // page) for n in lengths]
    # pages in random order; page 0 is the padding page, in the table wherever a request has no page
    order = (torch.randperm(sum(need), device=DEV, generator=g) + 1).to(torch.int32).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    st["table"], st["lengths"], st["page_count"] = _ints(rows), _ints(lengths), sum(need) + 1
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st["starts"] = _ints(starts) if c["ragged_tokens"] else None
    st["k_codes"], st["k_scale"] = _cache(c, st["page_count"], g)
    st["v_codes"], st["v_scale"] = _cache(c, st["page_count"], g)
    N = starts[-1]
    if c["kind"] == "append":
        st["k"] = _normal((N, c["kv_heads"], c["dim"]), g, 1.5).to(dt)
        st["v"] = _normal((N, c["kv_heads"], c["dim"]), g).to(dt)
    else:
        st["q"] = _normal((N, c["heads"], c["dim"]), g, 2.0).to(dt)
        st["out"] = torch.zeros((N, c["heads"], c["dim"]), dtype=dt, device=DEV)
        st["scale"] = c["dim"] ** -0.5
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _cached(codes, scale, table, block):
    """The table's tokens as the values that they stand for: [B, HKV, L, D] in 32 bits."""
    x = codes.view(torch.uint8)[table.long()].view(F8).float()                  # [B, P, HKV, page, D]
    x = x * scale[table.long()].repeat_interleave(block, dim=3)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _rows(st, c):
    """Each request's new tokens as rows of a padded [B, T]: their places in the call's tensors, whether there is
    one, and their positions in the context."""
    B, T = c["requests"], c["tokens"]
    t = torch.arange(T, device=DEV)
    if st["starts"] is None:
        first, count = T * torch.arange(B, device=DEV), torch.full((B,), T, device=DEV)
    else:
        first, count = st["starts"][:-1].long(), st["starts"].diff().long()
    there = t < count[:, None]
    return torch.where(there, first[:, None] + t, 0), there, (st["lengths"].long() - count)[:, None] + t


def _plain_attend(st, c):
    B, H, G, D, T = c["requests"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["tokens"]
    place, there, position = _rows(st, c)
    k = _cached(st["k_codes"], st["k_scale"], st["table"], c["block"])
    q = st["q"].float()[place].view(B, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(st["scale"]).view(B, H, G, T, -1)
    del k, q
    seen = torch.arange(s.shape[-1], device=DEV) <= position[..., None]         # [B, T, L]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _cached(st["v_codes"], st["v_scale"], st["table"], c["block"])
    o = torch.matmul(p.view(B, H, G * T, -1), v).view(B, H, G, T, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, T, H * G, D)
    st["out"].view(-1, H * G, D)[place[there]] = o[there].to(st["out"].dtype)
    return st["out"]


def _power_of_two(amax):
    """The smallest power of two s with amax / s <= 448."""
    part, power = torch.frexp(amax)                     # amax = part * 2^power, part in [0.5, 1); 448 = 0.875 * 2^9
    power = (power - 9 + (part > 0.875)).clamp(TINY_EXP, BIG_EXP)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, power, TINY_EXP))


def _plain_append(st, c, new, codes, scale):
    H, D, page, block = c["kv_heads"], c["dim"], c["page"], c["block"]
    place, there, position = _rows(st, c)
    there = there & (position >= 0)
    request = torch.arange(c["requests"], device=DEV)[:, None].expand_as(place)[there]
    position, x = position[there], new.float()[place[there]]                    # [n], [n, HKV, D]
    at = st["table"].long()[request, position // page] * (page // block) + position % page // block
    # largest magnitude and first place of each block's new tokens; the old scale counts where there are earlier ones
    per = page // block
    top = torch.zeros(st["page_count"] * per, H, device=DEV)
    top.scatter_reduce_(0, at[:, None].expand(-1, H), x.abs().amax(-1), "amax")
    begin = torch.full((st["page_count"] * per,), block, device=DEV)
    begin.scatter_reduce_(0, at, position % block, "amin")
    old = scale.transpose(1, 2).reshape(-1, H)
    now = torch.maximum(_power_of_two(top), torch.where(begin[:, None] > 0, old, 0.0))
    now = torch.where(begin[:, None] < block, now, old)
    # codes of the earlier tokens in a block whose scale grew
    grown = (begin[:, None] > 0) & (now > old)                                  # [pages * blocks, HKV]
    which = grown.any(1).nonzero()[:, 0]
    blocks = codes.view(torch.uint8).view(-1, H, per, block, D)
    part = blocks[which // per, :, which % per]                                 # [n, HKV, block, D]
    less = (part.view(F8).float() * (old / now)[which][..., None, None]).to(F8).view(torch.uint8)
    early = torch.arange(block, device=DEV) < begin[which, None]
    change = grown[which][:, :, None, None] & early[:, None, :, None]
    blocks[which // per, :, which % per] = torch.where(change, less, part)
    scale.copy_(now.view(-1, per, H).transpose(1, 2))
    y = (x / now[at][..., None]).clamp(-F8_MAX, F8_MAX).to(F8)
    h = torch.arange(H, device=DEV)
    codes.view(torch.uint8)[(at // per)[:, None], h, (position % page)[:, None]] = y.view(torch.uint8)


def _plain_norm(st, c):
    N, W = c["rows"], c["width"]
    h = st["x"].float() + st["residual"].float()
    st["residual_out"].copy_(h)
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + NORM_EPS) * st["weight"].float()
    if c["grouped"]:
        pad = torch.nn.functional.pad(y, (0, -W % GROUP)).view(N, -1, GROUP)
        st["scale"].copy_(pad.abs().amax(-1).clamp(min=AMAX_FLOOR) / F8_MAX)
        s = st["scale"].repeat_interleave(GROUP, dim=1)[:, :W]
    else:
        st["scale"].copy_(y.abs().amax(-1).clamp(min=AMAX_FLOOR) / F8_MAX)
        s = st["scale"][:, None]
    st["codes"].copy_((y / s).clamp(-F8_MAX, F8_MAX))
    return {"residual": st["residual_out"], "codes": st["codes"], "scale": st["scale"]}


def run(state):
    st, c = state, state["case"]
    if c["kind"] == "norm":
        if not own:
            return _plain_norm(st, c)
        from carrykernel_b200.vllm_integration import residual_norm
        residual_norm.add_rms_norm_quant(st["x"], st["residual"], st["weight"], st["codes"], st["scale"], NORM_EPS,
                                         residual_out=st["residual_out"])
        return {"residual": st["residual_out"], "codes": st["codes"], "scale": st["scale"]}
    cache = (st["k_codes"], st["k_scale"], st["v_codes"], st["v_scale"])
    if c["kind"] == "append":
        if own:
            from carrykernel_b200.vllm_integration import quantized_kv_cache
            quantized_kv_cache.quantized_kv_append(st["k"], st["v"], *cache, st["table"], st["lengths"],
                                                   query_start=st["starts"], max_query_len=c["tokens"])
        else:
            _plain_append(st, c, st["k"], st["k_codes"], st["k_scale"])
            _plain_append(st, c, st["v"], st["v_codes"], st["v_scale"])
        return {"k_codes": cache[0], "k_scale": cache[1], "v_codes": cache[2], "v_scale": cache[3]}
    if not own:
        return _plain_attend(st, c)
    from carrykernel_b200.vllm_integration import quantized_kv_cache
    return quantized_kv_cache.quantized_paged_attention(st["q"], st["scale"], *cache, st["out"], st["table"],
                                                        st["lengths"], query_start=st["starts"],
                                                        max_query_len=c["tokens"])


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits, request by request
# ---------------------------------------------------------------------------

def _exact_attend(st, c):
    new, lengths = _lengths(c)
    G, page, block = c["heads"] // c["kv_heads"], c["page"], c["block"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    first = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        pages = st["table"][b, :-(-length // page)].long()
        for h in range(c["kv_heads"]):
            k, v = (st[x + "_codes"][:, h].view(torch.uint8)[pages].view(F8).double().view(-1, block, c["dim"])
                    * st[x + "_scale"][pages, h].double().view(-1, 1, 1) for x in "kv")
            k, v = (x.reshape(-1, c["dim"])[:length] for x in (k, v))
            late = torch.ones(n, length, dtype=torch.bool, device=DEV).triu(length - n + 1)
            for i in range(h * G, h * G + G):
                s = (st["q"][first:first + n, i].double() @ k.T * st["scale"]).masked_fill(late, -math.inf)
                out[first:first + n, i] = torch.softmax(s, -1) @ v
        first += n
    return out


def _exact_append(st, c, x):
    new, lengths = _lengths(c)
    page, block = c["page"], c["block"]
    codes, scale = st[x + "_codes"].double(), st[x + "_scale"].double()
    table, first = st["table"].tolist(), 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        rows = st[x][first:first + n].double()
        first += n
        start, at = length - n, 0
        while at < n:
            position = start + at
            p, offset = table[b][position // page], position % page
            j, skip = offset // block, offset % block
            m = min(n - at, block - skip)
            part = rows[at:at + m].transpose(0, 1)                              # [HKV, m, D]
            top = part.abs().amax((1, 2))
            power = torch.ceil(torch.log2(top / F8_MAX)).clamp(TINY_EXP, BIG_EXP)
            now = torch.where(top > 0, 2.0 ** power, 2.0 ** TINY_EXP)
            if skip:
                now = torch.maximum(now, scale[p, :, j])
                # only rounded codes were kept of the earlier tokens
                codes[p, :, offset - skip:offset] *= (scale[p, :, j] / now)[:, None, None]
            codes[p, :, offset:offset + m] = part / now[:, None, None]
            scale[p, :, j] = now
            at += m
    return codes, scale


def _exact_norm(st, c):
    h = st["x"].double() + st["residual"].double()
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / c["width"] + NORM_EPS) * st["weight"].double()
    size = GROUP if c["grouped"] else c["width"]
    scale = torch.stack([p.abs().amax(-1) for p in y.split(size, dim=1)], 1).clamp(min=AMAX_FLOOR) / F8_MAX
    codes = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(y.split(size, dim=1))], 1)
    return {"residual": h, "codes": codes, "scale": scale if c["grouped"] else scale[:, 0]}


def exact(case, seed):
    st, c = prepare(case, seed), dict(case)
    if c["kind"] == "norm":
        return _exact_norm(st, c)
    if c["kind"] == "append":
        (kc, ks), (vc, vs) = _exact_append(st, c, "k"), _exact_append(st, c, "v")
        return {"k_codes": kc, "k_scale": ks, "v_codes": vc, "v_scale": vs}
    return _exact_attend(st, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    act = SIZE[c["act"]]
    if c["kind"] == "norm":
        N, W = c["rows"], c["width"]
        scales = N * -(-W // GROUP) if c["grouped"] else N
        return {"bytes": N * W * (3.0 * act + 1) + W * act + 4.0 * scales, "flops": 7.0 * N * W}
    new, lengths = _lengths(c)
    D, H, block = c["dim"], c["kv_heads"], c["block"]
    index = sum(4.0 * -(-n // c["page"]) + 8 for n in lengths)
    if c["kind"] == "append":
        blocks = sum((n - 1) // block - (n - m) // block + 1 for m, n in zip(new, lengths))
        return {"bytes": 2.0 * H * (sum(new) * D * (act + 1) + 4 * blocks) + index, "flops": 4.0 * H * sum(new) * D}
    cached = sum(2.0 * H * (n * D + 4 * -(-n // block)) for n in lengths)
    seen = sum(m * n - m * (m - 1) / 2 for m, n in zip(new, lengths))           # pairs of a query and a key it sees
    return {"bytes": cached + 2.0 * sum(new) * c["heads"] * D * act + index, "flops": seen * c["heads"] * (4.0 * D + 4)}
