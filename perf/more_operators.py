"""What a prompt's way through a hybrid model's layers is measured on: the gated delta rule over whole sequences, in
front of the slot pool's decode step, and the norm and rotation of queries and keys, in front of the key/value cache.

A case is a dict of plain values with a ``kind``:

* ``delta``  the recurrence of the slot-indexed step over every token of ragged sequences, from a floating-point state (or
  none) to a floating-point state: prompts, chunks of a prompt, a few tokens, one token;
* ``rotate``  RMS norm of every query and key head and the rotation by the token's position, or its positions on
  several axes.

``prepare`` makes the inputs on the GPU from the seed, ``run`` is one pass (plain torch, or with ``own`` the
framework's calls), ``exact`` the same in 64 bits, ``work`` the bytes and operations that it cannot do without.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
L2_EPS, NORM_EPS, SOFTPLUS_TOP = 1e-6, 1e-6, 20.0
CHUNK = 64                                                # of the plain form


def _delta(name, requests, tokens, key_heads=16, heads=32, dim=128, act="bf16", l2norm=True, initial=False, ragged=False):
    """``tokens``: of a request (of the longest one, where ragged)."""
    return dict(name=name, kind="delta", requests=requests, tokens=tokens, key_heads=key_heads, heads=heads, dim=dim, act=act,
                l2norm=l2norm, initial=initial, ragged=ragged)


def _rotate(name, tokens, heads=32, kv_heads=8, dim=128, rotary=128, axes=1, act="bf16", interleaved=False):
    return dict(name=name, kind="rotate", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, axes=axes, act=act,
                interleaved=interleaved)


def listed():
    return [
        # one user's short prompt, where the call's latency is what counts
        _delta("delta_prompt_77", 1, 77),
        # a serving batch that decodes from a floating-point state: one token for each of 64 requests
        _delta("delta_step_64", 64, 1, initial=True),
        # five speculated tokens of every request, checked at once
        _delta("delta_verify_5", 32, 5, initial=True),
        # whole prompts of eight requests, of all lengths, in one call
        _delta("delta_prompts_8", 8, 2000, ragged=True),
        # a chunk of one long prompt, behind what came before it
        _delta("delta_chunk_8192", 1, 8192, initial=True),
        # the largest prefill batch
        _delta("delta_prompts_16", 16, 4096),
        # narrow heads in fp32, keys normed by the caller
        _delta("delta_narrow_fp32", 4, 777, key_heads=4, heads=8, dim=64, act="fp32", l2norm=False),
        # a prompt of odd length in fp16
        _delta("delta_fp16_3001", 2, 3001, key_heads=8, act="fp16"),
        # an attention layer's queries and keys: one token, a decode batch of partly rotated heads, a prompt
        _rotate("rotate_1", 1),
        _rotate("rotate_256", 256, heads=16, kv_heads=2, rotary=32),
        _rotate("rotate_16384", 16384),
        # a prompt with pictures in it: positions in time, height and width
        _rotate("rotate_axes_5001", 5001, heads=16, kv_heads=16, axes=3, act="fp16"),
    ]


# ---------------------------------------------------------------------------
# sizes: a function of the case alone, so that work() knows them
# ---------------------------------------------------------------------------

def _lengths(c):
    """Tokens of every request: spread evenly over 1..tokens in an order of no pattern; the last one is the longest."""
    B, top = c["requests"], c["tokens"]
    if not c["ragged"]:
        return [top] * B
    part = [math.modf((i + 1) * 0.6180339887498949)[0] for i in range(B)]
    return [1 + int((top - 1) * p) for p in part[:-1]] + [top]


def _sections(c):
    """Frequencies of each axis: in time a quarter of them, the rest in equal parts."""
    half = c["rotary"] // 2
    if c["axes"] == 1:
        return [half]
    first = half // 4
    rest = (half - first) // (c["axes"] - 1)
    return [half - rest * (c["axes"] - 1)] + [rest] * (c["axes"] - 1)


def _positions_top(c):
    return 32768 if c["axes"] == 1 else 8192


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    act = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    kind = rng.choice(["step", "few", "prompt", "prompt", "prompts", "prompts", "rotate", "rotate", "rotate"])
    if kind == "rotate":
        dim, kv = rng.choice([64, 96, 128, 256]), rng.choice([1, 2, 4, 8, 16])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        return _rotate("", _log_int(rng, 1, 32768), kv * rng.choice([1, 2, 4, 8]), kv, dim, rotary, rng.choice([1, 1, 2, 3]), act,
                       rng.random() < 0.3)
    key_heads = rng.choice([1, 2, 4, 8, 16])
    more = dict(key_heads=key_heads, heads=key_heads * rng.choice([1, 2, 4]), dim=rng.choice([64, 128, 128]), act=act,
                l2norm=rng.random() < 0.8, initial=rng.random() < 0.5)
    if kind == "step":
        return _delta("", _log_int(rng, 1, 128), 1, **more)
    if kind == "few":
        return _delta("", _log_int(rng, 1, 64), rng.randrange(2, 17), ragged=rng.random() < 0.5, **more)
    if kind == "prompt":
        return _delta("", 1, _log_int(rng, 17, 16384), **more)
    return _delta("", rng.randrange(2, 33), _log_int(rng, 17, 4096), ragged=rng.random() < 0.7, **more)


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _draw_once(rng)
        w = work(c)
        padded = 0
        if c["kind"] == "delta":                        # what the plain form holds: padded sequences in 32 bits
            padded = 40 * c["requests"] * c["tokens"] * c["heads"] * c["dim"]
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and padded <= 24e9:
            del c["name"]
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(shape, g, sigma=1.0):
    return torch.empty(shape, device=DEV).normal_(0.0, sigma, generator=g)


def _uniform(shape, g, lo, hi):
    return torch.empty(shape, device=DEV).uniform_(lo, hi, generator=g)


def _prepare_delta(st, c, g):
    dt = DTYPES[c["act"]]
    B, H, HV, D = c["requests"], c["key_heads"], c["heads"], c["dim"]
    lengths = _lengths(c)
    N = sum(lengths)
    # queries, keys and values leave a short convolution through x * sigmoid(x): keys of neighbouring tokens are alike
    x = torch.nn.functional.silu(_normal((N, 2 * H * D + HV * D), g))
    if not c["l2norm"]:
        qk = x[:, :2 * H * D].view(N, 2 * H, D)
        qk /= qk.square().sum(-1, keepdim=True).add_(L2_EPS).sqrt_()
    st["mixed"] = x.to(dt)
    st["a"], st["b"] = _normal((N, HV), g).to(dt), _normal((N, HV), g).to(dt)
    # decays as models begin with: rates up to 16, steps of 0.001 to 0.1
    st["A_log"] = torch.log(_uniform((HV,), g, 1.0, 16.0))
    step = torch.exp(_uniform((HV,), g, math.log(1e-3), math.log(1e-1)))
    st["dt_bias"] = step + torch.log(-torch.expm1(-step))
    st["scale"] = D ** -0.5
    st["initial"] = _normal((B, HV, D, D), g, 0.1) if c["initial"] else None
    st["final"] = torch.zeros((B, HV, D, D), device=DEV)
    st["out"] = torch.zeros((N, HV, D), dtype=dt, device=DEV)
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)


def _prepare_rotate(st, c, g):
    dt = DTYPES[c["act"]]
    N, HQ, HK, D, R, A = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"], c["axes"]
    # the projection's rows: queries, keys, and the values that the call leaves alone
    qkv = _normal((N, HQ + 2 * HK, D), g, 2.0).to(dt)
    st["q"], st["k"], st["v"] = qkv.split([HQ, HK, HK], dim=1)
    st["q_weight"] = (1.0 + _normal((D,), g, 0.1)).to(dt)
    st["k_weight"] = (1.0 + _normal((D,), g, 0.1)).to(dt)
    top = _positions_top(c)
    freq = 1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
    angle = torch.arange(top, dtype=torch.float64, device=DEV)[:, None] * freq
    st["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    if A == 1:                                          # a chunk that begins somewhere in its prompt, or requests' own places
        first = torch.randint(0, top, (1,), device=DEV, generator=g) if N > 512 else torch.randint(0, top, (N,), device=DEV, generator=g)
        st["positions"] = (first + torch.arange(N, device=DEV)) % top
    else:
        st["positions"] = torch.randint(0, top, (A, N), device=DEV, generator=g)
    st["q_out"] = torch.zeros((N, HQ, D), dtype=dt, device=DEV)
    st["k_out"] = torch.zeros((N, HK, D), dtype=dt, device=DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    st = {"case": c}
    (_prepare_delta if c["kind"] == "delta" else _prepare_rotate)(st, c, g)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _padded(st, c, tokens):
    """Where each request's tokens lie in the call's rows, [B, tokens], and which of them there are."""
    t = torch.arange(tokens, device=DEV)
    first, count = st["starts"][:-1].long(), st["starts"].long().diff()
    there = t < count[:, None]
    return torch.where(there, first[:, None] + t, 0), there


def _plain_delta(st, c):
    """In chunks: with G the running sum of the log decays within a chunk, S the state at its start and
    u_i = beta_i (v_i - exp(G_i) k_i S - sum_{j<i} exp(G_i - G_j) (k_i . k_j) u_j) the rows that a chunk adds to it,
    o_i = exp(G_i) q_i S + sum_{j<=i} exp(G_i - G_j) (q_i . k_j) u_j."""
    B, H, HV, D, C = c["requests"], c["key_heads"], c["heads"], c["dim"], CHUNK
    n = -(-c["tokens"] // C)
    place, there = _padded(st, c, n * C)
    x = st["mixed"].float()

    def heads(lo, count):                               # [B, count, n, C, D], zeros where there is no token
        y = x[:, lo:lo + count * D].view(-1, count, D)[place]
        y = torch.where(there[:, :, None, None], y, 0.0)
        return y.view(B, n, C, count, D).permute(0, 3, 1, 2, 4)

    q, k, v = heads(0, H), heads(H * D, H), heads(2 * H * D, HV)
    if c["l2norm"]:
        q, k = (y / torch.sqrt(y.square().sum(-1, keepdim=True) + L2_EPS) for y in (q, k))
    q = (q * st["scale"]).repeat_interleave(HV // H, dim=1)
    k = k.repeat_interleave(HV // H, dim=1)
    z = st["a"].double() + st["dt_bias"].double()
    g = -torch.exp(st["A_log"].double()) * torch.where(z <= SOFTPLUS_TOP, torch.log1p(torch.exp(z)), z)
    g, beta = (torch.where(there[..., None], y[place], 0.0).view(B, n, C, HV).permute(0, 3, 1, 2)
               for y in (g, 1.0 / (1.0 + torch.exp(-st["b"].float()))))
    G = g.cumsum(-1)                                    # [B, HV, n, C], in 64 bits: the decays are of its differences
    i = torch.arange(C, device=DEV)
    decay = torch.where(i[:, None] >= i, (G[..., :, None] - G[..., None, :]).clamp(max=0.0).exp(), 0.0).float()
    less = torch.matmul(k, k.transpose(-1, -2)) * decay * beta[..., None]
    less = torch.where(i[:, None] > i, less, 0.0)
    inverse = torch.eye(C, device=DEV).expand_as(less).contiguous()
    for r in range(1, C):
        inverse[..., r, :r] = -torch.matmul(less[..., r:r + 1, :r], inverse[..., :r, :r])[..., 0, :]
    own_rows = torch.matmul(inverse, v * beta[..., None])
    of_state = torch.matmul(inverse, k * (beta * G.exp().float())[..., None])
    among = torch.matmul(q, k.transpose(-1, -2)) * decay
    q = q * G.exp().float()[..., None]
    k = k * (G[..., -1:] - G).exp().float()[..., None]
    last = G[..., -1].exp().float()
    S = torch.zeros(B, HV, D, D, device=DEV) if st["initial"] is None else st["initial"].transpose(-1, -2)
    o = torch.empty(B, HV, n, C, D, device=DEV)
    for j in range(n):
        u = own_rows[:, :, j] - torch.matmul(of_state[:, :, j], S)
        o[:, :, j] = torch.matmul(q[:, :, j], S) + torch.matmul(among[:, :, j], u)
        S = S * last[:, :, j, None, None] + torch.matmul(k[:, :, j].transpose(-1, -2), u)
    st["out"][place[there]] = o.permute(0, 2, 3, 1, 4).reshape(B, n * C, HV, D)[there].to(st["out"].dtype)
    st["final"].copy_(S.transpose(-1, -2))
    return {"out": st["out"], "state": st["final"]}


def _angles(st, c):
    """cos and sin of every token's angles, [N, 1, rotary / 2]."""
    half, table, positions = c["rotary"] // 2, st["table"], st["positions"]
    if c["axes"] == 1:
        rows = table[positions]
        cos, sin = rows[:, :half], rows[:, half:]
    else:
        axis = torch.arange(c["axes"], device=DEV).repeat_interleave(torch.tensor(_sections(c), device=DEV))
        of = positions[axis].T                          # [N, half]: each frequency's own position
        j = torch.arange(half, device=DEV)
        cos, sin = table[of, j], table[of, half + j]
    return cos[:, None], sin[:, None]


def _plain_rotate(st, c):
    R = c["rotary"]
    cos, sin = _angles(st, c)
    for x, weight, out in ((st["q"], st["q_weight"], st["q_out"]), (st["k"], st["k_weight"], st["k_out"])):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + NORM_EPS) * weight.float()
        one, two = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        first, second = y[..., one], y[..., two]
        out[..., one] = (first * cos - second * sin).to(out.dtype)
        out[..., two] = (second * cos + first * sin).to(out.dtype)
        out[..., R:] = y[..., R:].to(out.dtype)
    return {"q": st["q_out"], "k": st["k_out"]}


def run(state):
    st, c = state, state["case"]
    if c["kind"] == "rotate":
        if not own:
            return _plain_rotate(st, c)
        from carrykernel_b200.vllm_integration import qk_norm_rope
        qk_norm_rope.qk_norm_rope(st["q"], st["k"], st["q_weight"], st["k_weight"], st["table"], st["positions"], NORM_EPS,
                                  q_out=st["q_out"], k_out=st["k_out"], sections=None if c["axes"] == 1 else _sections(c),
                                  interleaved=c["interleaved"])
        return {"q": st["q_out"], "k": st["k_out"]}
    if not own:
        return _plain_delta(st, c)
    from carrykernel_b200.vllm_integration import packed_prefill
    packed_prefill.gated_delta_rule_packed_prefill(st["mixed"], st["a"], st["b"], st["A_log"], st["dt_bias"], st["scale"], st["out"],
                                                   st["final"], initial_state=st["initial"], query_start=st["starts"],
                                                   max_query_len=c["tokens"], use_qk_l2norm_in_kernel=c["l2norm"])
    return {"out": st["out"], "state": st["final"]}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits: the recurrence token by token, the rotation as complex numbers
# ---------------------------------------------------------------------------

def _exact_delta(st, c):
    B, H, HV, D = c["requests"], c["key_heads"], c["heads"], c["dim"]
    group = HV // H
    lengths = _lengths(c)
    x = st["mixed"]
    alpha = torch.exp(-torch.exp(st["A_log"].double()) * torch.nn.functional.softplus(st["a"].double() + st["dt_bias"].double()))
    beta = torch.sigmoid(st["b"].double())
    S = torch.zeros(B, HV, D, D, dtype=torch.float64, device=DEV)               # [V, K]
    if st["initial"] is not None:
        S.copy_(st["initial"])
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV)
    order = sorted(range(B), key=lambda b: -lengths[b])                         # the longest first: those still there are a prefix
    S = S[order]
    first = st["starts"][order].long() if B > 1 else st["starts"][:1].long()
    live = B
    for t in range(c["tokens"]):
        while lengths[order[live - 1]] <= t:
            live -= 1
        rows = first[:live] + t
        y = x[rows].double()
        q, k, v = y[:, :H * D].view(live, H, D), y[:, H * D:2 * H * D].view(live, H, D), y[:, 2 * H * D:].view(live, HV, D)
        if c["l2norm"]:
            q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + L2_EPS)
            k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + L2_EPS)
        q, k = (z[:, :, None].expand(live, H, group, D).reshape(live, HV, D, 1) for z in (q * st["scale"], k))
        T = S[:live]
        T *= alpha[rows][..., None, None]
        u = beta[rows][..., None, None] * (v[..., None] - T @ k)
        T += u * k.transpose(-1, -2)
        out[rows] = (T @ q)[..., 0]
    final = torch.empty_like(S)
    final[order] = S
    return {"out": out, "state": final}


def _exact_rotate(st, c):
    half, R = c["rotary"] // 2, c["rotary"]
    table = st["table"].double()
    turn = torch.complex(table[:, :half], table[:, half:])
    positions = st["positions"].view(c["axes"], -1)
    parts, at = [], 0
    for axis, size in enumerate(_sections(c)):
        parts.append(turn[positions[axis], at:at + size])
        at += size
    turn = torch.cat(parts, 1)[:, None]
    found = {}
    for name in "qk":
        y = st[name].double()
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / c["dim"] + NORM_EPS) * st[name + "_weight"].double()
        pairs = y[..., :R].unflatten(-1, (half, 2)) if c["interleaved"] else y[..., :R].unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
        z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        found[name] = torch.cat([z, y[..., R:]], -1)
    return found


def exact(case, seed):
    st, c = prepare(case, seed), dict(case)
    return _exact_delta(st, c) if c["kind"] == "delta" else _exact_rotate(st, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    act, D = SIZE[c["act"]], c["dim"]
    if c["kind"] == "rotate":
        N, rows = c["tokens"], c["tokens"] * (c["heads"] + c["kv_heads"])
        table = 4.0 * c["rotary"] * min(N, _positions_top(c))
        return {"bytes": 2.0 * rows * D * act + 2.0 * D * act + table + 8.0 * N * c["axes"], "flops": rows * (4.0 * D + 3.0 * c["rotary"])}
    N, B, H, HV = sum(_lengths(c)), c["requests"], c["key_heads"], c["heads"]
    states = 4.0 * B * HV * D * D * (2 if c["initial"] else 1)
    # decay, what the state holds for the key, the row added, what it holds for the query
    return {"bytes": N * act * (2.0 * H * D + 2.0 * HV * D + 2.0 * HV) + states + 8.0 * HV + 4.0 * (B + 1), "flops": 7.0 * N * HV * D * D}
