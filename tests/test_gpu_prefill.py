"""The gated delta rule over whole sequences against the recurrence in 64 bits."""

import math

import pytest
import torch

from carrykernel_b200 import _lib
from carrykernel_b200.vllm_integration import packed_prefill as pp
from oracle import prompt_oracle as orc

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"
TOKEN_BY_TOKEN, IN_CHUNKS = 13, 14


def make(lengths, H, HV, D, dtype, initial=False, l2norm=True, seed=0, gates=None, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)
    new = lambda f, *shape: f(*shape, generator=g, device=device)  # noqa: E731
    N = sum(lengths)
    x = torch.nn.functional.silu(new(torch.randn, N, 2 * H * D + HV * D))
    if not l2norm:
        qk = x[:, :2 * H * D].view(N, 2 * H, D)
        qk /= qk.norm(dim=-1, keepdim=True) + 1e-3
    c = dict(mixed_qkv=x.to(dtype), a=new(torch.randn, N, HV).to(gates or dtype), b=new(torch.randn, N, HV).to(gates or dtype),
             A_log=torch.log(1 + 15 * new(torch.rand, HV)), dt_bias=new(torch.randn, HV) - 4, scale=D ** -0.5)
    state = new(torch.randn, len(lengths), HV, D, D) if initial else None
    return c, state


def starts(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)


def run(c, state, lengths, HV, D, l2norm=True, out_dtype=None, most=None, **more):
    N = sum(lengths)
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
    out = torch.full((N, HV, D), float("nan"), dtype=out_dtype or c["mixed_qkv"].dtype, device=DEV)
    final = torch.full((len(lengths), HV, D, D), float("nan"), device=DEV)
    pp.gated_delta_rule_packed_prefill(**dev, out=out, final_state=final, initial_state=None if state is None else state.to(DEV),
                                       query_start=starts(lengths).to(DEV), max_query_len=max(lengths) if most is None else most,
                                       use_qk_l2norm_in_kernel=l2norm, **more)
    return out, final


def bounds(out, wanted, in_chunks, fp32_operands):
    """What outputs and states may be off by.

    A token's own arithmetic is fp32: a product of the state with a key is a sum of 128 numbers (at most 32 roundings one after the
    other token by token; on the tensor cores 48 steps of sixteen, each of which may lose 2^-23 of the largest), key and query
    norms, gates (an exponential of an exponential and a logarithm: 8 roundings relative to the log decay) and a few products: 64
    roundings of 2^-24 token by token, 256 in chunks.  In chunks T comes as two bf16 numbers, 2^-18 off (three, 2^-26, for fp32
    operands, where what T is solved from counts: 16 roundings of 2^-24), and P T is a sum of products of such, 2^-16.  Then the rounding
    to the output's type.  Below 2^-126 fp32 has no relative precision, and below 2^-149 nothing (sigmoid(-200) is 2^-288, and a decay
    by exp(-100) is good to 2^-150): each factor and each number may lose 2^-126 of what it multiplies or is added to."""
    want_out, want_state, out_weight, weight = wanted
    floor = 2.0 ** -126
    own = (256 if in_chunks else 64) * 2.0 ** -24
    of_t = 0.0 if not in_chunks else 2.0 ** -20 if fp32_operands else 2.0 ** -18 + 2.0 ** -20
    state = own * weight[..., 0] + of_t * weight[..., 1] + floor * (1 + weight[..., 0])
    half_step = torch.finfo(out.dtype).eps / 2
    value = own * out_weight[..., 0] + 4 * of_t * out_weight[..., 1] + floor * (1 + out_weight[..., 0])
    return (1 + half_step) * value + half_step * want_out.abs() + torch.finfo(out.dtype).smallest_normal * half_step, state


def check(got, c, state, lengths, H, D, l2norm=True, in_chunks=None, rows=None, requests=None):
    out, final = got
    wanted = orc.delta_rule(**{k: v for k, v in c.items() if k != "mixed_qkv"}, mixed=c["mixed_qkv"], H=H, D=D, lengths=lengths, initial=state,
                            l2norm=l2norm)
    out_bound, state_bound = bounds(out, wanted, in_chunks, c["mixed_qkv"].dtype == F32)
    off, off_state = (out.cpu().double() - wanted[0]).abs(), (final.cpu().double() - wanted[1]).abs()
    rows, requests = slice(None) if rows is None else rows, slice(None) if requests is None else requests
    assert (off <= out_bound)[rows].all(), f"outputs off by up to {(off / out_bound)[rows].max():.2f} of the bound"
    assert (off_state <= state_bound)[requests].all(), f"states off by up to {(off_state / state_bound)[requests].max():.2f} of the bound"
    # In the mean: a split's error is as good as random, at most 2^-18 of T's entry (2^-22 with what counts for fp32 operands), and
    # what a token's own arithmetic loses is 16 roundings.
    weight = wanted[3][requests]
    mean = 2.0 ** -20 * weight[..., 0] + (2.0 ** -22 if c["mixed_qkv"].dtype == F32 else 2.0 ** -18) * weight[..., 2] + 2.0 ** -126
    assert off_state[requests].norm() <= mean.expand_as(off_state[requests]).norm() / D ** 0.5


def goes_in_chunks(lengths, dtype, many=False):
    """The rule by which a call of so many tokens a request goes in chunks; `many`: heads, more than a few hundred."""
    return max(lengths) > (96 if dtype == F32 else 40 if many else 64)


FEW = [[1], [3], [1, 1, 1], [5, 0, 2], [33], [64], [1, 64, 17]]
MANY = [[65], [128], [1, 0, 64, 65, 3], [97, 0, 64, 65, 3], [200, 77], [191, 1]]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", FEW + MANY, ids=str)
def test_against_recurrence(dtype, D, lengths):
    H, HV = (2, 4) if D == 64 else (1, 3)
    initial = len(lengths) % 2 == 1
    c, state = make(lengths, H, HV, D, dtype, initial)
    got = run(c, state, lengths, HV, D)
    in_chunks = goes_in_chunks(lengths, dtype)
    assert _lib.load_library().carry_gdn_last_kernel() == (IN_CHUNKS if in_chunks else TOKEN_BY_TOKEN)
    check(got, c, state, lengths, H, D, in_chunks=in_chunks)


@pytest.mark.parametrize("lengths", [[40], [130]], ids=str)
@pytest.mark.parametrize("H,HV", [(1, 1), (1, 8), (5, 5), (4, 8)])
def test_head_maps_and_unnormed_keys(lengths, H, HV):
    for dtype, out_dtype, gates in ((BF16, F32, F32), (F16, BF16, BF16), (F32, F16, F16)):
        c, state = make(lengths, H, HV, 64, dtype, True, l2norm=False, seed=H, gates=gates)
        got = run(c, state, lengths, HV, 64, l2norm=False, out_dtype=out_dtype)
        check(got, c, state, lengths, H, 64, l2norm=False, in_chunks=goes_in_chunks(lengths, dtype))


@pytest.mark.parametrize("lengths", [[3, 20], [100, 70]], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_alignment(lengths, dtype):
    """Rows of wider tensors that begin off the grid, states apart from one another, in place; what lies beside them stays."""
    H, HV, D = 1, 2, 64
    c, state = make(lengths, H, HV, D, dtype, True)
    plain = run(c, state, lengths, HV, D)
    N, width = c["mixed_qkv"].shape
    wide = torch.full((N, width + 3), 9.0, dtype=dtype, device=DEV)
    wide[:, 1:1 + width] = c["mixed_qkv"].to(DEV)
    gates = torch.full((N, 2 * HV + 1), 9.0, dtype=dtype, device=DEV)
    gates[:, :HV], gates[:, HV + 1:] = c["a"].to(DEV), c["b"].to(DEV)
    outs = torch.full((N + 2, HV * D + 7), 9.0, dtype=dtype, device=DEV)
    states = torch.full((4, HV, D, D), 9.0, device=DEV)
    states[::2] = state.to(DEV)
    out = outs[1:-1, 3:3 + HV * D].unflatten(1, (HV, D))
    pp.gated_delta_rule_packed_prefill(wide[:, 1:1 + width], gates[:, :HV], gates[:, HV + 1:], c["A_log"].to(DEV), c["dt_bias"].to(DEV), c["scale"],
                                       out, states[::2], initial_state=states[::2], query_start=starts(lengths).to(DEV),
                                       max_query_len=max(lengths), use_qk_l2norm_in_kernel=True)
    assert torch.equal(out, plain[0]) and torch.equal(states[::2], plain[1])
    assert (states[1::2] == 9).all() and (outs[[0, -1]] == 9).all() and (outs[:, :3] == 9).all() and (outs[:, 3 + HV * D:] == 9).all()


@pytest.mark.parametrize("most", [64, 200])
def test_rows_outside_of_the_requests(most):
    """Rows ahead of the first request and behind the last one are left as they were, whatever they hold."""
    H, HV, D, lengths = 1, 2, 128, [40, 90 if most > 64 else 30]
    c, state = make([7, *lengths, 70], H, HV, D, BF16, True)
    for x in (c["mixed_qkv"], c["a"], c["b"]):
        x[:7], x[7 + sum(lengths):] = float("nan"), float("inf")
    N = c["mixed_qkv"].shape[0]
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
    out, final = torch.full((N, HV, D), 9.0, dtype=BF16, device=DEV), torch.empty(2, HV, D, D, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    pp.gated_delta_rule_packed_prefill(**dev, out=out, final_state=final, initial_state=state[1:3].to(DEV), query_start=7 + starts(lengths).to(DEV),
                                       max_query_len=most, use_qk_l2norm_in_kernel=True, status=status)
    assert status.item() == 0 and (out[:7] == 9).all() and (out[7 + sum(lengths):] == 9).all()
    inner = {k: v[7:7 + sum(lengths)] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}
    check((out[7:7 + sum(lengths)], final), inner, state[1:3], lengths, H, D, in_chunks=most > 64)


@pytest.mark.parametrize("n", [20, 150])
def test_a_request_with_numbers_that_are_not_finite_spoils_no_other(n):
    H, HV, D, lengths = 2, 2, 64, [n, n, n]
    c, state = make(lengths, H, HV, D, BF16, True)
    clean = run(c, state, lengths, HV, D)
    c["mixed_qkv"][n + 5:n + 9] = float("nan")
    c["a"][n + 3], state[1, 0, 0, 0] = float("nan"), float("inf")
    got = run(c, state, lengths, HV, D)
    for r in (slice(0, n), slice(2 * n, None)):
        assert torch.equal(got[0][r], clean[0][r])
    assert torch.equal(got[1][::2], clean[1][::2]) and got[1][1].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,at", [(40, 17), (200, 3), (200, 70), (130, 127), (193, 192)])
def test_numbers_that_are_not_finite_reach_no_token_ahead_of_them(n, at, dtype):
    """A value spoils its column of the state from its token on, a key or a gate the heads that read it, a query its token's output."""
    H, HV, D = 2, 4, 64
    c, state = make([n], H, HV, D, dtype, True)
    clean = run(c, state, [n], HV, D)
    for where, bad in (("value", float("nan")), ("value", float("inf")), ("key", float("nan")), ("key", -float("inf")), ("query", float("nan")),
                       ("a", float("nan")), ("b", float("nan"))):
        d = {k: v.clone() if torch.is_tensor(v) else v for k, v in c.items()}
        heads, columns, rows = slice(2, 4), slice(None), slice(at, None)       # what it may reach: heads 2 and 3 read key head 1
        if where == "value":
            d["mixed_qkv"][at, 2 * H * D + 2 * D + 5] = bad
            heads, columns = slice(2, 3), slice(5, 6)
        elif where == "key":
            d["mixed_qkv"][at, H * D + D + 7] = bad
        elif where == "query":
            d["mixed_qkv"][at, D + 7] = bad
            rows = slice(at, at + 1)
        else:
            d[where][at, 2] = bad
            heads = slice(2, 3)
        out, final = run(d, state, [n], HV, D)
        reached = torch.zeros_like(out, dtype=torch.bool)
        reached[rows, heads, columns] = True
        assert torch.equal(out[~reached], clean[0][~reached]), where
        assert not out[reached].isfinite().any() or (where == "value" and bad == float("inf")), where
        if where != "query":
            spoilt = torch.zeros_like(final, dtype=torch.bool)
            spoilt[:, heads, columns] = True
            assert torch.equal(final[~spoilt], clean[1][~spoilt]) and not final[spoilt].isfinite().any(), where
        else:
            assert torch.equal(final, clean[1])


def test_bad_row_ranges_are_flagged_and_skipped():
    H, HV, D = 1, 1, 64
    c, _ = make([100], H, HV, D, BF16)
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
    for start, most in (([0, 70, 250], 90), ([-5, 20, 60], 64), ([0, 100, 40], 100), ([0, 90, 100], 70), ([0, 20, 100], 40)):
        out, final = torch.full((100, HV, D), 9.0, dtype=BF16, device=DEV), torch.empty(2, HV, D, D, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        pp.gated_delta_rule_packed_prefill(**dev, out=out, final_state=final, query_start=torch.tensor(start, dtype=torch.int32, device=DEV),
                                           max_query_len=most, use_qk_l2norm_in_kernel=True, status=status)
        assert status.item() == _lib.STATUS_BAD_RANGE, (start, most)
        assert final.isfinite().all() and out.isfinite().all()
        with pytest.raises(RuntimeError):
            _lib.raise_for_status(status)


@pytest.mark.parametrize("n", [30, 100])
def test_row_ranges_at_the_ends_of_32_bits(n):
    """Starts that are no rows of the call at all: nothing outside of it is read or written, and what has rows is done."""
    least, most = -2 ** 31, 2 ** 31 - 1
    H, HV, D = 1, 2, 64
    c, _ = make([n + 9], H, HV, D, BF16)
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
    alone = run({k: v[:n] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}, None, [n], HV, D)
    for start in ([0, n, least], [0, n, most], [0, n, least, most], [0, n, least, least]):
        B = len(start) - 1
        guarded = torch.full((n + 9 + 64, HV, D), 9.0, dtype=BF16, device=DEV)
        out, final = guarded[32:32 + n + 9], torch.empty(B, HV, D, D, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        pp.gated_delta_rule_packed_prefill(**dev, out=out, final_state=final, query_start=torch.tensor(start, dtype=torch.int32, device=DEV),
                                           max_query_len=n, use_qk_l2norm_in_kernel=True, status=status)
        assert status.item() == _lib.STATUS_BAD_RANGE, start
        assert (guarded[:32] == 9).all() and (guarded[32 + n + 9:] == 9).all() and torch.equal(final[:1], alone[1])
        if most not in start:
            assert torch.equal(out[:n], alone[0]) and (out[n:] == 9).all() and (final[1:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_prompt_in_parts_is_the_prompt(dtype):
    """Handing the state on at any token, from any of the two ways of working to the other, is within the bounds of one call."""
    H, HV, D, lengths = 1, 2, 128, [230]
    c, state = make(lengths, H, HV, D, dtype, True)
    outs, now, at = [], state.to(DEV), 0
    for n in (1, 70, 64, 30, 65):
        part = {k: v[at:at + n] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}
        out, now = run(part, now, [n], HV, D)
        outs.append(out)
        at += n
    check((torch.cat(outs), now), c, state, lengths, H, D, in_chunks=True)


def test_many_heads_go_in_chunks_sooner():
    for n, kernel in ((40, TOKEN_BY_TOKEN), (41, IN_CHUNKS)):
        c, state = make([n] * 40, 16, 32, 64, BF16, True)
        got = run(c, state, [n] * 40, 32, 64)
        assert _lib.load_library().carry_gdn_last_kernel() == kernel
        part = {k: v[:n] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}
        check((got[0][:n], got[1][:1]), part, state[:1], [n], 16, 64, in_chunks=kernel == IN_CHUNKS)


def test_launches_that_share_the_workspace_out():
    """A call too large for the workspace's bound is cut by chunks, or by requests: the same numbers as alone."""
    for D, H, HV, lengths in ((128, 32, 64, [9000, 64, 9500, 4097]), (64, 4, 64, [65] * 300 + [129])):
        c, state = make(lengths, H, HV, D, BF16, True, device=DEV)
        need = pp.prefill_workspace_bytes(c["mixed_qkv"], state, starts(lengths).to(DEV), max(lengths))
        chunks = sum(-(-n // 64) for n in lengths)
        assert need < chunks * (H * D * 256 + HV * 32768)          # it does not hold every chunk at once
        out, final = run(c, state, lengths, HV, D)
        for i in range(0, len(lengths), max(1, len(lengths) // 4)):
            rows = slice(sum(lengths[:i]), sum(lengths[:i + 1]))
            part = {k: v[rows] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}
            alone = run(part, state[i:i + 1], lengths[i:i + 1], HV, D)
            if lengths[i] > 64:
                assert torch.equal(out[rows], alone[0]) and torch.equal(final[i:i + 1], alone[1])


def test_extreme_gates():
    """Decays of 0 and 1, write strengths of 0 and 1, and products of decays far below fp32."""
    for lengths in ([30], [140]):
        H, HV, D = 1, 4, 64
        c, state = make(lengths, H, HV, D, BF16, True, gates=F32)
        n = sum(lengths)
        c["A_log"] = torch.tensor([-30.0, 5.0, 0.0, 60.0])
        c["dt_bias"] = torch.zeros(HV)
        c["b"][:, 0], c["b"][n // 2:, 1], c["b"][:, 2] = 100.0, -200.0, torch.where(torch.arange(n) % 2 == 0, 90.0, -90.0)
        c["a"][:, 2] = torch.where(torch.arange(n) % 7 == 0, 300.0, -300.0)
        got = run(c, state, lengths, HV, D)
        check(got, c, state, lengths, H, D, in_chunks=n > 64)


def test_alike_keys_and_zero_rows():
    """A chunk whose keys are all one direction (the triangular system at its fullest), and tokens of zeros."""
    for lengths in ([30], [150]):
        H, HV, D = 1, 2, 128
        c, state = make(lengths, H, HV, D, BF16, True)
        x = c["mixed_qkv"]
        x[:, D:2 * D] = x[0, D:2 * D]
        x[3], x[100:105] = 0.0, 0.0
        c["a"].fill_(-30.0)
        c["b"].fill_(3.0)
        got = run(c, state, lengths, HV, D)
        check(got, c, state, lengths, H, D, in_chunks=max(lengths) > 64)


@pytest.mark.parametrize("dtype,D,H,HV,lengths", [(F32, 64, 2, 4, [97]), (BF16, 128, 8, 16, [300, 77, 64, 500]), (F32, 128, 8, 16, [300, 77, 64, 500]),
                                                  (F16, 128, 16, 32, [130] * 20), (BF16, 64, 1, 2, [700]), (BF16, 128, 16, 32, [1000, 1, 90]),
                                                  (F16, 128, 16, 32, [1000, 1, 90]), (F32, 64, 16, 32, [500, 90, 200])])
def test_repeated_calls_give_the_same_numbers(dtype, D, H, HV, lengths):
    """Warps and copies that meet at other times: every call's numbers are the first one's."""
    c, state = make(lengths, H, HV, D, dtype, True)
    first = run(c, state, lengths, HV, D)
    for _ in range(40):
        again = run(c, state, lengths, HV, D)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_no_rows_at_all():
    state = torch.randn(2, 3, 64, 64, device=DEV)
    for initial, want in ((None, torch.zeros_like(state)), (state, state)):
        final = torch.full_like(state, 9.0)
        pp.gated_delta_rule_packed_prefill(torch.empty(0, 5 * 64, dtype=BF16, device=DEV), torch.empty(0, 3, device=DEV), torch.empty(0, 3, device=DEV),
                                           torch.zeros(3, device=DEV), torch.zeros(3, device=DEV), 1.0, torch.empty(0, 3, 64, dtype=BF16, device=DEV),
                                           final, initial_state=initial)
        assert torch.equal(final, want)


@pytest.mark.parametrize("n", [16, 150])
def test_captured_graphs_that_share_a_workspace(n):
    H, HV, D = 2, 4, 128
    cases = [make([n, n], H, HV, D, BF16, True, seed=s) for s in (1, 2)]
    need = pp.prefill_workspace_bytes(cases[0][0]["mixed_qkv"].to(DEV), cases[0][1].to(DEV))
    assert (need > 0) == (n > 64)
    work = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    graphs = []
    for c, state in cases:
        dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
        out, final, first = torch.zeros(2 * n, HV, D, dtype=BF16, device=DEV), torch.zeros(2, HV, D, D, device=DEV), state.to(DEV)
        call = lambda: pp.gated_delta_rule_packed_prefill(**dev, out=out, final_state=final, initial_state=first, use_qk_l2norm_in_kernel=True, workspace=work)  # noqa: E731,B023
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        out.zero_(), final.zero_()
        graphs.append((graph, out, final, dev, first))                             # a graph does not keep its inputs
    for _ in range(2):
        for graph, *_ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (c, state), (_, out, final, *_) in zip(cases, graphs):
        alone = run(c, state, [n, n], HV, D)
        assert torch.equal(out, alone[0]) and torch.equal(final, alone[1])


def test_a_workspace_that_is_too_small_is_refused():
    c, _ = make([100], 1, 1, 64, BF16)
    with pytest.raises(ValueError):
        run(c, None, [100], 1, 64, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        run(c, None, [100], 1, 64, workspace=torch.empty(1 << 24, dtype=torch.uint8, device=DEV)[8:])


def test_prompt_then_decode_on_the_slot_pool():
    """A prompt, its state into the requests' slots, and decoded tokens from there: near the recurrence on the unquantized state."""
    from carrykernel_b200.vllm_integration import quantized_packed_decode as qpd
    from carrykernel_b200.vllm_integration.state_pool import load_state, store_state
    H, HV, D, lengths, steps = 2, 4, 128, [100, 131], 4
    c, _ = make([n + steps for n in lengths], H, HV, D, BF16)
    c["A_log"], c["dt_bias"] = torch.full((HV,), math.log(0.1)), torch.zeros(HV)
    first = starts([n + steps for n in lengths])
    pick = lambda lo, hi: torch.cat([torch.arange(first[i] + lo(n), first[i] + hi(n)) for i, n in enumerate(lengths)])  # noqa: E731
    prompt = {k: v[pick(lambda n: 0, lambda n: n)] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}
    out, final = run(prompt, None, lengths, HV, D)
    pool = qpd.init_quantized_state(4, HV, D, D, DEV, resid_fmt=qpd.RESID_INT8)
    slots = torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    store_state(final, pool, slots, keep_error=True)
    back = load_state(pool, slots)
    assert (back - final).norm() <= 1e-3 * final.norm()          # int8 codes and an int8 residual
    want = orc.delta_rule(**{k: v for k, v in c.items() if k != "mixed_qkv"}, mixed=c["mixed_qkv"], H=H, D=D, lengths=[n + steps for n in lengths])[0]
    for t in range(steps):
        rows = torch.tensor([first[i] + n + t for i, n in enumerate(lengths)])
        got = torch.empty(2, 1, HV, D, dtype=BF16, device=DEV)
        qpd.quantized_gated_delta_rule_packed_decode(c["mixed_qkv"][rows].to(DEV), c["a"][rows].to(DEV), c["b"][rows].to(DEV), c["A_log"].to(DEV),
                                                     c["dt_bias"].to(DEV), c["scale"], *pool, got, slots, use_qk_l2norm_in_kernel=True,
                                                     resid_fmt=qpd.RESID_INT8)
        # rows of int8 codes: half a step of 127 against a row's largest number in each of `steps` tokens, and the output's rounding
        assert (got[:, 0].cpu().double() - want[rows]).norm() <= (steps / 127 + 2 ** -8) * want[rows].norm()


@pytest.mark.parametrize("lengths", [[20, 7], [200, 90, 130]], ids=str)
def test_two_streams_at_once_and_a_state_for_all(lengths):
    """Calls side by side, each with the workspace that it allocates; an initial state that is one tensor for all requests."""
    H, HV, D, B = 4, 8, 128, len(lengths)
    cases = [make(lengths, H, HV, D, BF16, True, seed=s) for s in (1, 2)]
    first = [state[:1].to(DEV).expand(B, -1, -1, -1) for _, state in cases]
    alone = [run(c, state[:1].expand(B, -1, -1, -1).clone(), lengths, HV, D) for c, state in cases]
    on = [{k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()} for c, _ in cases]
    start = starts(lengths).to(DEV)
    results = [(torch.zeros_like(alone[i][0]), torch.zeros_like(alone[i][1])) for i in (0, 1) for _ in range(8)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for n in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                out, final = results[8 * i + n]
                pp.gated_delta_rule_packed_prefill(**on[i], out=out, final_state=final, initial_state=first[i], query_start=start,
                                                   max_query_len=max(lengths), use_qk_l2norm_in_kernel=True)
    torch.cuda.synchronize()
    for j, (out, final) in enumerate(results):
        assert torch.equal(out, alone[j // 8][0]) and torch.equal(final, alone[j // 8][1]), j


@pytest.mark.parametrize("lengths", [[35, 34, 1], [5, 65, 0]], ids=str)
def test_offsets_beyond_32_bits(lengths):
    """Rows, outputs and states that lie more than 2^31 numbers apart."""
    H, HV, D, N, B = 1, 2, 64, sum(lengths), len(lengths)
    c, state = make(lengths, H, HV, D, BF16, True)
    alone = run(c, state, lengths, HV, D)
    stride, state_stride = 2 ** 25, 2 ** 30 + 4
    buffer = torch.empty(N * stride, dtype=BF16, device=DEV)
    width = c["mixed_qkv"].shape[1]
    mixed, out = buffer.as_strided((N, width), (stride, 1)), buffer.as_strided((N, HV, D), (stride, D, 1), 4096)
    mixed.copy_(c["mixed_qkv"])
    states = torch.empty(2 * state_stride + HV * D * D, device=DEV).as_strided((B, HV, D, D), (state_stride, D * D, D, 1))
    states.copy_(state)
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items() if k != "mixed_qkv"}
    pp.gated_delta_rule_packed_prefill(mixed, **dev, out=out, final_state=states, initial_state=states, query_start=starts(lengths).to(DEV),
                                       max_query_len=max(lengths), use_qk_l2norm_in_kernel=True)
    assert (N - 1) * stride > 2 ** 31 and torch.equal(out, alone[0]) and torch.equal(states, alone[1])


@pytest.mark.parametrize("dtype,D,lengths", [(F16, 128, [130, 77]), (F16, 64, [65, 3, 140]), (F32, 64, [97, 64, 129]), (BF16, 128, [70, 130])], ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_more_heads_than_processors(dtype, D, lengths, shift):
    """The forms that share a processor, or have more of a state's columns: aligned rows and others, and a value that is not finite."""
    H, HV = 16, 32
    c, state = make(lengths, H, HV, D, dtype, True)
    width, N = c["mixed_qkv"].shape[1], sum(lengths)
    rows = torch.empty(N, width + 3, dtype=dtype, device=DEV)[:, shift:shift + width] if shift else torch.empty(N, width, dtype=dtype, device=DEV)
    rows.copy_(c["mixed_qkv"])
    got = run(dict(c, mixed_qkv=rows), state, lengths, HV, D)
    assert _lib.load_library().carry_gdn_last_kernel() == IN_CHUNKS
    check(got, c, state, lengths, H, D, in_chunks=True)
    head, column, at = HV - 1, D - 1, lengths[0] - 1
    rows[at, 2 * H * D + head * D + column] = float("inf")
    out, final = run(dict(c, mixed_qkv=rows), state, lengths, HV, D)
    bad, bad_state = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(final, dtype=torch.bool)
    bad[at, head, column], bad_state[0, head, column] = True, True
    assert torch.equal(out[~bad], got[0][~bad]) and torch.equal(final[~bad_state], got[1][~bad_state])
    assert not out[bad].isfinite().any() and not final[bad_state].isfinite().any()
