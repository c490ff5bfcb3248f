"""Plain 64-bit definitions, on the CPU, of a prompt's way through a hybrid model's layers: the gated delta rule over whole
sequences, and the norm and rotation of queries and keys.  Test infrastructure, written from the formulas."""

from __future__ import annotations

import torch

CHUNK = 64


def delta_rule(mixed, a, b, A_log, dt_bias, scale, H, D, lengths, initial=None, l2norm=True):
    """(out, state, out_weight, state_weight) of requests whose rows follow one another.

    The recurrence S <- alpha S (I - beta k k^T) + beta v k^T does not stretch a row of S while beta |k|^2 <= 2, so an error
    made on the way only fades.  ``state_weight [B, HV, V, 1, 3]`` sums, for each row of S, what errors can be relative to:

    * with a token's own arithmetic, the sizes |S| (1 + |log alpha|) + beta (|v| + |S|) that it goes through, counted once,
    * with T = (I + L)^-1 of a chunk, of which |T_ij| <= beta_i exp(G_i - G_j), the sizes beta_j (|v_j| + |S_0|) behind it,

    and a third number has the second's parts as the root of the sum of their squares, for errors that are as good as independent.
    ``out_weight [N, HV, V, 3]`` is the same for the outputs."""
    B, HV = len(lengths), a.shape[1]
    group = HV // H
    x = mixed.double()
    g = -torch.exp(A_log.double()) * torch.nn.functional.softplus(a.double() + dt_bias.double())
    beta = torch.sigmoid(b.double())
    out = torch.zeros(x.shape[0], HV, D, dtype=torch.float64)
    out_weight = torch.zeros(x.shape[0], HV, D, 3, dtype=torch.float64)
    state = torch.zeros(B, HV, D, D, dtype=torch.float64) if initial is None else initial.double().clone()
    weight = torch.zeros(B, HV, D, 3, dtype=torch.float64)
    row = 0
    for i, n in enumerate(lengths):
        S, w = state[i], weight[i]
        for t in range(n):
            if t % CHUNK == 0:
                start, behind, squares = S.norm(dim=-1), torch.zeros(HV, D, dtype=torch.float64), torch.zeros(HV, D, dtype=torch.float64)
            q = x[row, :H * D].view(H, D).repeat_interleave(group, 0)
            k = x[row, H * D:2 * H * D].view(H, D).repeat_interleave(group, 0)
            v = x[row, 2 * H * D:].view(HV, D)
            if l2norm:
                q, k = (y / torch.sqrt((y * y).sum(-1, keepdim=True) + 1e-6) for y in (q, k))
            q = q * scale
            alpha, be = torch.exp(g[row])[:, None], beta[row][:, None]
            size = S.norm(dim=-1)
            S *= alpha[..., None]
            u = be * (v - torch.einsum("hvk,hk->hv", S, k))
            S += u[..., None] * k[:, None]
            out[row] = torch.einsum("hvk,hk->hv", S, q)
            behind = behind * alpha + be * (v.abs() + start)
            squares = squares * alpha ** 2 + (be * (v.abs() + start)) ** 2
            w *= alpha[..., None]
            w[..., 0] += size * (1 + g[row].abs()[:, None]) + be * (v.abs() + size)
            w[..., 1] += be * behind
            w[..., 2] = (w[..., 2] ** 2 + be ** 2 * squares).sqrt()
            q_size = q.norm(dim=-1)[:, None]
            out_weight[row, ..., 0] = q_size * (w[..., 0] + S.norm(dim=-1))
            out_weight[row, ..., 1] = q_size * (w[..., 1] + CHUNK * behind)
            out_weight[row, ..., 2] = q_size * (w[..., 2] + (CHUNK * squares).sqrt())
            row += 1
    return out, state, out_weight, weight[..., None, :]


def qk_norm_rope(x, weight, cos_sin, positions, eps, sections=None, interleaved=False, offset=0.0):
    """(y, size): the normed and rotated heads, and |y1| + |y2| of every number's pair, what an error is relative to."""
    half = cos_sin.shape[1] // 2
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    positions = positions.view(-1, x.shape[0]).long()
    out, size = y.clone(), y.abs()
    axis = [i for i, s in enumerate(sections or [half]) for _ in range(s)]
    for f in range(half):
        p = positions[axis[f]].clamp(0, cos_sin.shape[0] - 1)
        c, s = cos_sin[p, f].double()[:, None], cos_sin[p, half + f].double()[:, None]
        i, j = (2 * f, 2 * f + 1) if interleaved else (f, f + half)
        out[..., i], out[..., j] = y[..., i] * c - y[..., j] * s, y[..., j] * c + y[..., i] * s
        size[..., i] = size[..., j] = y[..., i].abs() + y[..., j].abs()
    return out, size
