"""Block means, selection and attention over selected blocks in float64, by plain loops
over sequences and heads."""
import math

import numpy as np
import torch


def means(k, bs, lengths=None):
    k = k.detach().double().cpu()
    B, L, H, d = k.shape
    out = torch.zeros((B, -(-L // bs), H, d), dtype=torch.float64)
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        for j in range(-(-n // bs)):
            out[b, j] = k[b, j * bs:min(n, (j + 1) * bs)].mean(0)
    return out


def select(q, m, bs, count, causal=True, first=1, last=1, starts=None, lengths=None):
    """(blocks, scores) by sorting (-score, index) of each query's candidates."""
    q, m = q.detach().double().cpu(), m.detach().double().cpu()
    B, N, Hq, d = q.shape
    nblk, Hkv = m.shape[1:3]
    score = torch.einsum("bnhd,bjhd->bnhj", q.view(B, N, Hkv, -1, d).sum(3), m).numpy()
    out = np.full((B, N, Hkv, count), -1, np.int32)
    for b in range(B):
        nb = nblk if lengths is None else min(max(-(-int(lengths[b]) // bs), 0), nblk)
        for i in range(N):
            pos = i + (0 if starts is None else int(starts[b]))
            seen = nb if not causal else min(nb, max(pos, -1) // bs + 1)
            f = min(first, seen)
            l = min(last, seen - f)
            for h in range(Hkv):
                s = np.nan_to_num(score[b, i, h], nan=-np.inf, posinf=np.inf, neginf=-np.inf)
                c = sorted(range(f, seen - l), key=lambda j: (-s[j], j))[: max(0, min(count, seen) - f - l)]
                got = sorted([*range(f), *c, *range(seen - l, seen)])
                out[b, i, h, : len(got)] = got
    return torch.from_numpy(out), score


def visible(blocks, N, L, bs, causal, starts, lengths):
    """[B, Hkv, N, L]: key seen by query."""
    B, _, Hkv, _ = blocks.shape
    nblk = -(-L // bs)
    blocks = blocks.cpu().long()
    member = (blocks[..., None] == torch.arange(nblk)).any(3)  # B, N, Hkv, nblk
    ok = member.permute(0, 2, 1, 3)[..., torch.arange(L) // bs]
    for b in range(B):
        held = L if lengths is None else int(lengths[b])
        pos = torch.arange(N) + (0 if starts is None else int(starts[b]))
        ok[b] &= torch.arange(L) < held
        if causal:
            ok[b] &= torch.arange(L)[None, :] <= pos[:, None]
    return ok


def attend(q, k, v, ok, scale=None, do=None):
    """Outputs and the magnitudes that bound their errors: {name: (value, magnitude)}, and
    the largest magnitude of a score's terms."""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    B, N, Hq, d = q.shape
    L, Hkv = k.shape[1:3]
    G = Hq // Hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    top = 0.0
    clean = lambda x: torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
    for b in range(B):
        for h in range(Hkv):
            m = ok[b, h]
            # values that no query sees take no part, whatever they are
            use = m.any(0)
            K, V = (torch.where(use[:, None], x[b, :, h], torch.zeros(())) for x in (k, v))
            for i in range(h * G, h * G + G):
                S = torch.where(m, q[b, :, i] @ K.T * scale, -math.inf)
                A = clean(q[b, :, i].abs()) @ clean(K.abs()).T * abs(scale)
                top = max(top, float(torch.where(m, A, 0.0).max()) if m.any() else 0.0)
                P = torch.where(m, torch.exp(S - torch.where(S.amax(-1, keepdim=True) == -math.inf, 0.0, S.amax(-1, keepdim=True))), 0.0)
                P = P / torch.where(P.sum(-1, keepdim=True) == 0, 1.0, P.sum(-1, keepdim=True))
                O = P @ V
                out["o"][0][b, :, i], out["o"][1][b, :, i] = O, P @ V.abs()
                if do is None:
                    continue
                D = do[b, :, i].double().cpu()
                dS = P * (D @ V.T - (D * O).sum(-1, keepdim=True)) * scale
                M = P * (D.abs() @ V.abs().T + (D.abs() * (P @ V.abs())).sum(-1, keepdim=True)) * abs(scale)
                for n, x, y, at in (("dq", dS @ K, M @ K.abs(), i), ("dk", dS.T @ q[b, :, i], M.T @ q[b, :, i].abs(), h),
                                    ("dv", P.T @ D, P.T @ D.abs(), h)):
                    out[n][0][b, :, at] += x
                    out[n][1][b, :, at] += y
    return out, top


def tolerance(value, mag, dt, top, d, terms):
    """Bound of an output's error.  u = 2^-24.  Scores are sums of d products in float32, off
    by (d + 4) u of their magnitude, at most `top`; a weight is off by twice that (itself
    and the sum of weights), and by 8 u of exponential, logarithm and joining; products of
    `terms` terms by terms * u.  16-bit: P and dS are rounded to the inputs' type, half a
    step eps / 2 each (O: and so is the sum that divides them), and the result is."""
    u = 2.0 ** -24
    w = 2 * ((d + 4) * u * top) + 8 * u + (terms + 2 * d + 16) * u
    eps = torch.finfo(dt).eps
    if dt == torch.float32:
        return (w + eps) * mag + 1e-37
    # a weight below the type's smallest normal value keeps an absolute step only
    tiny = torch.finfo(dt).smallest_normal * eps
    return eps / 2 * value.abs() * (1 + eps) + (w + eps) * mag * (1 + eps) + tiny * (1 + mag)
