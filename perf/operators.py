"""The workloads of the operators around the masked attention: rotary positions, norms of
queries and keys with the rotation, selection of key blocks and attention over them.

A case is a dict of plain values:

  op        "rotary", "norm_rotary", "select" (block means and selection) or "attend"
            (attention over selected blocks)
  B, L, Lk  sequences, queries of each, keys of each (a cache's capacity where decode)
  Hq, Hkv, d, dtype ("bf16", "fp16", "fp32")
  grad      True: forward and backward, False: forward alone
  decode    True: the last L positions of sequences of ragged lengths in a cache
  layout, dim, scaling, far     rotary: pairing, rotated columns, frequencies' scaling,
            largest first position
  bs, count block size and blocks of a query

run() is the plain form (float32, elementary operations) or, where `own` is set, the calls
of this framework; exact() the same outputs in float64.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BASE = 10000.0
CONTEXT = 4096  # positions that the unscaled frequencies are meant for
EPS = 1e-6


def _rot(op, B, L, Hq, Hkv, d, *, dtype="bf16", grad=False, layout="half", dim=None, scaling="none", far=0):
    return dict(op=op, B=B, L=L, Lk=L, Hq=Hq, Hkv=Hkv, d=d, dtype=dtype, grad=grad, decode=False, layout=layout,
                dim=dim or d, scaling=scaling, far=far)


def _sel(op, B, L, Hq, Hkv, d, bs, count, *, Lk=None, dtype="bf16", grad=False, decode=False):
    return dict(op=op, B=B, L=L, Lk=Lk or L, Hq=Hq, Hkv=Hkv, d=d, dtype=dtype, grad=grad, decode=decode, bs=bs,
                count=count)


def listed():
    cases = {
        # One token of each of 64 sequences served far into a long context: a call whose cost is its launch.
        "rotary_decode_bf16": _rot("rotary", 64, 1, 32, 8, 128, scaling="parts", far=500000),
        # Training, interleaved pairs, the first 64 of 128 columns turned, a length of no round size.
        "rotary_train_fp16_part": _rot("rotary", 2, 4099, 16, 16, 128, dtype="fp16", grad=True, layout="interleaved", dim=64),
        # A prompt batch with grouped key heads: queries and keys normed and turned once, in one pass.
        "norm_rotary_prefill_bf16": _rot("norm_rotary", 4, 4096, 32, 8, 128),
        # One long sequence trained: the same with gradients of both tensors and both weights.
        "norm_rotary_train_bf16": _rot("norm_rotary", 1, 8192, 32, 32, 128, grad=True, scaling="linear"),
        # A small model trained in float32.
        "norm_rotary_train_fp32": _rot("norm_rotary", 2, 1000, 8, 8, 64, dtype="fp32", grad=True),
        # Selection for one long prompt: means of all blocks, and 16 blocks for each query and key head.
        "select_prefill_bf16": _sel("select", 1, 8192, 32, 8, 128, 64, 16),
        # The same over the longest context: 512 blocks to choose from.
        "select_long_bf16": _sel("select", 1, 32768, 8, 2, 128, 64, 16),
        # One token of each of 32 sequences: the newest block's mean is formed again, 64 blocks of up to 512 chosen.
        "select_decode_bf16": _sel("select", 32, 1, 32, 8, 128, 64, 64, Lk=32768, decode=True),
        # Training over the selected blocks of one long sequence with grouped key heads.
        "attend_train_bf16": _sel("attend", 1, 8192, 32, 8, 128, 64, 16, grad=True),
        # A long prompt over few wide blocks, float16, forward alone.
        "attend_prefill_wide_fp16": _sel("attend", 1, 16384, 16, 4, 128, 512, 4, dtype="fp16"),
        # A small model trained in float32, one key head for each query head, short blocks, an odd length.
        "attend_train_fp32": _sel("attend", 2, 1500, 8, 8, 64, 32, 8, dtype="fp32", grad=True),
        # One token of each of 32 sequences against caches of ragged lengths: 4096 keys of each.
        "attend_decode_bf16": _sel("attend", 32, 1, 32, 8, 128, 64, 64, Lk=32768, decode=True),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    def one():
        hkv = rng.choice((1, 2, 4, 8))
        hq = hkv * rng.choice((1, 2, 4))
        d = rng.choice((64, 64, 96, 128, 128))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        op = rng.choice(("rotary", "norm_rotary", "select", "select", "attend", "attend", "attend"))
        if op in ("rotary", "norm_rotary"):
            served = rng.random() < 0.25
            B = _log(rng, 1, 256) if served else rng.choice((1, 1, 2, 3))
            return _rot(op, B, 1 if served else max(2, _log(rng, 16, 16384) // B), hq, hkv, d, dtype=dtype,
                        grad=rng.random() < 0.6, layout=rng.choice(("half", "interleaved")), dim=rng.choice((d, d, d // 2)),
                        scaling=rng.choice(("none", "linear", "ntk", "parts")),
                        far=rng.choice((0, 0, _log(rng, 1000, 1000000))))
        bs = rng.choice((16, 32, 64, 64, 128, 256))
        if rng.random() < 0.35:  # served: the last few tokens of ragged sequences
            return _sel(op, _log(rng, 1, 32), rng.choice((1, 1, 1, 4)), hq, hkv, d, bs,
                        min(64, _log(rng, 4, 2048) // bs + 2), Lk=_log(rng, 100, 32768), dtype=dtype, decode=True)
        L = _log(rng, 64, 8192)
        return _sel(op, 1 if L > 2900 else rng.choice((1, 2)), L, hq, hkv, d, bs, min(32, _log(rng, 64, 1024) // bs + 2),
                    dtype=dtype, grad=op == "attend" and rng.random() < 0.6)

    most = [max(work(c)[n] for c in listed()) for n in ("bytes", "flops")]
    while True:
        c = one()
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return c


# ---- inputs ----------------------------------------------------------------------------


def _frequencies(case):
    """(inverse frequencies [dim / 2], factor of cos and sin) in float64: the plain ones;
    divided by 8 (linear); of a larger base (ntk); or by parts: the pairs that turn less
    than once over the context are divided, those that turn over 32 times kept, in a
    ramp between."""
    n = case["dim"]
    i = np.arange(0, n, 2) / n
    f = BASE ** -i
    if case["scaling"] == "linear":
        return f / 8.0, 1.0
    if case["scaling"] == "ntk":
        return (BASE * 8.0 ** (n / (n - 2))) ** -i, 1.0
    if case["scaling"] == "parts":
        turns = CONTEXT * f / (2 * math.pi)
        keep = np.clip((np.log(turns)) / math.log(32.0), 0.0, 1.0)
        return f * keep + f / 8.0 * (1 - keep), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _pick(q, k, case, lengths):
    """Blocks of each query as a program that attends has them: first and newest always,
    the best of the others by the dot product with the block's mean key; ascending, -1
    behind."""
    B, L, Hq, d = q.shape
    Hkv, bs, count = case["Hkv"], case["bs"], case["count"]
    nb = -(-case["Lk"] // bs)
    kp = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, nb * bs - case["Lk"]))
    m = kp.view(B, nb, bs, Hkv, d).mean(2, dtype=torch.float32)
    s = torch.matmul(q.float().view(B, L, Hkv, -1, d).sum(3).permute(0, 2, 1, 3), m.permute(0, 2, 3, 1).contiguous())
    pos = (lengths - L)[:, None] + torch.arange(L, device=q.device) if case["decode"] else torch.arange(L, device=q.device).expand(B, L)
    seen = (pos.clamp(min=-1).div(bs, rounding_mode="floor") + 1)[:, None, :, None]
    j = torch.arange(nb, device=q.device)
    s = s.masked_fill((j < 1) | (j >= seen - 1), 1e30).masked_fill(j >= seen, -math.inf)
    top, idx = s.topk(min(count, nb), dim=-1)
    idx = idx.masked_fill(top == -math.inf, nb).sort(-1).values
    idx = idx.masked_fill(idx == nb, -1).permute(0, 2, 1, 3)
    return torch.nn.functional.pad(idx, (0, count - idx.shape[-1]), value=-1).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, B, L, Lk, d = DTYPES[case["dtype"]], case["B"], case["L"], case["Lk"], case["d"]

    def normal(*shape, f=1.0, dtype=dt):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(f)

    s = {"case": case}
    f = d ** -0.25
    s["q"] = normal(B, L, case["Hq"], d, f=f)
    s["k"] = normal(B, Lk, case["Hkv"], d, f=f)
    if case["op"] in ("rotary", "norm_rotary"):
        first = torch.randint(0, case["far"] + 1, (B, 1), generator=gen, device="cuda")
        s["positions"] = (first + torch.arange(L, device="cuda")).to(torch.int32)
        inv, s["scale"] = _frequencies(case)
        s["inv_freq"] = torch.from_numpy(inv).cuda()
        leaves = ["q", "k"]
        if case["op"] == "norm_rotary":
            s["wq"], s["wk"] = (normal(d, f=0.2, dtype=torch.float32).add_(1.0) for _ in range(2))
            leaves += ["wq", "wk"]
        if case["grad"]:
            s["dq"], s["dk"] = normal(B, L, case["Hq"], d), normal(B, L, case["Hkv"], d)
    else:
        s["lengths"] = torch.randint(max(L, Lk // 2), Lk + 1, (B,), generator=gen, device="cuda", dtype=torch.int32) if case["decode"] else None
        s["starts"] = s["lengths"] - L if case["decode"] else None
        if case["op"] == "attend":
            s["v"] = normal(B, Lk, case["Hkv"], d, f=f)
            s["blocks"] = _pick(s["q"], s["k"], case, s["lengths"])
            if case["grad"]:
                s["do"] = normal(B, L, case["Hq"], d)
        elif case["decode"]:  # the means a server keeps beside its cache
            s["means"] = _means_plain(s["k"], case["bs"], s["lengths"])
        leaves = ["q", "k", "v"]
    if case["grad"]:
        for n in leaves:
            s[n].requires_grad_()
        s["leaves"] = [s[n] for n in leaves]
    return s


# ---- plain forms -----------------------------------------------------------------------


def _turn_plain(x, s):
    case = s["case"]
    n = case["dim"]
    angle = s["positions"].double()[:, :, None, None] * s["inv_freq"]
    c, t = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()
    x = x.float()
    if case["layout"] == "half":
        a, b = x[..., : n // 2], x[..., n // 2: n]
        return torch.cat((a * c - b * t, b * c + a * t, x[..., n:]), -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat((torch.stack((a * c - b * t, b * c + a * t), -1).flatten(-2), x[..., n:]), -1)


def _norm_plain(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _means_plain(k, bs, lengths):
    B, Lk, H, d = k.shape
    nb = -(-Lk // bs)
    if lengths is not None:
        k = k.masked_fill((torch.arange(Lk, device=k.device) >= lengths[:, None])[:, :, None, None], 0.0)
    k = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, nb * bs - Lk)).view(B, nb, bs, H, d)
    held = torch.full((B,), Lk, device=k.device) if lengths is None else lengths
    n = (held[:, None] - bs * torch.arange(nb, device=k.device)).clamp(1, bs)
    return (k.sum(2, dtype=torch.float64) / n[:, :, None, None]).float()


def _select_plain(s):
    case, q = s["case"], s["q"]
    B, L, Hq, d = q.shape
    bs, count = case["bs"], case["count"]
    if case["decode"]:  # the newest block's mean
        at = (s["lengths"] - 1).div(bs, rounding_mode="floor").long()
        rows = at[:, None] * bs + torch.arange(bs, device=q.device)
        in_ = (rows < s["lengths"][:, None])[:, :, None, None]
        kk = s["k"][torch.arange(B, device=q.device)[:, None], rows.clamp(max=case["Lk"] - 1)]
        new = kk.masked_fill(~in_, 0.0).sum(1, dtype=torch.float64) / in_.sum(1)
        means = s["means"].index_put_((torch.arange(B, device=q.device), at), new.float())
    else:
        means = _means_plain(s["k"], bs, None)
    nb = means.shape[1]
    # 64 bits: neighbours in the order lie closer than 32 bits hold them apart
    g = q.double().view(B, L, case["Hkv"], -1, d).sum(3).permute(0, 2, 1, 3)
    score = torch.matmul(g, means.double().permute(0, 2, 3, 1).contiguous())
    first = s["starts"][:, None] if case["decode"] else 0
    pos = first + torch.arange(L, device=q.device).expand(B, L)
    seen = (pos.div(bs, rounding_mode="floor") + 1).clamp(0, nb)[:, None, :, None]
    j = torch.arange(nb, device=q.device)
    score = score.masked_fill((j < 1) | (j >= seen - 1), math.inf).masked_fill(j >= seen, -math.inf)
    top, idx = score.sort(dim=-1, descending=True, stable=True)
    idx = idx.masked_fill(top == -math.inf, nb)[..., :count].sort(-1).values
    idx = torch.nn.functional.pad(idx, (0, max(0, count - nb)), value=nb)
    return means, idx.masked_fill(idx == nb, -1).permute(0, 2, 1, 3).to(torch.int32).contiguous()


def _attend_plain(s):
    """Over all keys under the blocks' mask; a served token over the keys gathered for it."""
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    B, L, Hq, d = q.shape
    Hkv, Lk, bs, count = case["Hkv"], case["Lk"], case["bs"], case["count"]
    nb = -(-Lk // bs)
    idx = s["blocks"].long().permute(0, 2, 1, 3)                                   # B, Hkv, L, count
    qg = q.float().view(B, L, Hkv, -1, d).permute(0, 2, 1, 3, 4)                   # B, Hkv, L, G, d
    if case["decode"]:
        pos = s["starts"][:, None] + torch.arange(L, device=q.device)
        key = (idx[..., None] * bs + torch.arange(bs, device=q.device)).flatten(-2)  # B, Hkv, L, n
        ok = (idx >= 0).repeat_interleave(bs, -1) & (key <= pos[:, None, :, None]) & (key < Lk)
        key = key.clamp(0, Lk - 1)
        at = (torch.arange(B, device=q.device)[:, None, None, None], key, torch.arange(Hkv, device=q.device)[:, None, None])
        kk, vv, ok = k[at].float(), v[at].float(), ok[..., None, :]                # B, Hkv, L, n, d
        score = torch.matmul(qg, kk.transpose(-1, -2)) * d ** -0.5
    else:
        in_ = torch.zeros((B, Hkv, L, nb + 1), dtype=torch.bool, device=q.device)
        in_.scatter_(-1, torch.where(idx < 0, nb, idx), True)
        j = torch.arange(Lk, device=q.device)
        ok = (in_[..., j // bs] & (j <= torch.arange(L, device=q.device)[:, None])).repeat_interleave(Hq // Hkv, 1)
        kk, vv = (x.float().repeat_interleave(Hq // Hkv, 2).permute(0, 2, 1, 3).contiguous() for x in (k, v))
        score = torch.matmul(q.float().permute(0, 2, 1, 3), kk.transpose(-1, -2)) * d ** -0.5
    score = score.masked_fill(~ok, -math.inf)
    top = score.detach().amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p / total.masked_fill(total == 0, 1.0), vv)
    if case["decode"]:
        return o.permute(0, 2, 1, 3, 4).reshape(B, L, Hq, d).to(q.dtype)
    return o.permute(0, 2, 1, 3).to(q.dtype)


# ---- one pass --------------------------------------------------------------------------


def _forward(s):
    case = s["case"]
    op = case["op"]
    if own:
        import jaxmodules_amd as jm

        if op == "rotary":
            return jm.rotary(s["q"], s["k"], s["positions"], inv_freq=s["inv_freq"], layout=case["layout"], scale=s["scale"])
        if op == "norm_rotary":
            return jm.norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["positions"], inv_freq=s["inv_freq"],
                                  layout=case["layout"], scale=s["scale"], eps=EPS)
        if op == "select":
            if case["decode"]:
                means = jm.block_means(s["k"], case["bs"], lengths=s["lengths"], out=s["means"], new=1)
            else:
                means = jm.block_means(s["k"], case["bs"])
            return means, jm.select_blocks(s["q"], means, case["bs"], case["count"], first=1, last=1, starts=s["starts"],
                                           lengths=s["lengths"])
        return jm.selected_attention(s["q"], s["k"], s["v"], s["blocks"], case["bs"], is_causal=True, starts=s["starts"],
                                     lengths=s["lengths"])
    if op == "rotary":
        return tuple(_turn_plain(x, s).to(x.dtype) for x in (s["q"], s["k"]))
    if op == "norm_rotary":
        return tuple(_turn_plain(_norm_plain(x, w), s).to(x.dtype) for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])))
    return _select_plain(s) if op == "select" else _attend_plain(s)


def run(state):
    case = state["case"]
    if not case["grad"]:
        with torch.no_grad():
            out = _forward(state)
        return {"out": out}
    out = _forward(state)
    up = state["do"] if case["op"] == "attend" else (state["dq"], state["dk"])
    grads = torch.autograd.grad(out, state["leaves"], up)
    return {"out": out.detach() if case["op"] == "attend" else tuple(x.detach() for x in out), "grads": grads}


def _pairs(case):
    """Visible (query, key) pairs of one sequence and query head, and its (query, block)
    pairs that a score is due for."""
    L, Lk, bs = case["L"], case["Lk"], case["bs"]
    p = np.arange(L) + (int(0.75 * Lk) if case["decode"] else 0)   # ragged lengths: three quarters on average
    seen = p // bs + 1
    n = np.minimum(seen, case["count"])
    return int(((n - 1) * bs + p % bs + 1).sum()), int(seen.sum())


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    B, L, Lk, Hq, Hkv, d = (case[n] for n in ("B", "L", "Lk", "Hq", "Hkv", "d"))
    if case["op"] in ("rotary", "norm_rotary"):
        n = B * L * (Hq + Hkv) * d
        passes = 2 if not case["grad"] else 4 if case["op"] == "rotary" else 5   # in, out; dz, dx; x again
        return {"bytes": passes * n * e, "flops": (2 if case["grad"] else 1) * (3 if case["op"] == "rotary" else 7) * n}
    pairs, scored = _pairs(case)
    if case["op"] == "select":
        nb = -(-Lk // case["bs"])
        keys = B * Hkv * d * (case["bs"] * e if case["decode"] else Lk * e)
        means = B * nb * Hkv * d * 4
        return {"bytes": B * L * Hq * d * e + keys + means + B * L * Hkv * case["count"] * 4, "flops": 2 * B * Hkv * d * scored}
    kv = B * Hkv * d * e * (min(Lk, pairs) if case["decode"] else Lk)
    qo = B * L * Hq * d * e
    if case["grad"]:  # q, k, v, do in; o, dq, dk, dv out
        return {"bytes": 4 * kv + 4 * qo, "flops": 14 * d * Hq * B * pairs}
    return {"bytes": 2 * kv + 2 * qo, "flops": 4 * d * Hq * B * pairs}


# ---- float64 ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)

    def turn(x, sign):
        """s R(sign p w) x on complex numbers, one (first, second) pair each."""
        n, half = case["dim"], case["layout"] == "half"
        z = torch.polar(torch.full_like(s["inv_freq"], s["scale"]).expand(*s["positions"].shape, n // 2).contiguous(),
                        sign * s["positions"].double()[..., None] * s["inv_freq"])[:, :, None]
        h = x[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2) if half else x[..., :n].unflatten(-1, (n // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(h.contiguous()) * z)
        y = y.transpose(-1, -2) if half else y
        return torch.cat((y.flatten(-2), x[..., n:]), -1)

    def rotation():
        outs, grads, weights = [], [], []
        for n in ("q", "k"):
            x = s[n].detach().double()
            if case["op"] == "norm_rotary":
                r = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) ** -0.5
                w = s["w" + n].detach().double()
                outs.append(turn(x * r * w, 1))
                if case["grad"]:
                    dy = turn(s["d" + n].double(), -1)
                    weights.append((dy * x * r).sum((0, 1, 2)))
                    grads.append(r * (dy * w - x * r * (dy * w * x * r).mean(-1, keepdim=True)))
            else:
                outs.append(turn(x, 1))
                if case["grad"]:
                    grads.append(turn(s["d" + n].double(), -1))
        return {"out": tuple(outs), "grads": tuple(grads + weights)} if case["grad"] else {"out": tuple(outs)}

    def select():
        bs, k = case["bs"], s["k"]
        B, Lk = k.shape[:2]
        nb = -(-Lk // bs)
        held = s["lengths"].tolist() if case["decode"] else [Lk] * B
        if case["decode"]:
            means = s["means"].double().clone()
        else:
            means = torch.zeros((B, nb, case["Hkv"], case["d"]), dtype=torch.float64, device=k.device)
        for b in range(B):
            for j in range((held[b] - 1) // bs if case["decode"] else 0, -(-held[b] // bs)):
                means[b, j] = k[b, j * bs:min(held[b], (j + 1) * bs)].double().mean(0)
        return {"out": (means, None)}

    def attend():
        q, k, v, blocks = (s[n].detach() for n in ("q", "k", "v", "blocks"))
        B, L, Hq, d = q.shape
        Hkv, bs, Lk, G = case["Hkv"], case["bs"], case["Lk"], Hq // case["Hkv"]
        o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in ((q, k, v) if case["grad"] else (q[:0],) * 3))
        j = torch.arange(Lk, device=q.device)
        for b in range(B):
            start = int(s["starts"][b]) if case["decode"] else 0
            for h in range(Hkv):
                listed_ = (blocks[b, :, h, :, None] == torch.arange(-(-Lk // bs), device=q.device)).any(1)
                ok = listed_[:, j // bs] & (j <= start + torch.arange(L, device=q.device)[:, None])
                K, V = k[b, :, h].double(), v[b, :, h].double()
                for i in range(h * G, h * G + G):
                    Q = q[b, :, i].double()
                    S = (Q @ K.T * d ** -0.5).masked_fill(~ok, -math.inf)
                    P = torch.softmax(S, -1).masked_fill(~ok, 0.0)
                    O = P @ V
                    o[b, :, i] = O
                    if case["grad"]:
                        dO = s["do"][b, :, i].double()
                        dS = P * (dO @ V.T - (dO * O).sum(-1, keepdim=True)) * d ** -0.5
                        dv[b, :, h] += P.T @ dO
                        dk[b, :, h] += dS.T @ Q
                        dq[b, :, i] = dS @ K
        return {"out": o, "grads": (dq, dk, dv)} if case["grad"] else {"out": o}

    with torch.no_grad():
        if case["op"] in ("rotary", "norm_rotary"):
            return rotation()
        return select() if case["op"] == "select" else attend()
