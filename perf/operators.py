"""The operators of the packed serving path, as they are measured: what each
case stands for, its inputs, its plain form in elementary torch operations, the
call a user makes, and its definition in 64 bits.

  qk_norm_rope        RMS norm of every query and key head and the rotate-half
                      position rotation, in one pass over the projections' output
  attn_varlen         attention over packed sequences of different lengths
                      (prompts, chunks of prompts behind a history, single
                      tokens), grouped heads, bottom-right causal
  attn_decode_shared  one token per request against a prefix that the whole
                      batch shares and the request's own keys behind it

Head dim 128 and bf16 throughout, as everywhere in this package.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
EPS = 1e-6
THETA = 1e6          # RoPE base of the package's benchmark layer
MAX_SCORES = 1 << 28  # elements of one score block of the plain forms (1 GiB in fp32)


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one decode step of a batch of 64: the smallest call, latency counts
        dict(name="norm_decode", op="norm", tokens=64, heads=32, kv_heads=8, layout="fused", positions=True),
        # an odd prompt in the package's own head-split layout, angles given per token
        dict(name="norm_odd", op="norm", tokens=1021, heads=28, kv_heads=4, layout="heads", positions=False),
        # the packed prompts of a whole prefill step (4 x 8192 tokens)
        dict(name="norm_prefill", op="norm", tokens=32768, heads=28, kv_heads=4, layout="fused", positions=True),
        # a handful of short questions: latency counts
        dict(name="varlen_short", op="varlen", seqs=5, min_q=1, max_q=40, min_hist=0, max_hist=0, heads=28, kv_heads=4,
             causal=True, empty=False, lens=11),
        # an ordinary batch of prompts of different lengths
        dict(name="varlen_prompts", op="varlen", seqs=24, min_q=64, max_q=2048, min_hist=0, max_hist=0, heads=32,
             kv_heads=8, causal=True, empty=False, lens=12),
        # odd group of five heads, idle slots of length zero, no causal mask (an encoder's batch)
        dict(name="varlen_full", op="varlen", seqs=9, min_q=200, max_q=1500, min_hist=0, max_hist=0, heads=10,
             kv_heads=2, causal=False, empty=True, lens=13),
        # the serving form: single tokens behind histories of very different lengths
        dict(name="varlen_tokens", op="varlen", seqs=64, min_q=1, max_q=1, min_hist=100, max_hist=16000, heads=32,
             kv_heads=8, causal=True, empty=False, lens=14),
        # the largest: long prompts, 28/4 heads
        dict(name="varlen_long", op="varlen", seqs=4, min_q=4096, max_q=12288, min_hist=0, max_hist=0, heads=28,
             kv_heads=4, causal=True, empty=False, lens=15),
        # a small batch behind a short instruction: latency counts
        dict(name="shared_small", op="shared", batch=4, heads=28, kv_heads=4, prefix=1000, capacity=64, lens=21),
        # odd sizes: 33 requests, groups of five heads
        dict(name="shared_odd", op="shared", batch=33, heads=40, kv_heads=8, prefix=5003, capacity=400, lens=22),
        # the decode batch of the benchmark (64 requests, 32768 keys), now with the prompt shared
        dict(name="shared_long", op="shared", batch=64, heads=32, kv_heads=8, prefix=32768, capacity=1024, lens=23),
        # many requests behind one document
        dict(name="shared_wide", op="shared", batch=256, heads=32, kv_heads=8, prefix=4096, capacity=512, lens=24),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads = rng.choice([(28, 4), (32, 8), (10, 2), (40, 8), (16, 16), (12, 4), (8, 1), (7, 7)])
    op = rng.choice(["norm", "varlen", "shared"])
    if op == "norm":
        return dict(op="norm", tokens=_between(rng, 1, 20000), heads=heads, kv_heads=kv_heads,
                    layout=rng.choice(["fused", "heads"]), positions=rng.random() < 0.5)
    if op == "varlen":
        kind = rng.choice(["prompts", "chunks", "tokens"])
        c = dict(op="varlen", heads=heads, kv_heads=kv_heads, causal=rng.random() < 0.75, empty=rng.random() < 0.3,
                 lens=rng.randrange(1 << 30))
        if kind == "prompts":
            top = _between(rng, 2, 8192)
            return dict(c, seqs=_between(rng, 1, max(1, min(64, 16384 // top))), min_q=max(1, top // rng.choice([2, 8, 64])),
                        max_q=top, min_hist=0, max_hist=0)
        if kind == "chunks":
            return dict(c, seqs=_between(rng, 1, 12), min_q=1, max_q=_between(rng, 2, 512), min_hist=0,
                        max_hist=_between(rng, 64, 8192))
        return dict(c, seqs=_between(rng, 1, 64), min_q=1, max_q=1, min_hist=rng.randrange(0, 64),
                    max_hist=_between(rng, 64, 16000))
    batch = _between(rng, 1, 256)
    return dict(op="shared", batch=batch, heads=heads, kv_heads=kv_heads,
                prefix=_between(rng, 1, min(32768, (1 << 26) // (batch * heads), (1 << 18) // kv_heads)),
                capacity=_between(rng, 1, min(1024, (1 << 19) // (batch * kv_heads))), lens=rng.randrange(1 << 30))


def _seq_lens(case):
    """(query lengths, key lengths) of a varlen case: the keys are the history and the new tokens."""
    r = random.Random(case["lens"])
    q_lens, k_lens = [], []
    for i in range(case["seqs"]):
        n = _between(r, case["min_q"], case["max_q"])
        h = _between(r, max(1, case["min_hist"]), case["max_hist"]) if case["max_hist"] > 0 else 0
        if case["empty"] and i % 4 == 1:
            n = 0
        q_lens.append(n)
        k_lens.append(n + h)
    return q_lens, k_lens


def _own_lens(case):
    """Keys of each request behind the shared prefix: 0 (nothing yet) up to the cache's capacity."""
    r = random.Random(case["lens"])
    return [r.randint(0, case["capacity"]) for _ in range(case["batch"])]


# ------------------------------------------------------------------ inputs --
def _rope_tables(positions):
    """cos, sin (fp32 [len, 128]) of the given positions; angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=positions.device) / D)
    ang = positions.double()[:, None] * inv[None]
    ang = torch.cat([ang, ang], -1)
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()

    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "norm":
        t = case["tokens"]
        if case["layout"] == "fused":  # the output of one q/k/v projection, sliced
            qkv = normal(t, h + 2 * hk, D, scale=1.7)
            q, k = qkv[:, :h], qkv[:, h:h + hk]
        else:  # [H, T, 128] as the package's projections write them, indexed [T, H, 128]
            q, k = normal(h, t, D, scale=1.7).transpose(0, 1), normal(hk, t, D, scale=1.7).transpose(0, 1)
        s = dict(op="norm", q=q, k=k, qw=1 + normal(D, scale=0.2), kw=1 + normal(D, scale=0.2), positions=None)
        if case["positions"]:  # packed prompts: positions restart, the table covers the longest context
            length = max(64, min(8192, t))
            s["positions"] = torch.randint(0, length, (t,), device="cuda", generator=g, dtype=torch.int32)
            s["rope"] = _rope_tables(torch.arange(length, device="cuda"))
        else:
            s["rope"] = _rope_tables(torch.arange(t, device="cuda") + (seed % 7) * 1000)
        return s
    if case["op"] == "varlen":
        q_lens, k_lens = _seq_lens(case)
        tq, tk = sum(q_lens), sum(k_lens)
        if case["max_hist"] == 0:  # prompts: slices of the packed projection
            qkv = normal(tq, h + 2 * hk, D)
            q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        else:
            q, k, v = normal(tq, h, D), normal(tk, hk, D), normal(tk, hk, D)
        cu = [torch.tensor([0] + n, device="cuda").cumsum(0).int() for n in (q_lens, k_lens)]
        return dict(op="varlen", q=q, k=k, v=v, cu_q=cu[0], cu_k=cu[1], max_k=max(k_lens), q_lens=q_lens, k_lens=k_lens,
                    causal=case["causal"])
    b, p, cap = case["batch"], case["prefix"], case["capacity"]
    lens = _own_lens(case)
    return dict(op="shared", q=normal(b, h, D), k_prefix=normal(hk, p, D), v_prefix=normal(hk, p, D),
                k=normal(b, hk, cap, D), v=normal(b, hk, cap, D),
                lens=torch.tensor(lens, device="cuda", dtype=torch.int32))


# ------------------------------------------------------------- plain forms --
def _norm_rotate(x, w, cos, sin):
    """x [T, H, 128], cos / sin [T, 128]: fp32, rounded once."""
    x = x.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    turned = torch.cat([-n[..., D // 2:], n[..., :D // 2]], -1)
    return (n * cos[:, None] + turned * sin[:, None]).bfloat16()


def _softmax_v(s, v):
    """fp32 scores [..., R, S] (-inf where masked) and values [..., S, 128]: output and log-sum-exp; rows that see
    nothing give zeros and -inf."""
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    z = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(z == 0, 1.0, z)
    return o, (torch.log(z) + m).squeeze(-1)


def _plain_varlen(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, hk = q.shape[1], k.shape[1]
    o = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    lse = torch.empty((h, q.shape[0]), dtype=torch.float32, device=q.device)
    q_lens, k_lens = s["q_lens"], s["k_lens"]
    mq, mk, n = max(q_lens), max(k_lens), len(q_lens)
    if n * h * mq * mk <= MAX_SCORES:  # everything at once, padded
        dev = q.device
        ql, kl = s["cu_q"].diff().long(), s["cu_k"].diff().long()
        iq, ik = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
        rows = (s["cu_q"][:-1, None] + iq).clamp(max=q.shape[0] - 1)
        keys = (s["cu_k"][:-1, None] + ik).clamp(max=k.shape[0] - 1)
        qf = q[rows].float().view(n, mq, hk, h // hk, D).permute(0, 2, 3, 1, 4).reshape(n, hk, h // hk * mq, D)
        kf, vf = k[keys].float().permute(0, 2, 1, 3), v[keys].float().permute(0, 2, 1, 3)
        see = (ik[None] < kl[:, None])[:, None]
        if s["causal"]:
            see = see & (ik[None, None] <= iq[None, :, None] + (kl - ql)[:, None, None])
        sc = torch.matmul(qf, kf.transpose(-1, -2)).view(n, hk, h // hk, mq, mk) * D ** -0.5
        sc = sc.masked_fill(~see[:, None, None], -math.inf).view(n, hk, h // hk * mq, mk)
        of, l = _softmax_v(sc, vf)
        live = iq[None] < ql[:, None]
        o[:] = of.view(n, h, mq, D).permute(0, 2, 1, 3)[live].bfloat16()
        lse[:] = l.view(n, h, mq).permute(1, 0, 2)[:, live]
        return o, lse
    q0 = k0 = 0
    for lq, lk in zip(q_lens, k_lens):  # long sequences one by one, in blocks of rows whose scores fit
        kf, vf = (x[k0:k0 + lk].float().transpose(0, 1) for x in (k, v))
        step = max(1, MAX_SCORES // (h * max(1, lk)))
        for a in range(0, lq, step):
            b = min(lq, a + step)
            qf = q[q0 + a:q0 + b].float().view(b - a, hk, h // hk, D).permute(1, 2, 0, 3).reshape(hk, -1, D)
            sc = torch.matmul(qf, kf.transpose(-1, -2)).view(h, b - a, lk) * D ** -0.5
            if s["causal"]:
                row = torch.arange(a, b, device=q.device)[:, None] + lk - lq
                sc = sc.masked_fill(torch.arange(lk, device=q.device)[None] > row, -math.inf)
            of, l = _softmax_v(sc.view(hk, -1, lk), vf)
            o[q0 + a:q0 + b] = of.view(h, b - a, D).transpose(0, 1).bfloat16()
            lse[:, q0 + a:q0 + b] = l.view(h, b - a)
        q0, k0 = q0 + lq, k0 + lk
    return o, lse


def _plain_shared(s):
    q, kp, vp, k, v = s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"]
    b, h = q.shape[:2]
    hk, p, cap = kp.shape[0], kp.shape[1], k.shape[2]
    qf = q.float().view(b, hk, h // hk, D)
    sp = torch.matmul(qf.transpose(0, 1).reshape(hk, -1, D), kp.float().transpose(-1, -2))
    sp = sp.view(hk, b, h // hk, p).transpose(0, 1)
    so = torch.matmul(qf, k.float().transpose(-1, -2))
    past = torch.arange(cap, device=q.device)[None] >= s["lens"][:, None]
    so = so.masked_fill(past[:, None, None], -math.inf)
    sc = torch.cat([sp, so], -1) * D ** -0.5
    m = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - m)
    z = e.sum(-1, keepdim=True)
    ep, eo = e[..., :p], e[..., p:]
    o = torch.matmul(ep.transpose(0, 1).reshape(hk, -1, p), vp.float()).view(hk, b, h // hk, D).transpose(0, 1)
    o = (o + torch.matmul(eo, v.float())) / z
    return o.reshape(b, 1, h, D).bfloat16(), (torch.log(z) + m).view(b, h)


def run(state):
    s = state
    if own:
        from mka_b200 import ops

        if s["op"] == "norm":
            return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], EPS, rope=s["rope"], positions=s["positions"])
        if s["op"] == "varlen":
            return ops.attn_varlen(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_k=s["max_k"], causal=s["causal"])
        return ops.attn_decode_shared(s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], s["lens"])
    if s["op"] == "norm":
        cos, sin = s["rope"]
        if s["positions"] is not None:
            cos, sin = cos[s["positions"]], sin[s["positions"]]
        return _norm_rotate(s["q"], s["qw"], cos, sin), _norm_rotate(s["k"], s["kw"], cos, sin)
    return _plain_varlen(s) if s["op"] == "varlen" else _plain_shared(s)


# -------------------------------------------------------------------- work --
def work(case):
    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "norm":
        t = case["tokens"]
        table = min(t, max(64, min(8192, t))) if case["positions"] else t
        return {"bytes": t * (h + hk) * D * 4 + table * D * 8 + (4 * t if case["positions"] else 0) + 4 * D,
                "flops": t * (h + hk) * D * 7}
    if case["op"] == "varlen":
        q_lens, k_lens = _seq_lens(case)
        pairs = 0
        for lq, lk in zip(q_lens, k_lens):
            pairs += lq * lk - (lq * (lq - 1) // 2 if case["causal"] else 0)
        live = sum(lk for lq, lk in zip(q_lens, k_lens) if lq > 0)
        return {"bytes": sum(q_lens) * h * (D * 4 + 4) + live * hk * D * 4 + 8 * (case["seqs"] + 1),
                "flops": 4 * D * h * pairs}
    b, n = case["batch"], sum(_own_lens(case))
    return {"bytes": b * h * (D * 4 + 4) + (case["prefix"] + n) * hk * D * 4 + 4 * b,
            "flops": 4 * D * h * (b * case["prefix"] + n)}


# ------------------------------------------------------- definition, 64 bits --
def _exact_norm(x, w, cos, sin):
    x = x.double()
    unit = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
    lo, hi = unit.split(D // 2, -1)
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([lo * cos[..., :D // 2] - hi * sin[..., :D // 2], hi * cos[..., D // 2:] + lo * sin[..., D // 2:]], -1)


def _exact_rows(q, keys, values, see):
    """q [R, D], keys / values [S, D] of one head in 64 bits; see [R, S] or None."""
    s = q @ keys.t() / math.sqrt(D)
    if see is not None:
        s = torch.where(see, s, torch.full_like(s, -math.inf))
    l = torch.logsumexp(s, -1)
    return torch.exp(s - l[:, None]) @ values, l


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        cos, sin = s["rope"]
        if s["positions"] is not None:
            at = s["positions"].long()
            cos, sin = cos.index_select(0, at), sin.index_select(0, at)
        return _exact_norm(s["q"], s["qw"], cos, sin), _exact_norm(s["k"], s["kw"], cos, sin)
    q = s["q"].double()
    if case["op"] == "varlen":
        h, group = q.shape[1], q.shape[1] // s["k"].shape[1]
        o, lse = torch.empty_like(q), torch.empty((h, q.shape[0]), dtype=torch.float64, device=q.device)
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for i in range(case["seqs"]):
            lq, lk = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
            at = torch.arange(lq, device=q.device)
            for a in at.split(4096):
                see = None
                if case["causal"]:
                    see = torch.arange(lk, device=q.device)[None] + (lq - lk) <= a[:, None]
                for j in range(h):
                    kj, vj = (x[ck[i]:ck[i + 1], j // group].double() for x in (s["k"], s["v"]))
                    o[cq[i] + a, j], lse[j, cq[i] + a] = _exact_rows(q[cq[i] + a, j], kj, vj, see)
        return o, lse
    b, h = q.shape[:2]
    group = h // s["k"].shape[1]
    o, lse = torch.empty((b, 1, h, D), dtype=torch.float64, device=q.device), torch.empty((b, h), dtype=torch.float64, device=q.device)
    for j in range(h // group):
        kp, vp = s["k_prefix"][j].double(), s["v_prefix"][j].double()
        rows = slice(j * group, (j + 1) * group)
        op, lp = _exact_rows(q[:, rows].reshape(-1, D), kp, vp, None)
        op, lp = op.view(b, group, D), lp.view(b, group)
        for i, n in enumerate(s["lens"].tolist()):
            oi, li = _exact_rows(q[i, rows], s["k"][i, j, :n].double(), s["v"][i, j, :n].double(), None)
            l = torch.logaddexp(lp[i], li)
            oi = torch.where(torch.isfinite(li)[:, None], oi, torch.zeros_like(oi))
            o[i, 0, rows] = op[i] * torch.exp(lp[i] - l)[:, None] + oi * torch.exp(li - l)[:, None]
            lse[i, rows] = l
    return o, lse
