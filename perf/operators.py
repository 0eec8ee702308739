"""Measured cases of the attention-block operators beside the cache.

Three operators, each through the framework's public entry points when ``own`` is true and as elementary torch
operations in 32 bits otherwise:

* ``attend``: softmax attention of packed sequences with grouped heads, causal by token or by block of tokens (a
  frame), over keys that may start earlier than the queries, optionally merged with the history part;
* ``rotary`` / ``tables``: rotary positions with several axes (time, height, width), applied to q and k after an
  optional RMS norm, or written out as the cos / sin tables that the K/V projection takes;
* ``norm``: gated residual with an optional norm of the block's output, then the next block's norm and modulation.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _pkg():
    import os
    import sys
    root = os.path.join(os.getcwd(), "hy-nomas-rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nomas_kv
    return nomas_kv


def _ints(text):
    return [int(v) for v in str(text).split(",")]


# ------------------------------------------------------------------ cases
def _attend(name, q_lens, k_lens, heads, kv_heads, head_dim, dtype, causal=True, block=1, history=False):
    return {"name": name, "op": "attend", "q_lens": q_lens, "k_lens": k_lens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "causal": causal, "block": block, "history": history}


def _rotary(name, tokens, heads, kv_heads, head_dim, dims, dtype, norm, interleaved, fused, far):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dims": dims, "dtype": dtype, "norm": norm, "interleaved": interleaved,
            "fused": fused, "far": far}


def _norm(name, tokens, dim, dtype, branch, post, norm, weight, groups, mod_dtype):
    return {"name": name, "op": "norm", "tokens": tokens, "dim": dim, "dtype": dtype, "branch": branch,
            "post": post, "norm": norm, "weight": weight, "groups": groups, "mod_dtype": mod_dtype}


def listed():
    return [
        # one new token of the 24-head model over the benchmark's rebuilt working set
        _attend("attend_token", "1", "29056", 24, 24, 128, "bf16"),
        # a whole segment (4 frames of 1,560 tokens and 256 text tokens), each frame seeing itself and the frames
        # before it, merged with the history part
        _attend("attend_segment", "6496", "6496", 24, 24, 128, "bf16", block=1560, history=True),
        # prompts of very different lengths packed into one call, grouped heads
        _attend("attend_prompts", "1,17,509,1024,2049,4093", "1,17,509,1024,2049,4093", 32, 8, 128, "f16"),
        # one long prompt with narrow heads
        _attend("attend_long", "16383", "16383", 16, 4, 64, "bf16"),
        # chunks of new tokens over caches of their own, some rows short, one sequence idle
        _attend("attend_chunks", "4,1,16,3,0,64", "9001,1,4096,777,130,64", 40, 8, 128, "bf16"),
        # q and k of one new token
        _rotary("rotary_token", 1, 24, 24, 128, "44,42,42", "bf16", True, True, False, False),
        # q and k of a whole segment, RMS norm and three axes
        _rotary("rotary_segment", 6496, 24, 24, 128, "44,42,42", "bf16", True, True, False, False),
        # far positions, half-split pairs, a part of the head rotated, q and k as views of one projection
        _rotary("rotary_far", 4099, 32, 8, 128, "32,24,24", "f16", False, False, True, True),
        # the tables of a whole segment, as the K/V projection takes them
        {"name": "tables_segment", "op": "tables", "tokens": 6496, "dims": "44,42,42", "far": False},
        # one new token between two blocks
        _norm("norm_token", 1, 2048, "bf16", True, "rms", "rms", True, 1, "f32"),
        # a whole segment between two blocks: gate, norms on both sides, one modulation per frame and one for text
        _norm("norm_segment", 6496, 5120, "bf16", True, "rms", "rms", True, 5, "f32"),
        # a layer norm before the first block, rows of an odd width
        _norm("norm_odd", 2047, 1155, "f16", False, "none", "layer", False, 3, "same"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _axes_dims(rng, head_dim):
    n = rng.choice([1, 2, 3, 3, 3])
    total = head_dim // 2 if rng.random() < 0.7 else rng.randint(n, max(n, head_dim // 2))
    cuts = sorted(rng.sample(range(1, total), n - 1)) if total >= n and n > 1 else []
    parts = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return ",".join(str(2 * p) for p in parts)


def draw(rng):
    op = rng.choice(["attend", "attend", "rotary", "norm", "tables"])
    if op == "attend":
        while True:
            kv = _log(rng, 1, 24)
            heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
            head_dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 16)])
            n = rng.choice([1, 1, 2, 3, 5, 8])
            q, k = [], []
            for _ in range(n):
                ql = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 8192), _log(rng, 64, 8192)])
                if n > 1 and rng.random() < 0.05:
                    ql = 0
                kl = ql if rng.random() < 0.5 else ql + _log(rng, 1, 16384)
                q.append(ql)
                k.append(kl)
            case = _attend("", ",".join(map(str, q)), ",".join(map(str, k)), heads, kv, head_dim,
                           rng.choice(["bf16", "bf16", "f16"]), causal=rng.random() < 0.8,
                           block=rng.choice([1, 1, _log(rng, 2, 2000)]), history=rng.random() < 0.3)
            area = sum(a * b for a, b in zip(q, k)) * heads * head_dim
            if heads <= 64 and sum(q) > 0 and area <= 6496 * 6496 * 24 * 128 and \
                    work(case)["flops"] <= 2.5e11 and work(case)["bytes"] <= 4e8:
                break
    elif op == "rotary":
        kv = _log(rng, 1, 24)
        heads = kv * rng.choice([1, 1, 2, 4])
        head_dim = rng.choice([64, 128, 128, 2 * rng.randint(8, 128)])
        tokens = _log(rng, 1, max(1, min(20000, 6496 * 48 * 128 // ((heads + kv) * head_dim))))
        case = _rotary("", tokens, heads, kv if rng.random() < 0.6 else 0, head_dim, _axes_dims(rng, head_dim),
                       rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.6, rng.random() < 0.6,
                       rng.random() < 0.3, rng.random() < 0.3)
        if case["dtype"] == "f32":
            case["tokens"] = max(1, tokens // 2)
    elif op == "tables":
        case = {"op": "tables", "tokens": _log(rng, 1, 30000), "dims": _axes_dims(rng, 2 * rng.randint(8, 64)),
                "far": rng.random() < 0.4}
    else:
        dim = rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 8, 1024)])
        tokens = _log(rng, 1, max(1, min(20000, 6496 * 5120 // dim)))
        branch = rng.random() < 0.7
        case = _norm("", tokens, dim, rng.choice(["bf16", "bf16", "f16", "f32"]), branch,
                     rng.choice(["none", "rms", "layer"]) if branch else "none",
                     rng.choice(["rms", "rms", "layer"]), rng.random() < 0.6, rng.choice([0, 1, rng.randint(2, 9)]),
                     rng.choice(["f32", "same"]))
        if case["dtype"] == "f32":
            case["tokens"] = max(1, tokens // 2)
    case.pop("name", None)
    return case


def _limits(case):
    """Per sequence: (q_len, k_len, list of (first row, rows, visible keys)) in runs of equal visibility."""
    out = []
    for ql, kl in zip(_ints(case["q_lens"]), _ints(case["k_lens"])):
        if not case["causal"]:
            out.append((ql, kl, ql * kl))
            continue
        b = case["block"]
        pairs = 0
        i = 0
        while i < ql:
            p = i + kl - ql
            lim = max(0, min(kl, (p // b + 1) * b))
            run = min(ql - i, b - p % b)  # rows up to the next block border share the limit
            pairs += run * lim
            i += run
        out.append((ql, kl, pairs))
    return out


def work(case):
    op = case["op"]
    if op == "attend":
        e = 2
        tq = sum(_ints(case["q_lens"]))
        lims = _limits(case)
        tk = sum(kl for ql, kl, _ in lims if ql)
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        bytes_ = 2 * tq * h * d * e + 2 * tk * kv * d * e + 4 * tq * h
        if case["history"]:
            bytes_ += tq * h * (d + 1) * 4
        return {"bytes": bytes_, "flops": 4 * d * h * sum(p for _, _, p in lims)}
    if op == "rotary":
        e = _DT[case["dtype"]].itemsize
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * e + case["tokens"] * len(_ints(case["dims"])) * 4,
                "flops": n * (6 if case["norm"] else 3)}
    if op == "tables":
        pairs = sum(_ints(case["dims"])) // 2
        return {"bytes": case["tokens"] * (8 * pairs + 4 * len(_ints(case["dims"]))),
                "flops": 40 * case["tokens"] * pairs}
    e = _DT[case["dtype"]].itemsize
    t, c = case["tokens"], case["dim"]
    me = 4 if case["mod_dtype"] == "f32" else e
    vecs = case["groups"] * (2 + case["branch"]) + case["weight"] + (case["post"] != "none")
    return {"bytes": t * c * e * (4 if case["branch"] else 2) + vecs * c * me + (4 * t if case["groups"] > 1 else 0),
            "flops": t * c * (6 + (4 if case["branch"] else 0) + (4 if case["post"] != "none" else 0))}


# ----------------------------------------------------------------- inputs
def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device=dev)

    op = case["op"]
    s = {}
    if op == "attend":
        dt = _DT[case["dtype"]]
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        tq, tk = sum(_ints(case["q_lens"])), sum(_ints(case["k_lens"]))
        # normed and rotated q / k: unit variance, k with a per-channel gain; v of a projection
        s["q"] = rnd(tq, h, d).to(dt)
        s["k"] = (rnd(tk, kv, d) * (1.0 + 0.3 * rnd(kv, d))).to(dt)
        s["v"] = (0.7 * rnd(tk, kv, d)).to(dt)
        if case["history"]:
            s["o_h"] = 0.05 * rnd(tq, h, d)
            s["lse_h"] = 8.0 + rnd(h, tq)
    elif op in ("rotary", "tables"):
        t = case["tokens"]
        n = len(_ints(case["dims"]))
        # frames, rows and columns of a video segment; far: a session hours long
        span = [200_000 if case["far"] else 64, 60, 104][:n]
        pos = [torch.randint(0, m, (t,), generator=g, device=dev, dtype=torch.int32) for m in span]
        s["positions"] = torch.stack(pos, dim=1).contiguous()
        if op == "rotary":
            dt = _DT[case["dtype"]]
            h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
            if case["fused"]:  # q | k | v of one projection
                x = rnd(t, h + 2 * max(kv, 1), d).to(dt)
                s["q"], s["k"] = x[:, :h], (x[:, h:h + kv] if kv else None)
            else:
                s["q"], s["k"] = rnd(t, h, d).to(dt), (rnd(t, kv, d).to(dt) if kv else None)
            s["qw"] = (1.0 + 0.1 * rnd(d)).to(dt) if case["norm"] else None
            s["kw"] = (1.0 + 0.1 * rnd(d)).to(dt) if case["norm"] and kv else None
    else:
        dt = _DT[case["dtype"]]
        md = torch.float32 if case["mod_dtype"] == "f32" else dt
        t, c, m = case["tokens"], case["dim"], case["groups"]
        s["x"] = (2.0 * rnd(t, c) + 0.5).to(dt)
        s["b"] = rnd(t, c).to(dt) if case["branch"] else None
        s["post_w"] = (1.0 + 0.1 * rnd(c)).to(md) if case["post"] != "none" else None
        s["w"] = (1.0 + 0.1 * rnd(c)).to(md) if case["weight"] else None
        s["gate"] = (0.5 * rnd(m, c)).to(md) if m and case["branch"] else None
        s["scale"] = (0.2 * rnd(m, c)).to(md) if m else None
        s["shift"] = (0.2 * rnd(m, c)).to(md) if m else None
        s["index"] = None
        if m > 1:  # tokens of one frame lie together
            per = -(-t // m)
            s["index"] = (torch.arange(t, device=dev) // per).to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        nk = _pkg()
        if case["op"] == "attend":
            s["plan"] = nk.AttendPlan(_ints(case["q_lens"]), case["heads"], kv_heads=case["kv_heads"],
                                      head_dim=case["head_dim"], k_lens=_ints(case["k_lens"]),
                                      causal=case["causal"], block=case["block"], device=s["q"].device)
        elif case["op"] in ("rotary", "tables"):
            s["axes"] = nk.RotaryAxes(tuple(_ints(case["dims"])), theta=10000.0,
                                      interleaved=case.get("interleaved", True))
    return s


# -------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)[case["op"]](case, state)


def _own_attend(case, s):
    nk = _pkg()
    history = (s["o_h"], s["lse_h"]) if case["history"] else None
    return nk.attend_packed(s["plan"], s["q"], s["k"], s["v"], history=history)


def _own_rotary(case, s):
    nk = _pkg()
    return nk.rotary(s["positions"], s["axes"], s["q"], k=s["k"], norm=case["norm"], q_weight=s["qw"],
                     k_weight=s["kw"])


def _own_tables(case, s):
    return _pkg().rope_tables(s["positions"], s["axes"])


def _own_norm(case, s):
    nk = _pkg()
    h, y = nk.residual_norm(s["x"], s["b"], gate=s["gate"], post=case["post"], post_weight=s["post_w"],
                            norm=case["norm"], weight=s["w"], scale=s["scale"], shift=s["shift"],
                            mod_index=s["index"])
    return (h, y) if case["branch"] else y


_run_own = {"attend": _own_attend, "rotary": _own_rotary, "tables": _own_tables, "norm": _own_norm}


def _plain_attend(case, s):
    q, k, v = s["q"], s["k"], s["v"]
    tq, h, d = q.shape
    kv = case["kv_heads"]
    grp = h // kv
    out = torch.zeros((tq, h, d), dtype=torch.float32, device=q.device)
    lse = torch.full((h, tq), -math.inf, dtype=torch.float32, device=q.device)
    q0 = k0 = 0
    for ql, kl in zip(_ints(case["q_lens"]), _ints(case["k_lens"])):
        if ql and kl:
            kk = k[k0:k0 + kl].float().permute(1, 2, 0)                    # kv, d, kl
            vv = v[k0:k0 + kl].float().permute(1, 0, 2)                    # kv, kl, d
            j = torch.arange(kl, device=q.device)
            step = max(1, min(ql, (1 << 28) // max(1, kl * h)))            # rows whose scores fit about 1 GB
            for r0 in range(0, ql, step):
                r1 = min(ql, r0 + step)
                qq = q[q0 + r0:q0 + r1].float().view(r1 - r0, kv, grp, d)
                qq = qq.permute(1, 2, 0, 3).reshape(kv, grp * (r1 - r0), d)
                sc = torch.matmul(qq, kk) * (1.0 / math.sqrt(d))
                sc = sc.view(kv, grp, r1 - r0, kl)
                if case["causal"]:
                    p = torch.arange(r0, r1, device=q.device) + (kl - ql)
                    lim = torch.div(p, case["block"], rounding_mode="floor") * case["block"] + case["block"]
                    sc = sc.masked_fill(j[None, :] >= lim[:, None], -math.inf)
                m = sc.amax(dim=-1, keepdim=True)
                m = torch.where(m == -math.inf, torch.zeros_like(m), m)
                e = torch.exp(sc - m)
                l = e.sum(dim=-1, keepdim=True)
                o = torch.matmul(e.view(kv, grp * (r1 - r0), kl), vv).view(kv, grp, r1 - r0, d)
                o = torch.where(l > 0, o / l, torch.zeros_like(o))
                out[q0 + r0:q0 + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, h, d)
                lse[:, q0 + r0:q0 + r1] = (m + torch.log(l)).view(h, r1 - r0)
        q0 += ql
        k0 += kl
    if case["history"]:
        m = torch.maximum(lse, s["lse_h"])
        a, b = torch.exp(lse - m), torch.exp(s["lse_h"] - m)
        wa, wb = (a / (a + b)).t()[:, :, None], (b / (a + b)).t()[:, :, None]
        out = out * wa + s["o_h"] * wb
        lse = m + torch.log(a + b)
    return out.to(q.dtype), lse


def _plain_angles(case, s):
    pos = s["positions"].to(torch.float64)
    cols = []
    for a, dims in enumerate(_ints(case["dims"])):
        i = torch.arange(0, dims, 2, device=pos.device, dtype=torch.float64)
        cols.append(pos[:, a:a + 1] * torch.pow(10000.0, -i / dims)[None, :])
    ang = torch.cat(cols, dim=1)
    return torch.cos(ang).float(), torch.sin(ang).float()


def _plain_rotary(case, s):
    cos, sin = _plain_angles(case, s)
    n = 2 * cos.shape[1]

    def one(x, w):
        f = x.float()
        if case["norm"]:
            f = f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + 1e-6) * w.float()
        c, sn = cos[:, None, :], sin[:, None, :]
        r = f[..., :n]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * c - b * sn, b * c + a * sn), dim=-1).flatten(-2)
        else:
            a, b = r[..., :n // 2], r[..., n // 2:]
            r = torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)
        return torch.cat((r, f[..., n:]), dim=-1).to(x.dtype)

    q = one(s["q"], s["qw"])
    return q if s["k"] is None else (q, one(s["k"], s["kw"]))


def _plain_norm(case, s):
    def nrm(f, kind):
        if kind == "layer":
            f = f - f.mean(dim=-1, keepdim=True)
        return f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + 1e-6)

    def row(v):
        v = v.float()
        return v[s["index"].long()] if s["index"] is not None else v

    h = s["x"].float()
    if case["branch"]:
        b = s["b"].float()
        if case["post"] != "none":
            b = nrm(b, case["post"]) * s["post_w"].float()
        h = h + (b * row(s["gate"]) if s["gate"] is not None else b)
    y = nrm(h, case["norm"])
    if s["w"] is not None:
        y = y * s["w"].float()
    if s["scale"] is not None:
        y = y * (1.0 + row(s["scale"])) + row(s["shift"])
    dt = s["x"].dtype
    return (h.to(dt), y.to(dt)) if case["branch"] else y.to(dt)


_run_plain = {"attend": _plain_attend, "rotary": _plain_rotary, "tables": _plain_angles, "norm": _plain_norm}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "attend":
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        q, k, v = s["q"].to(f64), s["k"].to(f64), s["v"].to(f64)
        out = torch.zeros(q.shape, dtype=f64, device=q.device)
        lse = torch.full((h, q.shape[0]), -math.inf, dtype=f64, device=q.device)
        qe = ke = 0
        for ql, kl in zip(_ints(case["q_lens"]), _ints(case["k_lens"])):
            qb, kb, qe, ke = qe, ke, qe + ql, ke + kl
            if not ql or not kl:
                continue
            key = torch.arange(kl, device=q.device)
            rows = max(1, min(ql, (1 << 26) // kl))
            for head in range(h):
                kh, vh = k[kb:ke, head * kv // h], v[kb:ke, head * kv // h]
                for a in range(0, ql, rows):
                    b = min(ql, a + rows)
                    sc = (q[qb + a:qb + b, head] @ kh.t()) / math.sqrt(d)
                    if case["causal"]:
                        last = torch.arange(a, b, device=q.device) + kl - ql
                        seen = (key[None, :] // case["block"]) <= torch.div(last, case["block"],
                                                                           rounding_mode="floor")[:, None]
                        sc = torch.where(seen, sc, torch.full_like(sc, -math.inf))
                    z = torch.logsumexp(sc, dim=1)
                    w = torch.exp(sc - torch.where(z.isinf(), torch.zeros_like(z), z)[:, None])
                    out[qb + a:qb + b, head] = w @ vh
                    lse[head, qb + a:qb + b] = z
        if case["history"]:
            o2, z2 = s["o_h"].to(f64), s["lse_h"].to(f64)
            z = torch.logaddexp(lse, z2)
            out = out * torch.exp(lse - z).t()[..., None] + o2 * torch.exp(z2 - z).t()[..., None]
            lse = z
        return out, lse
    if op in ("rotary", "tables"):
        parts = []
        for axis, dims in enumerate(_ints(case["dims"])):
            freq = torch.tensor([10000.0 ** (-2.0 * i / dims) for i in range(dims // 2)], dtype=f64,
                                device=s["positions"].device)
            parts.append(torch.outer(s["positions"][:, axis].to(f64), freq))
        angle = torch.cat(parts, dim=1)
        if op == "tables":
            return angle.cos(), angle.sin()
        half = angle.shape[1]
        turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]

        def rotate(x, w):
            y = x.to(f64)
            if case["norm"]:
                y = y / torch.sqrt((y * y).sum(dim=-1, keepdim=True) / y.shape[-1] + 1e-6) * w.to(f64)
            y = y.clone()
            first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
            second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q = rotate(s["q"], s["qw"])
        return q if s["k"] is None else (q, rotate(s["k"], s["kw"]))

    def unit(z, kind):
        mean = z.sum(dim=1, keepdim=True) / z.shape[1] if kind == "layer" else 0.0
        z = z - mean
        return z / ((z * z).sum(dim=1, keepdim=True) / z.shape[1] + 1e-6).sqrt()

    pick = s["index"].long() if s["index"] is not None else torch.zeros(case["tokens"], dtype=torch.long,
                                                                       device=s["x"].device)
    h = s["x"].to(f64)
    if case["branch"]:
        b = s["b"].to(f64)
        if case["post"] != "none":
            b = unit(b, case["post"]) * s["post_w"].to(f64)
        if s["gate"] is not None:
            b = b * s["gate"].to(f64).index_select(0, pick)
        h = h + b
    y = unit(h, case["norm"])
    if s["w"] is not None:
        y = y * s["w"].to(f64)
    if s["scale"] is not None:
        y = y + y * s["scale"].to(f64).index_select(0, pick) + s["shift"].to(f64).index_select(0, pick)
    return (h, y) if case["branch"] else y
