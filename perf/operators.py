"""Cases for timing and checking the operators around the expert GEMMs.

Four operators, each in a plain form (elementary torch operations) and, with
``own`` true, as a user's program calls them:

* ``norm``    residual addition + RMS norm + 1x128 FP8 rows (``ops.add_rms_norm``);
* ``route``   expert choice and weights from router logits, with the gradient
  of the logits in training cases (``ops.moe_route``, ``ops.moe_route_backward``);
* ``balance`` balance loss, per-expert counts and its gradient
  (``ops.moe_balance_loss``, ``ops.moe_balance_loss_backward``);
* ``int4``    few tokens times a 4-bit weight matrix (``ops.int4_linear``).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
COEF = 1e-2


# ------------------------------------------------------------------ the cases

def _norm(name, T, K, dtype="bf16", fp8=True, residual=True):
    return {"name": name, "op": "norm", "T": T, "K": K, "dtype": dtype, "fp8": fp8,
            "residual": residual}


def _route(name, T, E, topk, dtype="fp32", scoring="softmax", bias=False, groups=1, keep=1,
           group_top=2, renorm=True, pad=0.0, masked=0, train=False):
    return {"name": name, "op": "route", "T": T, "E": E, "topk": topk, "dtype": dtype,
            "scoring": scoring, "bias": bias, "groups": groups, "keep": keep,
            "group_top": group_top, "renorm": renorm, "pad": pad, "masked": masked, "train": train}


def _balance(name, T, E, topk, dtype="fp32", scoring="softmax", pad=0.0):
    return {"name": name, "op": "balance", "T": T, "E": E, "topk": topk, "dtype": dtype,
            "scoring": scoring, "pad": pad}


def _int4(name, T, K, N, group=32, dtype="bf16", zeros=False, bias=False):
    return {"name": name, "op": "int4", "T": T, "K": K, "N": N, "group": group, "dtype": dtype,
            "zeros": zeros, "bias": bias}


def listed():
    return [
        # one token's norm before the expert layer, latency alone
        _norm("norm_1_token", 1, 7168),
        # a ragged batch of a narrow model, no quantised output, odd row length
        _norm("norm_ragged_fp16", 1021, 1001, dtype="fp16", fp8=False),
        # the expert-parallel prefill batch: norm, residual stream and FP8 rows
        _norm("norm_prefill", 32768, 7168),
        # one decode batch of 128 tokens, sigmoid scores with a selection bias and 4 of 8 groups
        _route("route_decode_groups", 128, 256, 8, scoring="sigmoid", bias=True, groups=8, keep=4),
        # a small model's training batch: softmax weights not renormalised, padded rows, gradient
        _route("route_train_small", 4099, 60, 4, dtype="bf16", renorm=False, pad=0.1, train=True),
        # a prefill batch of 32768 tokens over 256 experts, sigmoid with bias, gradient too
        _route("route_prefill", 32768, 256, 8, scoring="sigmoid", bias=True, groups=8, keep=4,
               train=True),
        # 8 experts, a short batch: counts, loss, gradient
        _balance("balance_small", 256, 8, 2),
        # a padded training batch over 160 experts in bf16, sigmoid scores
        _balance("balance_padded_bf16", 5003, 160, 6, dtype="bf16", scoring="sigmoid", pad=0.2),
        # the whole prefill-sized training batch over 256 experts
        _balance("balance_large", 32768, 256, 8),
        # single-token decode through a shared expert's gate+up projection, group 32
        _int4("int4_1_token", 1, 7168, 4096),
        # five tokens through an odd-sized projection with zero points and a bias, fp16
        _int4("int4_zeros_fp16", 5, 2048, 7176, group=128, dtype="fp16", zeros=True, bias=True),
        # a decode batch of 16 tokens through a dense layer's wide projection
        _int4("int4_16_tokens", 16, 7168, 32768),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    case = _draw(rng, rng.choice(["norm", "route", "balance", "int4"]))
    del case["name"]
    return case


def _draw(rng, op):
    if op == "norm":
        fp8 = rng.random() < 0.6
        K = 128 * _log(rng, 1, 128) if fp8 else _log(rng, 64, 16384)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 2_000_000_000 // (K * (4 * SIZE[dtype] + 1))
        return _norm("", _log(rng, 1, max(1, min(32768, most))), K, dtype, fp8, rng.random() < 0.8)
    if op in ("route", "balance"):
        E = _log(rng, 8, 512)
        T = _log(rng, 1, max(1, min(32768, 8_000_000 // E)))
        topk = rng.randint(1 if T >= 64 else 2, min(E, 10))
        scoring = rng.choice(["softmax", "sigmoid"])
        pad = rng.choice([0.0, 0.0, rng.uniform(0.0, 0.5)])
        if op == "balance":
            return _balance("", T, E, topk, rng.choice(["fp32", "bf16"]), scoring, pad)
        groups, keep = 1, 1
        if rng.random() < 0.4:
            groups = rng.choice([2, 4])
            E = E // groups * groups
            keep = rng.randint(1, groups)
            topk = min(topk, keep * (E // groups))
        return _route("", T, E, topk, rng.choice(["fp32", "fp32", "bf16", "fp16"]), scoring,
                      rng.random() < 0.5, groups, keep, rng.choice([1, 2]), rng.random() < 0.6,
                      pad, rng.choice([0, 0, rng.randint(0, E - 1)]), rng.random() < 0.6)
    group = rng.choice([32, 64, 128])
    K = group * _log(rng, 256 // group, 16384 // group)
    T = _log(rng, 1, 32)
    N = 8 * _log(rng, 8, min(4096, 230_000_000 // (8 * K * max(1, T // 16))))
    return _int4("", T, K, N, group, rng.choice(["bf16", "fp16"]), rng.random() < 0.4,
                 rng.random() < 0.4)


# ----------------------------------------------------------------- the inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    T = case["T"]
    s = {"case": case}
    if case["op"] == "norm":
        K = case["K"]
        channel = torch.exp(0.5 * normal(K)).to(dt)        # some channels are much larger
        s["x"] = normal(T, K, dtype=dt) * channel
        s["residual"] = normal(T, K, dtype=dt) * channel if case["residual"] else None
        s["weight"] = (1 + 0.1 * normal(K)).to(dt)
        return s
    if case["op"] in ("route", "balance"):
        E, topk = case["E"], case["topk"]
        s["logits"] = (1.5 * normal(T, E) + 0.7 * normal(E)).to(dt)   # some experts are popular
        live = torch.rand(T, generator=g, device="cuda") >= case["pad"]
        live[:1] = True
        s["mask"] = live if case["pad"] > 0 else None
        if case["op"] == "route":
            if case["masked"]:                             # experts closed to some of the tokens
                shut = torch.rand(T, E, generator=g, device="cuda") < case["masked"] / E
                shut[:1] = False
                s["logits"].masked_fill_(shut, -math.inf)
            s["bias"] = 0.05 * normal(E) if case["bias"] else None
            s["grad"] = normal(T, topk) if case["train"] else None
        else:
            s["ids"] = s["logits"].float().argsort(dim=1, descending=True)[:, :topk] \
                .to(torch.int32).contiguous()
            if s["mask"] is not None:
                s["ids"].masked_fill_(~live[:, None], -1)  # as the router leaves padded rows
            s["grad"] = 1 + 0.1 * normal(1).reshape(())
        return s
    K, N, G = case["K"], case["N"], case["K"] // case["group"]
    s["x"] = normal(T, K, dtype=dt)
    s["w"] = torch.randint(-2 ** 31, 2 ** 31, (K // 8, N), generator=g, device="cuda",
                           dtype=torch.int64).to(torch.int32)
    s["scale"] = (0.01 * normal(G, N).abs() + 1e-4).to(dt)
    s["zero"] = torch.randint(-2 ** 31, 2 ** 31, (G, N // 8), generator=g, device="cuda",
                              dtype=torch.int64).to(torch.int32) if case["zeros"] else None
    s["bias"] = normal(N, dtype=dt) if case["bias"] else None
    return s


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"norm": _plain_norm, "route": _plain_route, "balance": _plain_balance,
            "int4": _plain_int4}[c["op"]](s, c)


def _own(s, c):
    from ferret_b200 import ops
    if c["op"] == "norm":
        return ops.add_rms_norm(s["x"], s["weight"], s["residual"], EPS, quant=c["fp8"])
    if c["op"] == "route":
        w, ids = ops.moe_route(s["logits"], c["topk"], scoring=c["scoring"], bias=s["bias"],
                               n_group=c["groups"], topk_group=c["keep"],
                               group_top=c["group_top"], renormalize=c["renorm"], scale=2.5,
                               token_mask=s["mask"])
        if not c["train"]:
            return w, ids
        return w, ids, ops.moe_route_backward(s["grad"], s["logits"], ids, scoring=c["scoring"],
                                              renormalize=c["renorm"], scale=2.5)
    if c["op"] == "balance":
        loss, counts, sums, live = ops.moe_balance_loss(s["logits"], s["ids"], COEF,
                                                        scoring=c["scoring"], token_mask=s["mask"])
        grad = ops.moe_balance_loss_backward(s["grad"], s["logits"], counts, live, c["topk"], COEF,
                                             scoring=c["scoring"], token_mask=s["mask"])
        return loss, counts, sums, live, grad
    return ops.int4_linear(s["x"], s["w"], s["scale"], w_zero=s["zero"], bias=s["bias"])


# ------------------------------------------------------------ the plain forms

def _plain_norm(s, c):
    dt = DTYPES[c["dtype"]]
    v = s["x"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    y = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    out = (y.to(dt), None if s["residual"] is None else v.to(dt))
    if not c["fp8"]:
        return out + (None, None)
    b = y.reshape(c["T"], c["K"] // 128, 128)
    amax = b.abs().amax(2, keepdim=True).clamp(min=1e-4)
    q = (b * (448.0 / amax)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return out + (q.reshape(c["T"], c["K"]), (amax / 448.0).squeeze(2))


def _plain_scores(z, scoring):
    """Scores of float64 logits; a row of nothing but -inf has zeros."""
    if scoring == "sigmoid":
        return torch.sigmoid(z)
    e = torch.exp(z - z.amax(1, keepdim=True).clamp(min=-1e300))
    return e / e.sum(1, keepdim=True).clamp(min=1e-300)


def _plain_route(s, c):
    T, E, k = c["T"], c["E"], c["topk"]
    # 64 bits: which of two near scores is the larger decides a whole number
    z = s["logits"].double()
    p = _plain_scores(z, c["scoring"])
    key = z if s["bias"] is None and (c["groups"] == 1 or c["group_top"] == 1) else p
    if s["bias"] is not None:
        key = p + s["bias"].double()
    key = key.masked_fill(torch.isneginf(z), -math.inf)
    if c["groups"] > 1:
        per = key.reshape(T, c["groups"], E // c["groups"])
        best = per.sort(dim=2, descending=True).values[:, :, :c["group_top"]]
        score = best.masked_fill(torch.isneginf(best), 0).sum(2)
        score = score.masked_fill(torch.isneginf(best[:, :, 0]), -math.inf)
        chosen = score.sort(dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        open_ = torch.zeros(T, c["groups"], dtype=torch.bool, device=z.device)
        open_.scatter_(1, chosen, True)
        key = per.masked_fill(~open_[:, :, None], -math.inf).reshape(T, E)
    top = key.sort(dim=1, descending=True, stable=True)
    ids, have = top.indices[:, :k], ~torch.isneginf(top.values[:, :k])
    if s["mask"] is not None:
        have = have & s["mask"][:, None]
    sel = torch.where(have, p.gather(1, ids), 0)
    total = sel.sum(1, keepdim=True)
    w = sel / torch.where(total > 0, total, 1) if c["renorm"] else sel
    out = ((2.5 * w).float(), torch.where(have, ids, -1).to(torch.int32))
    if not c["train"]:
        return out
    g = torch.where(have, 2.5 * s["grad"].double(), 0)
    if c["renorm"]:
        d_sel = (g - (g * w).sum(1, keepdim=True)) / torch.where(total > 0, total, 1)
        d_sel = torch.where(have, d_sel, 0)
    else:
        d_sel = g
    dp = torch.zeros(T, E, dtype=torch.float64, device=z.device).scatter_add_(1, ids, d_sel)
    if c["scoring"] == "sigmoid":
        dz = dp * p * (1 - p)
    else:
        dz = p * (dp - (dp * p).sum(1, keepdim=True))
    return out + (dz.to(DTYPES[c["dtype"]]),)


def _plain_balance(s, c):
    T, E, k = c["T"], c["E"], c["topk"]
    z = s["logits"].float()
    if c["scoring"] == "sigmoid":
        sig = torch.sigmoid(z)
        p = sig / sig.sum(1, keepdim=True)
    else:
        e = torch.exp(z - z.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    live = torch.ones(T, dtype=torch.bool, device=z.device) if s["mask"] is None else s["mask"]
    n = live.sum()
    ids = s["ids"].long()
    ok = (ids >= 0) & live[:, None]
    counts = torch.zeros(E, dtype=torch.int64, device=z.device)
    counts.scatter_add_(0, torch.where(ok, ids, 0).reshape(-1), ok.long().reshape(-1))
    sums = torch.where(live[:, None], p, 0).double().sum(0)      # long sums
    factor = COEF * E / (k * n.clamp(min=1).double().square())
    loss = factor * (counts * sums).sum()
    # the counts' mean taken off: what is left is the difference that matters
    centred = (counts - counts.double().mean()).float()
    inner = centred - (p * centred).sum(1, keepdim=True)
    dz = p * inner * (s["grad"] * factor.float())
    if c["scoring"] == "sigmoid":
        dz = dz * (1 - sig)
    dz = torch.where(live[:, None], dz, 0)
    return (loss.float(), counts.to(torch.int32), sums.float(),
            n.to(torch.int32).reshape(1), dz.to(DTYPES[c["dtype"]]))


def _plain_int4(s, c):
    K, N, group = c["K"], c["N"], c["group"]
    shift = torch.arange(0, 32, 4, device=s["w"].device, dtype=torch.int32)
    q = ((s["w"][:, None, :] >> shift[None, :, None]) & 15).reshape(K // group, group, N).float()
    if s["zero"] is None:
        zero = 8.0
    else:
        zero = ((s["zero"][:, :, None] >> shift) & 15).reshape(K // group, 1, N).float()
    w = ((q - zero) * s["scale"].float()[:, None, :]).reshape(K, N)
    y = s["x"].float() @ w
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[c["dtype"]])


# ----------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "route": _exact_route, "balance": _exact_balance,
            "int4": _exact_int4}[case["op"]](s, case)


def _exact_norm(s, c):
    v = s["x"].to(torch.float64)
    if s["residual"] is not None:
        v += s["residual"].to(torch.float64)
    norm2 = torch.linalg.vector_norm(v, dim=1, dtype=torch.float64) ** 2
    y = s["weight"].to(torch.float64) * v / torch.sqrt(norm2 / c["K"] + EPS)[:, None]
    r = None if s["residual"] is None else v
    if not c["fp8"]:
        return y, r, None, None
    blocks = y.unflatten(1, (-1, 128))
    top = torch.maximum(blocks.max(2).values, -blocks.min(2).values).clamp(min=1e-4)
    return y, r, (448 * blocks / top[:, :, None]).flatten(1), top / 448


def _exact_route(s, c):
    T, E, k = c["T"], c["E"], c["topk"]
    z = s["logits"].to(torch.float64)
    shut = z == -math.inf
    if c["scoring"] == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
    else:
        p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)).masked_fill(shut, 0)
    bare = s["bias"] is None and (c["groups"] == 1 or c["group_top"] == 1)
    key = z.clone() if bare else p if s["bias"] is None else p + s["bias"].to(torch.float64)
    key = key.masked_fill(shut, -math.inf)
    rows = torch.arange(T, device=z.device)
    if c["groups"] > 1:
        per = E // c["groups"]
        score = torch.full((T, c["groups"]), -math.inf, dtype=torch.float64, device=z.device)
        for j in range(c["groups"]):
            part = key[:, j * per:(j + 1) * per].clone()
            for n in range(min(c["group_top"], per)):
                v, at = part.max(1)
                score[:, j] = v if n == 0 else score[:, j] + torch.where(v == -math.inf, 0, v)
                part[rows, at] = -math.inf
        for _ in range(c["groups"] - c["keep"]):           # the worst, the last of equals first
            worst = c["groups"] - 1 - score.flip(1).argmin(1)
            at = worst[:, None] * per + torch.arange(per, device=z.device)
            key.scatter_(1, at, -math.inf)
            score[rows, worst] = math.inf
    chosen = torch.zeros(T, E, dtype=torch.bool, device=z.device)
    ids = []
    for _ in range(k):
        v = key.max(1, keepdim=True).values
        at = (key == v).to(torch.int8).argmax(1)           # the first of equals
        have = v[:, 0] > -math.inf
        if s["mask"] is not None:
            have = have & s["mask"]
        ids.append(torch.where(have, at, -1))
        chosen[rows, at] |= have
        key[rows, at] = -math.inf
    ids = torch.stack(ids, 1)
    sel = torch.where(chosen, p, 0)
    total = sel.sum(1, keepdim=True)
    w_all = sel / total.clamp(min=1e-320) if c["renorm"] else sel
    w = torch.where(ids >= 0, 2.5 * w_all.gather(1, ids.clamp(min=0)), 0)
    if not c["train"]:
        return w, None
    g = torch.zeros(T, E, dtype=torch.float64, device=z.device)
    for j in range(k):
        have = ids[:, j] >= 0
        g[rows[have], ids[have, j]] = 2.5 * s["grad"][have, j].to(torch.float64)
    mean = (g * w_all).sum(1, keepdim=True)
    if c["renorm"]:
        # d log w_i / d z_j = (log s_j)' (1[i = j] - w_j)
        slope = torch.where(chosen, 1 - p, 0) if c["scoring"] == "sigmoid" else chosen.double()
        dz = w_all * slope * (g - mean)
    elif c["scoring"] == "sigmoid":
        dz = g * sel * (1 - p)
    else:
        dz = g * sel - p * mean
    return w, None, dz


def _exact_balance(s, c):
    E, k = c["E"], c["topk"]
    keep = slice(None) if s["mask"] is None else s["mask"].nonzero()[:, 0]
    z = s["logits"][keep].to(torch.float64)
    n = z.shape[0]
    hit = s["ids"][keep].flatten()
    counts = torch.bincount(hit[hit >= 0].long(), minlength=E).to(torch.float64)
    if c["scoring"] == "sigmoid":
        sig = 1 / (1 + torch.exp(-z))
        p = sig / sig.sum(1, keepdim=True)
        slope = 1 - sig
    else:
        p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
        slope = torch.ones((), dtype=torch.float64, device=z.device)
    factor = COEF * E / (k * max(n, 1) ** 2)
    loss = factor * torch.dot(counts, p.sum(0))
    dz = torch.zeros(c["T"], E, dtype=torch.float64, device=z.device)
    dz[keep] = s["grad"].to(torch.float64) * factor * p * slope * (counts - (p @ counts)[:, None])
    return loss, None, p.sum(0), None, dz


def _exact_int4(s, c):
    K, N, G = c["K"], c["N"], c["K"] // c["group"]
    y = torch.zeros(c["T"], N, dtype=torch.float64, device=s["x"].device)
    scale = s["scale"].to(torch.float64).repeat_interleave(c["group"] // 8, 0)
    zero = 8.0
    if s["zero"] is not None:
        zero = torch.empty(G, N, dtype=torch.float64, device=s["x"].device)
        for j in range(8):
            zero[:, j::8] = s["zero"].bitwise_right_shift(4 * j).bitwise_and(15).double()
        zero = zero.repeat_interleave(c["group"] // 8, 0)
    for j in range(8):
        q = s["w"].bitwise_right_shift(4 * j).bitwise_and(15).to(torch.float64)
        y += s["x"][:, j::8].to(torch.float64) @ (scale * (q - zero))
    return y if s["bias"] is None else y + s["bias"].to(torch.float64)


# ------------------------------------------------------------------- the work

def work(case):
    T, size = case["T"], SIZE[case["dtype"]]
    if case["op"] == "norm":
        n = T * case["K"]
        moved = n * size * (4 if case["residual"] else 2) + case["K"] * size
        return {"bytes": moved + (n + n // 32 if case["fp8"] else 0), "flops": 8 * n}
    if case["op"] == "route":
        n, m = T * case["E"], T * case["topk"]
        train = n * size + 4 * m if case["train"] else 0
        return {"bytes": n * size + 8 * m + train + (T if case["pad"] else 0), "flops": 8 * n}
    if case["op"] == "balance":
        n = T * case["E"]
        return {"bytes": 2 * n * size + 4 * T * case["topk"] + 8 * case["E"]
                + (T if case["pad"] else 0), "flops": 12 * n}
    K, N, G = case["K"], case["N"], case["K"] // case["group"]
    return {"bytes": K * N // 2 + 2 * G * N + (G * N // 2 if case["zeros"] else 0)
            + 2 * T * (K + N) + (2 * N if case["bias"] else 0), "flops": 2 * T * K * N}
