"""The operators around the expert GEMMs in 64 bits on the CPU: plain
restatements from their definitions, used by the tests only."""
import math

import torch

U = 2.0 ** -24                       # half a step of fp32, relative


def half_step(t):
    """Largest relative rounding error of a type."""
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half of the type's smallest step (what a rounding in its subnormals costs)."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def norm(x, weight, residual, eps):
    s = x.double().cpu()
    if residual is not None:
        s = s + residual.double().cpu()
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + eps) * weight.double().cpu()
    return y, s


def clean(z):
    z = z.double().cpu()
    return torch.where(torch.isnan(z), -math.inf, z).clamp(max=float(torch.finfo(torch.float32).max))


def scores(z, scoring):
    """Scores of cleaned logits; closed experts and rows without an open one have zeros."""
    if scoring == "sigmoid":
        return torch.sigmoid(z)
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - torch.where(m == -math.inf, 0.0, m))
    return e / e.sum(1, keepdim=True).clamp(min=1e-300)


def route(logits, topk, scoring="softmax", bias=None, n_group=1, topk_group=1, group_top=2,
          renormalize=False, scale=1.0, token_mask=None):
    """(weights float64, ids int64), token by token in plain Python."""
    z = clean(logits)
    p = scores(z, scoring)
    T, E = z.shape
    monotone = bias is None and (n_group == 1 or group_top == 1)
    key = z.clone() if monotone else p.clone()
    if bias is not None:
        b = bias.double().cpu()
        key = key + b
        key[:, torch.isnan(b) | (b == -math.inf)] = -math.inf
    key[z == -math.inf] = -math.inf
    ids = torch.full((T, topk), -1, dtype=torch.int64)
    G = E // n_group
    for t in range(T):
        if token_mask is not None and not bool(token_mask[t]):
            continue
        row = key[t].tolist()
        live = [e for e in range(E) if row[e] > -math.inf]
        if n_group > 1:
            total = {}
            for g in range(n_group):
                best = sorted((row[e] for e in live if e // G == g), reverse=True)[:group_top]
                if best:
                    total[g] = math.fsum(best)
            kept = sorted(total, key=lambda g: (-total[g], g))[:topk_group]
            live = [e for e in live if e // G in kept]
        chosen = sorted(live, key=lambda e: (-row[e], e))[:topk]
        ids[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int64)
    return weights(z, ids, scoring, renormalize, scale), ids


def weights(z, ids, scoring, renormalize, scale):
    """Weights of given ids (negative: none) from cleaned logits."""
    at = ids.clamp(min=0)
    if not renormalize:
        return scale * torch.where(ids >= 0, scores(z, scoring).gather(1, at), 0.0)
    log = torch.nn.functional.logsigmoid(z) if scoring == "sigmoid" else z
    log = torch.where(ids >= 0, log.gather(1, at), -math.inf)
    m = log.detach().max(1, keepdim=True).values
    e = torch.exp(log - torch.where(m == -math.inf, 0.0, m))
    return scale * e / e.sum(1, keepdim=True).clamp(min=1e-300)


def route_grad(grad, logits, ids, scoring, renormalize, scale):
    """By automatic differentiation of the definition in 64 bits, ids fixed."""
    z = clean(logits).requires_grad_(True)
    ids = ids.long().cpu()
    ids = torch.where((ids >= 0) & (ids < z.shape[1]), ids, -1)
    w = weights(z, ids, scoring, renormalize, scale)
    w.backward(torch.where(ids >= 0, grad.double().cpu(), 0.0))
    return torch.where(torch.isinf(z.detach()), 0.0, torch.nan_to_num(z.grad))


def balance(logits, ids, coef, scoring="softmax", token_mask=None, grad=1.0):
    """(loss, counts, prob_sums, n, dlogits)."""
    z = clean(logits)
    T, E = z.shape
    live = torch.ones(T, dtype=torch.bool) if token_mask is None else token_mask.cpu()
    ids = ids.cpu().long()
    hit = ids[live]
    hit = hit[(hit >= 0) & (hit < E)]
    counts = torch.bincount(hit.flatten(), minlength=E)
    zl = z[live].requires_grad_(True)
    open_ = ~torch.isinf(zl).all(1, keepdim=True)
    if scoring == "sigmoid":
        s = torch.sigmoid(zl)
        p = s / torch.where(s.sum(1, keepdim=True) > 0, s.sum(1, keepdim=True), 1.0)
    else:
        p = torch.softmax(torch.where(open_, zl, 0.0), 1) * open_
    n = int(live.sum())
    dz = torch.zeros(T, E, dtype=torch.float64)
    if n == 0:
        return 0.0, counts, torch.zeros(E, dtype=torch.float64), 0, dz
    loss = coef * E / (ids.shape[1] * n * n) * (counts.double() * p.sum(0)).sum()
    (loss * grad).backward()
    dz[live] = torch.where(torch.isinf(zl.detach()), 0.0, torch.nan_to_num(zl.grad))
    return float(loss.detach()), counts, p.sum(0).detach(), n, dz


def int4(x, w, scale, zero=None, bias=None):
    """(y, sum of |products|)."""
    x, w, scale = x.double().cpu(), w.cpu().long(), scale.double().cpu()
    K, N = w.shape[0] * 8, w.shape[1]
    q = torch.stack([(w >> (4 * j)) & 15 for j in range(8)], 1).reshape(K, N).double()
    group = K // scale.shape[0]
    if zero is None:
        z = torch.full((scale.shape[0], N), 8.0, dtype=torch.float64)
    else:
        zl = zero.cpu().long()
        z = torch.stack([(zl >> (4 * j)) & 15 for j in range(8)], 2).reshape(-1, N).double()
    wd = (q - z.repeat_interleave(group, 0)) * scale.repeat_interleave(group, 0)
    y = x @ wd
    if bias is not None:
        y = y + bias.double().cpu()
    return y, x.abs() @ wd.abs()
