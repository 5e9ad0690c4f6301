"""64-bit CPU restatement of the token operators (attention with a bucketed relative bias, sandwich norm, token log probabilities) and of
their gradients, from the definitions; each also returns, where asked, the magnitudes that bound a 32-bit evaluation's error."""
import math

import torch

F64 = torch.float64


def rel_attention(q, k, v, table, bucket_map, heads, kv_heads, causal=False, scale=None, klen=None, qstart=None, dout=None):
    """q [B, Tq, H ch], k / v [B, Tk, Hk ch], table [nb, H], bucket_map [2R + 1] -> dict(out, lse[, dq, dk, dv, dtable]) and per-element error
    magnitudes e_* (see bound())."""
    q, k, v, table = (t.to(F64) for t in (q, k, v, table))
    B, Tq, C = q.shape
    Tk, ch, rep, R = k.shape[1], C // heads, heads // kv_heads, bucket_map.numel() // 2
    scale = 1.0 / math.sqrt(ch) if scale is None else scale
    out, lse = torch.zeros(B, Tq, heads, ch, dtype=F64), torch.full((B, heads, Tq), -math.inf, dtype=F64)
    r = dict(out=out, lse=lse, pv=torch.zeros_like(out), logit=torch.zeros_like(lse))
    if dout is not None:
        r.update(dq=torch.zeros_like(out), dk=torch.zeros(B, Tk, kv_heads, ch, dtype=F64), dv=torch.zeros(B, Tk, kv_heads, ch, dtype=F64),
                 dtable=torch.zeros_like(table))
        r.update({"a" + n: torch.zeros_like(r[n]) for n in ("dq", "dk", "dv", "dtable")})
        do = dout.to(F64).reshape(B, Tq, heads, ch)
    qh, kh, vh = q.reshape(B, Tq, heads, ch), k.reshape(B, Tk, kv_heads, ch), v.reshape(B, Tk, kv_heads, ch)
    for b in range(B):
        n = Tk if klen is None else max(0, min(Tk, int(klen[b])))
        pos = torch.arange(Tq) + (0 if qstart is None else int(qstart[b]))
        rel = torch.arange(n)[None] - pos[:, None]
        cell = bucket_map.long()[rel.clamp(-R, R) + R]
        ok = (cell >= 0) & (cell < table.shape[0])
        safe = torch.where(ok, cell, 0)
        seen = rel <= 0 if causal else torch.ones_like(rel, dtype=torch.bool)
        for h in range(heads):
            kk, vv, qq = kh[b, :n, h // rep], vh[b, :n, h // rep], qh[b, :, h]
            bias = torch.where(ok, table[safe, h], torch.zeros((), dtype=F64))
            s = torch.where(seen, scale * qq @ kk.T + bias, -math.inf)
            top = s.max(1).values if n else torch.full((Tq,), -math.inf, dtype=F64)
            live = top > -math.inf
            p = torch.where(live[:, None], torch.exp(s - torch.where(live, top, 0.0)[:, None]), 0.0)
            z = p.sum(1)
            p = p / torch.where(live, z, 1.0)[:, None]
            out[b, :, h] = p @ vv
            lse[b, h] = torch.where(live, top + torch.log(torch.where(live, z, 1.0)), -math.inf)
            r["pv"][b, :, h] = p @ vv.abs()
            size = abs(scale) * qq.abs() @ kk.abs().T + bias.abs()                  # magnitude behind each logit
            size = torch.where(p > 0, size, 0.0)
            r["logit"][b, h] = size.max(1).values if n else 0.0
            if dout is None:
                continue
            g = do[b, :, h]
            dp, D = g @ vv.T, (g * out[b, :, h]).sum(1, keepdim=True)
            ds = p * (dp - D)
            r["dq"][b, :, h] = scale * ds @ kk
            r["dk"][b, :n, h // rep] += scale * ds.T @ qq
            r["dv"][b, :n, h // rep] += p.T @ g
            r["dtable"][:, h].index_add_(0, safe.reshape(-1), torch.where(ok, ds, 0.0).reshape(-1))
            mag = p * (g.abs() @ vv.abs().T + (g.abs() * out[b, :, h].abs()).sum(1, keepdim=True))   # |dS| before cancellation
            r["adq"][b, :, h] = abs(scale) * mag @ kk.abs()
            r["adk"][b, :n, h // rep] += abs(scale) * mag.T @ qq.abs()
            r["adv"][b, :n, h // rep] += p.T @ g.abs()
            r["adtable"][:, h].index_add_(0, safe.reshape(-1), torch.where(ok, mag, 0.0).reshape(-1))
    flat = lambda t: t.reshape(t.shape[0], t.shape[1], -1)
    return {n: (flat(t) if t.dim() == 4 else t) for n, t in r.items()}


def _norm(t, kind, w, b, eps):
    if kind is None:
        return t
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    if w is not None:
        t = t * w
    return t if b is None else t + b


def sandwich_norm(x, y, post, post_w, post_b, gate, res_scale, pre, pre_w, pre_b, eps):
    """u = post(y); r = res_scale x + gate u; z = pre(r) in the tensors' own (64-bit) type; differentiable."""
    D = x.shape[-1]
    u = _norm(y, post, post_w, post_b, eps)
    if gate is not None:
        rows = x.numel() // D
        g = gate.reshape(-1, D)
        u = (u.reshape(g.shape[0], rows // g.shape[0], D) * g[:, None]).reshape(x.shape)
    r = res_scale * x + u
    return r, (_norm(r, pre, pre_w, pre_b, eps) if pre is not None else None)


def token_logprobs(logits, ids, k, t):
    """[rows, V] -> logprob, entropy, lse, top_ids, top_logprobs and all log probabilities in 64 bits; differentiable (top_ids aside).  The largest
    logit is taken off first: at -3e38 a 64-bit number has no room for a logarithm beside it."""
    x = logits.to(F64)
    top = x.max(1, keepdim=True).values.detach()
    live = top > -math.inf
    d = (x - torch.where(live, top, 0.0)) * t
    logs = torch.logsumexp(d, 1, keepdim=True)
    l = d - torch.where(live, logs, 0.0)
    lse = torch.where(live, top * t + logs, -math.inf)[:, 0]
    p = torch.exp(l)
    ent = -torch.where(p > 0, p * torch.where(p > 0, l, torch.zeros_like(l)), torch.zeros_like(p)).sum(1)
    V = x.shape[1]
    lp = torch.zeros_like(lse)
    if ids is not None:
        ok = (ids >= 0) & (ids < V)
        lp = torch.where(ok, l.gather(1, torch.where(ok, ids, 0)[:, None])[:, 0], lp)
    key = torch.nan_to_num(x, nan=math.inf, posinf=1.7e308, neginf=-math.inf)
    best = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    return lp, ent, lse, best, l.gather(1, best), l
