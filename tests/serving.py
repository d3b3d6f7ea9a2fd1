"""Plain forms in 64 bits of the serving operators (paged cache append, attention of one new token, expert routing) and the inputs
that their tests share."""
import ctypes as C
import math

import numpy as np
import torch

BF16_HALF, F32_HALF = 2.0 ** -8, 2.0 ** -24      # half a step of a rounding, relative to the value


def stream():
    return torch.cuda.current_stream().cuda_stream


def run(capi, entry, desc):
    """The call and everything in front of it done: its status, or the one that the kernels left."""
    st = stream()
    rc = entry(C.byref(desc), st)
    return rc if rc != capi.SUCCESS else capi.lib.b200dnn_stream_status(st)


class Cache:
    """A paged cache whose every byte that no test writes is a NaN (bf16) or has a NaN for a scale (s8)."""

    def __init__(self, pages, page, heads, dim, dt, layout="tokens", pad=0, device="cuda"):
        self.dt, self.page, self.heads, self.dim = dt, page, heads, dim
        shape = [pages, page, heads, dim + pad] if layout == "tokens" else [pages, heads, page, dim + pad]
        turn = (lambda t: t) if layout == "tokens" else (lambda t: t.transpose(1, 2))
        self.scale = [None, None]
        if dt == "s8":
            self.kv = [turn(torch.full(shape, 77, dtype=torch.int8, device=device))[..., :dim] for _ in range(2)]
            self.scale = [turn(torch.full(shape[:3], math.nan, device=device)) for _ in range(2)]
        else:
            self.kv = [turn(torch.full(shape, math.nan, dtype=torch.bfloat16, device=device))[..., :dim] for _ in range(2)]

    def desc(self, capi):
        return capi.make_kv_cache(*self.kv, *self.scale)

    def put(self, which, pages, offs, x):
        """x [n, heads, dim] f64 into the rows: rounded to bf16, or codes with a scale that leaves no code out of range."""
        if self.dt == "s8":
            s = (x.abs().amax(-1) / 127.0).float().clamp_(min=1e-10)
            self.scale[which][pages, offs] = s
            self.kv[which][pages, offs] = (x / s.double()[..., None]).round().clamp(-127, 127).to(torch.int8)
        else:
            self.kv[which][pages, offs] = x.to(torch.bfloat16)

    def rows(self, which, pages, offs):
        """[n, heads, dim] in 64 bits: what the cache holds there."""
        x = self.kv[which][pages, offs].double()
        return x * self.scale[which][pages, offs].double()[..., None] if self.dt == "s8" else x

    def bits(self):
        """A copy of every byte, to see what a call has left alone."""
        return [t.reshape(-1).clone().view(torch.uint8) for t in self.kv + [s for s in self.scale if s is not None]]


def tables(rows, rot, device="cuda", pad=0):
    """cos and sin [rows, rot / 2] f32 (rows `pad` elements longer than that apart)."""
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    got = []
    for t in (angle.cos(), angle.sin()):
        wide = torch.zeros(rows, rot // 2 + pad)
        wide[:, :rot // 2] = t.float()
        got.append(wide.to(device)[:, :rot // 2])
    return got


def rotated(x, positions, cos, sin, interleaved):
    """x [n, heads, dim] f64 rotated, and the sum |a| + |b| behind every element, by which its rounding errors are bounded."""
    rot = 2 * cos.shape[1]
    y, size = x.clone(), torch.zeros_like(x)
    first = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    c, s = (t.double()[positions.long()][:, None] for t in (cos, sin))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return y, size


def attention(q, cache, table, lens, scale=0.0, window=0, softcap=0.0, sinks=None):
    """out, lse and, for both, how far a computation in f32 with probabilities to 16 bits may lie from them.

    A score is a sum of dim products in f32, a few operations on it and an exponential: off by dz <= (dim + 8) 2^-24 sum |q k| scale + 2^-20 |z| (the scale, the cap's
    tanh and the change of base, each a few roundings).  A probability is off by 2 dz relatively, and by 2^-15 for its own roundings, a sum of n of them by n 2^-24."""
    B, H, D = q.shape
    g = H // cache.heads
    out, lse = torch.zeros(B, H, D, dtype=torch.float64, device=q.device), torch.full((B, H), -math.inf, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    scale = scale or D ** -0.5
    for i, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        at = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        pages, offs = table[i].long()[at // cache.page], at % cache.page
        k, v = (cache.rows(w, pages, offs).transpose(0, 1) for w in (0, 1))      # [key head, key, dim]
        x = q[i].double().view(-1, g, D)
        z, size = x @ k.transpose(1, 2) * scale, x.abs() @ k.abs().transpose(1, 2) * abs(scale)
        dz = ((D + 8) * F32_HALF * size + 2.0 ** -20 * z.abs()).amax(-1)
        if softcap:
            z = softcap * torch.tanh(z / softcap)
        w = torch.cat((z, sinks.double().view(-1, g, 1)), -1) if sinks is not None else z
        total = torch.logsumexp(w, -1)
        p = torch.exp(z - total[..., None])
        off = 2 * dz + 2.0 ** -15 + len(at) * F32_HALF
        out[i], lse[i] = (p @ v).view(H, D), total.view(H)
        tol[i], ltol[i] = (off[..., None] * (p @ v.abs())).view(H, D), (off + 2.0 ** -20 * total.abs()).view(H)
    return out, lse, tol, ltol


def gate(x, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renorm=True, scale=1.0):
    """numpy, in 64 bits: ids, weights, rows per expert and every slot's row."""
    T, E = x.shape
    x = x.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        s = 1.0 / (1.0 + np.exp(-x)) if score == "sigmoid" else np.exp(x - x.max(1, keepdims=True)) / np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)
    c = s if bias is None else s + bias.astype(np.float64)
    c = np.where(np.isnan(c), -np.inf, c)
    per = E // groups
    ids, w = np.zeros((T, k), np.int32), np.zeros((T, k))
    for t in range(T):
        row = c[t]
        if groups > 1:
            best = -np.sort(-row.reshape(groups, per), 1)
            rank = best[:, 0] if group_score == "max" or per == 1 else best[:, 0] + best[:, 1]
            out = np.argsort(-rank, kind="stable")[top_groups:]
            keep = np.ones(groups, bool)
            keep[out] = False
            candidates = np.flatnonzero(np.repeat(keep, per))
        else:
            candidates = np.arange(E)
        ids[t] = candidates[np.argsort(-row[candidates], kind="stable")[:k]]
        w[t] = s[t, ids[t]]
        if renorm:
            w[t] /= w[t].sum()
    flat = ids.reshape(-1)
    rows = np.empty(T * k, np.int32)
    rows[np.argsort(flat, kind="stable")] = np.arange(T * k, dtype=np.int32)
    return ids, w * scale, np.bincount(flat, minlength=E).astype(np.int32), rows.reshape(T, k)
