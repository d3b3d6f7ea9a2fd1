"""The operators that serve a decoder layer token by token, as cases that can be timed beside their plain form: appending rotated keys and
values to a paged cache (b200dnn_kv_append), attention of one new token over that cache (b200dnn_paged_attention), and the routing of tokens to
experts with a balance bias and groups (b200dnn_moe_gate).

  own               False: run() computes the plain form with elementary torch operations; True: it makes the library's calls
  listed()          the fixed cases
  draw(rng)         one more case of the same ranges
  prepare(case, s)  inputs of one case, made on the GPU from the seed s
  run(state)        one pass through the operator; returns its outputs
  work(case)        bytes and operations that no implementation can do without
  exact(case, s)    what run() returns, in 64 bits from the operator's definition
"""
import math

import numpy as np
import torch

own = False

DTYPES = dict(bf16=torch.bfloat16, f32=torch.float32, s8=torch.int8)
SIZES = dict(bf16=2, f32=4, s8=1)


def listed():
    return [
        # ---- appending to the cache
        # one user's new token: the smallest call, all latency
        dict(name="append_one_token", op="append", T=1, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, dt="bf16", cache="bf16", page=16,
             layout="tokens", pages=64, padded=False),
        # a decode batch into an 8-bit cache, some of its rows padding of a captured graph
        dict(name="append_decode_s8", op="append", T=256, heads=40, kv_heads=8, dim=128, rot=128, interleaved=False, dt="bf16", cache="s8", page=16,
             layout="tokens", pages=128, padded=True),
        # a prompt of several thousand tokens
        dict(name="append_prompt", op="append", T=8192, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, dt="bf16", cache="bf16", page=16,
             layout="tokens", pages=640, padded=False),
        # a ragged prompt of a small model: neighbouring pairs of part of the head are rotated, f32 activations, pages head by head, a page size that is no power of two
        dict(name="append_ragged_partial", op="append", T=1999, heads=12, kv_heads=12, dim=80, rot=32, interleaved=True, dt="f32", cache="bf16", page=24,
             layout="heads", pages=128, padded=True),
        # ---- attention of one new token
        # one user, a short conversation: all latency
        dict(name="attend_one_user", op="attend", B=1, heads=32, kv_heads=8, dim=128, cache="bf16", page=16, layout="tokens", longest=500, ragged=False,
             window=0, softcap=0.0, sinks=False, lse=False, out="bf16"),
        # a decode batch, every conversation of its own length, some rows padding
        dict(name="attend_batch_ragged", op="attend", B=32, heads=32, kv_heads=8, dim=128, cache="bf16", page=16, layout="tokens", longest=4096, ragged=True,
             window=0, softcap=0.0, sinks=False, lse=False, out="bf16"),
        # two users with very long documents: the split over the cache's length
        dict(name="attend_long", op="attend", B=2, heads=32, kv_heads=8, dim=128, cache="bf16", page=64, layout="heads", longest=131072, ragged=False,
             window=0, softcap=0.0, sinks=False, lse=True, out="bf16"),
        # a large batch over an 8-bit cache, five query heads to a key head, sinks beside the keys
        dict(name="attend_batch_s8", op="attend", B=64, heads=40, kv_heads=8, dim=128, cache="s8", page=32, layout="tokens", longest=8192, ragged=True,
             window=0, softcap=0.0, sinks=True, lse=False, out="bf16"),
        # a head for every query head, a head size and a page size that are no powers of two, a sliding window, capped scores, f32 out with the sums' logarithms
        dict(name="attend_window_odd", op="attend", B=16, heads=12, kv_heads=12, dim=80, cache="bf16", page=24, layout="heads", longest=3001, ragged=True,
             window=1000, softcap=30.0, sinks=False, lse=True, out="f32"),
        # ---- routing to experts
        # a decode batch, softmax scores, no groups
        dict(name="gate_decode", op="gate", T=32, E=64, k=6, score="softmax", bias=False, groups=1, top_groups=1, group_score="max", renorm=True, scale=1.0, dt="f32"),
        # a prompt batch over many experts: sigmoid scores, a bias for balance, the best groups first
        dict(name="gate_prompt_groups", op="gate", T=16384, E=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, group_score="top2", renorm=True,
             scale=2.5, dt="f32"),
        # a ragged batch, bf16 logits (many are equal), groups by their best expert, a number of experts that is no power of two
        dict(name="gate_ragged_bf16", op="gate", T=3001, E=60, k=4, score="softmax", bias=False, groups=6, top_groups=3, group_score="max", renorm=False,
             scale=16.0, dt="bf16"),
    ]


# ------------------------------------------------------------------------------------------------ ranges
def _log(rng, lo, hi):
    """Log-uniform over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["append", "attend", "attend", "gate"])
    if op == "gate":
        groups = rng.choice([1, 1, 2, 4, 6, 8])
        E = groups * rng.randint(2 if groups > 1 else 4, 256 // groups)
        top_groups = rng.randint(1, groups)
        return dict(op=op, T=_log(rng, 1, 16384), E=E, k=rng.randint(1, min(16, top_groups * (E // groups))), score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5, 16.0]),
                    dt=rng.choice(["f32", "f32", "bf16"]))
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    dim = rng.choice([64, 128, 128, 80, 96, 256])
    common = dict(heads=kv_heads * rng.randint(1, 64 // kv_heads if kv_heads > 2 else 16), kv_heads=kv_heads, dim=dim, page=rng.choice([1, 16, 16, 24, 32, 64, 128]),
                  layout=rng.choice(["tokens", "heads"]), cache=rng.choice(["bf16", "bf16", "s8"]) if dim % 16 == 0 else "bf16")
    if op == "append":
        T = _log(rng, 1, 8192)
        return dict(op=op, T=T, rot=rng.choice([dim, dim, dim // 2, 16]), interleaved=rng.random() < 0.3, dt=rng.choice(["bf16", "bf16", "f32"]),
                    pages=-(-int(T * rng.uniform(1.0, 1.5)) // common["page"]) + 2, padded=rng.random() < 0.5, **common)
    return dict(op=op, B=_log(rng, 1, 256), longest=_log(rng, 1, 131072), ragged=rng.random() < 0.7, window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]),
                softcap=rng.choice([0.0, 0.0, 30.0]), sinks=rng.random() < 0.3, lse=rng.random() < 0.3, out=rng.choice(["bf16", "bf16", "f32"]), **common)


def _held(case):
    """Bytes of the cache."""
    if case["op"] == "gate":
        return 0
    tokens = case["pages"] * case["page"] if case["op"] == "append" else case["B"] * case["longest"]
    return 2 * tokens * case["kv_heads"] * case["dim"] * SIZES[case["cache"]]


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def draw(rng):
    """Sizes over the whole range, no case dearer than the dearest listed one of its operator, no cache larger than theirs."""
    cases = listed()
    while True:
        case = _draw(rng)
        same = [c for c in cases if c["op"] == case["op"]]
        if _cost(case) <= max(_cost(c) for c in same) and _held(case) <= max(_held(c) for c in same):
            return case


# ------------------------------------------------------------------------------------------------ work
def _lengths(case):
    """Keys of each sequence, from the case alone: all of them `longest`, or spread evenly in the square root with a row of padding in ten."""
    B, n = case["B"], case["longest"]
    if not case["ragged"]:
        return [n] * B
    rng = np.random.default_rng(B * 1000003 + n)
    got = [max(1, int(n * rng.random() ** 0.5)) for _ in range(B)]
    got[0] = n
    return [-1 if i % 10 == 9 else g for i, g in enumerate(got)]


def work(case):
    if case["op"] == "gate":
        T, E, k = case["T"], case["E"], case["k"]
        return dict(bytes=T * E * SIZES[case["dt"]] + 4 * E * (2 if case["bias"] else 1) + T * k * 12, flops=T * E * 4)
    row = case["kv_heads"] * (case["dim"] * SIZES[case["cache"]] + (4 if case["cache"] == "s8" else 0))      # a token's keys or values
    if case["op"] == "append":
        T, x = case["T"], SIZES[case["dt"]]
        return dict(bytes=T * (2 * case["heads"] * case["dim"] * x + 2 * case["kv_heads"] * case["dim"] * x + 2 * row + 12 + 4 * case["rot"]),
                    flops=T * 3 * (case["heads"] + case["kv_heads"]) * case["rot"])
    lens = _lengths(case)
    keys = sum(max(0, min(n, case["window"]) if case["window"] else n) for n in lens)
    q = case["heads"] * case["dim"]
    return dict(bytes=keys * 2 * row + case["B"] * q * (2 + SIZES[case["out"]]) + 4 * sum(-(-max(0, n) // case["page"]) for n in lens) + 4 * case["B"],
                flops=4 * keys * q)


# ------------------------------------------------------------------------------------------------ inputs
def _cache(case, g, pages):
    """Keys, values and (8-bit) their scales as [page, token, head, dim] views of either storage order."""
    H, ps, D = case["kv_heads"], case["page"], case["dim"]
    shape = (pages, ps, H, D) if case["layout"] == "tokens" else (pages, H, ps, D)
    seen = (lambda t: t) if case["layout"] == "tokens" else (lambda t: t.transpose(1, 2))
    got = {}
    for name in ("key", "value"):
        if case["cache"] == "s8":
            got[name] = seen(torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda"))
            got[name + "_scale"] = seen(torch.rand(shape[:3], generator=g, device="cuda").mul_(0.02).add_(0.005))
        else:
            got[name] = seen(torch.randn(shape, generator=g, dtype=torch.bfloat16, device="cuda"))
    return got


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "gate":
        T, E, k = case["T"], case["E"], case["k"]
        st["logits"] = torch.randn(T, E, generator=g, device="cuda").to(DTYPES[case["dt"]])
        st["bias"] = torch.randn(E, generator=g, device="cuda").mul_(0.1) if case["bias"] else None
        st.update(ids=torch.empty(T, k, dtype=torch.int32, device="cuda"), weights=torch.empty(T, k, device="cuda"),
                  counts=torch.empty(E, dtype=torch.int32, device="cuda"), rows=torch.empty(T, k, dtype=torch.int32, device="cuda"))
        return st
    heads, H, D, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        T, dt, rot = case["T"], DTYPES[case["dt"]], case["rot"]
        st.update(_cache(case, g, case["pages"]))
        # q, k and v are the columns of one projection's output
        qkv = torch.randn(T, heads + 2 * H, D, generator=g, device="cuda").to(dt)
        st.update(q=qkv[:, :heads], k=qkv[:, heads:heads + H], v=qkv[:, heads + H:], q_out=torch.zeros(T, heads, D, dtype=dt, device="cuda"))
        st["slots"] = torch.randperm(case["pages"] * ps, generator=g, device="cuda")[:T].clone()
        if case["padded"]:
            st["slots"][9::10] = -1
        most = 32768
        st["positions"] = torch.randint(0, most, (T,), generator=g, device="cuda", dtype=torch.int32)
        angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        st.update(cos=angle.cos().float(), sin=angle.sin().float())
        if case["cache"] == "s8":      # what the codes stand for, for whoever reads the cache
            st.update({name + "_values": torch.empty(st[name].shape, dtype=torch.bfloat16, device="cuda") for name in ("key", "value")})
        return st
    B, lens = case["B"], _lengths(case)
    need = [-(-max(0, n) // ps) for n in lens]
    cols = -(-case["longest"] // ps)
    order = torch.randperm(sum(need) + 1, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table, at = np.full((B, cols), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    st.update(_cache(case, g, sum(need) + 1))
    st.update(q=torch.randn(B, heads, D, generator=g, device="cuda").to(torch.bfloat16), out=torch.zeros(B, heads, D, dtype=DTYPES[case["out"]], device="cuda"),
              table=torch.from_numpy(table).cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    st["sinks"] = torch.randn(heads, generator=g, device="cuda") if case["sinks"] else None
    st["lse"] = torch.zeros(B, heads, device="cuda") if case["lse"] else None
    return st


# ------------------------------------------------------------------------------------------------ the library's calls
def _descriptor(st):
    """What a program fills in once for its buffers and keeps from call to call."""
    from zendnn_b200 import capi
    case = st["case"]
    if case["op"] == "gate":
        return capi.lib.b200dnn_moe_gate, capi.make_moe_gate(
            st["logits"], case["k"], st["ids"], st["weights"], bias=st["bias"], score=case["score"], num_groups=case["groups"], topk_groups=case["top_groups"],
            group_score=case["group_score"], renorm=case["renorm"], scale=case["scale"], expert_counts=st["counts"], slot_to_row=st["rows"])
    cache = capi.make_kv_cache(st["key"], st["value"], st.get("key_scale"), st.get("value_scale"))
    if case["op"] == "append":
        return capi.lib.b200dnn_kv_append, capi.make_kv_append(
            cache, st["k"], st["v"], st["slots"], q=st["q"], q_out=st["q_out"], positions=st["positions"], cos=st["cos"], sin=st["sin"], interleaved=case["interleaved"])
    return capi.lib.b200dnn_paged_attention, capi.make_paged_attention(
        cache, st["q"], st["out"], st["table"], st["lens"], window=case["window"], softcap=case["softcap"], sinks=st["sinks"], lse=st["lse"])


def _call(st):
    import ctypes
    from zendnn_b200 import capi
    if "call" not in st:
        st["call"] = _descriptor(st)
    entry, desc = st["call"]
    capi.check(entry(ctypes.byref(desc), torch.cuda.current_stream().cuda_stream))


# ------------------------------------------------------------------------------------------------ the plain forms
def _rotate(x, cos, sin, rot, interleaved):
    """x [T, heads, dim] in 32 bits; cos, sin [T, 1, rot / 2]."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1 if interleaved else -2).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_append(st):
    case = st["case"]
    ps, rot = case["page"], case["rot"]
    cos, sin = (st[n][st["positions"].long()][:, None] for n in ("cos", "sin"))
    keep = st["slots"] >= 0
    q = _rotate(st["q"].float(), cos, sin, rot, case["interleaved"])
    st["q_out"].copy_(torch.where(keep[:, None, None], q.to(st["q_out"].dtype), st["q_out"]))
    rows = dict(key=_rotate(st["k"].float(), cos, sin, rot, case["interleaved"])[keep], value=st["v"].float()[keep])
    slots = st["slots"][keep]
    for name, x in rows.items():
        if case["cache"] == "s8":
            scale = x.abs().amax(-1) / 127.0
            st[name + "_scale"][slots // ps, slots % ps] = scale
            codes = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x)).round().clamp(-127, 127)
            st[name][slots // ps, slots % ps] = codes.to(torch.int8)
        else:
            st[name][slots // ps, slots % ps] = x.to(torch.bfloat16)


def _plain_attend(st):
    case = st["case"]
    B, H, D, ps = case["B"], case["kv_heads"], case["dim"], case["page"]
    at = torch.arange(case["longest"], device="cuda")
    page, off = st["table"][:, at // ps].clamp(min=0).long(), at % ps
    lens = st["lens"][:, None]
    seen = at < lens
    if case["window"]:
        seen = seen & (at >= lens - case["window"])

    def rows(name):
        x = st[name][page, off].float()
        if case["cache"] == "s8":
            x = x * st[name + "_scale"][page, off][..., None]
        return torch.where(seen[:, :, None, None], x, torch.zeros((), device="cuda")).permute(0, 2, 1, 3)      # [B, H, keys, D]

    q = st["q"].float().view(B, H, -1, D)
    s = torch.matmul(q, rows("key").transpose(2, 3)) / math.sqrt(D)
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    s = torch.where(seen[:, None, None], s, torch.full((), -math.inf, device="cuda"))
    top = s.amax(-1, keepdim=True)
    if case["sinks"]:
        sink = st["sinks"].view(1, H, -1, 1)
        top = torch.maximum(top, sink)
    live = lens[:, :, None, None] > 0
    top = torch.where(live, top, torch.zeros((), device="cuda"))
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    total = torch.where(live, total, torch.ones((), device="cuda"))
    o = (torch.matmul(p, rows("value")) / total).reshape(B, -1, D)
    write = st["lens"] >= 0
    st["out"].copy_(torch.where(write[:, None, None], o.to(st["out"].dtype), st["out"]))
    if case["lse"]:
        st["lse"].copy_(torch.where(write[:, None], (top + torch.log(total)).reshape(B, -1), st["lse"]))


def _plain_gate(st):
    """In 64 bits: two experts' scores may lie nearer to one another than 32 bits tell."""
    case = st["case"]
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    x = st["logits"].double()
    if case["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        s = torch.exp(x - x.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
    c = s if st["bias"] is None else s + st["bias"].double()
    if G > 1:
        best = c.view(T, G, -1).sort(-1, descending=True)[0]
        rank = best[..., 0] if case["group_score"] == "max" else best[..., :2].sum(-1)
        groups = rank.sort(dim=-1, descending=True, stable=True)[1][:, :case["top_groups"]]
        chosen = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, groups, True)
        c = torch.where(chosen[:, :, None], c.view(T, G, -1), torch.full((), -math.inf, dtype=torch.float64, device="cuda")).view(T, E)
    ids = c.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    flat = ids.reshape(-1)
    st["ids"].copy_(ids)
    st["weights"].copy_(w * case["scale"])
    st["counts"].copy_(torch.zeros(E, dtype=torch.int64, device="cuda").index_add_(0, flat, torch.ones_like(flat)))
    order = flat.sort(stable=True)[1]
    st["rows"].view(-1)[order] = torch.arange(T * k, dtype=torch.int32, device="cuda")


def run(state):
    op = state["case"]["op"]
    if own:
        _call(state)
    else:
        {"append": _plain_append, "attend": _plain_attend, "gate": _plain_gate}[op](state)
    if op == "gate":
        return {n: state[n] for n in ("ids", "weights", "counts", "rows")}
    if op == "attend":
        return {n: state[n] for n in ("out", "lse") if state[n] is not None}
    if state["case"]["cache"] == "s8":
        for name in ("key", "value"):
            torch.mul(state[name], state[name + "_scale"][..., None], out=state[name + "_values"])
        return {"q": state["q_out"], "key": state["key_values"], "value": state["value_values"], "key_scale": state["key_scale"], "value_scale": state["value_scale"]}
    return {"q": state["q_out"], "key": state["key"], "value": state["value"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gate":
        return _exact_gate(case, st)
    ps, D, H, g = case["page"], case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    if case["op"] == "append":
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"].long()][:, None]
        half = case["rot"] // 2

        def turned(x):
            x = x.double().clone()
            first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
            second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
            x[..., first], x[..., second] = z.real, z.imag
            return x

        on = (st["slots"] >= 0).nonzero()[:, 0]
        q = st["q_out"].double()
        q[on] = turned(st["q"])[on]
        got = {"q": q}
        pages, offs = st["slots"][on] // ps, st["slots"][on] % ps
        for name, x in (("key", turned(st["k"])), ("value", st["v"].double())):
            held = st[name].double()
            if case["cache"] == "s8":
                held = held * st[name + "_scale"].double()[..., None]
                step = x.abs().amax(-1, keepdim=True) / 127.0
                x = torch.round(x / step.clamp(min=1e-300)) * step
                scales = st[name + "_scale"].double()
                scales[pages, offs] = step[on, :, 0]
                got[name + "_scale"] = scales
            held[pages, offs] = x[on]
            got[name] = held
        return got
    out, lse = st["out"].double(), st["lse"].double() if case["lse"] else None
    for i, n in enumerate(st["lens"].tolist()):
        if n < 0:
            continue
        at = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        page, off = st["table"][i].long()[at // ps], at % ps
        for h in range(H):
            kv = []
            for name in ("key", "value"):
                x = st[name][page, off, h].double()
                kv.append(x * st[name + "_scale"][page, off, h].double()[:, None] if case["cache"] == "s8" else x)
            s = st["q"][i, h * g:(h + 1) * g].double() @ kv[0].T * D ** -0.5
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            z = torch.cat((s, st["sinks"][h * g:(h + 1) * g].double()[:, None]), 1) if case["sinks"] else s
            total = torch.logsumexp(z, 1, keepdim=True)
            out[i, h * g:(h + 1) * g] = torch.exp(s - total) @ kv[1]
            if lse is not None:
                lse[i, h * g:(h + 1) * g] = total[:, 0]
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_gate(case, st):
    """Token by token where the choice is made, on the host."""
    x = st["logits"].double().cpu().numpy()
    s = 1.0 / (1.0 + np.exp(-x)) if case["score"] == "sigmoid" else np.exp(x - x.max(1, keepdims=True)) / np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)
    c = s + st["bias"].double().cpu().numpy() if case["bias"] else s.copy()
    per = case["E"] // case["groups"]
    w = np.empty((case["T"], case["k"]))
    for t in range(case["T"]):
        row = c[t]
        if case["groups"] > 1:
            parts = np.sort(row.reshape(-1, per), 1)[:, ::-1]
            value = parts[:, 0] if case["group_score"] == "max" else parts[:, :2].sum(1)
            order = np.argsort(-value, kind="stable")
            row = row.copy()
            for lost in order[case["top_groups"]:]:
                row[lost * per:(lost + 1) * per] = -np.inf
        ids = np.argsort(-row, kind="stable")[:case["k"]]
        w[t] = s[t, ids] / s[t, ids].sum() if case["renorm"] else s[t, ids]
    return {"ids": None, "weights": w * case["scale"], "counts": None, "rows": None}
