"""Operators of a text tower's transformer block, measured one call at a time.

Kinds of cases:
  self    self attention with a learned relative position bias by buckets (forward, forward + backward, or one new token over a cache)
  cross   cross attention to an encoder's states of another length: per-sample lengths, a key mask, shared key / value heads
  norm    root-mean-square norm with the residual's addition: training (forward + backward), or an 8-bit output that feeds a projection
  linear  a projection in 8-bit integers: activations quantised by row, weights by output channel

`run` computes the plain form in elementary torch operations, or, with `own`, calls celebbasis_amd. `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
_T = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one prompt of the text tower's own length through one layer, in the training step's own type: latency
        dict(name="self_prompt", op="self", mode="fwd", dtype="f32", B=1, Nq=77, Nk=77, H=12, Hkv=12, d=64, causal=False, ragged=0.0, buckets=32, dist=128),
        # a training batch of padded captions
        dict(name="self_train", op="self", mode="train", dtype="bf16", B=8, Nq=512, Nk=512, H=12, Hkv=12, d=64, causal=False, ragged=0.5, buckets=32, dist=128),
        # a decoder's training step on long texts
        dict(name="self_train_long", op="self", mode="train", dtype="bf16", B=2, Nq=4096, Nk=4096, H=12, Hkv=12, d=64, causal=True, ragged=0.0, buckets=32, dist=128),
        # one new token for each of 32 texts over their caches
        dict(name="self_token", op="self", mode="token", dtype="bf16", B=32, Nq=1, Nk=8192, H=12, Hkv=12, d=64, causal=True, ragged=0.5, buckets=32, dist=128),
        # the image network's 64x64 level on padded prompts, guided batch, training
        dict(name="cross_image_train", op="cross", mode="train", dtype="bf16", B=8, Nq=4096, Nk=77, H=8, Hkv=8, d=40, causal=False, ragged=0.8, mask=False),
        # a prompt batch reading long encoder states with holes, shared key / value heads
        dict(name="cross_states", op="cross", mode="fwd", dtype="bf16", B=4, Nq=1024, Nk=2000, H=16, Hkv=4, d=128, causal=False, ragged=0.3, mask=True),
        # the 32x32 level in fp32 with its gradients, odd lengths
        dict(name="cross_f32_train", op="cross", mode="train", dtype="f32", B=2, Nq=1023, Nk=333, H=8, Hkv=8, d=80, causal=False, ragged=0.4, mask=True),
        # one new token for each of 64 texts over the encoder's states
        dict(name="cross_token", op="cross", mode="token", dtype="bf16", B=64, Nq=1, Nk=1500, H=16, Hkv=4, d=64, causal=False, ragged=0.5, mask=False),
        # four new tokens: residual, norm, 8 bits, the fused q/k/v projection of the text tower's width: latency
        dict(name="norm_token", op="norm", mode="i8", dtype="bf16", rows=4, C=768, N=2304),
        # a training step's norm over a batch of long texts
        dict(name="norm_train", op="norm", mode="train", dtype="bf16", rows=16384, C=2048),
        # one new token through a wide projection: bound by the weights
        dict(name="linear_token", op="linear", mode="i8", dtype="bf16", rows=1, N=8192, K=4096, bias=True),
        # a large prompt batch through a wide projection
        dict(name="linear_prompts", op="linear", mode="i8", dtype="bf16", rows=8192, N=8192, K=4096, bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["self", "self", "cross", "cross", "norm", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("self", "cross"):
        mode = rng.choice(["fwd", "train", "token"])
        d = rng.choice([40, 64, 64, 80, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 1, 2, 4])
        ragged = rng.choice([0.0, 0.3, 0.7])
        if mode == "token":
            Nq, Nk = 1, _log(rng, 64, 16384)
            B = _log(rng, 1, max(1, min(64, 400000 // Nk)))
        elif op == "self":
            Nq = Nk = _log(rng, 33, 3000)
            B = _log(rng, 1, 8)
        else:
            Nq, Nk, B = _log(rng, 33, 4096), _log(rng, 17, 2500), _log(rng, 1, 8)
        while B > 1 and B * H * Nq * Nk > 2 * 12 * 4096 * 2048:
            B -= 1
        c = dict(op=op, mode=mode, dtype=dtype, B=B, Nq=Nq, Nk=Nk, H=H, Hkv=Hkv, d=d, causal=op == "self" and (mode == "token" or rng.random() < 0.5), ragged=ragged)
        if op == "self":
            c.update(buckets=rng.choice([32, 32, 16, 64]), dist=rng.choice([128, 128, 64, 256]))
        else:
            c.update(mask=rng.random() < 0.5)
        return c
    if op == "norm":
        if rng.random() < 0.5:
            return dict(op="norm", mode="train", dtype=dtype, rows=_log(rng, 5, 16384), C=8 * _log(rng, 8, 512))
        return dict(op="norm", mode="i8", dtype="bf16", rows=_log(rng, 1, 4096), C=8 * _log(rng, 16, 512), N=_log(rng, 64, 5000))
    return dict(op="linear", mode="i8", dtype="bf16", rows=_log(rng, 1, 6000), N=_log(rng, 64, 8000), K=_log(rng, 100, 4096), bias=rng.random() < 0.5)


def _lengths(n, B, ragged):
    """B lengths of at most n, spread evenly over the last `ragged` share of it"""
    return [max(1, n - int(n * ragged * b / max(1, B - 1))) for b in range(B)]


def _pairs(c):
    """visible (query, key) pairs of one head, over the batch"""
    lens = _lengths(c["Nk"], c["B"], c["ragged"])
    if c["mode"] == "token":
        return sum(lens)
    pairs = 0
    for n in lens:
        nq = n if c["op"] == "self" else c["Nq"]
        pairs += n * (n + 1) // 2 if c["causal"] else nq * n
    return pairs * (0.75 if c.get("mask") else 1.0)


def work(c):
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] in ("self", "cross"):
        lens = _lengths(c["Nk"], c["B"], c["ragged"])
        nkv = sum(lens)
        nq = c["B"] * c["Nq"] if c["op"] == "cross" or c["mode"] == "token" else nkv
        q, kv = nq * c["H"] * c["d"] * e, nkv * c["Hkv"] * c["d"] * e
        per = 4 * c["d"] * c["H"] * _pairs(c)
        if c["mode"] == "train":                      # q, k, v, do in; o, dq, dk, dv out
            return dict(bytes=4 * q + 4 * kv, flops=3.5 * per)
        return dict(bytes=2 * q + 2 * kv, flops=per)
    if c["op"] == "norm":
        x = c["rows"] * c["C"] * e
        if c["mode"] == "train":                      # x, r, dy, dres in; h, y, dh out
            return dict(bytes=7 * x + 8 * c["C"], flops=20 * c["rows"] * c["C"])
        return dict(bytes=3 * x + c["C"] * c["N"] + 2 * c["rows"] * c["N"], flops=2 * c["rows"] * c["C"] * c["N"])
    return dict(bytes=c["rows"] * c["K"] * e + c["N"] * c["K"] + 2 * c["rows"] * c["N"], flops=2 * c["rows"] * c["N"] * c["K"])


# ------------------------------------------------------------------------------------------------ inputs
def _thresholds(buckets, dist, two_sided):
    """first distance of each bucket beyond the exact ones: the least n with n >= E (D/E)^(k/m), in whole numbers"""
    nb = buckets // 2 if two_sided else buckets
    E = nb // 2
    m = nb - E
    got = []
    for k in range(1, m):
        n = E
        lo, hi = E, dist
        while lo < hi:
            n = (lo + hi) // 2
            if n ** m * E ** k >= E ** m * dist ** k:
                hi = n
            else:
                lo = n + 1
        got.append(lo)
    return nb, E, got


_handles = {}


def _context():
    from celebbasis_amd import lib
    if "ctx" not in _handles:
        _handles["ctx"] = lib.Context()
    return lib, _handles["ctx"]


def _inputs(c, seed):
    """the case's tensors from the seed alone, on the GPU"""
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)
    t = _T[c["dtype"]]

    def rnd(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {"case": dict(c)}
    if c["op"] in ("self", "cross"):
        B, Nq, Nk, H, Hkv, d = (c[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "d"))
        lens = _lengths(Nk, B, c["ragged"])
        at = torch.randperm(B, generator=torch.Generator().manual_seed(int(seed))).tolist()
        s["kv_len"] = torch.tensor([lens[i] for i in at], dtype=torch.int32, device=DEV)
        s["scale"] = d ** -0.5
        if c["op"] == "self" and c["mode"] != "token":          # the fused projection's output
            s["qkv"] = rnd(B, Nk, (H + 2 * Hkv) * d, scale=1.2)
        else:
            s["q"] = rnd(B, Nq, H * d, scale=1.2)
            s["kv"] = rnd(B, Nk, 2 * Hkv * d, scale=1.2)
        if c["op"] == "self":
            s["table"] = rnd(c["buckets"], H, scale=0.7, dtype=torch.float32)
            s["two_sided"] = not c["causal"]
            nb, E, th = _thresholds(c["buckets"], c["dist"], s["two_sided"])
            s["nb"], s["E"] = nb, E
            s["th"] = torch.tensor(th, dtype=torch.int64, device=DEV)
        if c["mode"] == "token":
            s["q_pos"] = s["kv_len"] - 1
        if c.get("mask"):
            s["mask"] = torch.rand(B, Nk, generator=g, device=DEV) < 0.75
            s["mask"][:, 0] = True
        if c["mode"] == "train":
            s["do"] = rnd(B, Nq, H * d)
            if c["op"] == "self":                               # rows behind a text's end carry no gradient
                s["do"] *= (torch.arange(Nq, device=DEV)[None, :] < s["kv_len"][:, None]).to(t)[..., None]
    elif c["op"] == "norm":
        s["x"], s["r"] = rnd(c["rows"], c["C"], scale=0.5), rnd(c["rows"], c["C"], scale=2.0)
        s["g"] = 1.0 + rnd(c["C"], scale=0.2, dtype=torch.float32)
        if c["mode"] == "train":
            s["dy"], s["dres"] = rnd(c["rows"], c["C"]), rnd(c["rows"], c["C"])
        else:
            s["w"] = rnd(c["N"], c["C"], scale=c["C"] ** -0.5, dtype=torch.float32)
    else:
        s["x"] = rnd(c["rows"], c["K"])
        s["w"] = rnd(c["N"], c["K"], scale=c["K"] ** -0.5, dtype=torch.float32)
        s["bias"] = rnd(c["N"], dtype=torch.float32) if c["bias"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = s["case"]
    if "w" in s:                                                # weights are brought to 8 bits once, when they are loaded
        w = s.pop("w")
        amax = w.abs().amax(1)
        s["wq"] = torch.round(w * (127.0 / amax)[:, None]).to(torch.int8)
        s["ws"] = amax / 127.0
        pad = -w.shape[1] % 16                                  # rows of whole 16-byte pieces
        if pad:
            s["wq"] = torch.cat([s["wq"], torch.zeros(w.shape[0], pad, dtype=torch.int8, device=DEV)], 1)
    if own and c["op"] == "self":
        lib, ctx = _context()
        key = (c["buckets"], c["dist"], s["two_sided"])
        if key not in _handles:
            _handles[key] = lib.RelPos(ctx, num_buckets=c["buckets"], max_distance=c["dist"], bidirectional=s["two_sided"])
        s["relpos"] = _handles[key]
    return s


def _heads(s):
    """q, k, v as [B, N, heads, d] views of what the projections wrote"""
    c = s["case"]
    H, Hkv, d = c["H"], c["Hkv"], c["d"]
    if "qkv" in s:
        x = s["qkv"].view(c["B"], c["Nk"], H + 2 * Hkv, d)
        return x[:, :, :H], x[:, :, H:H + Hkv], x[:, :, H + Hkv:]
    kv = s["kv"].view(c["B"], c["Nk"], 2 * Hkv, d)
    return s["q"].view(c["B"], c["Nq"], H, d), kv[:, :, :Hkv], kv[:, :, Hkv:]


# ------------------------------------------------------------------------------------------------ plain forms
def _bucket(s, rel):
    n = rel.abs() if s["two_sided"] else (-rel).clamp(min=0)
    far = s["E"] + (n[..., None] >= s["th"]).sum(-1)
    b = torch.where(n < s["E"], n, far)
    return b + s["nb"] * (rel > 0) if s["two_sided"] else b


def _visible(s):
    c = s["case"]
    j = torch.arange(c["Nk"], device=DEV)
    i = torch.arange(c["Nq"], device=DEV)
    ok = (j[None] < s["kv_len"][:, None])
    if "mask" in s:
        ok = ok & s["mask"]
    ok = ok[:, None, None, :]
    if c["op"] == "self" and c["mode"] != "token":
        ok = ok & (i[None] < s["kv_len"][:, None])[:, None, :, None]
    if c["causal"] and c["mode"] != "token":
        ok = ok & (j[None, :] <= i[:, None])
    return ok


def _plain_attention(s):
    c = s["case"]
    B, Nq, Nk, H, Hkv, d = (c[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "d"))
    q, k, v = (x.float().transpose(1, 2) for x in _heads(s))
    k = k[:, :, None].expand(B, Hkv, H // Hkv, Nk, d).reshape(B, H, Nk, d)
    v = v[:, :, None].expand(B, Hkv, H // Hkv, Nk, d).reshape(B, H, Nk, d)
    sc = torch.matmul(q * s["scale"], k.transpose(-1, -2))
    if c["op"] == "self":
        j = torch.arange(Nk, device=DEV)
        if c["mode"] == "token":
            sc = sc + s["table"][_bucket(s, j[None] - s["q_pos"][:, None].long())].permute(0, 2, 1)[:, :, None, :]
        else:
            bk = _bucket(s, j[None] - j[:, None])
            sc = sc + s["table"][bk].permute(2, 0, 1)
    ok = _visible(s)
    sc = sc.masked_fill(~ok, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(sc - top)
    tot = p.sum(-1, keepdim=True)
    p = torch.where(tot > 0, p / tot, torch.zeros_like(p))
    o = torch.matmul(p, v)
    t = _T[c["dtype"]]
    out = o.transpose(1, 2).reshape(B, Nq, H * d).to(t)
    if c["mode"] != "train":
        return out
    do = s["do"].float().view(B, Nq, H, d).transpose(1, 2)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(-1, -2), q).view(B, Hkv, H // Hkv, Nk, d).sum(2) * s["scale"]
    dv = torch.matmul(p.transpose(-1, -2), do).view(B, Hkv, H // Hkv, Nk, d).sum(2)
    dq, dk, dv = (x.transpose(1, 2) for x in (dq, dk, dv))
    if c["op"] == "cross":
        return {"out": out, "dq": dq.reshape(B, Nq, H * d).to(t), "dkv": torch.cat([dk, dv], 2).reshape(B, Nk, 2 * Hkv * d).to(t)}
    # the table's gradient: sums along the diagonals j - i (a row of the padded copy starts one place further left than the one above it),
    # then over the distances of a bucket
    W = Nk + Nq - 1
    x = torch.nn.functional.pad(ds.sum(0).flip(1), (0, Nq)).reshape(H, -1)[:, :Nq * W].reshape(H, Nq, W)
    diag = x.sum(1, dtype=torch.float64)
    rel = torch.arange(W, device=DEV) - (Nq - 1)
    hot = (_bucket(s, rel)[:, None] == torch.arange(c["buckets"], device=DEV)).double()
    return {"out": out, "dqkv": torch.cat([dq, dk, dv], 2).reshape(B, Nk, (H + 2 * Hkv) * d).to(t), "dtable": torch.matmul(hot.t(), diag.t()).float()}


def _plain_norm(s):
    c = s["case"]
    t = _T[c["dtype"]]
    held = (s["x"].float() + s["r"].float()).to(t)
    h = held.float()
    rstd = torch.rsqrt(h.double().square().mean(-1, keepdim=True) + 1e-6).float()
    y = h * rstd * s["g"]
    if c["mode"] == "i8":
        return {"h": held, "y": _plain_product(y, s["wq"], s["ws"], None)}
    w = s["dy"].float() * s["g"]
    dh = rstd * (w - h * rstd.square() * (w * h).mean(-1, keepdim=True)) + s["dres"].float()
    dg = (s["dy"].float() * h * rstd).sum(0, dtype=torch.float64).float()
    return {"h": held, "y": y.to(t), "dh": dh.to(t), "dg": dg}


def _plain_product(x, wq, ws, bias):
    amax = x.abs().amax(1, keepdim=True)
    q = torch.round(x * (127.0 / amax))
    y = torch.matmul(q, wq[:, :x.shape[1]].float().t()) * (amax / 127.0) * ws
    return (y if bias is None else y + bias).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ one pass
def _own_attention(s):
    lib, ctx = _context()
    c = s["case"]
    q, k, v = _heads(s)
    more = dict(scale=s["scale"], causal=c["causal"], kv_len=s["kv_len"], kv_mask=s.get("mask"), q_pos=s.get("q_pos"),
                relpos=s.get("relpos"), table=s.get("table"))
    if c["op"] == "self" and c["mode"] != "token":
        more["q_len"] = s["kv_len"]
    flat = lambda x: x.reshape(c["B"], x.shape[1], -1)  # noqa: E731
    if c["mode"] != "train":
        return flat(lib.seq_attention(ctx, q, k, v, **more))
    out, tape = lib.seq_attention(ctx, q, k, v, need_grad=True, **more)
    do = s["do"].view(c["B"], c["Nq"], c["H"], c["d"])
    H, Hkv = c["H"], c["Hkv"]
    if c["op"] == "cross":
        dkv = torch.empty_like(s["kv"])
        x = dkv.view(c["B"], c["Nk"], 2 * Hkv, c["d"])
        g = lib.seq_attention_backward(ctx, tape, do, dk=x[:, :, :Hkv], dv=x[:, :, Hkv:])
        return {"out": flat(out), "dq": flat(g.dq), "dkv": dkv}
    dqkv = torch.empty_like(s["qkv"])
    x = dqkv.view(c["B"], c["Nk"], H + 2 * Hkv, c["d"])
    g = lib.seq_attention_backward(ctx, tape, do, dq=x[:, :, :H], dk=x[:, :, H:H + Hkv], dv=x[:, :, H + Hkv:])
    return {"out": flat(out), "dqkv": dqkv, "dtable": g.dtable}


def _own_norm(s):
    lib, ctx = _context()
    if s["case"]["mode"] == "i8":
        n = lib.rms_norm(ctx, s["x"], s["g"], residual=s["r"], eps=1e-6, out="i8")
        return {"h": n.h, "y": lib.linear_i8(ctx, n.y, n.scale, s["wq"], s["ws"], dtype="bf16")}
    n = lib.rms_norm(ctx, s["x"], s["g"], residual=s["r"], eps=1e-6, need_grad=True)
    dh, dg = lib.rms_norm_backward(ctx, s["dy"], n.h, s["g"], n.rstd, dres=s["dres"])
    return {"h": n.h, "y": n.y, "dh": dh, "dg": dg}


def run(s):
    op = s["case"]["op"]
    if op in ("self", "cross"):
        return _own_attention(s) if own else _plain_attention(s)
    if op == "norm":
        return _own_norm(s) if own else _plain_norm(s)
    if own:
        lib, ctx = _context()
        q, sc = lib.quantize_rows(ctx, s["x"])
        return lib.linear_i8(ctx, q, sc, s["wq"], s["ws"], bias=s["bias"], dtype="bf16")
    return _plain_product(s["x"].float(), s["wq"], s["ws"], s["bias"])


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _bucket64(c, two_sided, rel):
    """the definition by the logarithm, a hair above its borders"""
    nb = c["buckets"] // 2 if two_sided else c["buckets"]
    E = nb // 2
    n = (rel.abs() if two_sided else torch.clamp(-rel, min=0)).double()
    far = E + torch.floor(torch.log(n.clamp(min=1) / E) / math.log(c["dist"] / E) * (nb - E) + 1e-9).clamp(max=nb - E - 1)
    b = torch.where(n < E, n, far).long()
    return b + nb * (rel > 0).long() if two_sided else b


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] in ("self", "cross"):
        return _exact_attention(s)
    if c["op"] == "norm":
        t = _T[c["dtype"]]
        held = (s["x"].double() + s["r"].double()).to(t)
        h, g = held.double().requires_grad_(), s["g"].double().requires_grad_()
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / c["C"] + 1e-6) * g
        if c["mode"] == "i8":
            return {"h": held.double(), "y": _exact_product(y.detach(), s["wq"], s["ws"], None)}
        dh, dg = torch.autograd.grad((y * s["dy"].double()).sum(), (h, g))
        return {"h": held.double(), "y": y.detach(), "dh": dh + s["dres"].double(), "dg": dg}
    return _exact_product(s["x"].double(), s["wq"], s["ws"], s["bias"])


def _exact_product(x, wq, ws, bias):
    step = x.abs().max(dim=1).values / 127
    q = torch.round(x / step[:, None])
    y = (q @ wq.double()[:, :x.shape[1]].T.contiguous()) * step[:, None] * ws.double()[None, :]
    return y if bias is None else y + bias.double()


def _exact_attention(s):
    """text by text and head by head, on the visible keys alone; gradients by differentiation"""
    c = s["case"]
    B, H, Hkv, d = c["B"], c["H"], c["Hkv"], c["d"]
    grad = c["mode"] == "train"
    q, k, v = (x.double() for x in _heads(s))
    out = torch.zeros(B, c["Nq"], H, d, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    table = s["table"].double() if c["op"] == "self" else None
    dtable = torch.zeros_like(table) if table is not None else None
    for b in range(B):
        n = int(s["kv_len"][b])
        keys = torch.arange(n, device=DEV)
        if "mask" in s:
            keys = keys[s["mask"][b, :n]]
        nq = n if c["op"] == "self" and c["mode"] != "token" else c["Nq"]
        at = torch.arange(nq, device=DEV) + (n - 1 if c["mode"] == "token" else 0)
        rel = keys[None, :] - at[:, None]
        for g in range(Hkv):
            hs = slice(g * (H // Hkv), (g + 1) * (H // Hkv))
            qq, kk, vv = q[b, :nq, hs].transpose(0, 1).contiguous(), k[b, keys, g].contiguous(), v[b, keys, g].contiguous()
            tt = table[:, hs].contiguous() if table is not None else None
            ins = [x.requires_grad_() for x in (qq, kk, vv) + ((tt,) if tt is not None else ())] if grad else []
            z = torch.matmul(qq, kk.t().contiguous()) * s["scale"]
            if tt is not None:
                hot = torch.nn.functional.one_hot(_bucket64(c, s["two_sided"], rel), c["buckets"]).double()
                z = z + torch.matmul(hot, tt).permute(2, 0, 1)
            if c["causal"]:
                z = z + torch.where(rel > 0, -math.inf, 0.0)
            o = torch.matmul(torch.softmax(z, -1), vv)
            out[b, :nq, hs] = o.detach().transpose(0, 1)
            if grad:
                do = s["do"][b, :nq].double().view(nq, H, d)[:, hs].transpose(0, 1)
                got = torch.autograd.grad((o * do).sum(), ins)
                dq[b, :nq, hs] = got[0].transpose(0, 1)
                dk[b, keys, g], dv[b, keys, g] = got[1], got[2]
                if tt is not None:
                    dtable[:, hs] += got[3]
    out = out.view(B, c["Nq"], H * d)
    if not grad:
        return out
    if c["op"] == "cross":
        return {"out": out, "dq": dq.reshape(B, c["Nq"], H * d), "dkv": torch.cat([dk, dv], 2).reshape(B, c["Nk"], 2 * Hkv * d)}
    return {"out": out, "dqkv": torch.cat([dq, dk, dv], 2).reshape(B, c["Nk"], (H + 2 * Hkv) * d), "dtable": dtable}
