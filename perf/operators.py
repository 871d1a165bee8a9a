"""Measured cases of the training operators: relative attention, layer norm and AdamW.

``listed()`` names the cases, ``draw()`` makes more of the same ranges, ``run()`` is one
pass: the plain form in elementary torch operations, or, where ``own`` is set, the
framework's operators (:mod:`hive_neuralnet_b200.train_ops`).  ``exact()`` computes the
same outputs in 64 bits, written apart from the plain form.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
CLIP, CLIP_Z = 8, 2  # the hybrid network's offset clips (coordinates, heights)
BLOCK = 256          # AdamW: every tensor's state starts at a multiple of this; one 8-bit scale per block


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one position's CLS + 28 piece tokens through one block of the default network: latency
        _att("attention: one position", 1, 29, 29, 8, 8, "f32", grad=False),
        # a training batch of the default network in full precision
        _att("attention: 1024 positions f32", 1024, 29, 29, 8, 8, "f32"),
        # the search's leaf batch used as a training batch, activations in half precision
        _att("attention: 8192 positions f16", 8192, 29, 29, 8, 8, "f16"),
        # the large preset (hidden 128): tokens masked anywhere, not only at the end
        _att("attention: large preset bf16", 2048, 29, 29, 8, 16, "bf16", holes=True),
        # long sequences with wide heads, a ragged last tile
        _att("attention: 1023 tokens bf16", 2, 1023, 1023, 8, 64, "bf16"),
        # one position's tokens: latency
        _norm("norm: one position", 29, 64, "f32", residual=False),
        # the second norm of a block over a leaf batch's tokens, with the residual added
        _norm("norm: 8192 positions f16", 8192 * 29, 64, "f16", residual=True),
        # the successor encoder's norm over every successor of 32,768 positions, forward only
        _norm("norm: successor rows f32", 1_170_000, 64, "f32", residual=False, grad=False),
        # wide rows of odd length
        _norm("norm: wide odd rows bf16", 4095, 2047, "bf16", residual=False),
        # the default hybrid network's parameter tensors: many small ones
        dict(name="adamw: hybrid network", op="adamw", net="hybrid", tensors=89, total=0, dtype="f32", bits=32),
        # few large tensors, 32-bit states
        dict(name="adamw: 64M f32", op="adamw", net="", tensors=24, total=64_000_000, dtype="f32", bits=32),
        # half-precision parameters, 8-bit states
        dict(name="adamw: 16M bf16 8 bits", op="adamw", net="", tensors=24, total=16_000_000, dtype="bf16", bits=8),
    ]


def _att(name, batch, tokens, queries, heads, head_dim, dtype, grad=True, holes=False):
    return dict(name=name, op="attention", batch=batch, tokens=tokens, queries=queries, heads=heads,
                head_dim=head_dim, dtype=dtype, grad=grad, holes=holes)


def _norm(name, rows, width, dtype, residual, grad=True):
    return dict(name=name, op="norm", rows=rows, width=width, dtype=dtype, residual=residual, grad=grad)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "adamw"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "attention":
        n = rng.choice([_log(rng, 1, 64), _log(rng, 20, 33), _log(rng, 1, 1024)])
        h, d = rng.randint(1, 12), rng.choice([4, 8, 8, 12, 16, 16, 24, 32, 48, 64])
        pairs = n * n * h
        most = max(1, min(int(4e8 / (pairs * d)), int(5e7 / pairs), int(5e6 / (n * n)), 8192))
        c = _att("", _log(rng, 1, most), n, n if rng.random() < 0.8 else 1, h, d, dtype, grad=rng.random() < 0.8,
                 holes=rng.random() < 0.5)
    elif op == "norm":
        w = _log(rng, 1, 8192)
        c = _norm("", _log(rng, 1, min(1_000_000, int(3e7 / w))), w, dtype, residual=rng.random() < 0.5,
                  grad=rng.random() < 0.8)
    else:
        c = dict(op="adamw", net="", tensors=rng.randint(1, 60), total=_log(rng, 1000, 10_000_000), dtype=dtype,
                 bits=rng.choice([8, 32]))
    c.pop("name", None)
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _counts(case):
    """Valid tokens of each position: spread evenly from the opening (the CLS token
    and one piece) to a full board, the same total for every seed."""
    b, n = case["batch"], case["tokens"]
    lo = min(n, 2) if n <= 64 else n // 2
    return lo + ((np.arange(b) + 0.5) / b * (n - lo + 1)).astype(np.int64)


def hybrid_shapes(h=64, mlp=96, layers=4, heads=8, e=64, a=64, v=128):
    """Parameter shapes of the hybrid network (default preset)."""
    s = [(64, 122), (64,), (64,), (64,), (e, 64), (e,), (1, e), (1,), (a, 2 * e), (a,), (1, a), (1,)]
    s += [(h, 26), (h,), (1, 1, h)]
    for _ in range(layers):
        s += [(h,), (h,), (3 * h, h), (3 * h,), (h, h), (h,), (17, heads), (17, heads), (5, heads), (h,), (h,),
              (mlp, h), (mlp,), (h, mlp), (h,)]
    return s + [(h,), (h,), (e, h), (e,), (e, 31), (e,), (a, 4 * e), (a,), (1, a), (1,), (v, e + h + 6), (v,),
                (1, v), (1,)]


def tensor_shapes(case):
    if case["net"] == "hybrid":
        return hybrid_shapes()
    t, total = case["tensors"], case["total"]
    # tensor i takes a share that falls off geometrically, at least one value
    w = 0.8 ** np.arange(t)
    return [(max(1, int(x)),) for x in w / w.sum() * total]


def _offsets(sizes):
    return np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])]).astype(np.int64)


def _parts(flat, s):
    """The tensors' own parts of a flat state."""
    return [flat[o:o + n] for o, n in zip(s["offsets"], s["sizes"])]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "attention":
        b, n, nq, h, d = (case[k] for k in ("batch", "tokens", "queries", "heads", "head_dim"))
        s["qkv"] = randn(b, n, 3, h, d).to(dt)  # as the fused projection writes it
        counts = torch.from_numpy(_counts(case)).to(dev)[torch.randperm(b, generator=g, device=dev)]
        mask = torch.arange(n, device=dev)[None, :] < counts[:, None]
        if case["holes"]:  # valid tokens anywhere, the CLS token first
            order = torch.rand(b, n, generator=g, device=dev)
            order[:, 0] = -1
            mask = mask.gather(1, order.argsort(1).argsort(1))
        s["mask"] = mask
        spread = 6 if n <= 64 else 11
        for name in ("tq", "tr"):
            s[name] = torch.randint(-spread, spread + 1, (b, n), generator=g, device=dev, dtype=torch.int32)
        s["tz"] = ((torch.rand(b, n, generator=g, device=dev) < 0.15)
                   * torch.randint(1, 5, (b, n), generator=g, device=dev)).to(torch.int32)
        for name in ("tq", "tr", "tz"):
            s[name][:, 0] = 0
        s["bq"], s["br"], s["bz"] = (0.5 * randn(2 * c + 1, h) for c in (CLIP, CLIP, CLIP_Z))
        if case["grad"]:
            s["dout"] = randn(b, nq, h, d).to(dt)
    elif case["op"] == "norm":
        r, w = case["rows"], case["width"]
        s["x"] = (randn(r, w) * 1.5 + 0.3).to(dt)
        s["weight"], s["bias"] = 1 + 0.2 * randn(w), 0.1 * randn(w)
        if case["residual"]:
            s["residual"] = randn(r, w).to(dt)
        if case["grad"]:
            s["dy"] = randn(r, w).to(dt)
            if case["residual"]:  # the gradient that comes along the residual path
                s["dsum"] = randn(r, w).to(dt)
    else:
        shapes = tensor_shapes(case)
        sizes = [int(np.prod(x)) for x in shapes]
        s["params"] = [(0.1 * randn(*x)).to(dt) for x in shapes]
        s["grads"] = [(0.01 * randn(*x)).to(dt) for x in shapes]
        off = _offsets(sizes)
        s["sizes"], s["offsets"], s["padded"] = sizes, [int(o) for o in off[:-1]], int(off[-1])
        for name in ("m", "v"):
            value = torch.zeros(s["padded"], device=dev)
            for part in _parts(value, s):
                part.copy_(0.003 * randn(part.numel()))
                if name == "v":  # a running mean of squares
                    part.square_().add_(1e-9)
            if case["bits"] == 32:
                s[name] = value
                continue
            value = value.reshape(-1, BLOCK)
            value = value.sqrt() if name == "v" else value
            top = MAX_V if name == "v" else MAX_M
            scale = value.abs().amax(1) / top
            y = value.abs() / scale.clamp_min(1e-30)[:, None] * 2.0 ** -120
            code = (y.view(torch.int32) >> (19 if name == "v" else 20)).clamp_max(255 if name == "v" else 127)
            code = torch.where((value > 0) & (code == 0), 1, code) if name == "v" else code | ((value < 0).int() << 7)
            s[name], s[name + "_scale"] = code.to(torch.uint8).reshape(-1), scale
        s["step"] = 10
    return s


HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
SEED = 5  # of the 8-bit states' rounding


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _run_attention(state, case)
    if case["op"] == "norm":
        return _run_norm(state, case)
    return _run_adamw(state, case)


def _run_attention(s, case):
    nq = case["queries"]
    q, k, v = s["qkv"].unbind(2)
    q = q[:, :nq]
    if own:
        from hive_neuralnet_b200 import train_ops as ops
        args = (s["tq"], s["tr"], s["tz"], s["mask"], s["bq"], s["br"], s["bz"])
        out, saved = ops.relative_attention_forward(q, k, v, *args, save=case["grad"])
        if not case["grad"]:
            return [out]
        return [out, *ops.relative_attention_backward(s["dout"], q, k, v, *args, saved)]

    dt, scale = s["qkv"].dtype, case["head_dim"] ** -0.5
    mask = s["mask"]
    rows = mask[:, :nq]

    def heads(t, keep):  # [B, n, H, D] -> [B, H, n, D] in 32 bits, masked tokens cleared
        return torch.where(keep[:, :, None, None], t.float(), 0.0).permute(0, 2, 1, 3)

    def offset(t, clip):  # of key j from query i, clipped and shifted to an index
        return (t[:, None, :] - t[:, :nq, None]).clamp(-clip, clip) + clip

    q, k, v = heads(q, rows), heads(k, mask), heads(v, mask)
    iq, ir, iz = offset(s["tq"], CLIP), offset(s["tr"], CLIP), offset(s["tz"], CLIP_Z)
    bias = s["bq"][iq] + s["br"][ir] + s["bz"][iz]
    scores = q @ k.transpose(-2, -1) * scale + bias.permute(0, 3, 1, 2)
    keep = rows[:, None, :, None] & mask[:, None, None, :]
    scores = torch.where(keep, scores, -1e30)
    p = torch.exp(scores - scores.amax(-1, keepdim=True)) * keep
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = (p @ v).permute(0, 2, 1, 3).to(dt)
    if not case["grad"]:
        return [out]
    dout = heads(s["dout"], rows)
    dp = dout @ v.transpose(-2, -1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    grads = [ds @ k * scale, ds.transpose(-2, -1) @ q * scale, p.transpose(-2, -1) @ dout]
    by_pair = ds.permute(0, 2, 3, 1)  # [B, query, key, H]

    def table(index, size):  # sums of ds over the pairs of each offset, one query at a time first
        hot = (index[..., None] == torch.arange(size, device=index.device)).float()
        return (hot.transpose(-2, -1) @ by_pair).sum((0, 1))

    return [out, *(t.permute(0, 2, 1, 3).to(dt) for t in grads), table(iq, 2 * CLIP + 1), table(ir, 2 * CLIP + 1),
            table(iz, 2 * CLIP_Z + 1)]


def _run_norm(s, case):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        from hive_neuralnet_b200 import train_ops as ops
        y, total, mean, rstd = ops.layer_norm_forward(x, w, b, 1e-5, residual=s.get("residual"))
        outs = [y] + ([total] if case["residual"] else [])
        if case["grad"]:
            outs += ops.layer_norm_backward(s["dy"], total, w, mean, rstd, dsum=s.get("dsum"))
        return outs

    dt = x.dtype
    total = x
    if case["residual"]:
        total = (x.float() + s["residual"].float()).to(dt)  # the running stream keeps its type
    t = total.float()
    mean = t.mean(1, keepdim=True)
    centred = t - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    hat = centred * rstd
    outs = [(hat * w + b).to(dt)] + ([total] if case["residual"] else [])
    if case["grad"]:
        dy = s["dy"].float()
        dhat = dy * w
        dx = rstd * (dhat - dhat.mean(1, keepdim=True) - hat * (dhat * hat).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + s["dsum"].float()
        outs += [dx.to(dt), (dy * hat).sum(0), dy.sum(0)]
    return outs


# 8-bit states: the first moment as sign + 4 exponent + 3 mantissa bits, the root of the
# second as 4 exponent + 4 mantissa bits; code << 20 (19) are the bits of value * 2^-120.
MAX_M, MAX_V = 480.0, 496.0
M32 = 0xFFFFFFFF


def _values(code, scale, second):
    c = code.to(torch.int32)
    if second:
        y = (c << 19).view(torch.float32) * 2.0 ** 120
        r = y.reshape(-1, BLOCK) * scale[:, None]
        return (r * r).reshape(-1)
    y = ((c & 127) << 20).view(torch.float32) * 2.0 ** 120
    return (torch.where(c > 127, -y, y).reshape(-1, BLOCK) * scale[:, None]).reshape(-1)


def _noise(count, step, dev):
    """32 hashed bits for each state value and step (the rounding's random numbers)."""
    h = (torch.arange(count, device=dev) * 0x9E3779B1 + (SEED * 0x6A09E667 + step * 0xBB67AE85)) & M32
    h = ((h ^ (h >> 16)) * 0x6A09E667) & M32
    h = ((h ^ (h >> 13)) * 0xBB67AE85) & M32
    return h ^ (h >> 16)


def _codes(x, noise, second):
    x = x.reshape(-1, BLOCK)
    mag = x.sqrt() if second else x.abs()
    peak = mag.amax(1, keepdim=True)
    top = MAX_V if second else MAX_M
    live = peak >= 2.0 ** -100
    inv = torch.where(live, torch.full_like(peak, top) / peak, 0.0)
    bits = (mag * inv * 2.0 ** -120).view(torch.int32)
    noise = noise.reshape(-1, BLOCK)
    if second:
        code = ((bits + (noise >> 13).int()) >> 19).clamp_max(255)
        code = torch.where((mag > 0) & live, code.clamp_min(1), code)  # a live mean is never rounded to none
    else:
        code = ((bits + (noise & 0xFFFFF).int()) >> 20).clamp_max(127) | ((x < 0).int() << 7)
    code = torch.where(live, code, 0)
    scale = torch.where(live, peak / torch.full_like(peak, top), 0.0)
    return code.to(torch.uint8).reshape(-1), scale.reshape(-1)


def _run_adamw(s, case):
    step = s["step"] = s["step"] + 1
    small = case["bits"] == 8
    if own:
        from hive_neuralnet_b200 import train_ops as ops
        scales = (s["m_scale"], s["v_scale"]) if small else None
        ops.adamw_step(s["params"], s["grads"], s["m"], s["v"], step=step, scales=scales, seed=SEED, **HYPER)
        if small:
            m, v = ops.exp_avg_values(s["m"], s["m_scale"]), ops.exp_avg_sq_values(s["v"], s["v_scale"])
        else:
            m, v = s["m"], s["v"]
    else:
        (b1, b2), lr, eps, wd = HYPER["betas"], HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
        flat = [t.view(-1) for t in s["params"]]
        p, g = (torch.zeros(s["padded"], device=s["m"].device) for _ in range(2))  # in 32 bits, laid out as the states
        torch._foreach_copy_(_parts(p, s), flat)
        torch._foreach_copy_(_parts(g, s), [t.view(-1) for t in s["grads"]])
        m, v = (_values(s["m"], s["m_scale"], False), _values(s["v"], s["v_scale"], True)) if small else (s["m"], s["v"])
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        denom = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + eps
        p = p * (1 - lr * wd) - (m / denom) * (lr / (1 - b1 ** step))
        torch._foreach_copy_(flat, _parts(p, s))
        if small:
            noise = _noise(s["padded"], step, p.device)
            for name, x in (("m", m), ("v", v)):
                code, scale = _codes(x, noise, name == "v")
                s[name].copy_(code)
                s[name + "_scale"].copy_(scale)
            m, v = _values(s["m"], s["m_scale"], False), _values(s["v"], s["v_scale"], True)
        else:
            s["m"].copy_(m)
            s["v"].copy_(v)
            m, v = s["m"], s["v"]
    params = s["params"]
    return [m, v, *([torch.cat([p.reshape(-1) for p in params])] if len(params) > 60 else params)]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "attention":
        b, n, nq, h, d = (case[k] for k in ("batch", "tokens", "queries", "heads", "head_dim"))
        c = _counts(case)
        share = nq / n if case["holes"] and nq < n else 1.0
        rows = np.minimum(c, nq) if nq == n or not case["holes"] else np.maximum(1, c * share)
        pairs, live, keys = float((rows * c).sum()) * h, float(rows.sum()), float(c.sum())
        bytes_ = e * h * d * (live + 2 * keys + b * nq) + 13.0 * b * n
        flops = 4.0 * d * pairs
        if case["grad"]:
            bytes_ += e * h * d * (live + b * nq + 2.0 * b * n)
            flops += 8.0 * d * pairs
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "norm":
        r, w = case["rows"], case["width"]
        n = 2 + (2 if case["residual"] else 0) + ((2 + (1 if case["residual"] else 0)) if case["grad"] else 0)
        return {"bytes": float(e * r * w * n + 8 * w * (2 if case["grad"] else 1)),
                "flops": (8.0 + (10 if case["grad"] else 0)) * r * w}
    n = float(sum(int(np.prod(x)) for x in tensor_shapes(case)))
    state = 16.0 if case["bits"] == 32 else 4 + 8 + 16 / BLOCK  # 8 bits: the codes both ways, the values that come back
    return {"bytes": n * (3 * e + state), "flops": 14 * n}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s, case)
    if case["op"] == "norm":
        return _exact_norm(s, case)
    return _exact_adamw(s, case)


def _exact_attention(s, case):
    nq, d = case["queries"], case["head_dim"]
    full = s["qkv"].double()
    full = full.masked_fill(~s["mask"][:, :, None, None, None], 0.0).requires_grad_(case["grad"])
    rel = [torch.stack([t[:, j] for j in range(nq)], 1) if nq < 2 else t[:, :nq] for t in (s["tq"], s["tr"], s["tz"])]
    index = [torch.clamp(t.unsqueeze(1).long() - r.unsqueeze(2).long(), -c, c) + c
             for t, r, c in zip((s["tq"], s["tr"], s["tz"]), rel, (CLIP, CLIP, CLIP_Z))]
    bias = sum(torch.nn.functional.embedding(i, w.double()) for i, w in zip(index, (s["bq"], s["br"], s["bz"])))
    bias = bias.movedim(3, 1).contiguous().requires_grad_(case["grad"])
    logit = torch.einsum("bihd,bjhd->bhij", full[:, :nq, 0], full[:, :, 1]) / math.sqrt(d) + bias
    logit = logit.masked_fill(~s["mask"][:, None, None, :], -math.inf)
    out = torch.einsum("bhij,bjhd->bihd", torch.softmax(logit, -1), full[:, :, 2])
    live = s["mask"][:, :nq, None, None].double()
    out = out * live
    if not case["grad"]:
        return [out.detach()]
    dfull, dbias = torch.autograd.grad(out, (full, bias), s["dout"].double().masked_fill(live == 0, 0.0))
    tables = []
    for i, c in zip(index, (CLIP, CLIP, CLIP_Z)):
        tables.append(torch.stack([(dbias * (i == k).unsqueeze(1)).sum((0, 2, 3)) for k in range(2 * c + 1)]))
    return [out.detach(), dfull[:, :nq, 0], dfull[:, :, 1], dfull[:, :, 2], *tables]


def _exact_norm(s, case):
    x = s["x"].double()
    if case["residual"]:
        x = (x + s["residual"].double()).to(s["x"].dtype).double()  # kept in its type by definition
    outs = [x.clone()] if case["residual"] else []
    x = x.requires_grad_(case["grad"])
    w, b = (s[k].double().requires_grad_(case["grad"]) for k in ("weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    y = torch.addcmul(b, (x - mean) * torch.rsqrt(var + 1e-5), w)
    if case["grad"]:
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        outs += [dx + s["dsum"].double() if case["residual"] else dx, dw, db]
    return [y.detach(), *outs]


def _exact_adamw(s, case):
    (b1, b2), lr, eps, wd = HYPER["betas"], HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    t = s["step"] + 1
    if case["bits"] == 8:
        def decode(code, bits, scale):
            c = code.cpu().numpy().astype(np.int64)
            sign = np.where(c >> 7, -1.0, 1.0) if bits == 3 else 1.0
            c = c & 127 if bits == 3 else c
            e, f = c >> bits, (c & ((1 << bits) - 1)) / (1 << bits)
            y = sign * np.where(e > 0, (1 + f) * 2.0 ** (e - 7.0), f * 2.0 ** -6)
            return torch.from_numpy(y).to(scale.device) * scale.double().repeat_interleave(BLOCK)
        m0, v0 = decode(s["m"], 3, s["m_scale"]), decode(s["v"], 4, s["v_scale"]).square()
    else:
        m0, v0 = s["m"].double(), s["v"].double()
    off = s["offsets"]
    ms, vs, ps = torch.zeros_like(m0), torch.zeros_like(v0), []
    for p, g, o, n in zip(s["params"], s["grads"], off, s["sizes"]):
        g = g.double().flatten()
        m = torch.lerp(g, m0[o:o + n], b1)
        v = torch.lerp(g.square(), v0[o:o + n], b2)
        ms[o:o + n], vs[o:o + n] = m, v
        p = p.double().flatten()
        p = p - lr * wd * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
        ps.append(p)
    states = [None, None] if case["bits"] == 8 else [ms, vs]
    shapes = [p.shape for p in s["params"]]
    return [*states, *([torch.cat(ps)] if len(ps) > 60 else [p.view(x) for p, x in zip(ps, shapes)])]
