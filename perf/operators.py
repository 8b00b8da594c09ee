"""What is measured of the transformer-block operators: layer normalisation, dropout whose mask is
never stored, rotary positions over several axes, attention with a sliding window and sinks.

`listed()` names the cases, `draw(rng)` makes one more of the same ranges, `prepare(case, seed)`
makes what a training program holds before the call, `run(state)` is one pass, `exact(case, seed)`
the same outputs from the definition in 64 bits, `work(case)` the bytes and operations a pass
cannot do without.  With `own` false a pass is computed by elementary torch operations.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}

# the largest work of each operator among the listed cases; draws stay below it
_LN_ELEMENTS = 184 * 196 * 2048
_DROPOUT_ELEMENTS = 184 * 196 * 4096
_ROTARY_ELEMENTS = 184 * 196 * 16 * 64
_ATTN_SCORES = 16 * 15808 * 15808
_ATTN_FLOPS_D = 16 * 15808 * 128


# ------------------------------------------------------------------------------------- cases
def _ln(name, rows, dim, dtype, wtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "dim": dim, "dtype": dtype,
            "wtype": wtype, "train": train}


def _drop(name, rows, dim, dtype, p, train):
    return {"name": name, "op": "dropout", "rows": rows, "dim": dim, "dtype": dtype, "p": p,
            "train": train}


def _rot(name, batch, frames, height, width, heads, dim, sections, dtype, joint, interleaved,
         train):
    """`sections` is a text such as "16,16": rotated pairs per axis, as many axes as numbers; the
    axes are the last ones of (frame, row, column)."""
    return {"name": name, "op": "rotary", "batch": batch, "frames": frames, "height": height,
            "width": width, "heads": heads, "dim": dim, "sections": sections, "dtype": dtype,
            "joint": joint, "interleaved": interleaved, "train": train}


def _attn(name, batch, tokens, heads, kv_heads, dim, dtype, left, right, sinks, lengths, train):
    """`lengths`: "full", "ragged" (entry b of the padded batch holds T*(B-b)//B tokens) or
    "empty" (like ragged, but the last of several entries holds none)."""
    return {"name": name, "op": "attention", "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "left": left, "right": right,
            "sinks": sinks, "lengths": lengths, "train": train}


def listed():
    """196 tokens: a 224 x 224 image in patches of 16; 988: a 416 x 608 image (26 x 38 patches);
    184 and 11: the batches the benchmark trains those images at."""
    return [
        # the normalised class token of one image: latency
        _ln("layer_norm one row bf16", 1, 512, "bf16", "bf16", False),
        # a training step's norm in the framework's default type, one token more than patches
        _ln("layer_norm train 184x197x384 fp32", 184 * 197, 384, "fp32", "fp32", True),
        # the widest norm of a bf16 step with fp32 parameters
        _ln("layer_norm train 184x196x2048 bf16", 184 * 196, 2048, "bf16", "fp32", True),
        # the hidden layer of a block's feed-forward part
        _drop("dropout 184x196x4096 bf16", 184 * 196, 4096, "bf16", 0.1, False),
        # a residual branch of odd width, forward and backward
        _drop("dropout train 11x988x1023 fp32", 11 * 988, 1023, "fp32", 0.25, True),
        # queries of a batch of images, an axis for rows and one for columns
        _rot("rotary 184 images 14x14 bf16", 184, 1, 14, 14, 16, 64, "16,16", "bf16", False, False,
             False),
        # a short video: three axes over one range of frequencies, part of the head left as it is
        _rot("rotary train video 7x26x38 fp32", 1, 7, 26, 38, 12, 80, "10,11,12", "fp32", True, True,
             True),
        # one image reduced to one token: latency
        _attn("attention one token bf16", 1, 1, 8, 8, 64, "bf16", 128, 0, 4, "full", False),
        # a step's images, every patch sees a band of patches on both sides, and the first one
        _attn("attention 11x988 both sides bf16", 11, 988, 16, 16, 64, "bf16", 200, 200, 1, "full",
              False),
        # tokens of a long video in order, shared heads, training
        _attn("attention train 15808 window 1024 bf16", 1, 15808, 16, 4, 128, "bf16", 1024, 0, 4,
              "full", True),
        # the framework's default type on a padded batch of images
        _attn("attention train ragged fp32", 8, 197, 12, 12, 64, "fp32", 96, 96, 1, "ragged", True),
        # no window: every earlier token, an odd length
        _attn("attention train causal 4099 fp16", 2, 4099, 12, 6, 96, "fp16", -1, 0, 0, "full", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "rotary", "attention", "attention"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.6
    if op == "layer_norm":
        dim = _log_int(rng, 8, 8192)
        rows = _log_int(rng, 1, 184 * 197)
        rows = max(1, min(rows, _LN_ELEMENTS * 2 // (_BYTES[dtype] * dim)))
        return _unnamed(_ln("", rows, dim, dtype, rng.choice([dtype, "fp32"]), train))
    if op == "dropout":
        dim = _log_int(rng, 1, 4096)
        rows = _log_int(rng, 1, 184 * 196)
        # (a pass in both directions writes twice)
        rows = max(1, min(rows, _DROPOUT_ELEMENTS // (_BYTES[dtype] * dim)))
        p = rng.choice([0.0, 0.1, 0.5, round(rng.uniform(0.01, 0.95), 4)])
        return _unnamed(_drop("", rows, dim, dtype, p, train))
    if op == "rotary":
        axes = rng.randint(1, 3)
        heads = rng.randint(1, 32)
        sections = [rng.randint(1, 64 // axes) for _ in range(axes)]
        dim = 2 * sum(sections) + rng.choice([0, 0, rng.randint(1, 32)])
        frames = _log_int(rng, 1, 16) if axes == 3 else 1
        height = _log_int(rng, 1, 64) if axes > 1 else 1
        width = _log_int(rng, 1, 64) if axes > 1 else _log_int(rng, 1, 16384)
        batch = _log_int(rng, 1, 184)
        room = _ROTARY_ELEMENTS * 2 // (_BYTES[dtype] * (2 if train else 1))
        batch = max(1, min(batch, room // (frames * height * width * heads * dim)))
        while frames * height * width * heads * dim > room:
            heads = max(1, heads // 2)
            width = max(1, width // 2)
        return _unnamed(_rot("", batch, frames, height, width, heads, dim,
                             ",".join(str(s) for s in sections), dtype, rng.random() < 0.5,
                             rng.random() < 0.5, train))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, rng.randint(8, 128)])
    tokens = _log_int(rng, 1, 15808)
    batch = _log_int(rng, 1, 16)
    cap = min(_ATTN_SCORES, 256 << 20 if dtype == "fp32" else _ATTN_SCORES)
    batch = max(1, min(batch, cap // (heads * tokens * tokens)))
    tokens = min(tokens, int(math.sqrt(cap / (heads * batch))))
    left = rng.choice([-1, 0, _log_int(rng, 1, 2048), _log_int(rng, 1, 2048)])
    right = rng.choice([0, 0, 0, left])
    sinks = rng.choice([0, 1, 4, rng.randint(1, 80)])
    # a window of everything is kept to lengths whose work stays below the largest listed case's
    if left < 0 or right < 0 or sinks > 16:
        tokens = min(tokens, int(math.sqrt(_ATTN_FLOPS_D * 1024 / (heads * batch * dim))))
    return _unnamed(_attn("", batch, tokens, heads, kv_heads, dim, dtype, left, right, sinks,
                          rng.choice(["full", "full", "ragged", "empty"]), train))


def _unnamed(case):
    del case["name"]
    return case


# ------------------------------------------------------------------------------------ inputs
def _lengths(case):
    B, T = case["batch"], case["tokens"]
    if case["lengths"] == "full":
        return [T] * B
    out = [T * (B - b) // B for b in range(B)]
    if case["lengths"] == "empty" and B > 1:
        out[-1] = 0
    return out


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, device=dev, generator=g).mul_(scale).to(dtype)

    op = case["op"]
    t = {}
    if op == "layer_norm":
        rows, dim = case["rows"], case["dim"]
        # a residual stream: rows off centre, a few channels much larger than the rest
        x = torch.randn(rows, dim, device=dev, generator=g)
        x.mul_(0.5 + torch.rand(rows, 1, device=dev, generator=g))
        x.add_(torch.randn(rows, 1, device=dev, generator=g), alpha=0.5)
        x[:, :: max(1, dim // 4)] *= 8.0
        t["x"] = x.to(dt)
        wt = _DTYPES[case["wtype"]]
        t["weight"] = (1.0 + 0.2 * torch.randn(dim, device=dev, generator=g)).to(wt)
        t["bias"] = (0.1 * torch.randn(dim, device=dev, generator=g)).to(wt)
        if case["train"]:
            t["grad"] = randn(rows, dim, scale=0.1)
    elif op == "dropout":
        t["x"] = randn(case["rows"], case["dim"])
        t["p"] = case["p"]
        t["state"] = torch.randint(0, 1 << 62, (2,), device=dev, generator=g, dtype=torch.int64)
        if case["train"]:
            t["grad"] = randn(case["rows"], case["dim"], scale=0.1)
    elif op == "rotary":
        F, H, W = case["frames"], case["height"], case["width"]
        shape = (case["batch"], F * H * W, case["heads"], case["dim"])
        t["x"] = randn(*shape)
        n = torch.arange(F * H * W, device=dev)
        axes = [n // (H * W), n // W % H, n % W]
        # positions of a crop somewhere in the picture or the film
        start = torch.randint(0, 1000, (3,), device=dev, generator=g)
        t["positions"] = torch.stack([axes[a] + start[a] for a in range(3)])[
            3 - len(_sections(case)):].contiguous()
        if case["train"]:
            t["grad"] = randn(*shape, scale=0.1)
    else:
        B, T, D = case["batch"], case["tokens"], case["dim"]
        H, K = case["heads"], case["kv_heads"]
        # one projection's output, as a block computes it: q, k and v are views of it
        qkv = randn(B, T, H + 2 * K, D)
        t["q"], t["k"], t["v"] = qkv[:, :, :H], qkv[:, :, H:H + K], qkv[:, :, H + K:]
        if case["lengths"] != "full":
            t["lengths"] = torch.tensor(_lengths(case), device=dev, dtype=torch.int32)
        if case["train"]:
            t["grad"] = randn(B, T, H, D, scale=0.1)
    return t


def prepare(case, seed):
    return {"case": case, "in": _inputs(case, seed)}


def run(state):
    return (_run_own if own else _run_plain)(state["case"], state["in"])


# ------------------------------------------------------------------------ the framework's calls
def _run_own(case, t):
    from monet_amd import lm_ops
    op, train = case["op"], case["train"]
    if op == "layer_norm":
        y, mean, rstd = lm_ops.layernorm.layer_norm_forward(
            t["x"], (case["dim"],), t["weight"], t["bias"], 1e-5)
        if not train:
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dw, db = lm_ops.layernorm.layer_norm_backward(
            t["grad"], t["x"], mean, rstd, t["weight"], t["bias"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if op == "dropout":
        out = {"y": lm_ops.dropout.dropout_forward(t["x"], t["p"], t["state"])}
        if train:
            out["dx"] = lm_ops.dropout.dropout_backward(t["grad"], t["p"], t["state"])
        return out
    if op == "rotary":
        how = (t["positions"], _sections(case), 10000.0, case["joint"], case["interleaved"])
        out = {"y": lm_ops.rotary.rotary_forward(t["x"], *how)}
        if train:
            out["dx"] = lm_ops.rotary.rotary_backward(t["grad"], *how)
        return out
    how = dict(left=case["left"], right=case["right"], sinks=case["sinks"],
               lengths=t.get("lengths"))
    out, lse = lm_ops.attention.window_attention_forward(t["q"], t["k"], t["v"], **how)
    if not train:
        return {"out": out, "lse": lse} if case["lengths"] == "full" else {"out": out}
    dq, dk, dv = lm_ops.attention.window_attention_backward(t["grad"], t["q"], t["k"], t["v"], out,
                                                            lse, **how)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


# ------------------------------------------------------------------------------ the plain forms
def _run_plain(case, t):
    return {"layer_norm": _plain_layer_norm, "dropout": _plain_dropout, "rotary": _plain_rotary,
            "attention": _plain_attention}[case["op"]](case, t)


def _plain_layer_norm(case, t):
    dt = t["x"].dtype
    x, w, b = t["x"].float(), t["weight"].float(), t["bias"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
    xh = xc * rstd
    y = (xh * w + b).to(dt)
    if not case["train"]:
        return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0]}
    g = t["grad"].float()
    dw = (g * xh).sum(0, dtype=torch.float64).to(t["weight"].dtype)
    db = g.sum(0, dtype=torch.float64).to(t["bias"].dtype)
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dw": dw, "db": db}


_M32 = 0xFFFFFFFF


def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 (Salmon et al., Parallel random numbers: as easy as 1, 2, 3, 2011) on int64
    tensors that hold 32-bit words."""
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, \
            ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return c0, c1, c2, c3


def _uniform_words(n, state):
    """One 32-bit number for each of n elements: eight elements share a counter, whose four words
    give each element the high half of its number; the low half comes from the same counter with
    bit 31 of its second word set."""
    groups = torch.arange((n + 7) // 8, device=state.device)
    seed, offset = state[0], state[1]
    halves = []
    for low in (0, 1 << 31):
        words = _philox(groups & _M32, (groups >> 32) | low, offset & _M32, (offset >> 32) & _M32,
                        seed & _M32, (seed >> 32) & _M32)
        w = torch.stack(words, 1)
        halves.append(torch.stack((w & 0xFFFF, w >> 16), 2).reshape(-1)[:n])
    return (halves[0] << 16) | halves[1]


def _plain_dropout(case, t):
    p = t["p"]
    keep = _uniform_words(t["x"].numel(), t["state"]) >= min(round(p * 2 ** 32), 2 ** 32 - 1)
    keep = keep.view(t["x"].shape)
    scale = 1.0 / (1.0 - p)
    out = {"y": torch.where(keep, t["x"].float() * scale, 0.0).to(t["x"].dtype)}
    if case["train"]:
        out["dx"] = torch.where(keep, t["grad"].float() * scale, 0.0).to(t["x"].dtype)
    return out


def _angles(case, positions):
    """[T, pairs], in 64 bits."""
    sections = _sections(case)
    n = sum(sections)
    cols, first = [], 0
    for a, s in enumerate(sections):
        i = torch.arange(s, device=positions.device, dtype=torch.float64)
        power = (i + first) / n if case["joint"] else i / s
        cols.append(positions[a].double()[:, None] * torch.pow(10000.0, -power)[None, :])
        first += s
    return torch.cat(cols, 1)


def _turn(x, cos, sin, interleaved):
    n = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _plain_rotary(case, t):
    angle = _angles(case, t["positions"])
    cos, sin = angle.cos().float()[None, :, None], angle.sin().float()[None, :, None]
    out = {"y": _turn(t["x"].float(), cos, sin, case["interleaved"]).to(t["x"].dtype)}
    if case["train"]:
        out["dx"] = _turn(t["grad"].float(), cos, -sin, case["interleaved"]).to(t["x"].dtype)
    return out


def _visible(case, rows, T, lengths):
    """[B, 1, rows, T]: which keys the query rows see."""
    i, j = rows[:, None], torch.arange(T, device=rows.device)[None, :]
    see = torch.ones(i.shape[0], T, dtype=torch.bool, device=rows.device)
    if case["right"] >= 0:
        see &= j <= i + case["right"]
    if case["left"] >= 0:
        see &= (j >= i - case["left"]) | (j < case["sinks"])
    if lengths is None:
        return see[None, None]
    n = lengths.long()[:, None, None]
    return (see[None] & (j[None] < n) & (i[None] < n))[:, None]


def _plain_attention(case, t):
    B, T, H, D = t["q"].shape
    group = H // case["kv_heads"]
    dt = t["q"].dtype
    scale = 1.0 / math.sqrt(D)
    q = t["q"].float().transpose(1, 2)
    k = t["k"].float().transpose(1, 2).repeat_interleave(group, 1).contiguous()
    v = t["v"].float().transpose(1, 2).repeat_interleave(group, 1).contiguous()
    kt, vt = k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous()
    out = torch.empty_like(q)
    lse = q.new_empty(B, H, T)
    train = case["train"]
    if train:
        g = t["grad"].float().transpose(1, 2).contiguous()
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, min(T, (1 << 28) // (B * H * T)))
    for r0 in range(0, T, step):
        r1 = min(T, r0 + step)
        see = _visible(case, torch.arange(r0, r1, device=q.device), T, t.get("lengths"))
        s = torch.matmul(q[:, :, r0:r1], kt) * scale
        s = s.masked_fill(~see, -math.inf)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        p = torch.exp(s - m)
        total = p.sum(-1, keepdim=True)
        lse[:, :, r0:r1] = (m + torch.log(total))[..., 0]
        p = p / torch.where(total == 0, 1.0, total)
        o = torch.matmul(p, v)
        out[:, :, r0:r1] = o
        if train:
            gr = g[:, :, r0:r1]
            dv += torch.matmul(p.transpose(2, 3).contiguous(), gr)
            ds = p * (torch.matmul(gr, vt) - (gr * o).sum(-1, keepdim=True)) * scale
            dq[:, :, r0:r1] = torch.matmul(ds, k)
            dk += torch.matmul(ds.transpose(2, 3).contiguous(), q[:, :, r0:r1])
    out = out.transpose(1, 2).contiguous().to(dt)
    if not train:
        return {"out": out, "lse": lse} if case["lengths"] == "full" else {"out": out}
    shared = (B, case["kv_heads"], group, T, D)
    dk, dv = dk.view(shared).sum(2), dv.view(shared).sum(2)
    return {"out": out, "dq": dq.transpose(1, 2).contiguous().to(dt),
            "dk": dk.transpose(1, 2).contiguous().to(dt),
            "dv": dv.transpose(1, 2).contiguous().to(dt)}


# ------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    t = {k: (v.double() if torch.is_tensor(v) and v.is_floating_point() else v)
         for k, v in _inputs(case, seed).items()}
    return {"layer_norm": _exact_layer_norm, "dropout": _exact_dropout, "rotary": _exact_rotary,
            "attention": _exact_attention}[case["op"]](case, t)


def _exact_layer_norm(case, t):
    x, w, b = t["x"], t["weight"], t["bias"]
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + 1e-5)
    y = torch.addcmul(b, (x - mean) * rstd, w)
    if not case["train"]:
        return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0]}
    # through the chain rule: y <- normalised <- (centred, rstd) <- x
    g, n = t["grad"], x.shape[1]
    dxh = g * w
    dvar = (dxh * (x - mean)).sum(1, keepdim=True) * -0.5 * rstd ** 3
    dmean = -(dxh * rstd).sum(1, keepdim=True)
    dx = dxh * rstd + dvar * 2.0 * (x - mean) / n + dmean / n
    return {"y": y, "dx": dx, "dw": ((x - mean) * rstd).mul_(g).sum(0), "db": g.sum(0)}


def _exact_dropout(case, t):
    # the generator's words are whole numbers: what is computed is the product alone
    keep = (_uniform_words(t["x"].numel(), t["state"]) >=
            min(int(math.floor(t["p"] * 2 ** 32 + 0.5)), 2 ** 32 - 1)).view(t["x"].shape).double()
    out = {"y": t["x"] * keep / (1.0 - t["p"])}
    if case["train"]:
        out["dx"] = t["grad"] * keep / (1.0 - t["p"])
    return out


def _exact_rotary(case, t):
    # pairs as complex numbers, turned by exp(i angle)
    sections = _sections(case)
    n = sum(sections)
    freq, axis = [], []
    for a, s in enumerate(sections):
        for i in range(s):
            freq.append(10000.0 ** -((len(axis)) / n if case["joint"] else i / s))
            axis.append(a)
    freq = torch.tensor(freq, device=t["x"].device, dtype=torch.float64)
    pos = t["positions"].double()[torch.tensor(axis, device=freq.device)]      # [pairs, T]
    phase = torch.polar(torch.ones_like(pos), pos * freq[:, None]).t()[None, :, None]

    def turn(x, by):
        if case["interleaved"]:
            z = torch.complex(x[..., 0:2 * n:2].contiguous(), x[..., 1:2 * n:2].contiguous()) * by
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * by
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., 2 * n:]), -1)

    out = {"y": turn(t["x"], phase)}
    if case["train"]:
        out["dx"] = turn(t["grad"], phase.conj())
    return out


def _exact_attention(case, t):
    B, T, H, D = t["q"].shape
    K = case["kv_heads"]
    group = H // K
    dev = t["q"].device
    train = case["train"]
    out = torch.zeros(B, T, H, D, device=dev, dtype=torch.float64)
    lse = torch.full((B, H, T), -math.inf, device=dev, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(out), torch.zeros_like(t["k"]), torch.zeros_like(t["v"])
    lens = _lengths(case)
    left = T if case["left"] < 0 else case["left"]
    right = T if case["right"] < 0 else case["right"]
    rows = 512
    for b in range(B):
        n = lens[b]
        for r0 in range(0, n, rows):
            r1 = min(n, r0 + rows)
            # the keys some row of the block sees: the window's, and the sinks before it
            lo, hi = max(0, r0 - left), min(n, r1 + right)
            j = torch.cat((torch.arange(min(case["sinks"], lo), device=dev),
                           torch.arange(lo, hi, device=dev)))
            i = torch.arange(r0, r1, device=dev)[:, None]
            hidden = (j > i + right) | ((j < i - left) & (j >= case["sinks"]))
            for h in range(K):
                hs = slice(h * group, (h + 1) * group)
                kj, vj = t["k"][b, j, h], t["v"][b, j, h]
                qi = t["q"][b, r0:r1, hs].transpose(0, 1).contiguous()          # [group, rows, D]
                s = torch.matmul(qi, kj.t().contiguous()) / math.sqrt(D)
                s[:, hidden] = -math.inf
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - z[..., None])
                o = torch.matmul(p, vj)
                out[b, r0:r1, hs] = o.transpose(0, 1)
                lse[b, hs, r0:r1] = z
                if train:
                    g = t["grad"][b, r0:r1, hs].transpose(0, 1).contiguous()
                    dp = torch.matmul(g, vj.t().contiguous())
                    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[b, r0:r1, hs] = torch.matmul(ds, kj).transpose(0, 1)
                    # the group's query heads share the keys: one product over all their rows
                    dv[b, :, h].index_add_(0, j, torch.matmul(
                        p.reshape(-1, len(j)).t().contiguous(), g.reshape(-1, D)))
                    dk[b, :, h].index_add_(0, j, torch.matmul(
                        ds.reshape(-1, len(j)).t().contiguous(), qi.reshape(-1, D)))
    if not train:
        return {"out": out, "lse": lse} if case["lengths"] == "full" else {"out": out}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


# -------------------------------------------------------------------------------- what it takes
def _pairs(case):
    """Query-key pairs that see each other, over the batch, of one head."""
    total = 0
    T = case["tokens"]
    left = T if case["left"] < 0 else case["left"]
    right = T if case["right"] < 0 else case["right"]
    for n in _lengths(case):
        for i in range(n):
            lo, hi = max(0, i - left), min(n, i + right + 1)
            total += hi - lo + min(case["sinks"], lo)
    return total


def work(case):
    e = _BYTES[case["dtype"]]
    op, train = case["op"], case["train"]
    if op == "layer_norm":
        n, d, w = case["rows"] * case["dim"], case["dim"], _BYTES[case["wtype"]]
        if not train:
            return {"bytes": 2 * n * e + 2 * d * w + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 4 * n * e + 4 * d * w, "flops": 20 * n}
    if op == "dropout":
        n = case["rows"] * case["dim"]
        return {"bytes": (4 if train else 2) * n * e + 16, "flops": (2 if train else 1) * n}
    if op == "rotary":
        tokens = case["frames"] * case["height"] * case["width"]
        n = case["batch"] * tokens * case["heads"]
        axes = len(_sections(case))
        return {"bytes": (4 if train else 2) * n * case["dim"] * e + 8 * axes * tokens,
                "flops": (2 if train else 1) * 6 * n * sum(_sections(case))}
    B, T, D = case["batch"], case["tokens"], case["dim"]
    q, kv = B * T * case["heads"] * D * e, B * T * case["kv_heads"] * D * e
    pairs = _pairs(case) * case["heads"]
    if not train:
        lse = 4 * B * case["heads"] * T if case["lengths"] == "full" else 0
        return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * D * pairs}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * D * pairs}
