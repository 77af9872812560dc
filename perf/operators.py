"""Timing cases of the operators that serve a model in 8 and 4 bits (the
library's `quant` kernels): products in 8-bit integers with a scale for each
token and each channel, the norm and the row quantisation that feed them, and
a paged cache held in 4 bits with the decode attention that reads it.

A case is a dict of plain values; `kind` names the operator. `prepare` makes
its inputs on the GPU, `run` is one pass (in plain torch, or through the
library where `own` is set), `exact` the same outputs in 64 bits.
"""

import math

import numpy as np
import torch

own = False
DEV = "cuda"

# (outputs, inputs) of projections in the repository's configurations and tests.
PROJECTIONS = ((2560, 2048), (2048, 2048), (2048, 5632), (4096, 4096), (4096, 11008), (96, 64))
# (dim, ffn) of their MLPs.
BLOCKS = ((2048, 5632), (1024, 4000), (4096, 11008), (64, 128))
# (query heads, kv heads, head dimension).
HEADS = ((32, 4, 64), (32, 8, 128), (8, 2, 64), (16, 16, 64), (16, 1, 128), (4, 2, 16), (8, 4, 32))


def listed():
    return [
        # The QKV projection of one token: a single chat session's decode step.
        {"name": "linear_1_token", "kind": "linear", "rows": 1, "n": 2560, "k": 2048},
        # A product nobody padded: every dimension odd.
        {"name": "linear_odd", "kind": "linear", "rows": 777, "n": 1155, "k": 1001},
        # The MLP's first half for a full decode batch: weights from HBM.
        {"name": "gate_up_32", "kind": "gate_up", "rows": 32, "dim": 2048, "ffn": 5632},
        # The same of a wider model for 2048 prompt tokens: the matrix cores' case.
        {"name": "gate_up_prefill", "kind": "gate_up", "rows": 2048, "dim": 4096, "ffn": 11008},
        # The norm between two projections of a decode batch, with the residual's addition.
        {"name": "norm_32", "kind": "norm", "rows": 32, "cols": 2048, "add": True},
        # The same for a prompt of odd length.
        {"name": "norm_2001", "kind": "norm", "rows": 2001, "cols": 4096, "add": True},
        # SwiGLU's outputs on their way into the down projection, prompt and decode sized.
        {"name": "quantize_4096", "kind": "quantize", "rows": 4096, "cols": 5632},
        {"name": "quantize_7", "kind": "quantize", "rows": 7, "cols": 11008},
        # Keys and values of a decode batch into the cache, and of packed prompts.
        {"name": "kv_write_64", "kind": "kv_write", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        {"name": "kv_write_2003", "kind": "kv_write", "tokens": 2003, "heads": 32, "kv_heads": 4, "dim": 64, "page": 32},
        # Decode attention of few short sequences.
        {"name": "attention_5_short", "kind": "attention", "seqs": 5, "heads": 32, "kv_heads": 4, "dim": 64,
         "page": 16, "lo": 20, "hi": 333},
        # A serving batch over a long cache, lengths far apart.
        {"name": "attention_64_long", "kind": "attention", "seqs": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "lo": 128, "hi": 4096},
    ]


def _log(rng, lo, hi):
    """A whole number in lo .. hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """As `_log`; half of them as drawn (odd ones), the others multiples of 8 or 64."""
    n = _log(rng, lo, hi)
    step = rng.choice((1, 1, 8, 64))
    return max(lo, min(hi, (n + step - 1) // step * step))


def _drawn(rng):
    kind = rng.choice(("linear", "linear", "gate_up", "norm", "quantize", "kv_write", "attention", "attention"))
    if kind == "linear":
        n, k = rng.choice(PROJECTIONS) if rng.random() < 0.6 else (_size(rng, 16, 8192), _size(rng, 16, 8192))
        return {"kind": kind, "rows": _log(rng, 1, 4096), "n": n, "k": k}
    if kind == "gate_up":
        dim, ffn = rng.choice(BLOCKS) if rng.random() < 0.7 else (_size(rng, 64, 4096), _size(rng, 64, 8192))
        return {"kind": kind, "rows": _log(rng, 1, 2048), "dim": dim, "ffn": ffn}
    if kind == "norm":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": _size(rng, 64, 8192), "add": rng.random() < 0.7}
    if kind == "quantize":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": _size(rng, 16, 16384)}
    heads, kv, dim = rng.choice(HEADS)
    if kind == "kv_write":
        return {"kind": kind, "tokens": _log(rng, 1, 2048), "heads": heads, "kv_heads": kv, "dim": dim,
                "page": rng.choice((16, 32, 64))}
    hi = _log(rng, 16, 16384)
    return {"kind": kind, "seqs": _log(rng, 1, 64), "heads": heads, "kv_heads": kv, "dim": dim,
            "page": rng.choice((16, 16, 32, 64)), "lo": max(1, hi // rng.choice((1, 4, 32))), "hi": hi}


def draw(rng):
    while True:
        case = _drawn(rng)
        w = work(case)
        if w["flops"] <= 3.6e11 and w["bytes"] <= 1.6e8:
            return case


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape, scale=1.0, dtype=torch.float16):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(dtype)


def _rows8(g, rows, cols, scale):
    """Rows of normal values in 8 bits: codes, and a scale for each row."""
    x = torch.randn(rows, cols, generator=g, device=DEV).mul_(scale)
    s = x.abs().amax(1).clamp_min(1e-6) / 127
    return torch.round(x / s[:, None]).clamp_(-127, 127).to(torch.int8), s


def _linear_state(c, g):
    x, sx = _rows8(g, c["rows"], c["k"], 1.0)
    w, sw = _rows8(g, c["n"], c["k"], c["k"] ** -0.5)
    return {"x": x, "sx": sx, "w": w, "sw": sw, "y": torch.zeros(c["rows"], c["n"], dtype=torch.float16, device=DEV)}


def _gate_up_state(c, g):
    x, sx = _rows8(g, c["rows"], c["dim"], 1.0)
    (wg, sg), (wu, su) = (_rows8(g, c["ffn"], c["dim"], c["dim"] ** -0.5) for _ in range(2))
    return {"x": x, "sx": sx, "wg": wg, "sg": sg, "wu": wu, "su": su,
            "y": torch.zeros(c["rows"], c["ffn"], dtype=torch.float16, device=DEV)}


def _norm_state(c, g):
    """The residual stream with a few loud channels, a projection's output, and the norm's weights."""
    t, d = c["rows"], c["cols"]
    loud = torch.rand(d, generator=g, device=DEV) < 0.01
    r = _normal(g, t, d, dtype=torch.float32) * torch.where(loud, 12.0, 1.0)
    s = {"r": r, "w": (1.0 + _normal(g, d, scale=0.1, dtype=torch.float32)).half(),
         "q": torch.zeros(t, d, dtype=torch.int8, device=DEV), "s": torch.zeros(t, device=DEV), "eps": 1e-5}
    if c["add"]:
        s["x"] = _normal(g, t, d, scale=0.5)
    return s


def _quantize_state(c, g):
    """Gated activations: products of two normal values, a hundredth of the rows all zero (padding)."""
    m, k = c["rows"], c["cols"]
    x = _normal(g, m, k, dtype=torch.float32) * _normal(g, m, k, dtype=torch.float32)
    x *= (torch.rand(m, 1, generator=g, device=DEV) >= 0.01)
    return {"x": x.half(), "q": torch.zeros(m, k, dtype=torch.int8, device=DEV), "s": torch.zeros(m, device=DEV)}


def _tables(npos, d, theta=10000.0):
    inv = theta ** (-torch.arange(0, d, 2, device=DEV).double() / d)
    a = torch.arange(npos, device=DEV).double()[:, None] * inv
    return torch.cos(a).float(), torch.sin(a).float()


def _kv_write_state(c, g):
    """A step's QKV rows, positions and slots (each a place of its own, in the order of the pages' random
    allocation), a cache that holds something already."""
    t, h, kv, d, p = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    pages = (t + p - 1) // p + 1
    cos, sin = _tables(4096, d)
    pos = torch.randint(0, 4096, (t,), generator=g, device=DEV, dtype=torch.int32)
    slot = torch.randperm(pages * p, generator=g, device=DEV)[:t].to(torch.int32)
    return {"qkv": _normal(g, t, (h + 2 * kv) * d), "pos": pos, "slot": slot, "cos": cos, "sin": sin,
            **_cache(g, pages, kv, p, d), "k": torch.zeros(t, kv, d, dtype=torch.float16, device=DEV),
            "v": torch.zeros(t, kv, d, dtype=torch.float16, device=DEV)}


def _cache(g, pages, kv, p, d):
    """A pool of pages in 4 bits: two codes a byte, and (lowest value, step) of each token and head."""
    def codes(*shape):
        return torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8)

    def pairs():
        step = 0.25 + 0.25 * torch.rand(pages, kv, p, generator=g, device=DEV)
        low = -step * (6.0 + 3.0 * torch.rand(pages, kv, p, generator=g, device=DEV))
        return torch.stack([low, step], -1).half()

    return {"kc": codes(pages, kv, p, d // 2), "vc": codes(pages, kv, p // 16, d // 2, 16), "ks": pairs(), "vs": pairs()}


def _attention_state(c, g):
    """One query token for each sequence; its keys and values on pages in random order of a pool."""
    b, h, kv, d, p = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    lens = torch.randint(c["lo"], c["hi"] + 1, (b,), generator=g, device=DEV)
    per = (c["hi"] + p - 1) // p
    need = (lens + p - 1) // p
    pages = b * per
    table = torch.randperm(pages, generator=g, device=DEV).view(b, per)
    table = torch.where(torch.arange(per, device=DEV)[None] < need[:, None], table, 0)
    return {"q": _normal(g, b, h, d), **_cache(g, pages, kv, p, d), "table": table.to(torch.int32).contiguous(),
            "lens": lens.to(torch.int32), "o": torch.zeros(b, h, d, dtype=torch.float16, device=DEV),
            "scale": float(np.float32(d ** -0.5))}


STATES = {"linear": _linear_state, "gate_up": _gate_up_state, "norm": _norm_state, "quantize": _quantize_state,
          "kv_write": _kv_write_state, "attention": _attention_state}


def prepare(case, seed):
    return {"kind": case["kind"], **STATES[case["kind"]](case, _gen(seed))}


# ---------------------------------------------------------------- the library's calls

# The arguments of each kernel, as `tessel_amd.kernel` and `launch` take them.
CALLS = {"linear": ("linear", ("x", "sx", "w", "sw", "y"), ()),
         "gate_up": ("gate_up", ("x", "sx", "wg", "sg", "wu", "su", "y"), ()),
         "norm": ("rmsnorm", ("r", "w", "q", "s"), ("eps",)),
         "add_norm": ("add_rmsnorm", ("x", "r", "w", "q", "s"), ("eps",)),
         "quantize": ("quantize", ("x", "q", "s"), ()),
         "kv_write": ("kv_write", ("qkv", "pos", "slot", "cos", "sin", "kc", "vc", "ks", "vs", "k", "v"), ()),
         "attention": ("decode_attention", ("q", "kc", "vc", "ks", "vs", "table", "lens", "o"), ("scale",))}


def _call(state):
    """The kernel's handle and arguments, which a program keeps with its buffers. torch's own work goes to the
    library's stream from here on, so what reads a kernel's outputs follows it; what made the inputs on another
    stream is waited for, there."""
    import tessel_amd as T

    T.open()
    stream = torch.cuda.ExternalStream(T.lib().tsl_stream())
    stream.wait_stream(torch.cuda.current_stream())
    torch.cuda.set_stream(stream)
    name, arrays, scalars = CALLS["add_norm" if "x" in state and state["kind"] == "norm" else state["kind"]]
    kernel = T.kernel("quant", name, [tuple(state[a].shape) for a in arrays])
    args = [T.Buf(state[a].data_ptr(), state[a].numel() * state[a].element_size()) for a in arrays]
    return T.launch, kernel, args + [T.F32(state[s]) for s in scalars]


# ---------------------------------------------------------------- the plain forms

def _linear(s):
    sums = s["x"].float() @ s["w"].float().t()
    s["y"].copy_(sums * s["sx"][:, None] * s["sw"])


def _gate_up(s):
    x = s["x"].float()
    gate = (x @ s["wg"].float().t()) * s["sx"][:, None] * s["sg"]
    up = (x @ s["wu"].float().t()) * s["sx"][:, None] * s["su"]
    s["y"].copy_(gate / (1 + torch.exp(-gate)) * up)


def _codes8(y):
    """Each row's codes round(127 y / largest), in 64 bits: a quotient next to a border rounds as it is."""
    top = y.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * y / top), 0.0), top.squeeze(-1)


def _norm(s):
    if "x" in s:
        s["r"].add_(s["x"])
    r = s["r"].double()
    codes, top = _codes8(r * s["w"].double())
    s["q"].copy_(codes)
    s["s"].copy_(top / torch.sqrt(r.square().mean(-1) + s["eps"]) / 127)


def _quantize(s):
    codes, top = _codes8(s["x"].double())
    s["q"].copy_(codes)
    s["s"].copy_(top / 127)


def _rotated(x, c, s):
    """Halves (x1, x2) of each head turned to (x1 c - x2 s, x2 c + x1 s), in 16 bits: the second product rounded to
    32 bits, then one multiply-add, as the library rotates everywhere."""
    x1, x2 = x.double().chunk(2, -1)
    c, s = c.double(), s.double()
    a = x1 * c - (x2 * s).float().double()
    b = x2 * c + (x1 * s).float().double()
    return torch.cat([a, b], -1).float().half()


def _codes4(x):
    """Each head's 16 levels between its lowest and highest value: codes, and (lowest, step) in 16 bits."""
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    n = torch.where(hi > lo, torch.round(15 * (x - lo) / (hi - lo)), 0.0).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.cat([lo, ((hi - lo) / 15).float()], -1).half()


def _kv_write(s):
    kv, d = s["k"].shape[1:]
    x = s["qkv"][:, -2 * kv * d:].view(-1, 2, kv, d)
    at = s["pos"].long()
    s["k"].copy_(_rotated(x[:, 0], s["cos"][at][:, None], s["sin"][at][:, None]))
    s["v"].copy_(x[:, 1])
    p = s["kc"].shape[2]
    page, off = (s["slot"].long() // p)[:, None], (s["slot"].long() % p)[:, None]
    g = torch.arange(kv, device=DEV)[None]
    s["kc"][page, g, off], s["ks"][page, g, off] = _codes4(s["k"])
    s["vc"][page, g, off // 16, :, off % 16], s["vs"][page, g, off] = _codes4(s["v"])


def _nibbles(codes, dim):
    return torch.stack([codes & 15, codes >> 4], dim)


def _attention(s):
    b, h, d = s["q"].shape
    kv, p = s["kc"].shape[1:3]
    pages, tokens = s["table"].long(), s["table"].shape[1] * p
    k = _nibbles(s["kc"][pages], -1).flatten(-2)  # [b, pages, kv, p, d]
    v = _nibbles(s["vc"][pages], -2).flatten(-3, -2).transpose(-1, -2).flatten(3, 4)
    ks, vs = s["ks"][pages].float(), s["vs"][pages].float()
    k = (k * ks[..., 1:] + ks[..., :1]).transpose(1, 2).reshape(b, kv, tokens, d)
    v = (v * vs[..., 1:] + vs[..., :1]).transpose(1, 2).reshape(b, kv, tokens, d)
    score = (s["q"].float().view(b, kv, h // kv, d) @ k.transpose(-1, -2).contiguous()) * s["scale"]
    past = torch.arange(tokens, device=DEV) >= s["lens"][:, None, None, None]
    score = score.masked_fill(past, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    s["o"].copy_(((e @ v) / e.sum(-1, keepdim=True)).view(b, h, d))


PLAIN = {"linear": _linear, "gate_up": _gate_up, "norm": _norm, "quantize": _quantize, "kv_write": _kv_write,
         "attention": _attention}


# ---------------------------------------------------------------- the outputs

def _outputs(s):
    """What a pass wrote; codes as the values that they stand for (the cache's in the order it holds them)."""
    if s["kind"] in ("linear", "gate_up"):
        return s["y"]
    if s["kind"] == "attention":
        return s["o"]
    if s["kind"] == "quantize":
        return {"values": s["q"] * s["s"][:, None], "scale": s["s"]}
    if s["kind"] == "norm":
        return {"values": s["q"] * s["s"][:, None], "scale": s["s"], "residual": s["r"]}
    ks, vs = s["ks"].float(), s["vs"].float()
    kc = _nibbles(s["kc"], -1).flatten(-2) * ks[..., 1:] + ks[..., :1]
    vs = vs.unflatten(2, (-1, 16))[:, :, :, None]
    vc = _nibbles(s["vc"], -2).flatten(-3, -2) * vs[..., 1] + vs[..., 0]
    return {"k": s["k"], "v": s["v"], "k_cache": kc.half(), "v_cache": vc.half()}


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        launch, kernel, args = state["call"]
        launch(kernel, args)
    else:
        PLAIN[state["kind"]](state)
    return _outputs(state)


# ---------------------------------------------------------------- 64 bits

def _exact_rows(y):
    """Symmetric 8-bit rows by their definition: the whole number nearest to y / step, an even one on a tie."""
    top = y.abs().max(dim=1, keepdim=True).values
    t = torch.where(top > 0, y * 127 / top, torch.zeros_like(y))
    low = torch.floor(t)
    part = t - low
    up = (part > 0.5) | ((part == 0.5) & (torch.remainder(low, 2) == 1))
    return (low + up.double()) * top / 127, top.squeeze(1) / 127


def _exact_kv(c, s):
    """Rotation in 64 bits, rounded to 16; the cache's values by token, then in its order."""
    kv, d, p = c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].double()[:, c["heads"] * d:]
    k, v = x[:, : kv * d].reshape(-1, kv, d), x[:, kv * d:].reshape(-1, kv, d)
    cs, sn = s["cos"].double()[s["pos"].long()].unsqueeze(1), s["sin"].double()[s["pos"].long()].unsqueeze(1)
    h = d // 2
    k = torch.cat([k[..., :h] * cs - k[..., h:] * sn, k[..., h:] * cs + k[..., :h] * sn], -1).half().double()
    pages = s["kc"].shape[0]

    def held(codes_lo, codes_hi, pair):  # [slots, kv, d] of what the cache held
        both = torch.empty(*codes_lo.shape[:-1], d, device=DEV, dtype=torch.float64)
        both[..., 0::2], both[..., 1::2] = codes_lo.double(), codes_hi.double()
        low, step = (pair[..., i].double().permute(0, 2, 1).reshape(-1, kv, 1) for i in (0, 1))
        return both.permute(0, 2, 1, 3).reshape(-1, kv, d) * step + low

    def stored(t):
        low, high = t.min(-1, keepdim=True).values, t.max(-1, keepdim=True).values
        n = torch.where(high > low, torch.round((t - low) * 15 / (high - low)), torch.zeros_like(t))
        return low + n * ((high - low) / 15).half().double()

    kold = held(s["kc"] % 16, s["kc"] // 16, s["ks"])
    vb = s["vc"].permute(0, 1, 2, 4, 3).reshape(pages, kv, p, h)
    vold = held(vb % 16, vb // 16, s["vs"])
    at = s["slot"].long()
    kold[at], vold[at] = stored(k), stored(v)
    kc = kold.view(pages, p, kv, d).permute(0, 2, 1, 3)
    vc = vold.view(pages, p // 16, 16, kv, d).permute(0, 3, 1, 4, 2)
    return {"k": k, "v": v, "k_cache": kc, "v_cache": vc}


def _exact_attention(c, s):
    kv, d, p = c["kv_heads"], c["dim"], c["page"]
    out = torch.empty(c["seqs"], c["heads"], d, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lens"].tolist()):
        at = s["table"][i, : (n + p - 1) // p].long()
        kb, vb = s["kc"][at].double(), s["vc"][at].transpose(-1, -2).flatten(2, 3).double()
        for g in range(kv):
            def values(bytes_, pair):
                codes = torch.stack([torch.remainder(bytes_, 16), torch.floor(bytes_ / 16)], -1).reshape(-1, d)[:n]
                low, step = pair.double().reshape(-1, 2)[:n].unbind(1)
                return codes * step[:, None] + low[:, None]

            k, v = values(kb[:, g], s["ks"][at][:, g]), values(vb[:, g], s["vs"][at][:, g])
            r = c["heads"] // kv
            w = torch.softmax((s["q"][i, g * r:(g + 1) * r].double() @ k.t().contiguous()) * s["scale"], -1)
            out[i, g * r:(g + 1) * r] = w @ v
    return out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        return (s["x"].double() * s["sx"].double()[:, None]) @ (s["w"].double() * s["sw"].double()[:, None]).t()
    if kind == "gate_up":
        x = s["x"].double() * s["sx"].double()[:, None]
        g = x @ (s["wg"].double() * s["sg"].double()[:, None]).t()
        return torch.nn.functional.silu(g) * (x @ (s["wu"].double() * s["su"].double()[:, None]).t())
    if kind == "quantize":
        values, step = _exact_rows(s["x"].double())
        return {"values": values, "scale": step}
    if kind == "norm":
        # The residual is held in 32 bits: the sum rounds once, and the norm is of what is held.
        r = (s["r"].double() + s["x"].double()).float().double() if case["add"] else s["r"].double()
        y = r * s["w"].double()
        rms = torch.sqrt((r * r).sum(1, keepdim=True) / r.shape[1] + s["eps"])
        values, step = _exact_rows(y)
        return {"values": values / rms, "scale": step / rms.squeeze(1), "residual": r}
    return _exact_kv(case, s) if kind == "kv_write" else _exact_attention(case, s)


# ---------------------------------------------------------------- the work

def work(case):
    c, kind = case, case["kind"]
    if kind == "linear":
        m, n, k = c["rows"], c["n"], c["k"]
        return {"bytes": float(m * k + n * k + 4 * (m + n) + 2 * m * n), "flops": 2.0 * m * n * k}
    if kind == "gate_up":
        m, n, k = c["rows"], c["ffn"], c["dim"]
        return {"bytes": float(m * k + 2 * n * k + 4 * (m + 2 * n) + 2 * m * n), "flops": 4.0 * m * n * k}
    if kind == "norm":
        m, k = c["rows"], c["cols"]
        return {"bytes": float(m * k * (11 if c["add"] else 5) + 2 * k + 4 * m), "flops": 6.0 * m * k}
    if kind == "quantize":
        m, k = c["rows"], c["cols"]
        return {"bytes": float(3 * m * k + 4 * m), "flops": 3.0 * m * k}
    kv, d = c["kv_heads"], c["dim"]
    if kind == "kv_write":
        t = c["tokens"]
        # K and V of the projection in, both out in 16 bits and in 4 with their pairs; cos, sin, position, slot.
        return {"bytes": t * (4.0 * kv * d + 4 * kv * d + kv * (d + 8) + 4 * d + 8), "flops": 12.0 * t * kv * d}
    tokens = c["seqs"] * (c["lo"] + c["hi"]) / 2.0
    return {"bytes": tokens * kv * (d + 8.0) + 4.0 * c["seqs"] * c["heads"] * d + 4.0 * tokens / c["page"],
            "flops": 4.0 * tokens * c["heads"] * d}
