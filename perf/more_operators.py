"""4-bit weights with a scale per group, rows of 8-bit digits with a scale per block, and the
products of both, as cases that can be timed and checked.

W4, a matrix [d, n] in groups of 128 numbers of a row (the last one shorter): a scale s (bf16) and
a code c in -8..7 per number, which stands for s c.  A group of numbers w is written as
    s = bf16(max |w| / 7) (0 where that is below 2^-126),  c = clamp(rint(w (1 / s)), -7, 7)
Memory: panels of 16 rows (d and n rounded up to 16 and 128, zeros there); a panel has its codes
[groups, 4 pieces, 16 rows, 16 bytes], byte b of piece j with number 32 j + b of the group in the
low half and number 32 j + 16 + b in the high half (two's complement), then its scales
[4, groups, 4] (row 4 i + r of the panel at [i, group, r]).

Q8 and Q24, rows x [tokens, n] in blocks of 128 numbers (the last one shorter): a scale s (fp32)
and a whole number q per number, which stands for s q.
    Q8   s = max |x| / 127 (0 where that is below 2^-120),  q = clamp(rint(x (1 / s)), -127, 127)
    Q24  s the least power of two >= 2^-120 with max |x| < 127 2^16 s,  q = rint(x / s)
q is one digit, or three: d0 + 256 d1 + 65536 d2 with digits in -128..127.  Memory: panels of 16
tokens (tokens rounded up); a panel has its digits [blocks, digits, 2 halves, 4 pieces, 16 tokens,
16 bytes], byte b of half h and piece j for number 32 j + 16 h + b of the block, then its scales
[blocks, 16 tokens].
"""
import ctypes
import math

import torch

own = False

GROUP = 128
EPS = 1e-5


def listed():
    return [
        # the small model's output projection of one token, with its residual: latency
        dict(name="gemv_stories", kind="gemv", mode="residual", rows=288, n=288),
        # one token's output projection at the 8B shape
        dict(name="gemv_8b_wo", kind="gemv", mode="residual", rows=4096, n=4096),
        # one token's norm, gate and up projections and SwiGLU at the 70B shape
        dict(name="gemv_70b_gate_up", kind="gemv", mode="swiglu", rows=28672, n=8192, norm="bf16"),
        # one token's norm and LM head of a 128k vocabulary
        dict(name="gemv_8b_lm_head", kind="gemv", mode="normed", rows=128256, n=4096, norm="f32"),
        # one token's residual, norm and digits
        dict(name="norm_step", kind="norm", tokens=1, n=4096, digits=3, norm="bf16"),
        # a 2k prompt's
        dict(name="norm_prompt_2k", kind="norm", tokens=2048, n=4096, digits=1, norm="bf16"),
        # a paragraph of odd length and width
        dict(name="norm_odd", kind="norm", tokens=131, n=2080, digits=3, norm="f32"),
        # five drafted tokens through the 8B shape's down projection
        dict(name="gemm_draft", kind="gemm", mode="residual", tokens=5, rows=4096, n=14336, digits=3),
        # a short question through the query, key and value projections
        dict(name="gemm_qkv_41", kind="gemm", mode="qkv", tokens=41, heads=32, kv_heads=8, head=128,
             n=4096, digits=3, pos=900),
        # a follow-up turn of odd length, an odd matrix
        dict(name="gemm_turn_odd", kind="gemm", mode="residual", tokens=301, rows=5003, n=2080, digits=1),
        # a 2k prompt through gate and up, 8-bit rows
        dict(name="gemm_prompt_2k", kind="gemm", mode="swiglu", tokens=2048, rows=14336, n=4096, digits=1),
        # a 1k prompt through the output projection, rows as exact as fp32
        dict(name="gemm_prompt_1k", kind="gemm", mode="residual", tokens=1024, rows=4096, n=4096, digits=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gemv", "gemv", "gemv", "norm", "gemm", "gemm", "gemm"])
    n = rng.choice([288, 2048, 4096, 8192, 14336, _log(rng, 96, 16384)])
    if kind == "norm":
        return dict(kind=kind, tokens=_log(rng, 1, 2048), n=n, digits=rng.choice([1, 3]),
                    norm=rng.choice(["f32", "bf16"]))
    c = dict(kind=kind, mode=rng.choice(["residual", "swiglu", "qkv"] + ["normed"] * (kind == "gemv")),
             n=n)
    if c["mode"] == "qkv":
        heads, kv_heads, head = rng.choice([(32, 8, 128), (64, 8, 128), (6, 6, 48), (32, 8, 64),
                                            (18, 6, 96), (4, 1, 80), (14, 2, 64)])
        c.update(heads=heads, kv_heads=kv_heads, head=head, pos=_log(rng, 1, 4000))
    else:
        c["rows"] = _log(rng, 200, 32768)
    if kind == "gemv":
        return c if c["mode"] == "residual" else dict(c, norm=rng.choice(["f32", "bf16"]))
    c.update(tokens=_log(rng, 1, 2048), digits=rng.choice([1, 3]))
    while work(c)["flops"] > 4.8e11:  # (the listed ones' most)
        c["tokens"] = c["tokens"] * 2 // 3
    return c


# ---- inputs -----------------------------------------------------------------------------------
def _up(a, b):
    return (a + b - 1) // b * b


def _shapes(c):
    """Rows of the case's matrices, all of n numbers a row."""
    if c["mode"] == "swiglu":
        return [c["rows"], c["rows"]]
    if c["mode"] == "qkv":
        return [c["heads"] * c["head"], c["kv_heads"] * c["head"], c["kv_heads"] * c["head"]]
    return [c["rows"]]


def _w4(w):
    """A matrix w [d, n] (fp32) as W4 bytes."""
    d, n = w.shape
    dp, np_ = _up(d, 16), _up(n, GROUP)
    x = torch.zeros((dp, np_), device=w.device)
    x[:d, :n] = w
    x = x.view(dp, np_ // GROUP, GROUP)
    top = x.abs().amax(-1)
    # (quotients in 64 bits, rounded once: the same on every device)
    s = (top.double() / 7).float().bfloat16()
    s = torch.where(s.float() < 2.0 ** -126, torch.zeros_like(s), s)
    inv = torch.where(s > 0, (1 / s.double()).float(), 0.0)
    c = (x * inv[..., None]).round().clamp(-7, 7).to(torch.int16) & 15
    # [panel, row, group, piece, half, byte]
    c = c.view(dp // 16, 16, np_ // GROUP, 4, 2, 16)
    codes = (c[..., 0, :] | (c[..., 1, :] << 4)).to(torch.uint8).permute(0, 2, 3, 1, 4)
    scales = s.view(dp // 16, 4, 4, np_ // GROUP).transpose(2, 3).contiguous().view(torch.uint8)
    return torch.cat([codes.reshape(dp // 16, -1), scales.reshape(dp // 16, -1)], 1).view(-1)


def _digits(q, digits):
    """Whole numbers q (int32) as [digits, ...] int8."""
    out = []
    for _ in range(digits):
        low = ((q + 128) & 255) - 128
        out.append(low.to(torch.int8))
        q = (q - low) >> 8
    return torch.stack(out)


def _quantised(x, digits):
    """Rows x [tokens, n] (fp32): scales [tokens, blocks] and whole numbers [tokens, blocks, 128]."""
    t, n = x.shape
    y = torch.zeros((t, _up(n, GROUP)), device=x.device)
    y[:, :n] = x
    y = y.view(t, -1, GROUP)
    top = y.abs().amax(-1)
    if digits == 1:
        s = (top.double() / 127).float()
        s = torch.where(s < 2.0 ** -120, 0.0, s)
        inv = torch.where(s > 0, (1 / s.double()).float(), 0.0)
        return s, (y * inv[..., None]).round().clamp(-127, 127).to(torch.int32)
    # the exponent, one more where the fraction is at least 127 / 64
    e = ((top.view(torch.int32) + 0x20000) >> 23) - 127 - 22
    s = ((e.clamp(min=-120) + 127) << 23).view(torch.float32)
    return s, (y / s[..., None]).round().to(torch.int32)


def _rows(s, q, digits):
    """Scales and whole numbers of _quantised as Q8 or Q24 bytes."""
    t, blocks = s.shape
    tp = _up(t, 16)
    d = torch.zeros((digits, tp, blocks, GROUP), dtype=torch.int8, device=s.device)
    d[:, :t] = _digits(q, digits)
    # [digit, panel, token, block, piece, half, byte] -> [panel, block, digit, half, piece, token, byte]
    d = d.view(digits, tp // 16, 16, blocks, 4, 2, 16).permute(1, 3, 0, 5, 4, 2, 6)
    sp = torch.zeros((tp, blocks), device=s.device)
    sp[:t] = s
    sp = sp.view(tp // 16, 16, blocks).transpose(1, 2).contiguous().view(torch.uint8)
    return torch.cat([d.reshape(tp // 16, -1).view(torch.uint8), sp.reshape(tp // 16, -1)], 1).view(-1)


def _stream(g, tokens, n):
    """Rows as a residual stream has them: channels of their own size, a few of them far larger."""
    x = torch.empty((tokens, n), device="cuda").normal_(generator=g)
    size = torch.exp(0.5 * torch.empty(n, device="cuda").normal_(generator=g))
    size[torch.randint(n, (3,), device="cuda", generator=g)] *= 30
    return x * size


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    n, tokens = c["n"], c.get("tokens", 1)
    s = {"c": c}
    if c.get("norm"):
        w = 1 + 0.2 * torch.empty(n, device="cuda").normal_(generator=g)
        s["norm"] = w.bfloat16() if c["norm"] == "bf16" else w
    x = _stream(g, tokens, n)
    if c["kind"] == "norm":
        s["x"], s["r"] = x, 0.3 * _stream(g, tokens, n)
        return s
    s["w"] = []
    for d in _shapes(c):
        w = torch.empty((d, n), device="cuda").normal_(generator=g)
        s["w"].append(_w4(w.mul_(0.5 / math.sqrt(n))))
        del w
    if c["kind"] == "gemm":
        s["x"] = _rows(*_quantised(x, c["digits"]), c["digits"])
    else:
        s["x"] = x[0].contiguous()
    if c["mode"] == "residual":
        s["r"] = torch.empty((tokens, c["rows"]), device="cuda").normal_(generator=g)
    if c["mode"] == "qkv":
        s["step"] = torch.tensor([0, c["pos"]], dtype=torch.int32, device="cuda")
        at = torch.arange(c["pos"] + tokens, device="cuda").double()[:, None]
        i = torch.arange(0, c["head"], 2, device="cuda").double()
        angle = at * 500000.0 ** (-i / c["head"])
        s["table"] = torch.stack([torch.cos(angle), torch.sin(angle)], -1).float().contiguous()
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _matrix(bytes_, d, n):
    """The fp32 numbers [d, n] of W4 bytes."""
    groups = _up(n, GROUP) // GROUP
    p = bytes_.view(-1, groups * 1056)
    codes = p[:, :groups * 1024].reshape(-1, groups, 4, 16, 16)
    scales = p[:, groups * 1024:].contiguous().view(torch.bfloat16).view(-1, 4, groups, 4)
    c = torch.stack([codes & 15, codes >> 4], -2).to(torch.int8)  # [panel, group, piece, row, half, byte]
    c = (c ^ 8) - 8
    c = c.permute(0, 3, 1, 2, 4, 5).reshape(-1, groups, GROUP)
    s = scales.transpose(2, 3).reshape(-1, groups).float()
    return (c.float() * s[..., None]).reshape(c.shape[0], -1)[:d, :n]


def _values(bytes_, tokens, n, digits):
    """The fp32 numbers [tokens, n] of Q8 or Q24 bytes."""
    blocks = _up(n, GROUP) // GROUP
    p = bytes_.view(-1, blocks * (2048 * digits + 64))
    d = p[:, :blocks * 2048 * digits].reshape(-1, blocks, digits, 2, 4, 16, 16).view(torch.int8)
    s = p[:, blocks * 2048 * digits:].contiguous().view(torch.float32).view(-1, blocks, 16)
    q = d[:, :, 0].to(torch.int32)
    for i in range(1, digits):
        q = q + (d[:, :, i].to(torch.int32) << (8 * i))
    q = q.permute(0, 4, 1, 3, 2, 5).reshape(-1, blocks, GROUP)  # [panel, block, half, piece, token, byte]
    v = q.float() * s.transpose(1, 2).reshape(-1, blocks)[..., None]
    return v.reshape(v.shape[0], -1)[:tokens, :n]


def _normed(h, w):
    """w (h / sqrt(mean(h^2) + eps)): the mean in 64 bits, each product rounded to 32."""
    r = (1 / torch.sqrt((h.double() ** 2).mean(-1, keepdim=True) + float(torch.tensor(EPS)))).float()
    return w.float() * (r * h)


def _rotated(y, table, head):
    """Rows y [tokens, heads * head], pairs rotated by table [tokens, head / 2, 2]."""
    p = y.view(y.shape[0], -1, head // 2, 2)
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    return torch.stack([p[..., 0] * c - p[..., 1] * s, p[..., 0] * s + p[..., 1] * c], -1).view(y.shape)


def _run_plain(state):
    c = state["c"]
    n, tokens = c["n"], c.get("tokens", 1)
    if c["kind"] == "norm":
        h = state["x"] + state["r"]
        s, q = _quantised(_normed(h, state["norm"]), c["digits"])
        v = (q.float() * s[..., None]).view(tokens, -1)[:, :n].contiguous()
        return {"sum": h, "rows": v}
    if c["kind"] == "gemm":
        x = _values(state["x"], tokens, n, c["digits"])
    else:
        x = state["x"][None]
        if "norm" in state:
            x = _normed(x, state["norm"])
    y = [torch.matmul(x, _matrix(w, d, n).t()) for w, d in zip(state["w"], _shapes(c))]
    if c["mode"] == "residual":
        return {"y": state["r"] + y[0]}
    if c["mode"] == "swiglu":
        return {"y": y[0] * (1 / (1 + torch.exp(-y[0]))) * y[1]}
    if c["mode"] == "qkv":
        table = state["table"][c["pos"]:]
        return {"q": _rotated(y[0], table, c["head"]), "k": _rotated(y[1], table, c["head"]), "v": y[2]}
    return {"y": y[0]}


_RUNTIME = None


def _kept(state):
    """What a program keeps beside its weights: the runtime, pointers and its buffers."""
    global _RUNTIME
    import ammon_amd
    from ammon_amd import _abi
    if _RUNTIME is None:
        _RUNTIME = ammon_amd.Runtime(0)
    c, lib, rt = state["c"], _abi.lib, _RUNTIME
    tokens, n = c.get("tokens", 1), c["n"]
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    empty = lambda *shape, **kw: torch.empty(shape, device="cuda", **kw)  # noqa: E731
    kept = {"h": rt.handle, "call": _abi.call, "w4": _abi.W4, "x": p(state["x"])}
    if c.get("digits"):
        kept["dtype"] = _abi.Q8 if c["digits"] == 1 else _abi.Q24
    if c.get("norm"):
        kept["norm"] = (p(state["norm"]), _abi.BF16 if c["norm"] == "bf16" else _abi.F32)
    if "r" in state:
        kept["r"] = p(state["r"])
    if c["kind"] == "norm":
        out = {"sum": empty(tokens, n), "rows": empty(tokens, n)}
        kept["q"] = empty(int(lib.ammon_q8_bytes(kept["dtype"], tokens, n)), dtype=torch.uint8)
        kept["q_p"] = p(kept["q"])
    elif c["mode"] == "qkv":
        kept["step"], kept["table"] = p(state["step"]), p(state["table"])
        out = {x: empty(tokens, d) for x, d in zip("qkv", _shapes(c))}
    else:
        out = {"y": empty(tokens, c["rows"])}
    kept["out"], kept["out_p"] = out, [p(t) for t in out.values()]
    if c["kind"] != "norm":
        kept["w"] = [p(w) for w in state["w"]]
    if c["kind"] == "gemm":
        size = int(lib.ammon_prefill_gemm_workspace_bytes(sum(_shapes(c)), tokens))
        kept["ws"] = empty(size // 4)
        kept["ws_p"] = (p(kept["ws"]), size)
    return kept


def _run_own(state):
    c = state["c"]
    if "kept" not in state:
        state["kept"] = _kept(state)
    k = state["kept"]
    h, call, n, tokens = k["h"], k["call"], c["n"], c.get("tokens", 1)
    if c["kind"] == "norm":
        call("ammon_rmsnorm_q8", h, None, k["x"], k["r"], k["out_p"][0], *k["norm"], EPS, tokens, n,
             k["q_p"], k["dtype"])
        call("ammon_q8_load", h, None, k["q_p"], k["dtype"], tokens, n, k["out_p"][1])
        return k["out"]
    if c["mode"] == "qkv":
        shape = (n, c["heads"], c["kv_heads"], c["head"], *k["out_p"], c["pos"] + tokens, k["step"],
                 k["table"])
    if c["kind"] == "gemv":
        norm = (*k["norm"], EPS) if "norm" in k else (None, 0, 0.0)
        if c["mode"] == "residual":
            call("ammon_gemv", h, None, *k["w"], k["w4"], c["rows"], n, k["x"], *k["out_p"], k["r"])
        elif c["mode"] == "normed":
            call("ammon_gemv_rmsnorm", h, None, k["x"], *norm, *k["w"], k["w4"], c["rows"], n,
                 *k["out_p"])
        elif c["mode"] == "swiglu":
            call("ammon_gate_up_swiglu", h, None, k["x"], *norm, *k["w"], k["w4"], n, c["rows"],
                 *k["out_p"])
        else:
            call("ammon_qkv_rope", h, None, k["x"], *norm, *k["w"], k["w4"], *shape)
    elif c["mode"] == "residual":
        call("ammon_prefill_gemm_w4", h, None, *k["w"], c["rows"], n, k["x"], k["dtype"], tokens,
             *k["out_p"], k["r"], *k["ws_p"])
    elif c["mode"] == "swiglu":
        call("ammon_prefill_gate_up_swiglu_w4", h, None, k["x"], k["dtype"], tokens, *k["w"], n,
             c["rows"], *k["out_p"])
    else:
        call("ammon_prefill_qkv_rope_w4", h, None, k["x"], k["dtype"], tokens, *k["w"], *shape,
             *k["ws_p"])
    return k["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c = case
    n, t = c["n"], c.get("tokens", 1)
    norm = n * (2 if c.get("norm") == "bf16" else 4) if c.get("norm") else 0
    rows = t * (n * c.get("digits", 0) + 4 * _up(n, GROUP) // GROUP)
    if c["kind"] == "norm":  # x and r in, their sum and the rows out, the rows in, their numbers out
        return {"bytes": 16 * t * n + norm + 2 * rows, "flops": 6 * t * n}
    d = sum(_shapes(c))
    weights = sum(d_ * n // 2 + 2 * d_ * (_up(n, GROUP) // GROUP) for d_ in _shapes(c))
    out = 4 * t * (c["rows"] * (2 if c["mode"] == "residual" else 1) if "rows" in c else d)
    x = rows if c["kind"] == "gemm" else 4 * n
    return {"bytes": weights + x + norm + out, "flops": 2 * d * n * t}


# ---- the same in 64 bits ---------------------------------------------------------------------------
def _exact_matrix(bytes_, d, n):
    """The numbers of W4 bytes in float64, one position of a group at a time."""
    groups = _up(n, GROUP) // GROUP
    panels = _up(d, 16) // 16
    p = bytes_.view(panels, 1056 * groups)
    codes = p[:, :1024 * groups].view(panels, groups, 64, 16)
    scales = p[:, 1024 * groups:].contiguous().view(torch.bfloat16).view(panels, 4 * groups, 4).double()
    out = torch.empty((panels, 16, groups * GROUP), dtype=torch.float64, device=bytes_.device)
    for r in range(16):
        s = scales[:, r // 4 * groups:(r // 4 + 1) * groups, r % 4]
        for j in range(4):
            b = codes[:, :, 16 * j + r].double()
            high = torch.floor(b / 16)
            for h, v in enumerate((b - 16 * high, high)):
                v = torch.where(v > 7.5, v - 16, v) * s[..., None]
                out[:, r].view(panels, groups, GROUP)[:, :, 32 * j + 16 * h:32 * j + 16 * h + 16] = v
    return out.view(-1, groups * GROUP)[:d, :n]


def _exact_values(bytes_, tokens, n, digits):
    blocks = _up(n, GROUP) // GROUP
    panels = _up(tokens, 16) // 16
    p = bytes_.view(panels, -1)
    d = p[:, :2048 * digits * blocks].view(panels, blocks, digits, 8, 16, 16).to(torch.float64)
    d = torch.where(d > 127, d - 256, d)
    s = p[:, 2048 * digits * blocks:].contiguous().view(torch.float32).view(panels, blocks, 16).double()
    out = torch.empty((panels, 16, blocks, GROUP), dtype=torch.float64, device=bytes_.device)
    for i in range(8):
        q = sum(d[:, :, k, i] * 256.0 ** k for k in range(digits))  # [panel, block, token, byte]
        at = 32 * (i % 4) + 16 * (i // 4)
        out[:, :, :, at:at + 16] = (q * s[..., None]).transpose(1, 2)
    return out.view(16 * panels, -1)[:tokens, :n]


def _exact_normed(h, w, rounded):
    """The norm of rows h in float64; rounded: with the definition's roundings to fp32."""
    f = (lambda t: t.float().double()) if rounded else (lambda t: t)
    eps = torch.tensor(EPS).double().item()
    r = f((torch.mean(h * h, -1, keepdim=True) + eps) ** -0.5)
    return f(w.double() * f(r * h))


def _exact_norm_rows(x, r, w, digits):
    f32 = lambda t: t.float().double()  # noqa: E731
    h = f32(x.double() + r.double())
    v = _exact_normed(h, w, True)
    out = torch.empty_like(v)
    for at in range(0, v.shape[1], GROUP):
        y = v[:, at:at + GROUP]
        top = y.abs().max(-1, keepdim=True).values
        if digits == 1:
            s = f32(top / 127)
            s = torch.where(s < 2.0 ** -120, torch.zeros_like(s), s)
            inv = torch.where(s > 0, f32(1 / s), torch.zeros_like(s))
            q = torch.clamp(torch.round(f32(y * inv)), -127, 127)
        else:
            k = torch.frexp(top / (127 * 65536)).exponent  # below 2^k, at least 2^(k - 1)
            k = torch.clamp(torch.where(top > 0, k, -120), min=-120)
            s = ((k.long() + 1023) << 52).view(torch.float64)
            q = torch.round(y / s)
        out[:, at:at + GROUP] = f32(s * q)
    return {"sum": h, "rows": out}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    n, tokens = c["n"], c.get("tokens", 1)
    if c["kind"] == "norm":
        return _exact_norm_rows(s["x"], s["r"], s["norm"], c["digits"])
    if c["kind"] == "gemm":
        x = _exact_values(s["x"], tokens, n, c["digits"])
    else:
        x = s["x"].double()[None]
        if "norm" in s:
            x = _exact_normed(x, s["norm"], False)
    y = [x @ _exact_matrix(w, d, n).t() for w, d in zip(s["w"], _shapes(c))]
    if c["mode"] == "residual":
        return {"y": y[0] + s["r"].double()}
    if c["mode"] == "swiglu":
        return {"y": y[0] * torch.sigmoid(y[0]) * y[1]}
    if c["mode"] != "qkv":
        return {"y": y[0]}
    table = s["table"].double()[c["pos"]:]
    turn = torch.complex(table[..., 0], table[..., 1])[:, None]
    out = {"v": y[2]}
    for name, rows in zip("qk", y):
        z = torch.view_as_complex(rows.reshape(tokens, -1, c["head"] // 2, 2).contiguous()) * turn
        out[name] = torch.view_as_real(z).reshape(tokens, -1)
    return {x_: out[x_] for x_ in "qkv"}
