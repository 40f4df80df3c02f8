"""The 4-bit KV cache: writing it, reading it back, and attention over it, as cases that can be
timed and checked.

A KV4 cache of one layer holds, for every kv head and position, one row of ``head`` numbers in
groups of 32 (the last one shorter where head is no multiple of 32).  A group has a scale s and a
bias b, both fp16, and a code c in 0..15 per number; it stands for fp16(s (16 + c) + b).  Writing
a group of fp32 numbers x (every step rounds to fp32 unless it says fp16):
    x = min(max(x, -16384), 16384)
    s = fp16((max x - min x) / 15),  b = fp16(min x - 16 s)
    c = clamp(rint((x - b) (1 / s) - 16), 0, 15), 0 where s = 0
and a group with a number that is not finite has s = b = NaN.

Memory of one cache: the codes [kv_heads, seq, 4, groups] as 32-bit words -- word (p, j) has
numbers 32 j + 8 p .. + 7, number + e in bits 4 n .. 4 n + 3 with n = e / 2 for even e and
4 + e / 2 for odd e -- then s and b (low and high half of a word) as [kv_heads, seq, groups].
"""
import ctypes
import math

import torch

own = False


def listed():
    return [
        # one token's key and value rows, as a decode step writes them: latency
        dict(name="store_step", kind="store", kv_heads=8, head=128, seq=8192, start=8150, tokens=1),
        # a whole 2k prompt's rows of one layer
        dict(name="store_prompt_2k", kind="store", kv_heads=8, head=128, seq=8192, start=0, tokens=2048),
        # a paragraph of odd length into a cache whose heads are narrower
        dict(name="store_odd", kind="store", kv_heads=6, head=96, seq=4096, start=77, tokens=131),
        # a full 32k layer read back as bf16, to be moved to a cache of that type
        dict(name="load_layer_32k", kind="load", kv_heads=8, head=128, seq=32768, start=0,
             tokens=32768, out="bf16"),
        # decode attention of the small model's heads: one short story so far
        dict(name="attn_stories", kind="attn", heads=6, kv_heads=6, head=48, seq=256, pos=200),
        # ... of the 8B heads at the end of an 8k context
        dict(name="attn_8b_ctx8k", kind="attn", heads=32, kv_heads=8, head=128, seq=8192, pos=8150),
        # ... of heads of 64 at the last position of a 128k cache
        dict(name="attn_h64_ctx128k", kind="attn", heads=32, kv_heads=8, head=64, seq=131072,
             pos=131071),
        # the 70B-shaped layer's decode step over a full 32k cache: the new row is stored, then
        # attended to with the others
        dict(name="append_70b_ctx32k", kind="append", heads=64, kv_heads=8, head=128, seq=32768,
             pos=32760),
        # ... and the 8B heads' in the middle of an 8k cache
        dict(name="append_8b_ctx4k", kind="append", heads=32, kv_heads=8, head=128, seq=8192,
             pos=4000),
        # prompt attention of one 8B layer: a whole 2k prompt
        dict(name="prefill_attn_2k", kind="prefill", heads=32, kv_heads=8, head=128, seq=8192,
             start=0, tokens=2048),
        # a follow-up turn of odd length late in a long chat
        dict(name="prefill_attn_turn", kind="prefill", heads=32, kv_heads=8, head=128, seq=8192,
             start=7001, tokens=301),
        # a few words after a long text, three query heads per kv head of 96
        dict(name="prefill_attn_short", kind="prefill", heads=18, kv_heads=6, head=96, seq=4096,
             start=4000, tokens=19),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, head = rng.choice([(32, 8, 128), (64, 8, 128), (16, 16, 128), (24, 12, 128),
                                        (32, 8, 64), (18, 6, 96), (8, 8, 48), (4, 1, 80),
                                        (12, 2, 112), (5, 5, 32), (14, 2, 64)])
    kind = rng.choice(["store", "load", "attn", "attn", "append", "append", "prefill", "prefill"])
    if kind in ("store", "load"):
        tokens = _log(rng, 1, 2048)
        c = dict(kind=kind, kv_heads=kv_heads, head=head, seq=8192,
                 start=rng.choice([0, _log(rng, 1, 6000)]), tokens=tokens)
        return dict(c, out=rng.choice(["f32", "bf16"])) if kind == "load" else c
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, head=head)
    if kind == "prefill":
        c = dict(c, seq=8192, start=rng.choice([0, 0, _log(rng, 1, 6000)]), tokens=_log(rng, 2, 2000))
        while work(c)["flops"] > 34e9:  # (the listed ones' most)
            c["tokens"] = c["tokens"] * 2 // 3
        return c
    seq = rng.choice([512, 8192, 32768])
    return dict(c, seq=seq, pos=_log(rng, 4, seq - 1))


# ---- inputs -----------------------------------------------------------------------------------
def _groups(head):
    return (head + 31) // 32


def _codes_view(cache, c):
    """The cache's words: codes [kv_heads, seq, 4, groups] and scale | bias [kv_heads, seq, groups]."""
    n, rows = _groups(c["head"]), c["kv_heads"] * c["seq"]
    w = cache.view(torch.int32)
    return (w[:rows * 4 * n].view(c["kv_heads"], c["seq"], 4, n),
            w[rows * 4 * n:].view(c["kv_heads"], c["seq"], n))


def _quantise(x):
    """Rows x [..., head] (fp32) as words: codes [..., 4, groups] and scale | bias [..., groups]."""
    head, n = x.shape[-1], _groups(x.shape[-1])
    x = x.clamp(-16384.0, 16384.0)
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], 32 * n - head)], -1)
    x = x.view(*x.shape[:-1], n, 32)
    real = (torch.arange(32 * n, device=x.device) < head).view(n, 32)
    lo = torch.where(real, x, math.inf).amin(-1)
    hi = torch.where(real, x, -math.inf).amax(-1)
    # (quotients in 64 bits, rounded once: the same on every device)
    s = ((hi - lo).double() / 15).float().half()
    b = (lo - s.float() * 16).half()
    inv = torch.where(s > 0, (1 / s.double()).float(), 0.0)
    c = ((x - b.float()[..., None]) * inv[..., None] - 16).round().clamp(0, 15)
    bad = ~torch.isfinite(lo + hi)
    c = torch.where(real & ~bad[..., None], c, 0.0).to(torch.int32)
    s, b = (torch.where(bad, math.nan, t).half() for t in (s, b))
    # [group, piece, even / odd pairs]: even numbers in the low half of a word, odd in the high
    c = c.view(*c.shape[:-1], 4, 4, 2).transpose(-1, -2).reshape(*c.shape[:-1], 4, 8)
    words = (c << torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)
    sb = torch.stack([s, b], -1).view(torch.int32).squeeze(-1)
    return words.transpose(-1, -2).contiguous(), sb.contiguous()


def _rows(c, seed):
    """Keys and values [2, tokens or seq, kv_heads, head] in fp32: keys have channels of their own
    size and mean, as rotated keys do."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    n = c["tokens"] if c["kind"] == "store" else c["pos"] + 1 if "pos" in c else c["start"] + c["tokens"]
    x = torch.empty((2, n, c["kv_heads"], c["head"]), device="cuda").normal_(generator=g)
    size = torch.empty((c["kv_heads"], c["head"]), device="cuda").normal_(generator=g)
    mean = torch.empty((c["kv_heads"], c["head"]), device="cuda").normal_(generator=g)
    x[0].mul_(0.5 + size.abs()).add_(mean)
    return x, g


def prepare(case, seed):
    c = case
    n = _groups(c["head"])
    x, g = _rows(c, seed)
    # rows that nothing has written hold whatever was in memory: here NaN
    caches = torch.full((2, 20 * n * c["kv_heads"] * c["seq"]), 255, dtype=torch.uint8, device="cuda")
    s = {"c": c, "k": caches[0], "v": caches[1]}
    first = c.get("pos", c.get("start"))
    if c["kind"] in ("store", "append"):
        s["new"] = x[:, -1] if c["kind"] == "append" else x
        s["new"] = s["new"].contiguous()
    if c["kind"] != "store":
        # positions before the call's own row
        past = first if c["kind"] == "append" else x.shape[1]
        for cache, rows in zip(caches, x):
            words, sb = _codes_view(cache, c)
            w, b = _quantise(rows[:past].transpose(0, 1).contiguous())
            words[:, :past], sb[:, :past] = w, b
    s["step"] = torch.tensor([0, first], dtype=torch.int32, device="cuda")
    tokens = c["tokens"] if c["kind"] == "prefill" else 1
    if "heads" in c:
        s["q"] = torch.empty((tokens, c["heads"], c["head"]), device="cuda").normal_(generator=g)
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _values(words, sb, head):
    """The fp32 numbers [..., head] that words [..., 4, groups] and sb [..., groups] stand for."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=words.device)
    c = (words[..., None] >> shift) & 15  # [..., 4, groups, 8]
    p = sb.contiguous().view(torch.float16).view(*sb.shape, 2).float()
    s, b = p[..., 0], p[..., 1]
    v = s[..., None, :, None] * (c + 16).float() + b[..., None, :, None]
    v = v.half().float().transpose(-2, -3)  # [..., groups, 4, 8]
    return v.reshape(*v.shape[:-3], -1)[..., :head]


def _read(cache, c, first, last):
    words, sb = _codes_view(cache, c)
    return _values(words[:, first:last], sb[:, first:last], c["head"])


def _attend(q, k, v, first):
    """q [n, heads, head] at positions first.. over k, v [kv_heads, first + n, head]."""
    n, heads, head = q.shape
    g = heads // k.shape[0]
    rows = q.transpose(0, 1).reshape(k.shape[0], g * n, head)
    s = torch.matmul(rows, k.transpose(1, 2).contiguous()) / math.sqrt(head)
    if n > 1:
        at = torch.arange(n, device=q.device).repeat(g) + first
        s.masked_fill_(torch.arange(k.shape[1], device=q.device)[None, :] > at[:, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    return o.reshape(heads, n, head).transpose(0, 1).contiguous()


def _run_plain(state):
    c = state["c"]
    first = c.get("pos", c.get("start"))
    last = first + c.get("tokens", 1)
    if c["kind"] in ("store", "append"):
        rows = state["new"].view(2, last - first, c["kv_heads"], c["head"]).transpose(1, 2)
        new_words, new_sb = _quantise(rows.contiguous())
        (kw, ks), (vw, vs) = _codes_view(state["k"], c), _codes_view(state["v"], c)
        kw[:, first:last], ks[:, first:last] = new_words[0], new_sb[0]
        vw[:, first:last], vs[:, first:last] = new_words[1], new_sb[1]
        k, v = (_read(state[x], c, first, last) for x in ("k", "v"))
        if c["kind"] == "store":
            return {"k": k, "v": v}
    if c["kind"] == "load":
        to = torch.bfloat16 if c["out"] == "bf16" else torch.float32
        return {x: _read(state[x], c, first, last).to(to) for x in ("k", "v")}
    out = _attend(state["q"], _read(state["k"], c, 0, last), _read(state["v"], c, 0, last), first)
    return {"out": out, "k": k, "v": v} if c["kind"] == "append" else {"out": out}


_RUNTIME = None


def _kept(state):
    """What a program keeps beside its caches: the runtime, the split it took and its buffers."""
    global _RUNTIME
    import ammon_amd
    from ammon_amd import _abi
    if _RUNTIME is None:
        _RUNTIME = ammon_amd.Runtime(0)
    c, lib, rt = state["c"], _abi.lib, _RUNTIME
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    empty = lambda *shape, **kw: torch.empty(shape, device="cuda", **kw)  # noqa: E731
    kept = {"h": rt.handle, "call": _abi.call, "kv4": _abi.KV4, "k": p(state["k"]), "v": p(state["v"]),
            "step": p(state["step"])}
    if c["kind"] in ("store", "load", "append"):
        to = torch.bfloat16 if c.get("out") == "bf16" else torch.float32
        kept["to"] = _abi.BF16 if c.get("out") == "bf16" else _abi.F32
        kept["rows"] = [empty(c["kv_heads"], c.get("tokens", 1), c["head"], dtype=to) for _ in "kv"]
        kept["rows_p"] = [p(t) for t in kept["rows"]]
    if c["kind"] in ("store", "append"):
        kept["new_p"] = [p(t) for t in state["new"]]
    if c["kind"] in ("attn", "append"):
        kept["split"] = int(lib.ammon_attention_default_split_for(
            rt.handle, c["heads"], c["kv_heads"], c["head"], _abi.KV4, c["seq"]))
        kept["bytes"] = int(lib.ammon_attention_scratch_bytes(c["heads"], c["head"], c["seq"],
                                                              kept["split"]))
    if c["kind"] == "prefill":
        ctx, split = c["start"] + c["tokens"], 16
        while split < 1024 and c["kv_heads"] * c["tokens"] * int(
                lib.ammon_attention_splits(ctx, split)) > 2 * rt.info.compute_units:
            split *= 2
        kept["split"] = split
        kept["bytes"] = int(lib.ammon_attention_prefill_scratch_bytes(c["tokens"], c["heads"],
                                                                      c["head"], ctx, split))
    if "q" in state:
        kept["part"], kept["out"] = empty(kept["bytes"] // 4), torch.empty_like(state["q"])
        kept["q_p"], kept["part_p"], kept["out_p"] = p(state["q"]), p(kept["part"]), p(kept["out"])
    return kept


def _run_own(state):
    c = state["c"]
    if "kept" not in state:
        state["kept"] = _kept(state)
    w = state["kept"]
    h, call = w["h"], w["call"]
    if c["kind"] == "store":
        call("ammon_kv4_store", h, None, *w["new_p"], c["tokens"], c["kv_heads"], c["head"], w["k"],
             w["v"], c["seq"], w["step"])
    if c["kind"] == "attn":
        call("ammon_attention_decode", h, None, w["q_p"], c["heads"], w["k"], w["v"], w["kv4"],
             c["kv_heads"], c["head"], c["seq"], w["step"], w["split"], w["part_p"], w["bytes"],
             w["out_p"])
        return {"out": w["out"]}
    if c["kind"] == "prefill":
        call("ammon_attention_prefill", h, None, w["q_p"], c["tokens"], c["heads"], w["k"], w["v"],
             w["kv4"], c["kv_heads"], c["head"], c["seq"], w["step"], c["start"] + c["tokens"],
             w["split"], w["part_p"], w["bytes"], w["out_p"])
        return {"out": w["out"]}
    if c["kind"] == "append":
        call("ammon_attention_decode_append", h, None, w["q_p"], c["heads"], *w["new_p"], w["k"],
             w["v"], w["kv4"], c["kv_heads"], c["head"], c["seq"], w["step"], w["split"],
             w["part_p"], w["bytes"], w["out_p"])
    call("ammon_kv4_load", h, None, w["k"], w["v"], c["kv_heads"], c["head"], c["seq"],
         c.get("pos", c.get("start")), c.get("tokens", 1), *w["rows_p"], w["to"])
    rows = dict(zip("kv", w["rows"]))
    return dict(rows, out=w["out"]) if c["kind"] == "append" else rows


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c = case
    n, kv = c.get("tokens", 1), c["kv_heads"]
    row = 20 * _groups(c["head"])  # bytes of a cache row
    if c["kind"] == "store":  # fp32 rows in, the cache's out and in, fp32 values out
        return {"bytes": 2 * n * kv * (8 * c["head"] + 2 * row), "flops": 2 * n * kv * 8 * c["head"]}
    if c["kind"] == "load":
        to = 2 if c["out"] == "bf16" else 4
        return {"bytes": 2 * n * kv * (to * c["head"] + row), "flops": 2 * n * kv * 2 * c["head"]}
    first = c.get("pos", c.get("start"))
    pairs = n * first + n * (n + 1) // 2
    nbytes = 2 * kv * row * (first + n) + 8 * n * c["heads"] * c["head"]
    if c["kind"] == "append":
        nbytes += 2 * kv * (8 * c["head"] + row)
    return {"bytes": nbytes, "flops": 4 * c["heads"] * c["head"] * pairs}


# ---- the same in 64 bits ---------------------------------------------------------------------------
def _exact_values(cache, c, first, last):
    """The numbers of positions first..last - 1 in float64, byte by byte."""
    n, rows = _groups(c["head"]), c["kv_heads"] * c["seq"]
    codes = cache[:rows * 16 * n].view(c["kv_heads"], c["seq"], 4, n, 4)[:, first:last]
    sb = cache[rows * 16 * n:].view(torch.float16).view(c["kv_heads"], c["seq"], n, 2)[:, first:last]
    sb = sb.double()
    out = torch.empty((c["kv_heads"], last - first, 32 * n), dtype=torch.float64, device=cache.device)
    for d in range(32 * n):
        j, p, e = d // 32, d % 32 // 8, d % 8
        byte = e // 4 + 2 * (e % 2)  # two codes a byte, even numbers in the first two
        code = codes[:, :, p, j, byte].double()
        code = torch.floor(code / 16) if e // 2 % 2 else torch.remainder(code, 16)
        out[..., d] = (sb[:, :, j, 0] * (16 + code) + sb[:, :, j, 1]).half().double()
    return out[..., :c["head"]]


def _exact_stored(x):
    """What rows x [n, kv_heads, head] read back as, [kv_heads, n, head]: the definition's roundings
    (fp32, fp16) of float64 results."""
    f32 = lambda t: t.float().double()  # noqa: E731
    f16 = lambda t: t.float().half().double()  # noqa: E731
    x = torch.clamp(x.double().transpose(0, 1), -16384, 16384)
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], 32):
        y = x[..., at:at + 32]
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        s = f16(f32(f32(hi - lo) / 15))
        b = f16(f32(lo - 16 * s))
        inv = torch.where(s > 0, f32(1 / s), torch.zeros_like(s))
        code = torch.clamp(torch.round(f32(f32(f32(y - b) * inv) - 16)), 0, 15)
        out[..., at:at + 32] = f16(s * (16 + code) + b)
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    first = c.get("pos", c.get("start"))
    last = first + c.get("tokens", 1)
    if c["kind"] == "store":
        return dict(zip("kv", (_exact_stored(x) for x in s["new"])))
    if c["kind"] == "load":
        return {x: _exact_values(s[x], c, first, last) for x in ("k", "v")}
    past = first if c["kind"] == "append" else last
    kv = {x: _exact_values(s[x], c, 0, past) for x in ("k", "v")}
    result = {}
    if c["kind"] == "append":
        for x, new in zip("kv", s["new"]):
            result[x] = _exact_stored(new[None])
            kv[x] = torch.cat([kv[x], result[x]], 1)
    q = s["q"].double()
    g = c["heads"] // c["kv_heads"]
    out = torch.empty_like(q)
    late = torch.arange(last, device="cuda")[None, :] > torch.arange(first, last, device="cuda")[:, None]
    for i in range(c["heads"]):
        score = (q[:, i] @ kv["k"][i // g].t()) * c["head"] ** -0.5
        out[:, i] = torch.softmax(score.masked_fill(late, -math.inf), -1) @ kv["v"][i // g]
    return dict(result, out=out)
