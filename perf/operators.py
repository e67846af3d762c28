"""The 4-bit serving operators, as cases that can be timed and compared:

  cache      K/V rows quantised into a paged 4-bit cache and read back
             (KV4Cache.append, KV4Cache.read)
  attention  queries against such a cache (attention_kv4)
  linear     rows times 4-bit weights with group scales (dq4_gemm)

Each runs in its plain form (elementary torch operations in 32 bits) or, with
`own` set, through the library.

Cache format. A page holds 64 tokens of every K/V head; per (page, head) one
block of bytes: K codes (64 x 64), V codes (64 x 64), K pairs, V pairs. A
token's 128 values fall into groups of 32, 64 or 128; a pair is (scale, zero)
in bf16, low and high half of a 32-bit word, [token][group]:
  zero = min, scale = (max - min) / 15 of the group, rounded to bf16,
  code = round((x - zero) / scale) in 0 .. 15 (ties to even; 0 where scale is 0),
  value = zero + scale * code.
With nibble n of a byte string meaning the low (even n) or high (odd n) half of
byte n / 2, code d of token t is
  K: nibble ((d / 8) % 4) * 32 + (d / 32) * 8 + d % 8 of the 64 bytes at 64 t,
  V: nibble (d / 32) * 4 + d % 4 of the 8 bytes at
     512 (t / 8) + 64 ((d / 4) % 8) + 16 ((t % 8) / 2) + 8 (t % 2).

Weights: code w + 8 in 0 .. 15, two columns a byte (low half the even column),
value (code - 8) * scale with one scale per group of 32, 64 or 128 columns.
"""

import math
import pathlib
import random
import sys

import torch

own = False

PAGE = 64
HD = 128


def _ltxb():
    p = str(pathlib.Path(__file__).resolve().parents[1] / "ltx-zml_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    import ltxb
    return ltxb


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# `new` rows a sequence belong to the call (0: all of its tokens, ragged);
# lengths are drawn from [len_lo, len_hi] with the seed `lengths`.

def _cache(name, batch, new, lo, hi, kv_heads, group, lengths=1):
    return {"name": name, "op": "cache", "batch": batch, "new": new, "len_lo": lo, "len_hi": hi,
            "kv_heads": kv_heads, "group": group, "lengths": lengths}


def _attention(name, batch, new, lo, hi, heads, kv_heads, group, causal, lengths=1):
    return {"name": name, "op": "attention", "batch": batch, "new": new, "len_lo": lo, "len_hi": hi, "heads": heads,
            "kv_heads": kv_heads, "group": group, "causal": causal, "lengths": lengths}


def _linear(name, m, n, k, group, scales, bias):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "group": group, "scales": scales, "bias": bias}


def listed():
    return [
        # one generated token of each of 16 sequences goes into the cache
        _cache("cache step", 16, 1, 1, 4096, 8, 32),
        # the 28,160 tokens of a whole clip (22 x 32 x 40), all 32 heads of the block
        _cache("cache clip", 1, 28160, 28160, 28160, 32, 128),
        # one token against a short prompt: the latency of a call
        _attention("token short", 1, 1, 77, 77, 32, 8, 128, True),
        # a served batch of ragged lengths, heads shared in fours
        _attention("token batch", 64, 1, 17, 8192, 32, 8, 32, True),
        # one token against a long cache with a K/V head for every query head
        _attention("token long", 1, 1, 131009, 131009, 32, 32, 128, True),
        # four proposed tokens a sequence, checked at once
        _attention("four tokens", 8, 4, 900, 2500, 32, 8, 64, True),
        # ragged prompts, each attending to its own earlier tokens
        _attention("prompts", 4, 0, 250, 1501, 32, 8, 32, True),
        # one of eight parts of a clip (3,520 of 28,160 tokens) against the whole clip's cache
        _attention("clip part", 1, 3520, 28160, 28160, 32, 32, 128, False),
        # a square projection of one token (D = 4096)
        _linear("row square", 1, 4096, 4096, 128, "bf16", False),
        # the modulation linear of two timesteps (9 D outputs), scales as the checkpoint tools write them
        _linear("rows modulation", 2, 36864, 4096, 64, "f32", True),
        # the FFN's down projection for a batch of 16 tokens
        _linear("rows down", 16, 4096, 16384, 32, "bf16", True),
        # a prompt's rows through the FFN's up projection
        _linear("rows prompt", 1001, 16384, 4096, 128, "bf16", False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("cache", "attention", "attention", "linear"))
    group = rng.choice((32, 64, 128))
    if op == "linear":
        n = 32 * _log(rng, 8, 1152)
        k = 128 * _log(rng, 4, 128)
        m = _log(rng, 1, 1024)
        m = max(1, min(m, (1001 * 16384 * 4096) // (n * k)))
        c = _linear("", m, n, k, group, rng.choice(("bf16", "f32")), rng.random() < 0.5)
    else:
        kv_heads = rng.choice((1, 2, 4, 5, 8, 16, 32))
        batch = _log(rng, 1, 64)
        new = rng.choice((0, 1, 1, 2, 5, 16))
        most = 28160 * 32 if new == 0 else 131009 * 32  # tokens x heads, as in the largest listed cases
        hi = _log(rng, 1, 131072)
        hi = max(1, min(hi, most // (kv_heads * batch)))
        lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
        lengths = rng.randrange(1 << 20)
        if new > lo:
            new = 1
        if op == "cache":
            c = _cache("", batch, new, lo, hi, kv_heads, group, lengths)
        else:
            shared = rng.choice((1, 1, 2, 3, 4, 7, 8, 16))
            shared = max(1, min(shared, 64 // kv_heads))
            heads = shared * kv_heads
            if new == 0 and batch * heads * hi * hi > 3520 * 28160 * 32:
                hi = max(1, int(math.sqrt(3520 * 28160 * 32 / (batch * heads))))
                lo = max(1, min(lo, hi))
            c = _attention("", batch, new, lo, hi, heads, kv_heads, group, rng.random() < 0.8, lengths)
    del c["name"]
    return c


def _lengths(case):
    r = random.Random(case["lengths"])
    return [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def _new(case):
    return [n if case["new"] == 0 else case["new"] for n in _lengths(case)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _rows(rng, shape, device):
    """K/V-like rows [..., heads, 128]: channels of unequal size, some with an offset, some far larger."""
    x = torch.randn(*shape, generator=rng, device=device)
    size = torch.exp(0.5 * torch.randn(shape[-2], shape[-1], generator=rng, device=device))
    big = torch.rand(shape[-2], shape[-1], generator=rng, device=device) < 0.02
    shift = torch.randn(shape[-2], shape[-1], generator=rng, device=device)
    return ((x + 0.5 * shift) * size * torch.where(big, 4.0, 1.0)).to(torch.bfloat16)


def _group_codes(x, group):
    """codes uint8 [..., 128], scale and zero bf16 [..., 128 / group] of bf16 rows."""
    g = x.float().unflatten(-1, (HD // group, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    # 64 bits for both quotients: a value next to a border must not depend on their rounding
    scale = ((hi.double() - lo.double()) / 15.0).float().to(torch.bfloat16)
    q = torch.where(scale > 0, (g.double() - lo.double()) / scale.double(), 0.0)
    code = q.round().clamp_(0, 15).to(torch.uint8)
    return code.flatten(-2), scale.squeeze(-1), lo.to(torch.bfloat16).squeeze(-1)


def _nibbles(codes):
    """pairs of codes along the last axis -> bytes, the even one low"""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _halves(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _pack(kc, ks, kz, vc, vs, vz):
    """Blocks [..., bytes] from codes [..., 64, 128] and bf16 pairs [..., 64, groups] of K and V."""
    lead = kc.shape[:-2]
    k = _nibbles(kc.unflatten(-1, (4, 4, 8)).transpose(-3, -2))            # [t, c, j, 4]
    v = _nibbles(vc.unflatten(-1, (4, 8, 4)).transpose(-3, -2)).flatten(-2)  # [t, g, 8]
    v = v.unflatten(-3, (8, 4, 2)).movedim(-2, -4)                          # [octet, g, c, parity, 8]
    pair = lambda s, z: torch.stack((s, z), -1).contiguous().view(torch.uint8)
    return torch.cat([k.reshape(*lead, -1), v.reshape(*lead, -1), pair(ks, kz).reshape(*lead, -1),
                      pair(vs, vz).reshape(*lead, -1)], -1)


def _unpack(blocks, group):
    """The f32 K and V values [..., 64, 128] of blocks [..., bytes]."""
    lead = blocks.shape[:-1]
    kb, vb, pairs = blocks[..., :4096], blocks[..., 4096:8192], blocks[..., 8192:]
    kc = _halves(kb.unflatten(-1, (PAGE, 4, 4, 4))).transpose(-3, -2).reshape(*lead, PAGE, HD)
    vc = vb.unflatten(-1, (8, 8, 4, 2, 8)).movedim(-4, -2)                  # [octet, c, parity, g, 8]
    vc = _halves(vc.reshape(*lead, PAGE, 8, 4, 2)).transpose(-3, -2).reshape(*lead, PAGE, HD)
    p = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (2, PAGE, HD // group, 2))

    def values(codes, p):
        return (p[..., 1:] + p[..., :1] * codes.float().unflatten(-1, (HD // group, group))).flatten(-2)
    return values(kc, p[..., 0, :, :, :]), values(vc, p[..., 1, :, :, :])


def _make(case, seed):
    """The inputs, before any packing."""
    dev = torch.device("cuda")
    rng = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "linear":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        x = torch.randn(m, k, generator=rng, device=dev).to(torch.bfloat16)
        w = (torch.randn(n, k, generator=rng, device=dev) * 0.02).unflatten(-1, (k // group, group))
        scale = (w.abs().amax(-1) / 7.0).to(torch.bfloat16 if case["scales"] == "bf16" else torch.float32)
        code = (torch.round(w / scale.float().unsqueeze(-1)).clamp_(-8, 7) + 8).to(torch.uint8).flatten(-2)
        bias = (torch.randn(n, generator=rng, device=dev) * 0.1).to(torch.bfloat16) if case["bias"] else None
        return {"x": x, "code": code, "scale": scale, "bias": bias}
    lens, new = _lengths(case), _new(case)
    start = [0]
    for c in new:
        start.append(start[-1] + c)
    s = {"lens": torch.tensor(lens, dtype=torch.int32, device=dev),
         "start": torch.tensor(start, dtype=torch.int32, device=dev),
         "rows": start[-1], "max_pages": (max(lens) + PAGE - 1) // PAGE}
    pages = case["batch"] * s["max_pages"]
    s["table"] = torch.randperm(pages, generator=rng, device=dev).to(torch.int32).view(case["batch"], s["max_pages"])
    s["pages"] = pages
    hk = case["kv_heads"]
    if case["op"] == "cache":
        s["k"], s["v"] = _rows(rng, (s["rows"], hk, HD), dev), _rows(rng, (s["rows"], hk, HD), dev)
    else:
        tokens = (case["batch"], s["max_pages"], PAGE, hk, HD)
        s["kq"] = _group_codes(_rows(rng, tokens, dev), case["group"])
        s["vq"] = _group_codes(_rows(rng, tokens, dev), case["group"])
        s["q"] = torch.randn(s["rows"], case["heads"], HD, generator=rng, device=dev).to(torch.bfloat16)
    return s


def prepare(case, seed):
    s = _make(case, seed)
    s["case"] = case
    if case["op"] == "linear":
        s["wq"] = _nibbles(s.pop("code"))
        return s
    block = 8192 + 2 * PAGE * 4 * (HD // case["group"])
    blocks = torch.zeros(s["pages"], case["kv_heads"], block, dtype=torch.uint8, device=s["lens"].device)
    if case["op"] == "attention":
        kq, vq = s.pop("kq"), s.pop("vq")
        blocks[s["table"].long()] = _pack(*(t.transpose(2, 3) for t in kq + vq))
    s["blocks"] = blocks
    # sequences with equally many rows need no list of where their rows begin
    s["row_start"] = s["start"] if case["new"] == 0 else None
    if own:
        s["cache"] = _ltxb().KV4Cache.from_pages(blocks, s["table"], s["lens"], group=case["group"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _plain_cache(s):
    group = s["case"]["group"]

    def held(x):
        code, scale, zero = _group_codes(x, group)
        v = zero.float().unsqueeze(-1) + scale.float().unsqueeze(-1) * code.float().unflatten(-1, (HD // group, group))
        return v.flatten(-2).to(torch.bfloat16)
    return held(s["k"]), held(s["v"])


def _plain_attention(s):
    case = s["case"]
    b, h, hk, rows = case["batch"], case["heads"], case["kv_heads"], s["rows"]
    n = max(_new(case))
    dev = s["q"].device
    k, v = _unpack(s["blocks"][s["table"].long()], case["group"])  # [B, pages, heads, 64, 128]
    k, v = (t.transpose(1, 2).flatten(2, 3) for t in (k, v))       # [B, heads, tokens, 128]
    r = torch.arange(rows, device=dev)
    seq = torch.searchsorted(s["start"][1:].long(), r, right=True)
    at = r - s["start"].long()[seq]
    q = torch.zeros(b, n, h, HD, device=dev)
    q[seq, at] = s["q"].float()
    q = q.view(b, n, hk, h // hk, HD).permute(0, 2, 1, 3, 4).reshape(b, hk, n * (h // hk), HD)
    p = q @ k.transpose(-1, -2)
    p *= 1.0 / math.sqrt(HD)
    key = torch.arange(k.shape[2], device=dev)
    last = s["lens"].long()[:, None].expand(b, n) - 1
    if case["causal"]:
        count = (s["start"][1:] - s["start"][:-1]).long()
        last = last - count[:, None] + 1 + torch.arange(n, device=dev)
    hidden = (key > last.repeat_interleave(h // hk, 1)[:, None, :, None])
    p.masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True)
    p -= torch.where(top == -math.inf, 0.0, top)
    p.exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(b, hk, n, h // hk, HD).permute(0, 2, 1, 3, 4).reshape(b, n, h, HD)
    return o[seq, at].to(torch.bfloat16)


def _plain_linear(s):
    group = s["case"]["group"]
    w = _halves(s["wq"]).float().unflatten(-1, (s["scale"].shape[1], group)) - 8.0
    w = (w * s["scale"].float().unsqueeze(-1)).flatten(-2)
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(torch.bfloat16)


def run(state):
    op = state["case"]["op"]
    if own:
        ltxb = _ltxb()
        if op == "cache":
            state["cache"].append(state["k"], state["v"], row_start=state["row_start"])
            return state["cache"].read(state["rows"], row_start=state["row_start"])
        if op == "attention":
            return ltxb.attention_kv4(state["q"], state["cache"], row_start=state["row_start"],
                                      causal=state["case"]["causal"])
        return ltxb.dq4_gemm(state["x"], state["wq"], state["scale"], bias=state["bias"])
    if op == "cache":
        return _plain_cache(state)
    return _plain_attention(state) if op == "attention" else _plain_linear(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its exact result
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        sb = 2 if case["scales"] == "bf16" else 4
        return {"bytes": n * k // 2 + n * (k // case["group"]) * sb + 2 * m * k + 2 * m * n + 2 * n * case["bias"],
                "flops": 2 * m * n * k}
    lens, new, hk = _lengths(case), _new(case), case["kv_heads"]
    held = 2 * (HD // 2 + 4 * (HD // case["group"]))  # a token's K and V of one head in the cache
    rows = sum(new)
    if case["op"] == "cache":  # bf16 rows in, cache written and read, bf16 rows out
        return {"bytes": rows * hk * (8 * HD + 2 * held), "flops": rows * hk * 2 * HD * 8}
    seen = sum(sum(n - c + 1 + i for i in range(c)) if case["causal"] else n * c for n, c in zip(lens, new))
    return {"bytes": sum(lens) * hk * held + 4 * rows * case["heads"] * HD, "flops": 4 * HD * case["heads"] * seen}


def exact(case, seed):
    s = _make(case, seed)
    if case["op"] == "linear":
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device=s["x"].device)
        x = s["x"].double()
        for a in range(0, case["n"], 4096):
            c = s["code"][a:a + 4096].double() - 8
            w = c * s["scale"][a:a + 4096].double().repeat_interleave(case["group"], 1)
            y[:, a:a + 4096] = x @ w.t()
        return y if s["bias"] is None else y + s["bias"].double()
    group = case["group"]
    if case["op"] == "cache":
        out = []
        for x in (s["k"], s["v"]):
            y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
            for h in range(x.shape[1]):
                for a in range(0, HD, group):
                    g = x[:, h, a:a + group].double()
                    zero = g.min(1).values
                    # bf16 of a 64-bit quotient, by way of 32 bits: no quotient by 15 of two bf16 values'
                    # difference lies close enough to a bf16 border for the detour to matter
                    step = ((g.max(1).values - zero) / 15).float().bfloat16().double()
                    code = torch.round((g - zero[:, None]) / torch.where(step > 0, step, torch.inf)[:, None])
                    y[:, h, a:a + group] = zero[:, None] + step[:, None] * code.clamp(0, 15)
            out.append(y)
        return tuple(out)
    heads, hk = case["heads"], case["kv_heads"]
    per = heads // hk
    (kc, ks, kz), (vc, vs, vz) = s["kq"], s["vq"]
    y = torch.zeros(s["rows"], heads, HD, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (n, c) in enumerate(zip(_lengths(case), _new(case))):
        pages = (n + PAGE - 1) // PAGE
        for h in range(hk):
            def value(codes, scale, zero):
                rep = lambda t: t[b, :pages, :, h].double().reshape(pages * PAGE, -1).repeat_interleave(group, 1)[:n]
                return rep(zero) + rep(scale) * codes[b, :pages, :, h].double().reshape(pages * PAGE, HD)[:n]
            k, v = value(kc, ks, kz), value(vc, vs, vz)
            q = s["q"][at:at + c, h * per:(h + 1) * per].double()
            score = torch.einsum("ihd,td->hit", q, k) / HD ** 0.5
            if case["causal"]:
                i = torch.arange(c, device=k.device)[:, None] + (n - c)
                score = score.masked_fill(torch.arange(n, device=k.device)[None] > i, -math.inf)
            y[at:at + c, h * per:(h + 1) * per] = torch.einsum("hit,td->ihd", torch.softmax(score, -1), v)
        at += c
    return y
