"""The token path on packed weights: attention over packed sequences, rotary positions with several axes and 4-bit
matrix-vector products, as a serving or prompt-processing program uses them.

A case names its operator in "op" and gives its sizes. With own = False run() computes the operators in elementary torch
operations in 32 bits; with own = True it makes the package's calls. Sequence lengths follow from the case alone, values
from the seed. exact() computes each result in 64 bits from the definitions.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lib():
    path = str(Path(__file__).resolve().parents[1] / "idol.cpp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import idolq_lib
    return idolq_lib


def listed():
    return [
        # one query of one sequence after a short context: the smallest call, latency counts
        dict(name="attn_token", op="attention", form="step", dtype="bf16", seqs=1, new=1, longest=500, heads=16, kv=16,
             hd=64, causal=True),
        # a serving step: one new query for each of 48 sequences whose contexts differ widely, four queries a key head
        dict(name="attn_step_ragged", op="attention", form="step", dtype="bf16", seqs=48, new=1, longest=8192, heads=32,
             kv=8, hd=128, causal=True),
        # a piece of a long prompt: 500 new tokens that see 32 thousand earlier ones
        dict(name="attn_chunk", op="attention", form="step", dtype="bf16", seqs=1, new=500, longest=32768, heads=32,
             kv=8, hd=128, causal=True),
        # a batch of prompts of different lengths, one key head per query head (the denoiser's 24 heads of 64)
        dict(name="attn_prompts", op="attention", form="prompt", dtype="fp16", seqs=8, new=0, longest=4096, heads=24,
             kv=24, hd=64, causal=True),
        # one long prompt with grouped heads: the largest call
        dict(name="attn_long_prompt", op="attention", form="prompt", dtype="bf16", seqs=1, new=0, longest=16384,
             heads=32, kv=8, hd=128, causal=True),
        # point sets of different sizes attending to their own sets of latent tokens (the decoders' 16 heads of 64)
        dict(name="attn_points", op="attention", form="cross", dtype="bf16", seqs=6, new=1000, longest=8192, heads=16,
             kv=16, hd=64, causal=False),
        # a few new tokens of several requests before attention: latency
        dict(name="rotary_token", op="rotary", dtype="bf16", rows=7, heads=32, kv=8, hd=128, axes=1, style="halves",
             partial=False),
        # tokens of a video latent, (time, height, width) positions, queries and keys of the fused projection
        dict(name="rotary_video", op="rotary", dtype="bf16", rows=32760, heads=24, kv=24, hd=64, axes=3, style="halves",
             partial=False),
        # image patches in fp32 with two axes and fractional positions, neighbouring elements paired, odd row count
        dict(name="rotary_image", op="rotary", dtype="fp32", rows=5001, heads=16, kv=16, hd=64, axes=2,
             style="interleaved", partial=True),
        # one token through a 4-bit layer
        dict(name="q4_token", op="q4", kind="q4_0", dtype="bf16", m=1, n=4096, k=4096, bias=True, residual=False),
        # a small batch of tokens through a large layer of 4-bit super-blocks: weight bytes count
        dict(name="q4_large", op="q4", kind="q4_k", dtype="fp16", m=4, n=16384, k=8192, bias=False, residual=True),
        # fp32 activations, rows and outputs that fill no tile
        dict(name="q4_odd", op="q4", kind="q4_0", dtype="fp32", m=13, n=4099, k=1568, bias=True, residual=True),
    ]


def draw(rng):
    def log(lo, hi, step=1):
        return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)

    op = rng.choice(("attention", "attention", "rotary", "q4"))
    if op == "attention":
        form = rng.choice(("step", "step", "prompt", "prompt", "cross"))
        kv = rng.choice((1, 2, 3, 4, 8))
        heads = kv * rng.choice((1, 2, 3, 4) if kv > 4 else (1, 2, 4, 8))
        if form == "step":
            seqs = log(1, 64)
            new = 1 if rng.random() < 0.6 else log(2, max(4, 600 // seqs))
            longest = log(64, 65536 if seqs < 16 else 16384)
        elif form == "prompt":
            seqs, new = log(1, 16), 0
            longest = log(16, 8192 if seqs < 3 else 2048)
        else:
            seqs, new, longest = log(1, 8), log(16, 2048), log(64, 8192)
        return dict(op=op, form=form, dtype=rng.choice(("bf16", "bf16", "fp16")), seqs=seqs, new=new, longest=longest,
                    heads=heads, kv=kv, hd=rng.choice((64, 128)), causal=form != "cross" and rng.random() < 0.9)
    if op == "rotary":
        kv = rng.choice((0, 1, 2, 8, 16))
        return dict(op=op, dtype=rng.choice(("bf16", "fp16", "fp32")), rows=log(1, 32760),
                    heads=max(1, kv) * rng.choice((1, 2, 4)), kv=kv, hd=rng.choice((32, 64, 80, 96, 128)),
                    axes=rng.choice((1, 2, 3)), style=rng.choice(("halves", "interleaved")), partial=rng.random() < 0.4)
    kind = rng.choice(("q4_0", "q4_k"))
    return dict(op=op, kind=kind, dtype=rng.choice(("bf16", "fp16", "fp32")), m=log(1, 16), n=log(100, 16384),
                k=log(256, 8192, 256 if kind == "q4_k" else 32), bias=rng.random() < 0.5, residual=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen)


def _lengths(case):
    """(query lengths, key lengths) of the case's sequences: the longest context once, the others down to a sixteenth
    of it; a step adds `new` queries to each, a prompt is its own context, cross has query sets of its own."""
    r = random.Random("%s %d %d %d" % (case["form"], case["seqs"], case["new"], case["longest"]))
    spread = lambda top: max(1, int(top * 16.0 ** -r.random()))  # noqa: E731
    lk = [case["longest"]] + [spread(case["longest"]) for _ in range(case["seqs"] - 1)]
    r.shuffle(lk)
    if case["form"] == "prompt":
        return list(lk), lk
    if case["form"] == "cross":
        return [spread(case["new"]) for _ in lk], lk
    return [min(case["new"], n) for n in lk], lk


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _sections(case):
    """Pairs of a head that turn with each axis: all of them, or (partial) about half."""
    pairs = case["hd"] // 2
    if case["partial"]:
        pairs = max(case["axes"], pairs // 2)
    each = pairs // case["axes"]
    return [pairs - each * (case["axes"] - 1)] + [each] * (case["axes"] - 1)


def _q4_blocks(gen, kind, n, k):
    """GGUF blocks (uint8 [n, blocks, bytes]) of a random matrix of standard deviation about 0.02."""
    values, size = (32, 18) if kind == "q4_0" else (256, 144)
    b = torch.randint(0, 256, (n, k // values, size), device=DEV, generator=gen, dtype=torch.uint8)
    d = 0.02 * (0.5 + torch.rand((n, k // values, 1), device=DEV, generator=gen))
    if kind == "q4_0":   # codes around 8, standard deviation 4.6
        b[:, :, :2] = (d / 4.6).half().view(torch.uint8)
    else:                # 6-bit scales about 31 times codes about 7.5, less the minimums
        d = d / (31.0 * 4.6)
        b[:, :, :2] = d.half().view(torch.uint8)
        b[:, :, 2:4] = (7.5 * d).half().view(torch.uint8)
    return b


def _inputs(case, seed):
    gen, op, dt = _gen(seed), case["op"], DTYPES[case["dtype"]]
    if op == "attention":
        lq, lk = _lengths(case)
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        if case["form"] == "prompt":   # one fused projection
            x = _randn(gen, sum(lq), (heads + 2 * kv) * hd).to(dt)
            q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
        else:
            q = _randn(gen, sum(lq), heads * hd).to(dt)
            x = _randn(gen, sum(lk), 2 * kv * hd).to(dt)
            k, v = x[:, :kv * hd], x[:, kv * hd:]
        return dict(q=q, k=k, v=v, lq=lq, lk=lk)
    if op == "rotary":
        rows, heads, kv, hd, sections = case["rows"], case["heads"], case["kv"], case["hd"], _sections(case)
        x = _randn(gen, rows, (heads + kv) * hd).to(dt)
        # positions of a grid of tokens that starts anywhere on the first axis; fractional ones for images
        side = max(1, int(math.sqrt(rows / 8.0)))
        i = torch.arange(rows, device=DEV)
        grid = torch.stack([i // (side * side), i // side % side, i % side], 1)[:, 3 - case["axes"]:]
        if case["axes"] == 2:
            pos = (grid.float() + torch.rand((rows, 2), device=DEV, generator=gen)) * 0.37
        else:
            start = torch.randint(0, 100000, (1,), device=DEV, generator=gen)
            pos = grid.clone()
            pos[:, 0] += start
            if case["axes"] == 1:
                pos = i.unsqueeze(1) + start
            pos = pos.to(torch.int32)
        freqs = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections]).float().to(DEV)
        return dict(q=x[:, :heads * hd], k=x[:, heads * hd:] if kv else None, pos=pos.contiguous(), freqs=freqs,
                    sections=sections)
    m, n, k = case["m"], case["n"], case["k"]
    return dict(w=_q4_blocks(gen, case["kind"], n, k), x=_randn(gen, m, k).to(dt),
                bias=_randn(gen, n) * 0.1 if case["bias"] else None,
                residual=_randn(gen, m, n).to(dt) if case["residual"] else None)


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    if case["op"] == "attention":
        for side in ("q", "k"):
            s["cu_" + side] = torch.tensor(_offsets(s["l" + side]), device=DEV, dtype=torch.int32)
        s["max_k"] = max(s["lk"])
    elif case["op"] == "q4":
        s["w"] = s["w"].reshape(-1)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _attention_plain(s):
    c = s["case"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    g, scale = heads // kv, hd ** -0.5
    out = torch.zeros(s["q"].shape, device=DEV, dtype=s["q"].dtype)
    q0 = k0 = 0
    for lq, lk in zip(s["lq"], s["lk"]):
        k = s["k"][k0:k0 + lk].float().reshape(lk, kv, hd).permute(1, 2, 0)                       # [kv, hd, lk]
        v = s["v"][k0:k0 + lk].float().reshape(lk, kv, hd).transpose(0, 1)                        # [kv, lk, hd]
        step = max(1, (1 << 27) // max(1, lk * heads))
        for a in range(0, lq, step):
            b = min(a + step, lq)
            seen = max(0, min(lk, b + lk - lq)) if c["causal"] else lk
            q = s["q"][q0 + a:q0 + b].float().reshape(b - a, kv, g, hd).permute(1, 0, 2, 3).reshape(kv, -1, hd)
            p = torch.matmul(q, k[:, :, :seen]).reshape(kv, b - a, g, seen) * scale
            if c["causal"]:
                i = torch.arange(a, b, device=DEV).reshape(-1, 1, 1) + (lk - lq)
                p = torch.where(torch.arange(seen, device=DEV) <= i, p, -math.inf)
            p = torch.exp(p - p.amax(-1, keepdim=True))
            o = torch.matmul(p.reshape(kv, -1, seen), v[:, :seen]) / p.sum(-1).reshape(kv, -1, 1)
            o = o.reshape(kv, b - a, g, hd).transpose(0, 1).reshape(b - a, heads * hd)
            out[q0 + a:q0 + b] = o.to(out.dtype)
        q0, k0 = q0 + lq, k0 + lk
    return out


def _rotary_plain(x, s, heads):
    c = s["case"]
    hd, pairs = c["hd"], s["freqs"].numel()
    axis = torch.tensor([a for a, n in enumerate(s["sections"]) for _ in range(n)], device=DEV)
    turn = s["pos"].double()[:, axis] * s["freqs"].double()                                       # [rows, pairs]
    cos, sin = torch.cos(turn).float().unsqueeze(1), torch.sin(turn).float().unsqueeze(1)
    y = x.float().reshape(-1, heads, hd).clone()
    first, second = ((slice(0, pairs), slice(pairs, 2 * pairs)) if c["style"] == "halves"
                     else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)))
    a, b = y[:, :, first].clone(), y[:, :, second].clone()
    y[:, :, first] = a * cos - b * sin
    y[:, :, second] = b * cos + a * sin
    return y.reshape(x.shape).to(x.dtype)


def _q4_values(b, kind, real):
    """The matrix of GGUF blocks [n, blocks, bytes] in the type `real`."""
    half = lambda t: t.contiguous().view(torch.float16).to(real)  # noqa: E731
    n = b.shape[0]
    if kind == "q4_0":
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], dim=-1).to(real) - 8.0
        return (half(b[..., :2]) * q).reshape(n, -1)
    a, m, h = (b[..., 4 + 4 * i:8 + 4 * i].to(torch.int32) for i in range(3))
    sc = torch.cat([a & 63, (h & 15) | ((a >> 6) << 4)], dim=-1).to(real)
    mn = torch.cat([m & 63, (h >> 4) | ((m >> 6) << 4)], dim=-1).to(real)
    codes = b[..., 16:].reshape(*b.shape[:2], 4, 32)
    q = torch.stack([codes & 15, codes >> 4], dim=3).reshape(*b.shape[:2], 8, 32).to(real)
    return ((half(b[..., :2]) * sc).unsqueeze(-1) * q - (half(b[..., 2:4]) * mn).unsqueeze(-1)).reshape(n, -1)


def _q4_plain(s, real=torch.float32):
    c = s["case"]
    y = torch.matmul(s["x"].to(real), _q4_values(s["w"].reshape(c["n"], -1, 18 if c["kind"] == "q4_0" else 144),
                                                 c["kind"], real).t())
    if s["bias"] is not None:
        y = y + s["bias"].to(real)
    if s["residual"] is not None:
        y = y + s["residual"].to(real)
    return y


def run(s):
    c = s["case"]
    if c["op"] == "attention":
        if not own:
            return _attention_plain(s)
        return _lib().attention_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], c["heads"], c["kv"], c["hd"],
                                       causal=c["causal"], max_k=s["max_k"])
    if c["op"] == "rotary":
        if not own:
            q = _rotary_plain(s["q"], s, c["heads"])
            return (q, _rotary_plain(s["k"], s, c["kv"])) if s["k"] is not None else q
        return _lib().rotary(s["q"], c["heads"], c["hd"], s["pos"], s["freqs"], s["sections"], k=s["k"],
                             kv_heads=c["kv"], interleaved=c["style"] == "interleaved")
    if not own:
        return _q4_plain(s).to(s["x"].dtype)
    L = _lib()
    return L.q4_gemv(s["x"], s["w"], L.KIND_Q4_0 if c["kind"] == "q4_0" else L.KIND_Q4_K, c["n"], bias=s["bias"],
                     residual=s["residual"])


# --------------------------------------------------------------------------------------------------- work and exact
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        pairs = 0
        for a, b in zip(lq, lk):
            n = min(a, b)  # queries that see something; the last of them sees all b keys
            pairs += n * b - n * (n - 1) // 2 if case["causal"] else a * b
        return dict(bytes=size * hd * (2 * sum(lq) * heads + 2 * sum(lk) * kv) + 8 * (len(lq) + 1),
                    flops=4 * heads * hd * pairs)
    if case["op"] == "rotary":
        cells = case["rows"] * (case["heads"] + case["kv"])
        pairs = sum(_sections(case))
        return dict(bytes=2 * size * cells * case["hd"] + 4 * (case["rows"] * case["axes"] + pairs), flops=6 * cells * pairs)
    m, n, k = case["m"], case["n"], case["k"]
    return dict(bytes=n * k * 9 // 16 + size * (m * k + m * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0),
                flops=2 * m * n * k)


def _attention_exact(i, case):
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    out = torch.zeros(i["q"].shape, device=DEV, dtype=torch.float64)
    qo, ko = _offsets(i["lq"]), _offsets(i["lk"])
    for n, (lq, lk) in enumerate(zip(i["lq"], i["lk"])):
        for h in range(heads):
            kh = h // (heads // kv)
            k = i["k"][ko[n]:ko[n + 1], kh * hd:(kh + 1) * hd].double()
            v = i["v"][ko[n]:ko[n + 1], kh * hd:(kh + 1) * hd].double()
            for a in range(0, lq, 8192):
                rows = slice(qo[n] + a, qo[n] + min(a + 8192, lq))
                score = (i["q"][rows, h * hd:(h + 1) * hd].double() @ k.t()) / math.sqrt(hd)
                if case["causal"]:
                    # query a + r sees keys 0 .. a + r + lk - lq
                    hidden = torch.ones(score.shape, device=DEV, dtype=torch.bool).triu(a + lk - lq + 1)
                    score = score.masked_fill(hidden, -math.inf)
                weight = torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True))
                out[rows, h * hd:(h + 1) * hd] = weight @ v
    return out


def _rotary_exact(x, i, case, heads):
    """Each pair as a complex number, turned by the product with exp(i angle)."""
    hd, n = case["hd"], i["freqs"].numel()
    angle, at = [], 0
    for a, count in enumerate(i["sections"]):
        angle.append(i["pos"][:, a:a + 1].double() * i["freqs"][at:at + count].double())
        at += count
    turn = torch.polar(torch.ones_like(torch.cat(angle, 1)), torch.cat(angle, 1)).unsqueeze(1)
    y = x.double().reshape(-1, heads, hd)
    head, rest = y[..., :2 * n], y[..., 2 * n:]
    pairs = head.unflatten(-1, (2, n)).transpose(-1, -2) if case["style"] == "halves" else head.unflatten(-1, (n, 2))
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    turned = turned.transpose(-1, -2).flatten(-2) if case["style"] == "halves" else turned.flatten(-2)
    return torch.cat([turned, rest], -1).reshape(x.shape)


def _q4_exact(i, case):
    """sum over groups of scale * (codes . x) - minimum * (sum of x), group by group."""
    b, x = i["w"], i["x"].double()
    n, m = case["n"], case["m"]
    xg = x.reshape(m, -1, 32)
    bits = lambda t: t.contiguous().view(torch.float16).double()  # noqa: E731
    if case["kind"] == "q4_0":
        d = bits(b[..., :2]).squeeze(-1)
        minimum = 8.0 * d
        low, high = b[..., 2:].int() % 16, b[..., 2:].int() // 16
        codes = torch.cat([low, high], -1)
    else:
        s = b[..., 4:16].int()
        sc = torch.empty((*b.shape[:2], 8), device=DEV, dtype=torch.float64)
        mn = torch.empty_like(sc)
        for j in range(4):
            sc[..., j], mn[..., j] = s[..., j] % 64, s[..., 4 + j] % 64
            sc[..., 4 + j] = s[..., 8 + j] % 16 + 16 * (s[..., j] // 64)
            mn[..., 4 + j] = s[..., 8 + j] // 16 + 16 * (s[..., 4 + j] // 64)
        d = (bits(b[..., :2]) * sc).reshape(n, -1)
        minimum = (bits(b[..., 2:4]) * mn).reshape(n, -1)
        codes = torch.empty((*b.shape[:2], 8, 32), device=DEV, dtype=torch.int32)
        for j in range(4):
            chunk = b[..., 16 + 32 * j:48 + 32 * j].int()
            codes[..., 2 * j, :], codes[..., 2 * j + 1, :] = chunk % 16, chunk // 16
        codes = codes.reshape(n, -1, 32)
    y = -(xg.sum(-1) @ minimum.t())
    for r in range(m):
        for a in range(0, n, 2048):
            dots = (codes[a:a + 2048].double() * xg[r]).sum(-1)
            y[r, a:a + 2048] += (dots * d[a:a + 2048]).sum(-1)
    if i["bias"] is not None:
        y += i["bias"].double()
    if i["residual"] is not None:
        y += i["residual"].double()
    return y


def exact(case, seed):
    i = _inputs(case, seed)
    if case["op"] == "attention":
        return _attention_exact(i, case)
    if case["op"] == "rotary":
        q = _rotary_exact(i["q"], i, case, case["heads"])
        return (q, _rotary_exact(i["k"], i, case, case["kv"])) if i["k"] is not None else q
    return _q4_exact(i, case)
