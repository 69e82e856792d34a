"""Cases of the 8-bit serving operators and of attention for drafted tokens, with their plain forms.

Four operators:

``linear``  y = act(Q(x) @ Q(w)^T + bias) + residual, Q = e4m3 with one power-of-two scale per 128 values along K;
            the weights are quantised once, the activations within the call.
``cache``   K/V of new tokens quantised into an 8-bit cache (one scale per token, head and K or V), then some of
            the cache's slots read back.
``decode``  single-token attention over that cache: left padding, beams' lineage table, shared K/V heads.
``tree``    attention of up to 64 drafted tokens per row, each seeing the row's cached prefix and its own
            ancestors among the drafted tokens, over the 8-bit or the bf16 cache.

``run`` computes the plain form in float32, or calls the package where ``own`` is true.
"""
import math
import os
import sys

import torch

own = False

TOP = 448.0  # largest e4m3 value
BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "index-tts-dubbing_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from indextts.gpt import kv8
    from indextts.utils import fp8
    return kv8, fp8


# ---- the cases ----------------------------------------------------------------------------------


def listed():
    return [
        # c_fc of the decode step of one utterance: weight bytes and latency only
        dict(name="linear-1-row", op="linear", m=1, k=1024, n=4096, x="bf16", act=1, bias=True, residual=False, out="bf16"),
        # mlp.c_proj of a decode step of 32 utterances x 3 beams, added to the f32 residual stream
        dict(name="linear-96-rows", op="linear", m=96, k=4096, n=1024, x="bf16", act=0, bias=True, residual=True, out="f32"),
        # the vocabulary's logits at every position of a few sentences; sizes that fill no tile
        dict(name="linear-odd", op="linear", m=1337, k=1000, n=8194, x="f32", act=0, bias=True, residual=False, out="f32"),
        # c_fc of the teacher-forced pass over 32 utterances of 450 positions
        dict(name="linear-latent-pass", op="linear", m=14400, k=1024, n=4096, x="bf16", act=1, bias=True, residual=False, out="bf16"),
        # one decode step's K/V of 32 rows appended, the same slots read back
        dict(name="cache-step", op="cache", rows=32, heads=16, hd=64, smax=608, tokens=32, read=32, src="f32", out="bf16"),
        # the prompt and codes of 64 rows written at once, ragged, then moved rows read back
        dict(name="cache-prompt", op="cache", rows=64, heads=16, hd=64, smax=640, tokens=24000, read=24000, src="bf16", out="bf16"),
        # a single utterance's step early in its decode
        dict(name="decode-1-row", op="decode", rows=1, heads=16, group=1, hd=64, smax=608, longest=131, q="bf16", out="bf16", beams=1, pad=0),
        # 32 utterances x 3 beams with the lineage table and left padding
        dict(name="decode-beams", op="decode", rows=96, heads=16, group=1, hd=64, smax=608, longest=483, q="f32", out="bf16", beams=3, pad=23),
        # few rows with a long history and shared K/V heads
        dict(name="decode-long", op="decode", rows=8, heads=4, group=4, hd=128, smax=32768, longest=32749, q="bf16", out="bf16", beams=1, pad=0),
        # eight drafted tokens of one utterance over the bf16 cache
        dict(name="tree-1-row", op="tree", rows=1, heads=16, group=1, hd=64, smax=608, longest=289, tokens=8, q="bf16", out="bf16", cache="bf16", pad=0),
        # sixteen drafted tokens for each of 32 utterances, ragged, in the f32 form
        dict(name="tree-rows", op="tree", rows=32, heads=16, group=1, hd=64, smax=640, longest=565, tokens=16, q="f32", out="f32", cache="8", pad=11),
        # a full tree over a long history, shared K/V heads
        dict(name="tree-long", op="tree", rows=4, heads=8, group=4, hd=128, smax=16384, longest=16301, tokens=64, q="bf16", out="bf16", cache="8", pad=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        b, f = top.get(c["op"], (0, 0))
        top[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    op = rng.choice(["linear", "cache", "decode", "tree"])
    while True:
        if op == "linear":
            act = rng.choice([0, 1, 2])
            c = dict(op=op, m=_log_int(rng, 1, 14400), k=_log_int(rng, 64, 4096), n=_log_int(rng, 32, 8194), x=rng.choice(["bf16", "f32"]),
                     act=act, bias=rng.random() < 0.7, residual=act == 0 and rng.random() < 0.4, out=rng.choice(["bf16", "f32"]))
            if c["residual"]:
                c["out"] = "f32"
        elif op == "cache":
            rows, smax = _log_int(rng, 1, 128), _log_int(rng, 64, 2048)
            tokens = _log_int(rng, 1, max(1, rows * smax // 2))
            c = dict(op=op, rows=rows, heads=rng.choice([4, 8, 16]), hd=rng.choice([64, 128]), smax=smax, tokens=tokens,
                     read=_log_int(rng, 1, tokens + 1), src=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
        else:
            group = rng.choice([1, 1, 2, 4, 8])
            heads = rng.choice([2, 4, 8, 16])
            beams = 3 if op == "decode" and rng.random() < 0.3 else 1
            rows = _log_int(rng, 1, 128 // beams) * beams
            longest = _log_int(rng, 1, 32749 if op == "decode" else 16301)
            out = rng.choice(["bf16", "bf16", "f32"])
            c = dict(op=op, rows=rows, heads=heads, group=group, hd=rng.choice([64, 128]), smax=longest + rng.randrange(64, 200),
                     longest=longest, q=rng.choice(["bf16", "f32"]), out=out, pad=rng.choice([0, 0, rng.randrange(0, 40)]))
            if op == "decode":
                c["beams"] = beams
            else:
                c["tokens"] = _log_int(rng, 1, 64)
                c["cache"] = "8" if out == "f32" else rng.choice(["8", "bf16"])
        w = work(c)
        cache = c["rows"] * c["heads"] * c["smax"] * c["hd"] if op != "linear" else 0
        scores = c["rows"] * c["heads"] * c["group"] * c["smax"] * c.get("tokens", 1) if op in ("decode", "tree") else 0
        if w["bytes"] <= top[op][0] and w["flops"] <= top[op][1] and cache <= 1.4e8 and scores <= 1.4e8:
            return c


# ---- inputs -------------------------------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _quantise(x):
    """Codes (uint8) and scale bytes of the blocks x [..., block]: the scale is the smallest power of two that brings
    the block's largest finite magnitude within e4m3's range."""
    x = x.float()
    good = torch.isfinite(x)
    top = torch.where(good, x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 9 + (m > 0.875), 0).clamp(min=-126)
    inv = ((127 - e).int() << 23).view(torch.float32)
    x = torch.where(good, x * inv[..., None], float("nan"))
    return x.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, scale):
    return codes.view(torch.float8_e4m3fn).float() * (scale.int() << 23).view(torch.float32)[..., None]


def _pad_k(x):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK))


def _quantise_rows(x):
    """x [M, K] -> codes [M, K up to a whole block], scale bytes [M, K / 128 up to a multiple of 4] (127 behind the last)."""
    x = _pad_k(x.float())
    codes, scale = _quantise(x.view(x.shape[0], -1, BLOCK))
    return codes.view(x.shape[0], -1), torch.nn.functional.pad(scale, (0, -scale.shape[1] % 4), value=127)


def _inputs(case, seed):
    """Everything a case is made of, before any operator: shared by prepare() and exact()."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c = case
    if c["op"] == "linear":
        # layer-normed activations with a few loud channels, weights at the usual 1/sqrt(K)
        x = _normal(g, c["m"], c["k"]) * (1 + 7 * (torch.rand(c["k"], generator=g, device="cuda") < 0.01))
        return dict(x=x.to(DTYPES[c["x"]]), w=_normal(g, c["n"], c["k"]) / math.sqrt(c["k"]),
                    bias=_normal(g, c["n"]) * 0.1 if c["bias"] else None,
                    residual=_normal(g, c["m"], c["n"]) if c["residual"] else None)
    rows, heads, hd, smax = c["rows"], c["heads"], c["hd"], c["smax"]
    loud = torch.exp(0.4 * _normal(g, 2, heads, 1, hd))
    if c["op"] == "cache":
        d = DTYPES[c["src"]]
        qkv = (_normal(g, c["tokens"], 3, heads, hd) * torch.cat([loud[:1], loud]).view(3, heads, hd)).to(d)  # a c_attn output row
        old = [_normal(g, rows, heads, smax, hd) * loud[i] for i in range(2)]
        slots = torch.randperm(rows * smax, generator=g, device="cuda")[: c["tokens"]]
        back = torch.cat([slots, torch.randint(rows * smax, (max(1, c["read"] // 8),), generator=g, device="cuda")])
        back = back[torch.randperm(back.numel(), generator=g, device="cuda")[: c["read"]]]
        return dict(qkv=qkv, old=old, row=(slots // smax).int(), pos=(slots % smax).int(), read_row=(back // smax).int(),
                    read_pos=(back % smax).int())
    tokens = c.get("tokens", 1)
    d = dict(k=_normal(g, rows, heads, smax, hd) * loud[0], v=_normal(g, rows, heads, smax, hd) * loud[1])
    q = _normal(g, rows, tokens, heads * c["group"], hd) * 1.5
    d["q"] = q.to(DTYPES[c["q"]])
    lens = (c["longest"] * (0.6 + 0.4 * torch.rand(rows, generator=g, device="cuda"))).int()
    lens[rows // 2] = c["longest"]
    d["len"] = lens
    d["pad"] = torch.minimum(torch.randint(c["pad"] + 1, (rows,), generator=g, device="cuda").int(), lens) if c["pad"] else None
    if c["op"] == "decode":
        if c["beams"] > 1:  # a key comes from some beam of the same utterance, a prompt's from the first; the newest from its own row
            first = torch.arange(rows, device="cuda") // c["beams"] * c["beams"]
            at = torch.arange(smax, device="cuda")[None]
            kv_rows = first[:, None] + torch.where(at < lens[:, None] // 3, 0, torch.randint(c["beams"], (rows, smax), generator=g, device="cuda"))
            d["kv_rows"] = torch.where(at == lens[:, None] - 1, torch.arange(rows, device="cuda")[:, None], kv_rows).int()
        else:
            d["kv_rows"] = None
        return d
    # a random tree: each drafted token's parent is an earlier one or the prefix's last token; bit j of a token's mask: j is
    # the token itself or an ancestor
    up = (torch.rand(rows, tokens, generator=g, device="cuda") * torch.arange(tokens, device="cuda")).long() - 1
    up = torch.where(torch.rand(rows, tokens, generator=g, device="cuda") < 0.6, torch.arange(tokens, device="cuda") - 1, up)
    up = up.clamp(min=-1)
    mask = torch.zeros(rows, tokens + 1, dtype=torch.int64, device="cuda")
    for t in range(tokens):
        mask[:, t] = mask.gather(1, up[:, t:t + 1] % (tokens + 1))[:, 0] | (1 << t if t < 63 else -(1 << 63))
    d["mask"] = mask[:, :tokens].contiguous()
    n = torch.randint(1, tokens + 1, (rows,), generator=g, device="cuda").int()
    n[rows // 2] = tokens
    d["n"] = n
    return d


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    s = dict(case=c)
    if c["op"] == "linear":
        s["x"], s["bias"], s["residual"] = d["x"], d["bias"], d["residual"]
        s["w"], s["w_scale"] = _quantise_rows(d["w"])
        if own:  # the layer a program keeps: it holds these very tensors
            s["layer"] = _package()[1].Fp8Linear(s["w"], s["w_scale"], c["k"], s["bias"])
        return s
    if c["op"] == "cache":
        (k, ks), (v, vs) = (_quantise(t) for t in d["old"])
        s.update({n: d[n] for n in ("qkv", "row", "pos", "read_row", "read_pos")})
    else:
        s.update({n: d.get(n) for n in ("q", "len", "pad", "kv_rows", "mask", "n")})
        if c.get("cache") == "bf16":
            k, v, ks, vs = d["k"].bfloat16(), d["v"].bfloat16(), None, None
        else:
            (k, ks), (v, vs) = _quantise(d["k"]), _quantise(d["v"])
        if c["op"] == "tree":  # rows of tokens that were not drafted stay as they are
            s["o"] = torch.zeros(*d["q"].shape, dtype=DTYPES[c["out"]], device="cuda")
    s.update(k=k, v=v, k_scale=ks, v_scale=vs)
    if own:  # the cache object a program keeps: it holds these very tensors
        kv8 = _package()[0]
        s["cache"] = kv8.Kv16Cache(k, v) if ks is None else kv8.Kv8Cache(k, v, ks, vs)
    return s


# ---- one pass -----------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    c = s["case"]
    if c["op"] == "linear":
        return s["layer"](s["x"], act=c["act"], residual=s["residual"], bf16_out=c["out"] == "bf16")
    if c["op"] == "cache":
        s["cache"].write(s["qkv"][:, 1], s["qkv"][:, 2], s["row"], s["pos"])
        return s["cache"].read(s["read_row"], s["read_pos"], dtype=DTYPES[c["out"]])
    if c["op"] == "decode":
        return s["cache"].decode(s["q"][:, 0], s["len"], pad=s["pad"], kv_rows=s["kv_rows"], max_len=c["longest"], dtype=DTYPES[c["out"]])
    return s["cache"].tree(s["q"], s["len"], s["mask"], n_tokens=s["n"], pad=s["pad"], max_len=c["longest"], out=s["o"])


def _plain(s):
    c = s["case"]
    if c["op"] == "linear":
        codes, scale = _quantise_rows(s["x"])
        x, w = (_values(q.view(q.shape[0], -1, BLOCK), e[:, : q.shape[1] // BLOCK]).view(q.shape) for q, e in ((codes, scale), (s["w"], s["w_scale"])))
        y = x @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"]
        if c["act"] == 1:
            y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
        elif c["act"] == 2:
            y = y / (1 + torch.exp(-y))
        if s["residual"] is not None:
            y = y + s["residual"]
        return y.to(DTYPES[c["out"]])
    if c["op"] == "cache":
        got = []
        for i, (codes, scale) in enumerate(((s["k"], s["k_scale"]), (s["v"], s["v_scale"]))):
            codes[s["row"].long(), :, s["pos"].long()], scale[s["row"].long(), :, s["pos"].long()] = _quantise(s["qkv"][:, 1 + i])
            at = s["read_row"].long(), slice(None), s["read_pos"].long()
            got.append(_values(codes[at], scale[at]).to(DTYPES[c["out"]]))
        return tuple(got)
    q = s["q"].float()
    rows, tokens, hq, hd = q.shape
    k, v = (s["k"].float(), s["v"].float()) if s["k_scale"] is None else (_values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"]))
    if s["kv_rows"] is not None:
        heads, smax = k.shape[1], k.shape[2]
        at = s["kv_rows"].long()[:, None, :], torch.arange(heads, device=k.device)[None, :, None], torch.arange(smax, device=k.device)[None, None, :]
        k, v = k[at], v[at]
    heads, smax = k.shape[1], k.shape[2]
    p = torch.arange(smax, device=k.device)
    seen = p[None] < s["len"][:, None]
    if s["pad"] is not None:
        seen &= p[None] >= s["pad"][:, None]
    seen = seen[:, None]  # [rows, tokens, smax]
    if s["mask"] is not None:
        j = p[None] - s["len"][:, None]
        inside = (j >= 0) & (j < s["n"][:, None])
        bit = (s["mask"][:, :, None] >> j.clamp(0, 63)[:, None].long()) & 1
        seen = seen | (inside[:, None] & (bit == 1))
    q = q.view(rows, tokens, heads, hq // heads, hd).permute(0, 2, 1, 3, 4).reshape(rows, heads, -1, hd)
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    x = x.view(rows, heads, tokens, -1, smax)
    seen = seen[:, None, :, None]
    x = torch.where(seen, x, -torch.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.where(seen, torch.exp(x - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(rows, heads, -1, smax), v).view(rows, heads, tokens, -1, hd) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(rows, tokens, hq, hd).to(DTYPES[c["out"]])
    if c["op"] == "decode":
        return o[:, 0]
    drafted = torch.arange(tokens, device=k.device)[None] < s["n"][:, None]
    s["o"].copy_(torch.where(drafted[:, :, None, None], o, s["o"]))
    return s["o"]


# ---- 64 bits ------------------------------------------------------------------------------------


def _rounded64(x):
    """What the blocks x [..., block] stand for once they are held in 8 bits, in float64."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / TOP)).clamp(min=-126))
    x = x / scale
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step * scale


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "linear":
        if c["m"] * c["k"] * c["n"] > 2e11:
            return None
        x, w = (_rounded64(_pad_k(t.double()).view(t.shape[0], -1, BLOCK)).view(t.shape[0], -1) for t in (d["x"], d["w"]))
        y = x @ w.t()
        if d["bias"] is not None:
            y += d["bias"].double()
        if c["act"] == 1:
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        elif c["act"] == 2:
            y = y * torch.sigmoid(y)
        return y if d["residual"] is None else y + d["residual"].double()
    if c["op"] == "cache":
        got = []
        for i in (0, 1):
            held = _rounded64(d["old"][i])
            held[d["row"].long(), :, d["pos"].long()] = _rounded64(d["qkv"][:, 1 + i])
            got.append(held[d["read_row"].long(), :, d["read_pos"].long()])
        return tuple(got)
    tokens, group, hd = c.get("tokens", 1), c["group"], c["hd"]
    o = torch.zeros(c["rows"], tokens, c["heads"] * group, hd, dtype=torch.float64, device="cuda")
    lens, pads = d["len"].tolist(), d["pad"].tolist() if d["pad"] is not None else [0] * c["rows"]
    counts = d["n"].tolist() if "n" in d else [0] * c["rows"]
    for b in range(c["rows"]):
        end = lens[b] + counts[b]
        if d.get("kv_rows") is not None:
            at = d["kv_rows"][b, :end].long(), slice(None), torch.arange(end, device="cuda")
            k, v = d["k"][at].transpose(0, 1), d["v"][at].transpose(0, 1)
        else:
            k, v = d["k"][b, :, :end], d["v"][b, :, :end]
        k, v = (k.bfloat16().double(), v.bfloat16().double()) if c.get("cache") == "bf16" else (_rounded64(k), _rounded64(v))
        hide = torch.zeros(tokens, end, dtype=torch.bool, device="cuda")
        hide[:, : pads[b]] = True
        if counts[b]:
            hide[:, lens[b]:] = (torch.bitwise_right_shift(d["mask"][b][:, None], torch.arange(counts[b], device="cuda")) & 1) == 0
        for h in range(c["heads"] * group):
            x = (d["q"][b, :, h].double() @ k[h // group].t()) * hd ** -0.5
            o[b, :, h] = torch.softmax(x.masked_fill(hide, -1e300), -1) @ v[h // group]
            o[b, :, h][hide.all(-1)] = 0
        if c["op"] == "tree":
            o[b, counts[b]:] = 0
    return o[:, 0] if c["op"] == "decode" else o


def work(case):
    c = case
    size = {"bf16": 2, "f32": 4}
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        blocks = -(-k // BLOCK)
        b = m * k * size[c["x"]] + n * (k + blocks) + m * n * (size[c["out"]] + (4 if c["residual"] else 0)) + (4 * n if c["bias"] else 0)
        return {"bytes": b, "flops": 2 * m * n * k}
    if c["op"] == "cache":
        per = 2 * c["heads"] * c["hd"]
        held = 2 * c["heads"] * (c["hd"] + 1)
        return {"bytes": c["tokens"] * (per * size[c["src"]] + held + 8) + c["read"] * (held + per * size[c["out"]] + 8), "flops": 2 * per * (c["tokens"] + c["read"])}
    tokens = c.get("tokens", 1)
    drafted = tokens * 0.5 if c["op"] == "tree" else 0
    keys = c["rows"] * (0.8 * c["longest"] + drafted)  # lengths spread over 0.6 .. 1 of the longest
    per = 2 * c["heads"] * (c["hd"] * 2 if c.get("cache") == "bf16" else c["hd"] + 1)
    hq = c["heads"] * c["group"]
    b = keys * per + c["rows"] * tokens * hq * c["hd"] * (size[c["q"]] + size[c["out"]])
    return {"bytes": b, "flops": 4 * keys * max(1.0, drafted) * hq * c["hd"]}
