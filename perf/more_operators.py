"""Operators of a decoding step over an 8-bit KV cache, as cases to be timed.

A serving program with long contexts keeps keys and values in e4m3 with one scale per token and key
head: prompts and accepted drafts are quantised as they are written ("write"), decode and
verification steps attend to the 8-bit cache ("attention"), and a sequence is read back in 16 bits
for programs that know no 8-bit cache ("read").  Between the attention and the next block the output
is normalised, gated, added to the scaled residual stream and normalised again ("norm").

Each case is a dict of plain values.  `prepare` makes what a serving program holds before the call
on the GPU from the seed, `run` is one pass (elementary torch operations, or with `own` the
package's entry points), `work` the bytes and operations that a pass cannot do without, `exact`
the outputs in 64 bits.
"""
import math

import torch

own = False

BLK = 128                # values of a row that share a scale (norm)
E4M3 = 448.0             # the largest e4m3 value
TINY = 2.0 ** -100       # the smallest maximum that a scale is made for
F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One chat stream, one new token, a short cache: where latency is all there is.
        dict(name="attn8_one_token", kind="attention", B=1, N=1, Hq=32, Hkv=8, D=128, L=1000,
             ragged=False, page=0, mask="causal", dtype="bf16"),
        # A serving batch's decode step: one token of each sequence, ragged lengths, pages of 64.
        dict(name="attn8_decode_batch", kind="attention", B=64, N=1, Hq=32, Hkv=8, D=128, L=16384,
             ragged=True, page=64, mask="causal", dtype="bf16"),
        # A serving batch's draft trees of 16 nodes, ragged lengths, pages of 64.
        dict(name="attn8_tree_batch", kind="attention", B=24, N=16, Hq=32, Hkv=8, D=128, L=16384,
             ragged=True, page=64, mask="tree", dtype="bf16"),
        # Wide heads, few of them, a chain of drafts, small pages, fp16.
        dict(name="attn8_d256_chain", kind="attention", B=8, N=8, Hq=8, Hkv=4, D=256, L=5000,
             ragged=True, page=16, mask="causal", dtype="f16"),
        # Long documents: 128k cached tokens a sequence and a full tree of 33 nodes.
        dict(name="attn8_long", kind="attention", B=4, N=33, Hq=32, Hkv=8, D=128, L=131072,
             ragged=False, page=0, mask="tree", dtype="bf16"),
        # The accepted path of one tree into the cache of every layer.
        dict(name="write8_path", kind="write", layers=32, B=1, N=16, most=5, path=True, Hkv=8, D=128,
             page=0, cap=2048, dtype="bf16"),
        # Prompts of a batch into one layer's pages, as the layer has computed their keys and values.
        dict(name="write8_prompts", kind="write", layers=1, B=8, N=4096, most=4096, path=False, Hkv=8,
             D=128, page=64, cap=64, dtype="bf16"),
        # Sequences of a batch back in 16 bits, from pages of 64, for one layer.
        dict(name="read8_batch", kind="read", layers=1, B=16, Hkv=8, D=128, L=8192, ragged=True, page=64,
             dtype="bf16"),
        # One short sequence back in 16 bits, in every layer.
        dict(name="read8_one", kind="read", layers=32, B=1, Hkv=8, D=128, L=300, ragged=False, page=16,
             dtype="f16"),
        # Between two blocks of a tree step, to 8 bits.
        dict(name="sandwich_step_8bit", kind="norm", B=16, H=4096, post=True, gate="none", rs=1.0, bits8=True,
             offset=1.0, dtype="bf16"),
        # Between two blocks of a prompt chunk, a gate per channel, width no power of two.
        dict(name="sandwich_prompt", kind="norm", B=8000, H=5760, post=True, gate="channel", rs=0.5,
             bits8=False, offset=0.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "write", "write", "read", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([0, 16, 64, 256, rng.randint(1, 100)])
    if kind == "attention":
        D = rng.choice([64, 128, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8])
        G = rng.choice([1, 2, 4, 8])
        B = _log(rng, 1, 64)
        most = min(131072, (1 << 29) // (B * Hkv * D))
        return dict(kind="attention", B=B, N=rng.choice([1, 1, 1, rng.randint(2, 33), rng.randint(2, 64)]),
                    Hq=Hkv * G, Hkv=Hkv, D=D, L=_log(rng, 1, most), ragged=rng.random() < 0.6,
                    page=page, mask=rng.choice(["tree", "tree", "causal"]), dtype=dtype)
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
    if kind == "write":
        if rng.random() < 0.5:
            N = rng.randint(1, 64)
            return dict(kind="write", layers=_log(rng, 1, 48), B=_log(rng, 1, 64), N=N, most=rng.randint(1, min(N, 12)),
                        path=True, Hkv=Hkv, D=D, page=page, cap=_log(rng, 64, 256), dtype=dtype)
        B, N = _log(rng, 1, 32), _log(rng, 1, 8192)
        return dict(kind="write", layers=1, B=min(B, max(1, 32768 // N)), N=N, most=N, path=False, Hkv=Hkv, D=D,
                    page=page, cap=_log(rng, 1, 4096), dtype=dtype)
    if kind == "read":
        B, layers = _log(rng, 1, 32), rng.choice([1, 1, rng.randint(2, 32)])
        most = max(1, min(32768, (1 << 27) // (B * layers * Hkv * D)))
        return dict(kind="read", layers=layers, B=B, Hkv=Hkv, D=D, L=_log(rng, 1, most), ragged=rng.random() < 0.6,
                    page=page, dtype=dtype)
    H = 8 * _log(rng, 8, 2048)
    return dict(kind="norm", B=_log(rng, 1, min(16384, (1 << 25) // H)), H=H, post=rng.random() < 0.8,
                gate=rng.choice(["none", "number", "channel", "token"]), rs=rng.choice([1.0, 0.5, rng.uniform(0.1, 2.0)]),
                bits8=rng.random() < 0.6, offset=rng.choice([0.0, 1.0]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _spread(n, most, ragged):
    """n lengths: all of them `most`, or from a few tokens up to it."""
    return [max(1, int(most * ((i + 1) / n) ** 2)) if ragged else most for i in range(n)]


def _tree(g, B, N):
    """Ancestor-or-self masks [B, N, N] of random trees: node i's parent is an earlier node."""
    u = torch.rand((B, N), generator=g, device="cuda")
    parent = (u * torch.arange(N, device="cuda")).long()     # node 0: itself
    mask = torch.eye(N, dtype=torch.bool, device="cuda").repeat(B, 1, 1)
    rows = torch.arange(B, device="cuda")
    for i in range(1, N):
        mask[:, i] |= mask[rows, parent[:, i]]
    return mask


def _quantize(x):
    """e4m3 values and their scale per row [..., D] of 32-bit values."""
    # 448 x / max rather than x / scale: ties of the 8-bit rounding stay ties (448 x is exact for
    # 16-bit x, and the quotient is rounded once)
    top = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return (x * E4M3 / top).to(F8), (top / E4M3)[..., 0]


def _cache8(c, g, S):
    """An 8-bit cache for B sequences of S tokens, the values of a head together, token after token:
    values [layers, B, S, Hkv, D] and scales [layers, B, S, Hkv], or pages of them in any order with
    their table [B, blocks] and a few pages that belong to nobody."""
    B, Hkv, D, layers = c["B"], c["Hkv"], c["D"], c.get("layers", 1)
    if c["page"]:
        nblk = -(-S // c["page"])
        pages = torch.randperm(B * nblk + 3, generator=g, device="cuda")[:B * nblk]
        rows, page, table = B * nblk + 3, c["page"], pages.view(B, nblk).to(torch.int32)
    else:
        rows, page, table = B, S, None
    wide = torch.exp(0.5 * _normal(g, Hkv, 1, D))            # channels of unlike size, as trained models have
    out = []
    for w in (wide, 1.0):
        q = torch.empty((layers, rows, Hkv, page, D), dtype=F8, device="cuda")
        s = torch.empty((layers, rows, Hkv, page), device="cuda")
        for i in range(layers):
            v, s[i] = _quantize(_normal(g, rows, Hkv, page, D) * w)
            q[i].view(torch.uint8).copy_(v.view(torch.uint8))
        out += [q.transpose(2, 3), s.transpose(2, 3)]
    return out, table


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind, dt = c["kind"], TYPES[c["dtype"]]
    s = dict(kind=kind)
    if kind == "norm":
        B, H = c["B"], c["H"]
        wide = torch.exp(0.5 * _normal(g, H))
        s.update(x=(_normal(g, B, H) * wide).to(dt), residual=(3.0 * _normal(g, B, H) * wide).to(dt),
                 post=(1.0 - c["offset"] + 0.2 * _normal(g, H)).to(dt) if c["post"] else None,
                 pre=(1.0 - c["offset"] + 0.2 * _normal(g, H)).to(dt),
                 gate={"none": lambda: None, "number": lambda: 0.375, "channel": lambda: torch.tanh(_normal(g, H)).to(dt),
                       "token": lambda: torch.tanh(_normal(g, B, H)).to(dt)}[c["gate"]](),
                 rs=c["rs"], eps=1e-5, offset=c["offset"], bits8=c["bits8"])
        return s
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if kind == "attention":
        N, lens = c["N"], _spread(B, c["L"], c["ragged"])
        (kq, ks, vq, vs), s["table"] = _cache8(c, g, max(lens) + N)
        s.update(kq=kq[0], ks=ks[0], vq=vq[0], vs=vs[0], q=2.0 * _normal(g, B, N, c["Hq"], D, dtype=dt),
                 k=_normal(g, B, N, Hkv, D, dtype=dt), v=_normal(g, B, N, Hkv, D, dtype=dt),
                 lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 mask=_tree(g, B, N) if c["mask"] == "tree" else None)
        return s
    if kind == "read":
        lens = _spread(B, c["L"], c["ragged"])
        (s["kq"], s["ks"], s["vq"], s["vs"]), s["table"] = _cache8(c, g, c["L"])
        s.update(lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), L=c["L"], dtype=dt)
        return s
    N, most, layers = c["N"], c["most"], c["layers"]
    (s["kq"], s["ks"], s["vq"], s["vs"]), s["table"] = _cache8(c, g, c["cap"] + most)
    nodes = None
    if c["path"]:
        nodes = torch.rand((B, N), generator=g, device="cuda").argsort(1)[:, :most].sort(1).values.to(torch.int32)
    s.update(k=_normal(g, layers, B, N, Hkv, D, dtype=dt), v=_normal(g, layers, B, N, Hkv, D, dtype=dt), nodes=nodes,
             counts=torch.tensor(_spread(B, most, True), dtype=torch.int32, device="cuda"),
             lens=torch.randint(0, c["cap"], (B,), generator=g, device="cuda").to(torch.int32))
    return s


# ------------------------------------------------------------------ plain forms


def _plain_norm(s):
    dt = s["x"].dtype

    def rms(h, w):
        # the mean of squares in 64 bits: a last-bit change of the factor moves 8-bit roundings
        ms = h.double().square().mean(1, keepdim=True)
        return h * (1.0 / torch.sqrt(ms + s["eps"])).float() * (w.float() + s["offset"])
    h = s["x"].float()
    if s["post"] is not None:
        h = rms(h, s["post"])
    if s["gate"] is not None:
        h = h * (s["gate"].float() if torch.is_tensor(s["gate"]) else s["gate"])
    r = (s["residual"].float() * s["rs"] + h).to(dt)
    y = rms(r.float(), s["pre"])
    if not s["bits8"]:
        return [y.to(dt), r]
    B, H = y.shape
    n = -(-H // BLK)
    q, scale = _quantize(torch.nn.functional.pad(y, (0, n * BLK - H)).view(B, n, BLK))
    return [q.view(B, -1)[:, :H].contiguous(), scale, r]


def _rows(values, scales, table, S):
    """[..., B, S, Hkv, D] in 32 bits of an 8-bit cache: its own rows, or its pages in the table's order."""
    bits = values.view(torch.uint8)
    if table is not None:
        t = table.long()
        bits, scales = bits[..., t, :, :, :].flatten(-4, -3), scales[..., t, :, :].flatten(-3, -2)
    bits, scales = bits[..., :S, :, :], scales[..., :S, :]
    return bits.contiguous().view(F8).float() * scales[..., None]


def _plain_read(s):
    keep = torch.arange(s["L"], device=s["lens"].device) < s["lens"][:, None]
    out = []
    for a, b in (("kq", "ks"), ("vq", "vs")):
        x = _rows(s[a], s[b], s["table"], s["L"])
        out.append(x.masked_fill(~keep[:, :, None, None], 0.0).to(s["dtype"]))
    return out


def _plain_attention(s):
    q, lens, mask = s["q"], s["lens"], s["mask"]
    B, N, Hq, D = q.shape
    Hkv = s["k"].shape[2]
    S = s["kq"].shape[1] if s["table"] is None else s["table"].shape[1] * s["kq"].shape[1]
    if mask is None:
        mask = torch.ones(N, N, dtype=torch.bool, device=q.device).tril().expand(B, N, N)
    seen = torch.arange(S, device=q.device) < lens[:, None]
    seen = torch.cat((seen[:, None].expand(B, N, S), mask), 2)
    k = torch.cat((_rows(s["kq"], s["ks"], s["table"], S), s["k"].float()), 1).permute(0, 2, 1, 3)
    v = torch.cat((_rows(s["vq"], s["vs"], s["table"], S), s["v"].float()), 1).permute(0, 2, 1, 3)
    x = q.float().view(B, N, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    t = torch.matmul(x, k.transpose(2, 3)).mul_(D ** -0.5).view(B, Hkv, Hq // Hkv, N, S + N)
    t = t.masked_fill_(~seen[:, None, None], -math.inf)
    t = t.sub_(t.amax(4, keepdim=True)).exp_()
    t = t.div_(t.sum(4, keepdim=True))
    o = torch.matmul(t.view(B, Hkv, -1, S + N), v)
    return o.view(B, Hkv, Hq // Hkv, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D).to(q.dtype)


def _plain_write(s):
    lens, counts, table = s["lens"], s["counts"], s["table"]
    B, page_size = len(counts), s["kq"].shape[2]
    places = s["k"].shape[2] if s["nodes"] is None else s["nodes"].shape[1]
    j = torch.arange(places, device=lens.device)
    keep = j < counts[:, None]
    b = torch.arange(B, device=lens.device)[:, None].expand(B, places)[keep]
    node = (j.expand(B, places) if s["nodes"] is None else s["nodes"])[keep].long()
    at = (lens[:, None] + j)[keep].long()
    page, off = (b, at) if table is None else (table[b, at // page_size].long(), at % page_size)
    for x, values, scales in ((s["k"], s["kq"], s["ks"]), (s["v"], s["vq"], s["vs"])):
        q, scale = _quantize(x[:, b, node].float())
        values.view(torch.uint8)[:, page, off] = q.view(torch.uint8)
        scales[:, page, off] = scale
    return [s["kq"], s["ks"], s["vq"], s["vs"], lens + counts]


def run(s):
    kind = s["kind"]
    if own:
        return _own(s)
    if kind == "norm":
        return _plain_norm(s)
    if kind == "attention":
        return _plain_attention(s)
    return _plain_read(s) if kind == "read" else _plain_write(s)


def _own(s):
    import llima_amd
    kind = s["kind"]
    if kind == "norm":
        y, r = llima_amd.sandwich_norm(s["x"], s["post"], s["residual"], s["pre"], gate=s["gate"],
                                       residual_scale=s["rs"], eps=s["eps"], weight_offset=s["offset"],
                                       out="fp8" if s["bits8"] else "same")
        return [y.values, y.scales, r] if s["bits8"] else [y, r]
    kc, vc = llima_amd.Fp8Cache(s["kq"], s["ks"]), llima_amd.Fp8Cache(s["vq"], s["vs"])
    if kind == "attention":
        return llima_amd.tree_attention(s["q"], s["k"], s["v"], kc, vc, s["lens"], tree_mask=s["mask"],
                                        block_table=s["table"])
    if kind == "read":
        return list(llima_amd.cache_read(kc, vc, s["lens"], block_table=s["table"], dtype=s["dtype"], tokens=s["L"]))
    if s["nodes"] is not None:
        lens = llima_amd.tree_commit(s["k"], s["v"], s["nodes"], s["counts"], kc, vc, s["lens"], block_table=s["table"])
    else:
        lens = llima_amd.cache_write(s["k"], s["v"], kc, vc, s["lens"], counts=s["counts"], block_table=s["table"])
    return [s["kq"], s["ks"], s["vq"], s["vs"], lens]


def work(case):
    c, kind = case, case["kind"]
    if kind == "norm":
        n, e = c["B"] * c["H"], 4 if c["dtype"] == "f32" else 2
        b = n * e * 3 + c["H"] * e * (2 if c["post"] else 1)
        b += c["H"] * e if c["gate"] == "channel" else n * e if c["gate"] == "token" else 0
        b += n + 4 * c["B"] * -(-c["H"] // BLK) if c["bits8"] else n * e
        return dict(bytes=b, flops=10 * n)
    Hkv, D, B = c["Hkv"], c["D"], c["B"]
    if kind == "write":
        rows = c["layers"] * sum(_spread(B, c["most"], True)) * Hkv * 2
        return dict(bytes=rows * (3 * D + 4) + 12 * B, flops=2 * rows * D)
    tokens = sum(_spread(B, c["L"], c["ragged"]))
    if kind == "read":
        return dict(bytes=2 * c["layers"] * Hkv * (tokens * (D + 4) + 2 * B * c["L"] * D) + 4 * B, flops=2 * c["layers"] * tokens * Hkv * D)
    N, Hq = c["N"], c["Hq"]
    b = 2 * tokens * Hkv * (D + 4) + 4 * B * N * (Hkv + Hq) * D + (B * N * N if c["mask"] == "tree" else 0) + 4 * B
    return dict(bytes=b, flops=4 * (tokens + B * N) * N * Hq * D)


# ------------------------------------------------------------------ 64 bits


def _exact_rows(x):
    """The maximum over 448 along the last dimension, and the e4m3 values of the quotients."""
    top = x.abs().max(-1).values
    top = torch.where(top < TINY, torch.full_like(top, TINY), top)
    return (x / top[..., None] * E4M3).float().to(F8).double(), top / E4M3


def _exact_norm(s):
    dt, off = s["x"].dtype, s["offset"]
    h = s["x"].double()
    H = h.shape[1]
    if s["post"] is not None:
        h = h / torch.sqrt((h * h).sum(1, keepdim=True) / H + s["eps"]) * (s["post"].double() + off)
    if s["gate"] is not None:
        h = h * s["gate"]
    r = s["rs"] * s["residual"].double() + h
    z = r.to(dt).double()                                    # the stream is kept in its type
    y = z / torch.sqrt((z * z).sum(1, keepdim=True) / H + s["eps"]) * (s["pre"].double() + off)
    if not s["bits8"]:
        return [y, r]
    parts = [_exact_rows(y[:, i:i + BLK]) for i in range(0, H, BLK)]
    return [torch.cat([p[0] for p in parts], 1), torch.stack([p[1] for p in parts], 1), r]


def _exact_keys(values, scales, table, b, n):
    """The first n tokens of sequence b of one layer's cache, [n, Hkv, D]."""
    v, s = values.view(torch.uint8), scales
    if table is None:
        v, s = v[b, :n], s[b, :n]
    else:
        t = table[b].long()
        v, s = v[t].flatten(0, 1)[:n], s[t].flatten(0, 1)[:n]
    return v.contiguous().view(F8).double() * s[..., None].double()


def _exact_attention(s):
    q = s["q"].double()
    B, N, Hq, D = q.shape
    G = Hq // s["k"].shape[2]
    out = torch.empty_like(q)
    for b, n in enumerate(s["lens"].tolist()):               # one sequence after the other, its own keys alone
        k = torch.cat((_exact_keys(s["kq"], s["ks"], s["table"], b, n), s["k"][b].double()))
        v = torch.cat((_exact_keys(s["vq"], s["vs"], s["table"], b, n), s["v"][b].double()))
        mask = torch.ones(N, n + N, dtype=torch.bool, device=q.device)
        mask[:, n:] = s["mask"][b] if s["mask"] is not None else torch.ones_like(mask[:, n:]).tril()
        for h in range(Hq):
            t = (q[b, :, h] @ k[:, h // G].t() / math.sqrt(D)).masked_fill(~mask, -math.inf)
            out[b, :, h] = torch.softmax(t, 1) @ v[:, h // G]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _exact_norm(s)
    if kind == "attention":
        return _exact_attention(s)
    lens = s["lens"].tolist()
    if kind == "read":
        layers, L = case["layers"], case["L"]
        out = [torch.zeros(layers, case["B"], L, case["Hkv"], case["D"], dtype=torch.float64, device="cuda") for _ in range(2)]
        for o, a, b in ((out[0], "kq", "ks"), (out[1], "vq", "vs")):
            for i in range(layers):
                for at, n in enumerate(lens):
                    o[i, at, :n] = _exact_keys(s[a][i], s[b][i], s["table"], at, n)
        return out
    out = []
    for a, values, scales in ((s["k"], s["kq"], s["ks"]), (s["v"], s["vq"], s["vs"])):
        v, f = values.double(), scales.double()
        q, top = _exact_rows(a.double())
        for b, n in enumerate(s["counts"].tolist()):
            src = torch.arange(n, device="cuda") if s["nodes"] is None else s["nodes"][b, :n].long()
            at = lens[b] + torch.arange(n, device="cuda")
            if s["table"] is None:
                v[:, b, at], f[:, b, at] = q[:, b, src], top[:, b, src]
            else:
                page, off = s["table"][b].long()[at // case["page"]], at % case["page"]
                v[:, page, off], f[:, page, off] = q[:, b, src], top[:, b, src]
        out += [v, f]
    return out + [None]
