"""The operators of MLA attention over a paged latent cache, each in its plain
form (elementary torch operations in 32 bits, rounded once at the end) and as
the library's call, over the sizes that decoding and prompts meet:

    rope    rotary positions on part of each head (interleaved or half layout,
            YaRN frequencies for long contexts)
    write   new tokens' rows into the paged cache: RMSNorm of the latent part,
            rotary positions on the rest, 16-bit or 8-bit storage
    read    cache rows back, gathered through the page table
    attend  absorbed attention of one or several drafted tokens per sequence
            (a tree given by a bit mask, or a causal chain) over the cache

A cache row is `latent` values and 64 rotary values.  The 16-bit formats hold
them one after the other.  The 8-bit formats hold the latent values as e4m3
with one power-of-two scale for every 32 (the exponent plus 127 in a byte, at
the end of the row) and the rotary values in 16 bits; rows are padded to 16
bytes.
"""
import math

import torch

own = False

ROPE = 64                    # rotary values of a cache row
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = {"f16": torch.float16, "bf16": torch.bfloat16, "fp8_f16": torch.float16, "fp8_bf16": torch.bfloat16}


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the rotary part of one decoded token's 128 query heads, from the 32-bit projections
        dict(name="rope_token", op="rope", tokens=1, heads=128, head_dim=64, offset=0, dim=64, half=False, yarn=40.0,
             type="f32", to="bf16"),
        # a prompt chunk: whole heads of 128 + 64, the last 64 rotated, positions far into a long context
        dict(name="rope_prompt", op="rope", tokens=4096, heads=128, head_dim=192, offset=128, dim=64, half=False,
             yarn=40.0, type="bf16", to="bf16"),
        # another layout: half rotation, an odd number of tokens and heads, no scaling
        dict(name="rope_half_odd", op="rope", tokens=777, heads=17, head_dim=80, offset=0, dim=80, half=True, yarn=1.0,
             type="f16", to="f16"),
        # one decoded token into an 8-bit cache
        dict(name="write_token", op="write", seqs=1, tokens=1, latent=512, fmt="fp8_bf16", page=64, type="f32"),
        # a decode step of a batch into a 16-bit cache
        dict(name="write_batch", op="write", seqs=48, tokens=1, latent=512, fmt="bf16", page=64, type="bf16"),
        # two long prompts into an 8-bit cache, pages that end inside
        dict(name="write_prompt", op="write", seqs=2, tokens=16381, latent=512, fmt="fp8_bf16", page=64, type="f32"),
        # a short context back in 16 bits
        dict(name="read_short", op="read", seqs=1, tokens=700, latent=512, fmt="fp8_f16", page=16, type="f16"),
        # the contexts of a batch
        dict(name="read_batch", op="read", seqs=16, tokens=8192, latent=512, fmt="fp8_bf16", page=64, type="bf16"),
        # one token, a short context: latency
        dict(name="attend_token", op="attend", seqs=1, tokens=1, heads=128, ctx=900, latent=512, fmt="bf16", page=64,
             tree=False),
        # a decode step of a batch
        dict(name="attend_batch", op="attend", seqs=32, tokens=1, heads=128, ctx=8192, latent=512, fmt="bf16", page=64,
             tree=False),
        # trees of up to 13 drafted tokens over an 8-bit cache
        dict(name="attend_tree", op="attend", seqs=8, tokens=13, heads=128, ctx=16384, latent=512, fmt="fp8_bf16",
             page=64, tree=True),
        # a long context, 16 heads (a shard of the heads), a small tree
        dict(name="attend_long", op="attend", seqs=1, tokens=5, heads=16, ctx=131072, latent=512, fmt="f16", page=32,
             tree=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        heads = rng.choice([1, 7, 16, 17, 40, 64, 128])
        dim = rng.choice([32, 64, 80, 128])
        offset = rng.choice([0, 64, 128])
        tokens = _spread(rng, 1, max(1, 4096 * 128 * 192 // (heads * (offset + dim))) if heads > 16 else 4096)
        kind, to = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
        return dict(op=op, tokens=min(tokens, 4096), heads=heads, head_dim=offset + dim, offset=offset, dim=dim,
                    half=rng.random() < 0.5, yarn=rng.choice([1.0, 4.0, 40.0]), type=kind, to=to)
    latent = rng.choice([128, 256, 384, 512, 512, 512])
    fmt = rng.choice(sorted(FORMATS))
    if op in ("write", "read"):
        seqs = _spread(rng, 1, 64)
        kind = rng.choice(["f32", fmt.split("_")[-1]])
        return dict(op=op, seqs=seqs, tokens=_spread(rng, 1, 32000 // seqs), latent=latent, fmt=fmt, page=page,
                    type=kind)
    heads = rng.choice([1, 5, 16, 32, 64, 128])
    tokens = rng.choice([1, 1, 2, 4, 7, 16])
    seqs = _spread(rng, 1, 32)
    most = min(131072, 8 * 13 * 128 * 16384 // (seqs * tokens * max(heads, 32)), 32 * 8192 // seqs)
    return dict(op=op, seqs=seqs, tokens=tokens, heads=heads, ctx=_spread(rng, 1, most), latent=latent, fmt=fmt,
                page=page, tree=tokens > 1 and rng.random() < 0.7)


def _row_bytes(latent, fmt):
    if fmt.startswith("fp8"):
        return (latent + 2 * ROPE + latent // 32 + 15) // 16 * 16
    return 2 * (latent + ROPE)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return dict(bytes=n * case["head_dim"] * (size[case["type"]] + size[case["to"]]) + 4 * case["tokens"],
                    flops=3 * n * case["dim"])
    lens = _lengths(case)
    row, width = _row_bytes(case["latent"], case["fmt"]), case["latent"] + ROPE
    rows = sum(n for _, n in lens)
    if case["op"] in ("write", "read"):
        return dict(bytes=rows * (width * size[case["type"]] + row), flops=6 * rows * width)
    h = case["heads"]
    scored = sum(h * n * (c + n) for c, n in lens)
    return dict(bytes=sum(c + n for c, n in lens) * row + rows * h * (2 * (width + case["latent"]) + 4),
                flops=2 * scored * (width + case["latent"]))


# ------------------------------------------------------------------ the inputs
def _lengths(case):
    """(rows in the cache before the call, rows or tokens of the call) of each sequence: ragged, the first one full."""
    out = []
    for b in range(case["seqs"]):
        n = case["tokens"] if b == 0 else case["tokens"] - (b * 5) % max(1, case["tokens"] // 3 + 1)
        if case["op"] == "attend":
            out.append((case["ctx"] - (b * 911) % (case["ctx"] // 4 + 1), n))
        else:
            out.append(((b * 37 + 5) % case["page"], n))
    return out


def _ancestors(n, gen):
    """Bit masks of a random tree: token i sees its ancestors and itself."""
    rows = []
    parents = [-1] + [int(torch.randint(-1, i, (1,), generator=gen)) for i in range(1, n)]
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return rows


def _yarn(dim, theta, factor, orig, fast=32.0, slow=1.0):
    """Frequencies of the pairs: theta^(-2i/dim), those of long wavelengths divided by `factor`, a ramp between."""
    lo = math.floor(dim * math.log(orig / (fast * 2 * math.pi)) / (2 * math.log(theta)))
    hi = math.ceil(dim * math.log(orig / (slow * 2 * math.pi)) / (2 * math.log(theta)))
    lo, hi = max(lo, 0), min(hi, dim // 2 - 1)
    hi = max(hi, lo + 1)
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = theta ** (-2 * i / dim)
    ramp = ((i - lo) / (hi - lo)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp)


THETA, ORIG_CTX = 10000.0, 4096.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = {"case": case}
    if case["op"] == "rope":
        t = case["tokens"]
        s["x"] = randn(t, case["heads"], case["head_dim"]).to(TYPES[case["type"]])
        s["pos"] = (torch.randint(0, 160000 - t, (1,), generator=host).item() + torch.arange(t)).to(dev, torch.int32)
        s["freq"] = _yarn(case["dim"], THETA, case["yarn"], ORIG_CTX).to(dev)
    else:
        lens = _lengths(case)
        latent, page, fmt = case["latent"], case["page"], case["fmt"]
        per_seq = max(-(-(c + n) // page) for c, n in lens)
        used = sum(-(-(c + n) // page) for c, n in lens)
        n_pages = used + 3
        order = torch.randperm(n_pages, generator=host).tolist()
        table, at = torch.zeros(case["seqs"], per_seq, dtype=torch.int32), 0
        for b, (c, n) in enumerate(lens):
            k = -(-(c + n) // page)
            table[b, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
            at += k
        counts = torch.tensor([n for _, n in lens])
        starts = torch.zeros(case["seqs"] + 1, dtype=torch.int32)
        starts[1:] = counts.cumsum(0)
        total = int(starts[-1])
        s.update(table=table.to(dev), q_start=starts.to(dev), ctx=torch.tensor([c for c, _ in lens], dtype=torch.int32).to(dev),
                 n_tokens=total, n_pages=n_pages, per_seq=per_seq, longest=max(c + n for c, n in lens),
                 most=max(n for _, n in lens))
        # where token t of the call sits: its sequence and its number there
        s["seq_of"] = torch.repeat_interleave(torch.arange(case["seqs"]), counts).to(dev)
        s["nth"] = (torch.arange(total) - starts[:-1].long()[s["seq_of"].cpu()]).to(dev)
        if case["op"] == "write":
            s["kv"] = (randn(total, latent + ROPE) * 3).to(TYPES[case["type"]])
            s["norm"] = 1 + 0.2 * randn(latent)
            # rotary positions of a far part of a long context
            s["pos"] = (s["nth"] + torch.randint(0, 100000, (1,), generator=host).item()).to(torch.int32)
            s["freq"] = _yarn(ROPE, THETA, 40.0, ORIG_CTX).to(dev)
            s["cache"] = torch.zeros(n_pages, page, _row_bytes(latent, fmt), dtype=torch.uint8, device=dev)
        else:
            rows = n_pages * page
            s["cache"] = _pack(randn(rows, latent), randn(rows, ROPE), fmt).view(n_pages, page, -1)
        if case["op"] == "attend":
            h, t = case["heads"], FORMATS[fmt]
            s["q_latent"], s["q_rope"] = randn(total, h, latent).to(t), randn(total, h, ROPE).to(t)
            s["scale"] = (0.1 * math.log(40.0) + 1) ** 2 / math.sqrt(192)
            words = -(-s["most"] // 32)
            bits = [m for _, n in lens for m in (_ancestors(n, host) if case["tree"] else [(2 << i) - 1 for i in range(n)])]
            # sees[t, j]: whether token t sees token j of its sequence
            s["sees"] = torch.tensor([[m >> j & 1 for j in range(s["most"])] for m in bits], dtype=torch.bool).to(dev)
            packed = [[(m >> 32 * w) & 0xFFFFFFFF for w in range(words)] for m in bits]
            s["tree"] = torch.tensor(packed, dtype=torch.int64).to(torch.uint32).view(torch.int32).to(dev)
    if own:
        _handles(s)
    return s


# -------------------------------------------------------------- the plain forms
def _pack(latent, rope, fmt):
    """Cache rows (bytes) of 32-bit latent and rotary values."""
    t = FORMATS[fmt]
    if not fmt.startswith("fp8"):
        return torch.cat([latent, rope], -1).to(t).contiguous().view(torch.uint8)
    n = latent.shape[-1]
    groups = latent.view(-1, n // 32, 32)
    mant, expo = torch.frexp(groups.abs().amax(-1))          # amax = mant * 2^expo, mant in [1/2, 1)
    k = (expo - 9 + (mant > 0.875)).clamp(-15, 7)            # the least k with amax <= 448 * 2^k
    k = torch.where(mant == 0, torch.full_like(k, -15), k)
    codes = (torch.ldexp(groups, -k[..., None])).clamp(-448, 448).to(torch.float8_e4m3fn)
    row = torch.zeros(latent.shape[0], _row_bytes(n, fmt), dtype=torch.uint8, device=latent.device)
    row[:, :n] = codes.view(torch.uint8).view(-1, n)
    row[:, n:n + 2 * ROPE] = rope.to(t).contiguous().view(torch.uint8)
    row[:, n + 2 * ROPE:n + 2 * ROPE + n // 32] = (k + 127).to(torch.uint8)
    return row


def _unpack(rows, latent, fmt):
    """The 32-bit values that cache rows (bytes, last axis) stand for."""
    t = FORMATS[fmt]
    if not fmt.startswith("fp8"):
        return rows.view(t).float()
    k = rows[..., latent + 2 * ROPE:latent + 2 * ROPE + latent // 32].float() - 127
    codes = rows[..., :latent].contiguous().view(torch.float8_e4m3fn).float()
    values = codes.view(*codes.shape[:-1], latent // 32, 32) * torch.exp2(k)[..., None]
    rope = rows[..., latent:latent + 2 * ROPE].contiguous().view(t).float()
    return torch.cat([values.view(codes.shape), rope], -1)


def _rotate(x, pos, freq, half):
    """x [..., dim] rotated by pos (of x's first axis) times freq."""
    turn = pos.double()[:, None] * freq
    shape = (pos.shape[0],) + (1,) * (x.dim() - 2) + (freq.shape[0],)
    cos, sin = torch.cos(turn).float().view(shape), torch.sin(turn).float().view(shape)
    a, b = (x[..., :freq.shape[0]], x[..., freq.shape[0]:]) if half else (x[..., 0::2], x[..., 1::2])
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.cat([u, v], -1) if half else torch.stack([u, v], -1).flatten(-2)


def _place(s, seq, row):
    """(page, row in the page) of rows `row` of sequences `seq`."""
    page = s["case"]["page"]
    return s["table"][seq, row // page].long(), row % page


def _parts(cache, latent, fmt):
    """A cache's buffer as the values that it holds: views, nothing is copied."""
    if not fmt.startswith("fp8"):
        return {"rows": cache.view(FORMATS[fmt])}
    return {"codes": cache[..., :latent].view(torch.float8_e4m3fn),
            "rope": cache[..., latent:latent + 2 * ROPE].view(FORMATS[fmt]),
            "scales": cache[..., latent + 2 * ROPE:latent + 2 * ROPE + latent // 32].view(torch.float8_e8m0fnu)}


def _plain_rope(s):
    c = s["case"]
    x, lo, hi = s["x"].float(), c["offset"], c["offset"] + c["dim"]
    return torch.cat([x[..., :lo], _rotate(x[..., lo:hi], s["pos"], s["freq"], c["half"]), x[..., hi:]], -1).to(TYPES[c["to"]])


def _plain_write(s):
    c = s["case"]
    n = c["latent"]
    x = s["kv"].float()
    lat, rope = x[:, :n], x[:, n:]
    lat = lat * torch.rsqrt(lat.square().mean(-1, keepdim=True) + EPS) * s["norm"]
    rows = _pack(lat, _rotate(rope, s["pos"], s["freq"], False), c["fmt"])
    s["cache"][_place(s, s["seq_of"], s["ctx"][s["seq_of"]] + s["nth"])] = rows
    return _parts(s["cache"], n, c["fmt"])


def _plain_read(s):
    c = s["case"]
    rows = s["cache"][_place(s, s["seq_of"], s["ctx"][s["seq_of"]] + s["nth"])]
    return _unpack(rows, c["latent"], c["fmt"]).to(TYPES[c["type"]])


def _visible(s):
    """[sequence, token, row]: whether the token sees the row."""
    c = s["case"]
    row = torch.arange(s["longest"], device=s["ctx"].device)
    drafted = row[None, :] - s["ctx"][:, None]                                  # [sequence, row]
    sees = torch.zeros(c["seqs"], s["most"], s["most"], dtype=torch.bool, device=row.device)
    sees[s["seq_of"], s["nth"]] = s["sees"]
    index = drafted.clamp(0, s["most"] - 1)[:, None, :].expand(-1, s["most"], -1).long()
    inside = ((drafted >= 0) & (drafted < s["most"]))[:, None, :]
    return (drafted < 0)[:, None, :] | (sees.gather(2, index) & inside)


def _plain_attend(s):
    c = s["case"]
    n, h = c["latent"], c["heads"]
    q = torch.zeros(c["seqs"], s["most"], h, n + ROPE, device=s["ctx"].device)
    q[s["seq_of"], s["nth"]] = torch.cat([s["q_latent"], s["q_rope"]], -1).float()
    seq = torch.arange(c["seqs"], device=q.device)[:, None]
    row = torch.arange(s["longest"], device=q.device)[None, :].expand(c["seqs"], -1)
    kv = _unpack(s["cache"][_place(s, seq, row)], n, c["fmt"])                   # [sequence, row, n + 64]
    score = torch.bmm(q.view(c["seqs"], -1, n + ROPE), kv.transpose(1, 2)).mul_(s["scale"])
    score = score.view(c["seqs"], s["most"], h, -1).masked_fill_(~_visible(s)[:, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(c["seqs"], -1, s["longest"]), kv[..., :n]).view(c["seqs"], s["most"], h, n) / total
    lse = (total.log() + top).squeeze(-1)
    return {"out": out[s["seq_of"], s["nth"]].to(FORMATS[c["fmt"]]), "lse": lse[s["seq_of"], s["nth"]]}


PLAIN = {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}


# ---------------------------------------------------------- the library's calls
_context = None


def _handles(s):
    """What a program keeps beside its tensors: the context, the structures of the calls, the workspace."""
    global _context
    import flash_deepseek_b200 as F
    if _context is None:
        _context = F.MoE(F.MoeConfig(hidden=256, intermediate=256, n_experts=8, n_group=2, topk_group=1, top_k=2,
                                     max_tokens=1), device=torch.cuda.current_device())
    c = s["case"]
    s["types"] = {"f32": F.TYPE_F32, "f16": F.TYPE_F16, "bf16": F.TYPE_BF16}
    s["m"] = _context
    s["cfg"] = F.RopeConfig(dim=c.get("dim", ROPE), half_layout=c.get("half", False), theta=THETA,
                            scale=c.get("yarn", 40.0), orig_ctx=ORIG_CTX)
    if c["op"] != "rope":
        formats = {"f16": F.KV_F16, "bf16": F.KV_BF16, "fp8_f16": F.KV_FP8_F16, "fp8_bf16": F.KV_FP8_BF16}
        s["kvc"] = F.KVCache(s["cache"], formats[c["fmt"]], c["latent"], c["page"], s["n_pages"])
        s["batch"] = F.KVBatch(c["seqs"], s["n_tokens"], s["q_start"], s["ctx"], s["table"], s["per_seq"])
    if c["op"] == "attend":
        size = _context.mla_workspace_bytes(c["latent"])
        s["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")


def _own(s):
    c, m = s["case"], s["m"]
    stream = torch.cuda.current_stream().cuda_stream or 1   # 1: the legacy default stream by its own handle
    if c["op"] == "rope":
        t, h, d = s["x"].shape
        y = torch.empty(t, h, d, dtype=TYPES[c["to"]], device="cuda")
        m.rope_device(s["cfg"], s["x"], s["types"][c["type"]], (h * d, d), y, s["types"][c["to"]], (h * d, d), s["pos"],
                      t, h, d, c["offset"], stream)
        return y
    if c["op"] == "write":
        m.kv_write_device(s["kvc"], s["batch"], s["kv"], s["types"][c["type"]], c["latent"] + ROPE, s["norm"], EPS,
                          s["cfg"], s["pos"], stream)
        return _parts(s["cache"], c["latent"], c["fmt"])
    if c["op"] == "read":
        width = c["latent"] + ROPE
        y = torch.empty(s["n_tokens"], width, dtype=TYPES[c["type"]], device="cuda")
        m.kv_read_device(s["kvc"], s["batch"], y, s["types"][c["type"]], width, stream)
        return y
    h, n = c["heads"], c["latent"]
    out = torch.empty(s["n_tokens"], h, n, dtype=FORMATS[c["fmt"]], device="cuda")
    lse = torch.empty(s["n_tokens"], h, dtype=torch.float32, device="cuda")
    m.mla_attention_device(s["kvc"], s["batch"], s["q_latent"], (h * n, n), s["q_rope"], (h * ROPE, ROPE), h, s["scale"],
                           out, (h * n, n), s["ws"], s["ws"].numel(), lse=lse, tree=s["tree"] if c["tree"] else None,
                           tree_words=s["tree"].shape[1] if c["tree"] else 0, stream=stream)
    return {"out": out, "lse": lse}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------- the definition, in 64 bits
def _exact_turn(x, pos, freq, half):
    """Each pair as a complex number, times exp(i pos freq)."""
    m = freq.shape[0]
    z = torch.complex(x[..., :m], x[..., m:]) if half else torch.view_as_complex(x.reshape(*x.shape[:-1], m, 2).contiguous())
    angle = torch.outer(pos.double(), freq)
    w = torch.polar(torch.ones_like(angle), angle)
    z = z * (w[:, None, :] if x.dim() == 3 else w)
    return torch.cat([z.real, z.imag], -1) if half else torch.view_as_real(z).reshape(x.shape)


def _exact_rows(flat, latent, fmt):
    """Values of cache rows [n, bytes] in 64 bits."""
    if not fmt.startswith("fp8"):
        return flat.contiguous().view(FORMATS[fmt]).double()
    byte = flat[:, :latent].long()
    e, m = byte >> 3 & 15, (byte & 7).double()
    mag = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2((e - 10).double()))
    scale = torch.exp2(flat[:, latent + 2 * ROPE:latent + 2 * ROPE + latent // 32].double() - 127)
    lat = mag * torch.where(byte >= 128, -1.0, 1.0) * scale.repeat_interleave(32, 1)
    return torch.cat([lat, flat[:, latent:latent + 2 * ROPE].contiguous().view(FORMATS[fmt]).double()], 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        x = s["x"].double()
        lo, hi = case["offset"], case["offset"] + case["dim"]
        x[..., lo:hi] = _exact_turn(x[..., lo:hi].clone(), s["pos"], s["freq"], case["half"])
        return x
    n, fmt, page = case["latent"], case["fmt"], case["page"]
    table, ctx, start = s["table"].cpu(), s["ctx"].tolist(), s["q_start"].tolist()
    # the flat number of every row of a sequence, from the page table
    flat = [(table[b].long()[:, None] * page + torch.arange(page)).reshape(-1).cuda() for b in range(case["seqs"])]
    store = s["cache"].view(s["n_pages"] * page, -1)
    span = range(case["seqs"])
    if case["op"] == "read":
        return torch.cat([_exact_rows(store[flat[b][ctx[b]:ctx[b] + start[b + 1] - start[b]]], n, fmt) for b in span])
    if case["op"] == "write":
        x = s["kv"].double()
        lat = x[:, :n] / (x[:, :n].pow(2).mean(1, keepdim=True) + EPS).sqrt() * s["norm"].double()
        rope = _exact_turn(x[:, n:], s["pos"], s["freq"], False)
        at = torch.cat([flat[b][ctx[b]:ctx[b] + start[b + 1] - start[b]] for b in span])
        shape = (s["n_pages"], page, -1)
        if not fmt.startswith("fp8"):
            rows = torch.zeros(len(store), n + ROPE, dtype=torch.float64, device="cuda")
            rows[at] = torch.cat([lat, rope], 1)
            return {"rows": rows.view(shape)}
        g = lat.view(-1, n // 32, 32)
        k = torch.ceil(torch.log2(g.abs().amax(-1) / 448)).clamp(-15, 7)
        v = g / torch.exp2(k)[..., None]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)   # of e4m3 at v
        codes = torch.zeros(len(store), n, dtype=torch.float64, device="cuda")
        codes[at] = (torch.round(v / step) * step).view(-1, n)
        scales = torch.full((len(store), n // 32), 2.0 ** -127, dtype=torch.float64, device="cuda")
        scales[at] = torch.exp2(k)
        ropes = torch.zeros(len(store), ROPE, dtype=torch.float64, device="cuda")
        ropes[at] = rope
        return {"codes": codes.view(shape), "rope": ropes.view(shape), "scales": scales.view(shape)}
    outs, lses = [], []
    for b in span:
        t = slice(start[b], start[b + 1])
        count = start[b + 1] - start[b]
        kv = _exact_rows(store[flat[b][:ctx[b] + count]], n, fmt)
        q = torch.cat([s["q_latent"][t], s["q_rope"][t]], -1).double()
        logits = torch.einsum("thd,rd->thr", q, kv) * s["scale"]
        hidden = torch.zeros(count, ctx[b] + count, dtype=torch.bool, device="cuda")
        hidden[:, ctx[b]:] = ~s["sees"][t, :count]
        logits[hidden[:, None, :].expand_as(logits)] = -math.inf
        lses.append(torch.logsumexp(logits, -1))
        outs.append(torch.einsum("thr,rd->thd", torch.softmax(logits, -1), kv[:, :n]))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
