"""Rotary positions, a paged key/value cache in 4 bits and the attention that reads it, as measurable cases.

Every case goes through the raw-pointer calls of the `tensorcore_b200` binding on torch's current stream, as a server
calls them between the projections of a layer: `raw_rope` turns rows by their positions (back again for gradients),
`raw_kv_append` turns a step's queries and keys and writes keys and values into the pages of their sequences,
`raw_kv_read` gives rows of the cache back, `raw_attention_paged` attends over the pages.  The plain forms are torch
operations in fp32.

Pages hold `page` tokens of every K/V head in tiles of 16 tokens.  A tile of NB = head_dim / 32 blocks is 576 NB bytes:
  keys' codes     [token 16][t 4][block NB][4 bytes]: nibble j of the eight is element 32 block + 8 t + j
  keys' scales    [token 16][block NB] fp16
  values' codes   [h 2][g 8][t 4][block NB][e 2][2 bytes]: nibble i of the four is element 32 block + 4 g + i of token 8 h + 2 t + e
  values' scales  [h 2][t 4][block NB][e 2] fp16
A code c with scale d stands for (c - 8) d; blocks of 32 elements are quantised as the library's Q4_0 weights are.

listed()          the cases; draw(rng) one more of the same ranges
prepare / run     what a program has in hand before a call, and one pass
work              bytes and operations a pass cannot do without
exact             the same results in 64-bit torch, without this library
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BASE = 500000.0      # of the rotary frequencies


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    return [
        # Query rows of one token (a decode step of one sequence): the smallest call, where latency counts.
        dict(name="rope_decode_m1", op="rope", tokens=1, heads=32, D=128, rot=128, layout="half", dtype="f16", rows=8192, inverse=False, fused=0),
        # Gradient of a training batch's queries, neighbouring elements paired: the rotation backwards.
        dict(name="rope_grad_bf16_8k", op="rope", tokens=8192, heads=32, D=128, rot=128, layout="interleaved", dtype="bf16", rows=8192, inverse=True, fused=0),
        # fp32 rows inside wider rows (a fused projection's result), three quarters of a head of 96 turned, odd sizes.
        dict(name="rope_part_f32_ragged", op="rope", tokens=1531, heads=20, D=96, rot=72, layout="half", dtype="f32", rows=40000, inverse=False, fused=7),
        # A decode step of 64 sequences: one new token each, queries turned beside it.
        dict(name="append_decode_b64", op="append", seqs=64, mean=1, ctx=4000, H=32, Hkv=8, D=128, rot=128, layout="half", dtype="f16", page=16, qkv=True),
        # Prompts of a few sequences put into the cache, behind what two of them already have there.
        dict(name="append_prompts_bf16", op="append", seqs=5, mean=1900, ctx=700, H=32, Hkv=8, D=128, rot=64, layout="interleaved", dtype="bf16", page=64, qkv=False),
        # One token of one sequence over a short cache: latency.
        dict(name="attn_decode_b1_short", op="attn", seqs=1, q=1, ragged=False, ctx=611, H=32, Hkv=8, D=128, dtype="f16", page=16, causal=True, window=0, lse=False),
        # A server's decode batch: lengths from nothing (an idle slot) to eight thousand.
        dict(name="attn_decode_b64_ragged", op="attn", seqs=64, q=1, ragged=True, ctx=8192, H=32, Hkv=8, D=128, dtype="f16", page=64, causal=True, window=0, lse=True),
        # One token over a very long cache, eight queries to a K/V head.
        dict(name="attn_decode_b1_long", op="attn", seqs=1, q=1, ragged=False, ctx=100003, H=64, Hkv=8, D=128, dtype="f16", page=128, causal=True, window=0, lse=False),
        # The 7B shape: a K/V head for every query head.
        dict(name="attn_decode_mha_bf16", op="attn", seqs=8, q=1, ragged=True, ctx=4096, H=32, Hkv=32, D=128, dtype="bf16", page=32, causal=True, window=0, lse=False),
        # Five proposed tokens a sequence are checked at once, in a window, heads of 64.
        dict(name="attn_verify_window", op="attn", seqs=16, q=5, ragged=True, ctx=6000, H=16, Hkv=4, D=64, dtype="bf16", page=16, causal=True, window=1024, lse=True),
        # A piece of 512 tokens of a long prompt, over what is there already.
        dict(name="attn_prompt_512", op="attn", seqs=1, q=512, ragged=False, ctx=4608, H=32, Hkv=8, D=128, dtype="f16", page=64, causal=True, window=0, lse=False),
        # Prompts and single tokens of several sequences in one call.
        dict(name="attn_mixed_prompts", op="attn", seqs=7, q=640, ragged=True, ctx=2000, H=32, Hkv=8, D=128, dtype="bf16", page=32, causal=True, window=0, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "decode", "decode", "verify", "prompt"])
    D = rng.choice([64, 96, 128, 128, 128])
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    H = hkv * rng.choice([1, 2, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    layout = rng.choice(["half", "interleaved"])
    rot = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
    if kind == "rope":
        return dict(op="rope", tokens=_log(rng, 1, max(1, 8192 * 32 * 128 // (H * D * 2))), heads=H, D=D, rot=rot, layout=layout,
                    dtype=rng.choice(["f16", "bf16", "f32"]), rows=_log(rng, 8192, 100000), inverse=rng.random() < 0.5, fused=rng.choice([0, 0, 1, 8]))
    if kind == "append":
        seqs, qkv = _log(rng, 1, 128), rng.random() < 0.7
        return dict(op="append", seqs=seqs, mean=rng.choice([1, 1, _log(rng, 2, max(2, 9500 // seqs))]), ctx=_log(rng, 1, 4000), H=min(H, 64), Hkv=hkv, D=D,
                    rot=rot, layout=layout, dtype=rng.choice(["f16", "bf16", "f32"]), page=page, qkv=qkv)
    if kind == "decode":
        seqs = _log(rng, 1, 96)
        ctx = _log(rng, 1, min(100000, max(1, 64 * 8192 * 8 * 128 // (seqs * hkv * D))))
        return dict(op="attn", seqs=seqs, q=1, ragged=rng.random() < 0.7, ctx=ctx, H=H, Hkv=hkv, D=D, dtype=dtype, page=page, causal=True,
                    window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), lse=rng.random() < 0.5)
    if kind == "verify":
        seqs, q = _log(rng, 1, 32), rng.randint(2, 12)
        ctx = _log(rng, 16, min(16000, max(16, 64 * 8192 * 8 * 128 // (2 * seqs * hkv * D))))
        return dict(op="attn", seqs=seqs, q=q, ragged=rng.random() < 0.7, ctx=ctx, H=H, Hkv=hkv, D=D, dtype=dtype, page=page, causal=rng.random() < 0.8,
                    window=rng.choice([0, 0, _log(rng, 16, 4096)]), lse=rng.random() < 0.5)
    seqs, q = _log(rng, 1, 8), _log(rng, 24, 900)
    ctx = _log(rng, q, max(q, min(16000, 512 * 4608 * 32 * 128 // (seqs * q * H * D))))
    return dict(op="attn", seqs=seqs, q=q, ragged=rng.random() < 0.5, ctx=ctx, H=H, Hkv=hkv, D=D, dtype=dtype, page=page, causal=rng.random() < 0.9,
                window=rng.choice([0, 0, 0, _log(rng, 64, 4096)]), lse=rng.random() < 0.5)


# ---- sizes of a case's sequences: the same for every seed, so that every seed is as much work ----------
def _lengths(c):
    """Appending: tokens already in the cache and new ones, by sequence; attention: keys and queries."""
    rng = random.Random(77 * c["seqs"] + c["ctx"])
    if c["op"] == "append":
        new = [1] * c["seqs"] if c["mean"] == 1 else [max(1, int(c["mean"] * rng.uniform(0.3, 1.7))) for _ in range(c["seqs"])]
        if c["mean"] > 1:
            total = c["seqs"] * c["mean"]
            new = [max(1, n * total // sum(new)) for n in new]
        return [rng.randint(0, c["ctx"]) if c["mean"] == 1 or rng.random() < 0.4 else 0 for _ in range(c["seqs"])], new
    if not c["ragged"]:
        return [max(c["ctx"], c["q"])] * c["seqs"], [c["q"]] * c["seqs"]
    keys = [int(c["ctx"] * (1 - 0.98 * rng.random())) for _ in range(c["seqs"])]
    keys[0] = c["ctx"]
    qs = [c["q"]] * c["seqs"] if c["q"] <= 16 else [c["q"]] + [rng.choice([1, rng.randint(1, c["q"])]) for _ in range(c["seqs"] - 1)]
    keys = [max(k, n) for k, n in zip(keys, qs)]
    if c["q"] == 1 and c["seqs"] > 3:
        keys[c["seqs"] // 2] = 0          # a slot without a sequence
    return keys, qs


# ---- data ----------------------------------------------------------------------------------------
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + what)
    return g


def _normal(shape, g, scale=1.0, mean=0.0, dtype=torch.float32):
    t = torch.empty(shape, dtype=torch.float32, device="cuda")
    t.normal_(mean, scale, generator=g)
    return t.to(dtype)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(rows, rot):
    """cos and sin [rows, rot / 2], worked out in 64 bits as a program does once for a model."""
    freq = torch.pow(torch.tensor(BASE, dtype=torch.float64, device="cuda"), -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda").unsqueeze(1) * freq
    return torch.cos(angle).float(), torch.sin(angle).float()


def _page_table(c, tokens, seed):
    """Pages of the sequences in no order: [seqs, most pages], -1 behind a sequence's own; and how many there are."""
    n = [-(-k // c["page"]) for k in tokens]
    total = sum(n) + 3
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed + 9)).to(torch.int32)
    table, at = torch.full((len(n), max(1, max(n))), -1, dtype=torch.int32), 0
    for s, k in enumerate(n):
        table[s, :k] = perm[at:at + k]
        at += k
    return table.cuda(), total


def _quantise(x, dt=torch.float32):
    """Blocks of 32: codes 0 .. 15 (uint8, as x) and scales [.., D / 32] as fp16; elementwise steps rounded one by one."""
    b = x.to(dt).unflatten(-1, (-1, 32))
    most = b.abs().amax(dim=-1, keepdim=True)
    inv = torch.where(most > 0, 8.0 / most, torch.zeros_like(most))
    y = b * inv
    whole = torch.trunc(y)
    whole = whole + torch.sign(y) * ((y - whole).abs() >= 0.5)                   # half away from zero
    return (whole + 8.0).clamp_(0, 15).to(torch.uint8).flatten(-2), (most / 8.0).squeeze(-1).to(torch.float16)


def _cache_values(c, pages, seed):
    """Codes and scales of a cache in use, [pages, Hkv, page, D]: keys with channels of different size, values N(0, 1)."""
    shape = (c["Hkv"], c["page"], c["D"])
    size = torch.exp(_normal((c["Hkv"], 1, c["D"]), _gen(seed, 21), 0.4))
    out = []
    for what in (22, 23):
        g = _gen(seed, what)
        codes = torch.empty((pages,) + shape, dtype=torch.uint8, device="cuda")
        scales = torch.empty((pages,) + shape[:2] + (c["D"] // 32,), dtype=torch.float16, device="cuda")
        step = max(1, (1 << 26) // math.prod(shape))
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = _normal((n,) + shape, g)
            codes[p:p + n], scales[p:p + n] = _quantise(x * size if what == 22 else x)
        out += [codes, scales]
    return out


def _pack(kc, ks, vc, vs):
    """Codes [pages, Hkv, page, D] and scales to pages, uint8 [pages, Hkv, page / 16, 576 NB]."""
    n, h, p, D = kc.shape
    nb, lead = D // 32, (n, h, p // 16)
    k = kc.view(lead + (16, nb, 4, 4, 2)).permute(0, 1, 2, 3, 5, 4, 6, 7)
    k = (k[..., 0] | (k[..., 1] << 4)).reshape(lead + (256 * nb,))
    v = vc.view(lead + (2, 4, 2, nb, 8, 2, 2)).permute(0, 1, 2, 3, 7, 4, 6, 5, 8, 9)       # h g t block e, byte, nibble
    v = (v[..., 0] | (v[..., 1] << 4)).reshape(lead + (256 * nb,))
    ks = ks.reshape(lead + (16 * nb,)).view(torch.uint8)
    vs = vs.view(lead + (2, 4, 2, nb)).permute(0, 1, 2, 3, 4, 6, 5).reshape(lead + (16 * nb,)).view(torch.uint8)
    return torch.cat([k, ks, v, vs], dim=3)


def _attn_data(c, seed):
    keys, qs = _lengths(c)
    table, pages = _page_table(c, keys, seed)
    q = _normal((sum(qs), c["H"], c["D"]), _gen(seed, 24), dtype=DTYPES[c["dtype"]])
    return keys, qs, table, q, _cache_values(c, pages, seed)


def _append_data(c, seed):
    """Rows of queries, keys and values (one fused projection's rows, or tensors of their own), where they go."""
    old, new = _lengths(c)
    g, T, D = _gen(seed, 31), sum(new), c["D"]
    n = c["H"] + 2 * c["Hkv"] if c["qkv"] else 2 * c["Hkv"]
    x = _normal((T, n, D), g, dtype=DTYPES[c["dtype"]])
    pos = _int([o + i for o, k in zip(old, new) for i in range(k)])
    seq = _int([s for s, k in enumerate(new) for _ in range(k)])
    table, pages = _page_table(c, [o + k for o, k in zip(old, new)], seed)
    if c["qkv"]:
        q, k, v = x[:, :c["H"]], x[:, c["H"]:c["H"] + c["Hkv"]], x[:, c["H"] + c["Hkv"]:]
    else:
        q, k, v = None, x[:, :c["Hkv"]].contiguous(), x[:, c["Hkv"]:].contiguous()
    return q, k, v, pos, seq, table, pages, max(o + m for o, m in zip(old, new))


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    if c["op"] == "rope":
        wide = _normal((c["tokens"], c["heads"] + c["fused"], c["D"]), _gen(seed, 11), dtype=dt)
        pos = torch.randint(0, c["rows"], (c["tokens"],), generator=_gen(seed, 12), device="cuda", dtype=torch.int32)
        cos, sin = _tables(c["rows"], c["rot"])
        x = wide[:, :c["heads"]]
        return dict(c=c, x=x, pos=pos, cos=cos, sin=sin, y=torch.zeros(x.shape, dtype=dt, device="cuda"))
    if c["op"] == "append":
        q, k, v, pos, seq, table, pages, longest = _append_data(c, seed)
        cos, sin = _tables(longest, c["rot"])
        store = torch.zeros((pages, c["Hkv"], c["page"] // 16, 18 * c["D"]), dtype=torch.uint8, device="cuda")
        back = torch.zeros((2,) + k.shape, dtype=torch.float16, device="cuda")
        return dict(c=c, q=q, k=k, v=v, pos=pos, seq=seq, table=table, cos=cos, sin=sin, pages=store, back=back,
                    y=None if q is None else torch.zeros(q.shape, dtype=dt, device="cuda"))
    keys, qs, table, q, cache = _attn_data(c, seed)
    start = [0]
    for n in qs:
        start.append(start[-1] + n)
    return dict(c=c, q=q, pages=_pack(*cache), table=table, lens=_int(keys), start=_int(start), max_q=max(qs), o=torch.zeros_like(q),
                lse=torch.zeros(q.shape[:2], dtype=torch.float32, device="cuda"))


# ---- a pass in plain form ----------------------------------------------------------------------------
def _turn(x, cos, sin, pos, rot, layout, inverse=False):
    """Rows [tokens, heads, D] turned by their positions, in the type of the tables."""
    x = x.to(cos.dtype)
    c, s = cos[pos.long()].unsqueeze(1), sin[pos.long()].unsqueeze(1)
    if inverse:
        s = -s
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., rot:]], dim=-1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2), x[..., rot:]], dim=-1)


def _places(c, pos, seq, table):
    """For tokens' rows: where in the pages, counted in 16-bit words, their codes and scales are, [tokens, Hkv, ..]."""
    nb, P, dev = c["D"] // 32, c["page"], pos.device
    pos, seq = pos.long(), seq.long()
    page = table[seq, pos // P].long()
    head = torch.arange(c["Hkv"], device=dev)
    tile = ((page.unsqueeze(1) * c["Hkv"] + head) * (P // 16) + (pos % P // 16).unsqueeze(1)) * (288 * nb)
    r = pos % 16
    h, t, e = r // 8, r % 8 // 2, r % 2
    block, g = torch.arange(nb, device=dev), torch.arange(8, device=dev)
    kc = (r * (8 * nb)).unsqueeze(1) + torch.arange(8 * nb, device=dev)
    ks = 128 * nb + (r * nb).unsqueeze(1) + block
    vc = 144 * nb + ((((h * 32 + t).unsqueeze(1) + 4 * g).unsqueeze(2) * nb + block) * 2 + e.view(-1, 1, 1)).flatten(1)
    vs = 272 * nb + (((h * 4 + t) * nb).unsqueeze(1) + block) * 2 + e.unsqueeze(1)
    return [tile.unsqueeze(2) + x.unsqueeze(1) for x in (kc, ks, vc, vs)]


def _append_plain(s):
    c = s["c"]
    nb, words = c["D"] // 32, s["pages"].view(torch.int16).view(-1)
    kc, ks = _quantise(_turn(s["k"], s["cos"], s["sin"], s["pos"], c["rot"], c["layout"]))
    vc, vs = _quantise(s["v"])
    lead = kc.shape[:2]
    k = kc.view(lead + (nb, 4, 4, 2)).transpose(2, 3)
    k = (k[..., 0] | (k[..., 1] << 4)).reshape(lead + (-1,)).view(torch.int16)
    v = vc.view(lead + (nb, 8, 2, 2)).transpose(2, 3)
    v = (v[..., 0] | (v[..., 1] << 4)).reshape(lead + (-1,)).view(torch.int16)
    at = _places(c, s["pos"], s["seq"], s["table"])
    for where, what in zip(at, (k, ks.view(torch.int16), v, vs.view(torch.int16))):
        words[where] = what
    # the rows as the cache has them now
    k, ks, v, vs = (words[where] for where in at)
    k = _nibbles(k.view(torch.uint8)).view(lead + (4, nb, 8)).transpose(2, 3).reshape(lead + (nb, 32))
    v = _nibbles(v.view(torch.uint8)).view(lead + (8, nb, 4)).transpose(2, 3).reshape(lead + (nb, 32))
    kv = torch.stack([(x.float() - 8.0) * d.view(torch.float16).float().unsqueeze(-1) for x, d in ((k, ks), (v, vs))])
    out = {"k": kv[0].flatten(-2).to(torch.float16), "v": kv[1].flatten(-2).to(torch.float16)}
    if s["q"] is not None:
        out["q"] = _turn(s["q"], s["cos"], s["sin"], s["pos"], c["rot"], c["layout"]).to(s["q"].dtype)
    return out


def _nibbles(x):
    return torch.stack([x & 15, x >> 4], dim=-1).flatten(-2)


def _unpack(pages, table, c):
    """The sequences' keys and values as fp32, [seqs, Hkv, most tokens, D]; pages that are not theirs count as page 0."""
    nb = c["D"] // 32
    t = pages[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)          # [seqs, Hkv, tiles, bytes]
    lead = t.shape[:3]
    k, ks, v, vs = t.split([256 * nb, 32 * nb, 256 * nb, 32 * nb], dim=3)
    k = _nibbles(k).view(lead + (16, 4, nb, 8)).transpose(4, 5).reshape(lead + (16, nb, 32))
    k = (k.float() - 8.0) * ks.contiguous().view(torch.float16).float().view(lead + (16, nb, 1))
    v = _nibbles(v).view(lead + (2, 8, 4, nb, 2, 4)).permute(0, 1, 2, 3, 5, 7, 6, 4, 8).reshape(lead + (16, nb, 32))
    vs = vs.contiguous().view(torch.float16).float().view(lead + (2, 4, nb, 2)).transpose(5, 6).reshape(lead + (16, nb, 1))
    shape = lead[:2] + (lead[2] * 16, c["D"])
    return k.reshape(shape), ((v.float() - 8.0) * vs).reshape(shape)


def _attn_plain(s):
    c, q, dev = s["c"], s["q"], s["q"].device
    n, rep, mq = c["seqs"], c["H"] // c["Hkv"], s["max_q"]
    k, v = _unpack(s["pages"], s["table"], c)
    lens, start = s["lens"].long(), s["start"].long()
    nq = start[1:] - start[:-1]
    i = torch.arange(mq, device=dev)
    row = (start[:-1].unsqueeze(1) + i).clamp(max=q.shape[0] - 1)                 # [seqs, mq]
    there = i < nq.unsqueeze(1)
    qp = q[row].float().view(n, mq, c["Hkv"], rep, c["D"]).permute(0, 2, 3, 1, 4).reshape(n, c["Hkv"], rep * mq, c["D"])
    sc = torch.matmul(qp, k.transpose(2, 3)).mul_(1.0 / math.sqrt(c["D"])).view(n, c["Hkv"], rep, mq, -1)
    j = torch.arange(k.shape[2], device=dev)
    at = (lens - nq).unsqueeze(1) + i                                            # positions of the queries
    seen = (j < lens.view(-1, 1, 1)).expand(n, mq, -1)
    if c["causal"]:
        seen = seen & (j <= at.unsqueeze(2))
    if c["window"]:
        seen = seen & (at.unsqueeze(2) - j <= c["window"])
    sc.masked_fill_(~seen.view(n, 1, 1, mq, -1), -math.inf)
    m = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))))
    l = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(n, c["Hkv"], rep * mq, -1), v).view(n, c["Hkv"], rep, mq, c["D"])
    o = torch.where(l > 0, o / l, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(n, mq, c["H"], c["D"])
    out = {"o": o.to(q.dtype)[there]}
    if c["lse"]:
        out["lse"] = (m + torch.log(l)).view(n, c["H"], mq).transpose(1, 2)[there]
    return out


# ---- a pass ------------------------------------------------------------------------------------------
_ctx = None


def _call(s):
    """The same through the library's calls; what describes a call's shapes is made once."""
    global _ctx
    import tensorcore_b200 as tc
    if _ctx is None:
        _ctx = tc.Context()
    c, st = s["c"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "rope":
        if "desc" not in s:
            s["desc"] = tc.rope_desc(c["tokens"], c["heads"], c["D"], rot_dim=c["rot"], layout=c["layout"], dtype=c["dtype"], table_rows=c["rows"],
                                     x_strides=s["x"].stride()[:2], inverse=c["inverse"])
        tc.raw_rope(_ctx, s["desc"], s["x"].data_ptr(), s["y"].data_ptr(), s["cos"].data_ptr(), s["sin"].data_ptr(), s["pos"].data_ptr(), st)
        return s["y"]
    if "kv" not in s:
        s["kv"] = tc.kv_desc(s["pages"].shape[0], c["page"], c["Hkv"], c["D"])
    if c["op"] == "append":
        if "desc" not in s:
            s["desc"] = tc.kv_append_desc(s["pos"].shape[0], s["table"].shape[0], s["table"].shape[1], q_heads=c["H"] if c["qkv"] else 0, rot_dim=c["rot"],
                                          layout=c["layout"], dtype=c["dtype"], table_rows=s["cos"].shape[0], k_strides=s["k"].stride()[:2],
                                          v_strides=s["v"].stride()[:2], q_strides=s["q"].stride()[:2] if c["qkv"] else (0, 0))
            s["read"] = tc.kv_read_desc(s["pos"].shape[0], s["table"].shape[0], s["table"].shape[1], dtype="f16")
        where = (s["pos"].data_ptr(), s["seq"].data_ptr(), s["table"].data_ptr())
        q, y = (s["q"].data_ptr(), s["y"].data_ptr()) if c["qkv"] else (0, 0)
        tc.raw_kv_append(_ctx, s["kv"], s["desc"], s["pages"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), q, y, s["cos"].data_ptr(),
                         s["sin"].data_ptr(), *where, st)
        tc.raw_kv_read(_ctx, s["kv"], s["read"], s["pages"].data_ptr(), s["back"][0].data_ptr(), s["back"][1].data_ptr(), *where, st)
        out = {"k": s["back"][0], "v": s["back"][1]}
        return dict(out, q=s["y"]) if c["qkv"] else out
    if "desc" not in s:
        s["desc"] = tc.attention_paged_desc(s["q"].shape[0], c["seqs"], s["table"].shape[1], c["H"], max_q=s["max_q"], dtype=c["dtype"],
                                            causal=c["causal"], window_size=c["window"])
    tc.raw_attention_paged(_ctx, s["kv"], s["desc"], s["pages"].data_ptr(), s["q"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
                           s["start"].data_ptr(), s["o"].data_ptr(), s["lse"].data_ptr() if c["lse"] else 0, st)
    return {"o": s["o"], "lse": s["lse"]} if c["lse"] else {"o": s["o"]}


def run(state):
    if own:
        return _call(state)
    c = state["c"]
    if c["op"] == "rope":
        return _turn(state["x"], state["cos"], state["sin"], state["pos"], c["rot"], c["layout"], c["inverse"]).to(state["x"].dtype)
    return _append_plain(state) if c["op"] == "append" else _attn_plain(state)


# ---- what it costs at least -----------------------------------------------------------------------------
def _pairs(c, keys, queries):
    """Keys that the queries of one sequence see, together, and how many keys any of them sees."""
    total, lo = 0, keys
    for i in range(queries):
        at = keys - queries + i
        hi = min(keys, at + 1) if c["causal"] else keys
        first = max(0, at - c["window"]) if c["window"] else 0
        total += max(0, hi - first)
        lo = min(lo, first)
    return total, keys - lo if queries else 0


def work(case):
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["D"] * es + c["tokens"] * (c["rot"] * 4 + 4), "flops": 3 * n * c["rot"]}
    if c["op"] == "append":
        T = sum(_lengths(c)[1])
        rows = c["H"] if c["qkv"] else 0
        return {"bytes": T * c["D"] * (2 * rows * es + 2 * c["Hkv"] * (es + 2)) + T * c["Hkv"] * (c["D"] * 9 // 8) + T * (c["rot"] * 4 + 8),
                "flops": T * ((rows + c["Hkv"]) * 3 * c["rot"] + 2 * c["Hkv"] * 4 * c["D"])}
    keys, qs = _lengths(c)
    got = [_pairs(c, k, n) for k, n in zip(keys, qs)]
    T = sum(qs)
    return {"bytes": sum(n for _, n in got) * c["Hkv"] * (c["D"] * 9 // 8) + 2 * T * c["H"] * c["D"] * es + (4 * T * c["H"] if c["lse"] else 0),
            "flops": 4 * c["H"] * c["D"] * sum(p for p, _ in got)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _rotated64(x, cos, sin, pos, rot, layout, sign=1.0):
    """Pairs as complex numbers times exp(i angle)."""
    z = torch.complex(cos.double(), sign * sin.double())[pos.long()].unsqueeze(1)
    y = x.double().clone()
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    w = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _stored64(x):
    """Rows as blocks of 32 in 4 bits hold them."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(dim=-1, keepdim=True)
    code = torch.where(top > 0, b * 8.0 / top, torch.zeros_like(b))
    code = (torch.sign(code) * torch.floor(code.abs() + 0.5)).clamp(-8, 7)
    return (code * (top / 8.0).half().double()).flatten(-2)


def exact(case, seed):
    c = case
    if c["op"] == "rope":
        s = prepare(c, seed)
        return _rotated64(s["x"], s["cos"], s["sin"], s["pos"], c["rot"], c["layout"], -1.0 if c["inverse"] else 1.0)
    if c["op"] == "append":
        q, k, v, pos, _, _, _, longest = _append_data(c, seed)
        cos, sin = _tables(longest, c["rot"])
        out = {"k": _stored64(_rotated64(k, cos, sin, pos, c["rot"], c["layout"])), "v": _stored64(v)}
        if q is not None:
            out["q"] = _rotated64(q, cos, sin, pos, c["rot"], c["layout"])
        return out
    keys, qs, table, q, (kc, ks, vc, vs) = _attn_data(c, seed)
    rep, at, o, lse = c["H"] // c["Hkv"], 0, [], []
    for s, (nk, nq) in enumerate(zip(keys, qs)):
        own_pages = table[s, :-(-nk // c["page"])].long()
        k, v = (((x[own_pages].double() - 8.0).unflatten(-1, (-1, 32)) * d[own_pages].double().unsqueeze(-1)).flatten(-2)
                .transpose(0, 1).flatten(1, 2)[:, :nk] for x, d in ((kc, ks), (vc, vs)))
        rows = q[at:at + nq].double().view(nq, c["Hkv"], rep, c["D"])
        at += nq
        sc = torch.einsum("ihrd,hjd->ihrj", rows, k) / math.sqrt(c["D"])
        i = torch.arange(nk - nq, nk, device="cuda").view(-1, 1)
        j = torch.arange(nk, device="cuda")
        hidden = (j > i if c["causal"] else j < 0) | (i - j > c["window"] if c["window"] else j < 0)
        sc = sc.masked_fill(hidden.view(nq, 1, 1, nk) if hidden.dim() == 2 else hidden, -math.inf)
        m = torch.logsumexp(sc, dim=-1, keepdim=True) if nk else torch.full(sc.shape[:3] + (1,), -math.inf, dtype=torch.float64, device="cuda")
        p = torch.where(m > -math.inf, torch.exp(sc - m), torch.zeros_like(sc))
        o.append(torch.einsum("ihrj,hjd->ihrd", p, v).reshape(nq, c["H"], c["D"]))
        lse.append(m.reshape(nq, c["H"]))
    return {"o": torch.cat(o), "lse": torch.cat(lse)} if c["lse"] else {"o": torch.cat(o)}
