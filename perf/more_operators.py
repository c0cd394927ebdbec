"""Pages of the 4-bit key/value cache that sequences share, move and choose from, as measurable cases.

Every case goes through the raw-pointer calls of the `tensorcore_b200` binding on torch's current stream, as a server makes them
between the steps and the layers of a model:

  copy     `raw_kv_copy`: pages, or their first tokens, to other pages in all layers (a sequence that forks, pages moved together)
  compact  `raw_kv_compact`: chosen tokens of sequences moved down to consecutive places (accepted proposals, eviction)
  shared   `raw_attention_shared`: attention for groups of sequences with the same first keys, which are read once a group
  select   `raw_kv_bounds`, `raw_kv_select`: what a step's new keys do to their blocks' bounds, then the blocks to attend to
  blocks   `raw_attention_blocks`: single tokens over the chosen blocks, a list of pages for each K/V head

Pages hold `page` tokens of every K/V head in tiles of 16 tokens.  A tile of NB = head_dim / 32 blocks of elements is 576 NB bytes:
  keys' codes     [token 16][t 4][block NB][4 bytes]: nibble j of the eight is element 32 block + 8 t + j
  keys' scales    [token 16][block NB] fp16
  values' codes   [h 2][g 8][t 4][block NB][e 2][2 bytes]: nibble i of the four is element 32 block + 4 g + i of token 8 h + 2 t + e
  values' scales  [h 2][t 4][block NB][e 2] fp16
A code c with scale d stands for (c - 8) d.

Bounds of a page's keys, 2 head_dim + 16 bytes for each K/V head: int8 hi [head_dim], int8 lo [head_dim], fp32 step, 12 bytes of zero.
step = (largest magnitude) / 127, hi = ceil(largest / step), lo = floor(smallest / step).  The queries of a K/V head are rounded to
eight bits with one step for all of them; a page's score is (I step) (queries' step), where I is the sum over the heads and elements of
the larger of q hi and q lo: whole numbers and three fp32 roundings, so that every way to compute it chooses the same pages.

listed()          the cases; draw(rng) one more of the same ranges
prepare / run     what a program has in hand before a call, and one pass
work              bytes and operations a pass cannot do without
exact             the same results in 64-bit torch, without this library
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    return [
        # One sequence forks in the middle of a page: 37 tokens of that page, in every layer.  The smallest call, where latency counts.
        dict(name="copy_fork_one", op="copy", pairs=1, tokens=37, layers=32, Hkv=8, D=128, page=64),
        # A cache's pages are moved together so that its end can be given back.
        dict(name="copy_together", op="copy", pairs=230, tokens=0, layers=16, Hkv=8, D=128, page=64),
        # Three of eight proposed tokens are kept, not the first three, in each of 32 sequences.
        dict(name="compact_proposals_b32", op="compact", seqs=32, ctx=900, tree=8, kept=3, layers=32, Hkv=8, D=128, page=16),
        # A long sequence keeps its first four and its last eight thousand tokens.
        dict(name="compact_evict_long", op="compact", seqs=1, ctx=20001, tree=0, kept=8000, layers=16, Hkv=8, D=128, page=64),
        # Four answers to one prompt are sampled side by side.
        dict(name="shared_samples_b4", op="shared", seqs=4, groups=1, q=1, prefix=1500, own=150, H=32, Hkv=8, D=128, dtype="f16", page=64, lse=False),
        # A server's decode batch behind one long system prompt.
        dict(name="shared_prompt_b64", op="shared", seqs=64, groups=1, q=1, prefix=8192, own=1024, H=32, Hkv=8, D=128, dtype="f16", page=64, lse=True),
        # Several prompts with a few sequences each, whose three proposed tokens are checked at once; heads of 64.
        dict(name="shared_groups_verify", op="shared", seqs=37, groups=5, q=3, prefix=5000, own=700, H=16, Hkv=4, D=64, dtype="bf16", page=16, lse=True),
        # One token of a very long sequence picks 64 of its 1563 blocks.
        dict(name="select_b1_long", op="select", seqs=1, ragged=False, ctx=100003, blocks=64, first=1, last=2, H=64, Hkv=8, D=128, dtype="f16", page=64),
        # A decode batch of lengths from nothing (an idle slot) on.
        dict(name="select_b64_ragged", op="select", seqs=64, ragged=True, ctx=16000, blocks=96, first=1, last=4, H=32, Hkv=8, D=128, dtype="bf16", page=32),
        # What the two cases above lead to: one token over 64 blocks of a long cache,
        dict(name="blocks_b1", op="blocks", seqs=1, ragged=False, blocks=64, H=64, Hkv=8, D=128, dtype="f16", page=64, lse=False),
        # and a batch over up to 64 blocks each.
        dict(name="blocks_b64", op="blocks", seqs=64, ragged=True, blocks=64, H=32, Hkv=8, D=128, dtype="bf16", page=32, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["copy", "compact", "shared", "shared", "select", "blocks"])
    D = rng.choice([32, 64, 96, 128, 128, 128])
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    H = hkv * rng.choice([1, 2, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "copy":
        layers, page_bytes = _log(rng, 1, 40), hkv * page * D * 9 // 8
        tokens = rng.choice([0, rng.randint(1, page)])
        return dict(op="copy", pairs=_log(rng, 1, min(2000, max(1, 230 * 16 * 73728 // (layers * page_bytes)))), tokens=tokens, layers=layers, Hkv=hkv, D=D, page=page)
    if kind == "compact":
        layers, row = _log(rng, 1, 40), hkv * D * 9 // 8
        if rng.random() < 0.5:
            seqs, tree = _log(rng, 1, 64), rng.randint(4, 24)
            return dict(op="compact", seqs=seqs, ctx=_log(rng, 64, max(64, min(3000, 300_000_000 // (layers * seqs * row)))), tree=tree,
                        kept=rng.randint(2, max(2, tree // 2)), layers=layers, Hkv=hkv, D=D, page=page)
        seqs = _log(rng, 1, 8)
        ctx = _log(rng, 64, max(64, min(24000, 300_000_000 // (layers * seqs * row))))
        return dict(op="compact", seqs=seqs, ctx=ctx, tree=0, kept=_log(rng, 4, max(4, ctx * 2 // 5)), layers=layers, Hkv=hkv, D=D, page=page)
    if kind == "shared":
        groups = _log(rng, 1, 8)
        seqs, q = groups * _log(rng, 1, 64 // groups), rng.choice([1, 1, 1, 2, 3, 5, _log(rng, 6, 64)])
        room = 64 * 9216 * 32 * 128
        prefix = _log(rng, 16, max(16, min(30000, room // (2 * seqs * q * H * D), 200_000_000 // (seqs * hkv * D))))
        return dict(op="shared", seqs=seqs, groups=groups, q=q, prefix=prefix, own=max(q, _log(rng, 1, max(1, min(2000, room // (2 * seqs * q * H * D))))), H=H, Hkv=hkv, D=D,
                    dtype=dtype, page=page, lse=rng.random() < 0.5)
    if kind == "select":
        seqs = _log(rng, 1, 64)
        ctx = _log(rng, 1, max(1, min(100000, 64 * 16000 * 8 * 128 // (seqs * hkv * D))))
        first, last = rng.randint(0, 3), rng.randint(1, 5)
        return dict(op="select", seqs=seqs, ragged=rng.random() < 0.7, ctx=ctx, blocks=first + last + _log(rng, 1, 100), first=first, last=last, H=H, Hkv=hkv, D=D,
                    dtype=dtype, page=page)
    seqs = _log(rng, 1, 64)
    return dict(op="blocks", seqs=seqs, ragged=rng.random() < 0.7, blocks=_log(rng, 1, max(1, min(256, 64 * 64 * 8 * 32 * 128 // (seqs * page * hkv * D)))), H=H, Hkv=hkv, D=D,
                dtype=dtype, page=page, lse=rng.random() < 0.5)


# ---- sizes of a case's sequences: the same for every seed, so that every seed is as much work ----------
def _moves(c):
    """Compacting: by sequence its length, the place where the kept tokens go, and which they are.  None of them lies where another one goes,
    so that a pass can be repeated."""
    rng, out = random.Random(31 * c["seqs"] + c["ctx"] + c["kept"]), []
    for _ in range(c["seqs"]):
        n = max(2 * c["tree"], 8, int(c["ctx"] * (1 - 0.5 * rng.random())) if c["seqs"] > 1 else c["ctx"])
        if c["tree"]:                    # the first proposal and later ones
            to = n - c["tree"]
            k = min(c["kept"], 1 + (c["tree"] - 1) // 2)
            keep = [to] + sorted(rng.sample(range(to + k, n), k - 1))
        else:                            # behind the first four
            to = 4
            k = min(c["kept"], (n - to) // 2)
            keep = list(range(n - k, n))
        out.append((n, to, keep))
    return out


def _family(c):
    """Shared prefixes: by group its sequences and its shared keys, whole pages; by sequence its keys."""
    rng = random.Random(17 * c["seqs"] + c["prefix"] + c["own"])
    cuts = sorted(rng.sample(range(1, c["seqs"]), min(c["groups"], c["seqs"]) - 1)) if c["groups"] > 1 else []
    start = [0] + cuts + [c["seqs"]]
    prefix = [c["prefix"] if g == 0 else int(c["prefix"] * (1 - 0.7 * rng.random())) for g in range(len(start) - 1)]
    lens = [prefix[g] + max(c["q"], int(c["own"] * (1 - 0.95 * rng.random()))) for g in range(len(prefix)) for _ in range(start[g + 1] - start[g])]
    return start, [p // c["page"] * c["page"] for p in prefix], lens


def _contexts(c):
    """Keys of each sequence."""
    rng = random.Random(77 * c["seqs"] + c["ctx"])
    keys = [c["ctx"] if not c["ragged"] or s == 0 else int(c["ctx"] * (1 - 0.98 * rng.random())) for s in range(c["seqs"])]
    if c["ragged"] and c["seqs"] > 3:
        keys[c["seqs"] // 2] = 0          # a slot without a sequence
    return keys


def _chosen(c):
    """Attention over blocks: how many each token has, and the keys in them."""
    rng = random.Random(5 * c["seqs"] + c["blocks"])
    n = [c["blocks"] if not c["ragged"] or s == 0 else rng.randint(1, c["blocks"]) for s in range(c["seqs"])]
    return n, [(k - 1) * c["page"] + rng.randint(1, c["page"]) for k in n]


# ---- data ----------------------------------------------------------------------------------------
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + what)
    return g


def _normal(shape, g, scale=1.0, dtype=torch.float32):
    t = torch.empty(shape, dtype=torch.float32, device="cuda")
    t.normal_(0.0, scale, generator=g)
    return t.to(dtype)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bytes(c, pages, seed):
    """A cache in use whose numbers do not matter, [layers, pages, Hkv, tiles, bytes]."""
    shape = (c["layers"], pages, c["Hkv"], c["page"] // 16, 18 * c["D"])
    return torch.empty(shape, dtype=torch.uint8, device="cuda").random_(0, 256, generator=_gen(seed, 41))


def _page_table(c, keys, seed, common=()):
    """Pages of the sequences in no order, [seqs, most pages], -1 behind a sequence's own, and how many there are.  common: (first sequence,
    one behind the last, pages) that those have together."""
    n = [-(-k // c["page"]) for k in keys]
    total = sum(n) + 3
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed + 9)).to(torch.int32)
    table, at = torch.full((len(n), max(1, max(n))), -1, dtype=torch.int32), 0
    for s, k in enumerate(n):
        table[s, :k] = perm[at:at + k]
        at += k
    for a, b, k in common:
        table[a:b, :k] = table[a, :k].clone()
    return table.cuda(), total


def _quantise(x):
    """Blocks of 32: codes 0 .. 15 (uint8, as x) and scales [.., D / 32] as fp16; elementwise steps rounded one by one."""
    b = x.unflatten(-1, (-1, 32))
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


def _shared_data(c, seed):
    start, shared, lens = _family(c)
    table, pages = _page_table(c, lens, seed, [(start[g], start[g + 1], p // c["page"]) for g, p in enumerate(shared)])
    q = _normal((c["seqs"] * c["q"], c["H"], c["D"]), _gen(seed, 24), dtype=DTYPES[c["dtype"]])
    return start, shared, lens, table, q, _cache_values(c, pages, seed)


def _select_data(c, seed):
    """Queries, where the sequences' keys are, and the keys' codes and scales."""
    keys = _contexts(c)
    table, pages = _page_table(c, keys, seed)
    q = _normal((c["seqs"], c["H"], c["D"]), _gen(seed, 25), dtype=DTYPES[c["dtype"]])
    return keys, table, q, _cache_values(c, pages, seed)


def _blocks_data(c, seed):
    n, keys = _chosen(c)
    pages = c["seqs"] * c["blocks"] * 2 + 3               # the cache is longer than what is chosen of it
    g = torch.Generator().manual_seed(seed + 13)
    lists = torch.full((c["seqs"], c["Hkv"], c["blocks"]), -1, dtype=torch.int32)
    for t, k in enumerate(n):
        mine = torch.randperm(pages, generator=g)[:2 * c["blocks"]].to(torch.int32)
        for h in range(c["Hkv"]):
            pick = torch.randperm(2 * c["blocks"] - 1, generator=g)[:k - 1].sort().values
            lists[t, h, :k] = torch.cat([mine[pick], mine[-1:]])         # the last block is among them
    q = _normal((c["seqs"], c["H"], c["D"]), _gen(seed, 26), dtype=DTYPES[c["dtype"]])
    return keys, lists.cuda(), q, _cache_values(c, pages, seed)


def prepare(case, seed):
    c = case
    if c["op"] == "copy":
        n = 2 * c["pairs"] + 3
        perm = torch.randperm(n, generator=torch.Generator().manual_seed(seed + 7)).to(torch.int32).cuda()
        counts = torch.full((c["pairs"],), c["tokens"], dtype=torch.int32, device="cuda") if c["tokens"] else None
        return dict(c=c, pages=_bytes(c, n, seed), src=perm[:c["pairs"]].contiguous(), dst=perm[c["pairs"]:2 * c["pairs"]].contiguous(), counts=counts)
    if c["op"] == "compact":
        moves = _moves(c)
        table, n = _page_table(c, [m[0] for m in moves], seed)
        start = [0]
        for m in moves:
            start.append(start[-1] + len(m[2]))
        return dict(c=c, pages=_bytes(c, n, seed), table=table, to=_int([m[1] for m in moves]), start=_int(start), keep=_int([k for m in moves for k in m[2]]))
    if c["op"] == "shared":
        start, shared, lens, table, q, cache = _shared_data(c, seed)
        return dict(c=c, q=q, pages=_pack(*cache), table=table, lens=_int(lens), start=_int([s * c["q"] for s in range(c["seqs"] + 1)]), groups=_int(start),
                    shared=_int(shared), most=max(b - a for a, b in zip(start, start[1:])) * c["q"], o=torch.zeros_like(q),
                    lse=torch.zeros(q.shape[:2], dtype=torch.float32, device="cuda"))
    if c["op"] == "select":
        keys, table, q, cache = _select_data(c, seed)
        bounds = _bounds_of(_numbers(cache[0], cache[1]), torch.ones((cache[0].shape[0], c["page"]), dtype=torch.bool, device="cuda"))
        for s, k in enumerate(keys):                      # the step's new key is in none yet
            if k:
                bounds[table[s, (k - 1) // c["page"]].long()] = 0
        T = c["seqs"]
        return dict(c=c, q=q, pages=_pack(*cache), table=table, bounds=bounds, lens=_int(keys), before=_int([max(0, k - 1) for k in keys]),
                    pos=_int([k - 1 for k in keys]), scores=torch.zeros((T, c["Hkv"], table.shape[1]), dtype=torch.float32, device="cuda"),
                    picked=torch.zeros((T, c["Hkv"], c["blocks"]), dtype=torch.int32, device="cuda"), picked_lens=torch.zeros(T, dtype=torch.int32, device="cuda"))
    keys, lists, q, cache = _blocks_data(c, seed)
    return dict(c=c, q=q, pages=_pack(*cache), lists=lists, lens=_int(keys), o=torch.zeros_like(q), lse=torch.zeros(q.shape[:2], dtype=torch.float32, device="cuda"))


# ---- a pass in plain form ----------------------------------------------------------------------------
def _copy_plain(s):
    c, pages = s["c"], s["pages"]
    tiles = -(-c["tokens"] // 16) if c["tokens"] else c["page"] // 16
    src, dst = s["src"].long(), s["dst"].long()
    for layer in pages:
        layer[dst, :, :tiles] = layer[src, :, :tiles]
    return pages


def _places(c, pos, seq, table):
    """For tokens' rows: where in a layer's pages, counted in 16-bit words, all that they have is, [tokens, Hkv, 18 NB]."""
    nb, P, dev = c["D"] // 32, c["page"], pos.device
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
    return tile.unsqueeze(2) + torch.cat([kc, ks, vc, vs], dim=1).unsqueeze(1)


def _compact_plain(s):
    c, n = s["c"], s["keep"].shape[0]
    start = s["start"].long()
    i = torch.arange(n, device="cuda")
    seq = torch.searchsorted(start, i, right=True) - 1
    to = s["to"].long()[seq] + i - start[seq]
    a, b = _places(c, s["keep"].long(), seq, s["table"]), _places(c, to, seq, s["table"])
    for layer in s["pages"]:
        words = layer.view(-1).view(torch.int16)
        words[b] = words[a]
    return s["pages"]


def _nibbles(x):
    return torch.stack([x & 15, x >> 4], dim=-1).flatten(-2)


def _unpack(t, nb):
    """Tiles [.., tiles, bytes] to keys and values as fp32, [.., tokens, D]."""
    lead = t.shape[:-1]
    k, ks, v, vs = t.split([256 * nb, 32 * nb, 256 * nb, 32 * nb], dim=-1)
    k = _nibbles(k).view(lead + (16, 4, nb, 8)).transpose(-3, -2).reshape(lead + (16, nb, 32))
    k = (k.float() - 8.0) * ks.contiguous().view(torch.float16).float().view(lead + (16, nb, 1))
    v = _nibbles(v).view(lead + (2, 8, 4, nb, 2, 4))
    d = v.dim()
    v = v.permute(*range(d - 6), d - 6, d - 4, d - 2, d - 3, d - 5, d - 1).reshape(lead + (16, nb, 32))
    vs = vs.contiguous().view(torch.float16).float().view(lead + (2, 4, nb, 2)).transpose(-2, -1).reshape(lead + (16, nb, 1))
    shape = lead[:-1] + (lead[-1] * 16, nb * 32)
    return k.reshape(shape), ((v.float() - 8.0) * vs).reshape(shape)


def _attend(sc, seen, v):
    """Scores [.., rows, keys] of which `seen` count, values [.., keys, D]: results, and the log of the sum."""
    sc = sc.masked_fill_(~seen, -math.inf)
    m = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))))
    l = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v)
    return torch.where(l > 0, o / l, torch.zeros_like(o)), (m + torch.log(l)).squeeze(-1)


def _shared_plain(s):
    c, q = s["c"], s["q"]
    n, rep, mq = c["seqs"], c["H"] // c["Hkv"], c["q"]
    # every sequence by itself, its shared keys among its own
    k, v = _unpack(s["pages"][s["table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3), c["D"] // 32)
    lens = s["lens"].long().view(n, 1, 1)
    rows = q.float().view(n, mq, c["Hkv"], rep, c["D"]).permute(0, 2, 3, 1, 4).reshape(n, c["Hkv"], rep * mq, c["D"])
    sc = torch.matmul(rows, k.transpose(2, 3)).mul_(1.0 / math.sqrt(c["D"]))
    at = lens - mq + torch.arange(mq, device="cuda").view(1, mq, 1)
    seen = (torch.arange(k.shape[2], device="cuda") <= at).unsqueeze(1).expand(n, rep, mq, -1).reshape(n, 1, rep * mq, -1)
    o, lse = _attend(sc, seen, v)
    out = {"o": o.view(n, c["Hkv"], rep, mq, c["D"]).permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)}
    if c["lse"]:
        out["lse"] = lse.view(n, c["Hkv"], rep, mq).permute(0, 3, 1, 2).reshape(q.shape[:2])
    return out


def _blocks_plain(s):
    c, q = s["c"], s["q"]
    n, rep = c["seqs"], c["H"] // c["Hkv"]
    head = torch.arange(c["Hkv"], device="cuda").view(1, -1, 1)
    k, v = _unpack(s["pages"][s["lists"].clamp(min=0).long(), head].flatten(2, 3), c["D"] // 32)
    sc = torch.matmul(q.float().view(n, c["Hkv"], rep, c["D"]), k.transpose(2, 3)).mul_(1.0 / math.sqrt(c["D"]))
    seen = (torch.arange(k.shape[2], device="cuda") < s["lens"].view(-1, 1)).view(n, 1, 1, -1)
    o, lse = _attend(sc, seen, v)
    out = {"o": o.reshape(q.shape).to(q.dtype)}
    if c["lse"]:
        out["lse"] = lse.reshape(q.shape[:2])
    return out


def _numbers(codes, scales):
    return ((codes.float() - 8.0).unflatten(-1, (-1, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _bounds_of(k, there):
    """Records of pages' keys k [pages, Hkv, page, D], of the tokens that are there [pages, page]: uint8 [pages, Hkv, 2 D + 16]."""
    there = there.view(there.shape[0], 1, -1, 1)
    hi = k.masked_fill(~there, -math.inf).amax(dim=2)
    lo = k.masked_fill(~there, math.inf).amin(dim=2)
    most = torch.maximum(hi.abs(), lo.abs()).amax(dim=-1, keepdim=True)
    step = most / torch.full_like(most, 127.0)            # (a division, not a product with a rounded 1 / 127)
    some = step > 0
    by = torch.where(some, step, torch.ones_like(step))
    codes = [torch.where(some, f(x / by).clamp_(-127, 127), torch.zeros_like(x)).to(torch.int8).view(torch.uint8) for f, x in ((torch.ceil, hi), (torch.floor, lo))]
    return torch.cat(codes + [step.contiguous().view(torch.uint8), torch.zeros(step.shape[:2] + (12,), dtype=torch.uint8, device=k.device)], dim=-1)


def _pick(c, scores, counts):
    """Which blocks, [tokens, Hkv, blocks] rising, -1 behind them: the first and last ones, then by score, then by index."""
    T, h, n = scores.shape
    i, counts = torch.arange(n, device=scores.device), counts.view(T, 1, 1)
    rank = torch.where((i < c["first"]) | (i >= counts - c["last"]), torch.full_like(scores, math.inf), scores)
    order = rank.masked_fill(i >= counts, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    order = torch.nn.functional.pad(order, (0, max(0, c["blocks"] - n)), value=n)[..., :c["blocks"]]
    taken = torch.arange(c["blocks"], device=scores.device) < counts
    order = torch.where(taken, order, torch.full_like(order, n)).sort(dim=-1).values
    return torch.where(taken, order, torch.full_like(order, -1))


def _select_plain(s):
    c, dev, P = s["c"], s["q"].device, s["c"]["page"]
    T, D, nb = c["seqs"], c["D"], c["D"] // 32
    lens, table = s["lens"].long(), s["table"]
    # bounds of the blocks that have a new key
    at = (lens - 1).clamp(min=0)
    page = table[torch.arange(T, device=dev), at // P].long()
    live = lens > 0
    k, _ = _unpack(s["pages"][page[live]], nb)
    s["bounds"][page[live]] = _bounds_of(k, torch.arange(P, device=dev) <= (at % P)[live].unsqueeze(1))
    # scores
    rows = s["q"].float().view(T, c["Hkv"], -1, D)
    most = rows.abs().amax(dim=(2, 3), keepdim=True)
    qs = most / torch.full_like(most, 127.0)
    whole = torch.where(qs > 0, torch.round(rows / torch.where(qs > 0, qs, torch.ones_like(qs))), torch.zeros_like(rows)).double()
    both = torch.cat([whole.clamp(min=0).sum(dim=2), whole.clamp(max=0).sum(dim=2)], dim=-1)                 # [T, Hkv, 2 D]
    counts = (lens + P - 1) // P
    n = table.shape[1]
    records = s["bounds"][table.clamp(min=0).long()]                                                      # [T, blocks, Hkv, bytes]
    codes = records[..., :2 * D].view(torch.int8).double()
    step = records[..., 2 * D:2 * D + 4].contiguous().view(torch.float32).squeeze(-1).transpose(1, 2)
    total = torch.einsum("tnhd,thd->thn", codes, both)
    scores = total.float() * step * qs.view(T, c["Hkv"], 1)
    there = (torch.arange(n, device=dev) < counts.view(T, 1)).unsqueeze(1)
    scores = torch.where(there, scores, torch.zeros_like(scores))
    order = _pick(c, scores, counts)
    picked = torch.where(order >= 0, table.unsqueeze(1).expand(T, c["Hkv"], n).gather(2, order.clamp(min=0)), torch.full_like(order, -1).int())
    got = torch.clamp(counts, max=c["blocks"])
    return _selected(c, s["bounds"], scores, picked.int(), torch.where(live, (got - 1) * P + at % P + 1, torch.zeros_like(got)).int())


def _selected(c, bounds, scores, picked, lens):
    codes = bounds[..., :2 * c["D"]].view(torch.int8)
    return {"codes": codes, "steps": bounds.view(torch.float32)[..., 2 * c["D"] // 4], "scores": scores, "pages": picked, "lens": lens}


# ---- a pass ------------------------------------------------------------------------------------------
_ctx = None


def _call(s):
    """The same through the library's calls; what describes a call's shapes is made once."""
    global _ctx
    import tensorcore_b200 as tc
    if _ctx is None:
        _ctx = tc.Context()
    c, st, first = s["c"], torch.cuda.current_stream().cuda_stream, "desc" not in s
    if first:
        s["kv"] = tc.kv_desc(s["pages"].shape[1 if c["op"] in ("copy", "compact") else 0], c["page"], c["Hkv"], c["D"])
    if c["op"] == "copy":
        if first:
            s["desc"] = tc.kv_copy_desc(c["pairs"], layers=c["layers"])
        tc.raw_kv_copy(_ctx, s["kv"], s["desc"], s["pages"].data_ptr(), s["src"].data_ptr(), s["dst"].data_ptr(), s["counts"].data_ptr() if c["tokens"] else 0, st)
        return s["pages"]
    if c["op"] == "compact":
        if first:
            s["desc"] = tc.kv_compact_desc(s["keep"].shape[0], c["seqs"], s["table"].shape[1], layers=c["layers"])
        tc.raw_kv_compact(_ctx, s["kv"], s["desc"], s["pages"].data_ptr(), s["table"].data_ptr(), s["to"].data_ptr(), s["start"].data_ptr(), s["keep"].data_ptr(), st)
        return s["pages"]
    if c["op"] == "shared":
        if first:
            s["desc"] = tc.attention_shared_desc(s["q"].shape[0], c["seqs"], s["table"].shape[1], c["H"], s["shared"].shape[0], max_q=c["q"], max_group_q=s["most"],
                                                 dtype=c["dtype"])
        tc.raw_attention_shared(_ctx, s["kv"], s["desc"], s["pages"].data_ptr(), s["q"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(), s["start"].data_ptr(),
                                s["groups"].data_ptr(), s["shared"].data_ptr(), s["o"].data_ptr(), s["lse"].data_ptr() if c["lse"] else 0, st)
        return {"o": s["o"], "lse": s["lse"]} if c["lse"] else {"o": s["o"]}
    if c["op"] == "select":
        if first:
            s["update"] = tc.kv_bounds_desc(c["seqs"], s["table"].shape[1], max_new=1)
            s["desc"] = tc.kv_select_desc(c["seqs"], c["seqs"], s["table"].shape[1], c["H"], c["blocks"], first_blocks=c["first"], last_blocks=c["last"], dtype=c["dtype"])
        tc.raw_kv_bounds(_ctx, s["kv"], s["update"], s["pages"].data_ptr(), s["bounds"].data_ptr(), s["before"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(), st)
        tc.raw_kv_select(_ctx, s["kv"], s["desc"], s["bounds"].data_ptr(), s["q"].data_ptr(), s["pos"].data_ptr(), 0, s["table"].data_ptr(), s["scores"].data_ptr(),
                         s["picked"].data_ptr(), s["picked_lens"].data_ptr(), st)
        return _selected(c, s["bounds"], s["scores"], s["picked"], s["picked_lens"])
    if first:
        s["desc"] = tc.attention_blocks_desc(c["seqs"], c["blocks"], c["H"], dtype=c["dtype"])
    tc.raw_attention_blocks(_ctx, s["kv"], s["desc"], s["pages"].data_ptr(), s["q"].data_ptr(), s["lists"].data_ptr(), s["lens"].data_ptr(), s["o"].data_ptr(),
                            s["lse"].data_ptr() if c["lse"] else 0, st)
    return {"o": s["o"], "lse": s["lse"]} if c["lse"] else {"o": s["o"]}


def run(state):
    if own:
        return _call(state)
    return {"copy": _copy_plain, "compact": _compact_plain, "shared": _shared_plain, "select": _select_plain, "blocks": _blocks_plain}[state["c"]["op"]](state)


# ---- what it costs at least -----------------------------------------------------------------------------
def work(case):
    c = case
    row = c["Hkv"] * c["D"] * 9 // 8                     # keys and values of a token
    if c["op"] == "copy":
        tokens = -(-c["tokens"] // 16) * 16 if c["tokens"] else c["page"]
        return {"bytes": 2 * c["pairs"] * c["layers"] * tokens * row, "flops": 0}
    if c["op"] == "compact":
        n = sum(k != to + j for _, to, keep in _moves(c) for j, k in enumerate(keep))
        return {"bytes": 2 * n * c["layers"] * row, "flops": 0}
    if c["op"] == "shared":
        start, shared, lens = _family(c)
        T = c["seqs"] * c["q"]
        rest = sum(lens) - sum(p * (b - a) for p, a, b in zip(shared, start, start[1:]))
        pairs = sum(k - c["q"] + i + 1 for k in lens for i in range(c["q"]))
        return {"bytes": (sum(shared) + rest) * row + 4 * T * c["H"] * c["D"] + (4 * T * c["H"] if c["lse"] else 0), "flops": 4 * c["H"] * c["D"] * pairs}
    if c["op"] == "select":
        n, P = [-(-k // c["page"]) for k in _contexts(c)], c["page"]
        fresh = sum((k - 1) % P + 1 for k in _contexts(c) if k)
        return {"bytes": sum(n) * c["Hkv"] * (2 * c["D"] + 8) + fresh * row // 2 + c["seqs"] * (2 * c["H"] * c["D"] + 4 * c["Hkv"] * c["blocks"]),
                "flops": 4 * sum(n) * c["Hkv"] * c["D"]}
    keys = sum(_chosen(c)[1])
    return {"bytes": keys * row + 4 * c["seqs"] * c["H"] * c["D"] + (4 * c["seqs"] * c["H"] if c["lse"] else 0), "flops": 4 * c["H"] * c["D"] * keys}


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _row_parts(layer, nb):
    """A layer's pages by what a token has in them: four views whose indexes include the token's."""
    k, ks, v, vs = layer.split([256 * nb, 32 * nb, 256 * nb, 32 * nb], dim=-1)
    return k.unflatten(-1, (16, -1)), ks.unflatten(-1, (16, -1)), v.unflatten(-1, (2, 8, 4, nb, 2, 2)), vs.unflatten(-1, (2, 4, nb, 2, 2))


def _keys64(codes, scales, own_pages):
    x = (codes[own_pages].double() - 8.0).unflatten(-1, (-1, 32)) * scales[own_pages].double().unsqueeze(-1)
    return x.flatten(-2).transpose(0, 1).flatten(1, 2)                          # [Hkv, tokens, D]


def _softmax64(q, k, v, hidden):
    """q [Hkv, rows, D], k and v [Hkv, keys, D]."""
    sc = torch.einsum("hrd,hjd->hrj", q, k) / math.sqrt(q.shape[-1])
    if hidden is not None:
        sc = sc.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(sc, dim=-1)
    return torch.einsum("hrj,hjd->hrd", torch.exp(sc - lse.unsqueeze(-1)), v), lse


def _f32(x):
    return x.float().double()


def exact(case, seed):
    c = case
    rep, nb = c.get("H", 0) // c["Hkv"], c["D"] // 32
    if c["op"] == "copy":
        s = prepare(c, seed)
        tokens = -(-c["tokens"] // 16) if c["tokens"] else c["page"] // 16
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            s["pages"][:, b, :, :tokens].copy_(s["pages"][:, a, :, :tokens])
        return s["pages"]
    if c["op"] == "compact":
        s, old = prepare(c, seed), None
        moves, table = _moves(c), s["table"].long()
        pos = torch.tensor([k for m in moves for k in m[2]], device="cuda")
        to = torch.tensor([m[1] + j for m in moves for j in range(len(m[2]))], device="cuda")
        seq = torch.tensor([i for i, m in enumerate(moves) for _ in m[2]], device="cuda")

        def where(p):
            r = p % 16
            return table[seq, p // c["page"]], p % c["page"] // 16, r, r // 8, r % 8 // 2, r % 2
        (pa, ta, ra, ha, qa, ea), (pb, tb, rb, hb, qb, eb) = where(pos), where(to)
        for layer in s["pages"]:
            old = _row_parts(layer.clone(), nb)
            k, ks, v, vs = _row_parts(layer, nb)
            k[pb, :, tb, rb] = old[0][pa, :, ta, ra]
            ks[pb, :, tb, rb] = old[1][pa, :, ta, ra]
            v[pb, :, tb, hb, :, qb, :, eb] = old[2][pa, :, ta, ha, :, qa, :, ea]
            vs[pb, :, tb, hb, qb, :, eb] = old[3][pa, :, ta, ha, qa, :, ea]
        return s["pages"]
    if c["op"] == "shared":
        _, _, lens, table, q, (kc, ks, vc, vs) = _shared_data(c, seed)
        o, lse, mq = [], [], c["q"]
        for s, n in enumerate(lens):
            own_pages = table[s, :-(-n // c["page"])].long()
            k, v = _keys64(kc, ks, own_pages)[:, :n], _keys64(vc, vs, own_pages)[:, :n]
            rows = q[s * mq:(s + 1) * mq].double().view(mq, c["Hkv"], rep, c["D"]).transpose(0, 1).flatten(1, 2)
            i = torch.arange(n - mq, n, device="cuda").repeat_interleave(rep).view(-1, 1)
            got, l = _softmax64(rows, k, v, torch.arange(n, device="cuda") > i)
            o.append(got.unflatten(1, (mq, rep)).transpose(0, 1).reshape(mq, c["H"], c["D"]))
            lse.append(l.unflatten(1, (mq, rep)).transpose(0, 1).reshape(mq, c["H"]))
        return {"o": torch.cat(o), "lse": torch.cat(lse)} if c["lse"] else {"o": torch.cat(o)}
    if c["op"] == "blocks":
        keys, lists, q, (kc, ks, vc, vs) = _blocks_data(c, seed)
        o, lse = torch.zeros((c["seqs"], c["H"], c["D"]), dtype=torch.float64, device="cuda"), torch.zeros((c["seqs"], c["H"]), dtype=torch.float64, device="cuda")
        for t, n in enumerate(keys):
            m = -(-n // c["page"])
            for h in range(c["Hkv"]):
                mine = lists[t, h, :m].long()
                k, v = (_keys64(x[:, h:h + 1], d[:, h:h + 1], mine)[:, :n] for x, d in ((kc, ks), (vc, vs)))
                got, l = _softmax64(q[t, h * rep:(h + 1) * rep].double().unsqueeze(0), k, v, None)
                o[t, h * rep:(h + 1) * rep], lse[t, h * rep:(h + 1) * rep] = got[0], l[0]
        return {"o": o, "lse": lse} if c["lse"] else {"o": o}
    # Bounds and scores are defined by fp32 steps: each in 64 bits and rounded.
    s = prepare(c, seed)
    keys, table, q, (kc, ks, _, _) = _select_data(c, seed)
    P, D, bounds = c["page"], c["D"], s["bounds"]
    scores = torch.zeros((c["seqs"], c["Hkv"], table.shape[1]), dtype=torch.float32, device="cuda")
    picked = torch.full((c["seqs"], c["Hkv"], c["blocks"]), -1, dtype=torch.int32, device="cuda")
    picked_lens = torch.zeros(c["seqs"], dtype=torch.int32, device="cuda")
    for t, n in enumerate(keys):
        if n == 0:
            continue
        m, mine = -(-n // P), table[t].long()
        x = _keys64(kc, ks, mine[m - 1:m])[:, :n - (m - 1) * P]
        hi, lo = x.max(dim=1).values, x.min(dim=1).values
        step = _f32(x.abs().flatten(1).max(dim=1, keepdim=True).values / 127.0)
        code = torch.cat([torch.ceil(_f32(hi / step)), torch.floor(_f32(lo / step))], dim=1).clamp(-127, 127)
        bounds[mine[m - 1], :, :2 * D] = code.to(torch.int8).view(torch.uint8)
        bounds[mine[m - 1], :, 2 * D:2 * D + 4] = step.float().view(torch.uint8)
        record = bounds[mine[:m]]
        code, step = record[..., :2 * D].view(torch.int8).double(), record[..., 2 * D:2 * D + 4].contiguous().view(torch.float32).double().squeeze(-1)
        for h in range(c["Hkv"]):
            rows = q[t, h * rep:(h + 1) * rep].double()
            qs = _f32(rows.abs().max() / 127.0)
            whole = torch.round(_f32(rows / qs))
            total = torch.maximum(whole.unsqueeze(1) * code[:, h, :D], whole.unsqueeze(1) * code[:, h, D:]).sum(dim=(0, 2))
            mark = _f32(_f32(_f32(total) * step[:, h]) * qs)
            scores[t, h, :m] = mark.float()
            left = sorted(range(m), key=lambda i, v=mark.tolist(): (not (i < c["first"] or i >= m - c["last"]), -v[i], i))
            take = sorted(left[:c["blocks"]])
            picked[t, h, :len(take)] = table[t, torch.tensor(take, device="cuda")]
        picked_lens[t] = (min(m, c["blocks"]) - 1) * P + (n - 1) % P + 1
    return _selected(c, bounds, scores, picked, picked_lens)
