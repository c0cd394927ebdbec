"""Plain forms, in numpy and 64 bits or bit by bit in fp32, of the rotary, cache and paged-attention calls."""
import numpy as np


def turn64(x, cos, sin, positions, rot, layout, inverse=False):
    """x [tokens, heads, D] turned by positions; and what one fp32 evaluation can be off by at most, before its result is rounded."""
    x = x.astype(np.float64)
    c, s = cos[positions][:, None, :].astype(np.float64), sin[positions][:, None, :].astype(np.float64) * (-1 if inverse else 1)
    i = np.arange(rot // 2) if layout == "half" else 2 * np.arange(rot // 2)
    j = i + rot // 2 if layout == "half" else i + 1
    y, room = x.copy(), np.zeros_like(x)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    # two products and a sum, each rounded once (2^-24 of its size)
    room[..., i] = 2 * 2.0 ** -24 * (abs(x[..., i] * c) + abs(x[..., j] * s))
    room[..., j] = 2 * 2.0 ** -24 * (abs(x[..., i] * s) + abs(x[..., j] * c))
    return y, room


def turn32(x, cos, sin, positions, rot, layout):
    """The same with every fp32 operation rounded by itself: what the library's bits have to be."""
    x = x.astype(np.float32)
    c, s = cos[positions][:, None, :], sin[positions][:, None, :]
    i = np.arange(rot // 2) if layout == "half" else 2 * np.arange(rot // 2)
    j = i + rot // 2 if layout == "half" else i + 1
    y = x.copy()
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def quantise(x):
    """Blocks of 32 along the last axis, fp32 step by step: codes (uint8, as x) and fp16 scales."""
    b = x.astype(np.float32).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    with np.errstate(all="ignore"):
        most = abs(b).max(axis=-1, keepdims=True)                      # a NaN wins
        scale = (most / np.float32(8)).astype(np.float32)
        inv = np.where(scale > 0, np.float32(8) / most, np.float32(0)).astype(np.float32)
        y = (b * inv).astype(np.float32).astype(np.float64)
        whole = np.trunc(y)
        whole += np.sign(y) * (abs(y - whole) >= 0.5)
        code = np.clip(np.nan_to_num(whole, nan=0.0) + 8, 0, 15).astype(np.uint8)
        return code.reshape(x.shape), scale[..., 0].astype(np.float16)


def numbers(codes, scales):
    """What codes and scales stand for, exactly (fp64)."""
    b = codes.reshape(codes.shape[:-1] + (codes.shape[-1] // 32, 32)).astype(np.float64) - 8
    with np.errstate(all="ignore"):
        return (b * scales.astype(np.float64)[..., None]).reshape(codes.shape)


def pack(kc, ks, vc, vs):
    """Codes [pages, heads, tokens, D] and scales [.., D / 32] into pages, one byte at a time by the documented places."""
    n, h, P, D = kc.shape
    nb = D // 32
    out = np.zeros((n, h, P // 16, 576 * nb), np.uint8)
    for token in range(P):
        tile, r = out[:, :, token // 16], token % 16
        hh, t, e = r // 8, r % 8 // 2, r % 2
        for d in range(D):
            block, in_block = d // 32, d % 32
            at = ((r * 4 + in_block // 8) * nb + block) * 4 + in_block % 8 // 2
            tile[:, :, at] |= kc[:, :, token, d] << (4 * (in_block % 2))
            at = 288 * nb + ((((hh * 8 + in_block // 4) * 4 + t) * nb + block) * 2 + e) * 2 + in_block % 4 // 2
            tile[:, :, at] |= vc[:, :, token, d] << (4 * (in_block % 2))
        for block in range(nb):
            at = 256 * nb + (r * nb + block) * 2
            tile[:, :, at:at + 2] = np.ascontiguousarray(ks[:, :, token, block]).view(np.uint8).reshape(n, h, 2)
            at = 544 * nb + (((hh * 4 + t) * nb + block) * 2 + e) * 2
            tile[:, :, at:at + 2] = np.ascontiguousarray(vs[:, :, token, block]).view(np.uint8).reshape(n, h, 2)
    return out


def attention64(q, k, v, scale, causal, window):
    """q [tokens, H, D], k and v [Hkv, keys, D] of one sequence (fp64): O, LSE, and how far an evaluation may be off whose scores are off by
    2^-11 of their terms and whose values and weights by 2^-11 each."""
    nq, H, D = q.shape
    Hkv, nk, _ = k.shape
    rep = H // Hkv
    kk, vv = np.repeat(k, rep, axis=0), np.repeat(v, rep, axis=0)                # [H, keys, D]
    s = np.einsum("ihd,hjd->ihj", q, kk) * scale
    at, j = np.arange(nk - nq, nk)[:, None], np.arange(nk)[None, :]
    seen = np.ones((nq, nk), bool)
    if causal:
        seen &= j <= at
    if window > 0:
        seen &= at - j <= window
    s = np.where(seen[:, None, :], s, -np.inf)
    m = s.max(axis=-1, keepdims=True, initial=-np.inf)
    p = np.where(seen[:, None, :], np.exp(s - np.where(m > -np.inf, m, 0.0)), 0.0)
    l = p.sum(axis=-1, keepdims=True)
    some = l > 0
    p = np.where(some, p / np.where(some, l, 1), 0)
    o = np.einsum("ihj,hjd->ihd", p, vv)
    with np.errstate(all="ignore"):
        lse = np.where(some, m + np.log(np.where(some, l, 1)), -np.inf)[..., 0]
    u = 2.0 ** -11
    es = np.where(seen[:, None, :], u * scale * np.einsum("ihd,hjd->ihj", abs(q), abs(kk)), 0)
    off = es.max(axis=-1, initial=0.0)                                           # of a score
    room = (np.expm1(2 * off)[..., None] + 2 * u) * np.einsum("ihj,hjd->ihd", p, abs(vv))
    return o, lse, room, off
