"""64-bit CPU restatement of the 4-bit page cache for the kv4 tests: the format from its definition (include/unimp_hip.h, unimp_amd/csrc/kv4.h), token by token."""
import math

import torch

PAGE = 32
MAG = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def blocks(hd):
    return (hd + 31) // 32


def page_bytes(hd):
    return 32 * hd + 64 * blocks(hd)


def quantise(x):
    """x [..., hd] (any float type) -> codes [..., hd] int64, scale bytes [..., blocks] int64"""
    x = x.double()
    codes, scales = torch.zeros(x.shape, dtype=torch.int64), torch.zeros(x.shape[:-1] + (blocks(x.shape[-1]),), dtype=torch.int64)
    for b in range(blocks(x.shape[-1])):
        y = x[..., 32 * b:32 * b + 32]
        bad = ~torch.isfinite(y).all(-1)
        top = torch.where(bad[..., None], torch.ones_like(y), y).abs().amax(-1)
        e = torch.where(top > 0, torch.frexp(top)[1] - 3, torch.full_like(top, -125).int()).clamp(min=-125)
        a = (y * torch.ldexp(torch.ones_like(top), -e)[..., None]).abs()
        off = (a[..., None] - MAG).abs()
        off = torch.where(torch.isnan(off), torch.zeros_like(off), off)
        low = off.amin(-1, keepdim=True)
        # nearest; of two equally near codes the even one
        c = torch.where(off[..., 0::2].amin(-1) == low[..., 0], 2 * (off[..., 0::2] == low).int().argmax(-1), 2 * (off[..., 1::2] == low).int().argmax(-1) + 1)
        c = torch.where(a > 6, torch.full_like(c, 7), c) + 8 * (y < 0)
        codes[..., 32 * b:32 * b + 32] = torch.where(bad[..., None], torch.zeros_like(c), c)
        scales[..., b] = torch.where(bad, torch.full_like(e, 255), e + 127).long()
    return codes, scales


def values(codes, scales):
    hd = codes.shape[-1]
    v = torch.where(codes >= 8, -MAG[codes & 7], MAG[codes & 7])
    s = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.float64), torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales - 127))
    return v * s.repeat_interleave(32, -1)[..., :hd]


def held(x):
    """what the cache holds of x"""
    return values(*quantise(x))


def put(page, t, k, v):
    """k, v [hd] into token t of ONE page (uint8 [page bytes], CPU)"""
    hd, nb = k.shape[-1], blocks(k.shape[-1])
    (kc, ks), (vc, vs) = quantise(k), quantise(v)
    g, nib = (t % 16) // 4, 4 * (t // 16) + t % 4
    for d in range(hd):
        at = 512 * (d // 32) + t * (min(32, hd - d // 32 * 32) // 2) + (d % 32) // 2
        page[at] = int(page[at]) & (0xf0 if d % 2 == 0 else 0x0f) | int(kc[d]) << 4 * (d % 2)
        at = 16 * hd + 4 * (g * hd + (d % 16) * (hd // 16) + d // 16) + nib // 2
        page[at] = int(page[at]) & (0xf0 if nib % 2 == 0 else 0x0f) | int(vc[d]) << 4 * (nib % 2)
    for b in range(nb):
        page[32 * hd + 32 * b + 2 * (t % 16) + t // 16] = int(ks[b])
        page[32 * hd + 32 * nb + 8 * nb * g + 8 * b + nib] = int(vs[b])


_WHERE = {}


def _where(hd):
    if hd not in _WHERE:
        nb, idx = blocks(hd), [[], [], [], [], [], []]
        for t in range(PAGE):
            g, nib = (t % 16) // 4, 4 * (t // 16) + t % 4
            for d in range(hd):
                idx[0].append(512 * (d // 32) + t * (min(32, hd - d // 32 * 32) // 2) + (d % 32) // 2), idx[1].append(4 * (d % 2))
                idx[2].append(16 * hd + 4 * (g * hd + (d % 16) * (hd // 16) + d // 16) + nib // 2), idx[3].append(4 * (nib % 2))
            for b in range(nb):
                idx[4].append(32 * hd + 32 * b + 2 * (t % 16) + t // 16), idx[5].append(32 * hd + 32 * nb + 8 * nb * g + 8 * b + nib)
        _WHERE[hd] = [torch.tensor(i) for i in idx]
    return _WHERE[hd]


def unpack(pages, hd):
    """pages uint8 [..., page bytes] (CPU) -> the values they hold, k and v [..., 32, hd] float64"""
    kb, ksh, vb, vsh, ks, vs = _where(hd)
    p = pages.long()
    f = lambda x, n: x.unflatten(-1, (PAGE, n))
    return (values(f((p[..., kb] >> ksh) & 15, hd), f(p[..., ks], blocks(hd))), values(f((p[..., vb] >> vsh) & 15, hd), f(p[..., vs], blocks(hd))))


def pack(k, v):
    """k, v [..., 32, hd] -> pages uint8 [..., page bytes] (CPU)"""
    hd = k.shape[-1]
    kb, ksh, vb, vsh, ks, vs = _where(hd)
    page = torch.zeros(k.shape[:-2] + (page_bytes(hd),), dtype=torch.int64)
    (kc, ksc), (vc, vsc) = quantise(k), quantise(v)
    for at, sh, c in ((kb, ksh, kc), (vb, vsh, vc)):
        page.index_add_(-1, at, c.flatten(-2) << sh)              # the nibbles of a byte are disjoint: their sum is their union
    page[..., ks], page[..., vs] = ksc.flatten(-2), vsc.flatten(-2)
    return page.to(torch.uint8)


def attend(q, pages, tables, lens, scale, alibi=None, width=None):
    """-> (o float64 [rows, heads, hd], bound [rows, heads, hd]): bound = how far a kernel may be off that forms the scores in fp32 from q held to 2^-17 of its
    32-block's largest magnitude, weights each token with p rounded to bf16, sums in fp32 and rounds the result to bf16 (half a step each: 2^-8)."""
    rows, heads, hd = q.shape
    n_pages, kvh = pages.shape[:2]
    G, width = heads // kvh, tables.shape[1] if width is None else width
    o, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for r in range(rows):
        n = min(max(int(lens[r]), 0), width * PAGE)
        if n == 0:
            continue
        cols = (n + PAGE - 1) // PAGE
        ids = tables[r, :cols].long()
        there = ((ids >= 0) & (ids < n_pages)).repeat_interleave(PAGE)[:n]
        if not bool(there.any()):
            continue
        k, v = unpack(pages[ids.clamp(0, n_pages - 1)], hd)        # [cols, kvh, 32, hd]
        k, v = (x.transpose(1, 2).flatten(0, 1)[:n][there] for x in (k, v))
        j = torch.arange(n, dtype=torch.float64)[there]
        for h in range(heads):
            qq, kk, vv = q[r, h].double(), k[:, h // G], v[:, h // G]
            s = (kk @ qq) * scale
            if alibi is not None:
                s = s + float(alibi[h]) * (j - (n - 1))
            p = torch.softmax(s, 0)
            o[r, h] = p @ vv
            qb = torch.zeros(hd, dtype=torch.float64)
            for b in range(blocks(hd)):
                qb[32 * b:32 * b + 32] = qq[32 * b:32 * b + 32].abs().amax()
            e = 2.0 ** -17 * (kk.abs() @ qb) * scale + (hd + 8) * 2.0 ** -24 * (kk.abs() @ qq.abs()) * scale        # of a score
            if alibi is not None:
                e = e + 2.0 ** -22 * (float(alibi[h]) * (n - 1 - j)).abs()
            e = e + 2.0 ** -21 * (1 + (s.amax() - s))              # exponent's argument and the exponential itself
            spread = (p * e).sum() + e                             # the normaliser moves as well
            bound[r, h] = 2.0 ** -8 * o[r, h].abs() + ((2.0 ** -8 + 2 * spread) * p) @ vv.abs() + 1e-30
    return o, bound
