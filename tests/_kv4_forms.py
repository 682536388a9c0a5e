"""Inputs and 64-bit results for tests/test_kv4_forms_{cpu,gpu}.py: the attention's bound with the precision that its kernels claim for p, expected pages of large writes, and
inputs on which that precision shows."""
import torch

import _kv4 as R

bf16 = torch.bfloat16


def attend(q, pages, tables, lens, scale, alibi=None, shared=None):
    """-> o float64 [rows, heads, hd], bound, and o with every p cut to the eight significant bits of one bf16.

    bound: the result is rounded to bf16, half a step: 2^-8 |o|.  p is held in two bf16 that are cut, not rounded: the first keeps 8 significant bits, what it leaves is below 2^-7 of it
    and keeps 8 more, so what is lost is below 2^-15 p.  Sums of n terms in 32 bits, over p v and over p: 2 n 2^-24, and 64 more for the joins.  A score is off by e: q held to 2^-17 of its
    32-block's largest magnitude, hd + 8 products and sums in 32 bits, the exponent's argument (of magnitude 10 or less at the largest score, plus the distance from it)
    and the exponential itself: 2^-19 (1 + distance); the normaliser moves with them.  2^-110: a p v is held in 32 bits, the smallest magnitudes are lost."""
    rows, heads, hd = q.shape
    kvh = pages.shape[1]
    G = heads // kvh
    o, cut, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape, 2.0 ** -110, dtype=torch.float64)
    qd = q.double()
    qb = torch.cat([qd[..., 32 * b:32 * b + 32].abs().amax(-1, keepdim=True).expand(-1, -1, min(32, hd - 32 * b)) for b in range(R.blocks(hd))], -1)
    for r in range(rows):
        n = int(lens[r])
        if n == 0:
            continue
        k, v = R.unpack(pages[tables[r, :(n + 31) // 32].long()], hd)
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(G, 0) for x in (k, v))          # [heads, n, hd]
        s = (k @ qd[r, :, :, None])[..., 0] * scale
        e = 2.0 ** -17 * (k.abs() @ qb[r, :, :, None])[..., 0] * scale + (hd + 8) * 2.0 ** -24 * (k.abs() @ qd[r, :, :, None].abs())[..., 0] * scale
        if alibi is not None:
            back = alibi.double()[:, None] * torch.arange(n - 1, -1, -1, dtype=torch.float64)
            s, e = s - back, e + 2.0 ** -22 * back.abs()
        top = s.amax(-1, keepdim=True)
        e = e + 2.0 ** -19 * (1 + top - s)
        p = torch.exp(s - top)
        low = (p.float().view(torch.int32) & -65536).view(torch.float32).double()
        total = p.sum(-1, keepdim=True)
        p = p / total
        spread = (p * e).sum(-1, keepdim=True) + e
        o[r] = (p[:, None] @ v)[:, 0]
        cut[r] = ((low / total)[:, None] @ v)[:, 0]
        bound[r] += 2.0 ** -8 * o[r].abs() + ((p * (2.0 ** -15 + (2 * n + 64) * 2.0 ** -24 + 2 * spread))[:, None] @ v.abs())[:, 0]
    return o, bound, cut


def opposite(n_pages, kvh, hd, seed):
    """pages whose values cancel: the second half of them holds the negated values of the first half, tokens in another order.  With scores close to each other the result is far
    below the terms it is summed of, and an error of every p shows beside the result's own rounding."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(n_pages, kvh, 32, hd, generator=g).to(bf16) for _ in range(2))
    half = n_pages // 2
    for i in range(half):
        v[half + i] = -v[i][:, torch.randperm(32, generator=g)]
    return R.pack(k, v)


# head dim, query heads to a key head: every split of p and of the scale blocks over the product's columns
ROWS = [(hd, G) for hd in (64, 80, 128) for G in (1, 2, 4, 6, 8, 16)]
# head dim, rows of a group, groups, key heads, query heads to a key head, columns of the table: read once per group, in every such split
GROUPS = [(80, 2, 8, 32, 1, 16), (128, 4, 4, 32, 1, 16), (128, 8, 2, 32, 1, 16), (64, 10, 2, 32, 1, 13), (64, 8, 2, 32, 1, 16), (80, 5, 2, 32, 3, 26), (128, 2, 2, 32, 8, 64), (128, 2, 2, 32, 4, 64)]


def rows_case(hd, G):
    rows, kvh = 3, 4
    pages = opposite(6 * rows, kvh, hd, seed=hd + G).view(6, rows, kvh, -1).transpose(0, 1)                     # [rows, 6]: halves 0 ... 2 and 3 ... 5
    pages = pages.reshape(6 * rows, kvh, -1).contiguous()
    g = torch.Generator().manual_seed(G)
    q = (0.02 * torch.randn(rows, kvh * G, hd, generator=g)).to(bf16)
    return q, pages, torch.arange(6 * rows, dtype=torch.int32).view(rows, 6), torch.tensor([192, 191, 160], dtype=torch.int32)


def groups_case(hd, K, groups, kvh, G, width):
    """shared columns: 12 that cancel; one or two columns of a row's own; the rest of the table is unused"""
    g = torch.Generator().manual_seed(width + K)
    rows = K * groups
    pages = opposite(12 + 2 * rows, kvh, hd, seed=K)
    half = pages.shape[0] // 2
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    both = torch.cat([torch.arange(6), half + torch.arange(6)]).to(torch.int32)
    for r in range(rows):
        tables[r, :12] = both
        tables[r, 12] = 6 + int(torch.randint(0, half - 6, (1,), generator=g))
    lens = torch.tensor([384 + 1 + (5 * r) % 32 for r in range(rows)], dtype=torch.int32)
    q = (0.02 * torch.randn(rows, kvh * G, hd, generator=g)).to(bf16)
    return q, pages, tables, lens, torch.full((groups,), 384 + 7, dtype=torch.int32)


def write_pages(before, slots, k, v):
    """the pages after k, v [tokens, heads, hd] went into slots: nothing else changes"""
    n_pages, heads, nbytes = before.shape
    hd = k.shape[-1]
    kb, ksh, vb, vsh, ks, vs = R._where(hd)
    nib = torch.stack([before & 15, before >> 4], -1).view(n_pages, heads, 2 * nbytes).clone()
    ok = (slots >= 0) & (slots < n_pages * 32)
    s = slots[ok]
    h = torch.arange(heads)[None, :, None]
    page, t = (s // 32)[:, None, None], s % 32
    for x, at, sh, scale_at in ((k, kb, ksh, ks), (v, vb, vsh, vs)):
        codes, scales = R.quantise(x[ok])
        where = (2 * at + sh // 4).view(32, hd)[t][:, None]
        nib[page, h, where] = codes.to(torch.uint8)
        where = 2 * scale_at.view(32, -1)[t][:, None]
        nib[page, h, where], nib[page, h, where + 1] = (scales & 15).to(torch.uint8), (scales >> 4).to(torch.uint8)
    nib = nib.view(n_pages, heads, nbytes, 2)
    return nib[..., 0] | nib[..., 1] << 4


def rotated(x, cos, sin, rot):
    """x [rows, heads, hd] float64, half-split pairs of the first rot dims turned by the rows' fp32 tables"""
    c, s, h = cos.double()[:, None], sin.double()[:, None], rot // 2
    return torch.cat([x[..., :h] * c - x[..., h:rot] * s, x[..., h:rot] * c + x[..., :h] * s, x[..., rot:]], -1)


def saturated(x):
    """values outside bf16's range, which only a rotation makes: their block's exponent stays 125, codes saturate at 6"""
    return x.clamp(-6 * 2.0 ** 125, 6 * 2.0 ** 125)
