"""The paged 4-bit decode cache on an MI355X: every kernel against the 64-bit restatement of tests/_kv4.py.

Codes, scales, page ids and slots are compared bit for bit.  Attention: per element, against a bound counted from the roundings (tests/_kv4.py attend)."""
import pytest
import torch

import _kv4 as R

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from unimp_amd import ops as o
    return o


def rnd(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(bf16)


def nan_equal(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a.double(), nan=0.0), torch.nan_to_num(b.double(), nan=0.0))


def paged(rows, width, kvh, hd, seed, extra=3, garbage=True):
    """a pool of rows * width + extra pages with random contents, and tables that name them in random order"""
    g = torch.Generator().manual_seed(seed)
    n = rows * width + extra
    k = torch.randn(n, kvh, 32, hd, generator=g) * torch.exp(0.5 * torch.randn(1, kvh, 1, hd, generator=g))
    pages = R.pack(k.to(bf16), torch.randn(n, kvh, 32, hd, generator=g).to(bf16))
    return pages, torch.randperm(n, generator=g)[:rows * width].view(rows, width).to(torch.int32)


def check(got, want, bound, name=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), name
    far = (got - want).abs() - bound
    assert far.max().item() <= 0, (name, (got - want).abs().max().item(), int(far.argmax()), far.max().item())


# ------------------------------------------------------------------------------------------------- write, read
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("tokens,heads,order", [(1, 1, "run"), (31, 3, "run"), (32, 2, "run"), (33, 2, "offset"), (100, 4, "offset"), (257, 2, "gaps"), (97, 3, "random"), (400, 5, "pieces")])
def test_write_read(ops, hd, tokens, heads, order):
    """runs of any length that start anywhere in a page, with padding between requests, and slots in random order; nothing but the named slots changes"""
    n_pages = (tokens + 40) // 32 + 3 if order != "pieces" else tokens
    g = torch.Generator().manual_seed(tokens)
    page = torch.randperm(n_pages, generator=g)
    first = {"run": 0, "offset": 13, "gaps": 5, "random": 0, "pieces": 0}[order]
    t = torch.arange(first, first + tokens)
    slots = page[t // 32] * 32 + t % 32
    if order == "random":
        slots = torch.randperm(n_pages * 32, generator=g)[:tokens]
    if order == "pieces":                                           # runs of 1 ... 16 tokens anywhere in their pages: whole, or in two parts the second of which comes first
        parts = []
        for pg in page.tolist():
            a, n = (int(x) for x in torch.randint(1, 17, (2,), generator=g))
            r = pg * 32 + a - 1 + torch.arange(n)
            parts.append(r if pg % 3 else torch.cat([r[n // 2:], r[:n // 2]]))
        slots = torch.cat(parts)[:tokens].contiguous()
    if order == "gaps":
        slots[torch.rand(tokens, generator=g) < 0.2] = -1
        slots[7] = n_pages * 32
        slots[9] = -(1 << 40)
    k, v = rnd(tokens, heads, hd, seed=1, scale=3.0), rnd(tokens, heads, hd, seed=2)
    before = torch.randint(0, 256, (n_pages, heads, R.page_bytes(hd)), generator=g).to(torch.uint8)
    want = before.clone()
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < n_pages * 32:
            for h in range(heads):
                R.put(want[s // 32, h], s % 32, k[i, h], v[i, h])
    pages = before.cuda()
    ops.kv4_write(k.cuda(), v.cuda(), pages, slots.cuda())
    assert torch.equal(pages.cpu(), want)
    ok = ((slots >= 0) & (slots < n_pages * 32))[:, None, None]
    gk, gv = ops.kv4_read(pages, slots.cuda(), hd)
    assert torch.equal(gk.cpu().double(), torch.where(ok, R.held(k), torch.zeros((), dtype=torch.float64)))
    assert torch.equal(gv.cpu().double(), torch.where(ok, R.held(v), torch.zeros((), dtype=torch.float64)))


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_write_every_magnitude(ops, hd):
    """all finite bf16 values, block maxima from the largest down to subnormals and zero; infinities and NaN make their block NaN and no other"""
    bits = torch.arange(0, 1 << 15, dtype=torch.int32)
    x = torch.cat([bits, bits + (1 << 15)]).to(torch.int16).view(bf16)
    x = x[torch.isfinite(x)]
    T = x.numel() // hd
    k = x[:T * hd].view(T, 1, hd)
    g = torch.Generator().manual_seed(3)
    v = x[torch.randperm(x.numel(), generator=g)][:T * hd].view(T, 1, hd).clone()
    v[5, 0, 3], v[6, 0, hd - 1], v[7, 0, 33] = float("inf"), float("-inf"), float("nan")
    v[8], k[9] = 0, 0
    slots = torch.arange(T)
    pages = torch.zeros(((T + 31) // 32, 1, R.page_bytes(hd)), dtype=torch.uint8, device="cuda")
    ops.kv4_write(k.cuda(), v.cuda(), pages, slots.cuda())
    gk, gv = ops.kv4_read(pages, slots.cuda(), hd)
    assert nan_equal(gk.cpu(), R.held(k)) and nan_equal(gv.cpu(), R.held(v))
    assert torch.isnan(gv[5, 0, :32]).all() and not torch.isnan(gv[5, 0, 32:]).any() and torch.isnan(gv[6, 0, hd - 1])


def test_write_views_and_layers(ops):
    """strided views (a prefill cache [rows, capacity, heads, hd]), one layer of a pool, two calls that fill one page"""
    hd, heads, L = 80, 4, 45
    cache = rnd(2, 2, 60, heads, hd, seed=4).cuda()
    pool = torch.zeros((3, 4, heads, R.page_bytes(hd)), dtype=torch.uint8, device="cuda")
    slots = torch.arange(2 * 64).view(2, 64)[:, :L]
    for r in range(2):
        for a, b in ((0, 17), (17, L)):
            ops.kv4_write(cache[0, r, a:b], cache[1, r, a:b], pool[1], slots[r, a:b].contiguous().cuda())
    gk, gv = ops.kv4_read(pool, slots.reshape(-1).cuda(), hd)
    assert gk.shape == (3, 2 * L, heads, hd) and not gk[0].any() and not gv[2].any()
    assert torch.equal(gk[1].cpu().double(), R.held(cache[0, :, :L].cpu()).flatten(0, 1))
    assert torch.equal(gv[1].cpu().double(), R.held(cache[1, :, :L].cpu()).flatten(0, 1))


# ------------------------------------------------------------------------------------------------- rotary append
@pytest.mark.parametrize("rows,heads,hd,rot,interleaved", [(1, 1, 64, 0, True), (10, 32, 80, 80, True), (7, 12, 64, 16, True), (33, 4, 128, 128, False), (2, 3, 128, 32, False)])
def test_rope_append(ops, rows, heads, hd, rot, interleaved):
    H = heads * hd
    qkv = rnd(rows, 3 * H + 8, seed=5).cuda()[:, :3 * H]
    hs, offs = (3 * hd, (0, hd, 2 * hd)) if interleaved else (hd, (0, H, 2 * H))
    g = torch.Generator().manual_seed(6)
    turn = torch.rand(rows, max(rot // 2, 1), generator=g).double()[:, :rot // 2] * 1000
    cos, sin = turn.cos().float(), turn.sin().float()
    n_pages = rows // 2 + 2
    slots = torch.randperm(n_pages * 32, generator=g)[:rows]       # rows that share a page among them
    if rows > 2:
        slots[1] = -1
    before = torch.randint(0, 256, (n_pages, heads, R.page_bytes(hd)), generator=g).to(torch.uint8)
    x = qkv.cpu().double()
    at = torch.arange(heads)[:, None] * hs + torch.arange(hd)
    q, k, v = (x[:, at + o] for o in offs)
    if rot:
        c, s, h = cos.double()[:, None], sin.double()[:, None], rot // 2
        q, k = (torch.cat([t[..., :h] * c - t[..., h:rot] * s, t[..., h:rot] * c + t[..., :h] * s, t[..., rot:]], -1) for t in (q, k))
    want = before.clone()
    for r, s in enumerate(slots.tolist()):
        for hh in range(heads):
            if s >= 0:
                R.put(want[s // 32, hh], s % 32, k[r, hh], v[r, hh])
    pages, kept = before.cuda(), qkv.clone()
    got = ops.kv4_rope_append(qkv, heads, hs, hd, offs, rot, cos.cuda(), sin.cuda(), pages, slots.cuda())
    assert torch.equal(pages.cpu(), want) and torch.equal(qkv, kept)
    assert ((got.cpu().double() - q).abs() <= 2.0 ** -8 * q.abs() * (1 + 2.0 ** -15)).all()          # one rounding to bf16 (through fp32)


# ------------------------------------------------------------------------------------------------- page tables
def tables_ref(tables, mapped, cached, new, cover, free, cursor, group, shared, max_tokens):
    rows, W = len(tables), len(tables[0])
    tables = [list(r) for r in tables]
    out, slots, cu, cur = [], [], [0], cursor
    for r in range(rows):
        c0, n = max(cached[r], 0), max(new[r], 0)
        need = min(W, (max(cover[r] if cover else 0, c0 + n) + 31) // 32)
        m = min(max(mapped[r], 0), W)
        first = r // group * group
        alias = min(max(shared[r // group], 0) // 32, need, out[first]) if shared and r != first else 0
        for c in range(m, need):
            if c < alias:
                tables[r][c] = tables[first][c]
            else:
                tables[r][c] = free[cur] if 0 <= cur < len(free) else -1
                cur += 1
        out.append(max(m, need))
        for t in range(c0, c0 + n):
            pg = tables[r][t // 32] if t // 32 < out[r] else -1
            slots.append(pg * 32 + t % 32 if pg >= 0 else -1)
        cu.append(cu[-1] + n)
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    return tables, out, cur, slots, cu


@pytest.mark.parametrize("case", range(15))
def test_page_tables_extend(ops, case):
    import random
    rng = random.Random(case)
    group = [1, 1, 1, 5, 10, 2, 1, 3, 1, 1, 4, 1, 1, 7, 1][case]
    rows = group * [1, 7, 300, 4, 8, 3, 1, 5, 700, 2, 1, 65, 1501, 200, 2][case]
    W = [1, 9, 40, 20, 20, 6, 3, 8, 5, 4, 6, 33, 7, 5, 900][case]
    cached = [rng.choice([0, 1, 31, 32, 33, rng.randint(0, W * 20)]) if group == 1 else 0 for _ in range(rows)]
    new = [rng.choice([0, 1, 31, 32, rng.randint(0, W * 12)]) for _ in range(rows)]
    if group > 1:
        new = [n if r % group == 0 else 0 for r, n in enumerate(new)]
    cover = [cached[r] + new[r // group * group if group > 1 else r] + rng.randint(0, 50) for r in range(rows)] if case % 2 else None
    if case == 6:
        cached, new, cover = [0], [0], None                         # nothing at all
    if case == 9:
        cached, new, cover = [-3, 5], [200, -7], [2 ** 31 - 1, -1]  # nonsense lengths, a table that is too narrow
    mapped = [min(W, (max(c, 0) + 31) // 32) for c in cached]
    shared = [rng.randint(0, new[g * group] + 40) for g in range(rows // group)] if group > 1 else None
    order = list(range(5000, 5000 + rows * W))
    rng.shuffle(order)
    if case == 7:
        order = order[:4]                                           # too few pages
    used = sum(mapped)
    tables = [[order[(sum(mapped[:r]) + c) % len(order)] if c < mapped[r] else -1 for c in range(W)] for r in range(rows)]
    max_tokens = [0, 3, 0, 5, 1, 0, 4, 2, 9, 1, 3, 0, 11, 6, 2][case] + (sum(max(n, 0) for n in new) if case != 11 else 17)
    want = tables_ref(tables, mapped, cached, new, cover, order, used, group, shared, max_tokens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda() if x is not None else None
    tab = i32(tables)
    for _ in range(2):                                              # the inputs are unchanged but for the filled-in columns: a second call gives the same
        m, c, s, cu = ops.page_tables_extend(tab, i32(mapped), i32(cached), i32(new), i32(order), i32([used]), max_tokens, cover=i32(cover), group=group,
                                             shared_len=i32(shared))
        assert (tab.tolist(), m.tolist(), c.item(), s.tolist(), cu.tolist()) == want


# ------------------------------------------------------------------------------------------------- beam reorder
@pytest.mark.parametrize("K,groups,heads,hd,layers", [(2, 1, 1, 64, 1), (5, 3, 4, 128, 2), (10, 2, 3, 80, 3), (16, 1, 2, 64, 2), (4, 2, 32, 80, 1)])
def test_reorder_beams(ops, K, groups, heads, hd, layers):
    W, R_ = 4, K * groups
    g = torch.Generator().manual_seed(K)
    pages = torch.randint(0, 256, (layers, R_ * W + 2, heads, R.page_bytes(hd)), generator=g).to(torch.uint8)
    tables = torch.randperm(R_ * W + 2, generator=g)[:R_ * W].view(R_, W).to(torch.int32)
    pos = torch.tensor([[37, 64, 127, 0, 128, 5][i % 6] for i in range(groups)]).repeat_interleave(K)
    if groups == 1:
        pos[:] = 50
    src = torch.randint(0, K, (R_,), generator=g)
    src[0] = K + 3                                                  # out of range: the row keeps its own
    wp, wt = pages.clone(), tables.clone()
    for r in range(R_):
        a = r // K * K + (int(src[r]) if 0 <= src[r] < K else r % K)
        c = int(pos[r]) // 32
        wt[r, :c] = tables[a, :c]
        if c < W and int(pos[r]) % 32:
            wp[:, tables[r, c]] = pages[:, tables[a, c]]
    gp, gt = pages.cuda(), tables.cuda()
    ops.kv4_reorder_beams(gp, gt, K, src.cuda(), pos.cuda())
    assert torch.equal(gt.cpu(), wt) and torch.equal(gp.cpu(), wp)


# ------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("rows,kvh,G,lens,alibi", [
    (1, 1, 1, [1], False), (5, 2, 1, [0, 1, 31, 32, 33], True), (3, 3, 2, [64, 7, 200], False), (2, 1, 16, [129, 300], True), (4, 2, 3, [96, 0, 1, 511], True),
    (2, 4, 8, [1500, 40], False), (1, 2, 1, [4500], True), (70, 16, 1, [5, 130, 64, 0, 513, 31, 200], False), (40, 32, 2, [77, 1, 90, 0], True),
    (9, 2, 4, [3000, 0, 1777, 2111], True), (3, 2, 6, [700, 33, 0], True), (1, 1, 5, [2500], False), (2, 1, 9, [95, 400], True),
    (9, 32, 1, [1400, 5, 300, 0, 64, 700, 31, 1, 1290], True)])
def test_attention(ops, hd, rows, kvh, G, lens, alibi):
    lens = (lens * rows)[:rows]
    W = (max(lens) + 31) // 32 + 1
    pages, tables = paged(rows, W, kvh, hd, seed=rows + G)
    for r, n in enumerate(lens):                                    # tables name nothing valid behind a row's pages, and the last page's unused tokens hold garbage
        c = (n + 31) // 32
        tables[r, c:] = torch.tensor([-1, 2 ** 31 - 1, pages.shape[0], -2 ** 31][r % 4], dtype=torch.int32)
        if n % 32:
            pages[int(tables[r, c - 1])] = poison_behind(pages[int(tables[r, c - 1])], n % 32, hd)
    q = rnd(rows, kvh * G, hd, seed=9, scale=2.0)
    slopes = torch.exp2(-8.0 * torch.arange(1, kvh * G + 1) / (kvh * G)) if alibi else None
    lens_t = torch.tensor(lens, dtype=torch.int32)
    want, bound = R.attend(q, pages, tables, lens_t, hd ** -0.5, slopes)
    a = (pages.cuda(), tables.cuda(), lens_t.cuda(), hd ** -0.5)
    got = ops.kv4_attn_decode(q.cuda(), *a, alibi=slopes.cuda() if alibi else None)
    check(got, want, bound)
    assert torch.equal(got, ops.kv4_attn_decode(q.cuda(), *a, alibi=slopes.cuda() if alibi else None))
    for r, n in enumerate(lens):
        if n == 0:
            assert not got[r].any()


def poison_behind(page, n, hd):
    """every byte and nibble of tokens n ... 31 of a page [heads, bytes] set, the scales to NaN: what an allocator may leave there"""
    page = page.clone()
    nb = R.blocks(hd)
    for t in range(n, 32):
        g, nib = (t % 16) // 4, 4 * (t // 16) + t % 4
        for d in range(hd):
            page[:, 512 * (d // 32) + t * (min(32, hd - d // 32 * 32) // 2) + (d % 32) // 2] |= 15 << 4 * (d % 2)
            page[:, 16 * hd + 4 * (g * hd + (d % 16) * (hd // 16) + d // 16) + nib // 2] |= 15 << 4 * (nib % 2)
        for b in range(nb):
            page[:, 32 * hd + 32 * b + 2 * (t % 16) + t // 16] = 255
            page[:, 32 * hd + 32 * nb + 8 * nb * g + 8 * b + nib] = 255
    return page


@pytest.mark.parametrize("hd,K,groups,kvh,G,prompt,more", [(80, 10, 1, 4, 1, 100, 20), (128, 4, 2, 2, 2, 64, 70), (64, 5, 3, 1, 3, 31, 40), (80, 16, 1, 2, 1, 333, 1),
                                                          (128, 10, 1, 2, 4, 200, 90), (64, 2, 2, 2, 8, 1000, 33),
                                                          # from 8 192 pages of all rows and key heads on the shared pages are read once per group
                                                          (80, 10, 2, 32, 1, 400, 20), (64, 16, 2, 32, 1, 290, 40), (128, 2, 5, 32, 8, 930, 70), (128, 4, 3, 32, 4, 700, 30),
                                                          (80, 3, 2, 16, 2, 2700, 40), (64, 5, 2, 16, 3, 1663, 3), (80, 3, 4, 32, 5, 800, 40),
                                                          (128, 2, 3, 32, 1, 1400, 20), (80, 4, 2, 32, 1, 1000, 80), (128, 2, 2, 32, 3, 2100, 20), (64, 2, 4, 32, 1, 1100, 10), (64, 5, 2, 32, 1, 860, 60)])
def test_attention_beam_groups(ops, hd, K, groups, kvh, G, prompt, more):
    """the beams of a prompt name its whole pages together; with and without room for all their queries in one tile; ragged lengths behind the prompt"""
    rows = K * groups
    W = (prompt + more + 31) // 32
    pages, tables = paged(rows, W, kvh, hd, seed=K)
    full = prompt // 32
    for r in range(rows):
        tables[r, :full] = tables[r // K * K, :full]
    lens = torch.tensor([prompt + 1 + (r * 7) % more for r in range(rows)], dtype=torch.int32)
    lens[-1] = prompt // 2                                          # a row inside the shared part
    shared = torch.full((groups,), prompt, dtype=torch.int32)
    q = rnd(rows, kvh * G, hd, seed=10)
    slopes = torch.exp2(-8.0 * torch.arange(1, kvh * G + 1) / (kvh * G))
    for al in (None, slopes):
        want, bound = R.attend(q, pages, tables, lens, 0.1, al)
        got = ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), 0.1, alibi=None if al is None else al.cuda(), group=K, shared_len=shared.cuda())
        check(got, want, bound)


def test_attention_views_streams_graph(ops):
    """q as a slice of a projection, out as one, a table with a longer row stride; on a second stream; captured, replayed with other contents between"""
    hd, kvh, G, rows, W = 128, 2, 2, 6, 9
    pages, tables = paged(rows, W, kvh, hd, seed=21)
    lens = torch.tensor([288, 1, 100, 0, 33, 250], dtype=torch.int32)
    q = rnd(rows, kvh * G, hd, seed=22)
    want, bound = R.attend(q, pages, tables, lens, 0.09)
    big = torch.zeros(rows, 3, kvh * G, hd + 8, dtype=bf16, device="cuda")
    big[:, 1, :, :hd] = q.cuda()
    wide = torch.full((rows, W + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :W] = tables.cuda()
    o = torch.zeros(rows, kvh * G, 2 * hd, dtype=bf16, device="cuda")
    p, ln = pages.cuda(), lens.cuda()
    ops.kv4_attn_decode(big[:, 1, :, :hd], p, wide[:, :W], ln, 0.09, out=o[..., hd:])
    check(o[..., hd:], want, bound)
    assert not o[..., :hd].any()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.kv4_attn_decode(q.cuda(), p, tables.cuda(), ln, 0.09)
    torch.cuda.synchronize()
    check(got, want, bound)
    sq, sl = q.cuda(), ln.clone()
    graph = torch.cuda.CUDAGraph()
    ops.kv4_attn_decode(sq, p, wide[:, :W], sl, 0.09)
    with torch.cuda.graph(graph):
        go = ops.kv4_attn_decode(sq, p, wide[:, :W], sl, 0.09)
    for i in range(4):
        q2 = rnd(rows, kvh * G, hd, seed=30 + i)
        sq.copy_(q2.cuda())
        sl.copy_(torch.tensor([(n + 37 * i) % 289 for n in lens.tolist()], dtype=torch.int32).cuda())
        graph.replay()
        eager = ops.kv4_attn_decode(q2.cuda(), p, tables.cuda(), sl, 0.09)
        assert torch.equal(go, eager)
        w2, b2 = R.attend(q2, pages, tables, sl.cpu(), 0.09)
        check(go, w2, b2)


def test_attention_not_a_number(ops):
    """a NaN block inside the visible keys (values) makes NaN of that row and head (of its 32 dims), and of nothing else; an infinite query too"""
    hd, kvh, rows, W = 80, 2, 4, 3
    pages, tables = paged(rows, W, kvh, hd, seed=41)
    lens = torch.tensor([70, 70, 70, 70], dtype=torch.int32)
    nb = R.blocks(hd)
    pages[int(tables[0, 1]), 1, 32 * hd + 2 * 5] = 255              # row 0, head 1: key 37's first block
    t, g = 2, 0                                                     # row 1, head 0: value 2's second block, its codes zero as the writer leaves them
    pages[int(tables[1, 0]), 0, 32 * hd + 32 * nb + 8 * nb * g + 8 * 1 + t] = 255
    q = rnd(rows, kvh, hd, seed=42)
    q[2, 1, 3] = float("inf")
    got = ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), 0.1).cpu()
    nan = torch.zeros(rows, kvh, hd, dtype=torch.bool)
    nan[0, 1], nan[2, 1] = True, True
    seen = torch.isnan(got)
    assert seen[0, 1].all() and seen[2, 1].all() and (~torch.isfinite(got[1, 0, 32:64])).all()
    nan[1, 0, 32:64] = True
    assert torch.isfinite(got[~nan]).all()


def test_attention_wide_table(ops):
    """a table far wider than its rows (the width is what the launch is made for, never the lengths), and one row of 20 000 tokens"""
    hd, kvh, W = 64, 1, 40000
    pages, few = paged(2, 640, kvh, hd, seed=61)
    tables = torch.full((2, W), -1, dtype=torch.int32)
    tables[:, :640] = few
    lens = torch.tensor([20000, 45], dtype=torch.int32)
    q = rnd(2, 2, hd, seed=62)
    want, bound = R.attend(q, pages, tables[:, :640], lens, 0.125)
    check(ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), 0.125), want, bound)


def test_hidden_pages(ops):
    """a page id outside the pool hides its 32 tokens; a row all of whose pages are hidden gives zeros"""
    hd, kvh, W = 64, 2, 6
    pages, tables = paged(3, W, kvh, hd, seed=51)
    tables[0, 1], tables[0, 4], tables[1, :] = -1, pages.shape[0], -5
    lens = torch.tensor([180, 100, 192], dtype=torch.int32)
    q = rnd(3, kvh * 2, hd, seed=52)
    want, bound = R.attend(q, pages, tables, lens, 0.125)
    got = ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), 0.125)
    check(got, want, bound)
    assert not got[1].any()


def test_lengths_beyond_the_table_and_odd_views(ops):
    """a length above 32 x width stands for the whole table, a negative one for nothing; q and k / v views that no 16-byte load can read are copied; out may be q"""
    hd, kvh, W = 64, 2, 3
    pages, tables = paged(3, W, kvh, hd, seed=71)
    lens = torch.tensor([1000, -4, 2 ** 31 - 1], dtype=torch.int32)
    q = rnd(3, kvh, hd, seed=72)
    want, bound = R.attend(q, pages, tables, torch.tensor([96, 0, 96]), 0.125)
    raw = torch.zeros(3, kvh, hd + 3, dtype=bf16, device="cuda")
    raw[..., 1:hd + 1] = q.cuda()
    p, t, n = pages.cuda(), tables.cuda(), lens.cuda()
    check(ops.kv4_attn_decode(raw[..., 1:hd + 1], p, t, n, 0.125), want, bound)
    own = q.cuda()
    check(ops.kv4_attn_decode(own, p, t, n, 0.125, out=own), want, bound)
    k = rnd(40, kvh, hd + 1, seed=73).cuda()
    ops.kv4_write(k[..., 1:], k[..., :hd], p, torch.arange(40, device="cuda"))
    gk, gv = ops.kv4_read(p, torch.arange(40, device="cuda"), hd)
    assert torch.equal(gk.cpu().double(), R.held(k[..., 1:].cpu())) and torch.equal(gv.cpu().double(), R.held(k[..., :hd].cpu()))


def test_nothing_to_do(ops):
    """no rows, no tokens, no columns"""
    e = lambda *s, dt=bf16: torch.empty(s, dtype=dt, device="cuda")
    pages = torch.zeros((2, 3, R.page_bytes(80)), dtype=torch.uint8, device="cuda")
    assert ops.kv4_attn_decode(e(0, 3, 80), pages, e(0, 4, dt=torch.int32), e(0, dt=torch.int32), 1.0).shape == (0, 3, 80)
    q = rnd(2, 6, 80).cuda()
    assert not ops.kv4_attn_decode(q, pages, e(2, 0, dt=torch.int32), torch.tensor([5, 0], dtype=torch.int32, device="cuda"), 1.0).any()
    ops.kv4_write(e(0, 3, 80), e(0, 3, 80), pages, e(0, dt=torch.int64))
    assert ops.kv4_read(pages, e(0, dt=torch.int64), 80)[0].shape == (0, 3, 80)
    assert ops.kv4_rope_append(e(0, 720), 3, 240, 80, (0, 80, 160), 0, None, None, pages, e(0, dt=torch.int64)).shape == (0, 3, 80)
    assert not pages.any()
    # a pool of no pages: nothing is written, everything reads as zero; no free page is needed where none is taken
    none, s2 = pages[:0], torch.tensor([3, -1], device="cuda")
    ops.kv4_write(rnd(2, 3, 80).cuda(), rnd(2, 3, 80).cuda(), none, s2)
    assert not ops.kv4_read(none, s2, 80)[0].any()
    qkv = rnd(2, 720).cuda()
    assert torch.equal(ops.kv4_rope_append(qkv, 3, 240, 80, (0, 80, 160), 0, None, None, none, s2), qkv.view(2, 3, 240)[..., :80])
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    tab = i32(7, 9, 4, -1).view(2, 2)
    m, c, s, cu = ops.page_tables_extend(tab, i32(2, 1), i32(40, 1), i32(2, 3), e(0, dt=torch.int32), i32(11), 6)
    assert (tab.tolist(), m.tolist(), c.item(), s.tolist(), cu.tolist()) == ([[7, 9], [4, -1]], [2, 1], 11, [296, 297, 129, 130, 131, -1], [0, 2, 5])
    ops.kv4_reorder_beams(pages, e(0, 4, dt=torch.int32), 2, e(0, dt=torch.int64), e(0, dt=torch.int64))
    ops.kv4_reorder_beams(pages, e(2, 0, dt=torch.int32), 2, torch.ones(2, dtype=torch.long, device="cuda"), torch.full((2,), 40, device="cuda"))


def test_sums_beyond_32_bits(ops):
    """lengths whose sums pass 32 bits: the counts stay at the largest value, no slot is written behind the room"""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    big = 2 ** 31 - 1
    tab = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    m, c, s, cu = ops.page_tables_extend(tab, i32(0, 0, 0), i32(0, 0, 5), i32(big, big, big), i32(8, 3), i32(big - 1), 70)
    assert tab.tolist() == [[-1, -1]] * 3 and m.tolist() == [2, 2, 2] and c.item() == big and cu.tolist() == [0, big, big, big] and s.tolist() == [-1] * 70


def test_one_row_of_a_misaligned_buffer(ops):
    """views that count as contiguous and yet start at an odd element, or have one row and an odd row stride"""
    hd, kvh = 64, 2
    pages, tables = paged(1, 2, kvh, hd, seed=75)
    n = torch.tensor([50], dtype=torch.int32)
    q = rnd(1, kvh, hd, seed=76)
    want, bound = R.attend(q, pages, tables, n, 0.125)
    flat = torch.zeros(1 + kvh * hd, dtype=bf16, device="cuda")
    flat[1:] = q.cuda().view(-1)
    wide = torch.zeros(1, kvh * hd + 3, dtype=bf16, device="cuda")
    wide[:, :kvh * hd] = q.cuda().view(1, -1)
    p, slot = pages.cuda(), torch.tensor([int(tables[0, 1]) * 32 + 31], device="cuda")
    for view in (flat[1:].view(1, kvh, hd), wide[:, :kvh * hd].view(1, kvh, hd)):
        check(ops.kv4_attn_decode(view, p, tables.cuda(), n.cuda(), 0.125), want, bound)
        ops.kv4_write(view, view, p, slot)
        assert torch.equal(ops.kv4_read(p, slot, hd)[1].cpu().double(), R.held(q))


def test_a_pool_beyond_32_bits(ops):
    """pages at byte offsets above 4 GiB: written, appended to, read, attended to, moved"""
    hd, kvh, n_pages = 128, 4, 300_000                              # 5.2 GB
    pool = torch.zeros((n_pages, kvh, R.page_bytes(hd)), dtype=torch.uint8, device="cuda")
    ids = torch.tensor([[n_pages - 1, 5, n_pages - 70], [n_pages - 2, 5, n_pages - 71]], dtype=torch.int32)
    t = torch.arange(70)
    slots = torch.cat([ids[r].long()[t // 32] * 32 + t % 32 for r in range(2)])
    kv = rnd(2, 140, kvh, hd, seed=81)
    ops.kv4_write(kv[0].cuda(), kv[1].cuda(), pool, slots.cuda())
    qkv = rnd(2, 3 * kvh * hd, seed=82)
    ops.kv4_rope_append(qkv.cuda(), kvh, hd, hd, (0, kvh * hd, 2 * kvh * hd), 0, None, None, pool, (ids[:, 2].long() * 32 + 6).cuda())
    small = pool[ids.view(-1).long()].cpu()                         # what the two rows name, as a pool of six pages
    q = rnd(2, kvh, hd, seed=83)
    lens = torch.tensor([71, 71], dtype=torch.int32)
    want, bound = R.attend(q, small, torch.arange(6, dtype=torch.int32).view(2, 3), lens, 0.1)
    check(ops.kv4_attn_decode(q.cuda(), pool, ids.cuda(), lens.cuda(), 0.1), want, bound)
    k, v = R.unpack(small, hd)
    assert torch.equal(k[2, :, 6], R.held(qkv.view(2, 3, kvh, hd)[0, 1])) and torch.equal(v[5, :, 6], R.held(qkv.view(2, 3, kvh, hd)[1, 2]))
    gk, _ = ops.kv4_read(pool, slots[:32].cuda(), hd)
    assert torch.equal(gk.cpu().double(), R.held(kv[0, :32]))
    tab = ids.cuda()
    ops.kv4_reorder_beams(pool, tab, 2, torch.tensor([1, 1], device="cuda"), torch.tensor([71, 71], device="cuda"))
    assert tab.tolist() == [[n_pages - 2, 5, n_pages - 70], [n_pages - 2, 5, n_pages - 71]] and torch.equal(pool[n_pages - 70], pool[n_pages - 71])
    del pool
    torch.cuda.empty_cache()


def test_two_streams_at_once(ops):
    """the same pool read by calls on two streams, each with partials of its own, while a third writes other pages"""
    hd, kvh, rows, W = 80, 4, 8, 70
    pages, tables = paged(rows, W, kvh, hd, seed=91, extra=40)
    free = sorted(set(range(pages.shape[0])) - set(tables.view(-1).tolist()))
    p, t = pages.cuda(), tables.cuda()
    lens = torch.full((rows,), W * 32 - 5, dtype=torch.int32, device="cuda")
    qs = [rnd(rows, kvh, hd, seed=92 + i).cuda() for i in range(2)]
    want = [ops.kv4_attn_decode(q, p, t, lens, 0.11) for q in qs]
    k = rnd(32 * len(free), kvh, hd, seed=95).cuda()
    slots = (torch.tensor(free)[:, None] * 32 + torch.arange(32)).view(-1).cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.kv4_attn_decode(qs[i], p, t, lens, 0.11))
        with torch.cuda.stream(streams[2]):
            ops.kv4_write(k, k, p, slots)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
