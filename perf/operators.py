"""Decoding over a paged K/V cache that is held in 4 bits: the operators, their cases, and what each must return.

The cache.  A page holds 32 tokens of one head of one layer, keys and values, as MX blocks: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) with one power-of-two scale byte (value 2^(byte - 127), 255: not a number) per 32 consecutive dims of a token; where the head is not a multiple of
32 wide, its last block is narrower.  With D dims and B = ceil(D / 32) blocks a page is 32 D + 64 B bytes:

    0 ............. key codes     block b (512 b onwards): token t, its dims 32 b ... as consecutive nibbles, low first
    16 D .......... value codes   32-bit word (t % 16 / 4) D + (d % 16) (D / 16) + d / 16, nibble 4 (t / 16) + t % 4 of it
    32 D .......... key scales    byte 32 b + 2 (t % 16) + t / 16
    32 D + 32 B ... value scales  byte 8 B (t % 16 / 4) + 8 b + 4 (t / 16) + t % 4

A block's scale is 2^e, e = max(floor(log2 of its largest magnitude) - 2, -125); its codes are x / 2^e rounded to the nearest (ties to the even code),
at most 6.  A block that holds an infinity or a NaN is not a number.  Slot s of a pool is token s % 32 of page s / 32; a negative slot or page is none.

The operators: `attend` (one new token per row against its pages), `write` (prompt tokens into slots), `append` (rotary embedding of a decode step's q and
k, and the append of its k and v), `tables` (page tables and slots from the rows' lengths), `reorder` (beam search: rows take over other rows' states)."""
import math
import random

import torch

own = False

PAGE = 32


# ------------------------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one user's greedy token at the 3B tower's heads (32 x 80), the recommendation prompt of 469 tokens: latency
        dict(name="attend_one_user", op="attend", rows=1, heads=32, kv_heads=32, hd=80, max_len=469, ragged=False, alibi=False, group=1, prompt=0),
        # the same user with ten beams, half way through 50 new tokens: the beams read one copy of the prompt's pages
        dict(name="attend_ten_beams", op="attend", rows=10, heads=32, kv_heads=32, hd=80, max_len=494, ragged=False, alibi=False, group=10, prompt=469),
        # sixteen users of the 7B tower (32 x 128, ALiBi), prompts of any length up to its 2048 positions
        dict(name="attend_alibi_ragged", op="attend", rows=16, heads=32, kv_heads=32, hd=128, max_len=2048, ragged=True, alibi=True, group=1, prompt=0),
        # long contexts, four query heads to a key head
        dict(name="attend_long_shared_heads", op="attend", rows=48, heads=32, kv_heads=8, hd=128, max_len=16384, ragged=True, alibi=False, group=1, prompt=0),
        # the prompts of eight users after their prefill, padded as a batch (padding has no slot)
        dict(name="write_eight_prompts", op="write", requests=8, max_new=469, heads=32, hd=80),
        # sixteen long prompts
        dict(name="write_long_prompts", op="write", requests=16, max_new=4100, heads=32, hd=128),
        # a decode step of ten beams of the 3B tower (rotary over the whole head, per-head q k v)
        dict(name="append_ten_beams", op="append", rows=10, heads=32, hd=80, rot=80, interleaved=True),
        # a decode step of many users (q, k and v as blocks)
        dict(name="append_many_rows", op="append", rows=200, heads=32, hd=128, rot=128, interleaved=False),
        # eight users with ten beams each: prompts and room for 50 new tokens
        dict(name="tables_eight_users", op="tables", requests=8, group=10, max_cached=0, max_new=469, room=50, width=20),
        # a scheduler's step over two thousand requests, most with a long past
        dict(name="tables_many_requests", op="tables", requests=2000, group=1, max_cached=3000, max_new=1000, room=0, width=128),
        # one user, five beams, between two tokens; all layers
        dict(name="reorder_five_beams", op="reorder", layers=24, groups=1, group=5, heads=16, hd=128, width=10),
        # eight users with ten beams
        dict(name="reorder_eighty_beams", op="reorder", layers=32, groups=8, group=10, heads=32, hd=80, width=20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "append", "tables", "reorder"])
    if op == "attend":
        hd, kv = rng.choice([64, 80, 128]), rng.choice([8, 12, 16, 32])
        top = 48 * 16384 * 8 * 128                      # elements of the largest listed case
        if rng.random() < 0.35:
            group = rng.randint(2, 10)
            prompt = _log(rng, 1, 4096)
            rows = group * rng.randint(1, 4)
            return dict(op=op, rows=rows, heads=kv, kv_heads=kv, hd=hd, max_len=prompt + rng.randint(1, 600), ragged=False, alibi=rng.random() < 0.4, group=group,
                        prompt=prompt)
        rows, q = _log(rng, 1, 64), rng.choice([1, 1, 2, 3, 4, 8, 16])
        return dict(op=op, rows=rows, heads=kv * q, kv_heads=kv, hd=hd, max_len=_log(rng, 1, max(1, min(16384, top // (rows * kv * hd)))), ragged=rng.random() < 0.7,
                    alibi=rng.random() < 0.4, group=1, prompt=0)
    if op == "write":
        heads, hd, requests = rng.choice([8, 12, 16, 32]), rng.choice([64, 80, 128]), _log(rng, 1, 64)
        return dict(op=op, requests=requests, max_new=_log(rng, 1, 65600 // requests), heads=heads, hd=hd)
    if op == "append":
        hd = rng.choice([64, 80, 128])
        return dict(op=op, rows=_log(rng, 1, 200), heads=rng.choice([8, 12, 16, 32]), hd=hd, rot=rng.choice([0, 16, 32, hd]), interleaved=rng.random() < 0.5)
    if op == "tables":
        group = rng.choice([1, 1, 2, 5, 10])
        requests = _log(rng, 1, 2000 // group)
        cached, new, room = rng.choice([0, _log(rng, 1, 3000)]), _log(rng, 1, 1000), rng.choice([0, 50, 256])
        return dict(op=op, requests=requests, group=group, max_cached=0 if group > 1 else cached, max_new=new, room=room, width=(cached + new + room) // PAGE + 1)
    group = rng.randint(2, 10)
    return dict(op=op, layers=rng.choice([1, 12, 24, 32]), groups=rng.randint(1, 8), group=group, heads=rng.choice([8, 12, 16, 32]), hd=rng.choice([64, 80, 128]),
                width=rng.randint(1, 20))


def _lengths(case):
    """the rows' lengths (a fixed function of the case, so that work() counts what is there)"""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "attend":
        lens = [rng.randint(0, case["max_len"]) if case["ragged"] else case["max_len"] for _ in range(case["rows"])]
        lens[-1] = case["max_len"]
        return lens
    if case["op"] == "write":
        lens = [rng.randint((case["max_new"] + 1) // 2, case["max_new"]) for _ in range(case["requests"])]
        lens[0] = case["max_new"]
        return lens
    if case["op"] == "tables":
        cached, new, cover = [], [], []
        for _ in range(case["requests"]):
            c, n = rng.randint(0, case["max_cached"]), rng.randint(0, case["max_new"])
            for j in range(case["group"]):
                cached.append(c), new.append(n if j == 0 else 0), cover.append(c + n + case["room"])
        return cached, new, cover
    if case["op"] == "reorder":
        return [rng.randint(0, case["width"] * PAGE - 1) for _ in range(case["groups"])]
    return None


def _blocks(hd):
    return (hd + 31) // 32


def _page_bytes(hd):
    return 32 * hd + 64 * _blocks(hd)


def work(case):
    op = case["op"]
    if op == "attend":
        lens, D = _lengths(case), case["hd"]
        once = sum(lens) - case["prompt"] // PAGE * PAGE * (case["rows"] - case["rows"] // case["group"])      # shared pages are read for one beam
        held = D + 2 * _blocks(D)                                                                              # bytes of a token's key and value
        return {"bytes": once * case["kv_heads"] * held + case["rows"] * case["heads"] * D * 4 + 4 * once // PAGE + 4 * case["rows"],
                "flops": 4 * sum(lens) * case["heads"] * D}
    if op == "write":
        n = sum(_lengths(case)) * case["heads"] * case["hd"]
        rows = case["requests"] * case["max_new"]
        # k and v in, codes and scales out, and the same back as values
        return {"bytes": n * 4 + 2 * n * 17 // 16 + rows * case["heads"] * case["hd"] * 4 + 16 * rows, "flops": 4 * n}
    if op == "append":
        n = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": n * 6 + n * 2 + n * 17 // 16 + 32 * n * 17 // 16 + 32 * n * 4 + case["rows"] * (8 + 256 + 4 * case["rot"]), "flops": 12 * n + 64 * n}
    if op == "tables":
        cached, new, cover = _lengths(case)
        rows = len(cached)
        return {"bytes": 8 * sum(new) + 4 * sum((c + PAGE - 1) // PAGE for c in cover) * 2 + 24 * rows, "flops": 4 * sum(new)}
    R = case["groups"] * case["group"]
    page = case["layers"] * case["heads"] * _page_bytes(case["hd"])
    vals = case["layers"] * R * PAGE * case["heads"] * case["hd"] * 4
    return {"bytes": R * page * 3 + vals + 8 * R * case["width"], "flops": 2 * case["layers"] * R * PAGE * case["heads"] * case["hd"]}


# ------------------------------------------------------------------------------------------------------------------------------------ the format, plainly
def _places(hd, dev):
    """byte and shift of every key and value code [32, hd], and byte of every scale [32, blocks], inside a page"""
    t, d, b = torch.arange(PAGE, device=dev)[:, None], torch.arange(hd, device=dev)[None, :], torch.arange(_blocks(hd), device=dev)[None, :]
    wide = torch.clamp(hd - d // 32 * 32, max=32) // 2                                                         # bytes of a token in its block
    kb, ks = d // 32 * 512 + t * wide + d % 32 // 2, d % 2 * 4 + 0 * t
    j = t // 16 * 4 + t % 4
    vb, vs = 16 * hd + (t % 16 // 4 * hd + d % 16 * (hd // 16) + d // 16) * 4 + j // 2, j % 2 * 4 + 0 * d
    ksc = 32 * hd + 32 * b + t % 16 * 2 + t // 16
    vsc = 32 * hd + 32 * _blocks(hd) + t % 16 // 4 * 8 * _blocks(hd) + b * 8 + j
    return (kb, ks, ksc), (vb, vs, vsc)


def _two(e):
    """2^e, -126 <= e <= 127, from its bits (a power function may round)"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """x [..., hd] -> codes uint8 [..., hd], scale bytes uint8 [..., blocks]"""
    hd, nb = x.shape[-1], _blocks(x.shape[-1])
    x = torch.nn.functional.pad(x, (0, nb * 32 - hd)).unflatten(-1, (nb, 32))
    amax = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    e = torch.clamp(torch.frexp(torch.where(bad, torch.ones_like(amax), amax))[1] - 3, min=-125)               # floor(log2 amax) - 2
    e = torch.where(amax == 0, torch.full_like(e, -125), e)
    a = x.abs() * _two(-e)
    code = torch.zeros_like(a, dtype=torch.uint8)
    for at, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):      # midpoints; ties to the even code
        code += (a >= at) if up else (a > at)
    code += 8 * (x < 0)
    return torch.where(bad, torch.zeros_like(code), code).flatten(-2)[..., :hd].contiguous(), torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(-1).to(torch.uint8)


def _held(codes, scales):
    """the values that codes [..., hd] and scale bytes [..., blocks] stand for"""
    m = (codes & 7).float()
    v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, m * 2 - 8))
    v = torch.where(codes > 7, -v, v)
    s = _two(torch.where(scales == 255, 0, scales.to(torch.int32) - 127))
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return v * s.repeat_interleave(32, -1)[..., :codes.shape[-1]]


def _unpack(pages, hd, which):
    """pages [..., page bytes] -> the codes [..., 32, hd] and scales [..., 32, blocks] of its keys (0) or values (1)"""
    byte, shift, scale = _places(hd, pages.device)[which]
    return (pages[..., byte] >> shift.to(torch.uint8)) & 15, pages[..., scale]


def _pack(k, v):
    """k, v [..., 32, hd] -> pages [..., page bytes]"""
    hd = k.shape[-1]
    out = torch.zeros(k.shape[:-2] + (_page_bytes(hd),), dtype=torch.uint8, device=k.device)
    for x, (byte, shift, scale) in zip((k, v), _places(hd, k.device)):
        codes, sc = _quantise(x)
        codes = codes << shift.to(torch.uint8)
        for half in (0, 4):                                                                                    # a byte's two nibbles come from two dims or two tokens
            at = shift == half
            out[..., byte[at]] |= codes[..., at]
        out[..., scale] = sc
    return out


# ------------------------------------------------------------------------------------------------------------------------------------ inputs
def _slots_of(table, first, n):
    t = torch.arange(first, first + n, device=table.device)
    return table[t // PAGE].long() * PAGE + t % PAGE


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device=dev)
    op = case["op"]
    s = dict(op=op, case=case)
    if op == "attend":
        R, H, hd, K = case["rows"], case["kv_heads"], case["hd"], case["group"]
        W = (case["max_len"] + PAGE - 1) // PAGE
        full = case["prompt"] // PAGE                                           # columns that the rows of a group share
        n = R * W - (R - R // K) * full
        order = torch.randperm(n, generator=g, device=dev).to(torch.int32)      # a pool's pages are handed out in any order
        tables = torch.empty((R, W), dtype=torch.int32, device=dev)
        at = 0
        for r in range(R):
            own_from = full if r % K else 0
            if r % K:
                tables[r, :full] = tables[r // K * K, :full]
            tables[r, own_from:] = order[at:at + W - own_from]
            at += W - own_from
        width = torch.exp(0.5 * normal(H, 1, hd))                               # some channels of a key are much larger than others
        s["pages"] = torch.empty((n, H, _page_bytes(hd)), dtype=torch.uint8, device=dev)
        for i in range(0, n, 2048):
            m = min(2048, n - i)
            s["pages"][i:i + m] = _pack((normal(m, H, PAGE, hd) * width).bfloat16().float(), normal(m, H, PAGE, hd).bfloat16().float())
        s.update(q=normal(R, case["heads"], hd).bfloat16(), tables=tables, lens=torch.tensor(_lengths(case), dtype=torch.int32, device=dev), scale=hd ** -0.5,
                 alibi=torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device=dev) / case["heads"]) if case["alibi"] else None,
                 group=K, shared=torch.full((R // K,), case["prompt"], dtype=torch.int32, device=dev) if K > 1 else None)
    elif op == "write":
        lens, H, hd, L = _lengths(case), case["heads"], case["hd"], case["max_new"]
        cols = [(n + PAGE - 1) // PAGE for n in lens]
        order = torch.randperm(sum(cols), generator=g, device=dev).to(torch.int32)
        slots = torch.full((len(lens), L), -1, dtype=torch.int64, device=dev)
        at = 0
        for r, n in enumerate(lens):
            slots[r, :n] = _slots_of(order[at:at + cols[r]], 0, n)
            at += cols[r]
        kv = normal(2, len(lens) * L, H, hd).bfloat16()
        kv[0] *= torch.exp(0.5 * normal(H, hd)).bfloat16()
        s.update(k=kv[0], v=kv[1], slots=slots.view(-1), pages=torch.zeros((sum(cols), H, _page_bytes(hd)), dtype=torch.uint8, device=dev), hd=hd)
    elif op == "append":
        R, H, hd, rot = case["rows"], case["heads"], case["hd"], case["rot"]
        s["pages"] = _pack(normal(R, H, PAGE, hd).bfloat16().float(), normal(R, H, PAGE, hd).bfloat16().float())
        page = torch.randperm(R, generator=g, device=dev)
        s["slots"] = page * PAGE + torch.randint(0, PAGE, (R,), generator=g, device=dev)
        s["around"] = (page[:, None] * PAGE + torch.arange(PAGE, device=dev)).view(-1)
        s["qkv"] = normal(R, 3 * H * hd).bfloat16()
        s["stride"], s["offs"] = (3 * hd, (0, hd, 2 * hd)) if case["interleaved"] else (hd, (0, H * hd, 2 * H * hd))
        pos = torch.randint(0, 2048, (R, 1), generator=g, device=dev).double()
        turn = pos * 10000.0 ** (-torch.arange(0, rot, 2, device=dev).double() / max(rot, 1))
        s.update(cos=turn.cos().float(), sin=turn.sin().float(), heads=H, hd=hd, rot=rot)
    elif op == "tables":
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        cached, new, cover = _lengths(case)
        R, W = len(cached), case["width"]
        mapped = [(c + PAGE - 1) // PAGE for c in cached]
        n = sum((c + PAGE - 1) // PAGE for c in cover) + 7
        order = torch.randperm(n, generator=g, device=dev).to(torch.int32)
        have = torch.arange(W, device=dev)[None, :] < i32(mapped)[:, None]
        tables = torch.full((R, W), -1, dtype=torch.int32, device=dev)
        tables[have] = order[:sum(mapped)]
        s.update(tables=tables, mapped=i32(mapped), cached=i32(cached), new=i32(new), cover=i32(cover), free=order, cursor=i32([sum(mapped)]), group=case["group"],
                 shared=i32(new[::case["group"]]) if case["group"] > 1 else None, max_tokens=sum(new) + 5)
    else:
        Ly, G, K, H, hd, W = (case[k] for k in ("layers", "groups", "group", "heads", "hd", "width"))
        pos = torch.tensor(_lengths(case), device=dev).repeat_interleave(K)
        R = G * K
        order = torch.randperm(R * W, generator=g, device=dev).to(torch.int32)
        tables = order.view(R, W).clone()
        now = tables.gather(1, (pos // PAGE)[:, None]).long()
        s["pages"] = torch.zeros((Ly, R * W, H, _page_bytes(hd)), dtype=torch.uint8, device=dev)
        for i in range(Ly):
            s["pages"][i, now[:, 0]] = _pack(normal(R, H, PAGE, hd).bfloat16().float(), normal(R, H, PAGE, hd).bfloat16().float())
        # some beams go on, the others take over one of those
        rank = torch.argsort(torch.rand((G, K), generator=g, device=dev), 1)
        keep = max(1, K // 2)
        src = torch.empty((G, K), dtype=torch.int64, device=dev)
        src.scatter_(1, rank[:, :keep], rank[:, :keep])
        src.scatter_(1, rank[:, keep:], rank[:, :keep].gather(1, torch.randint(0, keep, (G, K - keep), generator=g, device=dev)))
        s.update(tables=tables, src=src.view(-1), pos=pos, group=K, hd=hd, around=(now * PAGE + torch.arange(PAGE, device=dev)).view(-1))
    return s


# ------------------------------------------------------------------------------------------------------------------------------------ one pass
def _attend(s):
    R, Hq, hd = s["q"].shape
    H = s["pages"].shape[1]
    held = s["pages"][s["tables"].long()].transpose(1, 2)                                                     # [R, H, W, page bytes]
    n = held.shape[2] * PAGE
    there = torch.arange(n, device=s["q"].device) < s["lens"][:, None]                                        # [R, n]
    q = s["q"].float().view(R, H, Hq // H, hd)
    k = _held(*_unpack(held, hd, 0)).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]                                      # [R, H, q heads of a key head, n]
    del k
    if s["alibi"] is not None:
        far = torch.arange(n, device=q.device)[None, :] - (s["lens"][:, None] - 1)                            # a shift by a row's last position changes no softmax
        score = score + s["alibi"].view(1, H, Hq // H, 1) * far.float()[:, None, None, :]
    there = there[:, None, None, :]
    score = torch.where(there, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    v = _held(*_unpack(held, hd, 1)).flatten(2, 3)
    o = torch.matmul(p, v)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total == 0, torch.zeros_like(o), o / total)                                               # a row of length 0 attends to nothing
    return o.view(R, Hq, hd).bfloat16()


def _place(pages, hd, slots, k, v):
    """the codes of k, v [T, H, hd] into their slots of pages [P, H, page bytes]"""
    ok = slots >= 0
    page, t = slots[ok] // PAGE, slots[ok] % PAGE
    head = torch.arange(pages.shape[1], device=pages.device)
    for x, (byte, shift, scale) in zip((k, v), _places(hd, pages.device)):
        codes, sc = _quantise(x[ok])
        for half in (0, 4):                                                                                    # two codes share a byte: the low halves first
            r, d = (shift[t] == half).nonzero(as_tuple=True)
            where = (page[r, None], head[None, :], byte[t[r], d][:, None])
            pages[where] = (pages[where] & (15 << (4 - half))) | (codes[r, :, d] << half)
        pages[page[:, None, None], head[:, None], scale[t][:, None, :]] = sc


def _values(pages, hd, slots):
    """the k, v values [..., T, H, hd] held in slots of pages [..., P, H, page bytes]"""
    at = torch.clamp(slots, min=0)
    held = pages[..., at // PAGE, :, :]                                                                       # [..., T, H, page bytes]
    out = []
    for byte, shift, scale in _places(hd, pages.device):
        t = at % PAGE
        pick = lambda where: torch.gather(held, -1, where[t][:, None, :].expand(held.shape[:-1] + (where.shape[1],)))
        codes = (pick(byte) >> shift[t].to(torch.uint8)[:, None, :]) & 15
        out.append(torch.where((slots >= 0)[:, None, None], _held(codes, pick(scale)), torch.zeros((), device=pages.device)).bfloat16())
    return tuple(out)


def _append(s):
    R, H, hd, rot = s["qkv"].shape[0], s["heads"], s["hd"], s["rot"]
    at = torch.arange(H, device=s["qkv"].device)[:, None] * s["stride"] + torch.arange(hd, device=s["qkv"].device)
    q, k, v = (s["qkv"][:, at + o].double() for o in s["offs"])                                               # codes are decided next to a border: 64 bits
    if rot:
        c, si, h = s["cos"].double()[:, None, :], s["sin"].double()[:, None, :], rot // 2
        q, k = (torch.cat([x[..., :h] * c - x[..., h:rot] * si, x[..., h:rot] * c + x[..., :h] * si, x[..., rot:]], -1) for x in (q, k))
    _place(s["pages"], hd, s["slots"], k, v)
    return (q.bfloat16(),) + _values(s["pages"], hd, s["around"])


def _tables(s):
    R, W = s["tables"].shape
    K, dev = s["group"], s["tables"].device
    new, cached, mapped = (s[k].long() for k in ("new", "cached", "mapped"))
    need = torch.clamp((torch.maximum(s["cover"].long(), cached + new) + PAGE - 1) // PAGE, max=W)
    first = torch.arange(R, device=dev) // K * K
    after = torch.maximum(mapped, need)
    alias = torch.zeros_like(need)
    if s["shared"] is not None:
        alias = torch.minimum(torch.minimum(s["shared"].long().repeat_interleave(K) // PAGE, need), after[first])
        alias = torch.where(first == torch.arange(R, device=dev), torch.zeros_like(alias), alias)
    begin = torch.maximum(mapped, alias)
    mine = torch.clamp(need - begin, min=0)
    at = s["cursor"].long() + torch.cumsum(mine, 0) - mine
    col = torch.arange(W, device=dev)[None, :]
    index = at[:, None] + col - begin[:, None]
    page = torch.where(index < len(s["free"]), s["free"][torch.clamp(index, 0, len(s["free"]) - 1)], torch.full_like(s["tables"], -1))
    got = torch.where((col >= begin[:, None]) & (col < need[:, None]), page, s["tables"])
    got = torch.where((col >= mapped[:, None]) & (col < alias[:, None]), got[first], got)
    s["tables"].copy_(got)
    cu = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    i = torch.arange(s["max_tokens"], device=dev)
    row = torch.clamp(torch.searchsorted(cu, i, right=True) - 1, max=R - 1)
    t = cached[row] + i - cu[row]
    page = got[row, torch.clamp(t // PAGE, 0, W - 1)].long()
    slots = torch.where((i < cu[-1]) & (t // PAGE < W) & (page >= 0), page * PAGE + t % PAGE, torch.full_like(i, -1))
    return got, after.int(), (s["cursor"] + mine.sum()).int(), slots, cu.int()


def _reorder(s):
    K, W = s["group"], s["tables"].shape[1]
    R = len(s["src"])
    src = torch.arange(R, device=s["src"].device) // K * K + s["src"]
    now = (s["pos"] // PAGE)[:, None]
    page = s["tables"].gather(1, now)[:, 0].long()
    s["pages"][:, page] = torch.where((s["pos"] % PAGE > 0)[None, :, None, None], s["pages"][:, page[src]], s["pages"][:, page])
    s["tables"].copy_(torch.where(torch.arange(W, device=src.device)[None, :] < now, s["tables"][src], s["tables"]))
    return (s["tables"],) + _values(s["pages"], s["hd"], s["around"])


def run(s):
    op = s["op"]
    if own:
        from unimp_amd import ops
        if op == "attend":
            return ops.kv4_attn_decode(s["q"], s["pages"], s["tables"], s["lens"], s["scale"], alibi=s["alibi"], group=s["group"], shared_len=s["shared"])
        if op == "write":
            ops.kv4_write(s["k"], s["v"], s["pages"], s["slots"])
            return ops.kv4_read(s["pages"], s["slots"], s["hd"])
        if op == "append":
            q = ops.kv4_rope_append(s["qkv"], s["heads"], s["stride"], s["hd"], s["offs"], s["rot"], s["cos"], s["sin"], s["pages"], s["slots"])
            return (q,) + ops.kv4_read(s["pages"], s["around"], s["hd"])
        if op == "tables":
            mapped, cursor, slots, cu = ops.page_tables_extend(s["tables"], s["mapped"], s["cached"], s["new"], s["free"], s["cursor"], s["max_tokens"], cover=s["cover"],
                                                               group=s["group"], shared_len=s["shared"])
            return s["tables"], mapped, cursor, slots, cu
        ops.kv4_reorder_beams(s["pages"], s["tables"], s["group"], s["src"], s["pos"])
        return (s["tables"],) + ops.kv4_read(s["pages"], s["around"], s["hd"])
    if op == "attend":
        return _attend(s)
    if op == "write":
        _place(s["pages"], s["hd"], s["slots"], s["k"].float(), s["v"].float())
        return _values(s["pages"], s["hd"], s["slots"])
    return {"append": _append, "tables": _tables, "reorder": _reorder}[op](s)


# ------------------------------------------------------------------------------------------------------------------------------------ 64 bits, from the definition
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(x):
    """x [..., hd] in 64 bits -> the values that its MX blocks hold"""
    parts = []
    for b in range(0, x.shape[-1], 32):
        y = x[..., b:b + 32]
        top = y.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(top, min=2.0 ** -140))) - 2, min=-125.0))
        a, best = (y / step).abs(), None
        for i in (0, 2, 4, 6, 1, 3, 5, 7):                                       # the even codes first: they keep their ties
            off = (a - _E2M1[i]).abs()
            best = (off, torch.full_like(a, _E2M1[i])) if best is None else tuple(torch.where(off < best[0], n, o) for n, o in
                                                                                  ((off, best[0]), (torch.full_like(a, _E2M1[i]), best[1])))
        parts.append(torch.where(torch.isfinite(y).all(-1, keepdim=True), torch.sign(y) * best[1] * step, torch.full_like(y, math.nan)))
    return torch.cat(parts, -1)


def _tokens(pages, hd, values):
    """pages [..., page bytes] -> what their tokens hold [..., 32, hd], in 64 bits"""
    B, at, sc, high = _blocks(hd), [], [], []
    for t in range(PAGE):
        nib = 4 * (t // 16) + t % 4
        for d in range(hd):
            if values:
                at.append(16 * hd + 4 * ((t % 16) // 4 * hd + (d % 16) * (hd // 16) + d // 16) + nib // 2)
                sc.append(32 * hd + 32 * B + 8 * B * ((t % 16) // 4) + 8 * (d // 32) + nib)
                high.append(nib % 2)
            else:
                at.append(512 * (d // 32) + t * (min(32, hd - d // 32 * 32) // 2) + d % 32 // 2)
                sc.append(32 * hd + 32 * (d // 32) + 2 * (t % 16) + t // 16)
                high.append(d % 2)
    at, sc, high = (torch.tensor(x, device=pages.device) for x in (at, sc, high))
    lut = torch.tensor(_E2M1 + tuple(-m for m in _E2M1), dtype=torch.float64, device=pages.device)
    code = torch.where(high == 1, pages[..., at].long() // 16, pages[..., at].long() % 16)
    return (lut[code] * torch.exp2(pages[..., sc].double() - 127)).unflatten(-1, (PAGE, hd))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    dev = "cuda"
    if op == "attend":
        R, Hq, hd = s["q"].shape
        H = case["kv_heads"]
        o = torch.zeros((R, Hq, hd), dtype=torch.float64, device=dev)
        for r, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            cols = (n + PAGE - 1) // PAGE
            page = s["pages"][s["tables"][r, :cols].long()]                     # [cols, H, page bytes]
            k, v = (_tokens(page, hd, values).transpose(1, 2).flatten(0, 1)[:n] for values in (False, True))     # [n, H, hd]
            for j in range(Hq // H):
                q = s["q"][r, j::Hq // H].double()                              # [H, hd]
                a = (k * q).sum(-1) * s["scale"]
                if s["alibi"] is not None:
                    a = a + s["alibi"].double()[j::Hq // H] * torch.arange(n, device=dev, dtype=torch.float64)[:, None]
                o[r, j::Hq // H] = (torch.softmax(a, 0)[..., None] * v).sum(0)
        return o
    if op == "write":
        ok = (s["slots"] >= 0)[:, None, None]
        return tuple(torch.where(ok, _nearest(x.double()), torch.zeros((), dtype=torch.float64, device=dev)) for x in (s["k"], s["v"]))
    if op == "append":
        H, hd, rot = case["heads"], case["hd"], case["rot"]
        R = case["rows"]
        whole = s["qkv"].double().view((R, H, 3, hd) if case["interleaved"] else (R, 3, H, hd))
        q, k, v = whole.unbind(2 if case["interleaved"] else 1)
        q, k = q.clone(), k.clone()
        for x in (q, k):
            for i in range(rot // 2):
                a, b = x[..., i].clone(), x[..., i + rot // 2].clone()
                c, si = s["cos"][:, i, None].double(), s["sin"][:, i, None].double()
                x[..., i], x[..., i + rot // 2] = a * c - b * si, a * si + b * c
        page, t = s["slots"] // PAGE, s["slots"] % PAGE
        res = []
        for values, x in ((False, k), (True, v)):
            y = _tokens(s["pages"][page], hd, values).transpose(1, 2)           # [R, 32, H, hd]
            y[torch.arange(R, device=dev), t] = _nearest(x)
            res.append(y.flatten(0, 1))
        return (q,) + tuple(res)
    if op == "tables":
        return None                                                             # whole numbers
    K, out = case["group"], []
    pos, src, old = s["pos"].tolist(), s["src"].tolist(), s["tables"].tolist()
    new = [list(row) for row in old]
    take = []
    for r in range(len(src)):
        a = r // K * K + src[r]
        c = pos[r] // PAGE
        new[r][:c] = old[a][:c]
        take.append(old[a][c] if pos[r] % PAGE else old[r][c])
    out.append(None)
    page = s["pages"][:, torch.tensor(take, device=dev)]                        # [layers, R, H, page bytes]
    for values in (False, True):
        out.append(torch.cat([_tokens(p, case["hd"], values).transpose(1, 2).flatten(0, 1)[None] for p in page]))
    return tuple(out)
