"""The 4-bit page cache's kernels in every form that their launch rules choose, at the precision that they claim, and at the ends of the value range; 64-bit results and bounds in
tests/_kv4_forms.py (tests/test_kv4_forms_cpu.py shows that a p of one bf16 leaves them)."""
import pytest
import torch

import _kv4 as R
import _kv4_forms as F

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from unimp_amd import ops as o
    return o


def check(got, want, bound, name=""):
    got = got.double().cpu()
    lost, over = int((~torch.isfinite(got)).sum()), (got - want).abs() / bound
    assert lost == 0, (name, lost)
    assert over.max().item() <= 1, (name, over.max().item(), int((over > 1).sum()))


# ------------------------------------------------------------------------------------------------- p in two bf16
@pytest.mark.parametrize("hd,G", F.ROWS)
def test_precision_of_p(ops, hd, G):
    q, pages, tables, lens = F.rows_case(hd, G)
    want, bound, _ = F.attend(q, pages, tables, lens, hd ** -0.5)
    check(ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), hd ** -0.5), want, bound)


@pytest.mark.parametrize("hd,K,groups,kvh,G,width", F.GROUPS)
def test_precision_of_p_in_groups(ops, hd, K, groups, kvh, G, width):
    q, pages, tables, lens, shared = F.groups_case(hd, K, groups, kvh, G, width)
    want, bound, _ = F.attend(q, pages, tables, lens, hd ** -0.5)
    check(ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), hd ** -0.5, group=K, shared_len=shared.cuda()), want, bound)


# ------------------------------------------------------------------------------------------------- forms that small calls do not reach
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("order", ["offset", "gaps", "random", "pieces", "mixed"])
def test_write_read_of_large_chunks(ops, hd, order):
    """66 chunks of 32 rows x 4 blocks of heads: above 256 workgroups a chunk has 32 rows; runs that start in its middle, end behind it, or are a few rows long"""
    tokens, heads = 2100, 16
    g = torch.Generator().manual_seed(hd)
    n_pages = 400
    page = torch.randperm(n_pages, generator=g)
    t = torch.arange(13, 13 + tokens)
    slots = page[t // 32] * 32 + t % 32
    if order == "gaps":
        slots[torch.rand(tokens, generator=g) < 0.05] = -1
        slots[70], slots[71] = n_pages * 32, -(1 << 40)
    if order == "random":
        slots = torch.randperm(n_pages * 32, generator=g)[:tokens]
    if order in ("pieces", "mixed"):                                # runs of 1 ... 16 (32) tokens anywhere in their pages
        parts = []
        for pg in page.tolist():
            n = int(torch.randint(1, 17 if order == "pieces" else 33, (1,), generator=g))
            a = int(torch.randint(0, 33 - n, (1,), generator=g))
            r = pg * 32 + a + torch.arange(n)
            parts.append(r if pg % 3 else torch.cat([r[n // 2:], r[:n // 2]]))
        slots = torch.cat(parts)[:tokens].contiguous()
        assert slots.numel() == tokens
    k, v = (torch.randn(tokens, heads, hd, generator=g).to(bf16) for _ in range(2))
    before = torch.randint(0, 256, (n_pages, heads, R.page_bytes(hd)), generator=g).to(torch.uint8)
    pages = before.cuda()
    ops.kv4_write(k.cuda(), v.cuda(), pages, slots.cuda())
    assert torch.equal(pages.cpu(), F.write_pages(before, slots, k, v))
    ok = ((slots >= 0) & (slots < n_pages * 32))[:, None, None]
    zero = torch.zeros((), dtype=torch.float64)
    for got, x in zip(ops.kv4_read(pages, slots.cuda(), hd), (k, v)):
        assert torch.equal(got.cpu().double(), torch.where(ok, R.held(x), zero))


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("hd,G", [(64, 1), (80, 2), (128, 1), (64, 3), (64, 6), (80, 3), (128, 4)])
def test_one_wave_workgroups(ops, hd, G, alibi):
    """1 024 pairs of rows and key heads on tables of at most 16 columns: a wave each"""
    rows, kvh, W = 64, 16, 4
    g = torch.Generator().manual_seed(G)
    pages = R.pack(*(torch.randn(40, kvh, 32, hd, generator=g).to(bf16) for _ in range(2)))
    tables = torch.randint(0, 40, (rows, W), generator=g).to(torch.int32)
    lens = torch.tensor([[5, 128, 64, 0, 97, 31, 1, 33][r % 8] for r in range(rows)], dtype=torch.int32)
    q = torch.randn(rows, kvh * G, hd, generator=g).to(bf16)
    slopes = torch.exp2(-8.0 * torch.arange(1, kvh * G + 1) / (kvh * G)) if alibi else None
    want, bound, _ = F.attend(q, pages, tables, lens, hd ** -0.5, slopes)
    got = ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), hd ** -0.5, alibi=None if slopes is None else slopes.cuda())
    check(got, want, bound)
    assert not got[lens == 0].any()


@pytest.mark.parametrize("hd,K,groups,kvh,G,width", [(80, 2, 4, 16, 1, 300), (128, 3, 2, 32, 1, 150), (64, 2, 2, 16, 8, 300), (128, 2, 2, 16, 3, 600)])
def test_long_shared_chunks(ops, hd, K, groups, kvh, G, width):
    """shared columns in chunks of 18 ... 37 pages (16 is the least); one row ends inside them, one behind the first chunk"""
    rows = K * groups
    assert width * groups * kvh // 512 > 16 and K * G <= 16
    g = torch.Generator().manual_seed(width)
    pages = R.pack(*(torch.randn(50, kvh, 32, hd, generator=g).to(bf16) for _ in range(2)))
    shared = torch.tensor([(width - 3) * 32 + 5 - 100 * i for i in range(groups)], dtype=torch.int32)
    tables = torch.randint(0, 50, (rows, width), generator=g).to(torch.int32)
    for r in range(rows):
        c = int(shared[r // K]) // 32
        tables[r, :c] = tables[r // K * K, :c]
    lens = torch.tensor([int(shared[r // K]) + 1 + 17 * (r % K) for r in range(rows)], dtype=torch.int32)
    lens[1], lens[-1] = 40, 32 * (width // 2) + 1
    q = torch.randn(rows, kvh * G, hd, generator=g).to(bf16)
    want, bound, _ = F.attend(q, pages, tables, lens, hd ** -0.5)
    args = q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), hd ** -0.5
    check(ops.kv4_attn_decode(*args, group=K, shared_len=shared.cuda()), want, bound)
    check(ops.kv4_attn_decode(*args), want, bound)


# ------------------------------------------------------------------------------------------------- the ends of the value range
@pytest.mark.parametrize("hd", [64, 80, 128])
def test_append_beyond_bf16(ops, hd):
    """a rotation may take two bf16 beyond bf16's largest value: such a block saturates, what is read back is finite, and the other blocks and rows are those of any append"""
    rows, heads, rot = 4, 2, hd
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(rows, 3, heads, hd, generator=g).to(bf16)
    qkv[0, 1] = 3e38
    qkv[1, 1, 1, :16] = 3e38                                        # pairs of one large and one small value
    qkv[2, 1, 0, 3], qkv[2, 1, 0, 3 + rot // 2] = 3.3e38, -3.3e38
    cos, sin = (torch.full((rows, rot // 2), 0.5 ** 0.5) for _ in range(2))
    slots = torch.tensor([0, 33, 5, 40])
    pages = torch.zeros((2, heads, R.page_bytes(hd)), dtype=torch.uint8, device="cuda")
    ops.kv4_rope_append(qkv.view(rows, -1).cuda(), heads, hd, hd, (0, heads * hd, 2 * heads * hd), rot, cos.cuda(), sin.cuda(), pages, slots.cuda())
    k, v = (x.cpu().double() for x in ops.kv4_read(pages, slots.cuda(), hd))
    turned = F.rotated(qkv[:, 1].double(), cos, sin, rot)
    assert turned.abs().max() > torch.finfo(bf16).max
    lost = int((~torch.isfinite(k)).sum())
    assert lost == 0
    assert torch.equal(k, R.held(F.saturated(turned))) and torch.equal(v, R.held(qkv[:, 2]))


@pytest.mark.parametrize("G", [1, 4, 8, 16])
@pytest.mark.parametrize("hd,power", [(64, 125), (80, 125), (128, 125), (64, -74), (80, -74), (128, -74)])
def test_values_of_any_magnitude(ops, hd, power, G):
    """values up to bf16's largest and down to 2^-74: no sum of p v leaves 32 bits, whether scores rise along the row (the maximum lags behind them), are all alike or fall"""
    kvh, W = 2, 100
    g = torch.Generator().manual_seed(hd + G)
    k = torch.randn(2 * W, kvh, 32, hd, generator=g).to(bf16)
    v = torch.randn(2 * W, kvh, 32, hd, generator=g).clamp(-3.9, 3.9)
    v[W:] = v[W:].abs()                                             # the second row's values do not cancel
    pages = R.pack(k, (v.double() * 2.0 ** power).to(bf16))
    tables = torch.arange(2 * W, dtype=torch.int32).view(2, W)
    lens = torch.tensor([3200, 3111], dtype=torch.int32)
    q = (0.5 * torch.randn(2, kvh * G, hd, generator=g)).to(bf16)
    rise = torch.full((kvh * G,), 0.02)
    for slopes in (None, rise, -rise / 8):
        want, bound, _ = F.attend(q, pages, tables, lens, hd ** -0.5, slopes)
        check(ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), hd ** -0.5, alibi=None if slopes is None else slopes.cuda()), want, bound,
              "alike" if slopes is None else slopes[0].item())


@pytest.mark.parametrize("hd,K,groups,kvh,G,width", [F.GROUPS[0], F.GROUPS[1], F.GROUPS[2], F.GROUPS[5]])
@pytest.mark.parametrize("power", [125, -74])
def test_values_of_any_magnitude_in_groups(ops, hd, K, groups, kvh, G, width, power):
    g = torch.Generator().manual_seed(hd + G)
    rows = K * groups
    v = torch.randn(30, kvh, 32, hd, generator=g).clamp(-3.9, 3.9).abs()
    pages = R.pack(torch.randn(30, kvh, 32, hd, generator=g).to(bf16), (v.double() * 2.0 ** power).to(bf16))
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    tables[:, :12] = torch.arange(12, dtype=torch.int32)
    tables[:, 12] = torch.randint(12, 30, (rows,), generator=g).to(torch.int32)
    lens = torch.tensor([385 + r % 32 for r in range(rows)], dtype=torch.int32)
    q = (0.5 * torch.randn(rows, kvh * G, hd, generator=g)).to(bf16)
    shared = torch.full((groups,), 384, dtype=torch.int32)
    rise = torch.full((kvh * G,), 0.02)
    for slopes in (None, rise):
        want, bound, _ = F.attend(q, pages, tables, lens, hd ** -0.5, slopes)
        check(ops.kv4_attn_decode(q.cuda(), pages.cuda(), tables.cuda(), lens.cuda(), hd ** -0.5, alibi=None if slopes is None else slopes.cuda(), group=K, shared_len=shared.cuda()),
              want, bound, slopes is None)
