"""The inputs and bounds of tests/test_kv4_forms_gpu.py, without a GPU: a p of one bf16 leaves the attention's bound on every one of them, and the expected pages of a large write are those
of the token-by-token restatement."""
import pytest
import torch

import _kv4 as R
import _kv4_forms as F


@pytest.mark.parametrize("hd,G", F.ROWS)
def test_a_p_of_eight_bits_leaves_the_bound(hd, G):
    q, pages, tables, lens = F.rows_case(hd, G)
    o, bound, cut = F.attend(q, pages, tables, lens, hd ** -0.5)
    want, loose = R.attend(q, pages, tables, lens, hd ** -0.5)
    assert ((o - want).abs() <= 1e-12).all() and (bound < loose).all()
    assert ((cut - o).abs() > bound).double().mean() > 0.02


@pytest.mark.parametrize("hd,K,groups,kvh,G,width", F.GROUPS)
def test_a_p_of_eight_bits_leaves_the_bound_in_groups(hd, K, groups, kvh, G, width):
    q, pages, tables, lens, shared = F.groups_case(hd, K, groups, kvh, G, width)
    assert K * G <= 16 and K * groups * kvh * width >= 8192         # what the shared columns' form asks for
    o, bound, cut = F.attend(q[:K], pages, tables[:K], lens[:K], hd ** -0.5)
    assert ((cut - o).abs() > bound).double().mean() > 0.02


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_expected_pages(hd):
    g = torch.Generator().manual_seed(hd)
    slots = torch.tensor([5, -1, 64, 33, 200, 6])
    k, v = (torch.randn(6, 2, hd, generator=g).to(torch.bfloat16) for _ in range(2))
    before = torch.randint(0, 256, (3, 2, R.page_bytes(hd)), generator=g).to(torch.uint8)
    want = before.clone()
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 96:
            for h in range(2):
                R.put(want[s // 32, h], s % 32, k[i, h], v[i, h])
    assert torch.equal(F.write_pages(before, slots, k, v), want)


def test_what_is_held_is_finite_in_bf16():
    """two bf16 near the largest value, turned by 45 degrees, are beyond bf16: their block's scale stays one whose codes are values of bf16"""
    x = torch.full((1, 1, 64), 3e38, dtype=torch.bfloat16).double()
    y = F.rotated(x, torch.full((1, 32), 0.5 ** 0.5), torch.full((1, 32), 0.5 ** 0.5), 64)
    assert y.abs().max() > torch.finfo(torch.bfloat16).max and R.quantise(y)[1].max() == 253
    held = R.held(F.saturated(y))
    assert torch.equal(held.to(torch.bfloat16).double(), held) and R.quantise(F.saturated(y))[1].max() == 252
