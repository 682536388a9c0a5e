"""The 4-bit page cache inside the decode path: generate(kv_cache="mx4") on every tower form, the step's logits against a bf16 cache whose contents are rounded to the same
4 bits, and the operators run together over many steps against 64-bit histories."""
import pytest
import torch

import _kv4 as R
import _parity as P

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16
CONFIGS = {"neox80": P.TINY, "neox128_parallel": P.TINY_PAR, "opt64": P.TINY_OPT, "mpt64_alibi": P.TINY_MPT, "mosaic64_qkln": P.TINY_MOSAIC}


@pytest.fixture(scope="module", params=CONFIGS, ids=list(CONFIGS))
def tower(request):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    cfg = CONFIGS[request.param]
    om, layout = P.build_oracle(cfg)
    return cfg, P.build_hip(cfg, om, layout).eval(), layout


def _prompts(cfg, layout, n):
    b = P.make_batch(cfg, layout)
    return b["vision_x"].cuda()[:n], b["lang_x"].cuda()[:n]


def test_generate(tower):
    """greedy and beams, one prompt and two of different lengths, the step as a graph and kernel by kernel: the same tokens, of the right shape; the mode leaves a bf16
    call as it was"""
    cfg, model, layout = tower
    vx, ids = _prompts(cfg, layout, 2)
    ids = ids[:, :36]
    kw = dict(max_new_tokens=40, eos_token_id=-1, pad_token_id=layout.eos)                       # past two page boundaries
    before = model.generate(vx[:1], ids[:1], **kw)
    for beams in (1, 3):
        bk = dict(kw, num_beams=beams, num_return_sequences=beams, early_stopping=False)
        one = model.generate(vx[:1], ids[:1], kv_cache="mx4", **bk)
        assert one.shape == (beams, 36 + 40) and torch.equal(one[:, :36], ids[:1].expand(beams, -1))
        assert torch.equal(one, model.generate(vx[:1], ids[:1], kv_cache="mx4", use_graph=False, **bk))
        assert torch.equal(one, model.generate(vx[:1], ids[:1], kv_cache="mx4", **bk))             # a warm signature: captured from the first step on
        mask = torch.ones_like(ids)
        mask[1, 31:] = 0                                                                         # a row that ends one token before a page does
        two = model.generate(vx, ids, attention_mask=mask, kv_cache="mx4", **bk)
        assert two.shape == (2 * beams, 36 + 40)
        assert torch.equal(two, model.generate(vx, ids, attention_mask=mask, kv_cache="mx4", use_graph=False, **bk))
    assert torch.equal(before, model.generate(vx[:1], ids[:1], **kw))


def test_step_logits_are_those_of_rounded_keys_and_values(tower, monkeypatch):
    """The same steps on a bf16 cache whose keys and values are rounded to their 4-bit values before every attention.  What is left between the two is bf16 against fp32
    between rotation and rounding (about a hundredth of the new tokens' codes) and the attention kernels' own roundings; it must be a small part of what the 4 bits change."""
    from unimp_amd import functional as F_
    from unimp_amd import ops
    from unimp_amd.decode import DecodeSession
    cfg, model, layout = tower
    vx, ids = _prompts(cfg, layout, 1)
    ids = ids[:, :30]
    toks = torch.randint(0, 200, (6,), generator=torch.Generator().manual_seed(0)).tolist()

    def logits(kv_cache, rounded=False):
        with torch.no_grad(), monkeypatch.context() as mp:
            if rounded:
                mp.setattr(F_, "DECODE_FUSED", False)
                plain = F_._decode_attn

                def attn(q, k, v, *a, **kw):
                    for t in (k, v):
                        rows, cap, nh, hd = t.shape
                        pages = torch.zeros(((rows * cap + 31) // 32, nh, ops.kv4_page_bytes(hd)), dtype=torch.uint8, device=t.device)
                        slots = torch.arange(rows * cap, device=t.device)
                        flat = t.reshape(-1, nh, hd)
                        ops.kv4_write(flat, flat, pages, slots)
                        t.copy_(ops.kv4_read(pages, slots, hd)[0].view_as(t))
                    return plain(q, k, v, *a, **kw)
                mp.setattr(F_, "_decode_attn", attn)
            model.lang_encoder._use_cached_vision_x = True
            model._encode_vision_x(vision_x=vx[:1])
            s = DecodeSession(model, len(toks), reorder=False, graph=False, kv_cache=kv_cache)
            s.prefill(ids)
            out = torch.stack([s.step(torch.tensor([t], device="cuda")).float()[0].clone() for t in toks])
            model.clear_conditioned_layers()
            model.lang_encoder._use_cached_vision_x = False
            return out
    plain, rounded, paged = logits("bf16"), logits("bf16", True), logits("mx4")
    assert torch.isfinite(paged).all()
    effect, left = P.rel_l2(rounded, plain), P.rel_l2(paged, rounded)
    assert left <= effect / 2 + 2 ** -8, (left, effect)


def test_operators_together():
    """page tables, prompt writes, rotary appends, beam reorders and the attention as a decode runs them -- two prompts of different lengths, five beams, forty steps over two
    page boundaries, eager and as one captured graph -- against histories kept token by token in 64 bits"""
    from unimp_amd import ops
    K, G, nh, hd, new = 5, 2, 32, 80, 40
    rows, host_len = K * G, [52, 31]
    g = torch.Generator().manual_seed(0)
    cols = [-(-(n + new) // 32) for n in host_len]
    n_pages = sum(c + (K - 1) * (c - n // 32) for c, n in zip(cols, host_len))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    order = torch.randperm(n_pages, generator=g).to(torch.int32).cuda()
    length = i32(host_len).repeat_interleave(K)
    first = i32([1] + [0] * (K - 1)).repeat(G)
    shared, scale = i32(host_len), 0.2
    prompt = (torch.randn(2, sum(host_len), nh, hd, generator=g)).to(bf16)
    step_qkv = torch.randn(new, rows, 3 * nh * hd, generator=g).to(bf16)
    step_src = torch.randint(0, K, (new, rows), generator=g)
    turn = torch.rand(new, rows, hd // 2, generator=g).double() * 100

    def run(graph):
        pages = torch.randint(0, 256, (n_pages, nh, ops.kv4_page_bytes(hd)), dtype=torch.uint8, device="cuda")
        tables = torch.full((rows, max(cols)), -1, dtype=torch.int32, device="cuda")
        zero = torch.zeros(rows, dtype=torch.int32, device="cuda")
        mapped, cursor, slots, cu = ops.page_tables_extend(tables, zero, zero, length * first, order, zero[:1].clone(), sum(host_len), cover=length + new, group=K,
                                                           shared_len=shared)
        assert cursor.item() == n_pages and (slots >= 0).all()
        ops.kv4_write(prompt[0].cuda(), prompt[1].cuda(), pages, slots)
        ops.kv4_reorder_beams(pages, tables, K, torch.zeros(rows, dtype=torch.long, device="cuda"), length.long())
        qkv, src = torch.zeros(rows, 3 * nh * hd, dtype=bf16, device="cuda"), torch.zeros(rows, dtype=torch.long, device="cuda")
        cos, sin = torch.zeros(rows, hd // 2, device="cuda"), torch.zeros(rows, hd // 2, device="cuda")
        cached, ones = length.clone(), torch.ones_like(length)

        def body():
            ops.kv4_reorder_beams(pages, tables, K, src, cached.long())
            s = ops.page_tables_extend(tables, mapped, cached, ones, order, cursor, rows)[2]
            q = ops.kv4_rope_append(qkv, nh, 3 * hd, hd, (0, hd, 2 * hd), hd, cos, sin, pages, s)
            cached.add_(1)
            return ops.kv4_attn_decode(q, pages, tables, cached, scale, group=K, shared_len=shared)
        outs, cg = [], None
        for i in range(new):
            qkv.copy_(step_qkv[i].cuda()), src.copy_(step_src[i].cuda()), cos.copy_(turn[i].cos().float().cuda()), sin.copy_(turn[i].sin().float().cuda())
            if graph and i > 0:
                if cg is None:
                    cg = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(cg):
                        o = body()
                cg.replay()
            else:
                o = body()
            outs.append(o.clone())
        return torch.stack(outs).cpu()
    eager = run(False)
    assert torch.equal(eager, run(True))

    # the histories: per row a list of (k, v) of its tokens, as held
    hist, at = [], 0
    for n in host_len:
        k, v = R.held(prompt[0, at:at + n]), R.held(prompt[1, at:at + n])
        hist += [(k, v)] * K
        at += n
    for i in range(new):
        hist = [hist[r // K * K + int(step_src[i, r])] for r in range(rows)]
        x = step_qkv[i].double().view(rows, nh, 3, hd)
        c, s, h = turn[i].cos().float().double()[:, None], turn[i].sin().float().double()[:, None], hd // 2
        q, k = (torch.cat([t[..., :h] * c - t[..., h:] * s, t[..., h:] * c + t[..., :h] * s], -1) for t in (x[:, :, 0], x[:, :, 1]))
        q = q.to(bf16)
        k, v = R.held(k), R.held(x[:, :, 2])
        hist = [(torch.cat([hist[r][0], k[r:r + 1]]), torch.cat([hist[r][1], v[r:r + 1]])) for r in range(rows)]
        if i % 7 and i != new - 1:
            continue
        for r in range(rows):
            kk, vv = hist[r]
            n = kk.shape[0]
            pad = -n % 32
            z = lambda t: torch.cat([t, torch.zeros(pad, nh, hd, dtype=t.dtype)]).view(-1, 32, nh, hd).transpose(1, 2)
            want, bound = R.attend(q[r:r + 1], R.pack(z(kk), z(vv)), torch.arange((n + pad) // 32)[None].to(torch.int32), torch.tensor([n]), scale)
            far = (eager[i, r].double() - want[0]).abs() - bound[0]
            assert far.max().item() <= 0, (i, r, far.max().item())


def test_a_longer_session_of_a_warm_signature():
    """a step signature counts the cache in 128 slots: a second session of it that reaches further captures its first step at once and must find its rotary rows made"""
    from unimp_amd.decode import DecodeSession
    om, layout = P.build_oracle(P.TINY)
    model = P.build_hip(P.TINY, om, layout).eval()
    vx, ids = _prompts(P.TINY, layout, 1)
    long = ids.repeat(1, 12)[:, :500]
    for n, kv in ((460, "bf16"), (500, "bf16"), (460, "mx4"), (500, "mx4")):
        with torch.no_grad():
            model.lang_encoder._use_cached_vision_x = True
            model._encode_vision_x(vision_x=vx)
            s = DecodeSession(model, 12, reorder=False, kv_cache=kv)
            s.prefill(long[:, :n])
            for t in range(2):
                assert torch.isfinite(s.step(torch.tensor([t + 5], device="cuda"))).all()
            model.clear_conditioned_layers()
            model.lang_encoder._use_cached_vision_x = False
