"""A decode step of the 3B tower at cfg2 size on the bf16 cache and on 4-bit pages: ms per token-step and bytes of the cache, two passes of each in turn, and how far the logits of the two
are apart when both are fed the bf16 cache's greedy tokens (random-init weights).  Not a pytest file.
usage: python tools/bench_decode_cache.py"""
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch           # noqa: E402
import bench           # noqa: E402
from unimp_amd.decode import DecodeSession       # noqa: E402
from unimp_amd.synthetic import make_batch       # noqa: E402

dev = torch.device("cuda")
model, layout = bench.build_cfg2(dev, gate=0.5)
model.eval()
bt = make_batch(layout, 1, 8, 512, seed=7, device="cuda", vision_dtype=torch.bfloat16)
n = int(bt["attention_mask"][0].sum())
ids, vx = bt["lang_x"][:1, :n - 2], bt["vision_x"][:1]


@torch.no_grad()
def run(beams, users, kv, steps, length=None, feed=None):
    """ms per step, cache bytes; with feed (tokens [steps] of one row, or []: its own greedy tokens are appended): every step's logits"""
    prompt = ids.repeat(users, 1) if length is None else ids.repeat(users, 1 + length // ids.shape[1])[:, :length]
    model.lang_encoder._use_cached_vision_x = True
    model._encode_vision_x(vision_x=vx.repeat(users, 1, 1, 1, 1, 1))
    s = DecodeSession(model, steps + 8, reorder=beams > 1, beams=beams, kv_cache=kv)
    tok = s.prefill(prompt).float().argmax(-1)
    src = torch.arange(tok.shape[0], device=dev) if beams > 1 else None
    logits, own = [], feed is not None and not feed
    for i in range(4 + steps):
        if i == 4:
            torch.cuda.synchronize()
            t0 = time.perf_counter()
        if feed is not None:
            if own:
                feed.append(tok.clone())
            tok = feed[i]
        out = s.step(tok, src)
        if feed is not None:
            logits.append(out.float().clone())
        tok = out.float().argmax(-1)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t0) / steps * 1e3
    size = s.cache.pages.numel() if kv == "mx4" else 2 * s.cache.kv.numel()
    model.clear_conditioned_layers()
    return ms, size, logits


for beams, users, length in ((1, 1, None), (10, 1, None), (10, 4, None), (1, 16, None), (1, 1, 2000), (10, 1, 2000), (10, 4, 2000)):
    for _ in range(2):
        for kv in ("bf16", "mx4"):
            ms, size, _ = run(beams, users, kv, 40, length)
            print(f"{beams:2d} beams x {users:2d} users, prompt {length or ids.shape[1]}, {kv:4s}: {ms:.3f} ms per step, cache {size / 1e6:.0f} MB", flush=True)
for length in (None, 2000):
    feed = []
    a = torch.cat(run(1, 1, "bf16", 60, length, feed)[2])
    b = torch.cat(run(1, 1, "mx4", 60, length, feed)[2])
    print(f"greedy, prompt {length or ids.shape[1]}: logits of the 4-bit cache, relative L2 distance {float((b - a).norm() / a.norm()):.4f}, the same largest logit in "
          f"{int((a.argmax(-1) == b.argmax(-1)).sum())} of {a.shape[0]} steps", flush=True)
