"""Grouped-query layers over an 8-bit paged KV cache, as cases for timing.

A grouped-query layer has H query heads that share H_kv key / value heads (H a
multiple of H_kv) of D channels.  Its cache is pages of 64 tokens, e4m3fn codes
with one power-of-two scale for each (page, kv head) of K and one of V:

* K values, head h, token r, channel c: byte (64 h + r) D + c;
* V values after all K values, head h, channel c, token r: byte (D h + c) 64 + at(r),
  at(r) = 16 ((r / 4) % 4) + 4 (r / 16) + r % 4;
* then the fp32 K scales [H_kv], then the fp32 V scales [H_kv].

A summary record, kept for each page by a layer that attends to selected blocks, is the mean
key of each head as D int8 codes, then the fp32 power-of-two scales [H_kv].

Kinds of cases:

* ``norm``: RMS norms of queries and keys for each head and the position rotation.
* ``write``: the step's keys and values into the cache (``prep``: from the raw
  projections, norm and rotation included; ``summary``: with the pages' mean keys).
* ``attn``: causal attention over the cache, ``rows`` query tokens a sequence.
* ``block``: each query token and kv head picks ``blocks`` pages by their mean
  keys and attends to them.

Inputs come from the seed alone; sequence lengths come from the case, so that
its work is the same for every seed.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
PAGE = 64
KEEP_FIRST, KEEP_LAST = 1, 2  # blocks that every row attends to: the first, and its last two
F64 = torch.float64


def _ops():
    root = str(Path(__file__).resolve().parents[1] / "vllm-ernie_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from ernie_kv import ops

    return ops


# --------------------------------------------------------------------------- cases
def listed() -> list:
    return [
        # a decode step's norms and rotation on their own, 64 users: launch and latency count
        dict(name="norm_64", kind="norm", rows=64, heads=64, kv_heads=8, dim=128, rope=128, offset=0, inter=False),
        # a prompt's chunk with the rotation on interleaved pairs of the last 64 of 256 channels
        dict(name="norm_8191", kind="norm", rows=8191, heads=64, kv_heads=8, dim=256, rope=64, offset=192, inter=True),
        # a decode step's cache write of 64 users, norm and rotation included
        dict(name="write_64x1", kind="write", seqs=64, lo=500, hi=9000, rows=1, heads=64, kv_heads=8, dim=128,
             prep=True, summary=False),
        # prompts' chunks into the cache of a layer that selects blocks, from the middle of a page on
        dict(name="write_16x8192", kind="write", seqs=16, lo=777, hi=900, rows=8192, heads=32, kv_heads=8, dim=128,
             prep=False, summary=True),
        # one user's chat turn: the fewest bytes
        dict(name="attn_decode_1x4k", kind="attn", seqs=1, lo=4096, hi=4096, rows=1, heads=32, kv_heads=8, dim=128,
             window=0, sinks=False),
        # a server's ordinary batch at mixed, ragged contexts, with attention sinks
        dict(name="attn_decode_13x2k_48k", kind="attn", seqs=13, lo=2000, hi=48000, rows=1, heads=64, kv_heads=8,
             dim=128, window=0, sinks=True),
        # the benchmark's decode batch: 128K contexts
        dict(name="attn_decode_32x128k", kind="attn", seqs=32, lo=131072, hi=131072, rows=1, heads=64, kv_heads=8,
             dim=128, window=0, sinks=False),
        # decode with two draft tokens a sequence, three query heads a kv head, wide heads
        dict(name="attn_draft_9x16k_3", kind="attn", seqs=9, lo=9000, hi=16384, rows=3, heads=24, kv_heads=8, dim=256,
             window=0, sinks=False),
        # a chunk of a long prompt (chunked prefill)
        dict(name="attn_prefill_4096_32k", kind="attn", seqs=1, lo=32768, hi=32768, rows=4096, heads=32, kv_heads=8,
             dim=128, window=0, sinks=False),
        # short prompts prefilled whole through a sliding-window layer with a kv head for each query head
        dict(name="attn_prefill_3x777", kind="attn", seqs=3, lo=777, hi=777, rows=777, heads=16, kv_heads=16, dim=64,
             window=128, sinks=True),
        # the benchmark's decode batch, 64 selected blocks a row
        dict(name="block_decode_32x128k", kind="block", seqs=32, lo=131072, hi=131072, rows=1, heads=64, kv_heads=8,
             dim=128, blocks=64),
        # a short chunk behind a long context, 32 selected blocks a row
        dict(name="block_chunk_333_48k", kind="block", seqs=1, lo=48000, hi=48000, rows=333, heads=32, kv_heads=4,
             dim=128, blocks=32),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "write", "chunk", "attn", "attn", "attn", "prefill", "block", "block"])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16])
    dim = rng.choice([64, 128, 128, 128, 256])
    if kind == "norm":
        dim = rng.choice([64, 80, 128, 128, 192, 256, 512])
        rope = rng.choice([32, 64, dim])
        rope, offset = min(rope, dim), rng.choice([0, dim - min(rope, dim)])
        return dict(kind="norm", rows=_log(rng, 1, 8192 * 128 // max(dim, 128)), heads=min(heads, 64), kv_heads=kv,
                    dim=dim, rope=rope, offset=offset, inter=rng.random() < 0.5)
    if kind == "write":
        prep = rng.random() < 0.6
        hi = _log(rng, 64, 16384)
        return dict(kind="write", seqs=_log(rng, 1, 64), lo=hi // 3, hi=hi, rows=rng.choice([1, 1, 1, 2, 3, 7]),
                    heads=heads, kv_heads=kv, dim=dim, prep=prep, summary=not prep and rng.random() < 0.6)
    if kind == "chunk":
        prep, rows = rng.random() < 0.4, _log(rng, 33, 8192)
        return dict(kind="write", seqs=rng.randint(1, max(1, min(12, 60_000 // rows))), lo=0,
                    hi=rng.choice([0, 64, 1000]), rows=rows, heads=min(heads, 64), kv_heads=kv, dim=dim, prep=prep,
                    summary=not prep and rng.random() < 0.6)
    if kind == "attn":
        seqs = _log(rng, 1, 48)
        hi = _log(rng, 40, min(131072, 1_500_000 // seqs))
        return dict(kind="attn", seqs=seqs, lo=max(8, int(hi * rng.uniform(0.2, 1.0))), hi=hi,
                    rows=rng.choice([1, 1, 1, 2, 3, 5, 8]), heads=heads, kv_heads=kv, dim=dim,
                    window=rng.choice([0, 0, 0, 128, 1000, 4096]), sinks=rng.random() < 0.4)
    if kind == "prefill":
        rows, seqs = _log(rng, 40, 2500), rng.randint(1, 3)
        hi = rows if rng.random() < 0.4 else _log(rng, rows, 24000 // seqs + rows)
        return dict(kind="attn", seqs=seqs, lo=max(rows, hi // 2), hi=hi, rows=rows, heads=min(heads, 32), kv_heads=kv,
                    dim=dim, window=rng.choice([0, 0, 0, 128, 1000]), sinks=rng.random() < 0.4)
    n = rng.choice([8, 16, 32, 50, 64, 128])
    few = rng.random() < 0.75
    rows = rng.choice([1, 1, 1, 2, 3]) if few else _log(rng, 20, 300)
    seqs = _log(rng, 1, 48) if few else 1
    hi = _log(rng, 300, min(131072, 2_000_000 // seqs))
    return dict(kind="block", seqs=seqs, lo=max(rows, int(hi * rng.uniform(0.3, 1.0))), hi=max(rows, hi), rows=rows,
                heads=heads, kv_heads=kv, dim=dim, blocks=n if few else min(n, 32))


def _contexts(case: dict) -> list:
    """Tokens of each sequence before a write's new rows, or with the query rows of the
    attending kinds; the same for every seed."""
    r = random.Random("%(seqs)d/%(lo)d/%(hi)d" % case)
    least = 0 if case["kind"] == "write" else case["rows"]
    return [max(least, r.randint(case["lo"], case["hi"])) for _ in range(case["seqs"])]


# --------------------------------------------------------------------------- formats
def _exponent(amax: torch.Tensor, top: float) -> torch.Tensor:
    """The smallest e with fl32(max(amax, 1e-10) * fl32(1 / top)) <= 2^e."""
    v = amax.float().clamp_min(1e-10) * torch.tensor(1.0 / top, dtype=torch.float32, device=amax.device)
    m, e = torch.frexp(v)
    return e - (m == 0.5).to(e.dtype)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _codes(x: torch.Tensor) -> torch.Tensor:
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).to(dtype)


def _at(dev) -> torch.Tensor:
    """The byte of each token within a channel's 64 of V."""
    r = torch.arange(PAGE, device=dev)
    return 16 * (r // 4 % 4) + 4 * (r // 16) + r % 4


def _parts(cache: torch.Tensor, kv: int, dim: int):
    """Views of a cache: K [N, kv, 64, dim], V [N, kv, dim, 64] bytes, scales [N, 2, kv] fp32."""
    n = kv * PAGE * dim
    k, v = cache[:, :n].unflatten(1, (kv, PAGE, dim)), cache[:, n:2 * n].unflatten(1, (kv, dim, PAGE))
    return k, v, cache[:, 2 * n:2 * n + 8 * kv].view(torch.float32).unflatten(1, (2, kv))


def _summary_parts(summary: torch.Tensor, kv: int, dim: int):
    return summary[:, :kv * dim].view(torch.int8).unflatten(1, (kv, dim)), summary[:, kv * dim:].view(torch.float32)


def _round16(n: int) -> int:
    return (n + 15) // 16 * 16


# --------------------------------------------------------------------------- preparation
def _tables(ctxs: list, g, dev):
    pps = [(c + PAGE - 1) // PAGE for c in ctxs]
    pages = max(1, sum(pps))
    perm = torch.randperm(pages, device=dev, generator=g).int()
    bt = torch.full((len(ctxs), max(1, max(pps))), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(pps):
        bt[b, :n] = perm[at:at + n]
        at += n
    return pages, bt


def _filled(pages: int, kv: int, dim: int, g, dev) -> torch.Tensor:
    """Pages of keys with a mean in each channel, a drift from page to page, and N(0, 1) values."""
    cache = torch.empty((pages, _round16(kv * (2 * PAGE * dim + 8))), dtype=torch.uint8, device=dev)
    k, v, scales = _parts(cache, kv, dim)
    mean = 24 * torch.randn(kv, 1, dim, device=dev, generator=g)
    step = max(1, (1 << 27) // (kv * PAGE * dim))
    for a in range(0, pages, step):
        n = min(pages, a + step) - a
        drift = 16 * torch.randn(n, kv, 1, dim, device=dev, generator=g)
        x = torch.randn(n, kv, PAGE, dim, device=dev, generator=g)
        k[a:a + n] = _codes(x.mul_(40).add_(mean).add_(drift))
        v[a:a + n] = _codes(torch.randn(n, kv, dim, PAGE, device=dev, generator=g).mul_(64))
    scales.copy_(_pow2(torch.randint(-7, -4, (pages, 2, kv), device=dev, generator=g)))
    return cache


def _table(n: int, rope: int, dev) -> torch.Tensor:
    inv = 2.5e6 ** (-torch.arange(rope // 2, device=dev, dtype=F64) * 2 / rope)
    ang = torch.arange(n, device=dev, dtype=F64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    kind, H, kv, D, rows = case["kind"], case["heads"], case["kv_heads"], case["dim"], case["rows"]
    st = dict(kind=kind, heads=H, kv=kv, dim=D, rows=rows)
    if kind == "norm":
        top = 32768
        qkv = rnd(rows, (H + 2 * kv) * D).bfloat16()  # one projection's rows, split without copies
        return {**st, "q": qkv[:, :H * D].view(rows, H, D), "k": qkv[:, H * D:(H + kv) * D].view(rows, kv, D),
                "q_w": 1 + 0.1 * rnd(D), "k_w": 1 + 0.1 * rnd(D), "table": _table(top, case["rope"], dev),
                "positions": torch.randint(0, top, (rows,), device=dev, generator=g), "inter": case["inter"],
                "offset": case["offset"]}
    ctxs = _contexts(case)
    S, T = len(ctxs), len(ctxs) * rows
    first = [c if kind == "write" else c - rows for c in ctxs]
    pages, bt = _tables([c + rows for c in first], g, dev)
    start = torch.tensor(first, device=dev)
    st.update(bt=bt, start=start, qsl=(torch.arange(S + 1, device=dev) * rows).int(),
              positions=(start[:, None] + torch.arange(rows, device=dev)).flatten().contiguous(),
              req=torch.arange(S, dtype=torch.int32, device=dev).repeat_interleave(rows),
              max_len=max(first) + rows, scale=D ** -0.5, cache=_filled(pages, kv, D, g, dev))
    if kind == "write":
        # a few rows in a hundred are larger than what their page's scale was made for
        big = 1 + 7 * (torch.rand(T, 1, 1, device=dev, generator=g) < 0.05)
        qkv = rnd(T, H + 2 * kv, D)
        qkv[:, H:] *= big
        qkv = qkv.bfloat16()
        touched = [(b, p) for b, c in enumerate(first) for p in range(c // PAGE, (c + rows - 1) // PAGE + 1)]
        st.update(q=qkv[:, :H], k=qkv[:, H:H + kv], v=qkv[:, H + kv:], prep=case["prep"], inter=False, offset=0,
                  touched=torch.tensor(touched, device=dev), summary=None)
        if case["prep"]:
            st.update(q_w=1 + 0.1 * rnd(D), k_w=1 + 0.1 * rnd(D), table=_table(st["max_len"], D, dev))
        if case["summary"]:
            st["summary"] = torch.zeros((pages, _round16(kv * (D + 4))), dtype=torch.uint8, device=dev)
        return st
    st.update(q=(2 * rnd(T, H, D)).bfloat16(), sinks=rnd(H) if case.get("sinks") else None,
              window=case.get("window", 0), out=torch.empty((T, H, D), dtype=torch.bfloat16, device=dev),
              lse=torch.empty((T, H), dtype=torch.float32, device=dev))
    if kind == "block":
        st["summary"] = torch.zeros((pages, _round16(kv * (D + 4))), dtype=torch.uint8, device=dev)
        step = max(1, (1 << 27) // (kv * PAGE * D))
        for a in range(0, pages, step):
            at = torch.arange(a, min(pages, a + step), device=dev)
            _summarize(st, at, torch.full_like(at, PAGE))
        st["ids"] = torch.empty((T, kv, case["blocks"]), dtype=torch.int32, device=dev)
    return st


def _summarize(st: dict, pages: torch.Tensor, count: torch.Tensor) -> None:
    """Mean keys of the first `count` tokens of `pages`: sums of codes, which are exact in fp32."""
    kv, D = st["kv"], st["dim"]
    codes, scales = _summary_parts(st["summary"], kv, D)
    k, _, s = _parts(st["cache"], kv, D)
    live = torch.arange(PAGE, device=pages.device) < count[:, None]
    mean = _values(k[pages]).masked_fill(~live[:, None, :, None], 0).sum(2) / count[:, None, None]
    e = _exponent(mean.abs().amax(-1), 127.0)
    codes[pages] = torch.round(mean / _pow2(e)[..., None]).clamp(-127, 127).to(torch.int8)
    scales[pages.unsqueeze(1), torch.arange(kv, device=pages.device)] = _pow2(e) * s[pages, 0]


# --------------------------------------------------------------------------- one pass
def run(st: dict):
    if own:
        return _run_own(st)
    return {"norm": _plain_norm, "write": _plain_write, "attn": _plain_attn, "block": _plain_block}[st["kind"]](st)


def _written(st: dict, q) -> dict:
    kv, D = st["kv"], st["dim"]
    n = 2 * kv * PAGE * D
    out = {"codes": st["cache"][:, :n].view(torch.float8_e4m3fn),
           "scales": st["cache"][:, n:n + 8 * kv].view(torch.float32), "q": q}
    if st["summary"] is not None:
        out["summary"], out["summary_scales"] = _summary_parts(st["summary"], kv, D)
        out["summary_scales"] = out["summary_scales"][:, :kv]
    return out


def _run_own(st: dict):
    ops = _ops()
    kind = st["kind"]
    if kind == "norm":
        q, k = ops.qk_norm_rope(st["q"], st["k"], st["q_w"], st["k_w"], EPS, st["table"], st["positions"],
                                interleaved=st["inter"], rope_offset=st["offset"])
        return {"q": q, "k": k}
    if kind == "write":
        q = None
        if st["prep"]:
            q = ops.gqa_prologue(st["q"], st["k"], st["v"], st["q_w"], st["k_w"], EPS, st["table"], st["positions"],
                                 st["qsl"], st["rows"], st["bt"], st["cache"], summary=st["summary"])
        else:
            ops.gqa_append(st["k"], st["v"], st["positions"], st["qsl"], st["rows"], st["bt"], st["cache"],
                           summary=st["summary"])
        return _written(st, q)
    if kind == "attn":
        ops.gqa_attention(st["q"], st["cache"], st["kv"], st["bt"], st["positions"], st["qsl"], st["rows"],
                          st["max_len"], st["scale"], st["out"], st["lse"], sinks=st["sinks"], window=st["window"])
        return {"out": st["out"], "lse": st["lse"]}
    ops.gqa_block_select(st["q"], st["summary"], st["kv"], st["bt"], st["positions"], st["req"], st["max_len"],
                         st["ids"], keep_first=KEEP_FIRST, keep_last=KEEP_LAST)
    ops.gqa_block_attention(st["q"], st["cache"], st["kv"], st["bt"], st["positions"], st["req"], st["ids"],
                            st["scale"], st["out"], st["lse"], sinks=st["sinks"])
    return {"out": st["out"], "lse": st["lse"], "ids": st["ids"]}


def _norm_rotate(x: torch.Tensor, w: torch.Tensor, st: dict) -> torch.Tensor:
    """x [T, heads, D]: RMS norm of each head, then the rotation of `rope` channels from `offset` on."""
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    cs = st["table"][st["positions"]][:, None]
    half, a = cs.shape[-1] // 2, st["offset"]
    c, s, y = cs[..., :half], cs[..., half:], x[..., a:a + 2 * half]
    if st["inter"]:
        e, o = y[..., 0::2], y[..., 1::2]
        y = torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)
    else:
        e, o = y[..., :half], y[..., half:]
        y = torch.cat([e * c - o * s, o * c + e * s], -1)
    return torch.cat([x[..., :a], y, x[..., a + 2 * half:]], -1).bfloat16()


def _plain_norm(st: dict):
    return {"q": _norm_rotate(st["q"], st["q_w"], st), "k": _norm_rotate(st["k"], st["k_w"], st)}


def _plain_write(st: dict):
    kv, D, rows = st["kv"], st["dim"], st["rows"]
    q, new_k, new_v = None, st["k"], st["v"]
    if st["prep"]:
        q, new_k = _norm_rotate(st["q"], st["q_w"], st), _norm_rotate(new_k, st["k_w"], st)
    k, v, scales = _parts(st["cache"], kv, D)
    b, p = st["touched"].unbind(1)
    page = st["bt"][b, p].long()
    pos = p[:, None] * PAGE + torch.arange(PAGE, device=b.device)
    rel = pos - st["start"][b, None]
    new, old = (rel >= 0) & (rel < rows), rel < 0
    at = b[:, None] * rows + rel.clamp(0, rows - 1)
    held = (k[page], v[page][..., _at(b.device)].transpose(2, 3))  # [n, kv, 64, D] bytes
    stored = []
    for i, (x, codes) in enumerate(((new_k, held[0]), (new_v, held[1]))):
        x = x.float()[at].transpose(1, 2).masked_fill(~new[:, None, :, None], 0)  # [n, kv, 64, D]
        s = _pow2(_exponent(x.abs().amax((2, 3)), 448.0))
        was = scales[page, i]
        s = torch.where(old.any(1, keepdim=True), torch.maximum(s, was), s)
        again = _codes(_values(codes) * (was / s)[..., None, None])
        codes = torch.where(old[:, None, :, None], again, codes)
        stored.append(torch.where(new[:, None, :, None], _codes(x / s[..., None, None]), codes))
        scales[page, i] = s
    k[page] = stored[0]
    inv = torch.argsort(_at(b.device))
    v[page] = stored[1].transpose(2, 3)[..., inv]
    if st["summary"] is not None:
        _summarize(st, page, (new | old).sum(1))
    return _written(st, q)


def _softmax(x: torch.Tensor, sinks):
    """x [..., keys] with -inf at what is masked -> (weights, lse); `sinks` broadcasts against x[..., 0]."""
    m = x.amax(-1)
    if sinks is not None:
        m = torch.maximum(m, sinks)
    x = x.sub_(m[..., None]).exp_()
    l = x.sum(-1)
    lse = m + l.log()
    return x.div_((l if sinks is None else l + (sinks - m).exp())[..., None]), lse


def _plain_attn(st: dict):
    kv, D, rows, H = st["kv"], st["dim"], st["rows"], st["heads"]
    G, S = H // kv, st["bt"].shape[0]
    k, v, scales = _parts(st["cache"], kv, D)
    page = st["bt"].clamp_min(0).long()
    L = page.shape[1] * PAGE
    q = st["q"].float().view(S, rows, kv, G, D).transpose(1, 2).reshape(S * kv, rows * G, D)
    keys = (_values(k[page]) * scales[page, 0][..., None, None]).transpose(1, 2).reshape(S * kv, L, D)
    x = torch.bmm(q, keys.transpose(1, 2)).mul_(st["scale"]).view(S, kv, rows, G, L)
    del keys
    pos, at = st["positions"].view(S, 1, rows, 1, 1), torch.arange(L, device=q.device)
    seen = at <= pos
    if st["window"]:
        seen &= at > pos - st["window"]
    x.masked_fill_(~seen, -math.inf)
    sinks = st["sinks"]
    w, lse = _softmax(x, None if sinks is None else sinks.view(1, kv, 1, G))
    vals = (_values(v[page]) * scales[page, 1][..., None, None])[..., _at(q.device)]  # [S, P, kv, D, 64]
    vals = vals.permute(0, 2, 1, 4, 3).reshape(S * kv, L, D)
    out = torch.bmm(w.view(S * kv, rows * G, L), vals).view(S, kv, rows, G, D)
    return {"out": out.transpose(1, 2).reshape(S * rows, H, D).bfloat16(),
            "lse": lse.transpose(1, 2).reshape(S * rows, H)}


def _plain_select(st: dict) -> torch.Tensor:
    """[T, kv, blocks] blocks of the largest scores, the first and the last ones before them, ascending, -1 behind."""
    kv, D, rows, n = st["kv"], st["dim"], st["rows"], st["ids"].shape[2]
    S, G = st["bt"].shape[0], st["heads"] // kv
    codes, scales = _summary_parts(st["summary"], kv, D)
    page = st["bt"].clamp_min(0).long()
    q = st["q"].float().view(-1, kv, G, D)
    e = _exponent(q.abs().amax((2, 3)), 127.0)
    q = torch.round(q / _pow2(e)[..., None, None]).clamp(-127, 127)
    q = q.view(S, rows, kv, G, D).transpose(1, 2).reshape(S * kv, rows * G, D)
    m = codes[page].float().transpose(1, 2).reshape(S * kv, -1, D)
    dot = torch.bmm(q, m.transpose(1, 2)).view(S, kv, rows, G, -1)  # whole numbers below 2^24
    score = dot.amax(3) * scales[page][..., :kv].transpose(1, 2)[:, :, None]
    P = score.shape[-1]
    j, last = torch.arange(P, device=q.device), (st["positions"] // PAGE).view(S, 1, rows, 1)
    score = score.masked_fill((j < KEEP_FIRST) | (j > last - KEEP_LAST), math.inf).masked_fill(j > last, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True)
    ids = order.indices[..., :n].masked_fill(order.values[..., :n] == -math.inf, P)
    ids = torch.nn.functional.pad(ids, (0, max(0, n - P)), value=P).sort(-1).values
    return ids.masked_fill(ids == P, -1).int().transpose(1, 2).reshape(S * rows, kv, n)


def _plain_block(st: dict):
    kv, D, H = st["kv"], st["dim"], st["heads"]
    G, T = H // kv, st["q"].shape[0]
    ids = _plain_select(st)
    k, v, scales = _parts(st["cache"], kv, D)
    n, h = ids.shape[2], torch.arange(kv, device=ids.device)[:, None]
    page = st["bt"][st["req"].long()[:, None, None], ids.clamp_min(0).long()].long()
    q = st["q"].float().view(T * kv, G, D)
    keys = (_values(k[page, h]) * scales[page, 0, h][..., None, None]).view(T * kv, n * PAGE, D)
    x = torch.bmm(q, keys.transpose(1, 2)).mul_(st["scale"]).view(T, kv, G, n, PAGE)
    del keys
    at = ids.long()[..., None] * PAGE + torch.arange(PAGE, device=ids.device)
    seen = (ids >= 0)[..., None] & (at <= st["positions"].view(T, 1, 1, 1))
    x = x.masked_fill_(~seen[:, :, None], -math.inf).flatten(3)
    sinks = st["sinks"]
    w, lse = _softmax(x, None if sinks is None else sinks.view(1, kv, G))
    vals = (_values(v[page, h]) * scales[page, 1, h][..., None, None])[..., _at(ids.device)]  # [T, kv, n, D, 64]
    vals = vals.transpose(3, 4).reshape(T * kv, n * PAGE, D)
    out = torch.bmm(w.view(T * kv, G, -1), vals).view(T, H, D)
    return {"out": out.bfloat16(), "lse": lse.view(T, H), "ids": ids}


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    kind, H, kv, D, rows = case["kind"], case["heads"], case["kv_heads"], case["dim"], case["rows"]
    if kind == "norm":
        return {"bytes": 4 * rows * (H + kv) * D + rows * (4 * case["rope"] + 8), "flops": 8 * rows * (H + kv) * D}
    ctxs, G = _contexts(case), H // kv
    T = len(ctxs) * rows
    if kind == "write":
        pages = sum((c + rows - 1) // PAGE - c // PAGE + 1 for c in ctxs)
        size = T * kv * D * 6 + pages * kv * 8  # two rows of bf16 in, of codes out
        size += (T * (4 * H * D + 4 * D + 8)) if case["prep"] else 0
        if case["summary"]:  # the page's earlier keys are part of its mean
            size += sum(c % PAGE for c in ctxs) * kv * D + pages * kv * (D + 4)
        return {"bytes": size, "flops": T * (8 * kv * D + (8 * (H + kv) * D if case["prep"] else 0))}
    ends = T * H * (4 * D + 4)  # q in, out and lse back
    token = kv * (2 * D + 8 / PAGE)
    if kind == "attn":
        w = case["window"] or 1 << 60
        seen = [min(p + 1, w) for n in ctxs for p in range(n - rows, n)]
        tokens = sum(min(n, w - 1 + rows) for n in ctxs)
        return {"bytes": int(tokens * token) + ends, "flops": 4 * D * H * sum(seen)}
    size, flops = ends + 4 * T * kv * case["blocks"], 0
    for n in ctxs:
        blocks = (n - 1) // PAGE + 1
        size += blocks * kv * (D + 4)  # every page's mean key once, and each selected page once where rows share it
        taken = [min(case["blocks"], p // PAGE + 1) for p in range(n - rows, n)]
        size += int(min(blocks, sum(taken)) * PAGE * token)
        flops += sum(2 * D * H * (p // PAGE + 1) + 4 * D * H * PAGE * t for p, t in zip(range(n - rows, n), taken))
    return {"bytes": size, "flops": flops}


# --------------------------------------------------------------------------- 64-bit restatement
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if st["kind"] == "norm":
        return {"q": _exact_turn(st["q"], st["q_w"], st), "k": _exact_turn(st["k"], st["k_w"], st)}
    return {"write": _exact_write, "attn": _exact_attn, "block": _exact_block}[st["kind"]](st)


def _exact_turn(x, w, st):
    """Each pair of channels as a complex number, turned by its angle."""
    x = x.double()
    x = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    half, a = st["table"].shape[1] // 2, st["offset"]
    turn = torch.complex(st["table"][:, :half].double(), st["table"][:, half:].double())[st["positions"], None]
    i = torch.arange(half, device=x.device)
    first, second = (a + 2 * i, a + 2 * i + 1) if st["inter"] else (a + i, a + half + i)
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_write(st):
    """Unrounded codes: what each value is in units of its page's scale (a prepared key is one of bf16)."""
    kv, D, rows = st["kv"], st["dim"], st["rows"]
    q, new = None, [st["k"].double(), st["v"].double()]
    if st["prep"]:
        q, new[0] = _exact_turn(st["q"], st["q_w"], st), _exact_turn(st["k"], st["k_w"], st).bfloat16().double()
    k, v, scales = _parts(st["cache"], kv, D)
    values = [_values(k, F64), _values(v, F64)[..., _at(k.device)].transpose(2, 3).contiguous()]
    scales = scales.double().clone()
    for b, c in enumerate(st["start"].tolist()):
        for p in range(c // PAGE, (c + rows - 1) // PAGE + 1):
            page = int(st["bt"][b, p])
            lo, hi = max(c, p * PAGE), min(c + rows, (p + 1) * PAGE)
            at = lo - p * PAGE
            for i in (0, 1):
                x = new[i][b * rows + lo - c:b * rows + hi - c].transpose(0, 1)  # [kv, n, D]
                s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)).clamp_min(1e-10) / 448)))
                if at:
                    s = torch.maximum(s, scales[page, i])
                    values[i][page, :, :at] *= (scales[page, i] / s)[:, None, None]
                values[i][page, :, at:at + hi - lo] = x / s[:, None, None]
                scales[page, i] = s
    inv = torch.argsort(_at(k.device))
    codes = torch.cat([values[0].flatten(1), values[1].transpose(2, 3)[..., inv].flatten(1)], 1)
    out = {"codes": codes, "scales": scales.flatten(1), "q": q}
    return {**out, "summary": None, "summary_scales": None} if st["summary"] is not None else out


def _exact_pages(st, page, h):
    """fp64 keys and values [n * 64, D] of the pages of one head."""
    k, v, scales = _parts(st["cache"], st["kv"], st["dim"])
    s = scales[page][:, :, h].double()
    keys = _values(k[page, h], F64) * s[:, 0, None, None]
    vals = _values(v[page, h], F64)[..., _at(page.device)].transpose(1, 2) * s[:, 1, None, None]
    return keys.flatten(0, 1), vals.flatten(0, 1)


def _exact_rows(st, t, h, keys, vals, seen, out, lse):
    """Rows t of kv head h over keys [L, D]; seen [rows, L]."""
    G = st["heads"] // st["kv"]
    hs = slice(h * G, (h + 1) * G)
    x = (st["q"][t, hs].double().reshape(-1, st["dim"]) @ keys.t()).view(len(t), G, -1) * st["scale"]
    x.masked_fill_(~seen[:, None], -math.inf)
    lse[t, hs] = x.logsumexp(-1)
    full = lse[t, hs] if st["sinks"] is None else torch.logaddexp(lse[t, hs], st["sinks"][hs].double())
    out[t, hs] = (x.sub_(full[..., None]).exp_().view(-1, keys.shape[0]) @ vals).view(len(t), G, -1)


def _exact_attn(st):
    out, lse = (torch.empty(st["q"].shape[:n], dtype=F64, device=st["q"].device) for n in (3, 2))
    rows = st["rows"]
    for b, c in enumerate(st["start"].tolist()):
        page = st["bt"][b, :(c + rows + PAGE - 1) // PAGE].long()
        at = torch.arange(len(page) * PAGE, device=page.device)
        step = max(1, (1 << 24) // len(at))
        for h in range(st["kv"]):
            keys, vals = _exact_pages(st, page, h)
            for a in range(0, rows, step):
                t = torch.arange(b * rows + a, b * rows + min(rows, a + step), device=page.device)
                pos = st["positions"][t, None]
                seen = (at <= pos) & (at > pos - (st["window"] or 1 << 60))
                _exact_rows(st, t, h, keys, vals, seen, out, lse)
    return {"out": out, "lse": lse}


def _exact_block(st):
    """The selection is one of whole numbers and powers of two: exact as it is."""
    T, kv = st["q"].shape[0], st["kv"]
    if T * kv > 6000:
        return None
    ids = _plain_select(st)
    out, lse = (torch.empty(st["q"].shape[:n], dtype=F64, device=st["q"].device) for n in (3, 2))
    for t in range(T):
        pos = int(st["positions"][t])
        for h in range(kv):
            j = ids[t, h][ids[t, h] >= 0].long()
            keys, vals = _exact_pages(st, st["bt"][int(st["req"][t]), j].long(), h)
            at = (j[:, None] * PAGE + torch.arange(PAGE, device=j.device)).flatten()
            _exact_rows(st, torch.tensor([t], device=j.device), h, keys, vals, (at <= pos)[None], out, lse)
    return {"out": out, "lse": lse, "ids": None}
