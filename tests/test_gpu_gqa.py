"""GPU: grouped-query layers over 8-bit pages against the numpy oracle: norm
and rotation, cache write and summaries (bit for bit from given rows),
attention (dense, windowed, selected blocks) and block selection (bit for
bit), and a run of them together, eager and as a replayed graph."""

import numpy as np
import pytest
import torch

from helpers import bf16_tensor, bf16_values, randn_bf16, to_dev
from oracle import gqa
from oracle.fp8 import bf16_round

pytestmark = pytest.mark.gpu

NAN_CODE = 0x7F


def rope_table(n, rope, theta=1e4):
    ang = np.arange(n)[:, None] * theta ** (-np.arange(rope // 2) * 2.0 / rope)
    return np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)


# --------------------------------------------------------------------------- norm and rotation
def check_bf16(got, ref, rows, steps=1.0):
    """Half a bf16 step of the value, and fp32 sums and products (a few 2^-24
    of the row's largest value, 16 of them with the norm's)."""
    tol = steps * 2.0 ** -8 * np.abs(ref) + 16 * 2.0 ** -24 * rows
    err = np.abs(got - ref)
    assert np.all(err <= tol), f"worst {np.max(err - tol)} over, of {np.max(np.abs(ref))}"


@pytest.mark.parametrize("T,H,KV,D,rope,offset,inter,w", [
    (1, 1, 1, 64, 64, 0, False, "f32"), (7, 6, 2, 128, 128, 0, False, "f32"), (7, 6, 2, 128, 64, 64, True, "bf16"),
    (3, 5, 1, 80, 32, 48, False, "f32"), (3, 5, 1, 16, 16, 0, True, "f32"), (5, 4, 4, 192, 64, 128, True, None),
    (130, 24, 8, 256, 64, 192, True, "f32"), (2, 3, 1, 512, 512, 0, False, "bf16"), (9, 4, 2, 128, 0, 0, False, "f32"),
    (5000, 40, 8, 64, 64, 0, False, "f32"), (3, 4, 0, 128, 128, 0, False, "f32"), (3, 0, 4, 96, 32, 8, False, "f32"),
])
def test_qk_norm_rope(dev, T, H, KV, D, rope, offset, inter, w):
    from ernie_kv import ops

    rng = np.random.default_rng(T + D)
    q, k = randn_bf16(rng, (T, H, D)), randn_bf16(rng, (T, KV, D), 3.0)
    ws = [bf16_round((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2)]
    wt = [None if w is None else torch.from_numpy(x).to(dev, torch.float32 if w == "f32" else torch.bfloat16) for x in ws]
    pos = rng.integers(0, 300, T)
    pos[0] = -1 if T > 1 else 299
    pos[-1] = 300 if T > 2 else 5  # outside the table: unrotated
    cs = rope_table(300, rope) if rope else None
    # rows of one projection, q and k as strided views
    qk = torch.empty((T, (H + KV) * D + 8), dtype=torch.bfloat16, device=dev)
    qv, kv = qk[:, :H * D].view(T, H, D), qk[:, H * D:(H + KV) * D].view(T, KV, D)
    qv.copy_(bf16_tensor(q, dev)), kv.copy_(bf16_tensor(k, dev))
    args = (None if cs is None else to_dev(cs, dev), to_dev(pos, dev))
    got = ops.qk_norm_rope(qv, kv, *wt, 1e-5, *args, interleaved=inter, rope_offset=offset)
    odd = torch.empty(T * H * D + 1, dtype=torch.bfloat16, device=dev)[1:].view(T, H, D).copy_(qv)  # 2-byte aligned
    again = ops.qk_norm_rope(odd, kv, *wt, 1e-5, *args, interleaved=inter, rope_offset=offset)
    for g, g2, x, ww in zip(got, again, (q, k), ws):
        assert torch.equal(g, g2) and g.is_contiguous()
        if not x.size:
            continue
        ref = gqa.norm_rope(x, None if w is None else ww, 1e-5, cs, pos, inter, offset)
        check_bf16(bf16_values(g).astype(np.float64), ref, np.abs(ref).max(-1, keepdims=True))


# --------------------------------------------------------------------------- cache write
class Layer:
    """A cache of ragged sequences, on the host and on the device.  Pages are
    permuted; what no token was written to holds NaN codes."""

    def __init__(self, dev, rng, lens, KV, D, extra=0, summary=True, spread=1.0):
        self.dev, self.rng, self.KV, self.D, self.lens = dev, rng, KV, D, list(lens)
        P = max(1, max((n + extra + 63) // 64 for n in lens)) + 1
        B = len(lens)
        self.bt = rng.permutation(B * P + 3)[:B * P].astype(np.int32).reshape(B, P)
        pages = B * P + 3
        self.cache = np.full((pages, gqa.page_bytes(KV, D) + 16), NAN_CODE, np.uint8)
        self.summary = np.full((pages, gqa.summary_bytes(KV, D) + 16), NAN_CODE, np.uint8) if summary else None
        T = sum(lens)
        scale = spread * 2.0 ** rng.integers(-3, 4, (T, 1, 1))
        self.k = bf16_round((rng.standard_normal((T, KV, D)) * np.minimum(scale, 2)).astype(np.float32))
        self.v = bf16_round((rng.standard_normal((T, KV, D)) * scale).astype(np.float32))
        qsl = np.concatenate([[0], np.cumsum(lens)])
        pos = np.concatenate([np.arange(n) for n in lens]) if T else np.zeros(0, np.int64)
        gqa.append(self.k, self.v, pos, qsl, self.bt, self.cache, self.summary)
        self.d_cache = to_dev(self.cache, dev)
        self.d_summary = None if self.summary is None else to_dev(self.summary, dev)
        self.d_bt = to_dev(self.bt, dev)

    def step(self, rows, first=None):
        """(k, v, positions, qsl) of ``rows[b]`` new tokens a sequence."""
        first = self.lens if first is None else first
        T = sum(rows)
        scale = 2.0 ** self.rng.integers(-4, 6, (T, 1, 1))
        k, v = (bf16_round((self.rng.standard_normal((T, self.KV, self.D)) * scale).astype(np.float32)) for _ in "kv")
        pos = np.concatenate([np.arange(n) + f for n, f in zip(rows, first)] + [np.zeros(0)]).astype(np.int64)
        return k, v, pos, np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)

    def same(self):
        assert np.array_equal(self.d_cache.cpu().numpy(), self.cache), "cache bytes differ"
        if self.summary is not None:
            assert np.array_equal(self.d_summary.cpu().numpy(), self.summary), "summary bytes differ"


@pytest.mark.parametrize("KV,D", [(1, 64), (3, 128), (2, 256)])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1, 1, 1], [1, 2, 0, 64, 63, 65], [130, 1, 7, 0, 200, 3]])
@pytest.mark.parametrize("summary", [False, True])
def test_append(dev, KV, D, rows, summary):
    from ernie_kv import ops

    rng = np.random.default_rng(KV * D + rows[0])
    layer = Layer(dev, rng, [0, 1, 5, 63, 64, 130], KV, D, extra=400, summary=summary)
    for again in range(2):
        k, v, pos, qsl = layer.step(rows)
        tk, tv = bf16_tensor(k, dev), torch.empty((len(v), KV, D + 3), dtype=torch.bfloat16, device=dev)[..., :D]
        tv.copy_(bf16_tensor(v, dev))  # rows at odd strides
        ops.gqa_append(tk, tv, to_dev(pos, dev), to_dev(qsl, dev), max(rows), layer.d_bt, layer.d_cache, layer.d_summary)
        gqa.append(k, v, pos, qsl, layer.bt, layer.cache, layer.summary)
        layer.same()
        layer.lens = [a + b for a, b in zip(layer.lens, rows)]
    # rows taken back and written again
    back = [max(0, n - 3) for n in layer.lens]
    k, v, pos, qsl = layer.step([2] * 6, back)
    ops.gqa_append(bf16_tensor(k, dev), bf16_tensor(v, dev), to_dev(pos, dev), to_dev(qsl, dev), 2, layer.d_bt,
                   layer.d_cache, layer.d_summary)
    gqa.append(k, v, pos, qsl, layer.bt, layer.cache, layer.summary)
    layer.same()


def test_append_skips_what_has_no_place(dev):
    """A negative first position, pages outside the cache, positions behind the
    table's row, rows behind the last sequence: nothing is written for them."""
    from ernie_kv import ops

    rng = np.random.default_rng(8)
    layer = Layer(dev, rng, [10, 20, 30, 60], 2, 64, extra=0)
    layer.bt[1, 0], layer.bt[2, 0] = -1, 10_000
    k, v, pos, qsl = layer.step([2, 2, 2, 200])
    pos[:2] = -2, -1
    d_bt = to_dev(layer.bt, dev)
    more = np.zeros((5, 2, 64), np.float32)  # padding rows
    ops.gqa_append(bf16_tensor(np.concatenate([k, more]), dev), bf16_tensor(np.concatenate([v, more]), dev),
                   to_dev(np.concatenate([pos, np.zeros(5, np.int64)]), dev), to_dev(qsl, dev), 200, d_bt,
                   layer.d_cache, layer.d_summary)
    gqa.append(k, v, pos, qsl, layer.bt, layer.cache, layer.summary)
    layer.same()


def test_append_extreme_values(dev):
    """Zeros, the smallest and the largest bf16 values, and an infinity as the largest one."""
    from ernie_kv import ops

    rng = np.random.default_rng(9)
    layer = Layer(dev, rng, [0, 0, 0], 1, 64)
    k = np.zeros((3, 1, 64), np.float32)
    k[1, 0, :3] = [9.2e-41, -1e-38, 3e-39]
    k[2, 0, :3] = [3.3895e38, -3.3895e38, 1.0]
    k = bf16_round(k)
    args = (np.zeros(3, np.int64), np.arange(4, dtype=np.int32))
    ops.gqa_append(bf16_tensor(k, dev), bf16_tensor(k, dev), *(to_dev(x, dev) for x in args), 1, layer.d_bt,
                   layer.d_cache, layer.d_summary)
    gqa.append(k, k, *args, layer.bt, layer.cache, layer.summary)
    layer.same()
    inf = k[2:].copy()
    inf[0, 0, 1] = np.inf
    one = (to_dev(np.zeros(1, np.int64), dev), to_dev(np.arange(2, dtype=np.int32), dev), 1, layer.d_bt[2:])
    ops.gqa_append(bf16_tensor(inf, dev), bf16_tensor(inf, dev), *one, layer.d_cache)
    got = layer.d_cache.cpu().numpy()
    # the largest value is 255 * 2^120, 448 * 2^119 is less: scale 2^120, where it is 256 and the infinity 448
    assert np.array_equal(gqa.k_codes(got, layer.bt[2, 0], 1, 64, 0)[0, :2], [0x78, 0x7E])


@pytest.mark.parametrize("KV,D,H", [(2, 64, 6), (4, 128, 4), (1, 256, 16)])
@pytest.mark.parametrize("inter,w", [(False, True), (True, False)])
def test_prologue_is_norm_then_append(dev, KV, D, H, inter, w):
    from ernie_kv import ops

    rng = np.random.default_rng(D)
    rows = [1, 3, 70, 0]
    layer = Layer(dev, rng, [0, 61, 64, 5], KV, D, extra=80)
    k, v, pos, qsl = layer.step(rows)
    q = randn_bf16(rng, (len(k) + 2, H, D))  # two padding rows
    pad = np.zeros((2, KV, D), np.float32)
    k, v, pos = np.concatenate([k, pad]), np.concatenate([v, pad]), np.concatenate([pos, [3, -1]])
    tq, tk, tv = (bf16_tensor(x, dev) for x in (q, k, v))
    tw = torch.from_numpy((1 + 0.1 * rng.standard_normal((2, D))).astype(np.float32)).to(dev) if w else (None, None)
    cs, tpos, tqsl = to_dev(rope_table(200, 32), dev), to_dev(pos, dev), to_dev(qsl, dev)
    kw = dict(interleaved=inter, rope_offset=D - 32)
    c1, s1, c2, s2 = layer.d_cache.clone(), layer.d_summary.clone(), layer.d_cache.clone(), layer.d_summary.clone()
    wq, wk = ops.qk_norm_rope(tq, tk, tw[0], tw[1], 1e-6, cs, tpos, **kw)
    ops.gqa_append(wk, tv, tpos, tqsl, 70, layer.d_bt, c1, s1)
    gq = ops.gqa_prologue(tq, tk, tv, tw[0], tw[1], 1e-6, cs, tpos, tqsl, 70, layer.d_bt, c2, s2, **kw)
    assert torch.equal(gq, wq) and torch.equal(c1, c2) and torch.equal(s1, s2)
    assert not torch.equal(c1, layer.d_cache)


# --------------------------------------------------------------------------- attention
def check_rows(layer, q, out, lse, scale, rows, sinks, seen):
    """rows: (t, sequence) to check; seen(t): the row's tokens, as a function of
    the kv head.  The weights are rounded to bf16 once (2^-8 of sum |w v|), the
    result once; a score is off by D 2^-24 of sum |q k| (its fp32 sum) and a few
    2^-24 of its size, which moves each weight by as much; a sum of n weights
    in a tree of 16-token steps by (n / 16 + 64) 2^-24."""
    H, D, KV = q.shape[1], q.shape[2], layer.KV
    G = H // KV
    held = {}
    for t, b in rows:
        for h in range(KV):
            if (b, h) not in held:
                pages = layer.bt[b][:-1] if layer.bt.shape[1] > 1 else layer.bt[b]
                held[b, h] = gqa.tokens(layer.cache, pages, KV, D, h)
            keys, vals = held[b, h]
            idx = seen(t, h)
            for g in range(G):
                hq = h * G + g
                o, ref_lse, mass, big = gqa.attend(q[t, hq], keys[idx], vals[idx], scale,
                                                   None if sinks is None else sinks[hq])
                if not len(idx):
                    assert np.all(out[t, hq] == 0) and lse[t, hq] == -np.inf
                    continue
                es = (D + 8) * 2.0 ** -24 * big + (len(idx) / 16 + 64) * 2.0 ** -24
                tol = (2.0 ** -8 + 2 * es) * mass + 2.0 ** -8 * np.abs(o) + 1e-30
                err = np.abs(out[t, hq] - o)
                assert np.all(err <= tol), f"row {t} head {hq}: {np.max(err / tol)} of the tolerance"
                assert abs(lse[t, hq] - ref_lse) <= es + 2.0 ** -22 * max(1.0, abs(ref_lse))


def attn_case(dev, lens, rows, H, KV, D, window=0, with_sinks=False, q_scale=1.0, max_len=None, max_rows=None,
              odd=False, sample=None, seed=0):
    from ernie_kv import ops

    rng = np.random.default_rng(seed + D + H + sum(lens))
    layer = Layer(dev, rng, lens, KV, D, summary=False)
    T = sum(rows)
    q = randn_bf16(rng, (T, H, D), q_scale)
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]).astype(np.int64)
    seq = np.repeat(np.arange(len(lens)), rows)
    qsl = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    sinks = rng.standard_normal(H).astype(np.float32) * 3 if with_sinks else None
    tq = bf16_tensor(q, dev)
    if odd:
        wide = torch.empty((T, H, D + 5), dtype=torch.bfloat16, device=dev)
        wide[..., 1:D + 1] = tq
        tq = wide[..., 1:D + 1]
    big = torch.full((T + 3, H + 1, D + 4), 7.0, dtype=torch.bfloat16, device=dev)
    out = big[:T, :H, :D]
    lse = torch.full((T + 3, H), 7.0, dtype=torch.float32, device=dev)
    ops.gqa_attention(tq, layer.d_cache, KV, layer.d_bt, to_dev(pos, dev), to_dev(qsl, dev), max_rows or max(rows),
                      max_len or max(lens), D ** -0.5, out, lse[:T], sinks=None if sinks is None else to_dev(sinks, dev),
                      window=window)
    torch.cuda.synchronize()
    assert torch.all(big[T:] == 7) and torch.all(big[:, H:] == 7) and torch.all(big[..., D:] == 7)
    assert torch.all(lse[T:] == 7)
    ts = range(T) if sample is None else sorted(set([0, T - 1] + list(rng.integers(0, T, sample))))
    check_rows(layer, q, bf16_values(out.contiguous()).astype(np.float64), lse.cpu().numpy(), D ** -0.5,
               [(t, seq[t]) for t in ts], sinks,
               lambda t, h: np.arange(max(0, pos[t] - window + 1) if window else 0, pos[t] + 1))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,KV", [(1, 1), (6, 2), (8, 1), (16, 1), (20, 1), (40, 1)])
def test_attention_decode(dev, D, H, KV):
    lens = [1, 2, 63, 64, 65, 200, 1000]
    attn_case(dev, lens, [1] * 7, H, KV, D)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, False), (64, True), (100, True), (0, True)])
@pytest.mark.parametrize("rows", [[1, 0, 3, 2, 5], [9, 1, 40, 0, 70]])
def test_attention_rows_window_sinks(dev, D, window, sinks, rows):
    attn_case(dev, [9, 40, 130, 64, 700], rows, 8, 2, D, window, sinks, odd=True)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 3, 5, 66])
def test_attention_window_at_every_offset(dev, D, window):
    """One row at each place of two pages: every token of a page once as the first and once as the last one seen."""
    attn_case(dev, [n + 1 for n in range(130)], [1] * 130, 2, 1, D, window)


@pytest.mark.parametrize("H,KV,D,rows", [(16, 2, 128, [1, 1]), (24, 8, 64, [2, 1]), (4, 1, 256, [3, 2])])
def test_attention_long(dev, H, KV, D, rows):
    """Split over many workgroups, peaked scores (the reference moves late), bounds larger than the lengths."""
    attn_case(dev, [20_000, 3_333], rows, H, KV, D, q_scale=4.0, with_sinks=True, max_len=30_000, max_rows=4)


@pytest.mark.parametrize("H,KV,D,lens,rows,window", [
    (8, 1, 128, [300, 150], [300, 129], 0), (4, 4, 64, [777], [777], 128), (6, 2, 128, [1500, 70], [513, 70], 0),
    (16, 2, 256, [400], [257], 0), (12, 1, 64, [640], [100], 0), (3, 3, 128, [200, 1, 64], [200, 1, 64], 7),
])
def test_attention_prefill(dev, H, KV, D, lens, rows, window):
    attn_case(dev, lens, rows, H, KV, D, window, with_sinks=bool(window), sample=40, odd=D == 64)


def test_attention_large_scores_and_ties(dev):
    """Scores in the thousands: one token takes all the weight, or equal ones share it."""
    attn_case(dev, [130, 700], [1, 2], 4, 2, 128, q_scale=200.0)
    attn_case(dev, [130, 700], [1, 2], 4, 2, 128, q_scale=0.0)


def test_attention_rows_without_tokens(dev):
    """Negative positions (one with a sink, one in a draft next to live rows),
    an unmapped page in the middle, rows of no sequence."""
    from ernie_kv import ops

    rng = np.random.default_rng(3)
    KV, H, D = 2, 8, 128
    layer = Layer(dev, rng, [300, 200, 80], KV, D, summary=False)
    q = randn_bf16(rng, (8, H, D))
    pos = np.array([299, -1, 100, -1, -1, 79, 5, 5], np.int64)
    qsl = np.array([0, 3, 5, 6], np.int32)  # rows 6, 7: no sequence
    seq = [0, 0, 0, 1, 1, 2]
    layer.bt[0, 2] = -1
    for sinks in (None, rng.standard_normal(H).astype(np.float32)):
        out = torch.full((8, H, D), 7.0, dtype=torch.bfloat16, device=dev)
        lse = torch.full((8, H), 7.0, device=dev)
        ops.gqa_attention(bf16_tensor(q, dev), layer.d_cache, KV, to_dev(layer.bt, dev), to_dev(pos, dev),
                          to_dev(qsl, dev), 3, 300, 0.1, out, lse, sinks=None if sinks is None else to_dev(sinks, dev))
        assert torch.all(out[6:] == 7) and torch.all(lse[6:] == 7)

        def seen(t, h):
            at = np.arange(pos[t] + 1)
            return at[(at // 64 != 2)] if seq[t] == 0 else at

        check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), 0.1,
                   [(t, seq[t]) for t in range(6)], sinks, seen)


# --------------------------------------------------------------------------- selected blocks
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,KV,n", [(1, 1, 3), (6, 2, 8), (20, 1, 16), (64, 1, 5), (8, 4, 70)])
def test_block_select_and_attention(dev, D, H, KV, n):
    from ernie_kv import ops

    rng = np.random.default_rng(D + H + n)
    lens = [1, 64, 65, 640, 4500]
    layer = Layer(dev, rng, lens, KV, D)
    req = np.array([0, 1, 2, 3, 4, 4, 4, -1, 9, 3], np.int32)
    pos = np.array([0, 63, 64, 639, 4499, 4490, 2047, 5, 5, -1], np.int64)
    T = len(req)
    q = randn_bf16(rng, (T, H, D), 2.0)
    sinks = rng.standard_normal(H).astype(np.float32)
    tq, tpos, treq = bf16_tensor(q, dev), to_dev(pos, dev), to_dev(req, dev)
    ids = torch.full((T, KV, n + 2), 7, dtype=torch.int32, device=dev)
    ops.gqa_block_select(tq, layer.d_summary, KV, layer.d_bt, tpos, treq, 4500, ids[..., :n], keep_first=1, keep_last=2)
    got = ids.cpu().numpy()
    assert np.all(got[..., n:] == 7) and np.all(got[7:9] == 7)
    live = [t for t in range(T) if 0 <= req[t] < len(lens)]
    for t in live:
        want = gqa.select(q[t], layer.summary, KV, layer.bt[req[t]], int(pos[t]), n, 1, 2)
        assert np.array_equal(got[t, :, :n], want), f"row {t}"
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((T, H), 7.0, device=dev)
    ops.gqa_block_attention(tq, layer.d_cache, KV, layer.d_bt, tpos, treq, ids[..., :n], D ** -0.5, out, lse,
                            sinks=to_dev(sinks, dev))
    assert torch.all(out[7:9] == 7) and torch.all(lse[7:9] == 7)

    def seen(t, h):
        j = got[t, h, :n]
        at = (j[j >= 0][:, None] * 64 + np.arange(64)).ravel()
        return at[at <= pos[t]]

    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), D ** -0.5, [(t, req[t]) for t in live],
               sinks, seen)


def test_block_attention_lists_of_a_user(dev):
    """Lists in any order, with gaps, pages behind the row and a page listed twice (counted twice)."""
    from ernie_kv import ops

    rng = np.random.default_rng(12)
    KV, H, D = 2, 4, 64
    layer = Layer(dev, rng, [1000], KV, D, summary=False)
    q = randn_bf16(rng, (2, H, D))
    pos = np.array([500, 999], np.int64)
    lists = np.array([[[9, 3, -1, 7, 0, 1 << 30], [-1, -1, -1, -1, -1, -1]], [[4, 4, 15, -5, 2, 1], [8, -1, 7, 6, 5, 4]]],
                     np.int32)
    out = torch.empty((2, H, D), dtype=torch.bfloat16, device=dev)
    lse = torch.empty((2, H), device=dev)
    ops.gqa_block_attention(bf16_tensor(q, dev), layer.d_cache, KV, layer.d_bt, to_dev(pos, dev),
                            to_dev(np.zeros(2, np.int32), dev), to_dev(lists, dev), 0.2, out, lse)

    def seen(t, h):
        j = lists[t, h]
        at = (j[(j >= 0) & (j < 16)][:, None] * 64 + np.arange(64)).ravel()
        return at[at <= pos[t]]

    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), 0.2, [(0, 0), (1, 0)], None, seen)


@pytest.mark.parametrize("blocks", [3000, 32768])
def test_block_select_ties_and_long_rows(dev, blocks):
    """Few distinct scores over up to 2^21 tokens: ties go to the lowest page;
    the pages' records are shared, so that the table alone is long."""
    from ernie_kv import ops

    rng = np.random.default_rng(blocks)
    KV, H, D = 1, 4, 64
    summary = np.zeros((40, gqa.summary_bytes(KV, D)), np.uint8)
    for p in range(40):
        codes, s = gqa.summary_parts(summary, p, KV, D)
        codes[:], s[:] = rng.integers(-2, 3, (KV, D)), 2.0 ** rng.integers(-2, 2)
    bt = rng.integers(0, 40, (1, blocks)).astype(np.int32)
    q = randn_bf16(rng, (2, H, D))
    pos = np.array([blocks * 64 - 1, blocks * 32], np.int64)
    for n in (1, 64, 2500):
        ids = torch.empty((2, KV, n), dtype=torch.int32, device=dev)
        keep = (0, 1) if n == 1 else (1, 2)
        ops.gqa_block_select(bf16_tensor(q, dev), to_dev(summary, dev), KV, to_dev(bt, dev), to_dev(pos, dev),
                             to_dev(np.zeros(2, np.int32), dev), blocks * 64, ids, keep_first=keep[0], keep_last=keep[1])
        for t in range(2):
            want = gqa.select(q[t], summary, KV, bt[0], int(pos[t]), n, *keep)
            assert np.array_equal(ids[t].cpu().numpy(), want), (n, t)


# --------------------------------------------------------------------------- together
def run_step(ops, layer, st, ws):
    """A layer's step: prologue, dense attention, block selection and attention."""
    q = ops.gqa_prologue(st["q"], st["k"], st["v"], st["w"], st["w"], 1e-6, st["cs"], st["pos"], st["qsl"], st["most"],
                         layer.d_bt, layer.d_cache, layer.d_summary)
    ops.gqa_attention(q, layer.d_cache, layer.KV, layer.d_bt, st["pos"], st["qsl"], st["most"], st["len"], 0.09, st["o1"],
                      st["l1"], workspace=ws[0])
    ops.gqa_block_select(q, layer.d_summary, layer.KV, layer.d_bt, st["pos"], st["req"], st["len"], st["ids"])
    ops.gqa_block_attention(q, layer.d_cache, layer.KV, layer.d_bt, st["pos"], st["req"], st["ids"], 0.09, st["o2"],
                            st["l2"], workspace=ws[1])


def step_state(dev, rng, layer, rows, H, n):
    k, v, pos, qsl = layer.step(rows)
    T = len(k)
    new = lambda *s: torch.full(s, 7.0, device=dev)  # noqa: E731
    return dict(q=bf16_tensor(randn_bf16(rng, (T, H, layer.D)), dev), k=bf16_tensor(k, dev), v=bf16_tensor(v, dev),
                w=torch.ones(layer.D, device=dev), cs=to_dev(rope_table(6000, layer.D), dev), pos=to_dev(pos, dev),
                qsl=to_dev(qsl, dev), req=to_dev(np.repeat(np.arange(len(rows)), rows).astype(np.int32), dev),
                most=max(rows), len=max(a + b for a, b in zip(layer.lens, rows)), o1=new(T, H, layer.D).bfloat16(),
                l1=new(T, H), o2=new(T, H, layer.D).bfloat16(), l2=new(T, H),
                ids=torch.full((T, layer.KV, n), 7, dtype=torch.int32, device=dev))


def workspaces(ops, st, layer, H, n, dev):
    T, B = st["q"].shape[0], st["qsl"].numel() - 1
    return (ops.gqa_attention_workspace(T, B, st["most"], st["len"], H, layer.KV, layer.D, dev),
            ops.gqa_block_attention_workspace(T, H, layer.KV, layer.D, n, dev))


def test_a_step_of_all_of_them(dev):
    """Every page of a short sequence selected: both attentions see the same tokens."""
    from ernie_kv import ops

    rng = np.random.default_rng(31)
    layer = Layer(dev, rng, [700, 64, 0, 1300], 2, 128, extra=4)
    st = step_state(dev, rng, layer, [1, 3, 2, 1], 12, 32)
    run_step(ops, layer, st, workspaces(ops, st, layer, 12, 32, dev))
    layer.cache, layer.summary = layer.d_cache.cpu().numpy(), layer.d_summary.cpu().numpy()
    q = bf16_values(ops.qk_norm_rope(st["q"], st["k"], st["w"], st["w"], 1e-6, st["cs"], st["pos"])[0])
    pos, req = st["pos"].cpu().numpy(), st["req"].cpu().numpy()
    for o, l in (("o1", "l1"), ("o2", "l2")):
        check_rows(layer, q, bf16_values(st[o]).astype(np.float64), st[l].cpu().numpy(), 0.09, list(enumerate(req)), None,
                   lambda t, h: np.arange(pos[t] + 1))
    ids = st["ids"].cpu().numpy()
    for t in range(len(pos)):
        nb = pos[t] // 64 + 1
        assert np.array_equal(ids[t], np.tile(np.where(np.arange(32) < nb, np.arange(32), -1), (2, 1)))


def test_step_graph_replay_and_streams(dev):
    """The step captured once and replayed on new inputs and on another stream,
    eager work of its own between the replays: every replay gives the eager bytes."""
    from ernie_kv import ops

    rng = np.random.default_rng(32)
    H, n, lens, rows = 16, 6, [2000, 640, 65, 5000], [1, 2, 1, 1]
    layer = Layer(dev, rng, lens, 2, 128, extra=8)
    clean = layer.d_cache.clone(), layer.d_summary.clone()
    st = step_state(dev, rng, layer, rows, H, n)
    ws = workspaces(ops, st, layer, H, n, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_step(ops, layer, st, ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_step(ops, layer, st, ws)
    outs = ("o1", "l1", "o2", "l2", "ids")
    for rep in range(4):
        new = step_state(dev, rng, layer, rows, H, n)
        layer.d_cache.copy_(clean[0]), layer.d_summary.copy_(clean[1])
        run_step(ops, layer, new, workspaces(ops, new, layer, H, n, dev))
        want = {k: new[k].clone() for k in outs}, layer.d_cache.clone(), layer.d_summary.clone()
        layer.d_cache.copy_(clean[0]), layer.d_summary.copy_(clean[1])
        for k in ("q", "k", "v"):
            st[k].copy_(new[k])
        for k in outs:
            st[k].fill_(7)
        torch.cuda.synchronize()
        with torch.cuda.stream(side if rep % 2 else torch.cuda.current_stream()):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(st[k], want[0][k]) for k in outs), f"replay {rep}"
        assert torch.equal(layer.d_cache, want[1]) and torch.equal(layer.d_summary, want[2]), f"replay {rep}"


def test_torch_operators_are_the_wrappers(dev):
    """torch.ops.ernie_kv.*: the wrappers' bytes."""
    import ernie_kv.torch_ops  # noqa: F401
    from ernie_kv import ops

    rng = np.random.default_rng(33)
    H, n = 8, 5
    layer = Layer(dev, rng, [500, 70], 2, 64, extra=8)
    clean = layer.d_cache.clone(), layer.d_summary.clone()
    st = step_state(dev, rng, layer, [2, 1], H, n)
    outs, got = ("o1", "l1", "o2", "l2", "ids"), []
    for o in (ops, torch.ops.ernie_kv):
        layer.d_cache.copy_(clean[0]), layer.d_summary.copy_(clean[1])
        for k in outs:
            st[k].fill_(7)
        q, k = o.qk_norm_rope(st["q"], st["k"], st["w"], st["w"], 1e-6, st["cs"], st["pos"])
        o.gqa_append(k, st["v"], st["pos"], st["qsl"], st["most"], layer.d_bt, layer.d_cache, layer.d_summary)
        first = layer.d_cache.clone()
        layer.d_cache.copy_(clean[0])
        run_step(o, layer, st, workspaces(ops, st, layer, H, n, dev))
        assert torch.equal(first, layer.d_cache)
        got.append([q, k, layer.d_cache.clone(), layer.d_summary.clone()] + [st[x].clone() for x in outs])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and not torch.equal(got[0][2], clean[0])


def test_wrappers_refuse(dev):
    from ernie_kv import _lib, ops

    rng = np.random.default_rng(1)
    layer = Layer(dev, rng, [100], 2, 64)
    q, k = bf16_tensor(randn_bf16(rng, (1, 4, 64)), dev), bf16_tensor(randn_bf16(rng, (1, 2, 64)), dev)
    pos, qsl = to_dev(np.array([99], np.int64), dev), to_dev(np.array([0, 1], np.int32), dev)
    out, req = torch.empty_like(q), qsl[:1]
    attn = (layer.d_cache, 2, layer.d_bt, pos, qsl, 1, 100, 1.0)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        ops.gqa_attention(q[:, :3], layer.d_cache, 2, *attn[2:], out[:, :3])
    with pytest.raises(ValueError, match="out bf16"):
        ops.gqa_attention(q, *attn, out.float())
    with pytest.raises(ValueError, match="positions"):
        ops.gqa_attention(q, *attn[:3], pos.int(), *attn[4:], out)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.gqa_attention(q.half(), *attn, out)
    with pytest.raises(ValueError, match="workspace too small"):
        ops.gqa_attention(q, *attn[:6], 100_000, 1.0, out, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    with pytest.raises(_lib.EkvError, match="page_stride"):
        ops.gqa_append(k, k, pos, qsl, 1, layer.d_bt, layer.d_cache[:, :-32].contiguous())
    with pytest.raises(ValueError, match="like k"):
        ops.gqa_append(k, q, pos, qsl, 1, layer.d_bt, layer.d_cache)
    with pytest.raises(ValueError, match="blocks int32"):
        ops.gqa_block_attention(q, layer.d_cache, 2, layer.d_bt, pos, req, torch.zeros((1, 4, 3), dtype=torch.int32,
                                                                                     device=dev), 1.0, out)
    with pytest.raises(_lib.EkvError, match="keep_first"):
        ops.gqa_block_select(q, layer.d_summary, 2, layer.d_bt, pos, req, 100,
                             torch.zeros((1, 2, 2), dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="unit channel stride"):
        ops.qk_norm_rope(q.transpose(1, 2), k, None, None, 1e-6, None, pos)
