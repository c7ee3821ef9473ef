"""GPU: edges of the grouped-query operators that a serving program reaches --
many sequences at once, caches past 4 GiB, captured prompts, several streams,
shared and odd strides, rows that the bounds leave out -- against the same
calls in a plain setting, or the oracle."""

import numpy as np
import pytest
import torch

from helpers import bf16_tensor, bf16_values, randn_bf16, to_dev
from oracle import gqa
from test_gpu_gqa import Layer, check_rows, rope_table

pytestmark = pytest.mark.gpu


def attend(ops, layer, q, pos, qsl, max_len, max_rows, window=0, sinks=None, bt=None, workspace=None):
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=q.device)
    lse = torch.full(q.shape[:2], 7.0, device=q.device)
    ops.gqa_attention(q, layer.d_cache, layer.KV, layer.d_bt if bt is None else bt, pos, qsl, max_rows, max_len,
                      q.shape[2] ** -0.5, out, lse, sinks=sinks, window=window, workspace=workspace)
    return out, lse


def batch(dev, rng, lens, rows, H, D):
    T = sum(rows)
    q = randn_bf16(rng, (T, H, D))
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]).astype(np.int64)
    qsl = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    return q, pos, np.repeat(np.arange(len(lens)), rows), bf16_tensor(q, dev), to_dev(pos, dev), to_dev(qsl, dev)


@pytest.mark.parametrize("seqs", [2, 63, 64, 65, 150])
@pytest.mark.parametrize("window", [0, 90])
def test_many_ragged_sequences(dev, seqs, window):
    """Up to 64 sequences share the chip by their lengths, more take equal parts; some are empty, one is long."""
    from ernie_kv import ops

    rng = np.random.default_rng(seqs)
    lens = [int(n) for n in rng.integers(1, 400, seqs)]
    rows = [int(min(n, r)) for n, r in zip(lens, rng.integers(0, 4, seqs))]
    lens[seqs // 2], rows[seqs // 2], rows[0] = 6000, 2, 0
    layer = Layer(dev, rng, lens, 2, 64, summary=False)
    q, pos, seq, tq, tpos, tqsl = batch(dev, rng, lens, rows, 6, 64)
    out, lse = attend(ops, layer, tq, tpos, tqsl, 6000, 3, window)
    some = sorted(set(rng.integers(0, len(pos), 40)) | set(np.nonzero(seq == seqs // 2)[0]))
    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), 64 ** -0.5, [(t, seq[t]) for t in some],
               None, lambda t, h: np.arange(max(0, pos[t] - window + 1) if window else 0, pos[t] + 1))


def test_results_do_not_depend_on_the_company(dev):
    """A sequence's rows alone, or with 20 others of any length: what differs is
    the order of the sums over its parts, within the tolerance of both."""
    from ernie_kv import ops

    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(100, 9000, 21)]
    layer = Layer(dev, rng, lens, 1, 128, summary=False)
    q, pos, seq, tq, tpos, tqsl = batch(dev, rng, lens, [1] * 21, 8, 128)
    out, lse = attend(ops, layer, tq, tpos, tqsl, 9000, 1)
    again = attend(ops, layer, tq, tpos, tqsl, 9000, 1)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])  # no order of atomics in it
    for t in (0, 7, 20):
        one, l1 = attend(ops, layer, tq[t:t + 1], tpos[t:t + 1], to_dev(np.array([0, 1], np.int32), dev), lens[t], 1,
                         bt=layer.d_bt[t:t + 1])
        assert torch.allclose(one[0].float(), out[t].float(), rtol=2.0 ** -7, atol=2.0 ** -7 * float(out[t].abs().max()))
        assert torch.allclose(l1[0], lse[t], rtol=1e-5, atol=1e-5)


def test_caches_past_4_gib(dev):
    """Pages whose byte offsets pass 32 bits: the same bytes and results as in a small cache."""
    from ernie_kv import ops

    rng = np.random.default_rng(6)
    KV, D, H, pages = 8, 128, 16, 34_000
    stride = ops.gqa_page_bytes(KV, D)
    assert pages * stride > 1 << 32
    big = torch.empty((pages, stride), dtype=torch.uint8, device=dev)
    small = torch.zeros((8, stride), dtype=torch.uint8, device=dev)
    far = torch.tensor([[pages - 1, 17, pages - 9, 33_000, 16_400, pages - 2, 5, 32_768]], dtype=torch.int32, device=dev)
    near = torch.arange(8, dtype=torch.int32, device=dev)[None]
    n = 500
    k, v = (bf16_tensor(randn_bf16(rng, (n, KV, D)), dev) for _ in "kv")
    pos, qsl = torch.arange(n, device=dev), to_dev(np.array([0, n], np.int32), dev)
    sums = [torch.zeros((c.shape[0], ops.gqa_summary_bytes(KV, D)), dtype=torch.uint8, device=dev) for c in (big, small)]
    for c, bt, s in ((big, far, sums[0]), (small, near, sums[1])):
        ops.gqa_append(k, v, pos, qsl, n, bt, c, s)
    assert torch.equal(big[far[0].long(), :2 * KV * 64 * D][:7], small[:7, :2 * KV * 64 * D])
    q = bf16_tensor(randn_bf16(rng, (n, H, D)), dev)
    req = torch.zeros(n, dtype=torch.int32, device=dev)
    for rows in (1, 3, n):
        res = []
        for c, bt, s in ((big, far, sums[0]), (small, near, sums[1])):
            out, lse = torch.empty_like(q[:rows]), torch.empty((rows, H), device=dev)
            p, sq = pos[n - rows:].contiguous(), to_dev(np.array([0, rows], np.int32), dev)
            ops.gqa_attention(q[:rows], c, KV, bt, p, sq, rows, n, 0.1, out, lse)
            ids = torch.empty((rows, KV, 4), dtype=torch.int32, device=dev)
            ops.gqa_block_select(q[:rows], s, KV, bt, p, req[:rows], n, ids)
            o2 = torch.empty_like(out)
            ops.gqa_block_attention(q[:rows], c, KV, bt, p, req[:rows], ids, 0.1, o2)
            res.append((out, lse, ids, o2))
        assert all(torch.equal(a, b) for a, b in zip(*res)), rows


@pytest.mark.parametrize("D,H,KV", [(64, 4, 2), (128, 8, 2), (256, 4, 1)])
def test_captured_prompt(dev, D, H, KV):
    """Write and attention of whole prompts (the kernel of many rows) in a graph,
    replayed on other rows, eager work between: the eager bytes each time."""
    from ernie_kv import ops

    rng = np.random.default_rng(D)
    lens = [300, 70]
    layer = Layer(dev, rng, [0, 0], KV, D, extra=300)
    T = sum(lens)
    pos = to_dev(np.concatenate([np.arange(n) for n in lens]).astype(np.int64), dev)
    qsl = to_dev(np.array([0, 300, 370], np.int32), dev)
    w, cs = torch.ones(D, device=dev), to_dev(rope_table(400, D), dev)
    st = {n: torch.empty((T, h, D), dtype=torch.bfloat16, device=dev) for n, h in (("q", H), ("k", KV), ("v", KV))}
    out, lse = torch.empty_like(st["q"]), torch.empty((T, H), device=dev)
    ws = ops.gqa_attention_workspace(T, 2, 300, 300, H, KV, D, dev)

    def step(ws):
        q = ops.gqa_prologue(st["q"], st["k"], st["v"], w, w, 1e-6, cs, pos, qsl, 300, layer.d_bt, layer.d_cache,
                             layer.d_summary)
        ops.gqa_attention(q, layer.d_cache, KV, layer.d_bt, pos, qsl, 300, 300, D ** -0.5, out, lse, workspace=ws)

    def fill():
        for x in st.values():
            x.copy_(bf16_tensor(randn_bf16(rng, tuple(x.shape)), dev))

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ws)
    for rep in range(3):
        fill()
        step(None)
        want = out.clone(), lse.clone(), layer.d_cache.clone(), layer.d_summary.clone()
        out.fill_(7), lse.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out, lse, layer.d_cache, layer.d_summary
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {rep}"


def test_two_streams_at_once(dev):
    """The same call on two streams, each with its own workspace, over and over: no result changes."""
    from ernie_kv import ops

    rng = np.random.default_rng(9)
    lens = [5000, 900, 64]
    layer = Layer(dev, rng, lens, 2, 128, summary=False)
    _, _, _, tq, tpos, tqsl = batch(dev, rng, lens, [1, 2, 1], 16, 128)
    want = attend(ops, layer, tq, tpos, tqsl, 5000, 2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [ops.gqa_attention_workspace(4, 3, 2, 5000, 16, 2, 128, dev) for _ in range(2)]
    got = []
    for _ in range(8):
        for s, w in zip(streams, ws):
            with torch.cuda.stream(s):
                got.append(attend(ops, layer, tq, tpos, tqsl, 5000, 2, workspace=w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


def test_strided_tables_and_rows(dev):
    """Block tables as part of a wider one, query rows every other token of a
    larger buffer, heads before tokens, lse into a strided buffer."""
    from ernie_kv import ops

    rng = np.random.default_rng(10)
    lens = [200, 90]
    layer = Layer(dev, rng, lens, 2, 64)
    q, pos, seq, tq, tpos, tqsl = batch(dev, rng, lens, [2, 1], 4, 64)
    want = attend(ops, layer, tq, tpos, tqsl, 200, 2)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=dev)
    wide[:, 2:2 + layer.bt.shape[1]] = layer.d_bt
    bt = wide[:, 2:2 + layer.bt.shape[1]]
    spread = torch.zeros((6, 4, 64), dtype=torch.bfloat16, device=dev)
    spread[::2] = tq
    swapped = torch.empty((4, 3, 64), dtype=torch.bfloat16, device=dev).copy_(tq.transpose(0, 1)).transpose(0, 1)
    for x in (spread[::2], swapped):
        assert torch.equal(x, tq)
        lse = torch.empty((3, 9), device=dev)[:, :4]
        out = torch.empty((4, 3, 64), dtype=torch.bfloat16, device=dev).transpose(0, 1)
        ops.gqa_attention(x, layer.d_cache, 2, bt, tpos, tqsl, 2, 200, 0.125, out, lse)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        ids = torch.empty((2, 3, 5), dtype=torch.int32, device=dev).transpose(0, 1)
        ids2 = torch.empty((3, 2, 5), dtype=torch.int32, device=dev)
        req = to_dev(seq.astype(np.int32), dev)
        ops.gqa_block_select(x, layer.d_summary, 2, bt, tpos, req, 200, ids)
        ops.gqa_block_select(tq, layer.d_summary, 2, layer.d_bt, tpos, req, 200, ids2)
        assert torch.equal(ids, ids2)
        out2 = torch.empty_like(tq)
        ops.gqa_block_attention(x, layer.d_cache, 2, bt, tpos, req, ids, 0.125, out2)
        for t in range(3):
            assert np.array_equal(ids[t].cpu().numpy(), gqa.select(q[t], layer.summary, 2, layer.bt[seq[t]], int(pos[t]), 5, 1, 2))


def test_what_the_bounds_leave_out(dev):
    """max_query_len below a sequence's rows: the rows past it are not written to
    the cache; a table without columns, a sequence without pages: zeros and -inf."""
    from ernie_kv import ops

    rng = np.random.default_rng(11)
    layer = Layer(dev, rng, [0], 1, 64, extra=200, summary=False)
    before = layer.d_cache.clone()
    k, v, pos, qsl = layer.step([130])
    ops.gqa_append(bf16_tensor(k, dev), bf16_tensor(v, dev), to_dev(pos, dev), to_dev(qsl, dev), 64, layer.d_bt,
                   layer.d_cache)
    changed = (layer.d_cache != before).any(1).nonzero().flatten().cpu().tolist()
    assert set(changed) <= {int(layer.bt[0, 0]), int(layer.bt[0, 1])}
    q = bf16_tensor(randn_bf16(rng, (2, 2, 64)), dev)
    one = to_dev(np.array([0, 2], np.int32), dev)
    for bt in (layer.d_bt[:, :0], torch.full_like(layer.d_bt, -1)):
        out, lse = attend(ops, layer, q, to_dev(np.array([3, 900], np.int64), dev), one, 1000, 2, bt=bt)
        assert torch.all(out == 0) and torch.all(torch.isneginf(lse))
        ids = torch.full((2, 1, 4), 7, dtype=torch.int32, device=dev)
        summary = torch.zeros((layer.d_cache.shape[0], ops.gqa_summary_bytes(1, 64)), dtype=torch.uint8, device=dev)
        req = torch.zeros(2, dtype=torch.int32, device=dev)
        ops.gqa_block_select(q, summary, 1, bt, to_dev(np.array([3, 900], np.int64), dev), req, 1000, ids)
        assert torch.all(ids == -1)
        out.fill_(7)
        ops.gqa_block_attention(q, layer.d_cache, 1, bt, to_dev(np.array([3, 900], np.int64), dev), req, ids, 0.1, out)
        assert torch.all(out == 0)


def test_a_row_that_is_not_finite_stays_alone(dev):
    """NaN or infinite queries: that row and head, no other."""
    from ernie_kv import ops

    rng = np.random.default_rng(13)
    for lens, rows in (([700, 200], [2, 1]), ([300, 200], [150, 90])):
        layer = Layer(dev, rng, lens, 1, 64, summary=False)
        _, _, _, tq, tpos, tqsl = batch(dev, rng, lens, rows, 4, 64)
        want = attend(ops, layer, tq, tpos, tqsl, 700, max(rows))
        tq[1, 2, 5], tq[2, 0, 0] = float("nan"), float("inf")
        out, lse = attend(ops, layer, tq, tpos, tqsl, 700, max(rows))
        bad = torch.zeros(tq.shape[:2], dtype=torch.bool, device=dev)
        bad[1, 2] = bad[2, 0] = True
        assert torch.all(torch.isnan(out[1, 2])) and torch.all(torch.isnan(out[2, 0]))
        assert torch.allclose(out[~bad].float(), want[0][~bad].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
        assert torch.allclose(lse[~bad], want[1][~bad], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("D,blocks", [(64, 90), (128, 65), (256, 41)])
@pytest.mark.parametrize("window,with_sinks", [(0, True), (700, False)])
def test_units_that_fill_the_chip(dev, D, blocks, window, with_sinks):
    """Decode rows of more than 128 (row, kv head) pairs: no parts, each wave
    walks several pages; of ragged sequences, some empty, and of lists."""
    from ernie_kv import ops

    rng = np.random.default_rng(D + window)
    KV, H, seqs = 6, 18, 25
    lens = [int(n) for n in rng.integers(1, 90, seqs)]
    lens[3], lens[11], lens[24] = blocks * 64 - 5, blocks * 40, blocks * 64
    rows = [1] * seqs
    rows[7], rows[20] = 0, 2
    lens[20] += 1
    layer = Layer(dev, rng, lens, KV, D, summary=False)
    q, pos, seq, tq, tpos, tqsl = batch(dev, rng, lens, rows, H, D)
    sinks = (2 * rng.standard_normal(H)).astype(np.float32) if with_sinks else None
    st = None if sinks is None else to_dev(sinks, dev)
    assert ops.gqa_attention_workspace(len(pos), seqs, 2, blocks * 64, H, KV, D, dev, window=window).numel() == 16
    out, lse = attend(ops, layer, tq, tpos, tqsl, blocks * 64, 2, window, st)
    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), D ** -0.5, list(enumerate(seq)), sinks,
               lambda t, h: np.arange(max(0, pos[t] - window + 1) if window else 0, pos[t] + 1))

    # lists of any order with gaps, of the same rows
    ids = np.stack([[rng.permutation(blocks) for _ in range(KV)] for _ in pos]).astype(np.int32)
    ids[rng.random(ids.shape) < 0.1] = -1
    ids[5, 2] = -1
    o2, l2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    assert ops.gqa_block_attention_workspace(len(pos), H, KV, D, blocks, dev).numel() == 16
    ops.gqa_block_attention(tq, layer.d_cache, KV, layer.d_bt, tpos, to_dev(seq.astype(np.int32), dev), to_dev(ids, dev),
                            D ** -0.5, o2, l2, sinks=st)

    def seen(t, h):
        at = (ids[t, h][ids[t, h] >= 0][:, None] * 64 + np.arange(64)).ravel()
        return at[at <= pos[t]]

    check_rows(layer, q, bf16_values(o2).astype(np.float64), l2.cpu().numpy(), D ** -0.5, list(enumerate(seq)), sinks, seen)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 130])
def test_a_cache_of_zeros(dev, D, rows):
    """Pages that nothing was written to, their scales 0 as in a warm-up's
    cache: scores of 0 over the tokens a row sees, and values of 0."""
    from ernie_kv import ops

    KV, H, n = 2, 4, 150
    cache = torch.zeros((3, ops.gqa_page_bytes(KV, D)), dtype=torch.uint8, device=dev)
    bt = torch.arange(3, dtype=torch.int32, device=dev)[None]
    pos = torch.arange(n - rows, n, device=dev)
    q = bf16_tensor(randn_bf16(np.random.default_rng(D), (rows, H, D)), dev)
    for scale in (0.1, 1e-38):
        out = torch.full((rows, H, D), 7.0, dtype=torch.bfloat16, device=dev)
        lse = torch.empty((rows, H), device=dev)
        ops.gqa_attention(q, cache, KV, bt, pos, to_dev(np.array([0, rows], np.int32), dev), rows, n, scale, out, lse)
        assert torch.all(out == 0)
        want = torch.log(pos.double() + 1)[:, None]
        assert torch.all((lse.double() - want).abs() <= 2.0 ** -20 * want + 2.0 ** -20)  # 32-bit sums of up to 150 ones
    ids = torch.arange(3, dtype=torch.int32, device=dev).expand(rows, KV, 3)
    out.fill_(7.0)
    ops.gqa_block_attention(q, cache, KV, bt, pos, torch.zeros(rows, dtype=torch.int32, device=dev), ids.contiguous(),
                            0.1, out, lse)
    assert torch.all(out == 0) and torch.isfinite(lse).all()


@pytest.mark.parametrize("D,seqs", [(64, 40), (128, 70), (256, 130)])
def test_a_prompt_among_many_rows(dev, D, seqs):
    """One long chunk among sequences of single rows, some without any, rows
    behind the last one: the write's bytes and the attention of every sequence,
    and the same of a call of up to the bounds' lengths."""
    from ernie_kv import ops

    rng = np.random.default_rng(seqs)
    KV, H = 1, 8
    rows = [int(r) for r in rng.integers(0, 3, seqs)]
    rows[0], rows[seqs // 2], rows[-1] = 0, 700, 1
    ctx = [int(n) for n in rng.integers(0, 100, seqs)]
    layer = Layer(dev, rng, ctx, KV, D, extra=700)
    k, v, pos, qsl = layer.step(rows)
    T = len(pos)
    pad = [np.concatenate([x, np.ones((5,) + x.shape[1:], x.dtype)]) for x in (k, v)]
    tpos = np.concatenate([pos, np.zeros(5, np.int64)])
    gqa.append(k, v, pos, qsl, layer.bt, layer.cache, layer.summary)
    for bound in (700, 8192):
        c, s = layer.d_cache.clone(), layer.d_summary.clone()
        ops.gqa_append(*(bf16_tensor(x, dev) for x in pad), to_dev(tpos, dev), to_dev(qsl, dev), bound, layer.d_bt, c, s)
        assert np.array_equal(c.cpu().numpy(), layer.cache) and np.array_equal(s.cpu().numpy(), layer.summary)
    layer.d_cache = c
    q = randn_bf16(rng, (T + 5, H, D))
    out, lse = attend(ops, layer, bf16_tensor(q, dev), to_dev(tpos, dev), to_dev(qsl, dev), 800, 700)
    assert torch.all(out[T:] == 7) and torch.all(lse[T:] == 7)
    seq = np.repeat(np.arange(seqs), rows)
    some = sorted(set(np.nonzero(seq != seqs // 2)[0]) | set(T // 2 + rng.integers(-340, 340, 30)) | {0, T - 1})
    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), D ** -0.5, [(t, seq[t]) for t in some],
               None, lambda t, h: np.arange(pos[t] + 1))
    again = attend(ops, layer, bf16_tensor(q, dev), to_dev(tpos, dev), to_dev(qsl, dev), 800, 8192)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("seqs,spike", [(64, 9000), (100, 0), (100, 9000), (256, 0), (256, 9000), (257, 9000)])
def test_sequences_of_like_and_unlike_lengths(dev, seqs, spike):
    """Decode rows whose sequences are nearly equal (one part each), or one of
    them long (shared out by pages), at both ends of what is shared out."""
    from ernie_kv import ops

    rng = np.random.default_rng(seqs + spike)
    lens = [int(n) for n in rng.integers(590, 641, seqs)]
    if spike:
        lens = [n - 400 for n in lens]
        lens[seqs // 3] = spike
    KV, D, H = 8, 64, 8
    few = sorted({0, seqs // 3, seqs - 1} | set(int(b) for b in rng.integers(0, seqs, 9)))
    layer = Layer(dev, rng, [lens[b] for b in few], KV, D, summary=False)
    bt = np.zeros((seqs, layer.bt.shape[1]), np.int32)  # the other sequences read pages of the same cache
    bt[:] = layer.bt[rng.integers(0, len(few), seqs)]
    bt[few] = layer.bt
    q, pos, seq, tq, tpos, tqsl = batch(dev, rng, lens, [1] * seqs, H, D)
    out, lse = attend(ops, layer, tq, tpos, tqsl, max(lens), 1, bt=to_dev(bt, dev))
    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), D ** -0.5,
               [(b, i) for i, b in enumerate(few)], None, lambda t, h: np.arange(pos[t] + 1))


@pytest.mark.parametrize("D,window", [(64, 0), (128, 0), (128, 900), (128, 8700), (256, 0)])
def test_long_single_rows_beside_a_chunk(dev, D, window):
    """Single rows far behind a chunk of the same call, in parts each; the
    workspace holds what an earlier call might have left there."""
    from ernie_kv import ops

    rng = np.random.default_rng(D + window)
    KV, H = 1, 8
    rows = [1, 2, 300, 0, 1, 3, 1, 1, 2, 1]
    lens = [9000, 700, 900, 40, 1, 2000, 66, 3000, 129, 17]
    layer = Layer(dev, rng, lens, KV, D, summary=False)
    q, pos, seq, tq, tpos, tqsl = batch(dev, rng, lens, rows, H, D)
    sinks = rng.standard_normal(H).astype(np.float32)
    n = ops.gqa_attention_workspace(len(pos), len(rows), 300, 9000, H, KV, D, dev, window=window).numel()
    assert n > 16
    some = sorted(set(np.nonzero(seq != 2)[0]) | {3 + int(i) for i in rng.integers(0, 300, 25)} | {3, 302})
    for left in (2, 1 << 16 | 3, -1):
        ws = torch.full((n // 4 + 1,), left, dtype=torch.int32, device=dev).view(torch.uint8)
        out, lse = attend(ops, layer, tq, tpos, tqsl, 9000, 300, window, to_dev(sinks, dev), workspace=ws)
        check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), D ** -0.5, [(t, seq[t]) for t in some],
                   sinks, lambda t, h: np.arange(max(0, pos[t] - window + 1) if window else 0, pos[t] + 1))


def block_rows(dev, layer, q, pos, req, ids, scale, sinks=None, some=None):
    """Block attention of rows whose table is ``layer.bt``, checked against the oracle; (out, lse) as they came."""
    from ernie_kv import ops

    T, H, D = q.shape
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((T, H), 7.0, device=dev)
    bt = layer.d_bt
    ops.gqa_block_attention(bf16_tensor(q, dev), layer.d_cache, layer.KV, bt, to_dev(pos, dev), to_dev(req, dev),
                            to_dev(ids, dev), scale, out, lse, sinks=None if sinks is None else to_dev(sinks, dev))
    known = [(t, req[t]) for t in (range(T) if some is None else some) if 0 <= req[t] < bt.shape[0]]
    off = [t for t in range(T) if not 0 <= req[t] < bt.shape[0]]
    assert torch.all(out[off] == 7) and torch.all(lse[off] == 7)
    pages = layer.bt.shape[1] - 1

    def seen(t, h):
        j = ids[t, h]
        at = (j[(j >= 0) & (j < pages)].astype(np.int64)[:, None] * 64 + np.arange(64)).ravel()
        return at[at <= pos[t]]

    check_rows(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), scale, known, sinks, seen)
    return out, lse


@pytest.mark.parametrize("D,H,KV", [(64, 12, 4), (128, 16, 2), (128, 16, 16), (128, 16, 8), (256, 32, 8), (256, 10, 2)])
@pytest.mark.parametrize("n,T", [(5, 70), (24, 131), (33, 260)])
def test_lists_of_neighbouring_rows(dev, D, H, KV, n, T):
    """A chunk's rows, whose lists are joined: like and unlike lists, gaps, pages
    listed again (they count again), pages behind the row or outside the table,
    rows of no request, and rows of another request between them."""
    rng = np.random.default_rng(D + n + T)
    layer = Layer(dev, rng, [64 * 40 - 7, 900], KV, D, summary=False)
    q = randn_bf16(rng, (T, H, D))
    pos = np.sort(rng.integers(64 * 20, 64 * 40 - 7, T)).astype(np.int64)
    req = np.zeros(T, np.int32)
    ids = np.sort(np.argsort(rng.random((T, KV, 40)), axis=2)[..., :n], axis=2).astype(np.int32)
    ids[T // 3:T // 2] = ids[T // 3]  # neighbours that agree
    ids[rng.random(ids.shape) < 0.1] = -1
    ids[3, 0] = -1
    ids[8:12, :, 1:3] = ids[8:12, :, :1]  # three mentions
    ids[20, 0, 0], ids[21, 0, 0] = 1 << 30, -(1 << 31)
    req[30:33], req[40], req[41], req[T - 2] = 1, -1, 2, 1
    pos[req == 1] = rng.integers(0, 900, int((req == 1).sum()))
    pos[50] = -1
    sinks = rng.standard_normal(H).astype(np.float32)
    some = sorted(set(range(0, 52, 3)) | {8, 9, 10, 11, 20, 29, 30, 31, 32, 40, 41, 50, T // 3, T // 2 - 1, T - 3, T - 2, T - 1})
    first = block_rows(dev, layer, q, pos, req, ids, D ** -0.5, sinks, some)
    again = block_rows(dev, layer, q, pos, req, ids, D ** -0.5, sinks, some[:1])
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_joined_lists_over_long_tables(dev):
    """Pages past the first 2,048 of a request, which are joined range by range."""
    rng = np.random.default_rng(77)
    KV, H, D, T, n, pages = 8, 32, 128, 70, 20, 5000
    layer = Layer(dev, rng, [64 * 30], KV, D, summary=False)
    full = layer.bt[0, :30]
    layer.bt = full[rng.integers(0, 30, (1, pages + 1))].astype(np.int32)
    layer.d_bt = to_dev(layer.bt, dev)
    q = randn_bf16(rng, (T, H, D))
    pos = (64 * pages - 1 - 50 * np.arange(T)[::-1]).astype(np.int64)
    ids = np.sort(rng.choice(pages, (T, KV, n)), axis=2).astype(np.int32)
    ids[:, :, :3] = [2047, 2048, 4095]
    block_rows(dev, layer, q, pos, np.zeros(T, np.int32), ids, 0.1, some=[0, 17, 42, 69])
