"""GPU: calls of grouped-query attention that several kernels or parts share:
bounds below a call's rows, workspaces that another call has used, single rows
and drafts beside chunks -- against the oracle."""

import numpy as np
import pytest
import torch

from helpers import bf16_tensor, bf16_values, randn_bf16, to_dev
from oracle import gqa
from test_gpu_gqa import Layer, check_rows

pytestmark = pytest.mark.gpu


def batch(rng, lens, rows, H, D):
    q = randn_bf16(rng, (sum(rows), H, D))
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]).astype(np.int64)
    return q, pos, np.repeat(np.arange(len(lens)), rows), np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def call(layer, q, pos, qsl, most, max_len, window=0, sinks=None, workspace=None, bt=None):
    from ernie_kv import ops

    dev, (T, H, D) = layer.dev, q.shape
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((T, H), 7.0, device=dev)
    ops.gqa_attention(bf16_tensor(q, dev), layer.d_cache, layer.KV, layer.d_bt if bt is None else bt, to_dev(pos, dev),
                      to_dev(qsl, dev), most, max_len, D ** -0.5, out, lse, sinks=None if sinks is None else to_dev(sinks, dev),
                      window=window, workspace=workspace)
    return bf16_values(out).astype(np.float64), lse.cpu().numpy()


def size(q, qsl, most, max_len, KV, window=0):
    """Workspace bytes that a call of these bounds needs."""
    from ernie_kv import _lib

    return _lib.load().ekv_gqa_attention_workspace_size(q.shape[0], len(qsl) - 1, most, max_len, q.shape[1], KV, q.shape[2],
                                                        window)


@pytest.mark.parametrize("D,H,KV", [(64, 12, 2), (128, 8, 1), (256, 16, 2)])
@pytest.mark.parametrize("lens,rows,told", [([2000], [9], 1), ([2000], [2], 1), ([2000, 700, 1000], [7, 11, 0], 1),
                                            ([2000, 900], [90, 200], 30), ([2000], [400], 120),
                                            ([2000, 300, 1000, 66], [40, 1, 300, 2], 20)])
def test_rows_past_the_bound(dev, D, H, KV, lens, rows, told):
    """More rows in a sequence than max_query_len says, in a workspace that holds
    other calls' records: rows within the bound are right, each head of those past
    it is right too or left as it was."""
    rng = np.random.default_rng(D + told + sum(rows))
    layer = Layer(dev, rng, lens, KV, D, summary=False)
    q, pos, seq, qsl = batch(rng, lens, rows, H, D)
    need, most = size(q, qsl, told, 9000, KV), max(rows)  # a bound of lengths far above them: parts of few pages
    assert need
    seen = lambda t, h: np.arange(pos[t] + 1)  # noqa: E731
    sure = [t for t in range(len(pos)) if t - qsl[seq[t]] < told]
    some = sorted(set(sure[:6] + sure[-6:]) | set(int(t) for t in rng.integers(0, len(pos), 12)) | {len(pos) - 1})
    held, refs = [gqa.tokens(layer.cache, layer.bt[b][:-1], KV, D, h) for b in range(len(lens)) for h in range(KV)], {}

    def ref(t, hq):
        if (t, hq) not in refs:
            keys, vals = held[seq[t] * KV + hq * KV // H]
            refs[t, hq] = gqa.attend(q[t, hq], keys[:pos[t] + 1], vals[:pos[t] + 1], D ** -0.5)[:2]
        return refs[t, hq]

    for left in (2, 1 << 8 | 3, 1 << 16 | 2, "a call"):
        n = max(need, size(q, qsl, most, 9000, KV)) // 4 + 1
        ws = torch.full((n,), 0 if left == "a call" else left, dtype=torch.int32, device=dev).view(torch.uint8)
        if left == "a call":
            call(layer, q, pos, qsl, most, 9000, workspace=ws)
        out, lse = call(layer, q, pos, qsl, told, 9000, workspace=ws)
        kept = (out == 7).all(2) & (lse == 7)
        assert not kept[sure].any()
        for t, hq in zip(*np.nonzero(kept)):
            if t in some:
                out[t, hq], lse[t, hq] = ref(t, hq)
        check_rows(layer, q, out, lse, D ** -0.5, [(t, seq[t]) for t in some], None, seen)


def shared_call(dev, D, H, KV, lens, rows, window=0, held=None, max_len=1 << 20):
    """A call that both kernels may share, checked against the oracle; (parts,
    kernel) of each row, 0 the kernel of few rows, as the workspace names them.
    held: the sequences with pages of their own, of which the others read some."""
    rng = np.random.default_rng(D + H + sum(rows))
    held = list(range(len(lens))) if held is None else held
    layer = Layer(dev, rng, [lens[b] for b in held], KV, D, summary=False)
    bt = np.full((len(lens), layer.bt.shape[1]), -1, np.int32)
    bt[:] = layer.bt[rng.integers(0, len(held), len(lens))]
    bt[held] = layer.bt
    q, pos, seq, qsl = batch(rng, lens, rows, H, D)
    sinks = rng.standard_normal(H).astype(np.float32)
    n = size(q, qsl, max(rows), max_len, KV, window)
    assert n, "one kernel, no parts"
    some = [t for t in range(len(pos)) if seq[t] in held and rows[seq[t]] < 20]
    some += [int(t) for b in held if rows[b] >= 20 for t in (qsl[b], qsl[b + 1] - 1, *rng.integers(qsl[b], qsl[b + 1], 5))]
    for left in (2, -1):
        ws = torch.full((n // 4 + 1,), left, dtype=torch.int32, device=dev).view(torch.uint8)
        out, lse = call(layer, q, pos, qsl, max(rows), max_len, window, sinks, ws, to_dev(bt, dev))
        check_rows(layer, q, out, lse, D ** -0.5, [(t, held.index(seq[t])) for t in some], sinks,
                   lambda t, h: np.arange(max(0, pos[t] - window + 1) if window else 0, pos[t] + 1))
    y = ws[:8 * len(pos) * H].view(torch.int32).view(len(pos), H, 2)[..., 1].cpu().numpy()
    return y & 255, y >> 16, np.array(rows)[seq]


@pytest.mark.parametrize("D,H,KV", [(64, 8, 1), (128, 8, 1), (128, 12, 4), (256, 8, 1)])
@pytest.mark.parametrize("lens,rows", [([9000, 600], [1, 500]), ([700, 9000, 5000], [500, 1, 500]),
                                       ([3000, 400, 900, 20, 2000], [1, 400, 300, 1, 1])])
@pytest.mark.parametrize("window", [0, 100_000])
def test_a_single_row_beside_a_chunk(dev, D, H, KV, lens, rows, window):
    """However few they are: single rows go to the kernel of few rows, in parts, where they may see many pages."""
    parts, kernel, n = shared_call(dev, D, H, KV, lens, rows, window)
    assert np.all(kernel[n == 1] == 0) and np.all(kernel[n > 1] == 1)
    assert np.all(parts[(n == 1) & (np.repeat(lens, rows) >= 1000)] > 1)


def test_chunks_alone_are_one_launch(dev):
    """No sequence of a call can be short: no second kernel."""
    parts, kernel, n = shared_call(dev, 128, 8, 1, [900, 700], [400, 399])
    assert np.all(kernel == 0)


@pytest.mark.parametrize("seqs", [100, 260])
def test_many_single_rows_beside_a_chunk(dev, seqs):
    """More than 64 sequences, and more than are shared out by their lengths."""
    rng = np.random.default_rng(seqs)
    lens, rows = [int(n) for n in rng.integers(1, 900, seqs)], [1] * seqs
    lens[7], rows[7], lens[50], rows[60] = 9000, 1, 800, 0
    rows[50] = 600
    parts, kernel, n = shared_call(dev, 128, 8, 1, lens, rows, held=sorted({0, 7, 20, 50, 77, seqs - 1}))
    assert np.all(kernel[n == 1] == 0) and np.all(kernel[n > 1] == 1)


@pytest.mark.parametrize("D,H,KV,rows", [
    (128, 8, 1, [3, 300, 2, 4]), (64, 8, 1, [4, 300, 1]), (64, 16, 1, [3, 300, 3]), (128, 16, 1, [3, 300, 4, 2]),
    (256, 8, 1, [3, 300, 3]), (256, 4, 1, [4, 500, 1]), (128, 20, 1, [1, 300, 1]), (256, 20, 1, [1, 300, 1]),
    (64, 40, 1, [1, 300, 1]), (128, 40, 1, [1, 300, 1]), (64, 64, 1, [1, 200, 1]),
])
def test_drafts_and_wide_groups_beside_a_chunk(dev, D, H, KV, rows):
    """What the kernel of few rows holds goes to it: drafts, and many heads a kv head."""
    lens = [9000 if n < 20 else 700 for n in rows]
    parts, kernel, n = shared_call(dev, D, H, KV, lens, rows)
    assert np.all(kernel[n < 20] == 0) and np.all(parts[n < 20] > 1) and np.all(kernel[n >= 20] == 1)


def test_drafts_of_many_sequences_beside_a_chunk(dev):
    rng = np.random.default_rng(4)
    lens, rows = [int(n) for n in rng.integers(4, 900, 90)], [int(n) for n in rng.integers(1, 5, 90)]
    lens[7], lens[50], rows[50] = 9000, 800, 600
    parts, kernel, n = shared_call(dev, 128, 8, 1, lens, rows, held=[0, 7, 20, 50, 89])
    assert np.all(kernel[n < 20] == 0) and np.all(kernel[n >= 20] == 1)


@pytest.mark.parametrize("D,window", [(64, 0), (128, 100_000), (256, 0)])
def test_captured_mixed_call(dev, D, window):
    """Single rows, a draft and chunks in one captured call, both kernels and
    their joins: each replay gives the eager bytes, also on another stream and
    after other calls' use of the workspace."""
    from ernie_kv import ops

    rng = np.random.default_rng(D)
    H, KV, lens, rows = 8, 1, [9000, 500, 2000, 700], [1, 300, 2, 200]
    layer = Layer(dev, rng, lens, KV, D, summary=False)
    q, pos, seq, qsl = batch(rng, lens, rows, H, D)
    tq, tpos, tqsl = bf16_tensor(q, dev), to_dev(pos, dev), to_dev(qsl, dev)
    out, lse = torch.empty_like(tq), torch.empty(tq.shape[:2], device=dev)
    ws = torch.empty(size(q, qsl, 300, 1 << 20, KV, window), dtype=torch.uint8, device=dev)

    def step(workspace):
        ops.gqa_attention(tq, layer.d_cache, KV, layer.d_bt, tpos, tqsl, 300, 1 << 20, D ** -0.5, out, lse, window=window,
                          workspace=workspace)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ws)
    for rep in range(4):
        tq.copy_(bf16_tensor(randn_bf16(rng, q.shape), dev))
        step(None)
        want = out.clone(), lse.clone()
        out.fill_(7), lse.fill_(7), ws.fill_((0, 2, 255, 1)[rep])
        torch.cuda.synchronize()
        with torch.cuda.stream(side if rep % 2 else torch.cuda.current_stream()):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), f"replay {rep}"
