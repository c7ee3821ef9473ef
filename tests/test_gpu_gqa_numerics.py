"""GPU: how exact the grouped-query operators are -- attention weights of 11
bits, values of very different scales side by side -- against the oracle in 64
bits."""

import numpy as np
import pytest
import torch

from helpers import bf16_tensor, bf16_values, randn_bf16, to_dev
from oracle import gqa
from oracle.fp8 import bf16_round
from test_gpu_gqa import Layer

pytestmark = pytest.mark.gpu


def refill(layer, k, v):
    """The layer's tokens again, with other keys and values."""
    layer.cache[:] = 0
    pos = np.concatenate([np.arange(n) for n in layer.lens])
    gqa.append(k, v, pos, np.concatenate([[0], np.cumsum(layer.lens)]), layer.bt, layer.cache)
    layer.d_cache = to_dev(layer.cache, layer.dev)


def check_weights(layer, q, out, lse, scale, rows, sinks, seen):
    """As the oracle has it, but for: each weight rounded to 11 bits (2^-11 of
    it; of one far below, half the smallest fp16 step, which is 2^-30 of the row's
    largest: 2^-25 where that is 2^5 or more), a score's fp32 sum (D + 8 steps of
    2^-24 of sum |q k|) and the sum of n weights ((n / 16 + 64) 2^-24), each of
    which moves the weights by as much, and the result rounded to bf16 once.
    Weights rounded to bf16 would be off by up to 2^-8 of sum |w v|."""
    H, D, KV = q.shape[1], q.shape[2], layer.KV
    G, worst = H // KV, 0.0
    for t, b in rows:
        for h in range(KV):
            keys, vals = gqa.tokens(layer.cache, layer.bt[b], KV, D, h)
            idx = seen(t, h)
            for hq in range(h * G, (h + 1) * G):
                o, ref, mass, big = gqa.attend(q[t, hq], keys[idx], vals[idx], scale, None if sinks is None else sinks[hq])
                es = (D + 8) * 2.0 ** -24 * big + (len(idx) / 16 + 64) * 2.0 ** -24
                tol = (2.0 ** -11 + 2 * es) * mass + 2.0 ** -8 * np.abs(o) + len(idx) * 2.0 ** -30 * np.abs(vals[idx]).max(0)
                err = np.abs(out[t, hq] - o)
                worst = max(worst, np.max(err / (tol + 1e-300)))
                assert np.all(err <= tol + 1e-30), f"row {t} head {hq}: {np.max(err / tol)} of the tolerance"
                assert abs(lse[t, hq] - ref) <= es + 2.0 ** -22 * max(1.0, abs(ref))
    return worst


def attend(layer, q, pos, qsl, rows, max_len, scale, sinks=None, window=0):
    from ernie_kv import ops

    dev = layer.dev
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full(q.shape[:2], 7.0, device=dev)
    ops.gqa_attention(bf16_tensor(q, dev), layer.d_cache, layer.KV, layer.d_bt, to_dev(pos, dev), to_dev(qsl, dev), rows,
                      max_len, scale, out, lse, sinks=None if sinks is None else to_dev(sinks, dev), window=window)
    return bf16_values(out).astype(np.float64), lse.cpu().numpy()


def opposed(rng, n, KV, D):
    """Values that cancel in pairs of tokens, so that a result shows its weights' roundings whole."""
    v = rng.standard_normal((n, KV, D))
    v[1::2] = -v[0:n - n % 2:2]
    return bf16_round(v.astype(np.float32))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,KV,rows", [(4, 2, 1), (8, 1, 1), (16, 1, 2), (2, 1, 150)])
@pytest.mark.parametrize("n", [2, 9, 200, 1500])
def test_weights_keep_eleven_bits(dev, D, H, KV, rows, n):
    rng = np.random.default_rng(D + H + n)
    rows = min(rows, n)
    layer = Layer(dev, rng, [n], KV, D, summary=False)
    refill(layer, randn_bf16(rng, (n, KV, D), 0.5), opposed(rng, n, KV, D))
    q = randn_bf16(rng, (rows, H, D))
    pos = np.arange(n - rows, n, dtype=np.int64)
    out, lse = attend(layer, q, pos, np.array([0, rows], np.int32), rows, n, D ** -0.5)
    some = sorted({0, rows // 2, rows - 1})
    check_weights(layer, q, out, lse, D ** -0.5, [(t, 0) for t in some], None, lambda t, h: np.arange(pos[t] + 1))


@pytest.mark.parametrize("D,H,KV,rows", [(64, 4, 1, 40), (128, 8, 2, 3), (128, 4, 4, 70), (256, 4, 1, 2)])
def test_weights_of_listed_pages(dev, D, H, KV, rows):
    """Lists of one row a workgroup, and those that neighbouring rows join."""
    from ernie_kv import ops

    rng = np.random.default_rng(D + rows)
    n = 700
    layer = Layer(dev, rng, [n], KV, D, summary=False)
    refill(layer, randn_bf16(rng, (n, KV, D), 0.5), opposed(rng, n, KV, D))
    q = randn_bf16(rng, (rows, H, D))
    pos = rng.integers(n - 100, n, rows).astype(np.int64)
    ids = np.sort(np.argsort(rng.random((rows, KV, 9)), axis=2)[..., :4], axis=2).astype(np.int32)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full(q.shape[:2], 7.0, device=dev)
    ops.gqa_block_attention(bf16_tensor(q, dev), layer.d_cache, KV, layer.d_bt, to_dev(pos, dev),
                            torch.zeros(rows, dtype=torch.int32, device=dev), to_dev(ids, dev), D ** -0.5, out, lse)

    def seen(t, h):
        at = (ids[t, h][:, None] * 64 + np.arange(64)).ravel()
        return at[at <= pos[t]]

    check_weights(layer, q, bf16_values(out).astype(np.float64), lse.cpu().numpy(), D ** -0.5,
                  [(t, 0) for t in range(0, rows, 7)], None, seen)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,H", [(1, 8), (2, 24), (140, 2)])
@pytest.mark.parametrize("powers", [(0, 12), (-24, -24), (20, -18), (-12, 30), (90, 90), (-30, 3)])
def test_values_of_unlike_scales(dev, D, rows, H, powers):
    """Pages whose values are powers of two apart (a large one first, last or
    between), pages of zeros, values all tiny or all huge."""
    rng = np.random.default_rng(1000 + D + rows + 7 * powers[0] + powers[1])
    n = 64 * 11 + 5
    layer = Layer(dev, rng, [n], 1, D, summary=False)
    scale = np.repeat(2.0 ** rng.choice(powers, 12), 64)[:n, None, None]
    scale[64 * 3:64 * 5] = 0.0
    refill(layer, randn_bf16(rng, (n, 1, D), 0.5), bf16_round((opposed(rng, n, 1, D) * scale).astype(np.float32)))
    q = randn_bf16(rng, (rows, H, D))
    pos = np.arange(n - rows, n, dtype=np.int64)
    sinks = rng.standard_normal(H).astype(np.float32)
    out, lse = attend(layer, q, pos, np.array([0, rows], np.int32), rows, n, D ** -0.5, sinks)
    check_weights(layer, q, out, lse, D ** -0.5, [(t, 0) for t in sorted({0, rows // 2, rows - 1})], sinks,
                  lambda t, h: np.arange(pos[t] + 1))


@pytest.mark.parametrize("rows,H", [(1, 4), (130, 1)])
def test_many_small_weights(dev, rows, H):
    """One key far above 16,000 others, whose weights are 2^-18 of its own each
    and together 2^-4: none is lost."""
    rng = np.random.default_rng(rows)
    D, n = 64, 16_000
    layer = Layer(dev, rng, [n], 1, D, summary=False)
    k = np.zeros((n, 1, D), np.float32)
    k[100, 0, 0] = 12.5  # 12.5 nats above the others
    v = bf16_round((1 + 0.25 * rng.standard_normal((n, 1, D))).astype(np.float32))
    v[100] = 0
    refill(layer, k, v)
    q = np.zeros((rows, H, D), np.float32)
    q[:, :, 0] = 1
    pos = np.arange(n - rows, n, dtype=np.int64)
    out, lse = attend(layer, q, pos, np.array([0, rows], np.int32), rows, n, 1.0)
    check_weights(layer, q, out, lse, 1.0, [(0, 0), (rows - 1, 0)], None, lambda t, h: np.arange(pos[t] + 1))


@pytest.mark.parametrize("D,rows,H", [(64, 1, 4), (128, 2, 16), (256, 1, 3), (128, 130, 1), (256, 140, 1)])
@pytest.mark.parametrize("first", [1, 2 ** 7, 2 ** 11])
def test_small_values_beside_large_ones(dev, D, rows, H, first):
    """Values a thousandth of their page's largest, which sets the scale but has
    no weight, behind a page of values `first` times larger, which has none
    either: the small ones keep the bits that the cache holds."""
    rng = np.random.default_rng(D + rows + first)
    n = 64 * 5 + 40
    layer = Layer(dev, rng, [n], 1, D, summary=False)
    k = np.zeros((n, 1, D), np.float32)
    k[..., 1:] = randn_bf16(rng, (n, 1, D - 1), 0.25)
    v = opposed(rng, n, 1, D) * 2.0 ** -10
    large = np.concatenate([np.arange(64), np.arange(64, n, 64) + 7])
    k[large, :, 0], v[large] = -60, 1
    v[:64] *= first
    refill(layer, bf16_round(k), bf16_round(v.astype(np.float32)))
    q = randn_bf16(rng, (rows, H, D))
    q[..., 0] = 1
    pos = np.arange(n - rows, n, dtype=np.int64)
    out, lse = attend(layer, q, pos, np.array([0, rows], np.int32), rows, n, 1.0)
    check_weights(layer, q, out, lse, 1.0, [(t, 0) for t in sorted({0, rows // 2, rows - 1})], None,
                  lambda t, h: np.arange(pos[t] + 1))


@pytest.mark.parametrize("D,rows,H", [(64, 1, 4), (128, 3, 16), (256, 1, 2), (64, 130, 2), (256, 130, 1)])
@pytest.mark.parametrize("sign", [-1, 1])
def test_scores_far_from_zero(dev, D, rows, H, sign):
    """Scores of +-2^119, equal in all tokens (one product of powers of two): equal
    weights, so that only the weights' and the result's roundings are left."""
    rng = np.random.default_rng(D)
    n = 64 * 20 + 9
    layer = Layer(dev, rng, [n], 1, D, summary=False)
    k = np.zeros((n, 1, D), np.float32)
    k[..., 3] = sign * 2.0 ** 60
    refill(layer, k, opposed(rng, n, 1, D))
    q = np.zeros((rows, H, D), np.float32)
    q[..., 3] = 2.0 ** 59
    pos = np.arange(n - rows, n, dtype=np.int64)
    out, lse = attend(layer, q, pos, np.array([0, rows], np.int32), rows, 20_000, 1.0)
    _, vals = gqa.tokens(layer.cache, layer.bt[0], 1, D, 0)
    for t in {0, rows // 2, rows - 1}:
        v = vals[:pos[t] + 1]
        tol = (2.0 ** -11 + (len(v) / 16 + 64) * 2.0 ** -24) * np.abs(v).mean(0) + 2.0 ** -8 * np.abs(v.mean(0))
        assert np.all(np.abs(out[t] - v.mean(0)) <= tol)
        assert np.all(np.abs(lse[t] / (sign * 2.0 ** 119) - 1) <= 2.0 ** -21)


@pytest.mark.parametrize("D,H,KV", [(64, 4, 1), (128, 8, 2), (256, 2, 1)])
def test_selection_by_the_largest_keys(dev, D, H, KV):
    """Keys near the largest bf16 value: their scores, past 2^128, are still told apart."""
    from ernie_kv import ops

    rng = np.random.default_rng(D)
    n = 64 * 40
    layer = Layer(dev, rng, [n], KV, D)
    k = rng.standard_normal((n, KV, D)) + 2 * rng.standard_normal((40, KV, D)).repeat(64, 0)
    k *= 2.0 ** rng.integers(119, 124, (40, 1, 1)).repeat(64, 0)
    k = bf16_round(np.clip(k, -3.3e38, 3.3e38).astype(np.float32))
    gqa.append(k, k, np.arange(n), [0, n], layer.bt, layer.cache, layer.summary)
    q = randn_bf16(rng, (5, H, D))
    pos = np.array([n - 1, n - 70, 1000, 700, 64], np.int64)
    ids = torch.empty((5, KV, 7), dtype=torch.int32, device=dev)
    ops.gqa_block_select(bf16_tensor(q, dev), to_dev(layer.summary, dev), KV, layer.d_bt, to_dev(pos, dev),
                         torch.zeros(5, dtype=torch.int32, device=dev), n, ids)
    for t in range(5):
        assert np.array_equal(ids[t].cpu().numpy(), gqa.select(q[t], layer.summary, KV, layer.bt[0], int(pos[t]), 7, 1, 2))
