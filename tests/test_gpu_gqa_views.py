"""GPU: grouped-query caches and summaries that are part of a wider buffer."""

import numpy as np
import pytest
import torch

from helpers import bf16_tensor, randn_bf16, to_dev
from test_gpu_gqa import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("KV,D", [(1, 64), (2, 128), (3, 256)])
def test_views_narrower_than_a_page_are_refused(dev, KV, D):
    """Rows of a wider buffer that do not hold a page, or a record: refused,
    though the next row is far enough away; what lies beside stays."""
    from ernie_kv import _lib, ops

    rng = np.random.default_rng(D)
    page, rec = KV * (128 * D + 8), KV * (D + 4)
    pages, sums = (torch.zeros((3, 2 * n + 64 - 2 * n % 16), dtype=torch.uint8, device=dev) for n in (page, rec))
    k, q = bf16_tensor(randn_bf16(rng, (2, KV, D)), dev), bf16_tensor(randn_bf16(rng, (2, 2 * KV, D)), dev)
    pos, qsl = to_dev(np.arange(2), dev), to_dev(np.array([0, 2], np.int32), dev)
    bt, req, out = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), q.clone()
    ids = torch.zeros((2, KV, 3), dtype=torch.int32, device=dev)
    cache, summary = pages[:, :page], sums[:, :rec]
    with pytest.raises(_lib.EkvError, match="page_stride"):
        ops.gqa_append(k, k, pos, qsl, 2, bt, cache[:, :-1])
    with pytest.raises(_lib.EkvError, match="summary_stride"):
        ops.gqa_append(k, k, pos, qsl, 2, bt, cache, summary[:, :-1])
    with pytest.raises(_lib.EkvError, match="page_stride"):
        ops.gqa_prologue(q, k, k, None, None, 1e-6, None, pos, qsl, 2, bt, cache[:, :-16])
    with pytest.raises(_lib.EkvError, match="page_stride"):
        ops.gqa_attention(q, cache[:, :-8], KV, bt, pos, qsl, 2, 2, 1.0, out)
    with pytest.raises(_lib.EkvError, match="page_stride"):
        ops.gqa_block_attention(q, cache[:, :-8], KV, bt, pos, req, ids, 1.0, out)
    with pytest.raises(_lib.EkvError, match="summary_stride"):
        ops.gqa_block_select(q, summary[:, :-4], KV, bt, pos, req, 2, ids)
    assert not pages.any() and not sums.any() and torch.equal(out, q) and not ids.any()


@pytest.mark.parametrize("KV,D", [(1, 64), (3, 128)])
def test_layers_side_by_side_in_one_buffer(dev, KV, D):
    """Pages of two layers in each row of one buffer: the bytes and results of a
    cache of its own, and the other layer's bytes as they were."""
    from ernie_kv import ops

    rng = np.random.default_rng(KV)
    layer = Layer(dev, rng, [100, 64], KV, D, extra=80)
    n, m = layer.d_cache.shape[1], layer.d_summary.shape[1]
    both, sums = (torch.cat([x, torch.full_like(x, 9)], 1) for x in (layer.d_cache, layer.d_summary))
    k, v, pos, qsl = layer.step([3, 70])
    q = bf16_tensor(randn_bf16(rng, (73, 2 * KV, D)), dev)
    tk, tv, tpos, tqsl = bf16_tensor(k, dev), bf16_tensor(v, dev), to_dev(pos, dev), to_dev(qsl, dev)
    req = to_dev(np.repeat(np.arange(2), [3, 70]).astype(np.int32), dev)
    res = []
    for cache, summary in ((layer.d_cache, layer.d_summary), (both[:, :n], sums[:, :m])):
        ops.gqa_append(tk, tv, tpos, tqsl, 70, layer.d_bt, cache, summary)
        outs = [torch.empty_like(q) for _ in range(2)]
        ids = torch.empty((73, KV, 2), dtype=torch.int32, device=dev)
        ops.gqa_attention(q, cache, KV, layer.d_bt, tpos, tqsl, 70, 134, 0.1, outs[0])
        ops.gqa_block_select(q, summary, KV, layer.d_bt, tpos, req, 134, ids, keep_last=1)
        ops.gqa_block_attention(q, cache, KV, layer.d_bt, tpos, req, ids, 0.1, outs[1])
        res.append((cache, summary, ids, *outs))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert torch.all(both[:, n:] == 9) and torch.all(sums[:, m:] == 9)
