"""CPU: the grouped-query oracle against closed forms and torch's fp8 casts,
and the host's refusals (the C entry points' argument checks run before any
device work, so null or made-up pointers never reach a kernel)."""

import numpy as np
import pytest
import torch

from oracle import gqa
from oracle.fp8 import bf16_round, decode_e4m3


def test_v_order_is_a_permutation_of_the_page():
    at = gqa.v_at(np.arange(64))
    assert sorted(at) == list(range(64))
    # the 16 bytes of group g are tokens 16 t + 4 g + i
    for g in range(4):
        assert sorted(np.where(at // 16 == g)[0]) == sorted(16 * t + 4 * g + i for t in range(4) for i in range(4))


@pytest.mark.parametrize("amax,top,want", [(448.0, 448.0, 1.0), (449.0, 448.0, 2.0), (1.0, 448.0, 2.0 ** -8),
                                           (0.0, 448.0, 2.0 ** -42), (127.0, 127.0, 1.0), (3.5, 127.0, 2.0 ** -5)])
def test_scale_rule(amax, top, want):
    assert gqa.pow2_scale(np.float32(amax), top) == np.float32(want)


def test_append_matches_torch_casts_and_grows_once():
    rng = np.random.default_rng(5)
    KV, D = 2, 64
    cache = np.zeros((3, gqa.page_bytes(KV, D)), np.uint8)
    bt = np.array([[2, 0]], np.int32)
    a = bf16_round(rng.standard_normal((5, KV, D)).astype(np.float32))
    b = bf16_round((40 * rng.standard_normal((1, KV, D))).astype(np.float32))
    gqa.append(a, a, np.arange(5) + 60, [0, 5], bt, cache)  # rows 60..63 of page 2, row 0 of page 0
    s0 = gqa.scales(cache, 2, KV, D).copy()
    want = torch.from_numpy(a[:4, 1] / s0[0, 1]).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(gqa.k_codes(cache, 2, KV, D, 1)[60:], want)
    assert np.array_equal(gqa.v_codes(cache, 2, KV, D, 1).T[gqa.v_at(np.arange(60, 64))], want)
    before = decode_e4m3(gqa.k_codes(cache, 0, KV, D, 0)[0]).copy()
    old = gqa.scales(cache, 0, KV, D)[0, 0]
    gqa.append(b, b, np.array([65]), [0, 1], bt, cache)
    new = gqa.scales(cache, 0, KV, D)[0, 0]
    assert new > old
    want = torch.from_numpy(before * (old / new)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(gqa.k_codes(cache, 0, KV, D, 0)[0], want)
    # a page begun again forgets its scale
    gqa.append(a[:1], a[:1], np.array([64]), [0, 1], bt, cache)
    assert np.array_equal(gqa.scales(cache, 0, KV, D)[0], gqa.pow2_scale(np.abs(a[0]).max(-1), 448.0))


def test_summary_is_the_mean_of_the_stored_keys():
    rng = np.random.default_rng(6)
    KV, D = 1, 64
    cache = np.zeros((1, gqa.page_bytes(KV, D)), np.uint8)
    summary = np.zeros((1, gqa.summary_bytes(KV, D)), np.uint8)
    x = bf16_round(rng.standard_normal((23, KV, D)).astype(np.float32))
    gqa.append(x, x, np.arange(23), [0, 23], np.zeros((1, 1), np.int32), cache, summary)
    keys, _ = gqa.tokens(cache, [0], KV, D, 0)
    codes, s = gqa.summary_parts(summary, 0, KV, D)
    mean = keys[:23].mean(0)
    assert np.abs(codes[0] * s[0] - mean).max() <= s[0] / 2 * (1 + 1e-6)
    assert np.abs(codes).max() > 63


def test_norm_rope_keeps_the_norm_and_turns_pairs():
    rng = np.random.default_rng(7)
    x = rng.standard_normal((3, 2, 64))
    ang = rng.uniform(0, 6, (10, 16))
    cs = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    for inter in (False, True):
        y = gqa.norm_rope(x, np.ones(64), 0.0, cs, [3, 9, 10], inter, 32)
        assert np.allclose((y ** 2).mean(-1), 1.0)
        z = gqa.norm_rope(x, np.ones(64), 0.0, None, [0, 0, 0])
        assert np.array_equal(y[2], z[2]) and np.array_equal(y[:2, :, :32], z[:2, :, :32])
        pair = [32, 33] if inter else [32, 48]
        u = z[0, 0, pair[0]] + 1j * z[0, 0, pair[1]]
        w = u * np.exp(1j * ang[3, 0])
        assert np.allclose(y[0, 0, pair], [w.real, w.imag], atol=1e-6)


def test_select_takes_the_lowest_index_on_ties_and_the_forced_pages():
    KV, D = 1, 64
    summary = np.zeros((8, gqa.summary_bytes(KV, D)), np.uint8)
    for p in range(8):
        codes, s = gqa.summary_parts(summary, p, KV, D)
        codes[:], s[:] = [0, 5, 5, 9, 5, 5, 0, 0][p], 1.0
    q = np.ones((2, D), np.float32)
    got = gqa.select(q, summary, KV, np.arange(8), 7 * 64 + 3, 6, 1, 2)
    assert got.tolist() == [[0, 1, 2, 3, 6, 7]]
    assert gqa.select(q, summary, KV, np.array([0, -1, 2, 99]), 64 * 4, 6, 1, 2).tolist() == [[0, 2, -1, -1, -1, -1]]
    assert gqa.select(q, summary, KV, np.arange(8), -1, 2, 1, 1).tolist() == [[-1, -1]]


# --------------------------------------------------------------------------- refusals, on the host
@pytest.fixture(scope="module")
def lib():
    from ernie_kv import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libernie_kv.so not built (run __graft_entry__.build())")
    return _lib.load()


X = 1 << 20  # a 16-byte aligned address that no check dereferences


def _append(**o):
    a = dict(k=X, kt=1024, kh=128, v=X, vt=1024, vh=128, T=4, KV=8, D=128, pos=X, qsl=X, B=2, mq=2, bt=X, bts=4, btw=4,
             cache=X, ps=8 * (128 * 128 + 8), np=9, sm=None, ss=0, st=None)
    a.update(o)
    return list(a.values())


def _attn(**o):
    a = dict(q=X, qt=1024, qh=128, T=4, H=64, KV=8, D=128, cache=X, ps=8 * (128 * 128 + 8), np=9, bt=X, bts=4, btw=4,
             pos=X, qsl=X, B=2, mq=2, ml=100, win=0, sinks=None, scale=0.1, out=X, ot=8192, oh=128, lse=None, ls=0,
             ws=None, wb=0, st=None)
    a.update(o)
    return list(a.values())


def _select(**o):
    a = dict(q=X, qt=1024, qh=128, T=4, H=64, KV=8, D=128, sm=X, ss=8 * 132, np=9, bt=X, bts=4, btw=4, pos=X, req=X,
             B=2, ml=100, kf=1, kl=2, ids=X, it=64, ih=8, n=8, st=None)
    a.update(o)
    return list(a.values())


def _blocks(**o):
    a = dict(q=X, qt=1024, qh=128, T=4, H=64, KV=8, D=128, cache=X, ps=8 * (128 * 128 + 8), np=9, bt=X, bts=4, btw=4,
             pos=X, req=X, B=2, ids=X, it=64, ih=8, n=8, sinks=None, scale=0.1, out=X, ot=8192, oh=128, lse=None, ls=0,
             ws=None, wb=0, st=None)
    a.update(o)
    return list(a.values())


def _norm(**o):
    a = dict(q=X, qt=1024, qh=128, H=8, k=X, kt=1024, kh=128, KV=8, T=4, D=128, qw=X, kw=X, wb=0, eps=1e-6, cs=X, rows=10,
             rope=64, off=0, il=0, pos=X, qo=X, ko=X, st=None)
    a.update(o)
    return list(a.values())


@pytest.mark.parametrize("name,args,status,message", [
    ("ekv_qk_norm_rope", _norm(D=24), 1, "dim must be"),
    ("ekv_qk_norm_rope", _norm(D=528), 1, "dim must be"),
    ("ekv_qk_norm_rope", _norm(rope=24), 1, "rope must be"),
    ("ekv_qk_norm_rope", _norm(off=72), 1, "rope must be"),
    ("ekv_qk_norm_rope", _norm(off=4), 1, "rope must be"),
    ("ekv_qk_norm_rope", _norm(cs=None), 1, "cos_sin"),
    ("ekv_qk_norm_rope", _norm(cs=X + 4), 1, "cos_sin"),
    ("ekv_qk_norm_rope", _norm(pos=None), 1, "null"),
    ("ekv_qk_norm_rope", _norm(qo=X + 8), 1, "aligned"),
    ("ekv_gqa_append", _append(D=96), 1, "dim must be"),
    ("ekv_gqa_append", _append(KV=0), 1, "negative"),
    ("ekv_gqa_append", _append(ps=8 * (128 * 128 + 8) - 16), 1, "page_stride"),
    ("ekv_gqa_append", _append(ps=8 * (128 * 128 + 8) + 8), 1, "page_stride"),
    ("ekv_gqa_append", _append(sm=X, ss=8 * 132 - 16), 1, "summary_stride"),
    ("ekv_gqa_append", _append(qsl=None), 1, "null"),
    ("ekv_gqa_attention", _attn(H=60), 1, "multiple of kv_heads"),
    ("ekv_gqa_attention", _attn(D=512), 1, "dim must be"),
    ("ekv_gqa_attention", _attn(win=-1), 1, "negative"),
    ("ekv_gqa_attention", _attn(scale=0.0), 1, "scale"),
    ("ekv_gqa_block_attention", _blocks(scale=-1.0), 1, "scale"),
    ("ekv_gqa_attention", _attn(scale=float("inf")), 1, "scale"),
    ("ekv_gqa_attention", _attn(out=X + 2), 1, "8-byte"),
    ("ekv_gqa_attention", _attn(oh=130), 1, "8-byte"),
    ("ekv_gqa_attention", _attn(ml=100_000), 3, "workspace"),
    ("ekv_gqa_attention", _attn(ml=100_000, ws=X + 4, wb=1 << 40), 1, "16-byte"),
    ("ekv_gqa_block_select", _select(H=8 * 65), 1, "64 query heads"),
    ("ekv_gqa_block_select", _select(kf=7), 1, "keep_first"),
    ("ekv_gqa_block_select", _select(ml=(1 << 21) + 1), 1, "max_len"),
    ("ekv_gqa_block_select", _select(ss=1040), 1, "summary_stride"),
    ("ekv_gqa_block_attention", _blocks(req=None), 1, "null"),
    ("ekv_gqa_block_attention", _blocks(n=-1), 1, "negative"),
    ("ekv_gqa_block_attention", _blocks(n=64), 3, "workspace"),
])
def test_refusals(lib, name, args, status, message):
    assert getattr(lib, name)(*args) == status
    assert message in lib.ekv_last_error().decode()


@pytest.mark.parametrize("name,args", [
    ("ekv_qk_norm_rope", _norm(T=(1 << 31) - 1)), ("ekv_gqa_append", _append(T=1 << 26, B=1 << 20, mq=64)),
    ("ekv_gqa_append", _append(T=1 << 26, B=1 << 20, mq=8192)), ("ekv_gqa_attention", _attn(T=1 << 24, B=1 << 24, mq=1)),
    ("ekv_gqa_attention", _attn(T=(1 << 31) - 1, B=2, mq=(1 << 31) - 1)), ("ekv_gqa_block_select", _select(T=1 << 20)),
    ("ekv_gqa_block_attention", _blocks(T=1 << 24)),
])
def test_grids_past_the_limit(lib, name, args):
    """A grid holds fewer than 2^32 lanes: larger calls are refused, not cut off."""
    assert getattr(lib, name)(*args) == 1
    assert "too many rows" in lib.ekv_last_error().decode()


@pytest.mark.parametrize("name,args", [
    ("ekv_qk_norm_rope", _norm(T=0)), ("ekv_gqa_append", _append(T=0)), ("ekv_gqa_append", _append(B=0)),
    ("ekv_gqa_append", _append(mq=0)), ("ekv_gqa_attention", _attn(T=0)), ("ekv_gqa_attention", _attn(B=0)),
    ("ekv_gqa_attention", _attn(mq=0)), ("ekv_gqa_block_select", _select(n=0, kf=0, kl=0)),
    ("ekv_gqa_block_select", _select(T=0)), ("ekv_gqa_block_attention", _blocks(T=0)),
])
def test_empty_calls_launch_nothing(lib, name, args):
    assert getattr(lib, name)(*args) == 0


def test_sizes(lib):
    for kv, d in ((1, 64), (3, 128), (8, 256)):
        assert lib.ekv_gqa_page_bytes(kv, d) == gqa.page_bytes(kv, d)
        assert lib.ekv_gqa_summary_bytes(kv, d) == gqa.summary_bytes(kv, d)
    assert lib.ekv_gqa_page_bytes(8, 96) == 0 and lib.ekv_gqa_summary_bytes(0, 128) == 0
    ws = lib.ekv_gqa_attention_workspace_size
    assert ws(1, 1, 1, 64, 8, 8, 128, 0) == 0  # one page: no partial results
    assert ws(1, 1, 1, 131072, 8, 8, 128, 0) > 0
    assert ws(0, 1, 1, 131072, 8, 8, 128, 0) == 0 and ws(1, 1, 1, 131072, 8, 8, 96, 0) == 0


def test_wrappers_refuse_cpu_tensors():
    from ernie_kv import ops

    z = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i, p = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    cache = torch.zeros(1, gqa.page_bytes(1, 64), dtype=torch.uint8)
    with pytest.raises(ValueError, match="device tensors"):
        ops.gqa_append(z, z, p, i, 1, i[None], cache)
    with pytest.raises(ValueError, match="device tensors"):
        ops.gqa_attention(z, cache, 1, i[None], p, i, 1, 64, 1.0, torch.empty_like(z))
    with pytest.raises(ValueError, match="device tensors"):
        ops.qk_norm_rope(z, z, None, None, 1e-6, None, p)


def test_torch_ops_registered_and_traced():
    """The operators name what they write, and their fakes give what they return, without a launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import ernie_kv.torch_ops as T

    writes = {"qk_norm_rope": set(), "gqa_append": {"cache", "summary"}, "gqa_prologue": {"cache", "summary"},
              "gqa_attention": {"out", "lse", "workspace"}, "gqa_block_select": {"blocks"},
              "gqa_block_attention": {"out", "lse", "workspace"}}
    assert set(T.GQA_OPS) == set(writes)
    for name, expect in writes.items():
        schema = getattr(torch.ops.ernie_kv, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == expect, name
    with FakeTensorMode():
        q, k = torch.empty((3, 8, 64), dtype=torch.bfloat16), torch.empty((3, 2, 64), dtype=torch.bfloat16)
        pos, i = torch.empty(3, dtype=torch.int64), torch.empty(4, dtype=torch.int32)
        a, b = torch.ops.ernie_kv.qk_norm_rope(q[:, ::2], k, None, None, 1e-6, None, pos)
        assert a.shape == (3, 4, 64) and a.is_contiguous() and b.shape == k.shape
        cache = torch.empty((4, 2 * 128 * 64 + 16), dtype=torch.uint8)
        y = torch.ops.ernie_kv.gqa_prologue(q, k, k, None, None, 1e-6, None, pos, i, 1, i[None], cache, None)
        assert y.shape == q.shape and y.dtype == q.dtype
        assert torch.ops.ernie_kv.gqa_attention(q, cache, 2, i[None], pos, i, 1, 64, 0.1, y, None, None) is None
