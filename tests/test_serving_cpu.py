"""The serving operators without a GPU: what the library and the Python checks refuse, and the host-side helpers (rotary
frequencies, tree masks). Refusals come before any CUDA call, so the pointers here are never followed."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

P = 4096  # an aligned address that no refused call touches


def kv_args(**kw):
    a = dict(kq=P, ks=P, vq=P, vs=P, pages=8, page=16, kv_heads=2, head=64, bits=8, table=P, table_cols=4, cu=P, lens=P,
             batch=2, rows=3)
    a.update(kw)
    return a


def append(L, **kw):
    tail = dict(k=P, k_stride=128, v=P, v_stride=128, dtype=0, rope=P, pos=P, rot=64, table_rows=100, layout=0, q=P,
                q_stride=256, q_out=P, q_out_stride=256, heads=4)
    a = kv_args(**{k: v for k, v in kw.items() if k not in tail})
    tail.update({k: v for k, v in kw.items() if k in tail})
    return L.mvb_kv_append(*a.values(), *tail.values(), None)


def read(L, **kw):
    tail = dict(k_out=P, k_stride=128, v_out=P, v_stride=128, dtype=0)
    a = kv_args(**{k: v for k, v in kw.items() if k not in tail})
    tail.update({k: v for k, v in kw.items() if k in tail})
    return L.mvb_kv_read(*a.values(), *tail.values(), None)


def attention(L, **kw):
    tail = dict(heads=4, dtype=0, tree=P, words=1, scale=0.125, max_new=2, max_len=50, out=P, out_stride=256, lse=P, work=None,
                work_bytes=0)
    q = dict(q=P, q_stride=256)
    a = kv_args(**{k: v for k, v in kw.items() if k not in tail and k not in q})
    tail.update({k: v for k, v in kw.items() if k in tail})
    q.update({k: v for k, v in kw.items() if k in q})
    return L.mvb_tree_attention(*q.values(), *a.values(), *tail.values(), None)


CACHE_BAD = [dict(bits=6), dict(bits=16), dict(page=8), dict(page=24), dict(page=2048), dict(pages=0), dict(head=72),
             dict(head=144), dict(head=0), dict(kv_heads=0), dict(table_cols=0), dict(batch=0), dict(rows=-1),
             dict(kq=None), dict(ks=P + 4), dict(vq=P + 8), dict(table=None), dict(cu=P + 2), dict(lens=None)]


@pytest.mark.parametrize("bad", CACHE_BAD + [dict(dtype=3), dict(layout=2), dict(rot=0), dict(rot=72), dict(rot=12),
                                             dict(k=P + 4), dict(v=None), dict(k_stride=130), dict(rope=P + 4),
                                             dict(rope=None), dict(q_out=None), dict(heads=0), dict(q_stride=2)])
def test_append_refuses(mvb, bad):
    assert append(mvb.lib(), **bad) == -1
    assert "mvb_kv_append" in mvb.last_error()


@pytest.mark.parametrize("bad", CACHE_BAD + [dict(dtype=-1), dict(k_out=P + 8), dict(v_out=None), dict(v_stride=130)])
def test_read_refuses(mvb, bad):
    assert read(mvb.lib(), **bad) == -1
    assert "mvb_kv_read" in mvb.last_error()


@pytest.mark.parametrize("bad", CACHE_BAD + [dict(heads=3), dict(heads=0), dict(dtype=5), dict(batch=70000), dict(words=0),
                                             dict(max_new=-1), dict(max_len=-1), dict(scale=math.inf),
                                             dict(scale=math.nan), dict(q=P + 4), dict(out=None), dict(lse=P + 2),
                                             dict(tree=P + 4), dict(work=P + 8), dict(q_stride=258), dict(max_new=1 << 30, rows=1 << 30)])
def test_attention_refuses(mvb, bad):
    assert attention(mvb.lib(), **bad) == -1
    assert "mvb_tree_attention" in mvb.last_error()


def test_nothing_to_do(mvb):
    """No rows is no launch (and no GPU needed)."""
    L = mvb.lib()
    assert append(L, rows=0) == 0 and read(L, rows=0) == 0 and attention(L, rows=0) == 0 and attention(L, max_new=0) == 0
    assert L.mvb_rope(P, P, P, P, 0, 0, 4, 64, 64, 10, 0, 256, 256, None) == 0
    assert L.mvb_logprobs(P, 100, 0, 0, 100, P, 1, P, P, 5, P, P, None) == 0
    assert L.mvb_rope_table(P, P, 32, 0, 0, 1.0, None) == 0


@pytest.mark.parametrize("args", [
    (P, P, P, P, 3, 1, 4, 64, 64, 10, 0, 256, 256), (P, P, P, P, 0, 1, 4, 64, 64, 10, 2, 256, 256),
    (P, P, P, P, 0, 1, 4, 60, 32, 10, 0, 256, 256), (P, P, P, P, 0, 1, 4, 136, 64, 10, 0, 544, 544),
    (P, P, P, P, 0, 1, 4, 64, 72, 10, 0, 256, 256), (P, P, P, P, 0, 1, 4, 64, 12, 10, 0, 256, 256),
    (P, P, P, P, 0, -1, 4, 64, 64, 10, 0, 256, 256), (P + 4, P, P, P, 0, 1, 4, 64, 64, 10, 0, 256, 256),
    (P, None, P, P, 0, 1, 4, 64, 64, 10, 0, 256, 256), (P, P, P + 8, P, 0, 1, 4, 64, 64, 10, 0, 256, 256),
    (P, P, P, P, 0, 1, 4, 64, 64, 10, 0, 257, 256), (P, P, P, P, 0, 1, 4, 64, 64, -1, 0, 256, 256)])
def test_rope_refuses(mvb, args):
    assert mvb.lib().mvb_rope(*args, None) == -1
    assert "mvb_rope" in mvb.last_error()


@pytest.mark.parametrize("args", [(None, P, 32, 4, 0, 1.0), (P, P + 2, 32, 4, 0, 1.0), (P, P, 0, 4, 0, 1.0),
                                  (P, P, 32, -1, 0, 1.0), (P, P, 32, 4, -1, 1.0), (P, P, 32, 1 << 30, 1 << 30, 1.0)])
def test_rope_table_refuses(mvb, args):
    assert mvb.lib().mvb_rope_table(*args, None) == -1


@pytest.mark.parametrize("args", [
    (P, 100, 9, 2, 100, P, 1, P, P, 5, P, P), (P, 100, 0, -1, 100, P, 1, P, P, 5, P, P),
    (P, 100, 0, 2, 0, P, 1, P, P, 0, P, P), (P, 100, 0, 2, 100, P, 1, P, P, 65, P, P),
    (P, 4, 0, 2, 4, P, 1, P, P, 5, P, P), (None, 100, 0, 2, 100, P, 1, P, P, 5, P, P),
    (P + 2, 100, 0, 2, 100, P, 1, P, P, 5, P, P), (P, 100, 0, 2, 100, None, 1, P, P, 5, P, P),
    (P, 100, 0, 2, 100, P, 1, None, P, 5, P, P), (P, 100, 0, 2, 100, P, 1, P, P, 5, None, P),
    (P, 100, 0, 2, 100, P, 1, P, P + 1, 5, P, P), (P, 1 << 22, 0, 2, 1 << 22, P, 1, P, P, 5, P, P)])
def test_logprobs_refuses(mvb, args):
    assert mvb.lib().mvb_logprobs(*args, None) == -1
    assert "mvb_logprobs" in mvb.last_error()


def test_python_checks(mvb):
    """Shapes, types and devices that the C calls cannot see."""
    kq, ks = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2, 16)
    for bad in ((kq.float(), ks, kq, ks), (kq, ks[:3], kq, ks), (kq, ks, kq[:, :1], ks), (kq, ks.double(), kq, ks),
                (kq[..., :32], ks, kq[..., :32], ks)):
        with pytest.raises(ValueError):
            mvb.KvCache(*bad)
    with pytest.raises(ValueError):  # a cache on the CPU
        mvb.KvCache(kq, ks, kq, ks)
    x, pos, table = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(10, 64)
    for a in ((x[0], pos, table), (x, pos.long(), table), (x, pos[:2], table), (x, pos, table.half()),
              (x.double(), pos, table), (x.transpose(1, 2), pos, table), (x, pos, table)):
        with pytest.raises(ValueError):
            mvb.rope(*a)
    with pytest.raises(ValueError):
        mvb.rope(x, pos, table, layout="other")
    for a in ((torch.zeros(3), None), (torch.zeros(3, 4).T, None), (torch.zeros(3, 4), torch.zeros(3, 1)),
              (torch.zeros(3, 4), torch.zeros(2, 1, dtype=torch.int32)), (torch.zeros(3, 4), None)):
        with pytest.raises(ValueError):
            mvb.logprobs(*a)


def test_overlapping_outputs(mvb):
    """Rows that share memory may be read, not written."""
    x, pos, table = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(10, 64)
    for out in (torch.zeros(1, 4, 64).expand(3, 4, 64), torch.zeros(1000).as_strided((3, 4, 64), (128, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            mvb.rope(x, pos, table, out=out)
    with pytest.raises(ValueError, match="overlap"):  # in place
        mvb.rope(x[:1].expand(3, 4, 64), pos, table)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mvb.rope(x[:1].expand(3, 4, 64), pos, table, out=torch.zeros(3, 4, 64))


def test_cache_geometry():
    """The slots of a 4-bit cache: two elements a byte."""
    from conftest import load_pkg
    m = load_pkg()
    with pytest.raises(ValueError):
        m.KvCache.empty(4, 2, 16, 64, bits=5, device="cpu")
    with pytest.raises(ValueError):
        m.KvCache.empty(4, 2, 16, 63, bits=4, device="cpu")


def test_rope_frequencies(mvb):
    f, a = mvb.rope_frequencies(64, 1e6)
    assert f.dtype == np.float64 and a == 1.0
    assert np.allclose(f, [1e6 ** (-2 * i / 64) for i in range(32)], rtol=1e-15)
    g, a = mvb.rope_frequencies(64, 1e6, "linear", factor=4.0)
    assert np.array_equal(g, f / 4) and a == 1.0
    g, a = mvb.rope_frequencies(64, 1e6, "ntk", factor=4.0)
    assert g[0] == 1.0 and a == 1.0 and abs(g[-1] / f[-1] - 0.25) < 1e-12  # the slowest pair stretched by the factor
    g, a = mvb.rope_frequencies(64, 1e6, "yarn", factor=4.0, original=32768)
    assert abs(a - (0.1 * math.log(4) + 1)) < 1e-15
    turns = 32768 * f / (2 * math.pi)
    assert np.array_equal(g[turns > 64], f[turns > 64]) and np.allclose(g[turns < 0.5], f[turns < 0.5] / 4, rtol=1e-15)
    assert np.all(g <= f) and np.all(g >= f / 4) and np.all(np.diff(g) < 0)
    for bad in (dict(rot=63), dict(rot=0), dict(scaling="cubic"), dict(scaling="yarn", factor=2.0), dict(factor=0.5),
                dict(theta=0.0), dict(rot=2, scaling="ntk")):
        with pytest.raises(ValueError):
            mvb.rope_frequencies(**{"rot": 64, "theta": 1e4, **bad})


def test_tree_mask(mvb):
    w = mvb.tree_mask([-1, 0, 0, 2, -1, 3])
    assert w.dtype == torch.int64 and w.tolist() == [[1], [3], [5], [13], [16], [45]]
    chain = mvb.tree_mask(np.stack([np.arange(130) - 1, np.full(130, -1)]))
    assert tuple(chain.shape) == (2, 130, 3)
    bits = np.unpackbits(chain.numpy().view(np.uint8), axis=-1, bitorder="little")[..., :130]
    assert np.array_equal(bits[0], np.tril(np.ones((130, 130)))) and np.array_equal(bits[1], np.eye(130))
    assert tuple(mvb.tree_mask([]).shape) == (0, 1)
    for bad in ([0], [-1, 1], [-2]):
        with pytest.raises(ValueError):
            mvb.tree_mask(bad)


def test_status_names_every_code(mvb):
    assert set(mvb.serving.STATUS) == {0, 1, 2, 3, 4, 5}
    assert mvb.lib().mvb_serve_status.restype is C.c_int


def test_yarn_ramp_behind_the_last_pair(mvb):
    """Where no pair turns fewer than `slow` times, the ramp ends behind the last pair, at the rotary size at most: no pair is
    divided by the whole factor."""
    f, _ = mvb.rope_frequencies(64, 1e4)
    g, _ = mvb.rope_frequencies(64, 1e4, "yarn", factor=4.0, original=131072)
    turns = 131072 * f / (2 * math.pi)
    assert turns.min() > 2.7
    lo = math.floor(32 * math.log(131072 / (32 * 2 * math.pi)) / math.log(1e4))
    hi = math.ceil(32 * math.log(131072 / (2 * math.pi)) / math.log(1e4))
    assert (lo, hi) == (22, 35)
    keep = 1 - np.clip((np.arange(32) - lo) / (hi - lo), 0, 1)
    assert keep[31] > 0.3 and np.allclose(g, f / 4 * (1 - keep) + f * keep, rtol=1e-15)
    # never behind the rotary size
    g, _ = mvb.rope_frequencies(8, 2.0, "yarn", factor=4.0, original=1 << 20)
    f, _ = mvb.rope_frequencies(8, 2.0)
    assert np.array_equal(g, f)
