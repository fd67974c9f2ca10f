"""Calls of the serving operators at their borders: the decoder's log probabilities without a step, many rows at once, status
words, queries of the device that fail."""
import numpy as np
import pytest

import serving_reference as ref
from serving_reference import Case, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "a CUDA device is required"
    t.cuda.set_device(0)
    return t


def test_decoder_logprobs_need_a_step(torch, mvb, tmp_path):
    """Refused where the logits are of no step, of another head's, or of the step before a prompt."""
    path = str(tmp_path / "tiny.qwb")
    mvb.qwb.write_synthetic_qwb(path, mvb.qwb.QWEN_TINY, seed=11)
    dec = mvb.QwenDecoder(path, ctx=64)

    def refused():
        with pytest.raises(mvb.MatvecError, match="no step"):
            dec.logprobs([0], top=1)

    def fine(logits=None):
        logp, ent, top, top_logp = dec.logprobs([0], top=1)
        assert np.isfinite(logp[0]) and np.isfinite(ent) and logp[0] <= top_logp[0] <= 0
        assert logits is None or top[0] == int(np.argmax(logits))

    try:
        refused()
        fine(dec.forward(5, 0)[1])
        dec.full_head(False)  # the head in use already
        fine()
        dec.full_head(True)
        refused()
        fine(dec.forward(5, 0)[1])
        dec.full_head(False)
        refused()
        for feed in (dec.prefill, dec.prefill_tokenwise):
            fine(dec.forward(5, 0)[1])
            feed([3, 4, 5])
            refused()
            dec.decode(0)
            refused()
            dec.decode(2)
            fine()
        dec.prefill([3])
        refused()
        dec.trace(3, 0)
        fine()
    finally:
        dec.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompts_of_many_rows(torch, mvb, dtype):
    """Prompts whose rows together pass 32,768, and a max_new above that: 32 heads over 8 kv heads fit one call up to 262,140."""
    from test_attention_accuracy_gpu import bound
    new = [4200, 4100, 4225, 4150, 4200, 4000, 4300, 4200]
    c = Case(torch, mvb, [0] * 8, new, 8, 16, 8, 64)
    dt = getattr(torch, dtype)
    q = torch.randn(c.rows, 32, 16, device="cuda").to(dt)
    for max_new in (None, c.rows, 65536):
        out = torch.full_like(q, 9.0)
        mvb.tree_attention(q, c.cache, *c.batch(), out, max_new=max_new)
        assert mvb.serve_status() == 0 and not (out == 9).all(-1).any()
        vs = c.cache.vs.cpu().numpy().astype(np.float64)
        for b in (0, 2, 7):
            k, v = c.values(b, new[b], 0), c.values(b, new[b], 1)
            at = np.arange(new[b])
            for i in (0, 63, 2000, new[b] - 1):
                row = int(c.cu[b]) + i
                for h in (0, 7):
                    want, _, tol, _ = bound(torch, dt, f64(q[row:row + 1, 4 * h:4 * h + 4]), k[:i + 1, h], v[:i + 1, h],
                                            vs[c.pages[b, at // 64], h, at % 64][:i + 1], np.ones((1, i + 1), bool), 0.25,
                                            4096, 8 if dtype == "float32" else 12)
                    assert np.all(np.abs(f64(out[row:row + 1, 4 * h:4 * h + 4]) - want) <= tol)
    with pytest.raises(mvb.MatvecError, match="too many rows"):
        mvb.tree_attention(q, c.cache, *c.batch(), out, max_new=1 << 30)


def test_status_told_once(torch, mvb):
    """Two threads that ask while one of them makes bad calls: every report reaches one of them, once."""
    import threading
    assert mvb.serve_status() == 0
    f, _ = mvb.rope_frequencies(64, 1e4)
    table = mvb.rope_table(f, 10)
    x = torch.ones(1, 1, 64, device="cuda")
    pos = torch.full((1,), 10, dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    told, done = [0, 0], threading.Event()

    def other():
        while not done.is_set():
            told[1] += mvb.serve_status(stream=streams[1], device="cuda:0") != 0

    t = threading.Thread(target=other)
    t.start()
    n = 2000
    for _ in range(n):
        mvb.rope(x, pos, table, stream=streams[0])
        streams[0].synchronize()
        told[0] += mvb.serve_status(stream=streams[0]) != 0
    done.set()
    t.join()
    told[0] += mvb.serve_status() != 0
    assert sum(told) == n, told


def test_failed_occupancy_query_is_not_kept(torch, mvb):
    """A query of the device that fails (here: more threads than a block may have) says nothing about the next."""
    import ctypes as C
    L = mvb.lib()
    slots = L["_ZN3mvb4attn13cluster_slotsEPKviim"]
    slots.restype, slots.argtypes = C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_size_t]
    for name in ("_ZN3mvb4attn11join_kernelIfEEvNS0_10AttnParamsE", "_ZN3mvb4attn11join_kernelI6__halfEEvNS0_10AttnParamsE"):
        kernel = C.cast(L[name], C.c_void_p)
        for n in (1, 2, 4):
            assert slots(kernel, n, 4096, 0) == 0
            assert slots(kernel, n, 128, 0) >= 148 // n * n


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_more_rows_than_the_arrays_hold(torch, mvb, rows):
    """cu that ends behind the row arrays: the rows there are are done, the rest is reported."""
    c = Case(torch, mvb, [5, 0], [rows, 3], 2, 64, 8, 16)
    k = torch.randn(rows, 2, 64, device="cuda")
    mvb.kv_append(c.cache, k, k, *c.batch())
    assert mvb.serve_status() == 2
    ko, vo = torch.full_like(k, 5.0), torch.full_like(k, 5.0)
    mvb.kv_read(c.cache, *c.batch(), ko, vo)
    assert mvb.serve_status() == 2
    ints, scale = ref.quantize(f64(k), 8)
    want = ints * scale[..., None]
    assert np.all(np.abs(f64(ko) - want) <= 2 ** -23 * np.abs(want)) and torch.equal(ko, vo)
    exact = torch.tensor([0, rows, rows], dtype=torch.int32, device="cuda")
    mvb.kv_append(c.cache, k, k, c.pages_, exact, c.lens_)
    mvb.kv_read(c.cache, c.pages_, exact, c.lens_, ko, vo)
    assert mvb.serve_status() == 0


@pytest.mark.parametrize("cu", [[-3, 4, 8], [0, 9, 3, 8]])
def test_row_ranges_out_of_order(torch, mvb, cu):
    """cu that begins below 0 or falls: what was cached before stays, and the append reports rows whose sequence begins elsewhere;
    rows before the first are read as nobody's."""
    c = Case(torch, mvb, [20] * (len(cu) - 1), [4] * (len(cu) - 1), 2, 64, 8, 16)
    k = torch.randn(9, 2, 64, device="cuda")
    negative = cu[0] < 0
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    keep = c.cache.kq.clone()
    mvb.kv_append(c.cache, k, k, c.pages_, cu, c.lens_)
    assert mvb.serve_status() == 2
    for b in range(len(cu) - 1):
        for i in range(20):
            pg, sl = int(c.pages[b, i // 16]), i % 16
            assert torch.equal(c.cache.kq[pg, :, sl], keep[pg, :, sl])
    if negative:
        ko, vo = torch.full_like(k, 5.0), torch.full_like(k, 5.0)
        mvb.kv_read(c.cache, c.pages_, cu, c.lens_, ko, vo)
        assert mvb.serve_status() == 2 and (ko[:4] == 5).all() and not (ko[4:8] == 5).any()
