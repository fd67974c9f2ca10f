"""The serving operators as they are used together, and where calls meet: a step of drafted trees over a cache that the
framework's own matmul feeds, accepted tokens appended again; streams, CUDA graphs, caches whose offsets pass 32 bits; the
decoder's own log probabilities."""
import os
import subprocess
import sys

import numpy as np
import pytest

import serving_reference as ref
from conftest import ROOT, load_pkg
from serving_reference import Case, f64
from test_serving_gpu import attention_tolerance, check_attention, logprob_tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "a CUDA device is required"
    t.cuda.set_device(0)
    return t


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("lens,new,heads,kv_heads,head,page", [
    ([0], [30], 2, 2, 64, 16), ([63, 64, 65, 200], [10, 12, 1, 9], 8, 2, 128, 32), ([1], [26], 3, 3, 16, 16),
    ([300, 0], [100, 128], 5, 5, 48, 64), ([129], [33], 4, 4, 96, 16), ([70, 10], [64, 3], 4, 2, 64, 128),
    ([500, 0, 3], [129, 1, 140], 2, 1, 32, 16), ([40], [300], 2, 2, 112, 1024)])
def test_many_rows(torch, mvb, dtype, bits, tree, lens, new, heads, kv_heads, head, page):
    """25 to 128 rows a kv head (both softmax groups on one row tile) and more, at every head size's padding."""
    c = Case(torch, mvb, lens, new, kv_heads, head, bits, page, seed=sum(new), pad_rows=2)
    check_attention(torch, mvb, c, heads, dtype, tree, max_new=max(new))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("drafts,lens,heads,kv_heads,head,page", [
    (10, [0, 3, 700, 64, 65, 130, 1, 200, 63, 31], 4, 2, 128, 32), (12, list(range(0, 760, 40)), 2, 1, 96, 16),
    (60, [3000, 2000], 4, 2, 128, 64), (130, [2500, 40], 2, 1, 128, 16)])
def test_tiles_refilled(torch, mvb, dtype, bits, drafts, lens, heads, kv_heads, head, page):
    """17 to 24 rows of many sequences, and enough steps for every ring of the tensor-core kernel to come round."""
    c = Case(torch, mvb, lens, [drafts] * len(lens), kv_heads, head, bits, page, seed=drafts, pad_rows=1)
    check_attention(torch, mvb, c, heads, dtype, max_new=drafts)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("drafts", [1, 4, 7, 40, 150])
@pytest.mark.parametrize("max_len", [None, 17000, 300])
def test_long_context(torch, mvb, dtype, drafts, max_len):
    """Few sequences with a long context: clusters, and several clusters a sequence joined by a second kernel."""
    c = Case(torch, mvb, [16700, 5], [drafts, 1], 1, 64, 8, 64, seed=drafts)
    check_attention(torch, mvb, c, 3, dtype, max_new=drafts, max_len=max_len)


def test_no_workspace_and_too_small(torch, mvb):
    """The C call takes a workspace of any size, or none: the same result."""
    c = Case(torch, mvb, [20000], [2], 2, 128, 8, 32)
    q = torch.randn(2, 4, 128, device="cuda")
    want = mvb.tree_attention(q, c.cache, *c.batch(), torch.empty_like(q), max_new=2, max_len=20002)
    L, s = mvb.lib(), torch.cuda.current_stream().cuda_stream
    need = L.mvb_tree_attention_work(2, 4, 2, 128, 1, 2, 20002)
    assert need > 0 and L.mvb_tree_attention_work(2, 4, 2, 128, 64, 2, 20002) == 0
    for size in (0, 16, need // 8, need // 3, need):
        work = torch.empty(max(size, 16) + 64, dtype=torch.uint8, device="cuda").fill_(255)
        out = torch.full_like(q, 9.0)
        rc = L.mvb_tree_attention(q.data_ptr(), 512, *c.cache.args, c.pages_.data_ptr(), c.pages_.shape[1],
                                  c.cu_.data_ptr(), c.lens_.data_ptr(), 1, 2, 4, 0, None, 0, 128 ** -0.5, 2, 20002,
                                  out.data_ptr(), 512, None, work.data_ptr() if size else None, size, s)
        assert rc == 0 and (work[max(size, 16):] == 255).all()
        k, v = c.values(0, 20002, 0), c.values(0, 20002, 1)
        tol, _ = attention_tolerance(torch, torch.float32, f64(q), k, v, 128 ** -0.5, f64(want), 20002)
        assert np.all(np.abs(f64(out) - f64(want)) <= 2 * tol)


def test_speculative_step(torch, mvb, restatement):
    """One layer of a step with drafted trees: the projection by the framework's matmul (its rows sliced, not copied), keys
    and queries turned by the depth in the tree, cache written, attention, head, log probabilities of the drafts; then the
    longest path is kept: its rows appended again at the context's end, and the next single token attends to it. Each stage
    against 64 bits on what the stage before left."""
    rng = np.random.default_rng(3)
    torch.manual_seed(3)
    heads, kv, head, dim, page, bits = 14, 2, 64, 896, 16, 8
    lens, new = [37, 0, 130], [6, 3, 1]
    c = Case(torch, mvb, lens, new, kv, head, bits, page, seed=9, pad_rows=2)
    parents = [[-1, 0, 0, 1, 1, 3], [-1, -1, 1], [-1]]
    m, width = c.rows, (heads + 2 * kv) * head
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    w = rng.integers(0, 256, (width, dim // 2), dtype=np.uint8)
    ws = ((rng.integers(0, 2, width * dim // 32) << 15) | (rng.integers(5, 9, width * dim // 32) << 10)).astype(np.uint16)
    xq, xs = zip(*(restatement.quantize_qwen(rng.standard_normal(dim).astype(np.float32)) for _ in range(m)))
    ldx = (m + 3) // 4 * 4
    xs_gm = np.zeros((dim // 32, ldx), np.float32)
    xs_gm[:, :m] = np.stack(xs).T
    qkv = torch.empty(m, width, device="cuda")
    mvb.gemm4(dev(w), dev(ws.view(np.int16)), dev(np.stack(xq)), dev(xs_gm), qkv, dim, width, m, ldx, 4)
    assert mvb.gemm_status() == 0
    qkv = qkv.view(m, heads + 2 * kv, head)
    q, k, v = qkv.split([heads, kv, kv], 1)
    masks = [mvb.tree_mask(p) for p in parents]
    depth = [[int(bin(int(x) & (2 ** 64 - 1)).count("1")) - 1 for x in t[:, 0]] for t in masks]
    pos = torch.tensor([n + d for n, ds in zip(lens, depth) for d in ds] + [0] * 2, dtype=torch.int32, device="cuda")
    tree = torch.cat([t[:, :1] for t in masks] + [torch.zeros(2, 1, dtype=torch.int64)]).cuda()
    f, factor = mvb.rope_frequencies(head, 1e6)
    table = mvb.rope_table(f, 512, factor=factor)
    q_raw, k_raw, v_raw = f64(q), f64(k), f64(v)
    out, lse = torch.zeros(m, heads, head, device="cuda"), torch.zeros(m, heads, device="cuda")
    mvb.kv_append(c.cache, k, v, *c.batch(), positions=pos, rope=table, q=q, q_out=q)  # q in place, in the wide rows
    mvb.tree_attention(q, c.cache, *c.batch(), out, tree=tree, max_new=6, max_len=131, lse=lse)
    assert mvb.serve_status() == 0
    n = int(c.cu[-1])
    p, t64 = pos.cpu().numpy(), f64(table)
    q64 = ref.rope(q_raw, p, t64, "half")
    assert np.abs(f64(q)[:n] - q64[:n]).max() <= 2 ** -22 * np.abs(q_raw).max()
    assert np.array_equal(f64(k), k_raw) and np.array_equal(f64(v), v_raw) and np.array_equal(f64(q)[n:], q_raw[n:])
    at = ref.slots(c.pages, c.cu, c.lens, page)
    ints, scale = ref.quantize(ref.rope(k_raw, p, t64, "half")[:n], bits)
    assert np.array_equal(f64(c.cache.kq)[at[:, 0], :, at[:, 1]], ints)
    got_q = f64(q)
    for b in range(3):
        r0, nb, ctx = int(c.cu[b]), new[b], lens[b]
        allowed = np.ones((nb, ctx + nb), bool)
        bits_ = np.unpackbits(masks[b].numpy().view(np.uint8), axis=1, bitorder="little")[:, :nb]
        allowed[:, ctx:] = bits_
        kk, vv = c.values(b, ctx + nb, 0), c.values(b, ctx + nb, 1)
        want, _ = ref.attention(got_q[r0:r0 + nb], kk, vv, allowed, head ** -0.5)
        tol, _ = attention_tolerance(torch, torch.float32, got_q, kk, vv, head ** -0.5, want, ctx + nb)
        assert np.all(np.abs(f64(out)[r0:r0 + nb] - want) <= tol)
    # the head (a plain product stands for it) and the drafts' log probabilities under their parents' rows
    logits = out[:n].flatten(1) @ torch.randn(heads * head, 5000, device="cuda") * 0.1
    drafted = torch.randint(5000, (n, 2), device="cuda", dtype=torch.int32)
    r = mvb.logprobs(logits, drafted, top=3)
    y = f64(logits)
    lp = (y - y.max(1, keepdims=True)) - np.log(np.exp(y - y.max(1, keepdims=True)).sum(1, keepdims=True))
    want = np.take_along_axis(lp, drafted.cpu().numpy(), 1)
    assert np.all(np.abs(f64(r.logp) - want) <= logprob_tolerance(y, want))
    assert np.array_equal(r.top_ids.cpu().numpy(), np.argsort(-y, axis=1, kind="stable")[:, :3])
    # sequence 0 keeps drafts 0, 1, 3, 5 (one path): appended again behind the context, then one token attends
    path = torch.tensor([0, 1, 3, 5], device="cuda")
    cu1 = torch.tensor([0, 4, 4, 4], dtype=torch.int32, device="cuda")
    wide = qkv.index_select(0, path)
    mvb.kv_append(c.cache, wide[:, heads:heads + kv], wide[:, heads + kv:], c.pages_, cu1, c.lens_,
                  positions=pos[path].contiguous(), rope=table)
    kept = c.values(0, 41, 0)[37:]
    ints, scale = ref.quantize(ref.rope(k_raw, p, t64, "half")[[0, 1, 3, 5]], bits)
    assert np.array_equal(kept, ints * scale[..., None])
    q1, o1 = torch.randn(1, heads, head, device="cuda"), torch.empty(1, heads, head, device="cuda")
    lens1 = torch.tensor([40, 0, 130], dtype=torch.int32, device="cuda")
    cu2 = torch.tensor([0, 1, 1, 1], dtype=torch.int32, device="cuda")
    mvb.tree_attention(q1, c.cache, c.pages_, cu2, lens1, o1, max_new=1, max_len=41)
    kk, vv = c.values(0, 41, 0), c.values(0, 41, 1)
    want, _ = ref.attention(f64(q1), kk, vv, np.ones((1, 41), bool), head ** -0.5)
    tol, _ = attention_tolerance(torch, torch.float32, f64(q1), kk, vv, head ** -0.5, want, 41)
    assert np.all(np.abs(f64(o1) - want) <= tol) and mvb.serve_status() == 0


@pytest.mark.parametrize("new,ctx", [(1, 10), (3, 5000), (20, 100), (40, 5000), (90, 20000), (2, 20000)])
def test_out_over_q(torch, mvb, new, ctx):
    """out may be q: every row is read before one is written, however the work is split."""
    c = Case(torch, mvb, [ctx, 7], [new, 2], 2, 64, 8, 32)
    q = torch.randn(c.rows, 6, 64, device="cuda")
    want = mvb.tree_attention(q, c.cache, *c.batch(), torch.empty_like(q), max_new=max(new, 2))
    mvb.tree_attention(q, c.cache, *c.batch(), q, max_new=max(new, 2))
    assert torch.equal(q, want)


@pytest.mark.parametrize("drafts", [2, 40])
def test_graphs_and_streams(torch, mvb, drafts):
    """The same step eagerly, on another stream, and as two captured graphs replayed at once on two streams, with contents
    (queries, lengths, page table) changed after the capture: the same bits each time."""
    kv, heads, head = 1, 3, 64
    runs = []
    for i in range(2):
        c = Case(torch, mvb, [16900, 5], [drafts, 1], kv, head, 8, 64, seed=i)
        torch.manual_seed(i)
        x = torch.randn(c.rows, heads + 2 * kv, head, device="cuda")
        f, factor = mvb.rope_frequencies(head, 1e6)
        table = mvb.rope_table(f, 20000, factor=factor)
        pos = torch.randint(20000, (c.rows,), device="cuda", dtype=torch.int32)
        tree = torch.randint(1, 2 ** 40, (c.rows, 1), device="cuda") | 1
        out = torch.empty(c.rows, heads, head, device="cuda")
        lse = torch.empty(c.rows, heads, device="cuda")
        logits = torch.randn(3, 40000, device="cuda")
        runs.append([c, x, table, pos, tree, out, lse, kv, heads, logits])

    def copy(r, p):
        return [t.clone() for t in (r[5], r[6], r[0].cache.kq, *p[1:])]

    def attend(r):
        c, x, table, pos, tree, out, lse, kv, heads, logits = r
        q, k, v = x.split([heads, kv, kv], 1)
        turned = torch.empty_like(out)
        mvb.kv_append(c.cache, k, v, *c.batch(), positions=pos, rope=table, q=q, q_out=turned)
        mvb.tree_attention(turned, c.cache, *c.batch(), out, tree=tree, max_new=40, max_len=20000, lse=lse)
        return mvb.logprobs(logits, top=9)

    want = [copy(r, attend(r)) for r in runs]
    for r in runs:
        r[5].fill_(7.0)
    # another stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = copy(runs[0], attend(runs[0]))
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    # two graphs, captured with other contents
    graphs, results, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    keep = [(r[1].clone(), r[0].lens_.clone(), r[0].pages_.clone()) for r in runs]
    for r in runs:
        r[1].zero_()
        r[0].lens_.zero_()
    torch.cuda.synchronize()
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(attend(r))
        graphs.append(g)
    for r, (x, lens, pages) in zip(runs, keep):
        r[1].copy_(x)
        r[0].lens_.copy_(lens)
        r[0].pages_.copy_(pages)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for r, p, w in zip(runs, results, want):
        assert all(torch.equal(a, b) for a, b in zip(copy(r, p), w))
    assert mvb.serve_status() == 0


def test_first_call_in_a_capture():
    """A process whose first calls of all are captured."""
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch
from conftest import load_pkg
from serving_reference import Case
mvb = load_pkg()
c = Case(torch, mvb, [100, 3], [3, 40], 2, 64, 8, 16)
x = torch.randn(c.rows, 8, 64, device="cuda"); out = torch.empty(c.rows, 4, 64, device="cuda")
f, a = mvb.rope_frequencies(64, 1e4)
f = torch.from_numpy(f).cuda(); table = torch.empty(300, 64, device="cuda")
lg = torch.randn(2, 5000, device="cuda"); pos = torch.arange(c.rows, device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    mvb.rope_table(f, 300, out=table)
    mvb.rope(x, pos, table)
    mvb.kv_append(c.cache, x[:, 4:6], x[:, 6:], *c.batch())
    mvb.tree_attention(x[:, :4], c.cache, *c.batch(), out, max_new=3)
    mvb.tree_attention(x[:, :4], c.cache, *c.batch(), out, max_new=40)
    r = mvb.logprobs(lg, top=4)
keep = x.clone(); g.replay(); torch.cuda.synchronize()
first = out.clone(); x.copy_(keep); mvb.rope(x, pos, table)
mvb.tree_attention(x[:, :4], c.cache, *c.batch(), out, max_new=40)
assert torch.equal(first, out) and r.top_ids.tolist() == lg.topk(4).indices.tolist()
assert mvb.serve_status() == 2
print("fine")
""" % (ROOT + "/tests", ROOT)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "CUDA_MODULE_LOADING": "LAZY"})
    assert r.stdout.strip().endswith("fine"), r.stdout + r.stderr


def test_far_pages(torch, mvb):
    """A pool whose bytes pass 2^32 (and whose rows pass 2^25): the last pages, written, read and attended."""
    kv, head, page, bits = 8, 128, 64, 8
    pages = (1 << 32) // (kv * page * head) + 40
    cache = mvb.KvCache.empty(pages, kv, page, head, bits)
    table = torch.tensor([[pages - 1, pages - 7, 3], [pages - 2, 1, pages - 3]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 150, 290], dtype=torch.int32, device="cuda")
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    torch.manual_seed(0)
    k, v = torch.randn(290, kv, head, device="cuda"), torch.randn(290, kv, head, device="cuda")
    mvb.kv_append(cache, k, v, table, cu, zero)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    mvb.kv_read(cache, table, cu, zero, ko, vo)
    for a, b in ((k, ko), (v, vo)):
        ints, scale = ref.quantize(f64(a), bits)
        want = (ints * scale[..., None])
        assert np.all(np.abs(f64(b) - want) <= 2 ** -23 * np.abs(want))
    for rows in (1, 7):  # the few-row kernel and the tensor-core one
        q = torch.randn(2 * rows, kv * 4, head, device="cuda")
        out = torch.empty_like(q)
        lens = torch.tensor([150 - rows, 140 - rows], dtype=torch.int32, device="cuda")
        cq = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
        mvb.tree_attention(q, cache, table, cq, lens, out, max_new=rows, max_len=150)
        for b, n in ((0, 150), (1, 140)):
            kk, vv = f64(ko)[150 * b:150 * b + n], f64(vo)[150 * b:150 * b + n]
            allowed = np.arange(n)[None] <= n - rows + np.arange(rows)[:, None]
            want, _ = ref.attention(f64(q)[b * rows:(b + 1) * rows], kk, vv, allowed, head ** -0.5)
            tol, _ = attention_tolerance(torch, torch.float32, f64(q), kk, vv, head ** -0.5, want, n)
            # (the values read back are rounded once more: 2^-24 each)
            assert np.all(np.abs(f64(out)[b * rows:(b + 1) * rows] - want) <= tol + 2 ** -20)
    assert mvb.serve_status() == 0


def test_far_logits(torch, mvb):
    """Rows of logits whose offsets pass 2^32 elements' bytes and 2^31 elements."""
    big = torch.empty((1 << 31) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (2, 1000), ((1 << 31) + 7, 1))
    x.copy_(torch.randn(2, 1000, device="cuda"))
    r = mvb.logprobs(x, top=5)
    assert r.top_ids[1, 0] == int(x[1].float().argmax()) and r.entropy.isfinite().all()


def test_rows_outside_every_sequence(torch, mvb):
    """cu that begins behind row 0: the rows before it are nobody's."""
    c = Case(torch, mvb, [20], [4], 2, 64, 8, 16)
    cu = torch.tensor([3, 7], dtype=torch.int32, device="cuda")
    x = torch.randn(9, 2, 64, device="cuda")
    q = torch.randn(9, 4, 64, device="cuda")
    f, _ = mvb.rope_frequencies(64, 1e4)
    table = mvb.rope_table(f, 64)
    qo = torch.full_like(q, 5.0)
    mvb.kv_append(c.cache, x, x, c.pages_, cu, c.lens_, rope=table, q=q, q_out=qo)
    ko, vo = torch.full_like(x, 5.0), torch.full_like(x, 5.0)
    mvb.kv_read(c.cache, c.pages_, cu, c.lens_, ko, vo)
    out = torch.full_like(q, 5.0)
    mvb.tree_attention(q, c.cache, c.pages_, cu, c.lens_, out)
    for t in (qo, ko, vo, out):
        assert (t[:3] == 5).all() and (t[7:] == 5).all() and not (t[3:7] == 5).any()
    assert mvb.serve_status() == 0


def test_decoder_logprobs(torch, mvb, tmp_path):
    """The decoder's log probabilities against its downloaded logits; after a decode step too; refusals."""
    path = str(tmp_path / "tiny.qwb")
    mvb.qwb.write_synthetic_qwb(path, mvb.qwb.QWEN_TINY, seed=11)
    dec = mvb.QwenDecoder(path, ctx=64)
    try:
        for full in (False, True):
            dec.full_head(full)
            for pos, tok in enumerate((5, 9, 700)):
                row, logits = dec.forward(tok, pos)
                n = logits.size
                rows = [0, n - 1, row, 17]
                logp, ent, top, top_logp = dec.logprobs(rows, top=6)
                y = logits.astype(np.float64)
                lp = (y - y.max()) - np.log(np.exp(y - y.max()).sum())
                assert np.all(np.abs(logp - lp[rows]) <= logprob_tolerance(y, lp[rows]))
                assert abs(ent + (np.exp(lp) * lp).sum()) <= 2.0 ** -18 * np.log(n) * 8
                assert top[0] == row and np.array_equal(top, np.argsort(-y, kind="stable")[:6])
                assert np.all(np.abs(top_logp - lp[top]) <= logprob_tolerance(y, lp[top]))
        assert dec.logprobs()[0].size == 0
        for bad in (dict(rows=[n]), dict(rows=[-1]), dict(top=65), dict(rows=[0] * 1025)):
            with pytest.raises(mvb.MatvecError):
                dec.logprobs(**bad)
    finally:
        dec.close()
