"""The serving operators (csrc/rope.cu, kvcache.cu, tree_attention.cu, logprobs.cu) against plain forms in 64 bits, at the
types, head layouts, lengths, pages and masks where they can go wrong.

Tolerances (u = half a step of the output's type, relative: 2^-24 fp32, 2^-9 bf16... as torch.finfo(t).eps / 2):
  rope       x cos - y sin in fp32: one rounded product and one fused multiply-add, 2 * 2^-24 * (|x| + |y|), then u.
  cache      integers and scales are exact (equal); values read back are one fp32 product, then u.
  attention  derived in `attention_tolerance`.
  logprobs   derived in `logprob_tolerance`.
"""
import numpy as np
import pytest

import serving_reference as ref
from serving_reference import Case, f64

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "a CUDA device is required"
    t.cuda.set_device(0)
    return t


@pytest.fixture(autouse=True)
def clean_status(request):
    """Every test leaves the error word clear."""
    yield
    m = request.getfixturevalue("mvb")
    assert m.serve_status() == 0


def half_step(torch, dtype):
    return torch.finfo(dtype).eps / 2


def table_for(torch, mvb, positions, rot, theta=1e4, **kw):
    f, factor = mvb.rope_frequencies(rot, theta, **kw)
    return mvb.rope_table(f, positions, factor=factor)


# ---- rope ----

def test_rope_table(torch, mvb):
    f, factor = mvb.rope_frequencies(64, 1e6, "yarn", factor=4.0, original=32768)
    t = mvb.rope_table(f, 300, start=131072 - 200, factor=factor)
    a = (np.arange(300) + 131072 - 200)[:, None] * f
    want = np.concatenate([np.cos(a), np.sin(a)], 1) * factor
    # one rounding to fp32 of values up to factor, fp64 sine and cosine within 2^-50
    assert np.abs(f64(t) - want).max() <= 2 ** -24 * factor + 2 ** -40


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,head,rot,layout", [
    (1, 1, 64, 64, "half"), (1, 14, 64, 64, "pairs"), (5, 6, 48, 48, "half"), (7, 3, 128, 64, "half"),
    (33, 9, 80, 80, "pairs"), (3, 2, 128, 128, "half"), (2, 5, 96, 8, "half"), (2, 5, 96, 8, "pairs"),
    (4000, 17, 128, 96, "half"), (9000, 5, 40, 24, "half"), (3, 1, 8, 8, "half"), (0, 4, 64, 64, "half")])
def test_rope(torch, mvb, dtype, tokens, heads, head, rot, layout):
    dt = getattr(torch, dtype)
    table = table_for(torch, mvb, 500, rot)
    torch.manual_seed(tokens + head)
    x = torch.randn(tokens, heads, head, device="cuda").to(dt)
    pos = torch.randint(500, (tokens,), device="cuda", dtype=torch.int32)
    out = torch.full_like(x, float("nan"))
    mvb.rope(x, pos, table, out, layout=layout)
    want = ref.rope(f64(x), pos.cpu().numpy(), f64(table), layout)
    tol = 4 * 2 ** -24 * (np.abs(f64(x)).max() if tokens else 0) + half_step(torch, dt) * np.abs(want)
    assert np.all(np.abs(f64(out) - want) <= tol)
    # the elements behind rot are copies, in place gives the same bits, and so does a slice of a wider row
    assert torch.equal(out[..., rot:], x[..., rot:])
    y = x.clone()
    mvb.rope(y, pos, table, layout=layout)
    assert torch.equal(y, out)
    wide = torch.zeros(tokens, heads + 3, head, device="cuda", dtype=dt)
    wide[:, 2:2 + heads] = x
    mvb.rope(wide[:, 2:2 + heads], pos, table, layout=layout)
    assert torch.equal(wide[:, 2:2 + heads], out) and not wide[:, :2].any() and not wide[:, 2 + heads:].any()


def test_rope_position_outside(torch, mvb):
    table = table_for(torch, mvb, 10, 64)
    x = torch.ones(4, 2, 64, device="cuda")
    out = torch.full_like(x, 7.0)
    mvb.rope(x, torch.tensor([0, 10, -1, 9], dtype=torch.int32, device="cuda"), table, out)
    assert mvb.serve_status() == 3 and mvb.serve_status() == 0
    assert (out[1:3] == 7).all() and (out[0] == 1).all() and not (out[3] == 7).any()


# ---- the cache ----

LENGTHS = [([0], [1]), ([15], [1]), ([16], [17]), ([0, 31, 5, 100], [3, 0, 40, 1]), ([7] * 40, [1] * 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,new", LENGTHS)
@pytest.mark.parametrize("kv_heads,head,rot,layout,page", [(2, 64, 64, "half", 16), (3, 48, 32, "pairs", 32),
                                                           (1, 128, 128, "half", 64), (5, 80, 80, "pairs", 16),
                                                           (2, 16, 8, "half", 128)])
def test_append_and_read(torch, mvb, dtype, bits, lens, new, kv_heads, head, rot, layout, page):
    dt = getattr(torch, dtype)
    c = Case(torch, mvb, lens, new, kv_heads, head, bits, page, seed=head + page, pad_rows=2)
    heads, n = kv_heads * 3, int(c.cu[-1])
    torch.manual_seed(1)
    qkv = torch.randn(c.rows, heads + 2 * kv_heads, head, device="cuda").to(dt)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    table = table_for(torch, mvb, 200, rot)
    pos = torch.randint(200, (c.rows,), device="cuda", dtype=torch.int32)
    q_out = torch.full((c.rows, heads, head), 9.0, device="cuda", dtype=dt)
    before = [t.clone() for t in (c.cache.kq, c.cache.ks, c.cache.vq, c.cache.vs)]
    mvb.kv_append(c.cache, k, v, *c.batch(), positions=pos, rope=table, layout=layout, q=q, q_out=q_out)
    assert mvb.serve_status() == 0
    p, t64 = pos.cpu().numpy(), f64(table)
    at = ref.slots(c.pages, c.cu, c.lens, page)
    touched = np.zeros(before[1].shape, bool)
    touched[at[:, 0], :, at[:, 1]] = True
    for i, x in ((0, ref.rope(f64(k), p, t64, layout)[:n]), (2, f64(v)[:n])):
        ints, scale = ref.quantize(x, bits)
        got_q, got_s = (c.cache.kq, c.cache.ks, c.cache.vq, c.cache.vs)[i:i + 2]
        assert np.array_equal(ref.unpack(got_q.cpu().numpy(), bits)[at[:, 0], :, at[:, 1]], ints)
        assert np.array_equal(f64(got_s)[at[:, 0], :, at[:, 1]], scale)
        # no other slot changed
        assert np.array_equal(got_q.cpu().numpy()[~touched], before[i].cpu().numpy()[~touched])
        assert np.array_equal(got_s.cpu().numpy()[~touched], before[i + 1].cpu().numpy()[~touched], equal_nan=True)
    want = ref.rope(f64(q), p, t64, layout)[:n]
    tol = 4 * 2 ** -24 * np.abs(f64(q)).max() + half_step(torch, dt) * np.abs(want)
    assert np.all(np.abs(f64(q_out)[:n] - want) <= tol)
    assert (q_out[n:] == 9).all()
    # read back: the rows just written, in every type, into a slice of wider rows
    for out_type in TYPES:
        ot = getattr(torch, out_type)
        buf = torch.full((c.rows, 2 * kv_heads, head), 3.0, device="cuda", dtype=ot)
        mvb.kv_read(c.cache, *c.batch(), buf[:, :kv_heads], buf[:, kv_heads:])
        for half, which in ((buf[:, :kv_heads], 0), (buf[:, kv_heads:], 2)):
            got_q, got_s = (c.cache.kq, c.cache.ks, c.cache.vq, c.cache.vs)[which:which + 2]
            w = ref.unpack(got_q.cpu().numpy(), bits)[at[:, 0], :, at[:, 1]] * f64(got_s)[at[:, 0], :, at[:, 1]][..., None]
            assert np.all(np.abs(f64(half)[:n] - w) <= (2 ** -24 + half_step(torch, ot)) * np.abs(w))
            assert (half[n:] == 3).all()


def test_append_without_rope_and_with_cache_positions(torch, mvb):
    """No table: plain quantization. A table without positions: the position in the cache."""
    c = Case(torch, mvb, [5, 0, 33], [3, 2, 1], 2, 64, 8, 16)
    k, v = torch.randn(6, 2, 64, device="cuda"), torch.randn(6, 2, 64, device="cuda")
    at = ref.slots(c.pages, c.cu, c.lens, 16)
    mvb.kv_append(c.cache, k, v, *c.batch())
    ints, scale = ref.quantize(f64(k), 8)
    assert np.array_equal(f64(c.cache.kq)[at[:, 0], :, at[:, 1]], ints)
    table = table_for(torch, mvb, 64, 64)
    mvb.kv_append(c.cache, k, v, *c.batch(), rope=table)
    ints, scale = ref.quantize(ref.rope(f64(k), np.array([5, 6, 7, 0, 1, 33]), f64(table), "half"), 8)
    assert np.array_equal(f64(c.cache.kq)[at[:, 0], :, at[:, 1]], ints)
    assert np.array_equal(f64(c.cache.ks)[at[:, 0], :, at[:, 1]], scale)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_borders(torch, mvb, bits):
    """Ties between two integers (to even), zero rows, tiny and huge rows, infinities and NaN."""
    most = 127 if bits == 8 else 7
    c = Case(torch, mvb, [0], [10], 1, 32, bits, 16)
    v = torch.zeros(10, 1, 32, device="cuda")
    ties = torch.arange(31, device="cuda") % (2 * most) - most + 0.5
    v[0, 0, 0], v[0, 0, 1:] = most, ties          # scale 1: every other element a tie
    v[1, 0, 0], v[1, 0, 1:] = most * 2.0 ** -60, ties * 2.0 ** -60
    v[2] = 0.0
    v[3, 0] = torch.arange(32, device="cuda") * 2.0 ** -149   # subnormal rows: a scale of a few steps
    v[4, 0] = torch.linspace(-3.4e38, 3.4e38, 32, device="cuda")  # its step overflows: infinite and NaN elements
    v[9, 0] = torch.linspace(-1.0, 1.0, 32, device="cuda") * 3.4e38
    v[5, 0, 3], v[6, 0, 4], v[7, 0, 5] = float("inf"), float("nan"), float("-inf")
    v[8, 0] = torch.randn(32, device="cuda") * 1e-37
    mvb.kv_append(c.cache, v, v, *c.batch())
    at = ref.slots(c.pages, c.cu, c.lens, 16)
    assert not v[4].isfinite().all() and v[9].isfinite().all()
    fine = [0, 1, 2, 3, 8, 9]
    ints, scale = ref.quantize(f64(v)[fine], bits)
    got = ref.unpack(c.cache.vq.cpu().numpy(), bits)[at[:, 0], :, at[:, 1]]
    assert np.array_equal(got[fine], ints)
    assert np.array_equal(f64(c.cache.vs)[at[fine, 0], :, at[fine, 1]], scale)
    assert np.isnan(f64(c.cache.vs)[at[4:8, 0], :, at[4:8, 1]]).all()
    out = torch.zeros(10, 1, 32, device="cuda")
    mvb.kv_read(c.cache, *c.batch(), out, out.clone())
    assert out[4:8].isnan().all() and not out[:4].isnan().any() and not out[8:].isnan().any()


def test_bad_pages_and_lengths_are_skipped(torch, mvb):
    """A page number outside the pool, a position behind the table: reported, nothing else touched."""
    c = Case(torch, mvb, [10, 4], [10, 2], 2, 64, 8, 16)
    k = torch.randn(12, 2, 64, device="cuda")
    keep = c.pages_.clone()
    for bad in (-1, c.cache.pages, 1 << 30):
        c.pages_.copy_(keep)
        c.pages_[0, 1] = bad
        ks = c.cache.ks.clone()
        mvb.kv_append(c.cache, k, k, *c.batch())
        assert mvb.serve_status() == 1
        changed = (c.cache.ks != ks) & ~(c.cache.ks.isnan() & ks.isnan())
        assert int(changed.any(1).sum()) <= 8  # six rows of the first page and the second sequence's two
        out = torch.full((12, 2, 64), 5.0, device="cuda")
        mvb.kv_read(c.cache, *c.batch(), out, out.clone())
        assert mvb.serve_status() == 1 and (out[6:10] == 5).all() and not (out[:6] == 5).all()
        q = torch.randn(12, 4, 64, device="cuda")
        mvb.tree_attention(q, c.cache, *c.batch(), torch.empty_like(q))
        assert mvb.serve_status() == 1
    c.pages_.copy_(keep)
    for lens in ([30, 4], [-3, 4], [1 << 30, 4], [2147483647, 4]):
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        out = torch.full((12, 2, 64), 5.0, device="cuda")
        mvb.kv_read(c.cache, c.pages_, c.cu_, ln, out, out.clone())
        assert mvb.serve_status() in (1, 2)
        q = torch.randn(12, 4, 64, device="cuda")
        o = torch.full_like(q, 5.0)
        mvb.tree_attention(q, c.cache, c.pages_, c.cu_, ln, o)
        if lens[0] != 30:
            assert mvb.serve_status() == 2 and (o[:10] == 5).all()
        else:
            assert mvb.serve_status() in (1, 2)
        assert not (o[10:] == 5).any()


# ---- attention ----

def attention_tolerance(torch, dt, q, k, v, scale, want, keys):
    """Where an output may be off. S: fp32 sums of `head` exact products (fp32 q in two parts: 2^-22 of the row's largest
    element left out): |dS| <= head 2^-22 max|q| max|k| scale; a weight exp(S - m) / z then by 2 |dS| + 2^-20 (the exponential's
    2 ulp, fp32 sums); for 16-bit types each weight is rounded to fp16 once (2^-12), for fp32 held in two fp16 parts (2^-22); a
    weight below 2^-24 of the largest may vanish: keys 2^-24. All times max|v|, plus the output's own rounding."""
    head = q.shape[-1]
    ds = head * 2 ** -22 * np.abs(q).max() * np.abs(k).max() * abs(scale)
    p = 2 ** -12 if dt != torch.float32 else 2 ** -22
    return np.abs(v).max() * (2 * ds + 2 ** -20 + p + keys * 2 ** -24) + half_step(torch, dt) * np.abs(want), \
        ds + 2 ** -20


def mask_bits(torch, c, rng, empty_rows=True):
    """Random allowed pairs (not only trees) as words, with some rows of nothing."""
    n, words = c.rows, max(1, -(-int(c.new.max()) // 64))
    bits = rng.random((n, words * 64)) < 0.5
    if empty_rows:
        bits[::3] = False
    w = np.packbits(bits, axis=1, bitorder="little").view("<i8")
    return bits, torch.from_numpy(w.copy()).cuda()


def check_attention(torch, mvb, c, heads, dtype, tree=True, scale=None, seed=0, q_scale=2.0, max_new=None, max_len=None):
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(seed)
    torch.manual_seed(seed)
    q = (torch.randn(c.rows, heads, c.head, device="cuda") * q_scale).to(dt)
    out = torch.full_like(q, 9.0)
    lse = torch.full((c.rows, heads), 9.0, device="cuda")
    bits, words = mask_bits(torch, c, rng) if tree else (None, None)
    mvb.tree_attention(q, c.cache, *c.batch(), out, tree=words, scale=scale, lse=lse, max_new=max_new, max_len=max_len)
    assert mvb.serve_status() == 0
    sc = scale if scale is not None else c.head ** -0.5
    for b in range(len(c.lens)):
        ctx, n, r0 = int(c.lens[b]), int(c.new[b]), int(c.cu[b])
        if not n:
            continue
        k, v = c.values(b, ctx + n, 0), c.values(b, ctx + n, 1)
        allowed = np.ones((n, ctx + n), bool)
        allowed[:, ctx:] = bits[r0:r0 + n, :n] if tree else np.tril(np.ones((n, n), bool))
        want, want_lse = ref.attention(f64(q)[r0:r0 + n], k, v, allowed, sc)
        tol, lse_tol = attention_tolerance(torch, dt, f64(q), k, v, sc, want, ctx + n)
        got, got_lse = f64(out)[r0:r0 + n], f64(lse)[r0:r0 + n]
        assert np.all(np.abs(got - want) <= tol), (b, np.abs(got - want).max(), tol.min())
        seen = allowed.any(1)
        assert np.all(np.abs(got_lse[seen] - want_lse[seen]) <= lse_tol + 2 ** -22 * np.abs(want_lse[seen]))
        assert np.all(got[~seen] == 0) and np.all(got_lse[~seen] == -np.inf)
    n = int(c.cu[-1])
    assert (out[n:] == 9).all() and (lse[n:] == 9).all()  # rows behind the last sequence
    again = torch.full_like(q, 9.0)
    mvb.tree_attention(q, c.cache, *c.batch(), again, tree=words, scale=scale, max_new=max_new, max_len=max_len)
    assert torch.equal(again, out)  # the same bits
    return q, out


SHAPES = [  # lens, new, heads, kv_heads, head, page
    ([0], [1], 14, 2, 64, 16), ([0], [3], 1, 1, 64, 16), ([1], [1], 2, 2, 48, 32), ([1000], [1], 14, 2, 64, 16),
    ([511, 512, 513], [1, 1, 1], 8, 1, 128, 64), ([100, 0, 7, 300], [5, 1, 0, 9], 6, 6, 48, 16),
    ([17, 250], [16, 31], 9, 1, 96, 32), ([63], [130], 4, 2, 80, 128), ([3000], [2], 32, 8, 128, 16),
    ([40, 1], [70, 64], 7, 1, 64, 64), ([5] * 20, [2] * 20, 4, 4, 16, 16), ([900, 333], [40, 7], 32, 4, 112, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("lens,new,heads,kv_heads,head,page", SHAPES)
def test_attention(torch, mvb, dtype, bits, tree, lens, new, heads, kv_heads, head, page):
    c = Case(torch, mvb, lens, new, kv_heads, head, bits, page, seed=len(lens) + heads, pad_rows=1)
    check_attention(torch, mvb, c, heads, dtype, tree, max_new=max(new))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_long(torch, mvb, dtype, bits):
    """A context split over a cluster, in pages that end inside slices."""
    c = Case(torch, mvb, [20011, 3], [4, 4], 2, 128, bits, 16)
    check_attention(torch, mvb, c, 6, dtype, max_new=4, max_len=20015)


@pytest.mark.parametrize("max_len", [0, 1, 100, 1 << 30])
def test_attention_max_len_only_splits(torch, mvb, max_len):
    c = Case(torch, mvb, [700, 90], [3, 1], 2, 64, 8, 32)
    check_attention(torch, mvb, c, 4, "float32", max_new=3, max_len=max_len)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scales(torch, mvb, dtype):
    """Scales of keys and values over many magnitudes, a negative softmax scale, large logits."""
    c = Case(torch, mvb, [300], [6], 2, 64, 8, 16)
    c.cache.vs.mul_(torch.exp2(torch.randint(-6, 7, c.cache.vs.shape, device="cuda").float()))
    check_attention(torch, mvb, c, 4, dtype)
    check_attention(torch, mvb, c, 4, dtype, scale=-0.3)
    c.cache.vs.mul_(2.0 ** 60)
    check_attention(torch, mvb, c, 4, dtype if dtype != "float16" else "bfloat16")
    c = Case(torch, mvb, [300], [6], 2, 64, 8, 16)
    check_attention(torch, mvb, c, 4, dtype, q_scale=30.0)
    c.cache.vs.zero_()
    _, out = check_attention(torch, mvb, c, 4, dtype)
    assert not out.any()


@pytest.mark.parametrize("tokens", [3, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_poison_stays_in_its_rows(torch, mvb, dtype, tokens):
    """A new token whose key or value is NaN or infinite changes only the rows that see it; what it holds where the mask
    hides it does not matter."""
    c = Case(torch, mvb, [70], [tokens], 1, 64, 8, 16)
    q = torch.randn(tokens, 7, 64, device="cuda").to(getattr(torch, dtype))
    tree = mvb.tree_mask([-1] * tokens).cuda()  # every token sees the context and itself
    clean = torch.empty_like(q)
    mvb.tree_attention(q, c.cache, *c.batch(), clean, tree=tree)
    at = ref.slots(c.pages, c.cu, c.lens, 16)
    for which in (c.cache.ks, c.cache.vs):
        for bad in (float("nan"), float("inf")):
            keep = which.clone()
            which[at[1, 0], :, at[1, 1]] = bad
            out = torch.empty_like(q)
            mvb.tree_attention(q, c.cache, *c.batch(), out, tree=tree)
            others = [i for i in range(tokens) if i != 1]
            assert torch.equal(out[others], clean[others])
            assert not out[1].isfinite().all()
            which.copy_(keep)


def test_attention_lone_nan_key(torch, mvb):
    """The only key a row may see is NaN: NaN, not the zeros of an empty row."""
    c = Case(torch, mvb, [0], [1], 1, 64, 8, 16)
    at = ref.slots(c.pages, c.cu, c.lens, 16)
    c.cache.ks[at[0, 0], :, at[0, 1]] = float("nan")
    q = torch.randn(1, 2, 64, device="cuda")
    out = torch.zeros_like(q)
    mvb.tree_attention(q, c.cache, *c.batch(), out)
    assert out.isnan().all()


def test_attention_more_new_than_said(torch, mvb):
    c = Case(torch, mvb, [10, 20], [2, 5], 1, 64, 8, 16)
    q = torch.randn(7, 2, 64, device="cuda")
    out = torch.full_like(q, 9.0)
    mvb.tree_attention(q, c.cache, *c.batch(), out, max_new=4)
    assert mvb.serve_status() == 2 and (out[2:] == 9).all() and not (out[:2] == 9).any()


# ---- log probabilities ----

def logprob_tolerance(x, logp):
    """exp within 2 ulp and the fp32 rounding of x - m (2^-24 |x - m|) and of its product with log2 e: a term is off by
    2^-22 + 2^-23 |x - m| of itself, which is at most 2^-22 + 2^-23 * |ln p|; fp32 sums of 2^21 terms in at most 2^9 steps
    a thread and 13 joins: 2^-15 at worst, 2^-19 for signs that do not conspire (asserted: 2^-18 (1 + |logp|))."""
    return 2.0 ** -18 * (1 + np.abs(logp))


def check_logprobs(torch, mvb, x, ids, top):
    r = mvb.logprobs(x, ids, top=top)
    assert mvb.serve_status() == 0
    y = f64(x)
    m = y.max(1, keepdims=True)
    # (y - m) first: m + ln z would lose ln z in rows whose largest logit is the type's lowest value
    lp = (y - m) - np.log(np.exp(y - m).sum(1, keepdims=True))
    if ids is not None:
        i = ids.cpu().numpy()
        want = np.where(i == -1, 0, np.take_along_axis(lp, np.maximum(i, 0), 1))
        got = f64(r.logp)
        assert np.array_equal(np.isinf(got), np.isinf(want))
        fine = np.isfinite(want)
        assert np.all(np.abs(got - want)[fine] <= logprob_tolerance(y, want)[fine])
    with np.errstate(invalid="ignore"):
        ent = -(np.where(np.isfinite(lp), np.exp(lp) * lp, 0)).sum(1)
    assert np.all(np.abs(f64(r.entropy) - ent) <= 2.0 ** -18 * (1 + np.abs(ent)) * np.log(x.shape[1] + 1))
    order = np.argsort(-(y + 0.0), axis=1, kind="stable")[:, :top]
    assert np.array_equal(r.top_ids.cpu().numpy(), order)
    want = np.take_along_axis(lp, order, 1)
    got = f64(r.top_logp)
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine)
    assert np.all(np.abs(got - want)[fine] <= logprob_tolerance(y, want)[fine])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,nids,top", [
    (1, 1, 1, 1), (1, 2, 2, 2), (3, 7, 1, 7), (2, 33, 3, 5), (5, 1000, 2, 64), (2, 4097, 1, 20), (300, 4099, 1, 3),
    (1, 32000, 4, 10), (9, 65536, 1, 20), (1, 151936, 1, 5), (4, 151937, 2, 64), (700, 32001, 1, 0), (1, 700001, 1, 8)])
def test_logprobs(torch, mvb, dtype, rows, vocab, nids, top):
    torch.manual_seed(vocab)
    x = (torch.randn(rows, vocab, device="cuda") * 3).to(getattr(torch, dtype))
    ids = torch.randint(vocab, (rows, nids), device="cuda", dtype=torch.int32)
    if nids > 1:
        ids[:, 1] = -1
    check_logprobs(torch, mvb, x, ids, top)


@pytest.mark.parametrize("rows", [1, 40, 400])
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_masked_vocabulary(torch, mvb, dtype, rows):
    """A vocabulary masked to a few tokens by -inf or by the type's lowest value: the alternatives go on with the lowest
    ids of the equal rest; rows of equal logits; sorted rows, whose largest all come last."""
    dt = getattr(torch, dtype)
    vocab = 20003
    torch.manual_seed(rows)
    for fill in (float("-inf"), torch.finfo(dt).min, 0.0):
        x = torch.full((rows, vocab), fill, device="cuda", dtype=dt)
        for r in range(min(rows, 40)):
            x[r, torch.randint(vocab, (3,), device="cuda")] = torch.tensor([1.0, 2.0, 2.0], device="cuda", dtype=dt)
        x[-1, vocab - 1] = 3.0
        if fill == float("-inf"):
            x[40:, 17] = 1.0
        check_logprobs(torch, mvb, x, torch.full((rows, 1), vocab - 1, dtype=torch.int32, device="cuda"), 20)
    x = torch.arange(vocab, device="cuda").float().mul_(1e-3).to(dt).repeat(rows, 1)
    check_logprobs(torch, mvb, x, None, 33)
    check_logprobs(torch, mvb, x.flip(1).contiguous(), None, 33)
    x = torch.zeros(rows, vocab, device="cuda", dtype=dt)
    x[:, ::2] = -0.0
    check_logprobs(torch, mvb, x, None, 64)


def test_logprobs_strides(torch, mvb):
    """Rows of a wider matrix, at every alignment."""
    wide = torch.randn(6, 5013, device="cuda")
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        w = wide.to(dt)
        for off in range(9):
            check_logprobs(torch, mvb, w[:, off:off + 5000], None, 11)


def test_logprobs_not_numbers(torch, mvb):
    """NaN and +inf make a row NaN (ids still ordered, NaN last); a row without a finite logit too; its neighbours keep."""
    x = torch.randn(5, 3001, device="cuda")
    clean = mvb.logprobs(x, torch.full((5, 1), 7, dtype=torch.int32, device="cuda"), top=4)
    x[1, 100], x[2, 200], x[3] = float("nan"), float("inf"), float("-inf")
    r = mvb.logprobs(x, torch.full((5, 1), 7, dtype=torch.int32, device="cuda"), top=4)
    for t in (r.logp, r.entropy[:, None], r.top_logp):
        assert t[1:4].isnan().all() and t[[0, 4]].isfinite().all()
    for a, b in zip(r, clean):
        assert torch.equal(a[[0, 4]], b[[0, 4]])
    assert r.top_ids[2, 0] == 200 and r.top_ids[3].tolist() == [0, 1, 2, 3]
    keep = x[1].clone()
    keep[100] = float("-inf")
    assert r.top_ids[1].tolist() == keep.topk(4).indices.tolist()
    x = torch.full((1, 6), float("nan"), device="cuda")
    x[0, 4] = 1.0
    assert mvb.logprobs(x, top=6).top_ids.tolist() == [[4, 0, 1, 2, 3, 5]]


def test_logprobs_id_outside(torch, mvb):
    x = torch.randn(2, 50, device="cuda")
    r = mvb.logprobs(x, torch.tensor([[0, 50], [-2, 49]], dtype=torch.int32, device="cuda"))
    assert mvb.serve_status() == 4
    assert r.logp.isnan().tolist() == [[False, True], [True, False]]
