"""Attention over pages, heads into pages, copies of pages and sampling against plain float64 loops: sizes and masks where they can
go wrong, what masked places hold, refusals, and a run of them together."""
import importlib

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import float_oracle as fo

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "bfloat16"]
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}           # a rounding's most, relative


@pytest.fixture(scope="module")
def K(float_libpath):
    torch.backends.cuda.matmul.allow_tf32 = False
    return importlib.import_module(PKG + ".float_kernel")


def rnd(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(getattr(torch, dtype)).cuda()


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def np64(t):
    return t.double().cpu().numpy()


# ---- attention ---------------------------------------------------------------------------------------------------
def pool(dtype, new, lengths, page, heads, kv_heads, d, dv, seed=0, spare=3, fill=float("nan"), pad=0):
    """a batch over a pool: pages in no order, everything that no sequence holds is `fill`"""
    g = np.random.default_rng(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = g.permutation(pages)
    cols = max(need + [1]) + 1
    table = np.full((len(lengths), cols), -7, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    width = kv_heads * (d + dv) + pad
    both = torch.full((pages, page, width), fill, dtype=getattr(torch, dtype), device="cuda")
    for b, n in enumerate(lengths):
        for p in range(need[b]):
            lines = min(page, n - p * page)
            both[table[b, p], :lines] = rnd((lines, width), dtype, seed + 100 + 37 * b + p)
    rows = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    return dict(k=both[:, :, :kv_heads * d].unflatten(2, (kv_heads, d)),
                v=both[:, :, kv_heads * d:kv_heads * (d + dv)].unflatten(2, (kv_heads, dv)),
                table=torch.from_numpy(table).cuda(), rows=torch.from_numpy(rows).cuda(), lengths=i32(*lengths),
                q=rnd((int(rows[-1]), heads, d), dtype, seed + 1), host=(table, rows, lengths), new=new)


def attend(K, s, dtype, scale, window=0, gate=None, out_scale=1.0, behind=2, **kw):
    q, dv = s["q"], s["v"].shape[3]
    out = torch.full((q.shape[0] + behind, q.shape[1], dv), 5.0, dtype=q.dtype, device="cuda")
    qx = torch.cat([q, torch.full((behind,) + q.shape[1:], float("nan"), dtype=q.dtype, device="cuda")])
    gx = None if gate is None else torch.cat([gate, gate[:1].expand(behind, -1, -1)])
    K.paged_attention(qx, s["k"], s["v"], s["table"], s["rows"], s["lengths"], out, scale, window=window, gate=gx, out_scale=out_scale, **kw)
    assert (out[q.shape[0]:] == 5.0).all()              # rows behind the last sequence
    return out[:q.shape[0]]


def limit(dtype, size, score, d, keys):
    """Half steps that a result can be off by.  A weight: its score's sum of d products in 32 bits, both of score and maximum,
    the exponential's few ulps, its sum of `keys` weights; the weighted sum as many additions.  In bfloat16 also the weight's own
    rounding; the result's rounding is added by the caller."""
    e = 2.0 ** -24 * (2 * (d + 4) * score[..., None] + 3 * keys + 32)
    return size * (e + (HALF[dtype] if dtype == "bfloat16" else 0.0)) * 1.05


def check(K, s, dtype, scale=None, window=0, gate=None, out_scale=1.0, **kw):
    d = s["q"].shape[2]
    scale = d ** -0.5 if scale is None else scale
    got = np64(attend(K, s, dtype, scale, window, gate, out_scale, **kw))
    K.device_status(sync=True)
    table, rows, lengths = s["host"]
    want, size, score = fo.paged_attention(np64(s["q"]), np64(s["k"]), np64(s["v"]), table, rows, lengths, scale, window,
                                           None if gate is None else np64(gate), out_scale)
    off = np.abs(got - want) - limit(dtype, size, score, d, max(list(lengths) + [1])) - HALF[dtype] * np.abs(want)
    if gate is not None:
        off -= 2.0 ** -22 * np.abs(want)
    assert np.isfinite(got).all() and (off <= 1e-30).all(), float(off.max())
    return got


SHAPES = [  # new, lengths, page, heads, kv heads, d, dv, window
    ([1], [1], 8, 1, 1, 8, 8, 0), ([1], [4095], 64, 8, 2, 128, 128, 0), ([1, 1, 1], [17, 600, 64], 16, 8, 2, 64, 64, 0),
    ([2, 0, 1], [130, 40, 9], 32, 6, 2, 24, 40, 0), ([1, 3], [65, 64], 64, 7, 1, 40, 24, 5), ([16], [16], 16, 4, 4, 128, 128, 0),
    ([5, 1, 2], [300, 1, 77], 128, 12, 4, 96, 128, 64), ([100], [100], 16, 4, 2, 80, 80, 0), ([129, 1], [400, 33], 8, 3, 3, 16, 16, 33),
    ([33, 64], [512, 64], 1024, 16, 2, 128, 64, 1), ([70], [1000], 64, 9, 3, 72, 72, 129), ([300], [300], 32, 2, 1, 128, 128, 0),
    ([1] * 40, list(range(1, 400, 10)), 16, 4, 1, 64, 64, 0), ([3], [50], 16, 2, 2, 256, 200, 0), ([257, 1, 31], [700, 700, 31], 64, 8, 1, 128, 128, 200),
    ([1, 1], [9000, 3], 256, 16, 1, 128, 128, 0), ([40], [6000], 128, 32, 8, 64, 128, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(K, dtype, shape):
    new, lengths, page, heads, kv, d, dv, window = shape
    s = pool(dtype, new, lengths, page, heads, kv, d, dv, pad=8 * (page == 16))
    check(K, s, dtype, window=window)
    # sharper scores, a gate, and the bound on the rows of a sequence given
    check(K, s, dtype, scale=2.0 * d ** -0.5, window=window, gate=rnd((sum(new), heads, dv), dtype, 9), out_scale=0.7, max_tokens=max(new))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,length", [([1], [0]), ([5], [3]), ([40, 2], [7, 0]), ([200], [130])])
def test_rows_that_see_nothing_are_zero(K, dtype, new, length):
    s = pool(dtype, new, length, 16, 4, 2, 64, 64, fill=0.0)
    got = check(K, s, dtype)
    for b, (n, m) in enumerate(zip(new, length)):
        assert (got[sum(new[:b]):sum(new[:b]) + max(0, n - m)] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,window", [(1, 20), (4, 20), (90, 33), (300, 0)])
def test_what_masked_places_hold_has_no_part(K, dtype, bad, new, window):
    """keys and values that are infinite or NaN at a position that some rows see and others do not"""
    length = 310
    s = pool(dtype, [new], [length], 16, 4, 2, 64, 64)
    want = check(K, s, dtype, window=window)
    at = length - new // 2 - 1 if new > 1 else length - window - 1          # seen by the rows from there on, or by none
    page, line = s["host"][0][0][at // 16], at % 16
    for what in ("k", "v"):
        kept = s[what][page, line].clone()
        s[what][page, line] = bad
        got = np64(attend(K, s, dtype, 64 ** -0.5, window))
        s[what][page, line] = kept
        i = np.arange(length - new, length)
        blind = (i < at) | ((i - at >= window) if window else np.zeros(new, bool))
        assert blind.any() and np.isfinite(got[blind]).all()
        # the rows that do not see it, within the rounding of either run
        assert np.abs(got - want)[blind].max() <= 4 * HALF[dtype] * (np.abs(want).max() + 4.0) + (2e-5 if dtype == "float32" else 0)
        if what == "v" and not blind.all():
            assert not np.isfinite(got[~blind]).any()
    K.device_status(sync=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_without_a_finite_maximum(K, dtype):
    """every visible score -infinity gives NaN, as the formula does; one finite score among them takes all the weight"""
    s = pool(dtype, [1], [40], 16, 2, 1, 64, 64)
    s["q"][:] = 1.0
    s["k"].copy_(torch.full_like(s["k"], -1.0))
    s["k"][..., 0] = -float("inf")
    assert torch.isnan(attend(K, s, dtype, 0.125)).all()
    table = s["host"][0]
    s["k"][table[0][1], 3] = 0.0
    out = attend(K, s, dtype, 0.125)
    assert torch.equal(out, s["v"][table[0][1], 3, 0].expand_as(out))


# ---- heads into pages --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["pairs", "half"])
@pytest.mark.parametrize("new,lengths,page,heads,kv,d,dv,pairs", [
    ([1], [1], 8, 1, 1, 8, 8, 4), ([1, 1], [30, 7], 16, 5, 1, 64, 64, 16), ([3, 0, 9], [40, 5, 9], 8, 4, 2, 48, 24, 7),
    ([200], [333], 64, 8, 4, 128, 128, 64), ([2], [9], 32, 3, 3, 256, 8, 40), ([33, 1], [33, 65], 1024, 16, 2, 24, 40, 0)])
def test_heads_into_pages(K, dtype, layout, new, lengths, page, heads, kv, d, dv, pairs):
    s = pool(dtype, new, lengths, page, heads, kv, d, dv, fill=3.0, pad=16)
    n = sum(new)
    k, v = rnd((n, kv, d), dtype, 5), rnd((n, kv, dv), dtype, 6)
    angles = torch.outer(torch.arange(max(lengths) - 1).double(), 0.37 ** torch.arange(pairs).double())
    cos_sin = torch.stack((angles.cos(), angles.sin()), -1).float().cuda()      # one position fewer than the longest holds
    before, q_out = np64(s["k"]), torch.empty_like(s["q"])
    beforev = np64(s["v"])
    K.write_pages(k, v, s["k"], s["v"], s["table"], s["rows"], s["lengths"], q=s["q"], q_out=q_out, cos_sin=cos_sin, layout=layout)
    K.device_status(sync=True)
    wk, wv, wq = before, beforev, np64(s["q"])
    table, rows, _ = s["host"]
    cs = np64(cos_sin)
    for b, length in enumerate(lengths):
        for t in range(new[b]):
            i, r = length - new[b] + t, rows[b] + t
            turn = (lambda x: fo.turned(x, cs[i], layout)) if i < len(cs) else (lambda x: x)
            for g in range(kv):
                wk[table[b, i // page], i % page, g] = turn(np64(k)[r, g])
                wv[table[b, i // page], i % page, g] = np64(v)[r, g]
            for h in range(heads):
                wq[r, h] = turn(wq[r, h])
    # two products and their sum in 32 bits, one rounding
    for got, want, x in ((s["k"], wk, k), (q_out, wq, s["q"])):
        assert (np.abs(np64(got) - want) <= HALF[dtype] * np.abs(want) + 3 * 2.0 ** -24 * 2 * float(x.abs().max())).all()
    assert np.array_equal(np64(s["v"]), wv)
    # in place, and without queries or angles
    q2 = s["q"].clone()
    K.write_pages(k, v, s["k"], s["v"], s["table"], s["rows"], s["lengths"], q=q2, q_out=q2, cos_sin=cos_sin, layout=layout)
    assert torch.equal(q2, q_out)
    K.write_pages(k, v, s["k"], s["v"], s["table"], s["rows"], s["lengths"])
    for b, length in enumerate(lengths):
        if new[b]:
            i = length - 1
            assert torch.equal(s["k"][table[b, i // page], i % page], k[rows[b + 1] - 1])


# ---- copies ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layers,pages,page,width,moves,positions", [
    (1, 2, 8, 8, 1, None), (3, 40, 16, 24, 20, 5), (40, 9, 8, 8, 3, 8), (1, 900, 8, 16, 450, 7), (2, 7, 64, 4104, 3, 63), (2, 5, 16, 8, 2, 0)])
def test_copies_of_pages(K, layers, pages, page, width, moves, positions):
    g = np.random.default_rng(pages)
    # buffers of two formats, the second a part of a larger one
    bufs = [rnd((pages, page, width), DTYPES[i % 2], i) for i in range(layers - 1)] + [rnd((pages, 2, page, width), "bfloat16", 99)[:, 1]]
    order = g.permutation(pages).tolist()
    source, target = order[:moves], order[moves:2 * moves]
    if moves > 2:
        source[1] = source[0]                            # a page copied twice
    want = [b.clone() for b in bufs]
    n = page if positions is None else positions
    for w, b in zip(want, bufs):
        for s, t in zip(source, target):
            w[t, :n] = b[s, :n]
    K.copy_pages(bufs, source, target, positions=positions)
    for w, b in zip(want, bufs):
        assert torch.equal(w, b)


# ---- sampling ----------------------------------------------------------------------------------------------------
def sample_both(K, logits, u, **kw):
    got = K.sample(logits, u, **kw).cpu().tolist()
    l, r = np64(logits), np64(u)
    at = lambda x, i: float(x[i]) if isinstance(x, torch.Tensor) else x
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    full.update(kw)
    full = {k: (v.cpu().to(torch.float64) if isinstance(v, torch.Tensor) else float(np.float32(v)) if k != "top_k" else v) for k, v in full.items()}
    want = [fo.sample(l[i], r[i], at(full["temperature"], i), int(at(full["top_k"], i)), at(full["top_p"], i), at(full["min_p"], i))
            for i in range(len(l))]
    return got, want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (40, 1000), (7, 32768), (2, 129280), (160, 513), (3, 262144), (300, 40)])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.0), dict(temperature=0.6, top_k=20), dict(top_p=0.9), dict(min_p=0.05, temperature=1.7),
                                dict(temperature=0.8, top_k=50, top_p=0.7, min_p=0.02), dict(top_k=1), dict(top_p=0.0), dict(temperature=30.0, top_p=0.5)],
                         ids=str)
def test_sampling(K, dtype, rows, vocab, kw):
    logits = rnd((rows, vocab), dtype, vocab, 2.0)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(rows)).cuda()
    got, want = sample_both(K, logits, u, **kw)
    assert got == want


@pytest.mark.parametrize("dtype", DTYPES)
def test_sampling_by_row(K, dtype):
    """settings of their own for every row, rows of a wider tensor, many equal logits"""
    R, V = 200, 2500
    logits = rnd((R, V + 24), dtype, 3, 1.5)[:, 8:8 + V]
    logits[::3] = (logits[::3] * 2).round() / 2
    g = torch.Generator().manual_seed(1)
    f = lambda lo, hi: (torch.rand(R, generator=g) * (hi - lo) + lo).cuda()
    u, t, p, m = f(0, 1), f(0.3, 2.0), f(0.2, 1.1), f(-0.02, 0.1).clamp(min=0)
    k = torch.randint(0, 60, (R,), generator=g, dtype=torch.int32).cuda()
    t[5], k[6], p[7], m[8] = 0.0, V, 1.0, 1.0
    got, want = sample_both(K, logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert got == want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5), dict(temperature=0.0)], ids=str)
def test_sampling_of_odd_logits(K, dtype, kw):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(getattr(torch, dtype)).min
    rows = [[-inf] * 6, [nan] * 6, [nan, -inf, 1.0, 1.0, -inf, 0.5], [low] * 6, [low, low, 0.0, low, low, low], [inf, 1.0, inf, 2.0, nan, inf],
            [0.0, -0.0, 0.0, -0.0, 0.0, 0.0], [3e38, -3e38, 0.0, 3e38, 1.0, 2.0], [1.0] * 6]
    logits = torch.tensor(rows).to(getattr(torch, dtype)).cuda()
    for x in (0.0, 0.3, 0.5, 0.75, 1.0 - 2.0 ** -24):
        got, want = sample_both(K, logits, torch.full((len(rows),), x, device="cuda"), **kw)
        assert got == want and got[:2] == [-1, -1]


def test_every_kept_token_is_met_as_often_as_it_is_likely(K):
    """random numbers over the whole interval: each kept token's stretch of them, to the step of the numbers"""
    V, R = 37, 4096
    l = rnd((1, V), "float32", 8, 2.0)
    u = ((torch.arange(R) + 0.5) / R).cuda()
    got = K.sample(l.expand(R, V).contiguous(), u, temperature=0.9, top_k=12, top_p=0.95).cpu()
    index, w = fo.kept_tokens(np64(l)[0], float(np.float32(0.9)), 12, float(np.float32(0.95)), 0.0)
    share = np.bincount(got, minlength=V) / R
    assert set(got.tolist()) <= set(index.tolist())
    assert np.abs(share[index] - w / w.sum()).max() <= 1.0 / R and (np.diff(got.numpy()) >= 0).all()


# ---- the four together, and a model on pages ---------------------------------------------------------------------
def test_a_run_of_them_together(K):
    """a small decoder of one attention layer: two prompts of unequal lengths, forked, decoded with drawn tokens, compacted on the
    way; every step's attention and every token against plain float64 on the values that the pages should hold"""
    PC = importlib.import_module(PKG + ".paged_cache")
    G, H, d, V, page = 2, 4, 64, 500, 16
    cache = PC.PagedCache([2 * G * d], [0], 8, 128, torch.bfloat16, "cuda", page=page, pages=40)
    buf = cache.buffer(0)
    kp, vp = buf[..., :G * d].unflatten(2, (G, d)), buf[..., G * d:].unflatten(2, (G, d))
    angles = torch.outer(torch.arange(128).double(), 0.6 ** torch.arange(16).double())
    cos_sin = torch.stack((angles.cos(), angles.sin()), -1).float().cuda()
    head = rnd((H * d, V), "float32", 70, 0.7)
    emb = [rnd((V, n, d), "bfloat16", 80 + i) for i, n in enumerate((H, G, G))]
    history = {}                                       # slot -> token ids
    draws = torch.rand(64, generator=torch.Generator().manual_seed(5))

    def step(slots, tokens):
        """tokens of every slot, as many as it brings"""
        new = [len(t) for t in tokens]
        for s, t in zip(slots, tokens):
            cache.extend_all([s], len(history[s]), len(t))
            history[s] = history[s] + t
        rows = torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32).cuda()
        lengths = i32(*[len(history[s]) for s in slots])
        ids = torch.tensor(sum(tokens, [])).cuda()
        q, k, v = (e[ids] for e in emb)
        table = cache.table(slots).cuda()
        K.write_pages(k, v, kp, vp, table, rows, lengths, q=q, q_out=q, cos_sin=cos_sin, layout="half")
        out = torch.empty_like(q)
        K.paged_attention(q, kp, vp, table, rows, lengths, out, d ** -0.5, window=50, max_tokens=max(new))
        logits = (out[(rows[1:] - 1).long()].flatten(1).float() @ head)
        u = draws[:len(slots)].cuda()
        got = K.sample(logits, u, temperature=0.8, top_k=40, top_p=0.95).tolist()
        for i, s in enumerate(slots):
            ids = torch.tensor(history[s])
            turned = lambda e, i0=0: np.stack([[fo.turned(x, np64(cos_sin)[i0 + p], "half") for x in r] for p, r in enumerate(np64(e[ids.cuda()])[i0:])])
            bf = lambda x: torch.from_numpy(x).to(torch.bfloat16).double().numpy()
            kk, vv, qq = bf(turned(emb[1])), np64(emb[2][ids.cuda()]), bf(turned(emb[0], len(ids) - 1))
            pages = lambda x: x[:, None]
            want, size, score = fo.paged_attention(qq, pages(kk), pages(vv), [list(range(len(ids)))], [0, 1], [len(ids)], d ** -0.5, 50)
            mine = np64(out[int(rows[i + 1]) - 1])
            # the pages' own keys are rounded like the plain ones but for ties of the rounding: one step of a key more
            assert (np.abs(mine - want[0]) <= limit("bfloat16", size, score, d, 128)[0] * 3 + HALF["bfloat16"] * np.abs(want[0])).all()
            assert got[i] == fo.sample(np64(logits[i]), float(u[i]), float(np.float32(0.8)), 40, float(np.float32(0.95)))
        return got

    a, b = cache.acquire(), cache.acquire()
    history[a], history[b] = [], []
    g = np.random.default_rng(0)
    first = step([a, b], [g.integers(0, V, 37).tolist(), g.integers(0, V, 5).tolist()])
    slots, tokens = [a, b], list(first)
    for s, t in ((a, first[0]), (a, first[0]), (b, first[1])):
        slots.append(cache.fork(s))
        history[slots[-1]] = list(history[s])
        tokens.append(t)
    for n in range(14):
        tokens = step(slots, [[t] for t in tokens])
        if n == 4:
            gone = slots.pop(1)
            cache.release(gone)
            tokens.pop(1)
        if n == 6:
            assert cache.compact() > 0
    K.device_status(sync=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ["V_ODD", "V_PEAKED", "V_WIDE"])
def test_a_model_on_pages(float_libpath, tmp_path, case, dtype):
    """prompts, portions, recorded steps, forks and compaction against the oracle"""
    import float_cases as fc
    registry = importlib.import_module(PKG + ".registry")
    cfg = getattr(fc, case)
    W = fc.make_weights(cfg, 11)
    model = registry.load(fc.write_checkpoint(str(tmp_path), cfg, W), dtype=dtype, max_seq_len=300, max_batch_size=5, page=16, pages=45)
    rng = np.random.default_rng(5)
    toks = rng.integers(0, cfg["vocab"], 190).tolist()
    t = lambda x: torch.tensor([x])
    first, second = model.begin_batch(1), model.begin_batch(1)
    got = [model.step(t(toks[:70]), 0, first, want=range(70))[0].cpu().numpy()]
    model.step(t(toks[:33]), 0, second, want=[])
    got.append(model.step(t(toks[70:75]), 70, first, want=range(5))[0].cpu().numpy())
    for i in range(75, 90):
        got.append(model.step(t(toks[i:i + 1]), i, first)[0].cpu().numpy())
    model.end_batch(second)
    assert model.cache.compact() > 0
    # forks stand where their source does; each goes on by itself, in one batch, across the end of a page
    slots = model.fork(first, 3)
    tails = [toks[90:130], rng.integers(0, cfg["vocab"], 40).tolist(), rng.integers(0, cfg["vocab"], 40).tolist()]
    parts = [[], [], []]
    for i in range(40):
        l = model.step(torch.tensor([[x[i]] for x in tails]), 90 + i, slots)[0].cpu().numpy()
        for p, row in zip(parts, l):
            p.append(row[None])
    want = fc.Expected(cfg, W, toks[:130])
    assert want.ok(np.concatenate(got + parts[0]), dtype)
    for x, p in zip(tails[1:], parts[1:]):
        assert fc.Expected(cfg, W, toks[:90] + x).ok(np.concatenate(p), dtype, range(90, 130))
    model.end_batch(slots)
    assert model.cache.free_pages() == 45 and model.cache.free_slots() == 5
    importlib.import_module(PKG + ".float_kernel").device_status(sync=True)


def test_designs_with_latents_stay_in_slots(float_libpath, tmp_path):
    import float_cases as fc
    registry = importlib.import_module(PKG + ".registry")
    path = fc.write_checkpoint(str(tmp_path), fc.ODD, fc.make_weights(fc.ODD, 11))
    with pytest.raises(NotImplementedError):
        registry.load(path, page=16)


@pytest.mark.parametrize("case,page", [("V_PEAKED", 16), ("V_PEAKED", 0), ("PEAKED", 0)])
def test_completions_of_a_prompt(float_libpath, tmp_path, case, page):
    """several greedy completions are the single one's; drawn ones repeat with their seed and follow the oracle's kept tokens"""
    import float_cases as fc
    registry, gen = (importlib.import_module(PKG + "." + n) for n in ("registry", "generate"))
    Sampler = importlib.import_module(PKG + ".sampling").Sampler
    cfg = getattr(fc, case)
    W = fc.make_weights(cfg, 11)
    model = registry.load(fc.write_checkpoint(str(tmp_path), cfg, W), dtype="float32", max_seq_len=200, max_batch_size=6, page=page)
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, cfg["vocab"], n).tolist() for n in (41, 30)]
    alone = [gen.generate(model, [p], 8, -1, temperature=0.0)[0] for p in prompts]
    assert gen.generate(model, prompts, 8, -1, temperature=0.0, samples=3) == [alone[0]] * 3 + [alone[1]] * 3
    draw = lambda seed: gen.generate(model, prompts[:1], 8, -1, sampler=Sampler(1.3, top_k=5, seed=seed), samples=4)
    out, alike = draw(1), 1.0
    assert out == draw(1)
    for x in out:
        logits = fc.oracle_logits(cfg, W, prompts[0] + x)[len(prompts[0]) - 1:-1]
        for l, token in zip(logits, x):
            w = fo.kept_tokens(l, 1.3, 5, 1.0, 0.0)[1]
            alike *= w.max() / w.sum()
            # among the five largest, or so near to the fifth that 32 bits decide
            assert l[token] >= np.sort(l)[-5] - 1e-3 * l.std()
    # completions and seeds agree about as often as the likeliest token is drawn every time: where that is one in a million, they differ
    assert alike > 1e-6 or (out != draw(2) and len({tuple(x) for x in out}) > 1)
    assert model.cache.free_slots() == 6


def test_the_program_draws_tokens_on_pages(float_libpath, tmp_path, capsys):
    import json
    import float_cases as fc
    gen = importlib.import_module(PKG + ".generate")
    path = fc.write_checkpoint(str(tmp_path), fc.V_PEAKED, fc.make_weights(fc.V_PEAKED, 11))
    args = ["--model", path, "--tokens", "3,1,4,1,5", "--max-new-tokens", "6", "--max-seq-len", "64", "--dtype", "float32", "--samples", "3"]
    lines = []
    for more in (["--sample", "--top-k", "7", "--seed", "3", "--page", "8"], ["--sample", "--top-k", "7", "--seed", "3"], []):
        assert gen.main(args + more) == 0
        lines.append([json.loads(x) for x in capsys.readouterr().out.splitlines()])
        assert [len(x) for x in lines[-1]] == [6] * 3
    assert lines[0] == lines[1] and lines[2][0] == lines[2][1] == lines[2][2]


# ---- calls that the documentation allows -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_captured_calls_follow_their_inputs(K, dtype, new):
    """one graph of write, attention and sampling; rows, lengths, table and values change between replays; a second graph of the same
    calls in between"""
    B, page, H, G, d = 3, 16, 4, 2, 64
    a, b = (pool(dtype, [new] * B, lengths, page, H, G, d, d, seed=s) for s, lengths in ((1, [200, 90, 64]), (2, [41, 230, 77])))
    cols = max(a["table"].shape[1], b["table"].shape[1])
    pages = max(a["k"].shape[0], b["k"].shape[0])
    st = dict(q=a["q"].clone(), table=torch.zeros(B, cols, dtype=torch.int32, device="cuda"), rows=a["rows"].clone(), lengths=a["lengths"].clone(),
              pool=torch.zeros(pages, page, 2 * G * d, dtype=a["q"].dtype, device="cuda"), out=torch.empty_like(a["q"]),
              u=torch.rand(B * new, device="cuda"), token=torch.empty(B * new, dtype=torch.int64, device="cuda"), nk=rnd((B * new, G, d), dtype, 7))
    kp, vp = st["pool"][..., :G * d].unflatten(2, (G, d)), st["pool"][..., G * d:].unflatten(2, (G, d))

    def put(s):
        st["q"].copy_(s["q"])
        st["table"][:, :s["table"].shape[1]].copy_(s["table"])
        st["rows"].copy_(s["rows"])
        st["lengths"].copy_(s["lengths"])
        kp[:s["k"].shape[0]].copy_(s["k"].nan_to_num(0.0))
        vp[:s["v"].shape[0]].copy_(s["v"].nan_to_num(0.0))

    def calls():
        K.write_pages(st["nk"], st["nk"], kp, vp, st["table"], st["rows"], st["lengths"])
        K.paged_attention(st["q"], kp, vp, st["table"], st["rows"], st["lengths"], st["out"], 0.1, window=120, max_tokens=new)
        K.sample(st["out"].flatten(1), st["u"], st["token"], temperature=0.7, top_k=30, top_p=0.9)

    def plain(s):
        put(s)
        calls()
        return st["out"].clone(), st["token"].clone()

    want = [plain(s) for s in (a, b)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            calls()
    for i in (0, 1, 0):
        for g in graphs:
            put((a, b)[i])
            st["out"].zero_()
            st["token"].zero_()
            g.replay()
            # the same bits: nothing depends on the timing of a run
            assert torch.equal(st["out"], want[i][0]) and torch.equal(st["token"], want[i][1])
    K.device_status(sync=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_at_once_on_streams_of_their_own(K, dtype):
    s = [pool(dtype, [1 + 60 * (i % 2)] * 2, [700, 300], 32, 8, 2, 64, 64, seed=i, fill=0.0) for i in range(4)]
    logits = [rnd((40, 5000), dtype, i, 2.0) for i in range(4)]
    u = torch.rand(40, generator=torch.Generator().manual_seed(3)).cuda()
    want = [(attend(K, x, dtype, 0.1).clone(), K.sample(l, u, top_p=0.9)) for x, l in zip(s, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in s]
    for _ in range(5):
        got = []
        for x, l, stream in zip(s, logits, streams):
            with torch.cuda.stream(stream):
                got.append((attend_quietly(K, x, dtype), K.sample(l, u, top_p=0.9)))
        torch.cuda.synchronize()
        for (o, t), (wo, wt) in zip(got, want):
            assert torch.equal(o, wo) and torch.equal(t, wt)


def attend_quietly(K, s, dtype):
    """attend without its host checks, which wait"""
    out = torch.empty(s["q"].shape[:2] + s["v"].shape[3:], dtype=s["q"].dtype, device="cuda")
    return K.paged_attention(s["q"], s["k"], s["v"], s["table"], s["rows"], s["lengths"], out, 0.1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 3, 80])
def test_strided_heads(K, dtype, new):
    """queries, gate and result as parts of wider rows, in another order of heads and tokens"""
    s = pool(dtype, [new, 2], [150, 40], 16, 6, 3, 40, 24, fill=0.0, pad=24)
    n, gate = new + 2, rnd((new + 2, 6, 24), dtype, 9)
    want = attend(K, s, dtype, 0.2, 33, gate, 0.9)
    wide = rnd((n, 6 * 40 + 6 * 24 + 16), dtype, 4)
    q, g = wide[:, :240].unflatten(1, (6, 40)), wide[:, 240:384].unflatten(1, (6, 24))
    q.copy_(s["q"])
    g.copy_(gate)
    out = torch.zeros(6, n, 32, dtype=q.dtype, device="cuda").transpose(0, 1)[..., :24]         # heads first
    K.paged_attention(q, s["k"], s["v"], s["table"], s["rows"], s["lengths"], out, 0.2, window=33, gate=g, out_scale=0.9, max_tokens=new)
    assert torch.equal(out, attend(K, s, dtype, 0.2, 33, gate, 0.9, max_tokens=new))
    assert (out.double() - want.double()).abs().max() <= 6 * HALF[dtype] * float(want.abs().max()) + 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_beyond_32_bit_offsets(K, dtype):
    """the last pages of a pool of more than 2^32 bytes, and of 2^31 elements"""
    G, d, page, pages = 8, 128, 64, 16500
    small = pool(dtype, [2, 70], [100, 70], page, 16, G, d, d, fill=0.0)
    big = torch.empty(pages, page, 2 * G * d, dtype=getattr(torch, dtype), device="cuda")
    assert big.numel() > 2 ** 31 and big.numel() * big.element_size() > 2 ** 32
    n = small["k"].shape[0]
    kp, vp = big[..., :G * d].unflatten(2, (G, d)), big[..., G * d:].unflatten(2, (G, d))
    kp[-n:], vp[-n:] = small["k"], small["v"]
    table = torch.where(small["table"] >= 0, small["table"] + (pages - n), small["table"])
    for kw in (dict(max_tokens=1), dict()):
        out, want = torch.empty_like(small["q"]), torch.empty_like(small["q"])
        K.paged_attention(small["q"], kp, vp, table, small["rows"], small["lengths"], out, 0.09, **kw)
        K.paged_attention(small["q"], small["k"], small["v"], small["table"], small["rows"], small["lengths"], want, 0.09, **kw)
        assert torch.equal(out, want)
    new = rnd((72, G, d), dtype, 5)
    K.write_pages(new, new, kp, vp, table, small["rows"], small["lengths"])
    last = small["host"][0][1][1] + pages - n
    assert torch.equal(kp[last, 5], new[-1]) and torch.equal(vp[last, 5], new[-1])
    K.copy_pages([big], [int(last)], [7])
    assert torch.equal(big[7], big[int(last)])
    K.device_status(sync=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,heads,kv", [(1024, 2, 1), (1, 130, 1), (2, 128, 1), (300, 12, 12)])
def test_many_sequences_and_many_heads_of_a_group(K, dtype, batch, heads, kv):
    g = np.random.default_rng(batch)
    lengths = g.integers(1, 30, batch).tolist()
    for new in ([1] * batch, [min(n, int(k)) for n, k in zip(lengths, g.integers(0, 4, batch))]):
        check(K, pool(dtype, new, lengths, 8, heads, kv, 16, 16, fill=0.0), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_what_does_not_fit_is_reported(K, dtype, new):
    """page numbers outside the pool, more positions than the table has columns for, rows outside the batch: nothing of it is read or
    written, the other sequences come out right, and the status says so"""
    s = pool(dtype, [new, new, new], [100, 90, 60], 16, 4, 2, 64, 64, fill=0.0)
    want = attend(K, s, dtype, 0.1)
    K.device_status(sync=True)

    def wrong(name, edit, whole):
        kept = s[name].clone()
        edit(s[name])
        out = attend(K, s, dtype, 0.1)
        torch.cuda.synchronize()
        with pytest.raises(K.FloatOpsError):
            K.device_status(sync=True)
        for b in whole:                        # other lengths are cut elsewhere, so that sums come in another order
            mine = (out - want)[b * new:(b + 1) * new].double().abs().max()
            assert mine <= 4 * HALF[dtype] * float(want.abs().max()) + 1e-5
        before = s["k"].clone()
        K.write_pages(torch.ones_like(s["q"][:, :2]), torch.ones_like(s["q"][:, :2]), s["k"], s["v"], s["table"], s["rows"], s["lengths"])
        torch.cuda.synchronize()
        s["k"].copy_(before)
        try:
            K.device_status(sync=True)
        except K.FloatOpsError:
            pass
        s[name].copy_(kept)

    def page(value):
        def edit(t):
            t[1, 3] = value
        return edit
    values = s["v"].clone()
    for value in (-1, s["k"].shape[0], 2 ** 31 - 1, -2 ** 31):
        wrong("table", page(value), [0, 2])
        s["v"].copy_(values)
    for value in (16 * s["table"].shape[1] + 1, 2 ** 31 - 1, -5, -2 ** 31):
        wrong("lengths", lambda t: t[1:2].fill_(value), [0, 2])
        s["v"].copy_(values)
    wrong("rows", lambda t: t[3:].fill_(3 * new + 50), [0, 1])
    s["v"].copy_(values)
    wrong("rows", lambda t: t[2:3].fill_(-7), [0])
    s["v"].copy_(values)
    wrong("rows", lambda t: t[1:2].fill_(2 ** 31 - 1), [2])
    s["v"].copy_(values)
    assert torch.equal(attend(K, s, dtype, 0.1), want)
    K.device_status(sync=True)


def test_sampling_takes_any_number(K):
    """random numbers outside [0, 1) and settings that no row should have name a kept token all the same"""
    l = rnd((1, 300), "float32", 2, 2.0)
    kept = set(fo.kept_tokens(np64(l)[0], 1.0, 5, 1.0, 0.0)[0].tolist())
    for u in (1.0, -1.0, 7.0, float("nan"), float("inf"), -float("inf")):
        assert int(K.sample(l, torch.tensor([u], device="cuda"), top_k=5)) in kept
    f = lambda x: torch.tensor([x], dtype=torch.float32, device="cuda")
    best = int(l.argmax())
    half = f(0.5)
    assert int(K.sample(l, half, temperature=f(float("nan")))) == best and int(K.sample(l, half, temperature=f(-1.0))) == best
    assert int(K.sample(l, half, temperature=f(1e-30))) == best and int(K.sample(l, half, min_p=f(5.0))) == best
    assert int(K.sample(l, half, top_k=torch.tensor([-3], dtype=torch.int32, device="cuda"))) == fo.sample(np64(l)[0], 0.5)
    assert int(K.sample(l, half, temperature=float("inf"))) == 150 and int(K.sample(l, half, top_p=f(float("nan")))) == fo.sample(np64(l)[0], 0.5)


def test_calls_refuse_what_does_not_belong_together(K):
    s = pool("bfloat16", [2, 1], [30, 9], 16, 4, 2, 64, 64, fill=0.0)
    q, out, half = s["q"], torch.empty_like(s["q"]), s["q"].half()
    base = dict(q=q, k_pages=s["k"], v_pages=s["v"], table=s["table"], rows=s["rows"], lengths=s["lengths"], out=out, scale=0.1)
    K.paged_attention(**base)
    for bad in (dict(q=half), dict(q=q.float()), dict(out=out.float()), dict(q=q[:, :3]), dict(q=q[:2]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(out=q),
                dict(table=s["table"].long()), dict(table=s["table"][0]), dict(rows=s["rows"][:2]), dict(lengths=s["lengths"][:1]), dict(scale=-0.1),
                dict(window=-1), dict(max_tokens=-1), dict(k_pages=s["k"][:, :12]), dict(v_pages=s["v"][:, :8]), dict(v_pages=s["v"].float()),
                dict(gate=q[..., :32]), dict(q=torch.empty(3, 4, 68, device="cuda", dtype=q.dtype)[..., 4:]), dict(k_pages=s["k"][:0], v_pages=s["v"][:0]),
                dict(table=s["table"].t().contiguous().t()), dict(q=[1.0])):
        with pytest.raises(ValueError):
            K.paged_attention(**{**base, **bad})
    with pytest.raises(K.FloatOpsError):
        big = torch.zeros(2, 16, 1, 264, dtype=q.dtype, device="cuda")
        x = torch.zeros(3, 1, 264, dtype=q.dtype, device="cuda")
        K.paged_attention(x, big, big, s["table"], s["rows"], s["lengths"], torch.empty_like(x), 0.1)
    k, cs = rnd((3, 2, 64), "bfloat16"), torch.zeros(9, 32, 2, device="cuda")
    base = dict(k=k, v=k, k_pages=s["k"], v_pages=s["v"], table=s["table"], rows=s["rows"], lengths=s["lengths"], q=q, q_out=out, cos_sin=cs)
    K.write_pages(**base)
    for bad in (dict(k=k[:2]), dict(v=k[:, :1]), dict(q=None), dict(q_out=None), dict(q=q[:2]), dict(q_out=out[:, :2]), dict(layout="other"),
                dict(cos_sin=cs.double()), dict(cos_sin=cs[..., :1]), dict(cos_sin=torch.zeros(9, 33, 2, device="cuda")), dict(cos_sin=cs[:, ::2]), dict(k=k.float())):
        with pytest.raises(ValueError):
            K.write_pages(**{**base, **bad})
    b = torch.zeros(6, 16, 8, dtype=q.dtype, device="cuda")
    for bufs, src, dst, n in (([b], [0], [6], None), ([b], [0], [-1], None), ([b], [6], [0], None), ([b], [0], [1], 17), ([b], [0], [1], -1), ([b.cpu()], [0], [1], None),
                              ([b[:, :, :4]], [0], [1], None), ([b[0, 0]], [0], [1], None), ([b[:1].expand(6, 16, 8)], [0], [1], None), ([b, b[:3]], [0], [5], None),
                              ([torch.zeros(6, 16, 9, device="cuda", dtype=q.dtype)], [0], [1], 1)):
        with pytest.raises(ValueError):
            K.copy_pages(bufs, src, dst, positions=n)
    for src, dst in (([0, 1], [2, 2]), ([0, 2], [2, 3])):
        with pytest.raises(K.FloatOpsError):
            K.copy_pages([b], src, dst)
    l, u = rnd((3, 50), "float32"), torch.zeros(3, device="cuda")
    for bad in (dict(random=u[:2]), dict(random=u.double()), dict(logits=l.double()), dict(logits=l.t()), dict(logits=l[0]), dict(out=u), dict(temperature=-1.0),
                dict(top_k=1.5), dict(top_k=torch.zeros(3, device="cuda")), dict(top_p=torch.zeros(2, device="cuda")), dict(min_p=float("nan")),
                dict(random=torch.zeros(6, device="cuda")[::2])):
        with pytest.raises(ValueError):
            K.sample(**{**dict(logits=l, random=u), **bad})
    # nothing to do
    none = torch.empty(0, 4, 64, dtype=q.dtype, device="cuda")
    assert K.paged_attention(none, s["k"], s["v"], s["table"], s["rows"], s["lengths"], none.clone(), 0.1).shape == (0, 4, 64)
    assert K.sample(l[:0], u[:0]).shape == (0,)
    K.device_status(sync=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,lengths", [([5], [3]), ([40, 2], [7, 0]), ([200], [130]), ([1, 70], [90, 300])])
def test_a_window_of_any_size(K, dtype, new, lengths):
    """windows as long as the cache and longer, up to beyond 32 bits, see what no window sees, rows at negative positions among them"""
    s = pool(dtype, new, lengths, 16, 4, 2, 64, 64, fill=0.0)
    want = attend(K, s, dtype, 0.1)
    for window in (max(lengths), 2 ** 31 - 1, 2 ** 40):
        assert torch.equal(attend(K, s, dtype, 0.1, window), want)
    check(K, s, dtype, 0.1, 2 ** 31 - 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 2, 90])
def test_expanded_heads(K, dtype, new):
    """keys and values that all heads share, queries that all tokens or all heads share, none of them copied"""
    s = pool(dtype, [new, 1], [150, 40], 16, 4, 2, 64, 64, fill=0.0)
    s["k"], s["v"] = s["k"][:, :, :1].expand(-1, -1, 2, -1), s["v"][:, :, :1].expand(-1, -1, 2, -1)
    check(K, s, dtype)
    s = pool(dtype, [new, 1], [150, 40], 16, 4, 2, 64, 64, seed=3, fill=0.0)
    table, rows, lengths = s["host"]
    for q in (s["q"][:1].expand(new + 1, -1, -1), s["q"][:, :1].expand(-1, 4, -1)):
        out = K.paged_attention(q, s["k"], s["v"], s["table"], s["rows"], s["lengths"], torch.empty_like(s["q"]), 0.125)
        want, size, score = fo.paged_attention(np64(q), np64(s["k"]), np64(s["v"]), table, rows, lengths, 0.125)
        assert (np.abs(np64(out) - want) <= limit(dtype, size, score, 64, 150) + HALF[dtype] * np.abs(want)).all()
    q = s["q"]
    with pytest.raises(ValueError):
        K.paged_attention(q, s["k"], s["v"], s["table"], s["rows"], s["lengths"], q[:, :1].clone().expand(-1, 4, -1), 0.125)
    new_k = q[:, :2].contiguous()
    for bad in (dict(k_pages=s["k"][:, :, :1].expand(-1, -1, 2, -1)), dict(v_pages=s["v"][:1].expand(s["v"].shape)),
                dict(q_out=q[:, :1].clone().expand(-1, 4, -1))):
        with pytest.raises(ValueError):
            K.write_pages(**{**dict(k=new_k, v=new_k, k_pages=s["k"], v_pages=s["v"], table=s["table"], rows=s["rows"], lengths=s["lengths"], q=q, q_out=q), **bad})
    K.device_status(sync=True)


@pytest.mark.parametrize("rows,lengths", [([0, 3, 9], [20, 20]), ([-2, 3, 6], [20, 20]), ([0, 3, 6], [-1, 20])])
def test_rows_that_do_not_fit_are_reported_when_written(K, rows, lengths):
    s = pool("float32", [3, 3], [20, 20], 16, 2, 2, 32, 32, fill=0.0)
    before, x = s["k"].clone(), torch.ones(6, 2, 32, device="cuda")
    K.write_pages(x, x, s["k"], s["v"], s["table"], i32(*rows), i32(*lengths))
    torch.cuda.synchronize()
    with pytest.raises(K.FloatOpsError):
        K.device_status(sync=True)
    # the sequence that fits is written, the other one is not
    b = 0 if rows[2] == 9 else 1
    table = s["host"][0]
    page = int(table[b][1])
    assert (s["k"][page, 1:4] == 1).all()
    s["k"][page, 1:4] = before[page, 1:4]
    assert torch.equal(s["k"], before)


def test_the_path_of_a_call_without_heads(K):
    import ctypes
    a = K.PagedAttentionArgs()
    assert K.paged_path(ctypes.byref(a)) == 0


def test_calls_hold_on_to_nothing(K):
    """no tensor, page list or result is held by a call that is over"""
    import sys
    s = pool("bfloat16", [2, 1], [30, 9], 16, 4, 2, 64, 64, fill=0.0)
    out, k, cs, u = torch.empty_like(s["q"]), rnd((3, 2, 64), "bfloat16"), torch.zeros(40, 32, 2, device="cuda"), torch.zeros(3, device="cuda")
    l, source = rnd((3, 50), "float32"), [0]
    whole_k, whole_v = s["k"].contiguous(), s["v"].contiguous()
    watched = [s["q"], s["k"], s["v"], s["table"], s["rows"], s["lengths"], out, k, cs, u, l, whole_k, whole_v, source, torch.bfloat16, torch.float32, torch.int32]

    def calls():
        pages = s["k"], s["v"], s["table"], s["rows"], s["lengths"]
        K.paged_attention(s["q"], *pages, out, 0.1, gate=s["q"])
        K.write_pages(k, k, *pages, q=s["q"], q_out=out, cos_sin=cs)
        K.copy_pages([whole_k, whole_v], source, [1])
        K.sample(l, u, temperature=u, top_k=3)
        for bad in (lambda: K.paged_attention(s["q"], *pages, s["q"], 0.1), lambda: K.write_pages(k, k, *pages, q=s["q"]), lambda: K.copy_pages([whole_k, l], source, [90]),
                    lambda: K.sample(l, u, out=u)):
            with pytest.raises(ValueError):
                bad()
    calls()
    before, held = [sys.getrefcount(x) for x in watched], torch.cuda.memory_allocated()
    for _ in range(20):
        calls()
    after = [sys.getrefcount(x) for x in watched]
    # dtypes are referred to by whatever else is alive
    assert after[:-3] == before[:-3] and all(abs(a - b) < 20 for a, b in zip(after[-3:], before[-3:]))
    assert torch.cuda.memory_allocated() == held
    K.device_status(sync=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", list(range(1, 10)))
def test_every_number_of_few_rows(K, dtype, new):
    """three to 27 rows a key head, beside sequences with fewer, over stretches of keys that end in every way"""
    s = pool(dtype, [new, 1, new, max(new - 1, 0)], [new, 16 * new + 1, 400 + new, 129], 8, 6, 2, 40, 136 if new == 3 else 24)
    check(K, s, dtype, window=0 if new % 2 else 37, max_tokens=new)
    check(K, s, dtype, scale=1.0, window=100, max_tokens=1)


def test_tensors_that_require_gradients_are_read_all_the_same(K):
    s = pool("bfloat16", [2, 1], [30, 9], 16, 4, 2, 64, 64, fill=0.0)
    want = attend_quietly(K, s, "bfloat16")
    s["q"] = torch.nn.Parameter(s["q"])
    with torch.no_grad():
        assert torch.equal(attend_quietly(K, s, "bfloat16"), want)
    l, u = rnd((3, 50), "float32"), torch.full((3,), 0.4, device="cuda")
    assert torch.equal(K.sample(torch.nn.Parameter(l), u), K.sample(l, u))
    half = torch.arange(96, device="cuda", dtype=torch.float16).reshape(3, 2, 16)                # a type that no other call takes
    K.copy_pages([half], [0], [2])
    assert torch.equal(half[2], half[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_bound_on_rows_of_any_size(K, dtype):
    """and one that is too low, for tiles of rows that several CTAs take parts of"""
    s = pool(dtype, [90, 3], [2000, 700], 32, 16, 2, 64, 48, fill=0.0)
    for bound in (0, 1, 7, 90, 2 ** 31, 2 ** 62, 2 ** 70):
        check(K, s, dtype, max_tokens=bound)
