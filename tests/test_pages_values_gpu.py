"""Values that calls over pages meet rarely: scores that jump from one tile of keys to the next, keys that are NaN or infinite where a
row does see them, what lies behind the end of a sequence, infinities and NaN among heads that do not turn, the status of
what does not fit, and the bound on rows that is left out."""
import numpy as np
import pytest
import torch

from oracle import float_oracle as fo
from test_pages_gpu import DTYPES, HALF, K, attend, check, i32, limit, np64, pool, rnd  # noqa: F401 (K is a fixture)

pytestmark = pytest.mark.gpu
LN2 = float(np.float32(np.log(2.0)))                   # with it as scale, scores count in powers of two


# ---- jumps of the scores -----------------------------------------------------------------------------------------
TILE, LENGTH = 128, 400                                # keys of a tile; three tiles and a part of a fourth
LEVELS = {  # power of two that the keys of a position start from
    "many keys": lambda j, jump: jump if TILE <= j < 2 * TILE else 0,
    "one key": lambda j, jump: jump if j == 200 else 0,
    "last tile": lambda j, jump: jump if j >= 3 * TILE else 0,
    "one key of the last tile": lambda j, jump: jump if j == 3 * TILE else 0,
    "from there on": lambda j, jump: jump if j >= TILE else 0,
    "one key, a little less behind it": lambda j, jump: jump if j == 200 else jump - 4 if j >= 2 * TILE else 0,
    "up and up": lambda j, jump: j // TILE * jump,
}


def jumping(dtype, new, levels, jump, sequences, seed=0):
    """`sequences` times the same sequence, over the same pages"""
    s = pool(dtype, [new], [LENGTH], 16, 2, 1, 64, 64, seed=seed)
    table = s["host"][0][0]
    s["q"].zero_()
    s["q"][..., :2] = 1.0
    k = torch.zeros(LENGTH, 64)
    k[:, 0] = torch.tensor([float(levels(j, jump)) for j in range(LENGTH)])
    k[:, 1] = torch.rand(LENGTH, generator=torch.Generator().manual_seed(seed)) * 2 - 1
    j = torch.arange(LENGTH)
    pages, lines = torch.from_numpy(table)[j // 16].long().cuda(), (j % 16).cuda()
    s["k"][pages, lines, 0] = k.to(s["k"].dtype).cuda()
    s["v"][pages, lines, 0] = rnd((LENGTH, 64), dtype, seed + 5, 0.01)
    s["one"] = (s["q"], s["host"])
    s["q"] = s["q"].repeat(sequences, 1, 1)
    s["table"] = s["table"].repeat(sequences, 1)
    s["rows"] = torch.arange(sequences + 1, dtype=torch.int32, device="cuda") * new
    s["lengths"] = i32(*[LENGTH] * sequences)
    return s


def check_jumps(K, s, dtype, new, **kw):
    got = np64(attend(K, s, dtype, LN2, **kw))
    K.device_status(sync=True)
    q, (table, rows, lengths) = s["one"]
    want, size, score = fo.paged_attention(np64(q), np64(s["k"]), np64(s["v"]), table, rows, lengths, LN2)
    got = got.reshape((-1,) + want.shape)
    assert np.isfinite(got).all()
    # a score's own rounding, and those of its product with log2(e) and of its difference to the maximum, are counted by `limit`
    off = np.abs(got - want) - limit(dtype, size, score, 64, LENGTH) - HALF[dtype] * np.abs(want)
    assert (off <= 1e-30).all(), float(off.max())


@pytest.mark.parametrize("jump", [9, 60, 99, 101, 115, 121, 124, 126.5, 127.5, 129, 200])
@pytest.mark.parametrize("where", list(LEVELS))
@pytest.mark.parametrize("whole", [False, True])
def test_scores_that_jump(K, whole, where, jump):
    """one sequence, which several CTAs cut, and as many as the GPU has SMs, each of which takes one"""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    s = jumping("bfloat16", 20, LEVELS[where], jump, sms if whole else 1)
    check_jumps(K, s, "bfloat16", 20, max_tokens=20)


@pytest.mark.parametrize("jump", [60, 121, 126.5, 127.5, 129])
@pytest.mark.parametrize("where", list(LEVELS))
@pytest.mark.parametrize("dtype,new", [("bfloat16", 1), ("float32", 1), ("float32", 20)])
def test_scores_that_jump_in_the_other_kernels(K, dtype, new, where, jump):
    check_jumps(K, jumping(dtype, new, LEVELS[where], jump, 1), dtype, new, max_tokens=new)
    check_jumps(K, jumping(dtype, new, LEVELS[where], jump, 3), dtype, new, max_tokens=new)


def test_scores_that_jump_under_a_gate(K):
    s = jumping("bfloat16", 20, LEVELS["last tile"], 125, 148)
    gate = rnd((148 * 20, 2, 64), "bfloat16", 3)
    plain = np64(attend(K, s, "bfloat16", LN2, max_tokens=20))
    got = np64(attend(K, s, "bfloat16", LN2, gate=gate, out_scale=0.7, max_tokens=20))
    want = plain * 0.7 / (1 + np.exp(-np64(gate)))
    # either result is rounded once, and the sigmoid of bfloat16 results is good to more than they are
    assert (np.abs(got - want) <= 4 * HALF["bfloat16"] * np.abs(want) + 1e-30).all()
    K.device_status(sync=True)


# ---- keys that are seen ------------------------------------------------------------------------------------------
ENDS = [17, 33, 49, 65, 97, 129, 193, 257, 385, 641]   # the last position by itself in a warp's stretch, a block or a tile


def spoil(s, lengths, value, element=slice(None)):
    """the newest key of every sequence"""
    for b, n in enumerate(lengths):
        s["k"][s["host"][0][b][(n - 1) // 16], (n - 1) % 16, :, element] = value


@pytest.mark.parametrize("d", [64, 136])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,heads,kv", [(1, 3, 3), (1, 4, 1), (3, 4, 2), (20, 6, 3)])
@pytest.mark.parametrize("lengths", [[n] for n in ENDS] + [ENDS, ENDS[::-1] * 3, [385] * 7], ids=lambda x: "%dx%d" % (len(x), x[0]))
def test_a_newest_key_that_is_nan(K, dtype, d, new, heads, kv, lengths):
    """the rows that see it are NaN in every column, the others as if it were not there"""
    s = pool(dtype, [new] * len(lengths), lengths, 16, heads, kv, d, d)
    last = np.arange(1, len(lengths) + 1) * new - 1
    want = np64(attend(K, s, dtype, d ** -0.5, max_tokens=new))
    spoil(s, lengths, float("nan"))
    got = np64(attend(K, s, dtype, d ** -0.5, max_tokens=new))
    K.device_status(sync=True)
    blind = np.ones(len(got), bool)
    blind[last] = False
    assert np.isnan(got[last]).all(), np.isnan(got[last]).mean()
    assert np.isfinite(want).all() and np.isfinite(got[blind]).all()
    if blind.any():
        assert np.abs(got - want)[blind].max() <= 4 * HALF[dtype] * (np.abs(want).max() + 4.0) + (2e-5 if dtype == "float32" else 0)


@pytest.mark.parametrize("d", [64, 136])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new", [1, 20])
def test_an_element_of_the_newest_key_that_is_not_finite(K, dtype, d, new, bad):
    """+infinity as a score gives NaN, -infinity weighs nothing: what the formula says in 64 bits"""
    s = pool(dtype, [new] * len(ENDS), ENDS, 16, 4, 2, d, d)
    spoil(s, ENDS, bad, 3)
    got = np64(attend(K, s, dtype, d ** -0.5, max_tokens=new))
    K.device_status(sync=True)
    table, rows, lengths = s["host"]
    with np.errstate(invalid="ignore"):
        want, size, score = fo.paged_attention(np64(s["q"]), np64(s["k"]), np64(s["v"]), table, rows, lengths, d ** -0.5)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and (bad != bad or not np.isnan(want).all())
    fine = np.isfinite(want)
    # scores of normal numbers: |q k| scale stays below 8 for all but the spoiled key
    off = np.abs(got - want) - limit(dtype, size, np.full_like(score, 8.0), d, max(ENDS)) - HALF[dtype] * np.abs(want)
    assert (off[fine] <= 1e-30).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 20])
def test_a_scale_of_zero_is_the_mean(K, dtype, new):
    s = pool(dtype, [new] * 4, [17, 100, 385, 700], 16, 4, 2, 64, 64)
    check(K, s, dtype, scale=0.0, max_tokens=new)
    check(K, s, dtype, scale=0.0, window=33, max_tokens=new)


# ---- behind the end ----------------------------------------------------------------------------------------------
def test_stale_lines_cost_no_more_than_zeros(K):
    """a chunk whose last pages hold NaN behind the end of the sequence takes as long as over a zeroed pool (within a factor of two; rows
    that are all taken again one by one take many times as long)"""
    best = {}
    for fill in (0.0, float("nan"), 0.0, float("nan")):
        s = pool("bfloat16", [256], [4001], 64, 16, 4, 128, 128, fill=fill)
        out = torch.empty_like(s["q"])
        call = lambda: K.paged_attention(s["q"], s["k"], s["v"], s["table"], s["rows"], s["lengths"], out, 128 ** -0.5, max_tokens=256)
        for _ in range(3):
            call()
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            b.synchronize()
            best[fill == 0.0] = min(best.get(fill == 0.0, 1e9), a.elapsed_time(b))
    assert best[False] <= 2 * best[True], best


@pytest.mark.parametrize("length", [1, 5, 127, 128, 129, 250, 383, 4001])
@pytest.mark.parametrize("page", [8, 64, 256])
def test_stale_lines_of_any_kind(K, length, page):
    """bfloat16 chunks: infinities and NaN behind the end, over pages smaller and larger than a tile"""
    for fill in (float("nan"), float("inf"), -float("inf")):
        s = pool("bfloat16", [33, 40], [length, 77], page, 2, 1, 72, 80, fill=fill)
        check(K, s, "bfloat16", max_tokens=40)


# ---- heads that do not turn --------------------------------------------------------------------------------------
def odd(shape, dtype, seed):
    """normal numbers with infinities, zeros of both signs and NaN with bits of their own among them"""
    x = rnd(shape, dtype, seed)
    bits = x.view(torch.int16 if dtype == "bfloat16" else torch.int32)
    shift = 0 if dtype == "bfloat16" else 16
    g = torch.Generator().manual_seed(seed + 1)
    kind = torch.randint(0, 12, shape, generator=g).cuda()
    for i, b in enumerate((0x7f80, -0x80, 0x7fc0, 0x7fa5, -0x8000, 0)):
        bits[kind == i] = b << shift
    return x


def same_bits(a, b):
    t = torch.int16 if a.dtype == torch.bfloat16 else torch.int32
    return torch.equal(a.contiguous().view(t), b.contiguous().view(t))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["pairs", "half"])
@pytest.mark.parametrize("d,pairs", [(64, 16), (64, 5), (64, 32), (24, 3), (256, 40), (8, 0)])
def test_what_does_not_turn_is_copied(K, dtype, layout, d, pairs):
    new, lengths, page, heads, kv = [3, 0, 40], [9, 5, 33], 8, 5, 2
    s = pool(dtype, new, lengths, page, heads, kv, d, 16, fill=0.0)
    table, rows, _ = s["host"]
    n = sum(new)
    q, k, v = odd((n, heads, d), dtype, 3), odd((n, kv, d), dtype, 5), odd((n, kv, 16), dtype, 7)
    place = [(b, lengths[b] - new[b] + t) for b in range(3) for t in range(new[b])]

    def run(cos_sin):
        s["k"].zero_()
        s["v"].zero_()
        out = torch.empty_like(q)
        K.write_pages(k, v, s["k"], s["v"], s["table"], s["rows"], s["lengths"], q=q, q_out=out, cos_sin=cos_sin, layout=layout)
        K.device_status(sync=True)
        kept = [(r, table[b, i // page], i % page) for r, (b, i) in enumerate(place) if i >= 0]
        r, p, l = (torch.tensor(x).cuda() for x in zip(*kept))
        assert same_bits(s["v"][p, l], v[r])
        return out, s["k"][p, l], k[r], np.array([i for _, i in place]), np.array([i for _, i in place if i >= 0])

    out, got, want, pos, kpos = run(None)
    assert same_bits(out, q) and same_bits(got, want)
    if not pairs:
        return
    # angles for some of the positions only: the others keep their heads, and every head keeps its part behind the pairs
    held = 20
    angles = torch.outer(torch.arange(held).double(), 0.37 ** torch.arange(pairs).double())
    cos_sin = torch.stack((angles.cos(), angles.sin()), -1).float().cuda()
    out, got, want, pos, kpos = run(cos_sin)
    assert same_bits(out[..., 2 * pairs:], q[..., 2 * pairs:]) and same_bits(got[..., 2 * pairs:], want[..., 2 * pairs:])
    for x, y, i in ((out, q, pos), (got, want, kpos)):
        plain = torch.from_numpy((i < 0) | (i >= held)).cuda()
        assert same_bits(x[plain], y[plain]) and not plain.all()
        # the others: NaN where the formula has it, else two products and their sum in 32 bits and one rounding
        for r in np.nonzero(~plain.cpu().numpy())[0]:
            for h in range(x.shape[1]):
                with np.errstate(invalid="ignore"):
                    w = fo.turned(np64(y[r, h]), np64(cos_sin[i[r]]), layout)[:2 * pairs]
                g = np64(x[r, h])[:2 * pairs]
                big = np.abs(np64(y[r, h])[np.isfinite(np64(y[r, h]))]).max()
                assert np.array_equal(np.isnan(g), np.isnan(w))
                fine = np.isfinite(w)
                assert np.array_equal(g[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)])
                assert (np.abs(g[fine] - w[fine]) <= HALF[dtype] * np.abs(w[fine]) + 3 * 2.0 ** -24 * 2 * big).all()


# ---- the status --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,new,d", [("bfloat16", 1, 64), ("bfloat16", 40, 64), ("bfloat16", 1, 136), ("bfloat16", 40, 136), ("float32", 1, 64), ("float32", 40, 64)])
def test_a_status_of_its_own_for_what_does_not_fit(K, dtype, new, d):
    """pages outside the pool and rows outside the batch are no waits that ran out, whichever kernel meets them"""
    s = pool(dtype, [new, new], [100, 90], 16, 4, 2, d, d, fill=0.0)
    out, kv = torch.empty_like(s["q"]), torch.ones_like(s["q"][:, :2])
    attention = lambda: K.paged_attention(s["q"], s["k"], s["v"], s["table"], s["rows"], s["lengths"], out, 0.1, max_tokens=new)
    write = lambda: K.write_pages(kv, kv, s["k"], s["v"], s["table"], s["rows"], s["lengths"])
    K.device_status(sync=True)
    for name, at, value in (("table", (0, 6), -1), ("rows", (2,), 2 * new + 9)):
        kept = s[name].clone()
        s[name][at] = value
        for call in (attention, write):
            call()
            torch.cuda.synchronize()
            with pytest.raises(K.FloatOpsError, match="do not fit") as e:
                K.device_status()
            assert e.value.status == 2
            K.device_status()                          # it is said once
        s[name].copy_(kept)
    attention()
    K.device_status(sync=True)


# ---- the bound on rows -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,bound", [([1] * 40, 1), ([1], 1), ([7], 7), ([1, 1, 5, 1], 5), ([0, 0, 2], 1), ([2] * 9, 10)])
def test_a_bound_that_is_left_out(K, new, bound):
    """one row for each of the others is taken off; sequences without rows, or with more than that, come out right all the same"""
    s = pool("bfloat16", new, [100 + 3 * i for i in range(len(new))], 16, 16, 2, 64, 64)
    made, _ = K._calls.paged_attention(s["q"], s["k"], s["v"], s["table"], s["rows"], s["lengths"], torch.empty_like(s["q"]), 0.1, 0, None, None, 1.0)
    assert K.PagedAttentionArgs.from_buffer_copy(made).max_tokens == bound
    check(K, s, "bfloat16")
