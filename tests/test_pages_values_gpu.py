"""Values that calls over pages meet rarely: scores that jump from one tile of keys to the next, keys that are NaN or infinite where a
row does see them."""
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
