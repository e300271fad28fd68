"""Pages on the host: who holds which page, copies on write, forks, compaction; refusals of the calls; scaled rotations; several
completions of a prompt."""
import ctypes
import importlib
import math
import os
import random
import subprocess

import numpy as np
import pytest
import torch

import float_cases as fc
from conftest import PKG, ROOT
from oracle import float_oracle as fo
from test_float_cpu import FakeModel

PC = importlib.import_module(PKG + ".paged_cache")
SC = importlib.import_module(PKG + ".sequence_cache")
config = importlib.import_module(PKG + ".float_config")


def copy(buffers, source, target, positions=None):
    assert not set(source) & set(target) and len(set(target)) == len(target)
    for b in buffers:
        n = b.shape[1] if positions is None else positions
        b[target, :n] = b[source, :n]


def make(slots=6, capacity=40, page=8, pages=None, states=({"sums": ((4,), torch.float32)}, {})):
    return PC.PagedCache([None, 3], [None, 1], slots, capacity, torch.float32, "cpu", states, page, pages, copy)


def write(c, slot, start, values):
    for i, v in enumerate(values):
        at = start + i
        c.buffer(1)[c.held[slot][at // c.page], at % c.page] = v


def read(c, slot):
    t = c.table([slot])[0]
    return [int(c.buffer(1)[t[i // c.page], i % c.page, 0]) for i in range(c.lengths[slot])]


def consistent(c):
    counts = [0] * c.pages
    for held in c.held:
        for p in held:
            counts[p] += 1
    assert counts == c.counts and sorted(c._spare) == [p for p in range(c.pages) if not counts[p]]
    assert all(len(h) == -(-n // c.page) for h, n in zip(c.held, c.lengths))


def test_random_lives_of_sequences_keep_what_they_wrote():
    """thousands of steps, forks, truncations, releases and compactions against plain lists"""
    rng = random.Random(3)
    c = make(states=({}, {}), pages=17)
    mine, n = {}, 0
    for step in range(3000):
        what = rng.choice(["grow", "grow", "grow", "fork", "cut", "drop", "new", "compact"])
        consistent(c)
        if what == "new" and c.free_slots():
            mine[c.acquire()] = []
        elif what == "grow" and mine:
            length = len(mine[rng.choice(list(mine))])
            same = [s for s in mine if len(mine[s]) == length]
            slots = rng.sample(same, rng.randint(1, len(same)))
            k = rng.randint(0, 11)
            try:
                c.extend_all(slots, length, k)
            except PC.CacheFull:
                continue
            for s in slots:
                new = list(range(n, n + k))
                n += k
                write(c, s, length, new)
                mine[s] = mine[s] + new
        elif what == "fork" and mine and c.free_slots():
            s = rng.choice(list(mine))
            mine[c.fork(s)] = list(mine[s])
        elif what == "cut" and mine:
            s = rng.choice(list(mine))
            k = rng.randint(0, len(mine[s]))
            c.truncate(s, k)
            mine[s] = mine[s][:k]
        elif what == "drop" and mine:
            s = rng.choice(list(mine))
            c.release(s)
            del mine[s]
        elif what == "compact":
            before = c.compact()
            used = sum(1 for k in c.counts if k)
            assert all(p < used for h in c.held for p in h) and (before > 0) <= (used > 0)
        for s in mine:
            assert read(c, s) == mine[s]
    assert n > 1000


def test_a_fork_shares_pages_until_it_writes():
    c = make()
    a = c.acquire()
    c.extend(a, 0, 13)
    write(c, a, 0, range(13))
    c.state(0, "sums")[a] = 5.0
    b, d = c.fork(a), c.fork(a)
    assert c.held[a] == c.held[b] == c.held[d] and c.free_pages() == c.pages - 2 and c.state(0, "sums")[b].tolist() == [5.0] * 4
    v = c.version
    c.extend_all([a, b, d], 13, 1)
    # two copies of the second page: the last holder keeps the original
    assert c.held[a][0] == c.held[b][0] == c.held[d][0] and len({c.held[s][1] for s in (a, b, d)}) == 3 and c.version > v
    for i, s in enumerate((a, b, d)):
        write(c, s, 13, [100 + i])
    assert [read(c, s)[-2:] for s in (a, b, d)] == [[12, 100], [12, 101], [12, 102]]
    c.release(a)
    c.release(b)
    assert read(c, d) == list(range(13)) + [102] and c.free_pages() == c.pages - 2
    # a page that another holds is not written to by a step of one alone
    e = c.fork(d)
    c.extend(d, 14, 1)
    write(c, d, 14, [200])
    assert read(c, e) == list(range(13)) + [102]
    consistent(c)


def test_a_pool_that_is_too_small_refuses_and_changes_nothing():
    c = make(pages=3)
    a, b = c.acquire(), c.acquire()
    c.extend_all([a, b], 0, 8)
    before = (list(c.lengths), [list(h) for h in c.held], list(c.counts), c.version)
    with pytest.raises(PC.CacheFull):
        c.extend_all([a, b], 8, 1)
    with pytest.raises(PC.CacheFull):
        c.extend(a, 8, 33)
    with pytest.raises(ValueError):
        c.extend(a, 7, 1)
    with pytest.raises(ValueError):
        c.extend_all([a, a], 8, 1)
    assert before == (list(c.lengths), [list(h) for h in c.held], list(c.counts), c.version)
    c.extend(a, 8, 8)
    with pytest.raises(ValueError):
        c.truncate(a, 3)                       # a recurrent state cannot go back in part
    c.truncate(a, 0)
    c.release(a)
    for slot in (a, -1, 6):
        with pytest.raises(ValueError):
            c.release(slot)
        with pytest.raises(ValueError):
            c.fork(slot)
    for page in (0, 7, 12, 2048):
        with pytest.raises(ValueError):
            make(page=page)
    with pytest.raises(ValueError):
        PC.PagedCache([None, 16], [0, 1], 1, 4, torch.float32, "cpu", page=8)
    with pytest.raises(ValueError):
        make(pages=0)


def test_pages_are_the_lowest_free_ones():
    c = make()
    a, b = c.acquire(), c.acquire()
    c.extend(a, 0, 16)
    c.extend(b, 0, 9)
    assert c.held[a] == [0, 1] and c.held[b] == [2, 3]
    c.release(a)
    assert c.compact() == 2 and c.held[b] == [0, 1] and c.table([b]).tolist() == [[0, 1, -1, -1, -1]]
    assert c.compact() == 0


# ---- several completions of a prompt --------------------------------------------------------------------------------
class Forking(FakeModel):
    def fork(self, slots, n):
        out = []
        for s in slots:
            out.append(s)
            for _ in range(n - 1):
                new = self.free.pop()
                self.seen[new] = list(self.seen[s])
                out.append(new)
        return out


def test_completions_of_a_prompt_share_its_prefill():
    G = importlib.import_module(PKG + ".generate")
    m, drawn = Forking(8), []

    def sampler(logits):
        drawn.append(len(logits))
        return (logits.argmax(-1) + torch.arange(len(logits))) % 50

    out = G.generate(m, [[1, 2, 3], [5, 6, 7]], 2, eos_id=-7, sampler=sampler, samples=3)
    # sequence i adds i to every token that it draws
    want = [[s + i, (2 * s + 2 * i) % 50] for i, s in enumerate([6] * 3 + [18] * 3)]
    assert out == want and drawn == [6, 6] and m.calls == [(3, 0), (1, 3)] and len(m.free) == 8
    # prompts of unequal lengths: the longer one's tokens are not overwritten in any completion
    out = G.generate(m, [[1, 2, 3], [5]], 2, eos_id=-7, samples=2)
    assert out == [[6, 12], [6, 12], [5, 10], [5, 10]] and len(m.free) == 8
    assert G.generate(m, [[1, 2]], 0, eos_id=-7, samples=2) == [[], []]
    with pytest.raises(ValueError):
        G.generate(FakeModel(), [[1]], 2, eos_id=-7, samples=2)
    with pytest.raises(ValueError):
        G.generate(m, [[1]], 2, eos_id=-7, samples=0)
    with pytest.raises(IndexError):            # too few slots for the forks: what was begun is given back
        G.generate(m, [[1]], 2, eos_id=-7, samples=20)


@pytest.mark.parametrize("bad", [["--samples", "0"], ["--sample", "--top-p", "0"], ["--sample", "--min-p", "2"], ["--top-k", "-1"]])
def test_the_program_refuses_settings_out_of_range(bad):
    G = importlib.import_module(PKG + ".generate")
    with pytest.raises(SystemExit):
        G.main(["--model", "nowhere", "--tokens", "1"] + bad)


# ---- scaled rotations ---------------------------------------------------------------------------------------------
def test_scaled_rotations(float_libpath):
    M = importlib.import_module(PKG + ".float_model")
    plain = config.Rotary(10000.0, 64)
    base = M.rotary_table(plain, 40, "cpu").double()
    linear = M.rotary_table(config.Rotary(10000.0, 64, "pairs", config.RotaryScaling("linear", 4.0)), 160, "cpu").double()
    assert (linear[::4] - base).abs().max() <= 2.0 ** -23
    y = config.RotaryScaling("yarn", 8.0, original=256, magnitude=1.0)
    table = M.rotary_table(config.Rotary(10000.0, 64, "pairs", y), 40, "cpu").double()
    # pairs that turn more than 32 times in 256 positions keep their speed, those that turn less than once go 8 times slower
    turns = 256 * 10000.0 ** (-np.arange(32) / 32) / (2 * math.pi)
    for i in range(32):
        speed = math.atan2(table[1, i, 1], table[1, i, 0]) / 10000.0 ** (-i / 32)
        if turns[i] > 32:
            assert abs(speed - 1) < 1e-5
        elif turns[i] < 1 and turns[max(i - 1, 0)] < 1:
            assert abs(speed - 1 / 8) < 1e-5
        else:
            assert 1 / 8 - 1e-5 <= speed <= 1 + 1e-5
    full = M.rotary_table(config.Rotary(10000.0, 64, "pairs", config.RotaryScaling("yarn", 8.0, original=256)), 40, "cpu").double()
    assert (full - table * (1 + 0.1 * math.log(8))).abs().max() <= 2.0 ** -22


def test_scaled_rotations_are_read_from_the_configuration():
    cfg = fc.vifelix(40, 48, 1e-6, 2.0, [fc.parallel(4, 2, 16, 8, 4, 1, 8, 8, 8, [0.9], None)])
    cfg["layers"][0]["mixer"]["left"]["rot"]["scaling"] = {"type": "yarn", "factor": 4, "original": 128}
    left = config.parse_config(cfg).layers[0].mixer.left
    assert left.rot.scaling == config.RotaryScaling("yarn", 4.0, 128) and left.rot.layout == "half"
    lat = fc.config(40, 48, 1e-6, [fc.layer(2, 16, 8, 16, 24, 32, 4, None), fc.layer(2, 16, 8, 16, 24, 32, 4, None, kv_from=0)])
    lat["layers"][0]["mixer"]["rot"]["scaling"] = {"type": "linear", "factor": 2.5}
    del lat["layers"][1]["mixer"]["rot"]
    rots = [l.mixer.rot for l in config.parse_config(lat).layers]
    assert rots[0] == rots[1] and rots[0].scaling == config.RotaryScaling("linear", 2.5)
    for bad in ({"type": "other", "factor": 2}, {"type": "linear"}, {"type": "linear", "factor": 0.5}, {"type": "yarn", "factor": 2},
                {"type": "yarn", "factor": 2, "original": 64, "fast": 1, "slow": 2}):
        cfg["layers"][0]["mixer"]["left"]["rot"]["scaling"] = bad
        with pytest.raises(config.ConfigError):
            config.parse_config(cfg)


# ---- refusals, before anything touches a GPU ------------------------------------------------------------------------
@pytest.fixture(scope="module")
def K(float_libpath):
    return importlib.import_module(PKG + ".float_kernel")


def test_structures_match_the_header(K, tmp_path):
    names = {"zkfp_paged_attention_args": K.PagedAttentionArgs, "zkfp_write_pages_args": K.WritePagesArgs, "zkfp_page_table": K.PageTable,
             "zkfp_page_buffer": K.PageBuffer, "zkfp_sample_args": K.SampleArgs, "zkfp_heads_args": K.HeadsArgs}
    src = tmp_path / "sizes.c"
    lines = []
    for name, s in names.items():
        lines.append('printf("%%zu ", sizeof(%s));' % name)
        lines += ['printf("%%zu ", offsetof(%s, %s));' % (name, f[0]) for f in s._fields_]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "zkds_float.h"\nint main(void) { %s return 0; }\n' % "\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for s in names.values():
        want.append(ctypes.sizeof(s))
        want += [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


A = 1 << 20                                   # an aligned address that nothing reads


def attention_args(K, **kw):
    a = dict(q=A, k=A, v=A, out=A, gate=None, table=A, rows=A, lengths=A, scratch=A, q_tok=256, q_head=64, k_page=2048, k_pos=128, k_head=64,
             v_page=2048, v_pos=128, v_head=64, o_tok=256, o_head=64, gate_tok=0, gate_head=0, tokens=3, pages=10, table_cols=4, table_ld=4,
             batch=2, max_tokens=2, heads=4, kv_heads=2, d=64, dv=64, page=16, window=0, dtype=1, scale=0.1, out_scale=1.0)
    a.update(kw)
    return K.PagedAttentionArgs(**a)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(table=None), dict(rows=None), dict(lengths=None), dict(scratch=None),
    dict(scratch=A + 4), dict(q=A + 8), dict(gate=A + 2), dict(q_tok=252), dict(k_pos=60), dict(v_page=4), dict(o_head=3), dict(gate_tok=1), dict(tokens=-1),
    dict(pages=0), dict(table_cols=0), dict(table_ld=3), dict(batch=0), dict(heads=5), dict(heads=0), dict(kv_heads=0), dict(d=60), dict(d=0), dict(dv=4),
    dict(page=0), dict(page=24), dict(page=4), dict(page=2048), dict(window=-1), dict(dtype=2), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(max_tokens=-1)], ids=str)
def test_attention_refuses(K, bad):
    a = attention_args(K, **bad)
    assert K._paged(ctypes.byref(a), None) == 1


@pytest.mark.parametrize("far", [dict(d=264), dict(dv=512), dict(batch=1025), dict(tokens=1 << 28)], ids=str)
def test_attention_has_no_kernel_for(K, far):
    a = attention_args(K, **far)
    assert K._paged(ctypes.byref(a), None) == 6 and K._paged_scratch(ctypes.byref(a)) == 0


def test_attention_takes_the_kernel_meant_for_the_shape(K):
    path = lambda **kw: K.paged_path(ctypes.byref(attention_args(K, **kw)))
    assert path() == 2 and path(max_tokens=8) == 2 and path(max_tokens=9) == 1 and path(dtype=0) == 0
    assert path(d=136, max_tokens=9) == 0 and path(d=136) == 0 and path(heads=516, kv_heads=2, max_tokens=1) == 0
    assert path(heads=256, kv_heads=2, max_tokens=1) == 1 and path(batch=1024) == 2


@pytest.mark.parametrize("bad", [dict(k=None), dict(v_pages=None), dict(table=None), dict(q_out=None), dict(k=A + 8), dict(cos_sin=A + 4), dict(k_tok=4),
                                 dict(page=12), dict(pairs=33), dict(pairs=-1), dict(half=2), dict(dtype=5), dict(tokens=-1), dict(d=20), dict(heads=0),
                                 dict(table_ld=1), dict(pages=0), dict(batch=0), dict(positions=-1)], ids=str)
def test_writes_refuse(K, bad):
    a = dict(q=A, k=A, v=A, q_out=A, k_pages=A, v_pages=A, cos_sin=A, table=A, rows=A, lengths=A, q_tok=256, q_head=64, k_tok=128, k_head=64, v_tok=128,
             v_head=64, qo_tok=256, qo_head=64, k_page=2048, k_pos=128, kp_head=64, v_page=2048, v_pos=128, vp_head=64, tokens=3, pages=10,
             table_cols=4, table_ld=4, batch=2, positions=64, heads=4, kv_heads=2, d=64, dv=64, page=16, pairs=32, half=0, dtype=1)
    a.update(bad)
    assert K._write_pages(ctypes.byref(K.WritePagesArgs(**a)), None) == 1


@pytest.mark.parametrize("source,target", [([0], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([10], [1]), ([-1], [1]), ([1], [10]), ([1], [-2])], ids=str)
def test_copies_refuse(K, source, target):
    n = len(source)
    call = lambda b, s, t: K._copy_pages(b, 1, (ctypes.c_int * n)(*s), (ctypes.c_int * n)(*t), n, None)
    buffers = (K.PageBuffer * 1)((A, 1024, 1024, 10))
    assert call(buffers, source, target) == 1
    for bad in ((A + 4, 1024, 1024, 10), (A, 512, 1024, 10), (A, 1024, 1000, 10), (None, 1024, 1024, 10), (A, 1024, -16, 10), (A, 1024, 1024, 0)):
        assert call((K.PageBuffer * 1)(bad), list(range(n)), list(range(5, 5 + n))) == 1
    assert call((K.PageBuffer * 1)((A, 1024, 0, 10)), list(range(n)), list(range(5, 5 + n))) == 0          # nothing of them


@pytest.mark.parametrize("bad", [dict(logits=None), dict(random=None), dict(out=None), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(dtype=2)], ids=str)
def test_sampling_refuses(K, bad):
    a = dict(logits=A, random=A, out=A, ld=100, rows=2, vocab=100, dtype=0)
    a.update(bad)
    assert K._sample(ctypes.byref(K.SampleArgs(**a)), None) == 1
    a = K.SampleArgs(logits=A, random=A, out=A, ld=1 << 20, rows=2, vocab=(1 << 18) + 1, dtype=0)
    assert K._sample(ctypes.byref(a), None) == 6


def test_calls_refuse_tensors_that_are_not_on_a_gpu(K):
    t, i = torch.zeros(4, 16, 2, 64), torch.zeros(2, 4, dtype=torch.int32)
    x = torch.zeros(3, 2, 64)
    for call in (lambda: K.paged_attention(x, t, t, i, i[0, :3], i[0, :2], x, 1.0), lambda: K.write_pages(x, x, t, t, i, i[0, :3], i[0, :2]),
                 lambda: K.copy_pages([t], [0], [1]), lambda: K.sample(x[0], x[0, 0]), lambda: K.sample([1.0], None)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        K.copy_pages([t], [0], [1, 2])
    assert K.copy_pages([], [0], [1]) is None and K.copy_pages([t], [], []) is None


# ---- the oracle -----------------------------------------------------------------------------------------------------
def test_oracle_of_sampling():
    l = np.log([0.5, 0.125, 0.25, 0.125])
    assert [fo.sample(l, u) for u in (0.0, 0.49, 0.51, 0.62, 0.63, 0.88)] == [0, 0, 1, 1, 2, 3]
    assert fo.kept_tokens(l, 1.0, 3, 1.0, 0.0)[0].tolist() == [0, 1, 2]                # of the equal ones the first
    assert fo.kept_tokens(l, 1.0, 0, 0.75, 0.0)[0].tolist() == [0, 2] and fo.kept_tokens(l, 1.0, 0, 0.76, 0.0)[0].tolist() == [0, 1, 2]
    assert fo.kept_tokens(l, 1.0, 0, 1.0, 0.3)[0].tolist() == [0, 2] and fo.kept_tokens(l, 0.0, 0, 1.0, 0.0)[0].tolist() == [0]
    assert fo.kept_tokens(l, 1.0, 3, 0.6, 0.0)[0].tolist() == [0, 2]                   # of the weight that top_k left
    assert fo.sample(np.full(3, -np.inf), 0.5) == -1


def test_oracle_of_pages_is_the_window_of_a_whole_sequence():
    rng = np.random.default_rng(1)
    k, v, q = rng.standard_normal((20, 1, 4)), rng.standard_normal((20, 1, 4)), rng.standard_normal((20, 2, 4))
    order = [2, 0, 1]
    pages = lambda x: np.concatenate([x, np.full((4, 1, 4), np.nan)]).reshape(3, 8, 1, 4)[np.argsort(order)]
    got = fo.paged_attention(q[15:], pages(k), pages(v), [order], [0, 5], [20], 0.5, 6)[0]
    for h in range(2):
        p = fo.softmax_rows(q[:, h] @ k[:, 0].T * 0.5, fo.window_mask(20, 6))
        assert np.abs(got[:, h] - (p @ v[:, 0])[15:]).max() < 1e-12


def test_calls_refuse_what_is_on_no_gpu(K):
    """and hold on to nothing that they refused"""
    import sys
    t = {n: torch.zeros(*shape, dtype=dt) for n, shape, dt in (("q", (3, 4, 16), torch.float32), ("pages", (5, 16, 2, 16), torch.float32),
         ("table", (1, 2), torch.int32), ("rows", (2,), torch.int32), ("lengths", (1,), torch.int32), ("logits", (2, 30), torch.float32), ("u", (2,), torch.float32))}
    pages = (t["pages"], t["pages"], t["table"], t["rows"], t["lengths"])
    kept = {n: sys.getrefcount(x) for n, x in t.items()}
    for _ in range(3):
        for call in (lambda: K.paged_attention(t["q"], *pages, t["q"], 0.1), lambda: K.write_pages(t["q"], t["q"], *pages), lambda: K.sample(t["logits"], t["u"]),
                     lambda: K.copy_pages([t["pages"]], [0], [1]), lambda: K.sample([1.0], t["u"]), lambda: K.write_pages(t["q"], t["q"], *pages, layout="other"),
                     lambda: K.copy_pages([t["pages"]], [0, 1], [2]), lambda: K.copy_pages([t["pages"]], [2 ** 40], [2]), lambda: K.copy_pages([3], [0], [1])):
            with pytest.raises(ValueError):
                call()
        for call in (lambda: K.copy_pages([t["pages"]], [0.5], [1]), lambda: K.copy_pages(7, [0], [1])):
            with pytest.raises(TypeError):
                call()
    assert K.copy_pages([], [], []) is None and K.copy_pages([t["pages"]], [], []) is None
    assert {n: sys.getrefcount(x) for n, x in t.items()} == kept


def test_a_copy_that_fails_changes_nothing():
    def fails(*args, **kw):
        raise RuntimeError("no copy")
    c = make()
    a = c.acquire()
    c.extend(a, 0, 11)
    write(c, a, 0, range(11))
    b = c.fork(a)
    before = [list(h) for h in c.held], list(c.lengths), c.free_pages(), c.free_slots()
    c.copy = fails
    for act in (lambda: c.extend_all([a, b], 11, 9), lambda: c.extend(b, 11, 1), lambda: c.fork(a), lambda: c.compact() or fails()):
        with pytest.raises(RuntimeError):
            act()
        assert ([list(h) for h in c.held], list(c.lengths), c.free_pages(), c.free_slots()) == before
        consistent(c)
    c.copy = copy
    c.extend_all([a, b], 11, 9)
    write(c, a, 11, range(9))
    assert read(c, a) == list(range(11)) + list(range(9)) and read(c, b)[:11] == list(range(11))
    consistent(c)
