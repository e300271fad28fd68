"""The operators of serving over a pool of pages, as cases that can be timed and compared: attention of new tokens over
paged keys and values, the write of rotated heads into pages, copies of pages, and sampling from given random numbers.

A program that serves holds one pool of pages per layer, a table of page numbers per sequence (in no order: pages come
back and are handed out again), the bounds of each sequence's rows in the batch, and how many positions each holds.
Sizes are those of the framework's grouped attention layers (width 7168: 128 heads over 16, 4096: 32 over 8,
2048: 16 over 4, heads of 128) and of its vocabularies.
"""
import importlib
import math
import random

import torch

own = False
PACKAGE = "zk-deepseek_b200"
DEVICE = "cuda"


def listed():
    return [
        # one sequence decoding, latency: a token over a cache that is full but for one position
        {"name": "attention_1", "op": "attention", "dtype": "bfloat16", "batch": 1, "new": 1, "mixed": False, "length": 4095, "heads": 32,
         "kv_heads": 8, "dim": 128, "vdim": 128, "window": 0, "page": 64, "gate": False},
        # a full serving batch decoding, every sequence at a length of its own
        {"name": "attention_64", "op": "attention", "dtype": "bfloat16", "batch": 64, "new": 1, "mixed": False, "length": 8192, "heads": 128,
         "kv_heads": 16, "dim": 128, "vdim": 128, "window": 0, "page": 64, "gate": True},
        # a chunk of a long prompt beside four sequences that decode
        {"name": "attention_mixed", "op": "attention", "dtype": "bfloat16", "batch": 5, "new": 517, "mixed": True, "length": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "vdim": 128, "window": 0, "page": 16, "gate": True},
        # a whole prompt
        {"name": "attention_prompt", "op": "attention", "dtype": "bfloat16", "batch": 1, "new": 4096, "mixed": False, "length": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "vdim": 128, "window": 0, "page": 64, "gate": False},
        # float32, heads that fill no tile, a window, small pages: short chunks of three requests
        {"name": "attention_f32", "op": "attention", "dtype": "float32", "batch": 3, "new": 100, "mixed": False, "length": 777, "heads": 16,
         "kv_heads": 4, "dim": 72, "vdim": 72, "window": 300, "page": 16, "gate": False},
        # the heads of one decoding step of eight sequences, half of each head rotated, pairs half a rotation apart
        {"name": "heads_8", "op": "heads", "dtype": "bfloat16", "batch": 8, "new": 1, "length": 3001, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotated": 64, "layout": "half", "page": 64},
        # the heads of two long prompts at the largest width, whole heads rotated in adjacent pairs
        {"name": "heads_8190", "op": "heads", "dtype": "bfloat16", "batch": 2, "new": 4095, "length": 5000, "heads": 128, "kv_heads": 16, "dim": 128,
         "rotated": 128, "layout": "pairs", "page": 64},
        # one request forked into four: its last, partly filled page is copied in every layer
        {"name": "pages_fork", "op": "pages", "dtype": "bfloat16", "layers": 24, "pages": 64, "moves": 3, "page": 64, "pitch": 2048, "positions": 37},
        # a pool that is compacted: half of its pages move
        {"name": "pages_compact", "op": "pages", "dtype": "bfloat16", "layers": 3, "pages": 3001, "moves": 1500, "page": 64, "pitch": 2048,
         "positions": 64},
        # the next token of one sequence, the full vocabulary of the integer model's configuration
        {"name": "sample_1", "op": "sample", "dtype": "float32", "rows": 1, "vocab": 129280, "sharpness": 2.5, "limits": "top_p"},
        # a serving batch in bfloat16 logits, whose values repeat
        {"name": "sample_64", "op": "sample", "dtype": "bfloat16", "rows": 64, "vocab": 32768, "sharpness": 1.7, "limits": "top_k"},
        # a large batch, every request with settings of its own
        {"name": "sample_256", "op": "sample", "dtype": "float32", "rows": 256, "vocab": 129280, "sharpness": 2.5, "limits": "mixed"},
    ]


def _between(rng, low, high):
    """a whole number spread over the logarithm of the range, often odd"""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n | rng.randrange(2)))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "heads", "pages", "sample", "sample"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv_heads = rng.choice([(16, 4), (32, 8), (128, 16), (12, 4), (7, 1), (6, 6)])
    if op == "attention":
        wide = 16 if dtype == "float32" else 128
        kind, dim = rng.choice(["decode", "few", "chunk"]), 8 * rng.randint(2, 16)
        new = {"decode": 1, "few": rng.randint(2, 16), "chunk": _between(rng, 17, 128 if wide == 16 else 2048)}[kind]
        batch = _between(rng, 1, {"decode": 64, "few": 32, "chunk": 4}[kind])
        heads, kv_heads = (heads, kv_heads) if heads <= wide and (kind != "chunk" or heads <= 32) else (16, 4)
        return {"op": op, "dtype": dtype, "batch": batch, "new": new, "mixed": rng.random() < 0.3,
                "length": _between(rng, max(new, 1), 1024 if wide == 16 else 8192 if kind != "chunk" else 4096), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "vdim": dim if rng.random() < 0.7 else 8 * rng.randint(2, 16),
                "window": rng.choice([0, 0, _between(rng, 1, 2000)]), "page": page, "gate": rng.random() < 0.5}
    if op == "heads":
        dim, new = 8 * rng.randint(2, 32), _between(rng, 1, 2048)
        return {"op": op, "dtype": dtype, "batch": _between(rng, 1, 4), "new": new, "length": _between(rng, new, 8192), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotated": min(dim, 4 * rng.randint(1, 64)), "layout": rng.choice(["pairs", "half"]), "page": page}
    if op == "pages":
        pages = _between(rng, 2, 2000)
        return {"op": op, "dtype": dtype, "layers": rng.choice([1, 2, 3, 40]) if pages < 100 else rng.choice([1, 2]), "pages": pages,
                "moves": rng.randint(1, pages // 2), "page": page, "pitch": 8 * _between(rng, 2, 128), "positions": rng.randint(1, page)}
    return {"op": op, "dtype": dtype, "rows": _between(rng, 1, 256), "vocab": _between(rng, 100, 129280), "sharpness": rng.uniform(0.3, 4.0),
            "limits": rng.choice(["none", "top_k", "top_p", "min_p", "mixed"])}


def _counts(case):
    """new tokens and positions of every sequence: the first at the case's bounds, the others spread over the logarithm"""
    rng = random.Random(case["batch"] * 1000003 + case["length"])
    new = [case["new"] if b == 0 or not case.get("mixed") else 1 for b in range(case["batch"])]
    return new, [case["length"] if b == 0 else _between(rng, n, case["length"]) for b, n in enumerate(new)]


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "pages":
        return {"bytes": 2 * case["layers"] * case["moves"] * case["positions"] * case["pitch"] * size, "flops": 0}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 4 * case["rows"] * case["vocab"]}
    new, lengths = _counts(case)
    heads, kv, rows = case["heads"], case["kv_heads"], sum(new)
    if case["op"] == "heads":
        turned = rows * (heads + kv) * case["rotated"]
        return {"bytes": 2 * rows * (heads + 2 * kv) * case["dim"] * size + rows * case["rotated"] * 4, "flops": 3 * turned}
    window = case["window"] or case["length"]
    seen = sum(min(length, window + n - 1) for n, length in zip(new, lengths))
    # pairs of a query and a visible key: rows at position i see min(i + 1, window) keys
    full = [(max(0, min(length, window) - (length - n)), n, length) for n, length in zip(new, lengths)]
    pairs = sum(a * (length - n) + a * (a + 1) // 2 + (n - a) * window for a, n, length in full)
    both = case["dim"] + case["vdim"]
    return {"bytes": size * (rows * heads * (both + (case["vdim"] if case["gate"] else 0)) + seen * kv * both), "flops": 2 * pairs * heads * both}


# ---- what a serving program has in hand --------------------------------------------------------------------------
class State:
    pass


def _pool(s, case, lengths, g):
    """page tables over a pool with a few pages to spare, page numbers in no order"""
    page = case["page"]
    need = [-(-length // page) for length in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEVICE)[:sum(need)].tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)
    s.table, s.lengths = i32(table), i32(lengths)
    return total


def _rows(s, new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    s.rows, s.total = torch.tensor(at, dtype=torch.int32, device=DEVICE), at[-1]


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)
    s = State()
    s.case = case
    if case["op"] == "pages":
        s.buffers = [normal(case["pages"], case["page"], case["pitch"]) for _ in range(case["layers"])]
        order = torch.randperm(case["pages"], generator=g, device=DEVICE).tolist()
        s.source, s.target = order[:case["moves"]], order[case["moves"]:2 * case["moves"]]
        return s
    if case["op"] == "sample":
        R = case["rows"]
        # a few likely tokens over a bulk of unlikely ones
        bulk = torch.randn(R, case["vocab"], generator=g, device=DEVICE) * case["sharpness"]
        tail = torch.rand(R, case["vocab"], generator=g, device=DEVICE).pow_(40).mul_(2 * case["sharpness"])
        s.logits = (bulk + tail).to(dtype)
        s.random = torch.rand(R, generator=g, device=DEVICE)
        pick = lambda low, high: torch.rand(R, generator=g, device=DEVICE) * (high - low) + low
        coin = lambda: torch.rand(R, generator=g, device=DEVICE) < 0.5
        mixed, limits = case["limits"] == "mixed", case["limits"]
        s.temperature = pick(0.5, 1.5)
        s.top_k = torch.randint(2, 200, (R,), generator=g, device=DEVICE, dtype=torch.int32)
        s.top_k = s.top_k * coin() if mixed else s.top_k if limits == "top_k" else torch.zeros_like(s.top_k)
        s.top_p = pick(0.7, 0.98)
        s.top_p = torch.where(coin(), s.top_p, 1.0) if mixed else s.top_p if limits == "top_p" else torch.ones_like(s.top_p)
        s.min_p = pick(0.01, 0.2)
        s.min_p = torch.where(coin(), s.min_p, 0.0) if mixed else s.min_p if limits == "min_p" else torch.zeros_like(s.min_p)
        s.out = torch.empty(R, dtype=torch.int64, device=DEVICE)
        return s
    new, lengths = _counts(case)
    _rows(s, new)
    pages = _pool(s, case, lengths, g)
    s.new, s.length = max(new), max(lengths)
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "heads":
        s.q, s.k, s.v = normal(s.total, H, d), normal(s.total, G, d), normal(s.total, G, d)
        s.q_out = torch.empty_like(s.q)
        s.k_pages, s.v_pages = (torch.zeros(pages, case["page"], G, d, dtype=dtype, device=DEVICE) for _ in range(2))
        i = torch.arange(case["rotated"] // 2, dtype=torch.float64, device=DEVICE)
        angles = torch.outer(torch.arange(case["length"], dtype=torch.float64, device=DEVICE), 10000.0 ** (-2.0 * i / case["rotated"]))
        s.cos_sin = torch.stack((angles.cos(), angles.sin()), dim=-1).float()
        return s
    s.q = normal(s.total, H, d)
    # keys and values of a layer lie side by side in its pages
    s.pool = normal(pages, case["page"], G * (d + case["vdim"]))
    s.k_pages, s.v_pages = s.pool[:, :, :G * d].unflatten(2, (G, d)), s.pool[:, :, G * d:].unflatten(2, (G, case["vdim"]))
    s.gate = normal(s.total, H, case["vdim"]) if case["gate"] else None
    s.out = torch.empty(s.total, H, case["vdim"], dtype=dtype, device=DEVICE)
    s.scale = 2.0 * d ** -0.5
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"attention": _attention, "heads": _heads, "pages": _pages, "sample": _sample}[s.case["op"]](s)


def _run_own(s):
    K = importlib.import_module(PACKAGE + ".float_kernel")
    op = s.case["op"]
    if op == "attention":
        return K.paged_attention(s.q, s.k_pages, s.v_pages, s.table, s.rows, s.lengths, s.out, s.scale, window=s.case["window"],
                                 max_tokens=s.new, gate=s.gate, out_scale=0.7 if s.case["gate"] else 1.0)
    if op == "heads":
        K.write_pages(s.k, s.v, s.k_pages, s.v_pages, s.table, s.rows, s.lengths, q=s.q, q_out=s.q_out, cos_sin=s.cos_sin,
                      layout=s.case["layout"])
        return s.q_out, s.k_pages, s.v_pages
    if op == "pages":
        K.copy_pages(s.buffers, s.source, s.target, positions=s.case["positions"])
        return s.buffers
    return K.sample(s.logits, s.random, s.out, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)


def _places(s):
    """sequence, place in it and position of every row of the batch"""
    r = torch.arange(s.total, device=DEVICE, dtype=torch.int32)
    b = torch.searchsorted(s.rows, r, right=True) - 1
    t = r - s.rows[b]
    return b, t.long(), (s.lengths[b] - (s.rows[b + 1] - s.rows[b]) + t).long()


def _attention(s):
    case, G = s.case, s.case["kv_heads"]
    group = case["heads"] // G
    b, t, _ = _places(s)
    n = (s.rows[1:] - s.rows[:-1]).long()
    place = torch.arange(s.new, device=DEVICE)
    row = (s.rows[:-1, None].long() + place).clamp(max=s.total - 1)
    j = torch.arange(s.length, device=DEVICE)
    held = j < s.lengths[:, None]
    pages = s.table[:, j // case["page"]].long()
    line = j % case["page"]
    k = torch.where(held[..., None, None], s.k_pages[pages, line].float(), 0.0)
    v = torch.where(held[..., None, None], s.v_pages[pages, line].float(), 0.0)
    q = s.q[row].float().unflatten(2, (G, group))
    i = (s.lengths - n)[:, None] + place
    seen = (j <= i[..., None]) & held[:, None]
    if case["window"]:
        seen &= i[..., None] - j < case["window"]
    seen = seen[:, None, None]
    score = torch.where(seen, torch.einsum("bnhgd,blhd->bhgnl", q, k) * s.scale, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.einsum("bhgnl,blhd->bnhgd", e, v) / e.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    o = o.flatten(2, 3)[b, t]
    if s.gate is not None:
        o = o / (1.0 + torch.exp(-s.gate.float())) * 0.7
    s.out.copy_(o)
    return s.out


def _turn(x, cos_sin, layout):
    p = cos_sin.shape[1]
    c, n = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    y = x.clone()
    one, two = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if layout == "pairs" else (slice(0, p), slice(p, 2 * p))
    y[..., one], y[..., two] = x[..., one] * c - x[..., two] * n, x[..., two] * c + x[..., one] * n
    return y


def _heads(s):
    b, _, i = _places(s)
    turns = s.cos_sin[i]
    s.q_out.copy_(_turn(s.q.float(), turns, s.case["layout"]))
    page, line = s.table[b, i // s.case["page"]].long(), i % s.case["page"]
    s.k_pages[page, line] = _turn(s.k.float(), turns, s.case["layout"]).to(s.k.dtype)
    s.v_pages[page, line] = s.v
    return s.q_out, s.k_pages, s.v_pages


def _pages(s):
    n = s.case["positions"]
    for buffer in s.buffers:
        buffer[s.target, :n] = buffer[s.source, :n]
    return s.buffers


def _sample(s):
    # running sums decide next to their borders, so they are taken in 64 bits
    x = s.logits.double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / s.temperature.double()[:, None])
    order = torch.sort(s.logits, dim=-1, descending=True, stable=True).indices
    falling = w.gather(1, order)
    rank = torch.arange(s.logits.shape[1], device=DEVICE)
    k = torch.where(s.top_k > 0, s.top_k.long(), s.logits.shape[1])[:, None]
    first = torch.where(rank < k, falling, 0.0)
    mass = first.cumsum(-1)
    top_p = s.top_p.double()[:, None]
    keep = (rank < k) & ((mass - first < top_p * first.sum(-1, keepdim=True)) | (top_p >= 1.0)) & (falling >= s.min_p.double()[:, None])
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, falling, 0.0))
    mass = kept.cumsum(-1)
    s.out.copy_((mass <= s.random.double()[:, None] * mass[:, -1:]).sum(-1))
    return s.out


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    """copies are not computed, and a token is a whole number: both have no such value"""
    if case["op"] == "attention":
        return _exact_attention(case, seed)
    if case["op"] == "heads":
        return _exact_heads(case, seed)
    return None


def _exact_attention(case, seed):
    s = prepare(case, seed)
    new, lengths = _counts(case)
    group, out, at = case["heads"] // case["kv_heads"], [], 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        count = -(-length // case["page"])
        mine = s.table[b, :count].long()
        low = max(0, length - n - case["window"] + 1) if case["window"] else 0
        rel = torch.arange(length - n, length, device=DEVICE)[:, None] - torch.arange(low, length, device=DEVICE)
        hidden = (rel < 0) | (rel >= case["window"]) if case["window"] else rel < 0
        heads = []
        for h in range(case["heads"]):
            k = s.k_pages[mine, :, h // group].flatten(0, 1)[low:length].double()
            v = s.v_pages[mine, :, h // group].flatten(0, 1)[low:length].double()
            p = torch.softmax((s.q[at:at + n, h].double() @ k.T * s.scale).masked_fill_(hidden, -math.inf), dim=-1)
            heads.append(p @ v)
        o = torch.stack(heads, dim=1)
        if s.gate is not None:
            o = o * torch.sigmoid(s.gate[at:at + n].double()) * 0.7
        out.append(o)
        at += n
    return torch.cat(out)


def _exact_heads(case, seed):
    s = prepare(case, seed)
    new, lengths = _counts(case)
    unit = torch.view_as_complex(s.cos_sin.double().contiguous())

    def turned(x, low, high):
        part, rest = x.double()[..., :case["rotated"]], x.double()[..., case["rotated"]:]
        z = part.unflatten(-1, (-1, 2)) if case["layout"] == "pairs" else part.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * unit[low:high, None])
        return torch.cat((z.flatten(-2) if case["layout"] == "pairs" else z.transpose(-1, -2).flatten(-2), rest), dim=-1)

    k_pages, v_pages, q, at = s.k_pages.double(), s.v_pages.double(), [], 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        rows, low = slice(at, at + n), length - n
        q.append(turned(s.q[rows], low, length))
        k = turned(s.k[rows], low, length)
        for p in range(low // case["page"], -(-length // case["page"])):
            first, last = max(low, p * case["page"]), min(length, (p + 1) * case["page"])
            where = (int(s.table[b, p]), slice(first - p * case["page"], last - p * case["page"]))
            k_pages[where], v_pages[where] = k[first - low:last - low], s.v[at + first - low:at + last - low].double()
        at += n
    return torch.cat(q), k_pages, v_pages
