"""The operators that a step over several conversations at once is made of, besides its products: keys and values
appended to a paged cache, attention of each conversation's new rows over its pages, and the logits' rules before a
token is sampled.

`listed()` are the measured cases, `draw(rng)` makes one more of the same ranges, `prepare` is what a program holds
before a call, `run` the call (in plain torch operations, or with `own` the package's operator), `work` the bytes and
operations no implementation can do without, `exact` the result in 64 bits.

The shapes are those of the benchmark and the tests: 16 query and 2 key/value heads of 256 with 64 rotated dims,
vocabularies of 151,936 and 248,320, contexts of 8,192 and 32,001, chains of 5 rows and trees of 17; beside them other
usual head layouts.
"""
import ctypes

import numpy as np
import torch

own = False
DEV = "cuda"
EPS, THETA = 1e-6, 1e7
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3}   # the package's element types


# ------------------------------------------------------------------ the cases
def _append(name, **k):
    return dict(dict(name=name, op="append", order="head", norm=True, interleaved=False, pad=0), **k)


def _attention(name, **k):
    return dict(dict(name=name, op="attention", order="head", tree=False, pad=0), **k)


def listed():
    return [
        # plain decoding of one conversation: one token's key and value; the launch is all there is
        _append("append_token", seqs=1, rows=1, longest=1003, spread="even", heads=16, kv_heads=2, dim=256, rope=64,
                type="f16", rows_type="f32", q_type="f32", page=64),
        # a verify step of 48 conversations with up to 4 drafts each, the int8 cache
        _append("append_chains_i8", seqs=48, rows=5, longest=4096, spread="ragged", heads=16, kv_heads=2, dim=256,
                rope=64, type="i8", rows_type="f32", q_type="f32", page=64, pad=3),
        # four prompts of different lengths read at once, 16-bit rows, the whole head rotated
        _append("append_prompts", seqs=4, rows=4096, longest=4096, spread="prompts", heads=32, kv_heads=8, dim=128,
                rope=128, type="bf16", rows_type="bf16", q_type="bf16", page=32, norm=False),
        # one token of a short chat
        _attention("attend_token", seqs=1, rows=1, longest=1003, spread="even", heads=16, kv_heads=2, dim=256,
                   type="f16", q_type="f32", page=64),
        # one token at the end of a very long document: one conversation has to fill the chip
        _attention("attend_long", seqs=1, rows=1, longest=131073, spread="even", heads=16, kv_heads=2, dim=256,
                   type="f16", q_type="f16", page=128),
        # plain decoding of 64 conversations of very different lengths
        _attention("attend_batch", seqs=64, rows=1, longest=8192, spread="ragged", heads=32, kv_heads=8, dim=128,
                   type="bf16", q_type="bf16", page=32),
        # a verify step of 32 conversations with up to 4 chained drafts each
        _attention("attend_chains", seqs=32, rows=5, longest=4096, spread="ragged", heads=16, kv_heads=2, dim=256,
                   type="f16", q_type="f32", page=64, pad=5),
        # one conversation's draft tree in a long document, the int8 cache
        _attention("attend_tree_i8", seqs=1, rows=17, longest=32001, spread="even", heads=16, kv_heads=2, dim=256,
                   type="i8", q_type="f32", page=64, tree=True),
        # one long conversation among thirty short ones, small pages, an odd head size, positions before heads
        _attention("attend_mixed", seqs=31, rows=1, longest=65537, spread="one", heads=24, kv_heads=4, dim=80,
                   type="bf16", q_type="bf16", page=16, order="position"),
        # one row before plain sampling
        dict(name="rules_row", op="rules", rows=1, vocab=151936, type="f32", history=300, shared=1, biases=0, masks=0),
        # one row each of 64 conversations under grammars, 16-bit logits, biases
        dict(name="rules_batch", op="rules", rows=64, vocab=151936, type="bf16", history=2048, shared=1, biases=40, masks=8),
        # the 5 rows each of 32 conversations' verify step: a row's history is the conversation's and the drafts before it
        dict(name="rules_chains", op="rules", rows=160, vocab=248320, type="f32", history=8192, shared=5, biases=0, masks=0),
    ]


def _log_int(rng, lo, hi):
    """an integer of [lo, hi], spread over its logarithm"""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


LAYOUTS = [(16, 2, 256), (32, 8, 128), (8, 8, 64), (24, 4, 80), (20, 4, 96), (28, 4, 128), (16, 1, 192), (9, 3, 48)]


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "rules"])
    if op == "rules":
        shared = rng.choice([1, 1, 3, 5])
        rows = shared * _log_int(rng, 1, 160 // shared)
        return dict(op=op, rows=rows, vocab=_log_int(rng, 4001, 248320), type=rng.choice(["f32", "f16", "bf16"]),
                    history=_log_int(rng, 1, 16384), shared=shared, biases=rng.choice([0, 0, 7, 300]),
                    masks=rng.choice([0, 0, 1, 5]))
    heads, kv_heads, dim = rng.choice(LAYOUTS)
    kind = rng.choice(["f16", "bf16", "i8"])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, type=kind, page=rng.choice([16, 32, 48, 64, 128, 256]),
                order=rng.choice(["head", "position"]), pad=rng.choice([0, 0, 4]))
    if op == "append":
        case["rope"] = rng.choice([dim, 16, 8 * (dim // 16), 0])
        case["norm"], case["interleaved"] = rng.random() < 0.5, rng.random() < 0.3
        case["rows_type"] = rng.choice(["f32", "f16", "bf16"])
        case["q_type"] = rng.choice(["f32", case["rows_type"]])
        if rng.random() < 0.3:
            case.update(seqs=rng.randint(1, 4), spread="prompts", rows=_log_int(rng, 33, 2048))
            case["longest"] = case["rows"]
        else:
            case.update(seqs=_log_int(rng, 1, 128), rows=_log_int(rng, 1, 17), longest=_log_int(rng, 32, 8192),
                        spread=rng.choice(["even", "ragged", "one"]))
        return case
    case["q_type"] = rng.choice(["f32", kind] if kind != "i8" else ["f32", "f16", "bf16"])
    case["seqs"] = _log_int(rng, 1, 64)
    case["rows"] = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 32)])
    case["tree"] = case["rows"] > 2 and rng.random() < 0.4
    longest = min(65536, (1 << 29) // (case["seqs"] * kv_heads * dim))
    case["longest"] = _log_int(rng, case["rows"], longest)
    case["spread"] = rng.choice(["even", "ragged", "one"])
    return case


# ------------------------------------------------------------------ what the cases are made of
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFFFFFF)


def _lengths(case):
    """each sequence's (positions, new rows): the case's own, the same for every seed"""
    n, hi = case["seqs"], case["longest"]
    r = np.random.default_rng([n, hi, case["rows"]])
    rows = np.full(n, case["rows"])
    if case["spread"] == "prompts":   # whole prompts: every position is new
        rows = np.maximum(1, np.rint(hi / (1.0 + 0.6 * np.arange(n)))).astype(int)
        return rows, rows
    if case["rows"] > 1 and n > 1:
        rows = r.integers(1, case["rows"] + 1, n)
        rows[0] = case["rows"]
    if case["spread"] == "even":
        lens = np.full(n, hi)
    elif case["spread"] == "ragged":
        lens = np.rint(hi * 16.0 ** -r.random(n)).astype(int)
    else:   # one long conversation among short ones
        lens = r.integers(1, max(2, hi // 128), n)
        lens[n // 2] = hi
    return np.maximum(lens, rows), rows


def _tables(case, seed):
    """the batch on the GPU: row starts, lengths, and pages of a pool handed out in a random order"""
    lens, rows = _lengths(case)
    need = -(-lens // case["page"])
    wide = int(need.max())
    pool = int(need.sum()) + 3
    order = torch.randperm(pool, device=DEV, generator=_gen(seed, 1)).to(torch.int32)
    used = torch.as_tensor(np.arange(wide)[None, :] < need[:, None], device=DEV)
    pages = torch.full((case["seqs"], wide), -1, dtype=torch.int32, device=DEV)
    pages[used] = order[:int(need.sum())]
    i32 = lambda a: torch.as_tensor(np.asarray(a, np.int32), device=DEV)   # noqa: E731
    return dict(lens=i32(lens), row_start=i32(np.concatenate([[0], np.cumsum(rows)])), pages=pages, pool=pool,
                total=int(rows.sum()), n_rows=int(rows.sum()) + case["pad"], longest=int(lens.max()),
                max_rows=int(rows.max()))


def _pool(case, pool):
    P, g, d = case["page"], case["kv_heads"], case["dim"]
    return (pool, g, P, d) if case["order"] == "head" else (pool, P, g, d)


def _by_head(case, t):
    """a pool tensor as [page, head, position, dim], whatever its order in memory"""
    return t if case["order"] == "head" else t.transpose(1, 2)


def _cache(case, t, seed, filled):
    shape, kind = _pool(case, t["pool"]), case["type"]
    scales = (t["pool"], case["kv_heads"], case["page"])
    c = {}
    for salt, name in ((2, "k"), (3, "v")):
        g = _gen(seed, salt)
        if not filled:
            c[name] = torch.zeros(shape, dtype=TYPES[kind], device=DEV)
        elif kind == "i8":
            c[name] = torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=g)
        else:
            c[name] = torch.randn(shape, dtype=TYPES[kind], device=DEV, generator=g)
        if kind == "i8":   # a row's largest value / 127
            c[name + "_scale"] = (2.0 + torch.rand(scales, device=DEV, generator=g)) / 127.0 if filled else \
                torch.zeros(scales, device=DEV)
    return c


def _tree_bits(case, rows):
    """each row's visible rows of its sequence as bits: itself and its ancestors in a tree of branches 4, 3, 1"""
    bits = []
    for n in rows:
        parent = [-1] + [(j - 1) // 4 if j <= 4 else 1 + (j - 5) // 3 if j <= 16 else j - 12 for j in range(1, n)]
        seen = []
        for j in range(n):
            seen.append((seen[parent[j]] if j else 0) | (1 << j))
        bits += seen
    return np.array(bits + [0] * case["pad"], np.uint32)


def prepare(case, seed):
    s = _prepare_rules(case, seed) if case["op"] == "rules" else _prepare_paged(case, seed)
    if own:   # (torch fills the inputs on a stream of its own; the package's waits for no other)
        torch.cuda.synchronize()
    return s


def _prepare_paged(case, seed):
    t = _tables(case, seed)
    g = _gen(seed, 4)
    T, h, kv, d = t["n_rows"], case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case, t=t, cache=_cache(case, t, seed, case["op"] == "attention"))
    if case["op"] == "append":
        # the q | k | v product's rows, fused; each head's queries beside its output gate where the rows are fp32, as
        # a gated attention has them
        s["gated"] = 2 if case["rows_type"] == "f32" else 1
        s["rows"] = (torch.randn(T, (s["gated"] * h + 2 * kv) * d, device=DEV, generator=g) * 1.5).to(TYPES[case["rows_type"]])
        s["q_norm"], s["k_norm"] = (torch.randn(d, device=DEV, generator=g) * 0.02 for _ in range(2))
        half = case["rope"] // 2
        angle = torch.arange(t["longest"], device=DEV, dtype=torch.float64)[:, None] * \
            THETA ** (-torch.arange(half, device=DEV, dtype=torch.float64) / max(half, 1))
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        s["q_out"] = torch.zeros(T, h * d, dtype=TYPES[case["q_type"]], device=DEV)
        s["read"] = torch.cuda.Event()
    else:
        s["q"] = (torch.randn(T, h * d, device=DEV, generator=g) * 1.5).to(TYPES[case["q_type"]])
        s["out"] = torch.zeros(T, h * d, dtype=TYPES[case["q_type"]], device=DEV)
        s["lse"] = torch.zeros(T, h, device=DEV)
        s["scale"] = float(np.float32(d ** -0.5))
        s["visible"] = None
        if case["tree"]:
            bits = _tree_bits(case, _lengths(case)[1])
            s["visible"] = torch.as_tensor(bits.view(np.int32), device=DEV)
    if own:   # the cache's and the batch's descriptions, and the workspace, that a program keeps for its steps
        _descriptions(s)
    return s


def _prepare_rules(case, seed):
    g, r = _gen(seed, 5), np.random.default_rng(seed)
    R, V, shared = case["rows"], case["vocab"], case["shared"]
    i32 = lambda a: torch.as_tensor(np.asarray(a, np.int32), device=DEV)   # noqa: E731
    # a conversation's tokens (its prompt, its answer, then its drafts), most of them from a few hundred; conversations
    # of different lengths
    lens = np.rint(case["history"] * 4.0 ** -np.random.default_rng(R).random(R // shared)).astype(int)
    begin = np.concatenate([[0], np.cumsum(lens + shared - 1)])
    tokens = np.minimum(V - 1, (V * r.random(int(begin[-1])) ** 4)).astype(np.int32)
    end = (begin[:-1] + lens)[:, None] + np.arange(shared)[None, :]   # row i of a chain also sees the drafts before it
    s = dict(case=case, tokens=i32(tokens), begin=i32(np.repeat(begin[:-1], shared)), end=i32(end.reshape(-1)),
             generated=i32(np.repeat(begin[:-1] + lens // 2, shared)),
             total=int((end - begin[:-1, None]).sum()))
    s["logits"] = (torch.randn(R, V, device=DEV, generator=g) * 3.0).to(TYPES[case["type"]])
    f32 = lambda a: torch.as_tensor(np.asarray(a, np.float32), device=DEV)   # noqa: E731
    s["repetition"], s["frequency"], s["presence"] = f32(r.uniform(1.0, 1.3, R)), f32(r.uniform(0, 0.5, R)), f32(r.uniform(0, 1, R))
    nb = case["biases"]
    s["bias_token"], s["bias_value"] = i32(r.integers(0, V, R * nb)), f32(r.uniform(-5, 5, R * nb))
    s["bias_begin"], s["bias_end"] = i32(np.arange(R) * nb), i32(np.arange(1, R + 1) * nb)
    words = -(-V // 32)
    if case["masks"]:   # a grammar leaves a part of the vocabulary; the last row is free
        s["masks"] = torch.randint(-2 ** 31, 2 ** 31, (case["masks"], words), dtype=torch.int32, device=DEV, generator=g) & \
            torch.randint(-2 ** 31, 2 ** 31, (case["masks"], words), dtype=torch.int32, device=DEV, generator=g)
        of = np.arange(R) % case["masks"]
        of[-1] = -1
        s["mask_of"] = i32(of)
    s["out"] = torch.zeros(R, V, device=DEV)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    """One pass. With `own` the call is queued on the package's stream, as a program queues the next one behind it: its
    outputs are whole once that stream has been waited for too (a wait for the whole device)."""
    op = s["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "rules": _own_rules}[op](s)
    return {"append": _plain_append, "attention": _plain_attention, "rules": _plain_rules}[op](s)


def _places(s):
    """of every new row: its sequence, its position, its page and the slot in it"""
    t, P = s["t"], s["case"]["page"]
    row = torch.arange(t["total"], device=DEV)
    seq = torch.searchsorted(t["row_start"], row.to(torch.int32), right=True) - 1
    pos = t["lens"][seq] - t["row_start"][seq + 1] + row
    return seq, pos, t["pages"][seq, pos // P].long(), pos % P


def _split_rows(s):
    """the fused rows' queries, keys and values, [row, head, dim]"""
    case, T = s["case"], s["t"]["total"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    rows = s["rows"][:T]
    q = rows[:, :s["gated"] * h * d].view(T, h, s["gated"] * d)[..., :d]
    k, v = rows[:, s["gated"] * h * d:].view(T, 2, kv, d).unbind(1)
    return q, k, v


def _plain_norm_rotate(s, x, w, pos):
    case = s["case"]
    x = x.float()
    if case["norm"]:
        ss = x.double().square().sum(-1, keepdim=True)
        x = x * (1.0 / torch.sqrt((ss / case["dim"]).float() + EPS)) * (1.0 + w)
    n = case["rope"]
    if n == 0:
        return x
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    if case["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([turned, x[..., n:]], -1)


def _int8_values(s, page, slot):
    """the new rows of the int8 cache as the values they stand for"""
    c = s["cache"]
    return tuple((_by_head(s["case"], c[n])[page, :, slot].float() * c[n + "_scale"][page, :, slot, None]).half()
                 for n in ("k", "v"))


def _plain_append(s):
    case, c = s["case"], s["cache"]
    _, pos, page, slot = _places(s)
    q, k, v = _split_rows(s)
    s["q_out"][:s["t"]["total"]] = _plain_norm_rotate(s, q, s["q_norm"], pos).flatten(1).to(s["q_out"].dtype)
    for name, x in (("k", _plain_norm_rotate(s, k, s["k_norm"], pos)), ("v", v.float())):
        if case["type"] == "i8":
            most = x.abs().amax(-1, keepdim=True)
            inv = torch.where(most > 0, 127.0 / most, torch.zeros_like(most))
            c[name + "_scale"][page, :, slot] = (most / 127.0)[..., 0]
            x = torch.round(x * inv).clamp(-127, 127)
        _by_head(case, c[name])[page, :, slot] = x.to(TYPES[case["type"]])
    if case["type"] == "i8":
        return (s["q_out"],) + _int8_values(s, page, slot)
    return s["q_out"], c["k"], c["v"]


def _plain_attention(s):
    case, t, c = s["case"], s["t"], s["cache"]
    S, h, kv, d, P = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    L, R, T = t["longest"], t["max_rows"], t["total"]
    pos = torch.arange(L, device=DEV)
    page = t["pages"][:, pos // P].clamp(min=0).long()
    seq, row_pos, _, _ = _places(s)
    j = torch.arange(T, device=DEV) - t["row_start"][seq]

    def cached(name):   # [sequence, kv head, position, dim]
        x = _by_head(case, c[name])[page, :, pos % P].float()
        if case["type"] == "i8":
            x = x * c[name + "_scale"][page, :, pos % P][..., None]
        return x.permute(0, 2, 1, 3).contiguous()

    q = torch.zeros(S, R, h, d, device=DEV)
    q[seq, j] = s["q"][:T].view(T, h, d).float()
    q = q.view(S, R, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(S, kv, R * (h // kv), d).contiguous()
    score = torch.matmul(q, cached("k").transpose(2, 3).contiguous()) * s["scale"]
    seen = torch.zeros(S, R, L, dtype=torch.bool, device=DEV)
    if s["visible"] is None:
        seen[seq, j] = pos[None, :] <= row_pos[:, None]
    else:
        first = (t["lens"] - (t["row_start"][1:] - t["row_start"][:-1]))[seq]   # the sequence's first new position
        bit = (pos[None, :] - first[:, None]).clamp(0, 31)
        own_rows = ((s["visible"][:T, None].long() >> bit) & 1).bool()
        seen[seq, j] = (pos[None, :] < first[:, None]) | (own_rows & (pos[None, :] < t["lens"][seq][:, None]))
    score = score.view(S, kv, R, h // kv, L).masked_fill(~seen[:, None, :, None, :], float("-inf"))
    most = score.amax(-1, keepdim=True)
    most = torch.where(most == float("-inf"), torch.zeros_like(most), most)
    weight = torch.exp(score - most)
    del score
    total = weight.sum(-1, keepdim=True)
    value = torch.matmul(weight.view(S, kv, R * (h // kv), L), cached("v")).view(S, kv, R, h // kv, d)
    value = value / torch.where(total > 0, total, torch.ones_like(total))
    back = lambda x: x.permute(0, 2, 1, 3, 4).reshape(S, R, h, -1)[seq, j]   # noqa: E731
    s["out"][:T] = back(value).flatten(1).to(s["out"].dtype)
    s["lse"][:T] = back(torch.log(total) + most)[..., 0]
    return s["out"], s["lse"]


def _plain_rules(s):
    case = s["case"]
    R, V = case["rows"], case["vocab"]
    x = s["logits"].float()
    n = (s["end"] - s["begin"]).long()
    row = torch.repeat_interleave(torch.arange(R, device=DEV), n, output_size=s["total"])
    at = torch.arange(s["total"], device=DEV) - (n.cumsum(0) - n)[row] + s["begin"][row]
    place = row * V + s["tokens"][at].long()
    seen = torch.zeros(R * V, dtype=torch.bool, device=DEV)
    seen[place] = True
    count = torch.zeros(R * V, device=DEV)
    count.scatter_add_(0, place, (at >= s["generated"][row]).float())
    seen, count = seen.view(R, V), count.view(R, V)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0).float()
    if case["biases"]:
        bias = torch.zeros(R * V, device=DEV, dtype=torch.float64)
        bias.scatter_add_(0, torch.arange(R, device=DEV).repeat_interleave(case["biases"]) * V + s["bias_token"].long(),
                          s["bias_value"].double())
        x = x + bias.view(R, V).float()
    if case["masks"]:
        v = torch.arange(V, device=DEV)
        allowed = ((s["masks"][:, v // 32] >> (v % 32).int()) & 1).bool()
        free = (s["mask_of"] < 0)[:, None]
        x = torch.where(free | allowed[s["mask_of"].clamp(min=0).long()], x, torch.full_like(x, float("-inf")))
    s["out"].copy_(x)
    return s["out"]


# ------------------------------------------------------------------ the package's operators
def _descriptions(s):
    import geode_amd as g

    case, t, c = s["case"], s["t"], s["cache"]
    P, kv, d = case["page"], case["kv_heads"], case["dim"]
    s["kv"] = g.GvPagedKv(type=CODES[case["type"]], n_kv_heads=kv, head_dim=d, page_size=P, n_pages=t["pool"],
                          k=c["k"].data_ptr(), v=c["v"].data_ptr(),
                          k_scale=c["k_scale"].data_ptr() if case["type"] == "i8" else None,
                          v_scale=c["v_scale"].data_ptr() if case["type"] == "i8" else None, page_stride=P * kv * d,
                          head_stride=P * d if case["order"] == "head" else d,
                          pos_stride=d if case["order"] == "head" else kv * d)
    s["batch"] = g.GvPagedBatch(n_seqs=case["seqs"], n_rows=t["n_rows"], max_rows=t["max_rows"], max_len=t["longest"],
                                row_start=t["row_start"].data_ptr(), lens=t["lens"].data_ptr(),
                                pages=t["pages"].data_ptr(), ld_pages=t["pages"].shape[1])
    if case["op"] == "attention":
        n = g.lib.gv_paged_attention_workspace_bytes(ctypes.byref(s["kv"]), ctypes.byref(s["batch"]), case["heads"])
        s["ws"] = torch.empty(max(1, n), dtype=torch.uint8, device=DEV)


def _own_append(s):
    import geode_amd as g

    case = s["case"]
    h, kv, d, e = case["heads"], case["kv_heads"], case["dim"], SIZE[case["rows_type"]]
    p, width = s["rows"].data_ptr(), s["rows"].shape[1]
    a = g.GvAppendRows(type=CODES[case["rows_type"]], n_heads=h, q=p, q_row=width, q_head=s["gated"] * d,
                       k=p + s["gated"] * h * d * e, k_row=width, k_head=d,
                       v=p + (s["gated"] * h + kv) * d * e, v_row=width, v_head=d,
                       q_norm=s["q_norm"].data_ptr() if case["norm"] else None,
                       k_norm=s["k_norm"].data_ptr() if case["norm"] else None, eps=EPS, rope_dim=case["rope"],
                       interleaved=int(case["interleaved"]), cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(),
                       n_positions=s["t"]["longest"], positions=None, q_type=CODES[case["q_type"]],
                       q_out=s["q_out"].data_ptr(), q_out_row=h * d)
    if case["type"] == "i8":   # (torch reads the cache on a stream of its own: the pass before has done so)
        s["read"].synchronize()
    g.check(g.lib.gv_paged_append(ctypes.byref(s["kv"]), ctypes.byref(s["batch"]), ctypes.byref(a)), "gv_paged_append")
    if case["type"] == "i8":
        g.check(g.lib.gv_synchronize(), "gv_synchronize")
        _, _, page, slot = _places(s)
        values = _int8_values(s, page, slot)
        s["read"].record()
        return (s["q_out"],) + values
    return s["q_out"], s["cache"]["k"], s["cache"]["v"]


def _own_attention(s):
    import geode_amd as g

    case = s["case"]
    w = case["heads"] * case["dim"]
    a = g.GvAttentionRows(type=CODES[case["q_type"]], n_heads=case["heads"], q=s["q"].data_ptr(), q_row=w,
                          out=s["out"].data_ptr(), out_row=w, lse=s["lse"].data_ptr(), scale=s["scale"],
                          visible=s["visible"].data_ptr() if s["visible"] is not None else None)
    g.check(g.lib.gv_paged_attention(ctypes.byref(s["kv"]), ctypes.byref(s["batch"]), ctypes.byref(a),
                                     s["ws"].data_ptr(), s["ws"].numel()), "gv_paged_attention")
    return s["out"], s["lse"]


def _own_rules(s):
    import geode_amd as g

    case = s["case"]
    R, V = case["rows"], case["vocab"]
    biased, masked = case["biases"] > 0, case["masks"] > 0
    rules = g.GvLogitsRules(repetition=s["repetition"].data_ptr(), frequency=s["frequency"].data_ptr(),
                            presence=s["presence"].data_ptr(), tokens=s["tokens"].data_ptr(),
                            n_tokens=s["tokens"].numel(), begin=s["begin"].data_ptr(),
                            generated=s["generated"].data_ptr(), end=s["end"].data_ptr(),
                            bias_token=s["bias_token"].data_ptr() if biased else None,
                            bias_value=s["bias_value"].data_ptr() if biased else None,
                            n_biases=R * case["biases"], bias_begin=s["bias_begin"].data_ptr() if biased else None,
                            bias_end=s["bias_end"].data_ptr() if biased else None,
                            masks=s["masks"].data_ptr() if masked else None, n_masks=case["masks"],
                            ld_mask=-(-V // 32), mask_of=s["mask_of"].data_ptr() if masked else None)
    g.check(g.lib.gv_process_logits(ctypes.byref(rules), s["logits"].data_ptr(), CODES[case["type"]], V, R, V,
                                    s["out"].data_ptr(), V), "gv_process_logits")
    return s["out"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "rules":
        R, V, per = case["rows"], case["vocab"], case["shared"]
        lens = np.rint(case["history"] * 4.0 ** -np.random.default_rng(R).random(R // per)).astype(int)
        n = int((lens + per - 1).sum())
        by = R * V * (SIZE[case["type"]] + 4) + 4 * n + R * (8 * case["biases"] + 32) + case["masks"] * -(-V // 32) * 4
        return {"bytes": by, "flops": 2 * R * V}
    lens, rows = _lengths(case)
    h, kv, d, T = case["heads"], case["kv_heads"], case["dim"], int(rows.sum())
    cell = d * SIZE[case["type"]] + (4 if case["type"] == "i8" else 0)   # a (position, head)'s key or value
    if case["op"] == "append":
        row = (h + 2 * kv) * d * SIZE[case["rows_type"]] + h * d * SIZE[case["q_type"]] + 2 * kv * cell
        # (rows of different sequences at the same position share its angles, but few are)
        return {"bytes": T * (row + case["rope"] * 4 + 4), "flops": T * (h + kv) * d * (8 if case["norm"] else 4)}
    read = int(lens.sum()) * kv * 2 * cell + int((-(-lens // case["page"])).sum()) * 4
    return {"bytes": read + T * h * (2 * d * SIZE[case["q_type"]] + 4), "flops": 4 * int((lens * rows).sum()) * h * d}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "rules": _exact_rules}[case["op"]](s)


def _exact_append(s):
    case, t = s["case"], s["t"]
    d, n, P = case["dim"], case["rope"], case["page"]
    T, h, kv = t["total"], case["heads"], case["kv_heads"]
    rows = s["rows"].double()
    lens, starts, pages = t["lens"].tolist(), t["row_start"].tolist(), t["pages"].cpu()
    pos, page, slot = [], [], []
    for i in range(case["seqs"]):
        for r in range(starts[i], starts[i + 1]):
            p = lens[i] - starts[i + 1] + r
            pos.append(p), page.append(int(pages[i, p // P])), slot.append(p % P)
    pos = torch.tensor(pos, device=DEV)

    def turned(x, w):
        if case["norm"]:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * (1.0 + w.double())
        y = x.clone()
        for f in range(n // 2):   # one frequency after the other
            i, j = (2 * f, 2 * f + 1) if case["interleaved"] else (f, f + n // 2)
            c, sn = s["cos"][pos, f].double()[:, None], s["sin"][pos, f].double()[:, None]
            y[..., i] = x[..., i] * c - x[..., j] * sn
            y[..., j] = x[..., i] * sn + x[..., j] * c
        return y

    w = s["gated"] * d
    q = torch.stack([rows[:T, i * w:i * w + d] for i in range(h)], 1)
    k = torch.stack([rows[:T, h * w + i * d:h * w + (i + 1) * d] for i in range(kv)], 1)
    v = torch.stack([rows[:T, h * w + (kv + i) * d:h * w + (kv + i + 1) * d] for i in range(kv)], 1)
    q_out = torch.zeros(t["n_rows"], h * d, dtype=torch.float64, device=DEV)
    q_out[:T] = turned(q, s["q_norm"]).reshape(T, h * d)
    k = turned(k, s["k_norm"])
    if case["type"] == "i8":
        step = [x.abs().amax(-1, keepdim=True) / 127.0 for x in (k, v)]
        return (q_out,) + tuple(torch.round(x / u) * u for x, u in zip((k, v), step))
    whole = []
    for x, pool in ((k, s["cache"]["k"]), (v, s["cache"]["v"])):
        pool = pool.double()
        view = pool if case["order"] == "head" else pool.transpose(1, 2)
        view[torch.tensor(page, device=DEV), :, torch.tensor(slot, device=DEV)] = x
        whole.append(pool)
    return q_out, whole[0], whole[1]


def _exact_attention(s):
    case, t, c = s["case"], s["t"], s["cache"]
    h, kv, d, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(t["n_rows"], h, d, dtype=torch.float64, device=DEV)
    lse = torch.zeros(t["n_rows"], h, dtype=torch.float64, device=DEV)
    lens, starts = t["lens"].tolist(), t["row_start"].tolist()
    for i in range(case["seqs"]):
        n, first = lens[i], lens[i] - (starts[i + 1] - starts[i])
        ids = t["pages"][i, :-(-n // P)].long()
        side = {}
        for name in ("k", "v"):
            x = c[name][ids].double()
            x = x if case["order"] == "head" else x.transpose(1, 2)
            if case["type"] == "i8":
                x = x * c[name + "_scale"][ids].double()[..., None]
            side[name] = x.transpose(0, 1).reshape(kv, -1, d)[:, :n]
        for r in range(starts[i], starts[i + 1]):
            j = r - starts[i]
            see = list(range(j + 1)) if s["visible"] is None else [b for b in range(32) if int(s["visible"][r]) >> b & 1]
            keep = torch.zeros(n, dtype=torch.bool, device=DEV)
            keep[:first] = True
            keep[[first + b for b in see]] = True
            q = s["q"][r].double().view(kv, h // kv, d)
            score = (q @ side["k"].transpose(1, 2) * s["scale"]).masked_fill(~keep, float("-inf"))
            p = torch.softmax(score, -1)
            out[r] = (p @ side["v"]).reshape(h, d)
            lse[r] = torch.logsumexp(score, -1).reshape(h)
    return out.flatten(1), lse


def _exact_rules(s):
    case = s["case"]
    V = case["vocab"]
    out = s["logits"].double()
    begin, mid, end = s["begin"].tolist(), s["generated"].tolist(), s["end"].tolist()
    for r in range(case["rows"]):
        x = out[r]
        tok = s["tokens"][begin[r]:end[r]].long()
        used = tok.unique()
        rep = s["repetition"][r].double()
        x[used] = torch.where(x[used] > 0, x[used] / rep, x[used] * rep)
        made = torch.bincount(s["tokens"][max(begin[r], mid[r]):end[r]].long(), minlength=V)
        x -= s["frequency"][r].double() * made + s["presence"][r].double() * (made > 0)
        if case["biases"]:
            at = slice(r * case["biases"], (r + 1) * case["biases"])
            x.index_put_((s["bias_token"][at].long(),), s["bias_value"][at].double(), accumulate=True)
        if case["masks"] and int(s["mask_of"][r]) >= 0:
            words = s["masks"][int(s["mask_of"][r])].cpu().numpy().view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:V]
            x[torch.as_tensor(bits == 0, device=DEV)] = float("-inf")
    return out
