"""Cases, plain forms and exact values of the paged-cache operators: forking,
copying and compacting pages, writing a step's keys and values, and attention
for a batch whose sequences share a prefix.

A pool holds keys and values as [layers][pages][kv heads][page tokens][dims];
a sequence is a length and a list of pages, and pages are handed out lowest
free number first, so page numbers are part of the result.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LAYER = 1  # the layer of a two-layer pool that write and attend work on


def listed():
    return [
        # two verdicts asked of one prompt that has just been read: the smallest fork, all launch latency
        _pages("fork_two", "fork", "f16", 26, 8, 128, 16, parents=1, each=2, lo=293, hi=293, pick=1),
        # a policy prompt forked for 256 requests, whose last page is 28 of 64 rows full
        _pages("fork_wide", "fork", "f16", 26, 8, 128, 64, parents=1, each=256, lo=1500, hi=1500, pick=2),
        # 24 conversations moved to pages of their own, the old ones dropped, the pool packed down again
        _pages("copy_compact", "compact", "bf16", 26, 8, 128, 32, parents=24, each=1, lo=200, hi=1000, pick=3),
        # one layer's rows of a decode step of 64 sequences, from the model's f32 activations
        _write("write_step", "f16", "f32", 8, 128, 64, seqs=64, new=1, before=700, pick=4),
        # one layer's rows of a micro-batch of prompts, from a fused projection's output
        _write("write_prompts", "bf16", "bf16", 8, 128, 64, seqs=16, new=1024, before=37, pick=5),
        # one token of one short conversation: latency alone
        _attend("attend_one", "f16", 32, 8, 128, 64, groups=1, each=1, prefix=0, own_len=(300, 300), new=(1, 1), pick=6),
        # one request of 256 tokens read at once
        _attend("attend_prompt", "f16", 32, 8, 128, 64, groups=1, each=1, prefix=0, own_len=(256, 256), new=(256, 256), pick=7),
        # a decode step of 128 conversations under one long policy
        _attend("step_shared", "f16", 32, 8, 128, 64, groups=1, each=128, prefix=8192, own_len=(1, 256), new=(1, 1), pick=8),
        # a decode step of unrelated long conversations
        _attend("step_long", "bf16", 32, 8, 128, 64, groups=24, each=1, prefix=0, own_len=(2000, 16384), new=(1, 1), pick=9),
        # drafts of up to 5 tokens checked under four policies, 7 query heads to a kv head
        _attend("drafts_groups", "bf16", 14, 2, 64, 16, groups=4, each=12, prefix=2741, own_len=(5, 400), new=(1, 5), pick=10),
        # a micro-batch of requests around 300 tokens behind one system prompt
        _attend("prompts_shared", "f16", 32, 8, 128, 64, groups=1, each=32, prefix=1500, own_len=(32, 900), new=(32, 900), pick=11),
        # long documents read at once
        _attend("prompts_long", "bf16", 32, 8, 128, 128, groups=3, each=1, prefix=0, own_len=(4096, 4096), new=(4096, 4096), pick=12),
    ]


def _pages(name, op, type, layers, kv_heads, dim, page, parents, each, lo, hi, pick):
    return {"name": name, "op": op, "type": type, "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page,
            "parents": parents, "each": each, "lo": lo, "hi": hi, "pick": pick}


def _write(name, type, src, kv_heads, dim, page, seqs, new, before, pick):
    return {"name": name, "op": "write", "type": type, "src": src, "kv_heads": kv_heads, "dim": dim, "page": page,
            "seqs": seqs, "new": new, "before": before, "pick": pick}


def _attend(name, type, heads, kv_heads, dim, page, groups, each, prefix, own_len, new, pick):
    return {"name": name, "op": "attend", "type": type, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "groups": groups, "each": each, "prefix": prefix, "own_lo": own_len[0], "own_hi": own_len[1],
            "new_lo": new[0], "new_hi": new[1], "pick": pick}


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """Another case of the same ranges."""
    kind = rng.choice(("fork", "compact", "write", "step", "step", "drafts", "prompts", "prompts"))
    pick, type, page = rng.randrange(1 << 30), rng.choice(("f16", "bf16")), rng.choice((16, 32, 64, 128))
    if kind in ("fork", "compact"):
        parents = _log(rng, 1, 16)
        c = _pages("", kind, type, _log(rng, 2, 26), rng.choice((2, 4, 8)), rng.choice((64, 128)), page, parents,
                   each=_log(rng, 1, max(1, 192 // parents)) if kind == "fork" else 1, lo=_log(rng, 1, 200), hi=0, pick=pick)
        c["hi"] = c["lo"] + _log(rng, 1, 1000)
    elif kind == "write":
        c = _write("", type, rng.choice(("f32", type)), rng.choice((1, 2, 5, 8)), rng.choice((64, 128)), page,
                   seqs=_log(rng, 1, 128), new=1, before=_log(rng, 1, 900), pick=pick)
        c["new"] = _log(rng, 1, 8192 // c["seqs"])
    else:
        dim = rng.choice((64, 128, 128))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 3, 4, 7, 8) if kv_heads < 8 else (1, 4))
        groups = rng.choice((1, 1, 2, 3))
        each = _log(rng, 1, {"step": 40, "drafts": 16, "prompts": 8}[kind])
        prefix = _log(rng, 16, {"step": 8192, "drafts": 3000, "prompts": 1500}[kind]) if each > 1 or rng.random() < 0.5 else 0
        lo = _log(rng, 1, 300)
        hi = lo + _log(rng, 1, {"step": 900, "drafts": 400, "prompts": 700}[kind])
        new = {"step": (1, 1), "drafts": (1, 6), "prompts": (lo, hi)}[kind]
        c = _attend("", type, heads, kv_heads, dim, page, groups, each, prefix, (max(lo, new[0]), hi), new, pick)
    del c["name"]
    return c


# ------------------------------------------------------------ page numbers

def _lens(case, n):
    rng = random.Random(case["pick"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(n)]


def _attend_shape(case):
    """Per sequence: its group, its own length behind the prefix, and the new tokens at its end."""
    rng = random.Random(case["pick"])
    rows = []
    for g in range(case["groups"]):
        for _ in range(case["each"]):
            length = _log(rng, case["own_lo"], case["own_hi"])
            new = length if case["new_hi"] >= case["own_lo"] and case["new_hi"] == case["own_hi"] else min(
                length, rng.randint(case["new_lo"], case["new_hi"]))
            rows.append((g, length, new))
    return rows


class _Numbers:
    """Page numbers of a fresh pool: lowest free first, nothing freed."""

    def __init__(self):
        self.used = 0

    def take(self, n):
        got = list(range(self.used, self.used + n))
        self.used += n
        return got


def _attend_tables(case):
    """Page lists and lengths of the batch's sequences, and the pages used."""
    pt, numbers, lists, lens = case["page"], _Numbers(), [], []
    shape = _attend_shape(case)
    parents = [numbers.take(-(-case["prefix"] // pt)) for _ in range(case["groups"])] if case["prefix"] else [[]] * case["groups"]
    for g, _, _ in shape:  # every fork first, then every extension
        whole = case["prefix"] // pt
        lists.append(parents[g][:whole] + (numbers.take(1) if case["prefix"] % pt else []))
    for i, (_, length, _) in enumerate(shape):
        lens.append(case["prefix"] + length)
        lists[i] += numbers.take(-(-lens[i] // pt) - len(lists[i]))
    return lists, lens, numbers.used


def _padded(lists):
    out = np.full((len(lists), max(map(len, lists))), -1, np.int32)
    for i, p in enumerate(lists):
        out[i, :len(p)] = p
    return out


# ----------------------------------------------------------------- prepare

def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return {"fork": _prepare_pages, "compact": _prepare_pages, "write": _prepare_write, "attend": _prepare_attend}[case["op"]](case, gen)


def _pool(s, case, layers, pages, gen):
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    for name in ("k", "v"):
        s[name] = torch.empty(shape, dtype=TYPES[case["type"]], device="cuda").normal_(generator=gen)
    s.update(case=case, op=case["op"], pt=case["page"], type=TYPES[case["type"]], pages=pages)
    if own:
        from llm_shield_b200 import binding
        s["ctx"] = binding.ShieldContext(1)
        s["stream"] = torch.cuda.current_stream().cuda_stream
        s["kv"] = s["ctx"].kv_create(case["type"], layers, case["kv_heads"], case["dim"], case["page"], pages,
                                     k=s["k"].data_ptr(), v=s["v"].data_ptr())


def _prepare_pages(case, gen):
    s, pt = {}, case["page"]
    lens = _lens(case, case["parents"])
    held = sum(-(-n // pt) for n in lens)
    _pool(s, case, case["layers"], held + (held if case["op"] == "compact" else case["parents"] * case["each"]), gen)
    numbers = _Numbers()
    s["lists"] = _padded([numbers.take(-(-n // pt)) for n in lens])  # the live sequences' pages
    s["lens"] = np.array(lens, np.int32)
    s["ref"] = np.zeros(s["pages"], np.int32)
    s["ref"][:numbers.used] = 1
    s["from"] = np.repeat(np.arange(case["parents"]), case["each"])  # a child's parent
    if own:
        s["seqs"] = s["ctx"].kv_open(s["kv"], case["parents"])
        s["ctx"].kv_extend(s["kv"], s["seqs"], s["lens"])
        s["parents"] = s["seqs"][s["from"]]
    return s


def _prepare_write(case, gen):
    s, pt, n, new, before = {}, case["page"], case["seqs"], case["new"], case["before"]
    rng = random.Random(case["pick"])
    had = [rng.randint(0, before) for _ in range(n)]
    numbers = _Numbers()
    lists = [numbers.take(-(-h // pt)) for h in had]
    for i, h in enumerate(had):
        lists[i] += numbers.take(-(-(h + new) // pt) - len(lists[i]))
    _pool(s, case, LAYER + 1, numbers.used, gen)
    at = [(lists[i][p // pt], p % pt) for i, h in enumerate(had) for p in range(h, h + new)]
    s["page_of"], s["row_of"] = torch.tensor(at, dtype=torch.int64, device="cuda").unbind(1)
    # keys and values lie in one projection's rows, as a fused Q/K/V product leaves them
    H, D = case["kv_heads"], case["dim"]
    fused = torch.empty(n * new, 3 * H * D, dtype=TYPES[case["src"]], device="cuda").normal_(generator=gen)
    s["k_new"], s["v_new"] = (fused[:, j * H * D:(j + 1) * H * D].unflatten(1, (H, D)) for j in (1, 2))
    if own:
        c = s["ctx"]
        seqs = c.kv_open(s["kv"], n)
        c.kv_extend(s["kv"], seqs, had)
        c.kv_extend(s["kv"], seqs, [new] * n)
        s["batch"] = c.kv_batch_create(s["kv"], n_heads=H, max_tokens=n * new, max_seqs=n, max_positions=before + new)
        c.kv_batch_set(s["batch"], seqs, [new] * n, stream=s["stream"])
    return s


def _prepare_attend(case, gen):
    s, pt = {}, case["page"]
    shape = _attend_shape(case)
    lists, lens, used = _attend_tables(case)
    _pool(s, case, LAYER + 1, used, gen)
    new = [r[2] for r in shape]
    T, n, longest = sum(new), len(shape), max(lens)
    s["q"] = torch.empty(T, case["heads"], case["dim"], dtype=s["type"], device="cuda").normal_(generator=gen)
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = case["dim"] ** -0.5
    # where each position of each sequence lies (positions behind its end: page 0, never seen), and
    # which (sequence, place among its new tokens) each packed token is
    pages = np.maximum(_padded(lists), 0)
    pos = np.minimum(np.arange(longest), np.array(lens)[:, None] - 1)
    seq = np.repeat(np.arange(n), new)
    place = np.concatenate([np.arange(m) for m in new])
    packed = np.zeros((n, max(new)), np.int64)
    packed[seq, place] = np.arange(T)
    last = np.array(lens)[:, None] - np.array(new)[:, None] + np.arange(max(new))  # position of a new token
    for name, v in (("page_of", np.take_along_axis(pages, pos // pt, 1)), ("row_of", pos % pt), ("seq_of", seq),
                    ("place_of", place), ("packed", packed), ("last", last)):
        s[name] = torch.tensor(v, dtype=torch.int64, device="cuda")
    if own:
        c = s["ctx"]
        seqs = None
        if case["prefix"]:
            parents = c.kv_open(s["kv"], case["groups"])
            c.kv_extend(s["kv"], parents, [case["prefix"]] * case["groups"])
            seqs = c.kv_fork(s["kv"], parents[[r[0] for r in shape]], stream=s["stream"])
            # the fork copied rows of the prefix's last page: every row of the pool is as it was drawn again
            gen.manual_seed(gen.initial_seed())
            for name in ("k", "v"):
                s[name].normal_(generator=gen)
        else:
            seqs = c.kv_open(s["kv"], n)
        c.kv_extend(s["kv"], seqs, [r[1] for r in shape])
        s["batch"] = c.kv_batch_create(s["kv"], n_heads=case["heads"], max_tokens=T, max_seqs=n, max_positions=longest)
        c.kv_batch_set(s["batch"], seqs, new, stream=s["stream"])
    return s


# --------------------------------------------------------------------- run

def run(s):
    return {"fork": _fork, "compact": _compact, "write": _write_rows, "attend": _attention}[s["op"]](s)


def _rows_to(pool, dst, src, rows):
    """Rows [0, rows[i]) of page dst[i] become those of page src[i], in every layer and head."""
    keep = torch.arange(pool.shape[3], device="cuda") < torch.as_tensor(rows, device="cuda")[:, None]
    dst, src = (torch.as_tensor(x, device="cuda") for x in (dst, src))
    pool[:, dst] = torch.where(keep[None, :, None, :, None], pool[:, src], pool[:, dst])


def _fork(s):
    """Every parent forked for its children, who are then freed again."""
    if own:
        c, kv = s["ctx"], s["kv"]
        kids = c.kv_fork(kv, s["parents"], stream=s["stream"])
        pages = c.kv_pages(kv, kids)
        c.kv_free(kv, kids)
        return {"k": s["k"], "v": s["v"], "pages": pages}
    pages, lens = s["lists"][s["from"]], s["lens"][s["from"]]
    tail = np.flatnonzero(lens % s["pt"])
    if len(tail):
        src = pages[tail, lens[tail] // s["pt"]]
        dst = np.flatnonzero(s["ref"] == 0)[:len(tail)]
        pages[tail, lens[tail] // s["pt"]] = dst
        _rows_to(s["k"], dst, src, lens[tail] % s["pt"])
        _rows_to(s["v"], dst, src, lens[tail] % s["pt"])
    return {"k": s["k"], "v": s["v"], "pages": pages}


def _compact(s):
    """Every sequence copied to pages of its own, the old ones freed, the pool compacted."""
    if own:
        c, kv = s["ctx"], s["kv"]
        moved = c.kv_copy(kv, s["seqs"], stream=s["stream"])
        c.kv_free(kv, s["seqs"])
        c.kv_compact(kv, stream=s["stream"])
        s["seqs"] = moved
        return {"k": s["k"], "v": s["v"], "pages": c.kv_pages(kv, moved)}
    held = s["lists"] >= 0
    src = s["lists"][held]
    dst = np.flatnonzero(s["ref"] == 0)[:len(src)]
    rows = np.minimum(s["lens"][:, None] - np.arange(held.shape[1]) * s["pt"], s["pt"])[held]
    _rows_to(s["k"], dst, src, rows)
    _rows_to(s["v"], dst, src, rows)
    s["ref"][src], s["ref"][dst] = 0, 1
    free, used = np.flatnonzero(s["ref"] == 0), dst[::-1]  # dst goes up: used goes down
    m = min(len(free), len(used))
    down = np.flatnonzero(free[:m] < used[:m])
    _rows_to(s["k"], free[down], used[down], rows[::-1][down])
    _rows_to(s["v"], free[down], used[down], rows[::-1][down])
    s["ref"][used[down]], s["ref"][free[down]] = 0, 1
    at = dst.copy()
    at[::-1][down] = free[down]
    s["lists"] = s["lists"].copy()
    s["lists"][held] = at
    return {"k": s["k"], "v": s["v"], "pages": s["lists"]}


def _write_rows(s):
    """The new tokens' keys and values into their rows of one layer."""
    if own:
        s["ctx"].kv_write(s["batch"], LAYER, s["k_new"].data_ptr(), s["v_new"].data_ptr(), s["case"]["src"],
                          k_stride=s["k_new"].stride(0), v_stride=s["v_new"].stride(0), stream=s["stream"])
        return {"k": s["k"], "v": s["v"]}
    s["k"][LAYER][s["page_of"], :, s["row_of"]] = s["k_new"].to(s["type"])
    s["v"][LAYER][s["page_of"], :, s["row_of"]] = s["v_new"].to(s["type"])
    return {"k": s["k"], "v": s["v"]}


def _attention(s):
    """One layer's attention of every new token over its sequence, itself included."""
    if own:
        s["ctx"].kv_attend(s["batch"], LAYER, s["q"].data_ptr(), s["out"].data_ptr(), s["scale"], stream=s["stream"])
        return s["out"]
    k = s["k"][LAYER][s["page_of"], :, s["row_of"]].float()  # sequences, positions, kv heads, dims
    v = s["v"][LAYER][s["page_of"], :, s["row_of"]].float()
    q = s["q"][s["packed"]].float()
    q = q.unflatten(2, (k.shape[2], -1))  # sequences, new tokens, kv heads, heads of a group, dims
    seen = torch.arange(k.shape[1], device="cuda") <= s["last"][:, :, None]
    x = torch.einsum("nqhgd,nlhd->nhgql", q, k) * s["scale"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    x = x / x.sum(-1, keepdim=True)
    o = torch.einsum("nhgql,nlhd->nqhgd", x, v).flatten(2, 3)
    return o[s["seq_of"], s["place_of"]].to(s["type"])


# -------------------------------------------------------------------- work

def work(case):
    size = 4 if case.get("src") == "f32" else 2
    row = case["kv_heads"] * case["dim"]
    if case["op"] in ("fork", "compact"):
        per_row = 2 * case["layers"] * row * 2
        lens = _lens(case, case["parents"])
        if case["op"] == "compact":  # every row out and back
            return {"bytes": 4 * sum(lens) * per_row, "flops": 0}
        tails = [n % case["page"] for n in lens]
        return {"bytes": sum(t * (1 + case["each"]) for t in tails) * per_row or 1, "flops": 0}
    if case["op"] == "write":
        return {"bytes": 2 * case["seqs"] * case["new"] * row * (size + 2), "flops": 0}
    shape = _attend_shape(case)
    pairs = sum(n * (case["prefix"] + length - n) + n * (n + 1) // 2 for _, length, n in shape)
    keys = case["groups"] * case["prefix"] + sum(r[1] for r in shape)
    tokens = sum(r[2] for r in shape)
    return {"bytes": 2 * (2 * keys * row + 2 * tokens * case["heads"] * case["dim"]),
            "flops": 4 * case["heads"] * case["dim"] * pairs}


# ------------------------------------------------------------------- exact

def exact(case, seed):
    """The values in 64 bits, sequence by sequence."""
    s = _plain_state(case, seed)
    if case["op"] == "attend":
        return _exact_attention(case, s)
    if case["op"] == "write":
        k, v = s["k"].double(), s["v"].double()
        for t, (p, r) in enumerate(zip(s["page_of"].tolist(), s["row_of"].tolist())):
            k[LAYER, p, :, r], v[LAYER, p, :, r] = s["k_new"][t].double(), s["v_new"][t].double()
        return {"k": k, "v": v}
    k, v, pt = s["k"].clone(), s["v"].clone(), case["page"]
    lists = [[p for p in row if p >= 0] for row in s["lists"].tolist()]
    free = sorted(set(range(s["pages"])) - {p for row in lists for p in row})
    lens = s["lens"].tolist()

    def move(src, dst, rows):
        for x in (k, v):
            x[:, dst, :, :rows] = x[:, src, :, :rows]

    kids = []
    for i in s["from"].tolist():
        kid = []
        for j, p in enumerate(lists[i]):
            rows = min(pt, lens[i] - j * pt)
            if case["op"] == "fork" and rows == pt:
                kid.append(p)
            else:
                kid.append(free.pop(0))
                move(p, kid[-1], rows)
        kids.append(kid)
    if case["op"] == "compact":
        free = sorted(free + [p for row in lists for p in row])
        where = {p: (i, j) for i, row in enumerate(kids) for j, p in enumerate(row)}
        while free and free[0] < max(where):
            top = max(where)
            i, j = where.pop(top)
            kids[i][j] = free.pop(0)
            move(top, kids[i][j], min(pt, lens[i] - j * pt))
            where[kids[i][j]] = (i, j)
    return {"k": k.double(), "v": v.double(), "pages": None}


def _plain_state(case, seed):
    """prepare()'s tensors without handles of the framework."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _exact_attention(case, s):
    lists, lens, _ = _attend_tables(case)
    out, t, pt, H = [], 0, case["page"], case["kv_heads"]
    for (_, _, new), pages, n in zip(_attend_shape(case), lists, lens):
        pages = torch.tensor(pages, device="cuda")
        k, v = (s[x][LAYER][pages].double().transpose(1, 2).flatten(0, 1)[:n] for x in ("k", "v"))  # positions, heads, dims
        q = s["q"][t:t + new].double()
        rows = torch.empty(new, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        pos = torch.arange(n - new, n, device="cuda")
        for h in range(case["heads"]):
            g = h * H // case["heads"]
            e = q[:, h] @ k[:, g].T / math.sqrt(case["dim"])
            e[torch.arange(n, device="cuda")[None] > pos[:, None]] = -math.inf
            rows[:, h] = torch.softmax(e, -1) @ v[:, g]
        out.append(rows)
        t += new
    return torch.cat(out)
