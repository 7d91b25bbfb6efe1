"""Paged-cache operators on the GPU, through the C ABI: pages forked, copied
and compacted, rows written, and attention over shared and private pages
against the definition in 64 bits."""
from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import pytest

from llm_shield_b200 import binding

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


class Cache:
    """A context, a pool in torch memory, and the pages' contents by name."""

    def __init__(self, type="f16", layers=2, kv_heads=2, dim=64, pt=16, pages=64, fill=1.0, seed=0):
        self.ctx = binding.ShieldContext(1)
        self.type, self.pt, self.dim, self.kv_heads, self.layers = type, pt, dim, kv_heads, layers
        self.dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[type]
        gen = torch.Generator("cuda").manual_seed(seed)
        shape = (layers, pages, kv_heads, pt, dim)
        self.k = torch.empty(shape, dtype=self.dtype, device="cuda").normal_(generator=gen)
        self.v = torch.empty(shape, dtype=self.dtype, device="cuda").normal_(generator=gen)
        self.gen = gen
        self.stream = torch.cuda.current_stream().cuda_stream
        self.kv = self.ctx.kv_create(type, layers, kv_heads, dim, pt, pages, k=self.k.data_ptr(), v=self.v.data_ptr())

    def rows(self, seq, layer, pool):
        """Positions x heads x dims of one sequence."""
        n = int(self.ctx.kv_lengths(self.kv, [seq])[0])
        pages = torch.from_numpy(self.ctx.kv_pages(self.kv, [seq])[0]).long().cuda()
        return pool[layer][pages].transpose(1, 2).flatten(0, 1)[:n]

    def batch(self, seqs, counts, heads, **caps):
        lens = self.ctx.kv_lengths(self.kv, seqs)
        caps = dict(dict(max_tokens=max(1, int(sum(counts))), max_seqs=max(1, len(seqs)), max_positions=max(1, int(lens.max(initial=1)))), **caps)
        b = self.ctx.kv_batch_create(self.kv, heads, **caps)
        self.ctx.kv_batch_set(b, seqs, counts, stream=self.stream)
        return b


def tree(c, rng, roots, kids, lo, hi, own_lo, own_hi, whole=0.5):
    """Sequences forked from roots of lo..hi positions and extended by own_lo..own_hi."""
    top = c.ctx.kv_open(c.kv, roots)
    c.ctx.kv_extend(c.kv, top, [rng.randint(lo, hi) for _ in top])
    ids = np.repeat(top, kids)
    lens = [int(c.ctx.kv_lengths(c.kv, [i])[0]) for i in ids]
    leaves = c.ctx.kv_fork(c.kv, ids, [n if rng.random() < whole else rng.randint(0, n) for n in lens], stream=c.stream)
    c.ctx.kv_extend(c.kv, leaves, [rng.randint(own_lo, own_hi) for _ in leaves])
    return leaves


def expect(c, seqs, counts, q, layer, scale):
    """The definition in 64 bits, and how far a kernel may be from it.

    With u = eps / 2 the half step of the type: a weight is rounded once (u),
    as is the output (u |o|). A score is a sum of dim products in f32; each of
    its roundings is at most 2^-23 of the sum of magnitudes (tensor cores may
    truncate), and scaling, subtracting the maximum and the exponential add a
    few 2^-23 of the score; a score's error enters a weight as the factor
    exp(error), above and below the line. Sums over n weights in f32 add
    n 2^-23. The weights' errors act on sum w |v|.
    """
    outs, tols, t = [], [], 0
    u = torch.finfo(c.dtype).eps / 2
    for s, m in zip(seqs, counts):
        if m == 0:
            continue
        k, v = c.rows(s, layer, c.k).double(), c.rows(s, layer, c.v).double()
        n, heads = k.shape[0], q.shape[1]
        k, v = (x.repeat_interleave(heads // x.shape[1], 1).transpose(0, 1) for x in (k, v))  # heads, positions, dims
        x = q[t:t + m].double().transpose(0, 1)
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
        e = (x @ k.transpose(1, 2)) * scale
        size = ((x.abs() @ k.abs().transpose(1, 2)) * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
        err = size * (c.dim + 8) * 2.0 ** -23
        w = torch.softmax(e.masked_fill(hidden, -math.inf), -1)
        o = w @ v
        tol = (u + 2 * err + (n + 8) * 2.0 ** -23) * (w @ v.abs()) * 1.01 + u * o.abs() + torch.finfo(c.dtype).tiny
        outs.append(o.transpose(0, 1))
        tols.append(tol.transpose(0, 1))
        t += m
    return torch.cat(outs), torch.cat(tols)


def check(c, seqs, counts, heads, layer=1, scale=None, sharp=1.0, batch=None):
    scale = c.dim ** -0.5 if scale is None else scale
    T = int(sum(counts))
    # queries inside wider rows, outputs too; rows behind the last token stay as they are
    q = torch.empty(T + 2, heads + 3, c.dim, dtype=c.dtype, device="cuda").normal_(0, sharp, generator=c.gen)[:, 1:heads + 1]
    out = torch.full((T + 3, heads + 1, c.dim), 7.0, dtype=c.dtype, device="cuda")
    b = c.batch(seqs, counts, heads) if batch is None else batch
    c.ctx.kv_attend(b, layer, q.data_ptr(), out.data_ptr(), scale, q_stride=q.stride(0), out_stride=out.stride(0), stream=c.stream)
    assert (out[T:] == 7).all() and (out[:, heads:] == 7).all()
    want, tol = expect(c, seqs, counts, q, layer, scale)
    got = out[:T, :heads].double()
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1, f"{worst} times the tolerance"
    return out[:T, :heads].clone()


# (type, dim, page tokens, kv heads, query heads)
SHAPES = [("f16", 128, 64, 8, 32), ("bf16", 128, 16, 2, 8), ("f16", 64, 32, 2, 14), ("bf16", 64, 128, 1, 1),
          ("f16", 128, 128, 1, 20), ("bf16", 128, 32, 3, 3), ("bf16", 64, 64, 2, 34)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("step", ["one", "drafts", "prompts", "mixed", "first"])
def test_attention_against_64_bits(shape, step):
    type, dim, pt, kv_heads, heads = shape
    rng = random.Random(f"{shape}{step}")
    c = Cache(type, 2, kv_heads, dim, pt, pages=-(-40000 // pt), seed=rng.randrange(1000))
    if step == "first":  # prompts of 1, 2, .. positions and nothing before them
        seqs = c.ctx.kv_open(c.kv, 9)
        counts = [1, 2, 15, 16, 17, 127, 128, 129, 333]
        c.ctx.kv_extend(c.kv, seqs, counts)
    else:
        seqs = tree(c, rng, roots=2, kids=6, lo=1, hi=1200, own_lo=1, own_hi=300)
        seqs = np.concatenate([seqs, tree(c, rng, roots=3, kids=1, lo=1, hi=3000, own_lo=1, own_hi=20)])
        lens = c.ctx.kv_lengths(c.kv, seqs)
        top = {"one": 1, "drafts": 7, "prompts": 10 ** 6, "mixed": 40}[step]
        counts = [min(int(n), top) if step in ("one", "prompts") else min(int(n), rng.randint(0, top)) for n in lens]
    check(c, seqs, counts, heads)


@pytest.mark.parametrize("shape", SHAPES[:4], ids=lambda s: "-".join(map(str, s)))
def test_long_prefix_shared_by_many(shape):
    type, dim, pt, kv_heads, heads = shape
    rng = random.Random(str(shape))
    c = Cache(type, 2, kv_heads, dim, pt, pages=-(-60000 // pt))
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [9000 + 13])
    seqs = c.ctx.kv_fork(c.kv, [root] * 50, stream=c.stream)
    c.ctx.kv_extend(c.kv, seqs, [rng.randint(1, 700) for _ in seqs])
    check(c, seqs, [1] * 50, heads)
    check(c, seqs, [rng.randint(1, 5) for _ in seqs], heads, sharp=4.0)
    order = rng.sample(range(50), 17)
    check(c, seqs[order], [1 + i % 3 for i in range(17)], heads, scale=-0.3)


def test_the_same_plan_gives_the_same_bits():
    c = Cache("f16", 2, 8, 128, 64, pages=400)
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [5000])
    seqs = c.ctx.kv_fork(c.kv, [root] * 20, stream=c.stream)
    c.ctx.kv_extend(c.kv, seqs, range(1, 21))
    b = c.batch(seqs, [1] * 20, 32)
    q = torch.randn(20, 32, 128, device="cuda").half()
    outs = [torch.empty_like(q) for _ in range(3)]
    for o in outs:
        c.ctx.kv_attend(b, 0, q.data_ptr(), o.data_ptr(), 0.1, stream=c.stream)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    mine = q.clone()  # the output may take the queries' place
    c.ctx.kv_attend(b, 0, mine.data_ptr(), mine.data_ptr(), 0.1, stream=c.stream)
    assert torch.equal(mine, outs[0])


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("new", [3, 150])
def test_what_a_row_may_not_see_has_no_effect(type, bad, new):
    c = Cache(type, 1, 2, 128, 32, pages=64)
    seqs = c.ctx.kv_open(c.kv, 2)
    c.ctx.kv_extend(c.kv, seqs, [200, 333])
    pages = c.ctx.kv_pages(c.kv, seqs)
    held = torch.zeros(c.k.shape[1], c.pt, dtype=torch.bool, device="cuda")
    for row, n in zip(pages, (200, 333)):
        for p in range(n):
            held[int(row[p // c.pt]), p % c.pt] = True
    for pool in (c.k, c.v):  # pages and rows that no sequence holds
        pool.masked_fill_(~held[None, :, None, :, None], bad)
    check(c, seqs, [new, new], 8, layer=0)
    # and positions behind a row's own
    first = new // 2
    at = 200 - new + first
    c.k[0, int(pages[0][at // c.pt]), :, at % c.pt] = bad
    c.v[0, int(pages[0][at // c.pt]), 1, at % c.pt, ::3] = bad
    q = torch.randn(2 * new, 8, 128, device="cuda").to(c.dtype)
    out = torch.empty_like(q)
    b = c.batch(seqs, [new, new], 8)
    c.ctx.kv_attend(b, 0, q.data_ptr(), out.data_ptr(), 128 ** -0.5, stream=c.stream)
    want, tol = expect(c, seqs, [new, new], torch.nan_to_num(q), 0, 128 ** -0.5)
    blind = torch.ones(2 * new, dtype=torch.bool, device="cuda")
    blind[first:new] = False
    assert torch.isfinite(out[blind]).all()
    assert not torch.isfinite(out[first:new]).all(-1).any()  # an infinite or undefined score takes the row
    # a value alone: its dims and only those, in the rows that see it
    c.k[0, int(pages[0][at // c.pt]), :, at % c.pt] = 0.25
    c.ctx.kv_attend(b, 0, q.data_ptr(), out.data_ptr(), 128 ** -0.5, stream=c.stream)
    hit = torch.zeros(2 * new, 8, 128, dtype=torch.bool, device="cuda")
    hit[first:new, 4:, ::3] = True
    assert torch.equal(~torch.isfinite(out), hit)
    if math.isinf(bad):
        assert (out[hit] == bad).all()
    c.v[0, int(pages[0][at // c.pt]), 1, at % c.pt, ::3] = 0.0
    want, tol = expect(c, seqs, [new, new], q, 0, 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol)[~hit].all()


def test_extreme_scores():
    """Scores of the type's largest values, equal scores, and a lone key far above the others."""
    c = Cache("f16", 1, 1, 64, 16, pages=256)
    (s,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [s], [900])
    c.k.fill_(0)
    check(c, [s], [5], 4, layer=0)  # every weight 1 / n
    page = int(c.ctx.kv_pages(c.kv, [s])[0][40])
    c.k[0, page, 0, 3] = 30.0
    check(c, [s], [5], 4, layer=0, sharp=3.0)
    c.k.fill_(60000.0)
    check(c, [s], [2], 4, layer=0, scale=1e-9)
    c.k.normal_(0, 40.0, generator=c.gen)
    check(c, [s], [200], 4, layer=0)


def test_offsets_beyond_32_bits():
    """The last layer of a pool of more than 2^32 bytes, through its last pages."""
    c = Cache.__new__(Cache)
    c.ctx, c.type, c.pt, c.dim, c.kv_heads, c.layers, c.dtype = binding.ShieldContext(1), "f16", 64, 128, 2, 9, torch.float16
    pages = 20000  # 9 * 20000 * 2 * 64 * 128 = 2.9e9 elements
    c.k = torch.empty(9, pages, 2, 64, 128, dtype=c.dtype, device="cuda")
    c.v = torch.empty_like(c.k)
    c.gen = torch.Generator("cuda").manual_seed(1)
    c.stream = torch.cuda.current_stream().cuda_stream
    c.kv = c.ctx.kv_create("f16", 9, 2, 128, 64, pages, k=c.k.data_ptr(), v=c.v.data_ptr())
    (low, s) = c.ctx.kv_open(c.kv, 2)
    c.ctx.kv_extend(c.kv, [low], [64 * (pages - 24)])
    c.ctx.kv_extend(c.kv, [s], [700])
    seqs = c.ctx.kv_fork(c.kv, [s] * 6, stream=c.stream)
    c.ctx.kv_extend(c.kv, seqs, [60, 1, 2, 3, 4, 5])
    c.k[8, pages - 24:].normal_(generator=c.gen)
    c.v[8, pages - 24:].normal_(generator=c.gen)
    assert int(c.ctx.kv_pages(c.kv, seqs).max()) > pages - 10
    check(c, seqs, [60, 1, 1, 1, 1, 1], 8, layer=8)
    new = torch.randn(60, 2, 128, device="cuda").half()
    b = c.batch(seqs[:1], [60], 8)
    c.ctx.kv_write(b, 8, new.data_ptr(), new.data_ptr(), "f16", stream=c.stream)
    assert torch.equal(c.rows(seqs[0], 8, c.v)[-60:], new) and torch.equal(c.rows(seqs[0], 8, c.k)[-60:], new)
    copy = c.ctx.kv_copy(c.kv, seqs[:1], [100], stream=c.stream)
    assert torch.equal(c.rows(copy[0], 8, c.k), c.rows(seqs[0], 8, c.k)[:100])


# ---------------------------------------------------------------- page moves

@pytest.mark.parametrize("type,dim,pt,heads", [("f16", 128, 16, 8), ("bf16", 64, 128, 3), ("f16", 64, 32, 1)])
def test_page_moves_against_plain_copies(type, dim, pt, heads):
    """Random forks, copies, frees and compactions: every sequence keeps its rows, and no other row changes."""
    rng = random.Random(f"{type}{pt}")
    c = Cache(type, 3, heads, dim, pt, pages=500)
    live = {}  # sequence -> (keys, values) it has to hold, positions x heads x dims per layer

    def read(s):
        return [torch.stack([c.rows(s, l, x) for l in range(3)]) for x in (c.k, c.v)]

    def held():
        h = torch.zeros(c.k.shape[1], pt, dtype=torch.bool, device="cuda")
        for s in live:
            pages, n = c.ctx.kv_pages(c.kv, [s])[0], int(c.ctx.kv_lengths(c.kv, [s])[0])
            for p in range(n):
                h[int(pages[p // pt]), p % pt] = True
        return h

    for step in range(24):
        op = "open" if not live else rng.choice(("open", "fork", "fork", "copy", "free", "compact"))
        try:
            if op == "open":
                (s,) = c.ctx.kv_open(c.kv, 1)
                c.ctx.kv_extend(c.kv, [s], [rng.choice((0, 1, pt - 1, pt, pt + 1, 300))])
                live[s] = read(s)
                continue
            before = (c.k.clone(), c.v.clone())
            if op in ("fork", "copy"):
                ids = [rng.choice(list(live)) for _ in range(rng.randint(1, 40))]
                lens = [rng.randint(0, live[i][0].shape[1]) for i in ids]
                kids = (c.ctx.kv_fork if op == "fork" else c.ctx.kv_copy)(c.kv, ids, lens, stream=c.stream)
                old = held()
                for i, n, k in zip(ids, lens, kids):
                    live[k] = [x[:, :n] for x in live[i]]
                new = held() & ~old
                assert torch.equal(torch.where(new[None, :, None, :, None], before[0], c.k), before[0])
                assert torch.equal(torch.where(new[None, :, None, :, None], before[1], c.v), before[1])
            elif op == "free":
                gone = rng.sample(list(live), rng.randint(1, len(live)))
                c.ctx.kv_free(c.kv, gone)
                for s in gone:
                    del live[s]
            else:
                c.ctx.kv_compact(c.kv, stream=c.stream)
                info = c.ctx.kv_info(c.kv)
                assert info["pages_spanned"] == info["pages_used"]
        except binding.ShieldError as e:
            assert e.code == binding.ERR_NOMEM
        for s, want in live.items():
            for a, b in zip(read(s), want):
                assert torch.equal(a, b)


def test_many_moves_in_one_call():
    """More moves than one launch carries."""
    c = Cache("f16", 1, 1, 64, 16, pages=2000)
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [16 * 10 + 5])
    want = c.rows(root, 0, c.k).clone()
    kids = c.ctx.kv_fork(c.kv, [root] * 901, stream=c.stream)
    for s in (kids[0], kids[299], kids[300], kids[600], kids[900]):
        assert torch.equal(c.rows(s, 0, c.k), want)
    c.ctx.kv_free(c.kv, kids[:890])
    assert c.ctx.kv_compact(c.kv, stream=c.stream) == 11
    for s in kids[890:]:
        assert torch.equal(c.rows(s, 0, c.k), want)


# -------------------------------------------------------------------- writes

@pytest.mark.parametrize("type,dim,pt,heads", [("f16", 128, 64, 8), ("bf16", 64, 16, 3), ("bf16", 128, 128, 1)])
@pytest.mark.parametrize("src", ["f32", "same"])
def test_written_rows(type, dim, pt, heads, src):
    rng = random.Random(pt)
    c = Cache(type, 2, heads, dim, pt, pages=300)
    seqs = c.ctx.kv_open(c.kv, 7)
    c.ctx.kv_extend(c.kv, seqs, [0, 1, pt - 1, pt, 100, 37, 5])
    counts = [1, 2, 3, pt + 5, 0, 200, 1]
    c.ctx.kv_extend(c.kv, seqs, counts)
    T = sum(counts)
    dtype = torch.float32 if src == "f32" else c.dtype
    rows = torch.randn(2, T + 2, heads * dim + 24, device="cuda").to(dtype)
    rows[0, 0, 0], rows[1, 1, 3] = math.inf, math.nan
    rows[0, 2, 1] = 70000.0 if type == "bf16" or src == "f32" else 65504.0
    before = c.k.clone(), c.v.clone()
    b = c.batch(seqs, counts, heads)
    c.ctx.kv_write(b, 1, rows[0, :, 8:].data_ptr(), rows[1, :, 8:].data_ptr(), src if src == "f32" else type,
                   k_stride=rows.stride(1), v_stride=rows.stride(1), stream=c.stream)
    want = before[0].clone(), before[1].clone()
    t = 0
    for s, n, m in zip(seqs, c.ctx.kv_lengths(c.kv, seqs), counts):
        pages = c.ctx.kv_pages(c.kv, [s])[0]
        for p in range(n - m, n):
            for x, y in zip(want, rows):
                x[1, int(pages[p // pt]), :, p % pt] = y[t, 8:8 + heads * dim].view(heads, dim).to(c.dtype)
            t += 1
    for got, x in zip((c.k, c.v), want):
        assert torch.equal(got.view(torch.int16), x.view(torch.int16))


# ------------------------------------------------------- a run, and its edges

def test_a_run_of_steps():
    """Prompt, forks, decode steps, an early end, compaction, more steps: always the attention of the tokens written so far."""
    c = Cache("bf16", 2, 2, 128, 32, pages=200)
    heads, rng = 8, random.Random(3)
    said = {}  # sequence -> tokens, which stand for their rows

    def row(token, layer, which):
        g = torch.Generator("cuda").manual_seed(token * 4 + layer * 2 + which)
        return torch.randn(2, 128, device="cuda", generator=g)

    batch = c.ctx.kv_batch_create(c.kv, heads, 400, 32, 600)

    def step(seqs, tokens):
        counts = [len(t) for t in tokens]
        c.ctx.kv_extend(c.kv, seqs, counts)
        c.ctx.kv_batch_set(batch, seqs, counts, stream=c.stream)
        flat = [t for x in tokens for t in x]
        for layer in range(2):
            k, v = (torch.stack([row(t, layer, w) for t in flat]) for w in (0, 1))
            c.ctx.kv_write(batch, layer, k.data_ptr(), v.data_ptr(), "f32", stream=c.stream)
        for s, x in zip(seqs, tokens):
            said[s] = said[s] + list(x)
        check(c, seqs, counts, heads, layer=rng.randint(0, 1), batch=batch)
        for s in seqs:
            want = torch.stack([row(t, 1, 1) for t in said[s]]).to(c.dtype)
            assert torch.equal(c.rows(s, 1, c.v), want)

    (root,) = c.ctx.kv_open(c.kv, 1)
    said[root] = []
    step([root], [range(0, 345)])
    kids = c.ctx.kv_fork(c.kv, [root] * 9, stream=c.stream)
    for s in kids:
        said[s] = list(said[root])
    step(kids, [range(1000 + 50 * i, 1000 + 50 * i + 3 * i + 1) for i in range(9)])
    for n in range(3):
        step(kids, [[2000 + 10 * n + i] for i in range(9)])
    c.ctx.kv_free(c.kv, np.concatenate([[root], kids[::2]]))
    q = torch.zeros(9, heads, 128, dtype=c.dtype, device="cuda")
    with pytest.raises(binding.ShieldError) as e:  # its sequences are gone
        c.ctx.kv_attend(batch, 0, q.data_ptr(), q.data_ptr(), 1.0, stream=c.stream)
    assert e.value.code == binding.ERR_STATE
    kids = kids[1::2]
    c.ctx.kv_batch_set(batch, kids, [1] * 4, stream=c.stream)
    assert c.ctx.kv_compact(c.kv, stream=c.stream) > 0
    with pytest.raises(binding.ShieldError) as e:
        c.ctx.kv_write(batch, 0, q.data_ptr(), q.data_ptr(), "bf16", stream=c.stream)
    assert e.value.code == binding.ERR_STATE
    for n in range(2):
        step(kids, [[3000 + 10 * n + i] for i in range(4)])
    more = c.ctx.kv_fork(c.kv, kids[:1], [100], stream=c.stream)
    said[more[0]] = said[kids[0]][:100]
    step(np.concatenate([kids, more]), [[4000], [4001], [4002], range(4100, 4130), range(4200, 4333)])


def test_captured_steps_follow_the_plan_set_last():
    c = Cache("f16", 1, 2, 128, 16, pages=3000)
    heads = 8
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [3000])
    seqs = c.ctx.kv_fork(c.kv, [root] * 12, stream=c.stream)
    c.ctx.kv_extend(c.kv, seqs, range(5, 17))
    lone = c.ctx.kv_open(c.kv, 3)
    c.ctx.kv_extend(c.kv, lone, [1, 400, 7000])
    every = np.concatenate([seqs, lone])
    caps = dict(max_tokens=400, max_seqs=20, max_positions=8000)
    b = c.batch(every[:1], [1], heads, **caps)
    q = torch.randn(400, heads, 128, device="cuda").half()
    out = torch.zeros_like(q)
    rows = torch.randn(2, 400, 2, 128, device="cuda")
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        c.ctx.kv_write(b, 0, rows[0].data_ptr(), rows[1].data_ptr(), "f32", stream=side.cuda_stream)
        c.ctx.kv_attend(b, 0, q.data_ptr(), out.data_ptr(), 0.09, stream=side.cuda_stream)
        with pytest.raises(binding.ShieldError) as e:
            c.ctx.kv_batch_set(b, every[:2], [1, 1], stream=side.cuda_stream)
        assert e.value.code == binding.ERR_STATE
        with pytest.raises(binding.ShieldError) as e:
            c.ctx.kv_fork(c.kv, every[:2], stream=side.cuda_stream)
        assert e.value.code == binding.ERR_STATE
    for ids, counts in [(every[:1], [1]), (every, [1] * 15), (seqs, [3] * 12), (lone, [1, 300, 60]), (every, [0] * 14 + [1]), (lone, [1, 1, 1])]:
        c.ctx.kv_batch_set(b, ids, counts, stream=c.stream)
        T = sum(counts)
        out.fill_(5)
        g.replay()
        k0 = c.k.clone(), c.v.clone()
        want, tol = expect(c, ids, counts, q, 0, 0.09)
        assert ((out[:T].double() - want).abs() <= tol).all() and (out[T:] == 5).all()
        now = torch.empty_like(out)
        c.ctx.kv_attend(b, 0, q.data_ptr(), now.data_ptr(), 0.09, stream=c.stream)
        assert torch.equal(now[:T], out[:T])
        t = 0
        for s, m in zip(ids, counts):
            if m:
                assert torch.equal(c.rows(s, 0, c.v)[-m:], rows[1, t:t + m].half())
            t += m
        assert torch.equal(k0[0], c.k) and torch.equal(k0[1], c.v)


def test_batches_on_streams_of_their_own():
    c = Cache("f16", 2, 8, 128, 64, pages=1200)
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [6000])
    seqs = c.ctx.kv_fork(c.kv, [root] * 32, stream=c.stream)
    c.ctx.kv_extend(c.kv, seqs, range(100, 132))
    q = torch.randn(2, 32, 32, 128, device="cuda").half()
    want = torch.empty_like(q)
    b = [c.batch(seqs[16 * i:16 * i + 16 + 16 * (1 - i)], [1] * (16 + 16 * (1 - i)), 32) for i in range(2)]
    for i in range(2):
        c.ctx.kv_attend(b[i], i, q[i].data_ptr(), want[i].data_ptr(), 0.1, stream=c.stream)
    torch.cuda.synchronize()
    out = torch.empty_like(q)
    side = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        out.fill_(0)
        torch.cuda.synchronize()
        for i in range(2):
            c.ctx.kv_attend(b[i], i, q[i].data_ptr(), out[i].data_ptr(), 0.1, stream=side[i].cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1, :16], want[1, :16])
    # the context's own stream, waited for through torch
    own = torch.cuda.ExternalStream(c.ctx.stream())
    out.fill_(0)
    own.wait_stream(torch.cuda.current_stream())
    c.ctx.kv_attend(b[0], 0, q[0].data_ptr(), out[0].data_ptr(), 0.1)
    torch.cuda.current_stream().wait_stream(own)
    assert torch.equal(out[0], want[0])


def test_library_memory_and_release():
    ctx = binding.ShieldContext(1)
    kv = ctx.kv_create("bf16", 2, 2, 64, 16, 100)
    info = ctx.kv_info(kv)
    assert info["k"] and info["v"] and info["n_pages"] == 100 and info["pages_used"] == 0
    s = ctx.kv_open(kv, 2)
    ctx.kv_extend(kv, s, [17, 40])
    b = ctx.kv_batch_create(kv, 4, 57, 2, 40)
    ctx.kv_batch_set(b, s, [17, 40])
    k = torch.randn(57, 2, 64, device="cuda").bfloat16()
    q, out = torch.randn(57, 4, 64, device="cuda").bfloat16(), torch.empty(57, 4, 64, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    ctx.kv_write(b, 1, k.data_ptr(), k.data_ptr(), "bf16")
    ctx.kv_attend(b, 1, q.data_ptr(), out.data_ptr(), 0.125)
    torch.cuda.synchronize()
    for lo, hi in ((0, 17), (17, 57)):
        x = k[lo:hi].double().repeat_interleave(2, 1).transpose(0, 1)
        e = (q[lo:hi].double().transpose(0, 1) @ x.transpose(1, 2)) * 0.125
        e = e.masked_fill(torch.triu(torch.ones(hi - lo, hi - lo, device="cuda", dtype=torch.bool), 1), -math.inf)
        w = torch.softmax(e, -1) @ x
        assert ((out[lo:hi].double().transpose(0, 1) - w).abs() <= 2.0 ** -7 * (torch.softmax(e, -1) @ x.abs()) + 1e-5).all()
    ctx.kv_batch_release(b)
    with pytest.raises(binding.ShieldError):
        ctx.kv_attend(b, 1, q.data_ptr(), out.data_ptr(), 0.125)
    b = ctx.kv_batch_create(kv, 4, 57, 2, 40)
    ctx.kv_release(kv)
    for call in (lambda: ctx.kv_open(kv, 1), lambda: ctx.kv_batch_set(b, s, [1, 1])):
        with pytest.raises(binding.ShieldError) as e:
            call()
        assert e.value.code == binding.ERR_ARG


def test_refusals():
    c = Cache("f16", 2, 2, 64, 16, pages=32)
    ctx, kv = c.ctx, c.kv
    a, b = ctx.kv_open(kv, 2).tolist()
    ctx.kv_extend(kv, [a, b], [20, 30])
    other = ctx.kv_create("f16", 2, 2, 64, 16, 8)
    (far,) = ctx.kv_open(other, 1)
    batch = ctx.kv_batch_create(kv, 4, 10, 2, 25)
    q = torch.zeros(64, 4, 64, dtype=torch.float16, device="cuda")
    p = q.data_ptr()
    arg, rng_, uns, st, shape, nomem = (binding.ERR_ARG, binding.ERR_RANGE, binding.ERR_UNSUPPORTED, binding.ERR_STATE,
                                        binding.ERR_SHAPE, binding.ERR_NOMEM)

    def refused(code, call):
        with pytest.raises(binding.ShieldError) as e:
            call()
        assert e.value.code == code, str(e.value)

    refused(st, lambda: ctx.kv_attend(batch, 0, p, p, 1.0))  # no plan yet
    refused(uns, lambda: ctx.kv_create("f32", 1, 1, 64, 16, 4))
    refused(uns, lambda: ctx.kv_create("f16", 1, 1, 96, 16, 4))
    refused(uns, lambda: ctx.kv_create("f16", 1, 1, 64, 48, 4))
    refused(arg, lambda: ctx.kv_create("f16", 0, 1, 64, 16, 4))
    refused(arg, lambda: ctx.kv_create("f16", 1, 1, 64, 16, 0))
    refused(arg, lambda: ctx.kv_create("f16", 1, 1, 64, 16, 4, k=c.k.data_ptr()))
    refused(arg, lambda: ctx.kv_create("f16", 1, 1, 64, 16, 4, k=c.k.data_ptr() + 16, v=c.v.data_ptr()))
    refused(rng_, lambda: ctx.kv_create("f16", 1, 1, 64, 128, 1 << 24, k=c.k.data_ptr(), v=c.v.data_ptr()))
    refused(rng_, lambda: ctx.kv_create("f16", 1, 1, 64, 16, 4, device=1))
    refused(arg, lambda: ctx.kv_open(12345, 1))
    refused(arg, lambda: ctx.kv_extend(kv, [far], [1]))
    refused(arg, lambda: ctx.kv_fork(kv, [a, far]))
    refused(nomem, lambda: ctx.kv_extend(kv, [a], [16 * 40]))
    refused(nomem, lambda: ctx.kv_copy(kv, [a] * 20, stream=c.stream))
    refused(shape, lambda: ctx.kv_batch_create(kv, 3, 1, 1, 1))
    refused(arg, lambda: ctx.kv_batch_create(kv, 4, 0, 1, 1))
    refused(arg, lambda: ctx.kv_batch_set(batch, [a, a], [1, 1]))
    refused(arg, lambda: ctx.kv_batch_set(batch, [far], [1]))
    refused(rng_, lambda: ctx.kv_batch_set(batch, [a], [21]))
    refused(rng_, lambda: ctx.kv_batch_set(batch, [a], [-1]))
    refused(rng_, lambda: ctx.kv_batch_set(batch, [a], [11]))
    refused(rng_, lambda: ctx.kv_batch_set(batch, [b], [1]))  # longer than max_positions
    ctx.kv_batch_set(batch, [a], [10], stream=c.stream)
    refused(rng_, lambda: ctx.kv_attend(batch, 2, p, p, 1.0))
    refused(rng_, lambda: ctx.kv_write(batch, -1, p, p, "f16"))
    refused(arg, lambda: ctx.kv_attend(batch, 0, None, p, 1.0))
    refused(arg, lambda: ctx.kv_attend(batch, 0, p, p + 2, 1.0))
    refused(arg, lambda: ctx.kv_attend(batch, 0, p, p, 1.0, q_stride=255))
    refused(arg, lambda: ctx.kv_attend(batch, 0, p, p, 1.0, q_stride=260))
    refused(arg, lambda: ctx.kv_attend(batch, 0, p, p, math.inf))
    refused(arg, lambda: ctx.kv_write(batch, 0, p, p, "f16", k_stride=64))
    refused(uns, lambda: ctx.kv_write(batch, 0, p, p, "bf16"))
    ctx.kv_batch_set(batch, [], [], stream=c.stream)  # an empty step is one
    ctx.kv_attend(batch, 0, p, p, 1.0, stream=c.stream)
    ctx.kv_batch_set(batch, [a], [0], stream=c.stream)
    ctx.kv_write(batch, 0, p, p, "f16", stream=c.stream)
    torch.cuda.synchronize()
    assert not q.any()


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[1], SHAPES[5]], ids=lambda s: "-".join(map(str, s)))
def test_more_work_than_the_gpu_holds_at_once(shape):
    """Several units per CTA, short and long, one tile and two, partial and whole: each the same every time, and right."""
    type, dim, pt, kv_heads, heads = shape
    rng = random.Random(7)
    c = Cache(type, 2, kv_heads, dim, pt, pages=-(-120000 // pt))
    seqs = np.concatenate([tree(c, rng, roots=3, kids=12, lo=1, hi=1500, own_lo=1, own_hi=300),
                           tree(c, rng, roots=60, kids=1, lo=1, hi=700, own_lo=1, own_hi=90)])
    lens = c.ctx.kv_lengths(c.kv, seqs)
    counts = [min(int(n), rng.choice((1, 3, 6, 20, 34, 70, 200))) for n in lens]
    b = c.batch(seqs, counts, heads)
    first = check(c, seqs, counts, heads, batch=b)
    T = sum(counts)
    q = torch.randn(T, heads, dim, device="cuda").to(c.dtype)
    outs = torch.empty(20, T, heads, dim, dtype=c.dtype, device="cuda")
    for o in outs:
        c.k.add_(0)  # something else in between
        c.ctx.kv_attend(b, 1, q.data_ptr(), o.data_ptr(), dim ** -0.5, stream=c.stream)
    assert torch.equal(outs, outs[:1].expand_as(outs)) and first.shape == outs[0].shape


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 2])
def test_short_pieces_that_a_warp_takes_alone(type, new):
    """More short sequences than the GPU holds CTAs, behind a prefix and without, with what their rows may not see."""
    c = Cache(type, 1, 8, 128, 16, pages=900)
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [700])
    kids = c.ctx.kv_fork(c.kv, [root] * 60, stream=c.stream)
    c.ctx.kv_extend(c.kv, kids, [new + i % 45 for i in range(60)])
    lone = c.ctx.kv_open(c.kv, 30)
    c.ctx.kv_extend(c.kv, lone, [new + 2 * i for i in range(30)])
    seqs = np.concatenate([kids, lone])
    check(c, seqs, [new] * 90, 32, layer=0)
    if new > 1:  # an infinite value at a sequence's end: its last row has it, the rows before do not
        pages, lens = c.ctx.kv_pages(c.kv, seqs), c.ctx.kv_lengths(c.kv, seqs)
        for i in range(0, 90, 7):
            p = int(lens[i]) - 1
            c.v[0, int(pages[i][p // 16]), 3, p % 16, 5] = math.inf
        b = c.batch(seqs, [new] * 90, 32)
        q = torch.randn(90 * new, 32, 128, device="cuda").to(c.dtype)
        out = torch.empty_like(q)
        c.ctx.kv_attend(b, 0, q.data_ptr(), out.data_ptr(), 128 ** -0.5, stream=c.stream)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit.view(90, new, 32, 128)[::7, -1, 12:16, 5] = True
        assert torch.equal(~torch.isfinite(out), hit) and (out[hit] == math.inf).all()


@pytest.mark.parametrize("type,dim", [("f16", 128), ("bf16", 64)])
def test_a_run_of_keys_in_many_pieces(type, dim):
    """60,000 keys of one kv head: more pieces than a joining warp has lanes, for few rows and for many."""
    c = Cache(type, 1, 1, dim, 64, pages=1100)
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [60000])
    check(c, [root], [1], 8, layer=0)
    kids = c.ctx.kv_fork(c.kv, [root] * 25, stream=c.stream)
    c.ctx.kv_extend(c.kv, kids, [1 + i for i in range(25)])
    check(c, kids, [1] * 25, 8, layer=0)


@pytest.mark.parametrize("shape", [SHAPES[2], SHAPES[3], SHAPES[6]], ids=lambda s: "-".join(map(str, s)))
def test_more_work_than_the_gpu_holds_at_once_heads_of_64(shape):
    test_more_work_than_the_gpu_holds_at_once(shape)


@pytest.mark.parametrize("shape", [("f16", 64, 64, 8, 8), ("bf16", 64, 16, 4, 16), ("bf16", 128, 64, 8, 8), ("f16", 128, 32, 4, 16)],
                         ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("grows", [(1,), (0,), (0, 1)], ids=["second", "first", "both"])
def test_tiles_with_unequal_work(shape, grows):
    """Units of two row tiles, of one and of one key block, where the scores of one tile's rows grow from key to key,
    so that its maxima grow in every half block, and the other's fall."""
    type, dim, pt, kv_heads, heads = shape
    G, rng = heads // kv_heads, random.Random(f"{shape}{grows}")
    c = Cache(type, 1, kv_heads, dim, pt, pages=-(-40000 // pt))
    rows = 512 // G
    before = [0, 0, 700, 100, 129, 1000, 255, 640, 900, 1, 383, 500] + [300] * (148 // kv_heads // 2)
    counts = [rows - rng.choice((0, 0, 1, 17)) for _ in before]
    counts += [rng.randint(20 // G + 1, 128 // G) for _ in range(60)]  # one key block, one tile
    before += [0] * 60
    counts += [100 // G + 1] * 8
    before += [rng.randint(100, 400) for _ in range(8)]
    seqs = c.ctx.kv_open(c.kv, len(counts))
    c.ctx.kv_extend(c.kv, seqs, [n + m for n, m in zip(before, counts)])
    # scale q.k is 0.1 a key upwards: 9 in log2 per half block, above the growth that the kernel lets pass
    sign = torch.randint(0, 2, (dim,), device="cuda", generator=c.gen).mul_(2).sub_(1)
    step = 0.1 / dim ** 0.5
    for s, n, m in zip(seqs, before, counts):
        pages = torch.from_numpy(c.ctx.kv_pages(c.kv, [s])[0]).long().cuda()
        at = torch.arange(pages.numel() * pt, device="cuda").view(-1, 1, pt, 1)
        c.k[0, pages] = (c.k[0, pages].float() * 0.05 + at * step * sign).to(c.dtype)
    q = torch.empty(sum(counts), heads, dim, device="cuda").normal_(0, 0.05, generator=c.gen)
    t = 0
    for m in counts:
        tile = (torch.arange(m, device="cuda") * G // 128) % 2
        up = sum((tile == g) for g in grows).clamp(max=1)
        q[t:t + m] += (2 * up - 1)[:, None, None] * sign
        t += m
    q = q.to(c.dtype)
    scale = dim ** -0.5
    b = c.batch(seqs, counts, heads)
    outs = torch.empty(6, *q.shape, dtype=c.dtype, device="cuda")
    for o in outs:
        c.ctx.kv_attend(b, 0, q.data_ptr(), o.data_ptr(), scale, stream=c.stream)
    torch.cuda.synchronize()
    c.ctx.kv_batch_set(b, seqs, counts, stream=c.stream)  # would say so if a wait had given up
    want, tol = expect(c, seqs, counts, q, 0, scale)
    worst = ((outs[0].double() - want).abs() / tol).max().item()
    assert worst <= 1, f"{worst} times the tolerance"
    assert torch.equal(outs, outs[:1].expand_as(outs))


class StaleError:
    """A failed call of the caller's own, whose error the runtime still holds for this thread."""

    def __enter__(self):
        torch.cuda.synchronize()
        self.rt = ctypes.CDLL("libcudart.so.12")  # torch's and the library's
        assert self.rt.cudaSetDevice(1000) != 0 and self.rt.cudaPeekAtLastError() != 0

    def __exit__(self, *_):
        self.rt.cudaGetLastError()


def scattered(c):
    """501 forks of a root, each with a page of its own, behind 400 free pages, and what they hold."""
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [16 * 10 + 5])
    want = c.rows(root, 0, c.k).clone()
    kids = c.ctx.kv_fork(c.kv, [root] * 901, stream=c.stream)
    gone = c.ctx.kv_pages(c.kv, kids[:400])[:, -1]
    c.ctx.kv_free(c.kv, kids[:400])
    c.k[:, torch.from_numpy(gone).long().cuda()] = 9.0
    return kids[400:], want


def test_a_compaction_that_fails_changes_nothing():
    c = Cache("f16", 1, 1, 64, 16, pages=2000)
    kids, want = scattered(c)
    with StaleError():
        try:
            c.ctx.kv_compact(c.kv, stream=c.stream)
        except binding.ShieldError as e:
            assert e.code == binding.ERR_CUDA
    for s in kids[::20]:
        assert torch.equal(c.rows(s, 0, c.k), want)
    c.ctx.kv_compact(c.kv, stream=c.stream)
    info = c.ctx.kv_info(c.kv)
    assert info["pages_spanned"] == info["pages_used"] == 10 + 1 + 501
    for s in kids:
        assert torch.equal(c.rows(s, 0, c.k), want)


def test_errors_of_other_calls_are_not_taken_for_a_launchs_own():
    """Forks, compactions, writes and attention after a failed allocation of the library's and a failed call of the caller's."""
    c = Cache("f16", 1, 1, 64, 16, pages=2000)
    kids, want = scattered(c)
    rt = ctypes.CDLL("libcudart.so.12")
    for _ in range(2):
        with pytest.raises(binding.ShieldError) as e:  # 4 TB
            c.ctx.kv_create("f16", 1, 128, 128, 128, 1 << 20)
        assert e.value.code == binding.ERR_NOMEM
        assert rt.cudaPeekAtLastError() == 0
        kids = np.concatenate([kids, c.ctx.kv_fork(c.kv, kids[:1], stream=c.stream)])
    q, out = (torch.zeros(40, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    new = torch.randn(40, 1, 64, device="cuda")
    with StaleError():
        kids = np.concatenate([kids, c.ctx.kv_fork(c.kv, np.repeat(kids[:1], 350), stream=c.stream)])
        assert c.ctx.kv_compact(c.kv, stream=c.stream) == 400 - 352
        (s,) = c.ctx.kv_copy(c.kv, kids[-1:], stream=c.stream)
        c.ctx.kv_extend(c.kv, [s], [40])
        lens = c.ctx.kv_lengths(c.kv, [s])
        b = c.ctx.kv_batch_create(c.kv, 4, 40, 1, int(lens[0]))
        for n in (40, 1):  # the kernel of many rows, the one of few
            c.ctx.kv_batch_set(b, [s], [n], stream=c.stream)
            c.ctx.kv_write(b, 0, new[-n:].data_ptr(), new[-n:].data_ptr(), "f32", stream=c.stream)
            c.ctx.kv_attend(b, 0, q.data_ptr(), out.data_ptr(), 0.125, stream=c.stream)
    for s in kids:
        assert torch.equal(c.rows(s, 0, c.k), want)


def test_a_wait_that_gave_up_is_told():
    """The error word, set from the host as a kernel's wait sets it: told once, by whichever call comes first."""
    c = Cache("bf16", 1, 2, 64, 16, pages=40)
    s = c.ctx.kv_open(c.kv, 2)
    c.ctx.kv_extend(c.kv, s, [30, 5])
    b, other = (c.batch(s, [3, 1], 4) for _ in range(2))
    q, out = (torch.zeros(4, 4, 64, dtype=c.dtype, device="cuda") for _ in range(2))
    k = torch.randn(4, 2, 64, device="cuda")
    calls = [lambda b: c.ctx.kv_batch_check(b), lambda b: c.ctx.kv_batch_set(b, s, [3, 1], stream=c.stream),
             lambda b: c.ctx.kv_write(b, 0, k.data_ptr(), k.data_ptr(), "f32", stream=c.stream),
             lambda b: c.ctx.kv_attend(b, 0, q.data_ptr(), out.data_ptr(), 0.1, stream=c.stream)]
    for call in calls:
        call(b)
    for first in calls:
        c.ctx.debug_kv_error(c.kv, b, 3)
        c.ctx.kv_batch_check(other)  # another batch's work
        with pytest.raises(binding.ShieldError) as e:
            first(b)
        assert e.value.code == binding.ERR_TIMEOUT and "gave up" in str(e.value)
        for call in calls:
            call(b)
    far = c.ctx.kv_create("bf16", 1, 2, 64, 16, 4)
    for bad in (lambda: c.ctx.kv_batch_check(b + 100), lambda: c.ctx.debug_kv_error(far, b, 1), lambda: c.ctx.debug_kv_error(c.kv, 0, 1)):
        with pytest.raises(binding.ShieldError) as e:
            bad()
        assert e.value.code == binding.ERR_ARG


def test_rows_of_two_sequences_are_not_written_to_one_place():
    c = Cache("f16", 1, 2, 64, 16, pages=40)
    (root,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [root], [32])
    kids = c.ctx.kv_fork(c.kv, [root] * 2, stream=c.stream)
    c.ctx.kv_extend(c.kv, kids, [3, 5])
    before = c.k.clone()
    k = torch.randn(48, 2, 64, device="cuda")
    b = c.batch(kids, [3, 5], 4, max_tokens=48)

    def write():
        c.ctx.kv_write(b, 0, k.data_ptr(), k.data_ptr(), "f32", stream=c.stream)

    for counts in ([4, 6], [35, 6], [3, 37]):  # back into the shared pages: both, both, one of them
        c.ctx.kv_batch_set(b, kids, counts, stream=c.stream)
        if counts[0] == 3:
            write()
            assert torch.equal(c.rows(root, 0, c.k), k[3:35].half())
            continue
        with pytest.raises(binding.ShieldError) as e:
            write()
        assert e.value.code == binding.ERR_STATE
        assert torch.equal(c.k, before)
    c.ctx.kv_batch_set(b, kids, [3, 5], stream=c.stream)
    write()
    check(c, kids, [4, 6], 4, layer=0)  # queries of shared positions are no conflict


def test_outputs_over_other_queries_are_refused():
    c = Cache("bf16", 1, 2, 64, 16, pages=40)
    (s,) = c.ctx.kv_open(c.kv, 1)
    c.ctx.kv_extend(c.kv, [s], [60])
    b = c.batch([s], [40], 4)
    w = 4 * 64
    x = torch.randn(200, 2 * w, device="cuda").to(c.dtype)
    q = x[:40, :w].clone()
    want, tol = expect(c, [s], [40], q.view(40, 4, 64), 0, 0.125)

    def attend(offset, q_stride, out_stride):
        x[:40 * q_stride // (2 * w) + 1].view(-1)[:40 * q_stride].view(40, q_stride)[:, :w] = q
        base = x.data_ptr()
        c.ctx.kv_attend(b, 0, base, base + 2 * offset, 0.125, q_stride=q_stride, out_stride=out_stride, stream=c.stream)
        out = torch.as_strided(x, (40, w), (out_stride, 1), offset)
        assert ((out.double().view(40, 4, 64) - want).abs() <= tol).all()

    attend(0, w, w)
    attend(0, 2 * w, 2 * w)
    attend(w, 2 * w, 2 * w)  # rows that take turns
    attend(40 * w, w, 2 * w)
    attend(40 * 2 * w, 2 * w, w)
    for offset, q_stride, out_stride in [(0, w, 2 * w), (0, 2 * w, w), (8, w, w), (w // 2, w, w), (w - 8, 2 * w, 2 * w), (w + 8, 2 * w, 2 * w),
                                         (39 * w, w, 2 * w), (w, 2 * w, w)]:
        with pytest.raises(binding.ShieldError) as e:
            attend(offset, q_stride, out_stride)
        assert e.value.code == binding.ERR_ARG
    c.ctx.kv_batch_set(b, [s], [1], stream=c.stream)
    one = x[0].clone()
    c.ctx.kv_attend(b, 0, x.data_ptr(), x.data_ptr(), 0.125, q_stride=w, out_stride=2 * w, stream=c.stream)
    want, tol = expect(c, [s], [1], one[:w].view(1, 4, 64), 0, 0.125)
    assert ((x[0, :w].double().view(1, 4, 64) - want).abs() <= tol).all()
