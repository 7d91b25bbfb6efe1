"""The model on a paged cache (shield_kv_forward): step by step, forked and
compacted, bit-identical to the oracle's operations around shield_kv_attend,
which tests/test_gpu_kv.py holds to its definition."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from llm_shield_b200 import binding, synth
from helpers import oracle_config, oracle_model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


class Twin:
    """The model's layers from the oracle's operations; keys and values rounded
    into the cache, attention by shield_kv_attend on a plan of its own."""

    def __init__(self, ctx, spec, tensors, type):
        self.ctx, self.spec, self.t, self.type = ctx, spec, tensors, type
        cfg = oracle_config(spec)
        self.freqs, self.mscale = cfg["rope_freqs"], cfg["rope_mscale"]
        pt, pages = 16, 300
        shape = (spec.n_layers, pages, spec.n_kv_heads, pt, spec.head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=DTYPES[type], device="cuda") for _ in range(2))
        self.kv = ctx.kv_create(type, spec.n_layers, spec.n_kv_heads, spec.head_dim, pt, pages,
                                k=self.k.data_ptr(), v=self.v.data_ptr())

    def mul(self, name, x):
        t = self.t[name]
        return oracle.qmatmul(t["type"], t["data"], t["rows"], t["cols"], x, x.shape[0])

    def norm(self, name, x):
        w = np.frombuffer(self.t[name]["data"].tobytes(), np.float32)
        return np.stack([oracle.rmsnorm(r, w, self.spec.rms_eps) for r in x])

    def rope(self, x, heads, positions):
        return np.stack([oracle.rope_apply(r, heads, self.spec.head_dim, int(p), self.freqs, self.mscale) for r, p in zip(x, positions)])

    def step(self, seqs, chunks):
        """What kv_forward(seqs, chunks) has to give and to leave in the pages, which is compared."""
        s = self.spec
        lens = self.ctx.kv_lengths(self.kv, seqs)
        counts = [len(c) for c in chunks]
        positions = np.concatenate([np.arange(n - c, n) for n, c in zip(lens, counts)])
        ids = np.concatenate(chunks)
        emb = self.t["token_embd.weight"]
        row = len(emb["data"]) // emb["rows"]
        h = np.stack([oracle.dequantize(emb["type"], emb["data"][i * row:(i + 1) * row], emb["cols"]) for i in ids])
        b = self.ctx.kv_batch_create(self.kv, s.n_heads, len(ids), len(seqs), int(lens.max()))
        self.ctx.kv_batch_set(b, seqs, counts)
        pages = self.ctx.kv_pages(self.kv, seqs)
        at = [(int(pages[i, p // 16]), p % 16) for i, (n, c) in enumerate(zip(lens, counts)) for p in range(n - c, n)]
        page, line = (torch.tensor(x, device="cuda") for x in zip(*at))
        for l in range(s.n_layers):
            p = f"blk.{l}."
            x = self.norm(p + "attn_norm.weight", h)
            q, k = self.rope(self.mul(p + "attn_q.weight", x), s.n_heads, positions), self.rope(self.mul(p + "attn_k.weight", x), s.n_kv_heads, positions)
            v = self.mul(p + "attn_v.weight", x)
            for got, want in ((self.k, k), (self.v, v)):
                want = torch.from_numpy(want).cuda().view(len(ids), s.n_kv_heads, s.head_dim).to(got.dtype)
                assert torch.equal(got[l][page, :, line], want), (l, "keys or values")
            q16 = torch.from_numpy(q).cuda().to(self.k.dtype).contiguous()
            out = torch.empty_like(q16)
            torch.cuda.synchronize()
            self.ctx.kv_attend(b, l, q16.data_ptr(), out.data_ptr(), s.head_dim ** -0.5)
            torch.cuda.synchronize()
            h = h + self.mul(p + "attn_output.weight", out.float().cpu().numpy())
            x = self.norm(p + "ffn_norm.weight", h)
            g, u = self.mul(p + "ffn_gate.weight", x), self.mul(p + "ffn_up.weight", x)
            h = h + self.mul(p + "ffn_down.weight", np.stack([oracle.swiglu(a, c) for a, c in zip(g, u)]))
        self.ctx.kv_batch_release(b)
        last = np.cumsum(counts) - 1
        return self.mul("token_embd.weight", self.norm("output_norm.weight", h[last]))


@pytest.fixture(scope="module", params=[(synth.Q4_0, "f16"), (synth.Q5_1, "bf16")], ids=["Q4_0-f16", "Q5_1-bf16"])
def twin(request, shield_lib):
    qtype, type = request.param
    spec = synth.small_spec(qtype=qtype, n_layers=2, seed=17 + qtype)
    tensors = synth.make_model(spec)
    ctx = binding.ShieldContext(1)
    ctx.set_config(spec, max_positions=512, max_batch_tokens=600)
    ctx.upload_model(tensors)
    yield Twin(ctx, spec, tensors, type)
    ctx.close()


def ids(spec, n, seed):
    return np.random.default_rng(seed).integers(1, spec.vocab, size=n, dtype=np.int32)


def test_steps_on_forked_sequences(twin):
    ctx, kv, spec = twin.ctx, twin.kv, twin.spec
    (root,) = ctx.kv_open(kv, 1)
    prompt = [ids(spec, 211, 1)]
    got = ctx.kv_forward(kv, [root], prompt)
    np.testing.assert_array_equal(got, twin.step([root], prompt))
    kids = ctx.kv_fork(kv, [root] * 5)
    for chunks in ([ids(spec, n, 2 + n) for n in (1, 30, 2, 100, 17)], [ids(spec, 1, 30 + i) for i in range(5)],
                   [ids(spec, 1, 40 + i) for i in range(5)]):
        got = ctx.kv_forward(kv, kids, chunks)
        np.testing.assert_array_equal(got, twin.step(kids, chunks))
    ctx.kv_free(kv, [root, kids[1]])
    ctx.kv_compact(kv)
    kids = kids[[0, 2, 3, 4]]
    chunks = [ids(spec, 1, 50 + i) for i in range(4)]
    got = ctx.kv_forward(kv, kids, chunks)
    np.testing.assert_array_equal(got, twin.step(kids, chunks))
    # more tokens than a batch takes at once: two batches
    chunks = [ids(spec, 230, 60 + i) for i in range(3)]
    seqs = ctx.kv_open(kv, 3)
    got = ctx.kv_forward(kv, seqs, chunks)
    np.testing.assert_array_equal(got[:2], twin.step(seqs[:2], chunks[:2]))
    np.testing.assert_array_equal(got[2:], twin.step(seqs[2:], chunks[2:]))
    ctx.kv_free(kv, np.concatenate([kids, seqs]))
    assert ctx.kv_info(kv)["pages_used"] == 0


def test_the_exact_paths_are_as_they_were(twin):
    """Exact forwards before, between and after paged ones."""
    ctx, kv, spec = twin.ctx, twin.kv, twin.spec
    om = oracle_model(spec, twin.t)
    prompt = ids(spec, 90, 7)
    want = om.forward(prompt, np.arange(spec.vocab, dtype=np.int32))
    s = ctx.seq_create(128)
    seqs = ctx.kv_open(kv, 1)
    ctx.kv_forward(kv, seqs, [prompt], want_logits=False)
    np.testing.assert_array_equal(ctx.seq_forward([s], [prompt])[0], want)
    ctx.kv_forward(kv, seqs, [prompt[:5]], want_logits=False)
    np.testing.assert_array_equal(ctx.last_logits([prompt])[0], want)
    ctx.seq_release(s)
    ctx.kv_free(kv, seqs)


def test_refusals_and_cancellation_change_nothing(twin):
    ctx, kv, spec = twin.ctx, twin.kv, twin.spec
    a, b = ctx.kv_open(kv, 2)
    ctx.kv_forward(kv, [a], [ids(spec, 40, 1)], want_logits=False)
    used = ctx.kv_info(kv)["pages_used"]
    other = ctx.kv_create(twin.type, spec.n_layers + 1, spec.n_kv_heads, spec.head_dim, 16, 4)
    (far,) = ctx.kv_open(other, 1)
    small = ctx.kv_create(twin.type, spec.n_layers, spec.n_kv_heads, spec.head_dim, 16, 2)
    (tight,) = ctx.kv_open(small, 1)
    stop = np.array([1], np.int32)
    one = ids(spec, 1, 2)
    for code, call in [
        (binding.ERR_SHAPE, lambda: ctx.kv_forward(other, [far], [one])),
        (binding.ERR_ARG, lambda: ctx.kv_forward(kv, [far], [one])),
        (binding.ERR_ARG, lambda: ctx.kv_forward(kv, [a, a], [one, one])),
        (binding.ERR_ARG, lambda: ctx.kv_forward(kv, [a, b], [one, one[:0]])),
        (binding.ERR_RANGE, lambda: ctx.kv_forward(kv, [a, b], [one, ids(spec, 513, 3)])),
        (binding.ERR_RANGE, lambda: ctx.kv_forward(kv, [b], [np.array([spec.vocab], np.int32)])),
        (binding.ERR_NOMEM, lambda: ctx.kv_forward(small, [tight], [ids(spec, 33, 4)])),
        (binding.ERR_CANCELLED, lambda: ctx.kv_forward(kv, [a, b], [ids(spec, 20, 5), one], cancel=stop)),
    ]:
        with pytest.raises(binding.ShieldError) as e:
            call()
        assert e.value.code == code, str(e.value)
        assert ctx.kv_lengths(kv, [a, b]).tolist() == [40, 0] and ctx.kv_info(kv)["pages_used"] == used
    ctx.kv_release(other)
    ctx.kv_release(small)
    ctx.kv_free(kv, [a, b])


def test_a_forward_whose_wait_gave_up_changes_nothing(twin):
    ctx, kv, spec = twin.ctx, twin.kv, twin.spec
    seqs = ctx.kv_open(kv, 2)
    first = [ids(spec, 40, 1), ids(spec, 3, 2)]
    ctx.kv_forward(kv, seqs, first, want_logits=False)
    used = ctx.kv_info(kv)["pages_used"]
    chunks = [ids(spec, 20, 3), ids(spec, 1, 4)]
    ctx.debug_kv_error(kv, 0, 3)
    with pytest.raises(binding.ShieldError) as e:
        ctx.kv_forward(kv, seqs, chunks)
    assert e.value.code == binding.ERR_TIMEOUT
    assert ctx.kv_lengths(kv, seqs).tolist() == [40, 3] and ctx.kv_info(kv)["pages_used"] == used
    got = ctx.kv_forward(kv, seqs, chunks)
    np.testing.assert_array_equal(got, twin.step(seqs, chunks))
    ctx.kv_free(kv, seqs)


def test_decode_steps_keep_their_batch(twin):
    """A word set in the batch of one step is there in the next: the batch has not been made anew for one more position."""
    ctx, spec = twin.ctx, twin.spec
    kv = ctx.kv_create(twin.type, spec.n_layers, spec.n_kv_heads, spec.head_dim, 16, 20)
    seqs = ctx.kv_open(kv, 3)
    ctx.kv_forward(kv, seqs, [ids(spec, 40, i) for i in range(3)], want_logits=False)
    for n in range(4):
        ctx.kv_forward(kv, seqs, [ids(spec, 1, 9 + i) for i in range(3)], want_logits=False)
        ctx.debug_kv_error(kv, 0, 3)
        with pytest.raises(binding.ShieldError) as e:
            ctx.kv_forward(kv, seqs, [ids(spec, 1, 9 + i) for i in range(3)], want_logits=False)
        assert e.value.code == binding.ERR_TIMEOUT
    ctx.kv_release(kv)


def test_a_model_of_few_positions(twin):
    """Paged forwards where the exact attention's scratch for so few positions would not hold a batch's queries and outputs."""
    ctx = binding.ShieldContext(1)
    ctx.set_config(twin.spec, max_positions=64, max_batch_tokens=600)
    ctx.upload_model(twin.t)
    small = Twin(ctx, twin.spec, twin.t, twin.type)
    seqs = ctx.kv_open(small.kv, 12)
    for chunks in ([ids(twin.spec, 50 - i, i) for i in range(12)], [ids(twin.spec, 14, 20 + i) for i in range(12)]):
        got = ctx.kv_forward(small.kv, seqs, chunks)
        np.testing.assert_array_equal(got, small.step(seqs, chunks))
    ctx.close()
