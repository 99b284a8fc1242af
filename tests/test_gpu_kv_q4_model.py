"""The whole model on a 4-bit KV cache (KV_Q4), and sequences of a paged model
that share pages (fork_seq).

Tolerance against the oracle: both quantize the same K and V rows, computed in
fp32 in different orders, so a value within their rounding (about 1e-6 of
it) of a border between two codes may be stored one step d apart - of the
40,000 values a test stores, one or two (15 borders x 2 x 1e-6 each).  One
step is at most a 15th of its group's range; in a key it moves one position's
score by |q_i| d / sqrt(Dh) < 0.1, so its weight and a head's output by at most
a tenth, one head of at least four behind a residual: 2e-2 of the logits.
Two models that run the same kernels are compared with the same bound: the
projections add their splits in the order in which CTAs finish, so two runs
of one model differ by rounding too (4e-7 to 7e-6 of logits around 1 with
fp32 to fp16 rows), and a value may be stored one step apart.  The step is a
15th of the range for 4-bit rows, 2 / 254 of it for int8, 2^-10 of the value
for fp16: 2e-2, and that times 15 / 127 and 15 x 2^-10, at least doubled; fp32 rows
keep the rounding itself."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from lmc_b200 import synth
from tests.conftest import rel_err

pytestmark = pytest.mark.gpu

GPT2 = ("gpt2", dict(L=2, D=256, H=4, S=128, V=1000, seed=5))
LLAMA = ("llama", dict(L=2, D=512, H=8, Hkv=2, F=768, S=128, V=1000, seed=5))
MQA = ("llama", dict(L=2, D=512, H=16, Hkv=1, F=768, S=66, V=500, seed=6))  # 16 query heads of 32 on one kv head, an odd context


TOL = {rt.KV_F32: 1e-4, rt.KV_F16: 1e-3, rt.KV_Q8: 5e-3, rt.KV_Q4: 2e-2}


@pytest.mark.parametrize("kind,kw", [GPT2, LLAMA, MQA])
def test_logits_against_the_oracle(cuda, orc, model_dir, kind, kw):
    path = synth.cached_model(kind, model_dir, **kw)
    toks = np.random.default_rng(1).integers(0, kw["V"], 40)
    om = orc.model(path).set_kv(rt.KV_Q4)
    m = rt.Model(path, max_batch=1, kv_dtype=rt.KV_Q4)
    for p, t in enumerate(toks):
        got, nxt = m.forward([t], [p])
        assert rel_err(got[0], om.forward(int(t), p)) < 2e-2, p
        assert nxt[0] == int(np.argmax(got[0]))
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("kind,kw", [GPT2, LLAMA])
def test_paged_and_contiguous_caches_agree(cuda, model_dir, kind, kw):
    """The same rows read through pages, two sequences of different lengths;
    and greedy generation with and without a graph: each id it picks has the
    largest logit, within the bound, when the ids are fed back one by one."""
    path = synth.cached_model(kind, model_dir, **kw)
    load = lambda page: rt.Model(path, max_batch=2, kv_dtype=rt.KV_Q4, page_size=page, n_pages=12)  # noqa: E731
    a, b = load(0), load(16)
    toks = np.random.default_rng(2).integers(0, kw["V"], (60, 2))
    for p in range(60):
        pos = [p, p // 2]
        x, y = (m.forward(toks[p], pos)[0] for m in (a, b))
        assert rel_err(x, y) < TOL[rt.KV_Q4], p
    prompt = toks[:12].T
    check = load(0)
    for m in (a, b):
        for graph in (True, False):
            ids = m.generate(prompt, 30, use_graph=graph)
            fed = np.concatenate([prompt, ids], 1)
            for p in range(fed.shape[1] - 1):
                lg, _ = check.forward(fed[:, p], [p, p])
                if p >= prompt.shape[1] - 1:
                    for r in range(2):
                        assert lg[r].max() - lg[r][fed[r, p + 1]] < TOL[rt.KV_Q4] * np.linalg.norm(lg[r]), (p, r)
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("kind,kw", [LLAMA, MQA])
def test_prompt_chunks(cuda, orc, model_dir, kind, kw):
    """A prompt in chunks of 8 rows (appended as a batch, each row attending to
    its own past), then single tokens, against the oracle token by token."""
    path = synth.cached_model(kind, model_dir, **kw)
    toks = np.random.default_rng(3).integers(0, kw["V"], 30)
    om = orc.model(path).set_kv(rt.KV_Q4)
    m = rt.Model(path, max_batch=1, kv_dtype=rt.KV_Q4, max_rows=8)
    for p, t in enumerate(toks[:27]):
        want = om.forward(int(t), p)
    got, _ = m.prefill(0, toks[:27])
    assert rel_err(got, want) < 2e-2
    for p in range(27, 30):
        got, _ = m.forward([toks[p]], [p])
        assert rel_err(got[0], om.forward(int(toks[p]), p)) < 2e-2, p
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("kvd", [rt.KV_Q4, rt.KV_F16, rt.KV_F32, rt.KV_Q8])
def test_forked_sequences(cuda, model_dir, kvd):
    """Samples of one prompt: forked sequences give the logits of sequences that
    were each fed the prompt themselves, while they write into shared pages,
    rewind into them, give pages back and fork again."""
    path = synth.cached_model(LLAMA[0], model_dir, **LLAMA[1])
    V = LLAMA[1]["V"]
    rng = np.random.default_rng(4)
    prompt = rng.integers(0, V, 37)
    own = rt.Model(path, max_batch=4, kv_dtype=kvd, max_rows=16, page_size=16, n_pages=32)
    forked = rt.Model(path, max_batch=4, kv_dtype=kvd, max_rows=16, page_size=16, n_pages=32)
    for b in range(4):
        own.prefill(b, prompt)
    forked.prefill(2, prompt)
    for b in (0, 1, 3):
        forked.fork_seq(2, b)
    assert forked.kv_pages() == (16, 32, 29) and own.kv_pages() == (16, 32, 20)

    def step(toks, pos):
        x, y = (m.forward(toks, pos)[0] for m in (own, forked))
        for b in range(4):
            assert rel_err(x[b], y[b]) < TOL[kvd], (pos, b)

    for i in range(20):  # into the shared third page, on to pages of their own
        step(rng.integers(0, V, 4), [37 + i] * 4)
    # the first two pages stay shared; third and fourth: one each
    assert forked.kv_pages() == (16, 32, 32 - 2 - 8)
    t = rng.integers(0, V, 4)
    step(t, [3, 57, 20, 57])  # rewound: sequences 0 and 2 write into shared pages 1 and 2
    assert forked.kv_pages()[2] == 32 - 2 - 8 - 2
    # sequence 1 becomes a copy of 0, in both models (there by the same tokens is not possible: by forking too)
    for m in (own, forked):
        m.release_seq(1)
        m.fork_seq(0, 1)
    for i in range(5):
        step(rng.integers(0, V, 4), [4 + i, 4 + i, 21 + i, 58 + i])
    for m in (own, forked):
        for b in range(4):
            m.release_seq(b)
        assert m.kv_pages() == (16, 32, 32)
    assert rt.lib().lmc_device_status() == 0


def test_fork_of_a_contiguous_cache_is_refused(cuda, model_dir):
    path = synth.cached_model(GPT2[0], model_dir, **GPT2[1])
    m = rt.Model(path, max_batch=2, kv_dtype=rt.KV_Q4)
    with pytest.raises(rt.LmcError) as e:
        m.fork_seq(0, 1)
    assert e.value.code == -2


def test_head_sizes_4_bit_rows_cannot_hold_are_refused(cuda, model_dir):
    path = synth.cached_model("gpt2", model_dir, L=1, D=64, H=4, S=32, V=100, seed=1)  # heads of 16
    with pytest.raises(rt.LmcError) as e:
        rt.Model(path, max_batch=1, kv_dtype=rt.KV_Q4)
    assert e.value.code == -2 and "4-bit" in str(e.value)
