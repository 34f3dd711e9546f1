"""The decoder's 8-bit cache mode and its branches, against a plain decoder in
numpy whose linears are the oracle's int8 kernel and whose keys and values are
quantised as the cache holds them.

Tolerance.  Sums in another order and CUDA's expf / sincosf differ from numpy's by
rounding; where a value lies on a border of the int8 packing, that turns into
one quantisation step.  Its size, in the input of a linear of width 256 whose
32-element groups of normal values have a largest element of about 2.2 rms:
2.2 / 127 / sqrt(256) = 1.1e-3 of an output's rms times a normal weight.  The
layers behind it re-round a vector perturbed by 1.1e-3 rms, 6 % of a step of 2.2
/ 127 rms: 6 % of 256 elements, 15 of them, go the other way, sqrt(15) * 1.1e-3 =
4.2e-3 rms, three times that, 1.3e-2, at the largest of 320 logits; two such
linears add to sqrt(2) * 1.3e-2 = 1.8e-2.  The bound is 2e-2 of the logits' rms
(an unrelated token's logits differ by about 3)."""
from __future__ import annotations

import numpy as np
import pytest

from kv_q8_oracle import stored
from oracle.llama import make_llama
from oracle.oracle import DT_Q4_K, DT_Q8_0

pytestmark = pytest.mark.gpu

TOL = 2e-2


def rms(x):
    return float(np.sqrt(np.mean(np.square(np.asarray(x, np.float64)))))


def err(got, want):
    return float(np.max(np.abs(np.asarray(got, np.float64) - want)) / rms(want))


class PlainDecoder:
    """eosi_text_step with an 8-bit cache (numpy)."""

    def __init__(self, oracle, model):
        self.o, self.m, self.c = oracle, model, model["config"]
        self.hd = self.c["n_embd"] // self.c["n_head"]
        self.k = [[] for _ in range(self.c["n_layer"])]
        self.v = [[] for _ in range(self.c["n_layer"])]

    def _mul(self, a, w, n, dt=None):
        dt = self.c["wdtype"] if dt is None else dt
        return self.o.matmul_q(np.ascontiguousarray(a, np.float32), w, dt, 1, n, a.size)[1].reshape(-1)

    def _norm(self, x, w):
        x = x.astype(np.float64)
        return (x / np.sqrt(np.mean(x * x) + self.c["rms_eps"]) * w).astype(np.float32)

    def _rope(self, x, pos):
        i = np.arange(0, self.hd, 2)
        th = np.float64(pos) * self.c["rope_base"] ** (-i / self.hd)
        cs, sn = np.cos(th), np.sin(th)
        y = x.reshape(-1, self.hd).astype(np.float64)
        out = np.empty_like(y)
        out[:, 0::2] = y[:, 0::2] * cs - y[:, 1::2] * sn
        out[:, 1::2] = y[:, 0::2] * sn + y[:, 1::2] * cs
        return out.astype(np.float32)

    def step(self, token):
        c, hd = self.c, self.hd
        E, H, KV, F = c["n_embd"], c["n_head"], c["n_kv_head"], c["n_ff"]
        x = self.m["tok_embd"].view(np.float16).reshape(-1, E)[token].astype(np.float32)
        pos = len(self.k[0])
        for L, lay in enumerate(self.m["layers"]):
            h = self._norm(x, lay["attn_norm"])
            q = self._rope(self._mul(h, lay["wq"], E), pos)
            k = self._rope(self._mul(h, lay["wk"], KV * hd), pos)
            v = self._mul(h, lay["wv"], KV * hd).reshape(KV, hd)
            self.k[L].append(stored(k)[0])
            self.v[L].append(stored(v)[0])
            ks, vs = np.stack(self.k[L]).astype(np.float64), np.stack(self.v[L]).astype(np.float64)
            out = np.empty((H, hd))
            for i in range(H):
                g = i * KV // H
                s = ks[:, g] @ q[i].astype(np.float64) / np.sqrt(hd)
                p = np.exp(s - s.max())
                out[i] = (p / p.sum()) @ vs[:, g]
            x = x + self._mul(out.reshape(-1).astype(np.float32), lay["wo"], E)
            h = self._norm(x, lay["ffn_norm"])
            gate, up = self._mul(h, lay["wg"], F), self._mul(h, lay["wu"], F)
            x = x + self._mul((gate / (1 + np.exp(-gate.astype(np.float64))) * up).astype(np.float32), lay["wd"], E)
        return self._mul(self._norm(x, self.m["output_norm"]), self.m["output"], c["n_vocab"], c["out_dtype"])


def decoder(model, q8=True):
    from eosllm_b200.text import TextDecoder
    d = TextDecoder(model)
    if q8:
        d.set_cache(TextDecoder.CACHE_Q8)
        assert d.cache == TextDecoder.CACHE_Q8
    return d


def toks(n, vocab, seed):
    return np.random.default_rng(seed).integers(0, vocab, n).astype(np.uint32)


@pytest.mark.parametrize("kw", [dict(), dict(n_kv_head=2), dict(wdtype=DT_Q8_0, out_dtype=DT_Q8_0),
                                dict(n_embd=512, n_head=4, n_kv_head=2), dict(n_embd=512, n_head=2, n_kv_head=1)])
def test_steps_match_the_plain_decoder(gpu, oracle, kw):
    model = make_llama(oracle, max_ctx=160, **kw)
    d, ref = decoder(model), PlainDecoder(oracle, model)
    for t in toks(12, model["config"]["n_vocab"], 1):
        want = ref.step(int(t))
        assert err(d.step(int(t)), want) <= TOL
    d.close()


def test_prefill_continues_like_steps_across_pages(gpu, oracle):
    """Prompts of 1 to 300 tokens in one pass, then steps, against stepping."""
    model = make_llama(oracle, n_layer=2, n_kv_head=2, max_ctx=400)
    prompt = toks(303, 320, 2)
    a, b = decoder(model), decoder(model)
    at = 0
    for n in (1, 3, 4, 5, 17, 98, 130, 42):     # blocks that end inside and at page borders
        a.prefill(prompt[at:at + n])
        for t in prompt[at:at + n]:
            b.step(int(t))
        at += n
        assert a.pos == b.pos == at
    for t in prompt[at:at + 3]:
        assert err(a.step(int(t)), b.step(int(t))) <= TOL
    a.close()
    b.close()


def test_generate_and_reset(gpu, oracle):
    model = make_llama(oracle, max_ctx=200)
    d, ref = decoder(model), PlainDecoder(oracle, model)
    prompt = toks(40, 320, 3)
    got = d.generate(prompt, 5)
    for t in prompt:
        lg = ref.step(int(t))
    for t in got:
        best = int(np.argmax(lg))
        assert t == best or lg[best] - lg[t] <= 2 * TOL * rms(lg)
        lg = ref.step(int(t))
    d.reset()
    assert np.array_equal(d.generate(prompt, 5), got)
    d.close()


def test_changing_the_cache_keeps_f32_results(gpu, oracle):
    from eosllm_b200.text import TextDecoder
    model = make_llama(oracle, max_ctx=64)
    d = decoder(model, q8=False)
    prompt = toks(20, 320, 4)
    first = [d.step(int(t)) for t in prompt]
    with pytest.raises(gpu.CudaBackendError):
        d.set_cache(TextDecoder.CACHE_Q8)        # not at position 0
    d.reset()
    d.set_cache(TextDecoder.CACHE_Q8)
    d.step(1)
    d.reset()
    d.set_cache(TextDecoder.CACHE_F32)
    for t, w in zip(prompt, first):
        assert np.array_equal(d.step(int(t)), w)
    with pytest.raises(gpu.CudaBackendError):
        d.set_cache(7)
    d.close()


@pytest.mark.parametrize("n_prompt", [0, 20, 127, 128, 200])
def test_branches_follow_their_own_tokens(gpu, oracle, n_prompt):
    """Three branches fed different tokens, most likely token drawn, against a
    decoder of their own each; then one is adopted and goes on."""
    model = make_llama(oracle, n_layer=2, n_kv_head=2, max_ctx=320)
    V = 320
    prompt = toks(n_prompt, V, 5)
    d = decoder(model)
    if n_prompt:
        d.prefill(prompt)
    d.fork(3, 40)
    feed = np.array([[3], [77], [200]], np.uint32)
    fed = [list(prompt) for _ in range(3)]
    refs = []
    for i in range(3):
        r = decoder(model)
        if n_prompt:
            r.prefill(prompt)
        refs.append(r)
    for s in range(12):
        out = d.branch_step(feed, np.full((3, 1), 0.3), temperature=0.0)
        for i in range(3):
            lg = refs[i].step(int(feed[i, 0]))
            fed[i].append(int(feed[i, 0]))
            best, t = int(np.argmax(lg)), int(out[i][0])
            assert len(out[i]) == 1 and (t == best or lg[best] - lg[t] <= 2 * TOL * rms(lg)), (s, i)
        feed = np.array([[o[0]] for o in out], np.uint32)
    d.adopt(1)
    assert d.pos == n_prompt + 12
    for t in (9, 10):
        assert err(d.step(t), refs[1].step(t)) <= TOL
    for r in refs + [d]:
        r.close()


def test_drafts_are_verified(gpu, oracle):
    """Drafts that follow the most likely path are accepted, others are not;
    the cache keeps only what was accepted."""
    model = make_llama(oracle, n_layer=2, max_ctx=300)
    prompt = toks(130, 320, 6)
    a = decoder(model)
    a.prefill(prompt)
    a.fork(1, 60)
    path, t = [], 5
    for _ in range(9):
        t = int(a.branch_step([[t]], [[0.5]], temperature=0.0)[0][0])
        path.append(t)
    a.close()
    b = decoder(model)
    b.prefill(prompt)
    b.fork(2, 60, max_draft=4)
    wrong = [(p + 1) % 320 for p in path]
    # branch 0: all right; branch 1: wrong at the third
    out = b.branch_step([[5] + path[:4], [5] + path[:2] + [wrong[2], path[3]]], np.full((2, 5), 0.5), temperature=0.0)
    assert list(out[0]) == path[:5]
    assert list(out[1]) == path[:3]
    # both go on, now with one draft (branch 1's is wrong at once)
    out = b.branch_step([[path[4], path[5]], [path[2], wrong[3]]], np.full((2, 2), 0.5), temperature=0.0)
    assert list(out[0]) == path[5:7]
    assert list(out[1]) == path[3:4]
    b.adopt(0)
    assert b.pos == 130 + 5 + 2
    b.close()


def test_draws_follow_the_random_numbers(gpu, oracle):
    """Eight branches, temperature 0.7: each drawn token sits where its number
    falls in the running sum of the step's own softmax."""
    model = make_llama(oracle, max_ctx=200)
    prompt = toks(33, 320, 7)
    d, r = decoder(model), decoder(model)
    d.prefill(prompt)
    r.prefill(prompt)
    d.fork(8, 5)
    u = np.linspace(0.0, 0.97, 8).astype(np.float32)[:, None]
    out = d.branch_step(np.full((8, 1), 11), u, temperature=0.7)
    lg = r.step(11).astype(np.float64) / 0.7
    p = np.exp(lg - lg.max())
    c = np.concatenate([[0], np.cumsum(p / p.sum())])
    # logits off by TOL of their rms move every probability by that much / 0.7
    slack = 2 * TOL * rms(lg)
    for i in range(8):
        t = int(out[i][0])
        assert c[t] - slack <= u[i, 0] <= c[t + 1] + slack
    d.close()
    r.close()


def test_drawn_drafts_use_their_probabilities(gpu, oracle):
    """Draft probabilities equal to the target's accept every draft; draft
    probabilities of a token that cannot follow reject it."""
    model = make_llama(oracle, max_ctx=200)
    d, r = decoder(model), decoder(model)
    prompt = toks(20, 320, 8)
    d.prefill(prompt)
    r.prefill(prompt)
    d.fork(2, 10, max_draft=1)
    lg = r.step(4).astype(np.float64)
    p = np.exp(lg - lg.max())
    p /= p.sum()
    x = int(np.argmax(p))
    q = np.zeros((2, 1, 320), np.float32)
    q[0, 0] = p
    q[1, 0, x] = 1.0
    # accepted when u q(x) < p(x): 0.9 p(x) < p(x) whatever the rounding; 0.999 * 1 is above p(x)
    assert p[x] < 0.9
    out = d.branch_step([[4, x], [4, x]], [[0.9, 0.1], [0.999, 0.1]], draft_probs=q, temperature=1.0)
    assert len(out[0]) == 2 and out[0][0] == x
    assert len(out[1]) == 1 and out[1][0] != x
    d.close()
    r.close()


def test_refusals(gpu, oracle):
    from eosllm_b200.text import TextDecoder
    E = gpu.CudaBackendError

    def refused(status, fn, *a, **k):
        with pytest.raises(E) as ex:
            fn(*a, **k)
        assert ex.value.status == status

    model = make_llama(oracle, max_ctx=64)
    d = decoder(model, q8=False)
    refused(gpu.EOS_E_UNSUPPORTED, d.fork, 2, 8)                       # f32 cache
    d.set_step_mode(TextDecoder.STEP_PERSISTENT)
    refused(gpu.EOS_E_UNSUPPORTED, d.set_cache, TextDecoder.CACHE_Q8)  # persistent step
    d.set_step_mode(TextDecoder.STEP_AUTO)
    d.set_cache(TextDecoder.CACHE_Q8)
    refused(gpu.EOS_E_UNSUPPORTED, d.set_step_mode, TextDecoder.STEP_PERSISTENT)
    d.prefill(toks(30, 320, 1))
    refused(gpu.EOS_E_INVALID_ARG, d.fork, 0, 8)
    refused(gpu.EOS_E_INVALID_ARG, d.fork, 33, 8, 1)                   # 66 rows, max_ctx 64
    refused(gpu.EOS_E_OUT_OF_MEMORY, d.fork, 2, 35)
    refused(gpu.EOS_E_INVALID_ARG, d.adopt, 0)
    d.fork(2, 4, max_draft=1)
    refused(gpu.EOS_E_INVALID_ARG, d.fork, 2, 4)
    refused(gpu.EOS_E_INVALID_ARG, d.step, 1)
    refused(gpu.EOS_E_INVALID_ARG, d.generate, toks(2, 320, 1), 2)
    refused(gpu.EOS_E_INVALID_ARG, d.prefill, toks(2, 320, 1))
    ok = np.zeros((2, 1), np.uint32), np.zeros((2, 1), np.float32)
    refused(gpu.EOS_E_INVALID_ARG, d.branch_step, ok[0] + 320, ok[1])
    refused(gpu.EOS_E_INVALID_ARG, d.branch_step, ok[0], ok[1] + 1)
    refused(gpu.EOS_E_INVALID_ARG, d.branch_step, ok[0], ok[1], temperature=-1.0)
    refused(gpu.EOS_E_INVALID_ARG, d.branch_step, np.zeros((2, 3), np.uint32), np.zeros((2, 3), np.float32))
    with pytest.raises(ValueError):
        d.branch_step(np.zeros((3, 1)), np.zeros((3, 1)))
    for _ in range(4):
        d.branch_step(*ok)
    refused(gpu.EOS_E_OUT_OF_MEMORY, d.branch_step, *ok)               # max_new reached
    refused(gpu.EOS_E_INVALID_ARG, d.adopt, 2)
    d.close_branches()
    assert d.pos == 30
    d.step(1)
    d.fork(2, 4)
    d.reset()                                                          # closes them
    d.step(1)
    d.close()
    q80 = decoder(make_llama(oracle, max_ctx=64, wdtype=DT_Q8_0, out_dtype=DT_Q8_0))
    q80.step(1)
    refused(gpu.EOS_E_UNSUPPORTED, q80.fork, 2, 4)
    q80.close()
    assert DT_Q4_K == 33
