"""Verification of drafted tokens on the GPU against a plain 64-bit form."""
import numpy as np
import pytest

from kv_q8_oracle import verify

pytestmark = pytest.mark.gpu

NO = 0xFFFFFFFF


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def make(n, kk, vocab, seed, noise=0.7, gain=2.5):
    rng = np.random.default_rng(seed)
    lg = gain * rng.standard_normal((n, kk + 1, vocab))
    p = softmax(lg)
    q = softmax(lg[:, :kk] + noise * rng.standard_normal((n, kk, vocab)))
    drafts = np.zeros((n, kk), np.uint32)
    for i in range(n):
        for j in range(kk):
            drafts[i, j] = rng.choice(vocab, p=q[i, j].astype(np.float64) / q[i, j].astype(np.float64).sum())
    u = rng.random((n, kk + 1)).astype(np.float32)
    return p, q, drafts, u


def run(B, p, q, drafts, n_draft, u, pad=0, stream=0):
    import torch
    n, k1, vocab = p.shape
    kk = k1 - 1
    stride = vocab + pad

    def rows(x):
        w = np.full(x.shape[:2] + (stride,), np.nan, np.float32)
        w[..., :vocab] = x
        return torch.from_numpy(w).cuda()

    pd, qd = rows(p), (rows(q) if kk else None)
    dd = torch.from_numpy(drafts.view(np.int32)).cuda() if kk else None
    nd = None if n_draft is None else torch.from_numpy(np.asarray(n_draft, np.int32)).cuda()
    ud = torch.from_numpy(u).cuda()
    tok = torch.full((n + 1, kk + 1), 77, dtype=torch.int32, device="cuda")
    cnt = torch.full((n + 1,), 77, dtype=torch.int32, device="cuda")
    B.verify_draft_dev(pd, qd, stride, dd, nd, kk, ud, n, vocab, tok, cnt, stream=stream)
    torch.cuda.synchronize()
    assert bool((tok[n] == 77).all()) and int(cnt[n]) == 77
    return tok[:n].cpu().numpy().view(np.uint32), cnt[:n].cpu().numpy()


def check(B, p, q, drafts, n_draft, u, pad=0):
    tok, cnt = run(B, p, q, drafts, n_draft, u, pad)
    kk = p.shape[1] - 1
    nd = np.full(p.shape[0], kk) if n_draft is None else np.minimum(np.asarray(n_draft).astype(np.uint32), kk)
    want = verify(p, q, drafts, nd, u)
    for i, w in enumerate(want):
        assert cnt[i] == len(w)
        assert list(tok[i]) == w + [NO] * (kk + 1 - len(w)), i
    return tok, cnt


@pytest.mark.parametrize("n,kk,vocab,pad", [(1, 0, 1, 0), (1, 0, 33, 3), (3, 1, 320, 0), (1, 4, 32000, 0), (5, 7, 4099, 1),
                                            (17, 3, 1000, 24), (2, 2, 128001, 0), (64, 5, 257, 0), (200, 2, 320, 0)])
def test_matches_the_plain_form(gpu, n, kk, vocab, pad):
    for seed in range(3):
        p, q, d, u = make(n, kk, vocab, seed + n)
        check(gpu, p, q, d, None, u, pad)


def test_ragged_draft_counts(gpu):
    p, q, d, u = make(9, 5, 640, 3, noise=0.1)
    check(gpu, p, q, d, [0, 1, 2, 3, 4, 5, 0, 5, 99], u)


def test_every_point_of_rejection(gpu):
    """u = 0 accepts, a draft without target probability is rejected, equal
    rows accept everything, a residual of nothing draws from the target."""
    p, q, d, u = make(6, 4, 50, 1)
    u[:, :4] = 0.0
    for i in range(4):
        p[i, i, d[i, i]] = 0.0          # rejected at i
    q[4] = p[4, :4]                     # always accepted
    u[4, :4] = np.nextafter(np.float32(1), np.float32(0))
    q[5, 0] = p[5, 0] * np.float32(2)   # p <= q everywhere: rejected at u = 0.9, residual empty
    u[5, 0] = 0.9
    _, cnt = check(gpu, p, q, d, None, u)
    assert list(cnt) == [1, 2, 3, 4, 5, 1]


def test_draw_covers_the_row(gpu):
    """The drawn token for u = 0, just below 1, and at every border of a row
    of powers of two (sums are exact, so is the border)."""
    vocab = 64
    w = np.zeros((1, 1, vocab), np.float32)
    w[0, 0, 5], w[0, 0, 6], w[0, 0, 40], w[0, 0, 63] = 0.25, 0.25, 0.25, 0.25
    us = [0.0, 0.25, 0.5, 0.75, float(np.nextafter(np.float32(1), np.float32(0))),
          float(np.nextafter(np.float32(0.25), np.float32(0)))]
    want = [5, 6, 40, 63, 63, 5]
    for u, t in zip(us, want):
        tok, cnt = run(gpu, w, w[:, :0], np.zeros((1, 0), np.uint32), None, np.full((1, 1), u, np.float32))
        assert int(tok[0, 0]) == t and int(cnt[0]) == 1


def test_rows_need_not_sum_to_one_and_bad_weights_count_zero(gpu):
    p, q, d, u = make(4, 2, 100, 9)
    p *= np.float32(37.0)
    q *= np.float32(37.0)
    p[:, :, 3] = np.nan
    p[:, :, 4] = -1.0
    p[:, :, 5] = np.inf
    q[:, :, 6] = np.nan
    d[d < 7] = 8
    check(gpu, p, q, d, None, u)


def test_row_without_weight_and_token_outside_the_vocabulary(gpu):
    p, q, d, u = make(3, 1, 40, 2)
    p[0] = 0.0
    d[1, 0] = 40
    d[2, 0] = NO
    tok, cnt = check(gpu, p, q, d, None, u)
    assert cnt[0] == 0 and np.all(tok[0] == NO)
    assert cnt[1] == 1 and cnt[2] == 1


def test_accepted_share_matches_the_distributions(gpu):
    """Drawn tokens follow the target: 4096 independent sequences, 8 tokens;
    5 standard deviations of a binomial count."""
    rng = np.random.default_rng(0)
    n, vocab = 4096, 8
    p = np.repeat(softmax(rng.standard_normal((1, 2, vocab)) * 1.5), n, 0)
    q = np.repeat(softmax(rng.standard_normal((1, 1, vocab)) * 1.5), n, 0)
    d = rng.choice(vocab, size=(n, 1), p=q[0, 0].astype(np.float64) / q[0, 0].astype(np.float64).sum()).astype(np.uint32)
    u = rng.random((n, 2)).astype(np.float32)
    tok, _ = run(gpu, p, q, d, None, u)
    counts = np.bincount(tok[:, 0], minlength=vocab)
    mean = n * p[0, 0].astype(np.float64)
    assert np.all(np.abs(counts - mean) <= 5 * np.sqrt(mean * (1 - p[0, 0])) + 1)


def test_captured_call_sees_new_numbers(gpu):
    import torch
    p, q, d, u = make(3, 2, 320, 5)
    pd, qd = torch.from_numpy(p).cuda(), torch.from_numpy(q).cuda()
    dd, ud = torch.from_numpy(d.view(np.int32)).cuda(), torch.from_numpy(u).cuda()
    tok = torch.zeros((3, 3), dtype=torch.int32, device="cuda")
    cnt = torch.zeros(3, dtype=torch.int32, device="cuda")

    def call(stream):
        gpu.verify_draft_dev(pd, qd, 320, dd, None, 2, ud, 3, 320, tok, cnt, stream=stream)

    s = torch.cuda.Stream()
    call(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call(torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2, 3):
        u2 = np.random.default_rng(seed).random(u.shape).astype(np.float32)
        ud.copy_(torch.from_numpy(u2).cuda())
        g.replay()
        torch.cuda.synchronize()
        want = verify(p, q, d, [2, 2, 2], u2)
        for i, w in enumerate(want):
            assert int(cnt[i]) == len(w) and list(tok[i, :len(w)].cpu().numpy()) == w
