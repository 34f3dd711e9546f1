"""The 8-bit key/value cache on the GPU: rows written and read back, and the
attention of sequences that share a prefix, against plain 64-bit forms."""
import numpy as np
import pytest

from kv_q8_oracle import PAGE, attention, stored

pytestmark = pytest.mark.gpu


class Cache:
    """A pool with scrambled pages and a page table per sequence (row 0 of
    `lengths` may be a shared prefix)."""

    def __init__(self, B, kvh, hd, lengths, spare=3, seed=0, fill=None):
        import torch
        self.B, self.torch, self.kvh, self.hd = B, torch, kvh, hd
        pages = [(n + PAGE - 1) // PAGE for n in lengths]
        self.n_pages = sum(pages) + spare
        order = np.random.default_rng(seed).permutation(self.n_pages)
        self.width = max(1, max(pages, default=1))
        table = np.full((len(lengths), self.width), -1, np.int32)
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        self.table_np = table
        self.table = torch.from_numpy(table).cuda()
        nbytes = self.n_pages * B.kv_q8_page_bytes(kvh, hd)
        # stale contents: every byte set, so scales of unwritten tokens are NaN
        self.pages = torch.full((nbytes,), 0xFF if fill is None else fill, dtype=torch.uint8, device="cuda")
        self.pool = B.kv_q8_pool(self.pages, self.n_pages, kvh, hd)

    def i32(self, x):
        return self.torch.tensor(np.asarray(x, np.int64).astype(np.uint32).view(np.int32).reshape(-1), device="cuda")

    def write(self, k, v, counts, pos, first=0, stream=0):
        t = self.torch
        kd, vd = t.from_numpy(np.ascontiguousarray(k)).cuda(), t.from_numpy(np.ascontiguousarray(v)).cuda()
        row0 = self.i32(np.concatenate([[0], np.cumsum(counts)]))
        tab = self.table[first:first + len(counts)].contiguous()
        self.B.kv_q8_write_dev(self.pool, kd, vd, self.kvh * self.hd, k.shape[0], row0, tab, self.width,
                               self.i32(pos), len(counts), stream=stream)
        t.cuda.synchronize()

    def read(self, counts, pos, first=0):
        t = self.torch
        n = int(sum(counts))
        k = t.full((n, self.kvh, self.hd), 7.0, device="cuda")
        v = t.full((n, self.kvh, self.hd), 7.0, device="cuda")
        row0 = self.i32(np.concatenate([[0], np.cumsum(counts)]))
        tab = self.table[first:first + len(counts)].contiguous()
        self.B.kv_q8_read_dev(self.pool, k, v, self.kvh * self.hd, n, row0, tab, self.width, self.i32(pos),
                              len(counts))
        return k.cpu().numpy(), v.cpu().numpy()


def same(a, b):
    return np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)])


def rows(rng, n, kvh, hd, spread=1.0):
    x = rng.standard_normal((n, kvh, hd)).astype(np.float32)
    return (x * np.exp(spread * rng.standard_normal((n, kvh, 1)))).astype(np.float32)


@pytest.mark.parametrize("hd,kvh", [(64, 2), (128, 8), (256, 3), (128, 1)])
@pytest.mark.parametrize("counts,pos", [([1], [0]), ([1, 1, 1], [127, 128, 300]), ([33], [0]), ([31, 0, 130], [5, 9, 96]),
                                        ([511], [0]), ([257, 1, 64, 32], [31, 255, 64, 32])])
def test_write_read(gpu, hd, kvh, counts, pos):
    rng = np.random.default_rng(hd + kvh + sum(counts))
    n = sum(counts)
    k, v = rows(rng, n, kvh, hd, 3.0), rows(rng, n, kvh, hd, 3.0)
    c = Cache(gpu, kvh, hd, [p + m for p, m in zip(pos, counts)])
    c.write(k, v, counts, pos)
    kr, vr = c.read(counts, pos)
    assert same(kr, stored(k)[0]) and same(vr, stored(v)[0])
    assert gpu.take_device_errors() == 0


@pytest.mark.parametrize("n_seq,most", [(32, 2), (33, 3), (70, 40), (1100, 1), (1100, 12)])
def test_write_read_many_sequences(gpu, n_seq, most):
    """More sequences than one look-up holds, empty ones among them, row by row and by quarters."""
    rng = np.random.default_rng(n_seq + most)
    counts = rng.integers(0, most + 1, n_seq)
    pos = rng.integers(0, 100, n_seq)
    counts[-1], counts[n_seq // 2:n_seq // 2 + 3] = most, 0
    k, v = rows(rng, int(counts.sum()), 1, 64), rows(rng, int(counts.sum()), 1, 64)
    c = Cache(gpu, 1, 64, list(pos + counts + 1), seed=3)
    c.write(k, v, list(counts), list(pos))
    kr, vr = c.read(list(counts), list(pos))
    assert same(kr, stored(k)[0]) and same(vr, stored(v)[0])
    assert gpu.take_device_errors() == 0


def test_write_edge_values(gpu):
    """Zeros, subnormals, the largest floats, exact halves (ties), values just
    beside a half, NaN and infinities."""
    hd, kvh = 64, 1
    rng = np.random.default_rng(5)
    big = np.finfo(np.float32).max
    tiny = np.float32(2.0 ** -149)
    x = np.zeros((12, 1, hd), np.float32)
    x[1] = tiny
    x[2, 0, ::2] = -127 * tiny
    x[2, 0, 1::2] = 64 * tiny
    x[3] = big
    x[3, 0, 3] = -big / 3
    x[4, 0] = np.arange(hd) + 0.5          # amax 127: every element an exact half
    x[4, 0, -1] = 127.0
    x[5, 0] = np.nextafter(np.arange(hd, dtype=np.float32) + np.float32(0.5), np.float32(1e9))
    x[5, 0, -1] = -127.0
    x[6, 0] = np.nextafter(np.arange(hd, dtype=np.float32) + np.float32(0.5), np.float32(-1e9))
    x[6, 0, -1] = 127.0
    x[7, 0, 10] = np.nan
    x[8, 0, 11] = np.inf
    x[9, 0, 12] = -np.inf
    x[10, 0] = rng.standard_normal(hd) * 1e-36
    x[11, 0] = rng.standard_normal(hd) * 1e-44
    c = Cache(gpu, kvh, hd, [12])
    c.write(x, x[::-1], [12], [0])
    kr, vr = c.read([12], [0])
    assert same(kr, stored(x)[0]) and same(vr, stored(x[::-1])[0])


def test_write_many_near_halves(gpu):
    """Elements whose quotient lies within rounding of a half: decided by the
    exact quotient in every one of 2^20 cases."""
    rng = np.random.default_rng(11)
    n, kvh, hd = 1024, 8, 128
    amax = np.exp(rng.uniform(-20, 20, (n, kvh, 1))).astype(np.float32)
    steps = rng.integers(-127, 127, (n, kvh, hd)) + 0.5
    x = (steps / 127.0 * amax).astype(np.float32)
    x = np.where(rng.random(x.shape) < 0.5, np.nextafter(x, np.float32(0)), x).astype(np.float32)
    x[..., 0] = amax[..., 0]
    c = Cache(gpu, kvh, hd, [n])
    c.write(x, -x, [n], [0])
    kr, vr = c.read([n], [0])
    assert same(kr, stored(x)[0]) and same(vr, stored(-x)[0])


def test_strided_rows_and_untouched(gpu):
    """Rows inside a wider projection row; rows behind the last sequence, bad
    pages and positions are left out, and everything else stays as it was."""
    import torch
    rng = np.random.default_rng(2)
    kvh, hd, h = 2, 128, 4
    n = 40
    qkv = rng.standard_normal((n, (h + 2 * kvh) * hd)).astype(np.float32)
    c = Cache(gpu, kvh, hd, [100, 200], fill=0x11)
    before = c.pages.clone()
    dev = torch.from_numpy(qkv).cuda()
    kd, vd = dev[:, h * hd:], dev[:, (h + kvh) * hd:]
    row0 = c.i32([0, 10, 30])                      # rows 30 .. 39 belong to no sequence
    gpu.kv_q8_write_dev(c.pool, kd, vd, qkv.shape[1], n, row0, c.table, c.width, c.i32([3, 120]), 2)
    kr, vr = c.read([10, 20], [3, 120])
    want_k = qkv[:30, h * hd:(h + kvh) * hd].reshape(30, kvh, hd)
    want_v = qkv[:30, (h + kvh) * hd:].reshape(30, kvh, hd)
    assert same(kr, stored(want_k)[0]) and same(vr, stored(want_v)[0])
    # a token's block bytes: K row, V column, two scales -- nothing else moved
    changed = int((c.pages != before).sum())
    assert changed <= 30 * kvh * (2 * hd + 8)
    assert gpu.take_device_errors() == 0
    # out-of-range page and position: skipped, reported, nothing written
    before = c.pages.clone()
    bad = c.table.clone()
    bad[0, 0] = c.n_pages
    gpu.kv_q8_write_dev(c.pool, kd, vd, qkv.shape[1], n, row0, bad, c.width, c.i32([3, c.width * PAGE]), 2)
    assert gpu.take_device_errors() == 1 << 5
    assert torch.equal(c.pages, before)
    out = torch.full((n, kvh, hd), 9.0, device="cuda")
    gpu.kv_q8_read_dev(c.pool, out, out.clone(), kvh * hd, n, row0, bad, c.width, c.i32([3, c.width * PAGE]), 2)
    assert gpu.take_device_errors() == 1 << 5
    assert bool((out == 9.0).all())


def test_read_leaves_rows_behind_the_last_sequence(gpu):
    import torch
    rng = np.random.default_rng(3)
    c = Cache(gpu, 2, 64, [50])
    x = rows(rng, 50, 2, 64)
    c.write(x, x, [50], [0])
    k = torch.full((60, 2, 64), 5.0, device="cuda")
    v = torch.full((60, 2, 64), 6.0, device="cuda")
    gpu.kv_q8_read_dev(c.pool, k, v, 128, 60, c.i32([0, 50]), c.table, c.width, c.i32([0]), 1)
    assert same(k[:50].cpu().numpy(), stored(x)[0])
    assert bool((k[50:] == 5.0).all()) and bool((v[50:] == 6.0).all())


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
class Batch:
    def __init__(self, B, H, kvh, hd, prefix, lens, counts, seed=0, q_gain=1.5, spread=0.5, edit=None):
        rng = np.random.default_rng(seed)
        self.B, self.H, self.kvh, self.hd = B, H, kvh, hd
        self.prefix, self.lens, self.counts = prefix, lens, counts
        self.kp, self.vp = rows(rng, prefix, kvh, hd, spread), rows(rng, prefix, kvh, hd, spread)
        self.ks = [rows(rng, n, kvh, hd, spread) for n in lens]
        self.vs = [rows(rng, n, kvh, hd, spread) for n in lens]
        self.q = (q_gain * rng.standard_normal((sum(counts), H, hd))).astype(np.float32)
        self.scale = 1.0 / np.sqrt(hd)
        if edit:
            edit(self)
        c = self.c = Cache(B, kvh, hd, [prefix] + list(lens), seed=seed)
        if prefix:
            c.write(self.kp, self.vp, [prefix], [0])
        if sum(lens):
            c.write(np.concatenate(self.ks), np.concatenate(self.vs), lens, [0] * len(lens), first=1)
        t = c.torch
        self.tab = c.table[1:].contiguous()
        self.ptab, self.plen = c.table[0].contiguous(), c.i32([prefix])
        self.len_d = c.i32(lens)
        self.row0 = c.i32(np.concatenate([[0], np.cumsum(counts)]))
        self.qd = t.from_numpy(self.q).cuda()
        self.out = t.full((sum(counts) + 2, H, hd), 3.0, device="cuda")  # two rows behind the last
        self.batch = B.attn_batch(prefix_table=self.ptab, prefix_len=self.plen, max_prefix=prefix, table=self.tab,
                                  table_stride=c.width, seq_len=self.len_d, max_len=max(lens), row0=self.row0,
                                  n_seq=len(lens), n_rows=max(1, sum(counts)), max_rows=max(1, max(counts)))
        self.scratch = t.empty(B.kv_q8_attn_scratch_bytes(c.pool, self.batch, H), dtype=t.uint8, device="cuda")

    def run(self, stream=0):
        w = self.H * self.hd
        self.B.kv_q8_attn_dev(self.c.pool, self.batch, self.qd, w, self.out, w, self.H, self.scale, self.scratch,
                              self.scratch.numel(), stream=stream)

    def want(self):
        st = lambda x: stored(x)[0]
        return attention(self.q, self.counts, st(self.kp) if self.prefix else None,
                         st(self.vp) if self.prefix else None, [st(k) for k in self.ks], [st(v) for v in self.vs],
                         self.scale)

    def check(self):
        self.run()
        n = sum(self.counts)
        got = self.out.cpu().numpy()
        assert np.all(got[n:] == 3.0)
        want, tol = self.want()
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got[:n]), nan)
        err = np.abs(got[:n].astype(np.float64) - want)
        err[nan] = 0
        with np.errstate(invalid="ignore"):
            over = err > np.where(np.isnan(tol), np.inf, tol)
        assert not over.any(), (float(err.max()), float(np.nanmax(err / tol)))
        assert self.B.take_device_errors() == 0
        return got[:n]


SHAPES = [(4, 4, 128), (8, 2, 64), (4, 2, 256), (8, 1, 128), (28, 4, 128)]


@pytest.mark.parametrize("H,kvh,hd", SHAPES)
@pytest.mark.parametrize("prefix,lens,counts", [
    (0, [1], [1]), (0, [128], [1]), (0, [129], [3]), (1, [1], [1]), (127, [5, 1], [2, 1]), (128, [31, 33, 200], [1, 1, 1]),
    (300, [7, 0, 64, 129], [4, 0, 1, 7]), (641, [1] * 9, [1] * 9), (0, [40, 300], [40, 33])])
def test_attention(gpu, H, kvh, hd, prefix, lens, counts):
    Batch(gpu, H, kvh, hd, prefix, lens, counts, seed=prefix + sum(lens)).check()


@pytest.mark.parametrize("prefix,lens,counts", [(5000, [3, 700], [1, 2]), (2049, [100] * 20, [1] * 20)])
def test_attention_long(gpu, prefix, lens, counts):
    Batch(gpu, 4, 2, 128, prefix, lens, counts, seed=1).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_units(gpu, hd):
    """More units (a head of a sequence) than CTAs: each takes several in turn."""
    Batch(gpu, 16, 16, hd, 200, [20, 5, 130] * 14, [5, 5, 6] * 14, seed=hd).check()


def test_rows_without_any_key(gpu):
    """Sequences with no visible token give 0, with and without neighbours."""
    b = Batch(gpu, 4, 2, 64, 0, [0, 1, 2], [1, 3, 2], seed=4)  # row 0 none; rows 1, 2 of sequence 1 none
    got = b.check()
    assert np.all(got[0] == 0) and np.all(got[1:3] == 0) and np.any(got[3] != 0)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_extreme_scales(gpu, hd):
    """Rows of very uneven magnitude, peaked and flat softmax, zero keys and
    values, one zero query."""
    def edit(b):
        b.vp[::3] *= 1e4
        b.vp[1::3] *= 1e-4
        b.vp[5] = 0
        b.kp[7] = 0
        b.ks[1][:] = 0
        b.vs[0] *= 1e-30
        b.q[0] = 0
        b.q[2] *= 20
    Batch(gpu, 4, 2, hd, 260, [140, 10], [2, 2], seed=8, edit=edit).check()


@pytest.mark.parametrize("scale", [0.0, -0.11, 1e-20, 3.0])
def test_softmax_scales(gpu, scale):
    """Scale 0 averages the visible values; a negative one turns the order."""
    def edit(b):
        b.scale = scale
    Batch(gpu, 4, 2, 128, 140, [20, 3], [3, 1], seed=17, q_gain=0.5, edit=edit).check()


@pytest.mark.parametrize("gain", [1e30, 1e-25])
def test_large_queries_small_keys_and_the_reverse(gpu, gain):
    """Scores of ordinary size from factors far apart."""
    def edit(b):
        b.q *= np.float32(gain)
        for x in [b.kp] + b.ks:
            x *= np.float32(1 / gain)
    Batch(gpu, 4, 2, 128, 300, [140, 40], [2, 30], seed=19, edit=edit).check()


@pytest.mark.parametrize("gain,prefix,counts", [(1e36, 300, [2, 30]), (1e36, 0, [1, 1]), (1e30, 300, [2, 30]), (1e30, 20, [2, 2])])
def test_scores_beyond_every_exponent(gpu, gain, prefix, counts):
    """Scores of 1e3 to 1e10: one value row each, no NaN."""
    def edit(b):
        b.q *= np.float32(gain)
        for x in [b.kp] + b.ks:
            x *= np.float32(1e-29)
        b.scale = 40.0
    b = Batch(gpu, 4, 2, 128, prefix, [140, 40], counts, seed=20, edit=edit)
    got = b.check()
    vals = np.concatenate([stored(b.vp)[0]] + [stored(v)[0] for v in b.vs])
    for r in {0, 1, min(10, sum(counts) - 1), sum(counts) - 1}:  # each output is one of the stored value rows
        for h in range(4):
            assert np.abs(vals[:, h // 2] - got[r, h]).max(-1).min() <= 1e-5 * np.abs(vals).max()


def test_nan_and_infinity_reach_only_rows_that_see_them(gpu):
    def edit(b):
        b.ks[0][3, 0, 5] = np.nan      # seen by every row of sequence 0's heads 0, 1
        b.vs[1][9, 1, 0] = np.inf      # token 9 of 10: only the last row of sequence 1 sees it
        b.q[4, 2, 7] = np.inf
    b = Batch(gpu, 4, 2, 64, 50, [20, 10, 6], [2, 2, 1], seed=3, edit=edit)
    want, _ = b.want()
    b.run()
    got = b.out.cpu().numpy()[:5]
    bad = np.isnan(got).all(-1)
    assert np.array_equal(np.isnan(got).any(-1), bad)
    expect = np.zeros((5, 4), bool)
    expect[0:2, 0:2] = True
    expect[3, 2:4] = True
    expect[4, 2] = True
    assert np.array_equal(bad, expect)
    ok = ~bad
    assert np.max(np.abs(got[ok] - want[ok])) < 1e-4


def test_results_do_not_depend_on_timing(gpu):
    b = Batch(gpu, 8, 2, 128, 3001, [50, 400, 17], [1, 3, 1], seed=6)
    b.run()
    first = b.out.clone()
    for _ in range(5):
        b.out.zero_()
        b.run()
        assert b.c.torch.equal(b.out[:5], first[:5])


def test_graph_replay_follows_lengths_and_tables(gpu):
    """One captured call, replayed after the sequences grew and moved."""
    import torch
    b = Batch(gpu, 4, 2, 128, 300, [64, 200], [1, 2], seed=9)
    full_prefix, full_lens = b.prefix, list(b.lens)
    s = torch.cuda.Stream()
    b.run(stream=s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        b.run(stream=torch.cuda.current_stream().cuda_stream)
    for plen, lens in ((300, [64, 200]), (5, [1, 2]), (0, [64, 129]), (299, [33, 131])):
        b.plen.copy_(b.c.i32([plen]))
        b.len_d.copy_(b.c.i32(lens))
        b.out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        kp, vp, ks, vs = b.kp, b.vp, b.ks, b.vs
        b.prefix, b.kp, b.vp = plen, kp[:plen], vp[:plen]
        b.ks, b.vs = [k[:n] for k, n in zip(ks, lens)], [v[:n] for v, n in zip(vs, lens)]
        want, tol = b.want()
        got = b.out.cpu().numpy()[:3]
        assert np.all(np.abs(got - want) <= tol)
        b.kp, b.vp, b.ks, b.vs, b.prefix = kp, vp, ks, vs, full_prefix
    assert full_lens == [64, 200]


def test_write_attend_verify_in_one_graph(gpu):
    """A decode step of four sequences -- rows written, attention over the shared
    prefix, drafts verified -- captured once and replayed as they grow."""
    import torch
    from kv_q8_oracle import verify
    H, kvh, hd, V, n, k = 8, 4, 64, 96, 4, 2
    rng = np.random.default_rng(77)
    b = Batch(gpu, H, kvh, hd, 150, [140] * n, [k] * n, seed=31)
    c = b.c
    head = torch.from_numpy(rng.standard_normal((H * hd, V)).astype(np.float32)).cuda()
    new_k = torch.zeros(n * k, kvh, hd, device="cuda")
    new_v = torch.zeros_like(new_k)
    pos, drafts = c.i32([0] * n), c.i32(rng.integers(0, V, n))
    qp = torch.softmax(torch.from_numpy(rng.standard_normal((n, 1, V)).astype(np.float32)).cuda(), -1)
    u = torch.zeros(n, k, device="cuda")
    probs = torch.zeros(n, k, V, device="cuda")
    tok, cnt = torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")

    def step(stream):
        gpu.kv_q8_write_dev(c.pool, new_k, new_v, kvh * hd, n * k, b.row0, b.tab, c.width, pos, n, stream=stream)
        b.run(stream=stream)
        probs.copy_(torch.softmax(b.out[:n * k].view(n * k, -1) @ head, -1).view(n, k, V))
        gpu.verify_draft_dev(probs, qp, V, drafts, None, k - 1, u, n, V, tok, cnt, stream=stream)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(torch.cuda.current_stream().cuda_stream)
    lens = [100, 126, 127, 64]
    base_k, base_v = [x.copy() for x in b.ks], [x.copy() for x in b.vs]
    for x in base_k + base_v:
        x[:k] = 0  # the pass before the capture wrote its zeros at position 0
    for it in range(3):
        kk = rng.standard_normal((n * k, kvh, hd)).astype(np.float32)
        vv = rng.standard_normal((n * k, kvh, hd)).astype(np.float32)
        un = rng.random((n, k)).astype(np.float32)
        new_k.copy_(torch.from_numpy(kk))
        new_v.copy_(torch.from_numpy(vv))
        u.copy_(torch.from_numpy(un))
        pos.copy_(c.i32(lens))
        b.len_d.copy_(c.i32([x + k for x in lens]))
        g.replay()
        torch.cuda.synchronize()
        for i in range(n):
            base_k[i][lens[i]:lens[i] + k] = kk[i * k:(i + 1) * k]
            base_v[i][lens[i]:lens[i] + k] = vv[i * k:(i + 1) * k]
        b.ks = [base_k[i][:lens[i] + k] for i in range(n)]
        b.vs = [base_v[i][:lens[i] + k] for i in range(n)]
        want, tol = b.want()
        assert np.all(np.abs(b.out[:n * k].cpu().numpy() - want) <= tol)
        got = verify(probs.cpu().numpy(), qp.cpu().numpy(), drafts.cpu().numpy().reshape(n, 1), [k - 1] * n, un)
        for i in range(n):
            assert int(cnt[i]) == len(got[i]) and list(tok[i, :len(got[i])].cpu().numpy()) == got[i]
        lens = [x + k for x in lens]
    assert gpu.take_device_errors() == 0


@pytest.mark.parametrize("counts,prefix", [([1, 2], 0), ([1, 1], 300), ([9, 40], 300), ([70, 3], 0)])
def test_rows_before_the_first_sequence(gpu, counts, prefix):
    """row0[0] > 0: rows that belong to nobody, in front."""
    import torch
    b = Batch(gpu, 4, 2, 128, prefix, [130, 50], counts, seed=23)
    skip = 5
    n = sum(counts)
    b.qd = torch.cat([torch.ones(skip, 4, 128, device="cuda"), b.qd])
    b.out = torch.full((skip + n + 2, 4, 128), 3.0, device="cuda")
    b.row0 = b.c.i32(np.concatenate([[0], np.cumsum(counts)]) + skip)
    b.batch = gpu.attn_batch(prefix_table=b.ptab, prefix_len=b.plen, max_prefix=prefix, table=b.tab,
                             table_stride=b.c.width, seq_len=b.len_d, max_len=130, row0=b.row0, n_seq=2,
                             n_rows=skip + n + 2, max_rows=max(counts))
    b.qd = torch.cat([b.qd, b.qd[:2]])
    b.scratch = torch.empty(gpu.kv_q8_attn_scratch_bytes(b.c.pool, b.batch, 4), dtype=torch.uint8, device="cuda")
    b.run()
    got = b.out.cpu().numpy()
    want, tol = b.want()
    assert np.all(got[:skip] == 3.0) and np.all(got[skip + n:] == 3.0)
    assert np.all(np.abs(got[skip:skip + n] - want) <= tol)
    # and the rows written: those of the sequences only
    k = torch.randn(skip + n + 2, 2, 128, device="cuda")
    pos = b.c.i32([40, 1])
    gpu.kv_q8_write_dev(b.c.pool, k, -k, 256, skip + n + 2, b.row0, b.tab, b.c.width, pos, 2)
    rk, rv = torch.full_like(k, 3.0), torch.full_like(k, 3.0)
    gpu.kv_q8_read_dev(b.c.pool, rk, rv, 256, skip + n + 2, b.row0, b.tab, b.c.width, pos, 2)
    for got, x in ((rk, k), (rv, -k)):
        got = got.cpu().numpy()
        assert np.array_equal(got[skip:skip + n], stored(x.cpu().numpy())[0][skip:skip + n])
        assert np.all(got[:skip] == 3.0) and np.all(got[skip + n:] == 3.0)
    assert gpu.take_device_errors() == 0


def test_nothing_to_attend_to_follows_its_inputs(gpu):
    """No prefix and no own tokens: zeros, with row0 written just before."""
    import torch
    b = Batch(gpu, 4, 2, 64, 0, [1, 1], [2, 3], seed=2)
    batch = gpu.attn_batch(table=b.tab, table_stride=b.c.width, seq_len=b.len_d, max_len=0, row0=b.row0, n_seq=2, n_rows=5,
                           max_rows=3)
    b.len_d.zero_()
    scratch = torch.empty(max(16, gpu.kv_q8_attn_scratch_bytes(b.c.pool, batch, 4)), dtype=torch.uint8, device="cuda")
    rows = [[0, 2, 5], [0, 3, 5], [1, 3, 4]]
    for r in rows:
        b.out.fill_(3.0)
        b.row0.copy_(b.c.i32(r))
        gpu.kv_q8_attn_dev(b.c.pool, batch, b.qd, 256, b.out, 256, 4, 0.1, scratch, scratch.numel())
        got = b.out.cpu().numpy()
        assert np.all(got[r[0]:r[2]] == 0) and np.all(got[:r[0]] == 3.0) and np.all(got[r[2]:] == 3.0)
    assert gpu.take_device_errors() == 0


FIRST_CALL = """
import torch
from eosllm_b200 import backend as B
pages = torch.empty(2 * B.kv_q8_page_bytes(1, 64), dtype=torch.uint8, device="cuda")
pool = B.kv_q8_pool(pages, 2, 1, 64)
k = torch.randn(130, 1, 64, device="cuda")
out = [torch.zeros_like(k) for _ in range(2)]
tab, pos = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [0]))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    B.kv_q8_write_dev(pool, k, k, 64, 130, None, tab, 2, pos, 1, stream=st)
    B.kv_q8_read_dev(pool, out[0], out[1], 64, 130, None, tab, 2, pos, 1, stream=st)
g.replay()
torch.cuda.synchronize()
assert float((out[0] - k).abs().max()) <= float(k.abs().max()) / 254 * 1.001 and torch.equal(out[0], out[1])
assert B.take_device_errors() == 0
"""


def test_first_call_on_a_device_may_be_captured(gpu):
    """In a process of its own, where nothing has set the library up."""
    import pathlib
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=pathlib.Path(__file__).parent.parent, timeout=300,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_calls_at_once_with_their_own_scratch(gpu):
    import torch
    a = Batch(gpu, 8, 4, 128, 2000, [100] * 4, [1] * 4, seed=21)
    b = Batch(gpu, 8, 4, 128, 1777, [90] * 5, [2] * 5, seed=22)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        a.run(stream=s1.cuda_stream)
        b.run(stream=s2.cuda_stream)
    torch.cuda.synchronize()
    a.check()
    b.check()


def test_bad_pages_and_lengths_are_left_out(gpu):
    """A page outside the pool hides its tokens; a length beyond its bound is
    cut; both are reported."""
    b = Batch(gpu, 4, 2, 64, 256, [30], [1], seed=12)
    b.ptab[1] = b.c.n_pages + 7
    b.run()
    got = b.out.cpu().numpy()[:1]
    assert gpu.take_device_errors() == 1 << 5
    b.prefix, b.kp, b.vp = 128, b.kp[:128], b.vp[:128]
    want, tol = b.want()
    assert np.all(np.abs(got - want) <= tol)
    b = Batch(gpu, 4, 2, 64, 256, [30], [1], seed=12)
    b.plen.copy_(b.c.i32([100000]))
    b.run()
    got = b.out.cpu().numpy()[:1]
    assert gpu.take_device_errors() == 1 << 5
    want, tol = b.want()
    assert np.all(np.abs(got - want) <= tol)


def test_strided_queries_and_outputs(gpu):
    import torch
    b = Batch(gpu, 4, 2, 64, 100, [20, 30], [2, 1], seed=13)
    w = 4 * 64
    wide = torch.full((3, w + 128), 2.0, device="cuda")
    wide[:, :w] = b.qd.view(3, w)
    out = torch.full((3, w + 64), 4.0, device="cuda")
    gpu.kv_q8_attn_dev(b.c.pool, b.batch, wide, w + 128, out, w + 64, 4, b.scale, b.scratch, b.scratch.numel())
    want, tol = b.want()
    assert np.all(np.abs(out[:, :w].cpu().numpy().reshape(3, 4, 64) - want) <= tol)
    assert bool((out[:, w:] == 4.0).all())


def test_uniform_rows_without_row0(gpu):
    b = Batch(gpu, 4, 2, 64, 100, [20, 30, 9], [2, 2, 2], seed=14)
    b.batch = gpu.attn_batch(prefix_table=b.ptab, prefix_len=b.plen, max_prefix=100, table=b.tab,
                             table_stride=b.c.width, seq_len=b.len_d, max_len=30, n_seq=3, n_rows=6, max_rows=2)
    b.check()


def test_pages_beyond_4_gib(gpu):
    """Offsets that pass 32 bits: the last pages of a pool of 4.3 GB."""
    import torch
    kvh, hd = 8, 128
    page = gpu.kv_q8_page_bytes(kvh, hd)
    n_pages = (1 << 32) // page + 8
    c = Cache(gpu, kvh, hd, [1])
    c.pages = None
    c.n_pages = n_pages
    c.pages = torch.zeros(n_pages * page, dtype=torch.uint8, device="cuda")
    c.pool = gpu.kv_q8_pool(c.pages, n_pages, kvh, hd)
    c.width = 2
    c.table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(0)
    k, v = rows(rng, 200, kvh, hd), rows(rng, 200, kvh, hd)
    c.write(k, v, [200], [0])
    kr, vr = c.read([200], [0])
    assert same(kr, stored(k)[0]) and same(vr, stored(v)[0])
    q = torch.from_numpy(rng.standard_normal((1, kvh, hd)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    ln = c.i32([200])
    b = gpu.attn_batch(table=c.table, table_stride=2, seq_len=ln, max_len=256, n_seq=1, n_rows=1, max_rows=1)
    scratch = torch.empty(gpu.kv_q8_attn_scratch_bytes(c.pool, b, kvh), dtype=torch.uint8, device="cuda")
    gpu.kv_q8_attn_dev(c.pool, b, q, kvh * hd, out, kvh * hd, kvh, 0.1, scratch, scratch.numel())
    want, tol = attention(q.cpu().numpy(), [1], None, None, [stored(k)[0]], [stored(v)[0]], 0.1)
    assert np.all(np.abs(out.cpu().numpy() - want) <= tol)


def test_host_pointers_are_refused(gpu):
    import torch
    c = Cache(gpu, 2, 64, [10])
    x = np.zeros((10, 2, 64), np.float32)
    with pytest.raises(gpu.CudaBackendError):
        gpu.kv_q8_write_dev(c.pool, torch.from_numpy(x), torch.from_numpy(x), 128, 10, c.i32([0, 10]), c.table,
                            c.width, c.i32([0]), 1)
