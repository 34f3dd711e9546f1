"""The attention over the 8-bit cache where its integers, masks and bounds end:
sums of one sign, tokens that a row may not see, rows that see nothing."""
import numpy as np
import pytest

from kv_q8_oracle import PAGE, stored
from test_gpu_kv_q8 import Batch, Cache, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("count", [1, 6, 20])
@pytest.mark.parametrize("pattern", ["flat", "alternating", "random"])
@pytest.mark.parametrize("opposed", [0.0, 0.5, 1.0])
def test_queries_along_and_against_the_keys(gpu, hd, count, pattern, opposed):
    """Every product of a score has the same sign: sums of head_dim * 127 * 128
    and a little less, both ways.  A flat query has the digits -32, -90, 127."""
    rng = np.random.default_rng(hd + count)
    sign = {"flat": np.ones(hd), "alternating": 1.0 - 2.0 * (np.arange(hd) % 2),
            "random": 1.0 - 2.0 * rng.integers(0, 2, hd)}[pattern].astype(np.float32)

    def edit(b):
        b.q[:] = 0.6 * sign
        for x in [b.kp] + b.ks:
            turn = np.where(rng.random((x.shape[0], x.shape[1], 1)) < opposed, -1.0, 1.0)
            x[:] = sign * turn * rng.uniform(0.2, 1.0, (x.shape[0], x.shape[1], 1))
    Batch(gpu, 4, 2, hd, 150, [140], [count], seed=hd, edit=edit).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,length,prefix", [(2, 90, 0), (2, 129, 40), (4, 130, 0), (3, 300, 200), (7, 131, 40), (20, 90, 0),
                                             (40, 290, 130)])
def test_later_tokens_leave_earlier_rows_as_they_are(gpu, hd, n, length, prefix):
    """Rows of one sequence whose later tokens -- the other drafts, the rest of a
    prompt -- hold values 1e4 and 1e9 times as large: the earlier rows keep the
    accuracy of what they see, and are the same to the bit whatever stands there.
    Up to four rows a head, and more (H = kv heads, and pairs of heads)."""
    for H in (2, 4):
        def edit(b):
            b.vs[0][length - 1] *= np.float32(1e4)
            b.vs[0][length - n // 2 - 1] *= np.float32(1e9)
            b.ks[0][length - 1] *= np.float32(3.0)
        b = Batch(gpu, H, 2, hd, prefix, [length], [n], seed=n + hd, edit=edit)
        got = b.check()
        rng = np.random.default_rng(5)
        for t in {0, n // 2, n - 2}:  # rows 0 .. t see tokens 0 .. length - n + t
            seen = length - n + t + 1
            k, v = rows(rng, length - seen, 2, hd), rows(rng, length - seen, 2, hd)
            b.c.write(k, np.float32(1e-9) * v if t else v, [length - seen], [seen], first=1)
            b.run()
            again = b.out.cpu().numpy()[:n]
            assert np.array_equal(again[:t + 1].view(np.uint32), got[:t + 1].view(np.uint32)), t
            b.c.write(b.ks[0], b.vs[0], [length], [0], first=1)


@pytest.mark.parametrize("n,prefix", [(1, 100), (3, 0), (3, 100), (40, 100)])
def test_lengths_are_reported_without_own_tokens(gpu, n, prefix):
    """max_len = 0: a sequence length above it is left out and reported, and so
    are rows beyond max_rows, whether or not there is a prefix."""
    b = Batch(gpu, 2, 2, 64, prefix, [1] * n, [1] * n, seed=n)

    def call(max_rows, row0):
        b.row0.copy_(b.c.i32(row0))
        b.batch = gpu.attn_batch(prefix_table=b.ptab, prefix_len=b.plen, max_prefix=prefix, table=b.tab,
                                 table_stride=b.c.width, seq_len=b.len_d, max_len=0, row0=b.row0, n_seq=n, n_rows=n,
                                 max_rows=max_rows)
        b.scratch = b.c.torch.empty(max(16, gpu.kv_q8_attn_scratch_bytes(b.c.pool, b.batch, 2)),
                                    dtype=b.c.torch.uint8, device="cuda")
        b.run()
        return gpu.take_device_errors()

    every = list(range(n + 1))
    b.len_d.zero_()
    assert call(1, every) == 0
    b.len_d[n - 1] = 1
    assert call(1, every) == 1 << 5
    b.len_d.zero_()
    if n > 1:  # the first sequence has two rows where one is the most, the second none
        assert call(1, [0, 2] + every[2:]) == 1 << 5


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("H,n,length,prefix", [(2, 3, 1, 0), (2, 3, 0, 0), (4, 9, 4, 0), (4, 9, 0, 0), (2, 40, 30, 0)])
def test_rows_that_see_nothing_are_zero_whatever_their_query(gpu, bad, H, n, length, prefix):
    """Rows 0 .. n - length - 1 see no token: 0, also where the query holds a NaN
    or an infinity and the sequence has tokens for later rows; a row that sees
    one is NaN."""
    def edit(b):
        b.q[:, :, 5] = bad
    b = Batch(gpu, H, 2, 64, prefix, [length, 3], [n, 1], seed=n, edit=edit)
    b.run()
    got = b.out.cpu().numpy()[:n + 1]
    assert np.all(got[:n - length] == 0) and np.all(np.isnan(got[n - length:]))
    assert gpu.take_device_errors() == 0


@pytest.mark.parametrize("hd,max_rows", [(64, 9), (128, 40)])
@pytest.mark.parametrize("row0", [[0, 9, 2, 9, 0], [9, 0, 1, 2, 3], [40, 40, 0, 40, 40], [0, 40, 0, 40, 0],
                                  [0, 0xFFFFFFFF, 5, 0xFFFFFFFF, 40]])
def test_row0_that_is_not_ascending(gpu, hd, max_rows, row0):
    """Row starts that go down or beyond n_rows: which rows are computed is not
    defined, but nothing outside the batch is touched and the next call is right."""
    n = 40
    b = Batch(gpu, 4, 2, hd, 140, [130, 1, 300, 7], [10] * 4, seed=hd)
    good_batch, good_row0, good_scratch = b.batch, b.row0, b.scratch
    b.row0 = b.c.i32(row0)
    b.batch = gpu.attn_batch(prefix_table=b.ptab, prefix_len=b.plen, max_prefix=140, table=b.tab,
                             table_stride=b.c.width, seq_len=b.len_d, max_len=300, row0=b.row0, n_seq=4, n_rows=n,
                             max_rows=max_rows)
    b.scratch = b.c.torch.empty(gpu.kv_q8_attn_scratch_bytes(b.c.pool, b.batch, 4), dtype=b.c.torch.uint8, device="cuda")
    b.run()
    b.c.torch.cuda.synchronize()
    assert np.all(b.out.cpu().numpy()[n:] == 3.0)
    k = b.c.torch.full((n + 2, 2, hd), 5.0, device="cuda")
    gpu.kv_q8_read_dev(b.c.pool, k, k.clone(), 2 * hd, n, b.row0, b.tab, b.c.width, b.c.i32([0] * 4), 4)
    assert bool((k[n:] == 5.0).all())
    gpu.take_device_errors()
    b.batch, b.row0, b.scratch = good_batch, good_row0, good_scratch
    b.check()


@pytest.mark.parametrize("count", [1, 2, 6, 20])
@pytest.mark.parametrize("q_gain,k_gain,scale", [(4e37, 1e-38, 1e6), (1e37, 1e-36, -1e4), (1e-28, 1e28, 2.0), (3e37, 1e-30, 1e-7)])
def test_factors_at_the_ends_of_the_range(gpu, count, q_gain, k_gain, scale):
    """Scores of ordinary size or far apart, from a query, a key and a scale whose
    products in another order leave the f32 range."""
    def edit(b):
        b.q *= np.float32(q_gain)
        for x in [b.kp] + b.ks:
            x *= np.float32(k_gain)
        b.scale = scale
    Batch(gpu, 4, 2, 64, 150, [40], [count], seed=count, edit=edit).check()


def value_whose_scale_is_just_below_a_power_of_two():
    for up in range(-40, 40):
        a = np.float32(127.0 * (2.0 - 2.0 ** -23)) * np.float32(1 + up * 2.0 ** -24)
        if (np.float32(a * (np.float32(1.0) / np.float32(127.0))).view(np.uint32) & 0x7FFFFF) == 0x7FFFFF:
            return a
    raise AssertionError


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("prefix,length,count", [(0, 1, 1), (1, 1, 3), (1, 4, 20), (200, 30, 3), (200, 30, 20), (300, 130, 40)])
def test_a_value_scale_just_below_a_power_of_two(gpu, hd, prefix, length, count):
    """A weight is rounded as probability 1 times the largest value scale of its
    page, whose mantissa is all ones; queries of 0 give every token that
    probability exactly, the others give it to one."""
    big = value_whose_scale_is_just_below_a_power_of_two()

    def edit(b):
        b.q[::2] = 0
        for x in [b.vp] + b.vs:
            x[:] = np.clip(x, -100, 100)
            x[::3, :, hd // 2] = big
    Batch(gpu, 4, 2, hd, prefix, [length], [count], seed=count + hd, spread=0.0, edit=edit).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("top", [1.01, 1.4, 1.98])
def test_weights_use_their_integers_whole(gpu, hd, top):
    """The rounding of probabilities times value scales, on rows where little else
    is rounded (queries of 1 and -1 are integers of any unit): one page, and the
    largest value scale anywhere between two powers of two.

    Bound.  A weight is off by up to half of u = vs_max / 8388604, evenly spread:
    u^2 / 12 in the mean square, times the square of the value integer, summed over
    the tokens.  A probability is off by ex2's 2^-22.5 at most, 2^-23.5 in the root
    mean square, and by the f32 roundings of its score z (in log2 units): the sum,
    the difference and the product, each 2^-24 |z| / sqrt(3) or less.  The rest (the
    sum of probabilities, folding, the quotient) is four times 2^-24 of the output or
    less.  Every part but the first is an upper bound, so the root mean square over
    24 x 2 x hd outputs (6144 weights, 1 % of it) is below their sum's; a unit of a
    power of two doubles the first part at worst."""
    rng = np.random.default_rng(hd)
    tokens = 128

    def edit(b):
        b.q[:] = np.where(rng.random(b.q.shape) < 0.5, -1.0, 1.0)
        b.scale = 1.5 * 0.125 * (64 / hd) ** 0.5
        s = rng.uniform(0.3, 1.0, (tokens, 2, 1))
        s[5] = top
        b.vp[:] = b.vp / np.abs(b.vp).max(-1, keepdims=True) * 127 * s
    b = Batch(gpu, 2, 2, hd, tokens, [0], [24], seed=hd, spread=0.0, edit=edit)
    b.run()
    got = b.out.cpu().numpy()[:24].astype(np.float64)
    k, (v, vs) = stored(b.kp)[0].astype(np.float64), stored(b.vp)
    v, vs = v.astype(np.float64), vs.astype(np.float64)
    err, pred = [], []
    for r in range(24):
        for h in range(2):
            z = (k[:, h] @ b.q[r, h].astype(np.float64)) * b.scale
            z -= z.max()
            p = np.exp(z)
            out = p @ v[:, h] / p.sum()
            z2 = np.log2(np.e) * (np.abs(z) + np.abs(z).max())
            rho2 = 2.0 ** -47 + 3 * (np.log(2) * 2.0 ** -24 * z2) ** 2 / 3
            ints = v[:, h] / vs[:, h, None]
            var = (vs[:, h].max() / 8388604) ** 2 / 12 * (ints ** 2).sum(0) + ((p[:, None] * v[:, h]) ** 2 * rho2[:, None]).sum(0)
            err.append(got[r, h] - out)
            pred.append(var / p.sum() ** 2 + (4 * 2.0 ** -24 * out) ** 2)
    err, pred = np.sqrt(np.mean(np.square(err))), np.sqrt(np.mean(pred))
    assert err <= pred, (err, pred, err / pred)
    assert gpu.take_device_errors() == 0
