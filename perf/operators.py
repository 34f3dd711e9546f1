"""Workloads of the quantised key/value cache operators.

Three operators that a decoder with several sequences uses one after the
other: key and value rows quantised to 8 bits as they enter the paged cache
(and read back), attention of a batch of sequences that share a prefix held in
that cache, and verification of drafted tokens against the target's
probabilities.

`own` chooses between the plain form (elementary torch operations in 32 bits,
64 where a value sits next to a rounding or sampling border) and the library's
kernels.  Sizes follow the decoder's 7B shape (32 heads of 128, vocabulary
32000, 511-token prompts, positions 512..767), its small test models (heads of
64, grouped heads) and generic serving sizes.
"""
import math

import torch

own = False

PAGE = 128        # tokens of a cache page
NO_TOKEN = -1     # output slots behind the last token of a sequence


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one new token of each of 16 sequences of the 7B shape enters one layer's cache
        dict(name="write_step_16", kind="write", seqs=16, rows=1, ragged=False, heads=32, kv_heads=32, dim=128, pos=700),
        # a 511-token prompt of the 7B shape, one layer
        dict(name="write_prompt_511", kind="write", seqs=1, rows=511, ragged=False, heads=32, kv_heads=32, dim=128,
             pos=0),
        # prompts of uneven lengths, grouped heads, continuing inside a page
        dict(name="write_batch_ragged", kind="write", seqs=9, rows=2049, ragged=True, heads=32, kv_heads=8, dim=128,
             pos=77),
        # a short odd span of a small model read back
        dict(name="read_777_d64", kind="read", seqs=1, rows=777, ragged=False, heads=8, kv_heads=2, dim=64, pos=5),
        # a whole long context of the 7B shape read back, one layer
        dict(name="read_16383", kind="read", seqs=1, rows=16383, ragged=False, heads=32, kv_heads=32, dim=128, pos=0),
        # one decode step of one sequence of the 7B shape, no shared prefix
        dict(name="attn_step_1", kind="attn", seqs=1, rows=1, ragged=False, heads=32, kv_heads=32, dim=128, prefix=0,
             own_min=640, own_max=640),
        # 16 samples of one 4096-token prompt, a few hundred tokens in
        dict(name="attn_samples_16", kind="attn", seqs=16, rows=1, ragged=False, heads=32, kv_heads=32, dim=128,
             prefix=4096, own_min=1, own_max=300),
        # drafted tokens of several branches over an odd prefix
        dict(name="attn_drafts_7", kind="attn", seqs=7, rows=6, ragged=True, heads=32, kv_heads=32, dim=128,
             prefix=1537, own_min=6, own_max=100),
        # a serving batch with grouped heads over a very long shared document
        dict(name="attn_batch_48_long", kind="attn", seqs=48, rows=1, ragged=False, heads=32, kv_heads=8, dim=128,
             prefix=65537, own_min=1, own_max=700),
        # a small model's heads of 64, some sequences without a key of their own yet
        dict(name="attn_small_d64", kind="attn", seqs=33, rows=2, ragged=True, heads=8, kv_heads=2, dim=64,
             prefix=1000, own_min=2, own_max=500),
        # one sequence's four drafted tokens
        dict(name="verify_1", kind="verify", seqs=1, drafts=4, ragged=False, vocab=32000),
        # a batch of branches with uneven draft lengths
        dict(name="verify_64", kind="verify", seqs=64, drafts=7, ragged=True, vocab=32000),
    ]


def _span(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "verify"])
    heads, kv_heads, dim = rng.choice([(32, 32, 128), (32, 8, 128), (8, 2, 64), (16, 16, 64), (8, 4, 256), (12, 4, 128),
                                       (28, 4, 128)])
    if kind == "verify":
        return dict(kind=kind, seqs=_span(rng, 1, 64), drafts=rng.randint(0, 7), ragged=rng.random() < 0.5,
                    vocab=_span(rng, 320, 32000))
    if kind == "attn":
        seqs = _span(rng, 1, 48)
        rows = rng.choice([1, 1, 2, 3, 6])
        prefix = rng.choice([0, _span(rng, 1, 16384), _span(rng, 100, 16384)])
        own_max = _span(rng, rows, 700)
        return dict(kind=kind, seqs=seqs, rows=rows, ragged=rng.random() < 0.5, heads=heads, kv_heads=kv_heads, dim=dim,
                    prefix=prefix, own_min=min(rows, own_max), own_max=own_max)
    seqs = _span(rng, 1, 16)
    return dict(kind=kind, seqs=seqs, rows=_span(rng, 1, 8192 // seqs), ragged=rng.random() < 0.5, heads=heads,
                kv_heads=kv_heads, dim=dim, pos=rng.choice([0, 1, 127, 128, rng.randint(0, 3000)]))


def _counts(case):
    """New rows of each sequence (ragged: between 1 and case["rows"])."""
    n, top = case["seqs"], case["rows"]
    if not case["ragged"]:
        return [top] * n
    return [1 + (7919 * i + 5 * top + 3) % top for i in range(n)]


def _own_lengths(case):
    """Cached tokens of each sequence behind the prefix, its new rows included."""
    lo, hi = case["own_min"], case["own_max"]
    return [max(lo + (104729 * i + 17 * hi) % (hi - lo + 1), c) for i, c in enumerate(_counts(case))]


def _draft_counts(case):
    n, top = case["seqs"], case["drafts"]
    if not case["ragged"]:
        return [top] * n
    return [(7919 * i + 3) % (top + 1) for i in range(n)]


def work(case):
    d = case.get("dim", 0)
    if case["kind"] in ("write", "read"):
        n = sum(_counts(case)) * case["kv_heads"]
        cache, values = n * (2 * d + 8), n * 2 * d * 4
        if case["kind"] == "read":
            return {"bytes": cache + values, "flops": 2 * n * d}
        return {"bytes": values + cache + values, "flops": 8 * n * d}  # rows in, cache, values out
    if case["kind"] == "attn":
        counts, lens = _counts(case), _own_lengths(case)
        rows = sum(counts)
        keys = case["prefix"] + sum(lens)
        pairs = sum(c * (case["prefix"] + n - c) + c * (c + 1) // 2 for c, n in zip(counts, lens))
        return {"bytes": keys * case["kv_heads"] * (2 * d + 8) + 2 * rows * case["heads"] * d * 4,
                "flops": 4 * pairs * case["heads"] * d}
    k = _draft_counts(case)
    # a sequence needs one row of the target and, after a rejection, the
    # draft's row too; which one happens depends on the numbers: count the target's
    return {"bytes": case["seqs"] * case["vocab"] * 4 + sum(k) * 16, "flops": 2 * case["seqs"] * case["vocab"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _kv_rows(g, n, kv_heads, dim):
    """Key and value rows: keys with a few large channels, rows of uneven size."""
    channel = 1.0 + 6.0 * (torch.rand(1, kv_heads, dim, generator=g, device="cuda") < 0.03).float()
    k = _normal(g, n, kv_heads, dim) * channel
    v = _normal(g, n, kv_heads, dim) * (0.25 + torch.rand(n, kv_heads, 1, generator=g, device="cuda"))
    return k, v


def _inputs(case, seed):
    """The operator's inputs as plain tensors, from the seed alone."""
    g = _generator(seed)
    if case["kind"] in ("write", "read"):
        n, h, kvh, d = sum(_counts(case)), case["heads"], case["kv_heads"], case["dim"]
        k, v = _kv_rows(g, n, kvh, d)
        if case["kind"] == "write":  # rows as the projection leaves them: [q heads | k heads | v heads]
            qkv = torch.empty(n, (h + 2 * kvh) * d, device="cuda", dtype=torch.float32)
            qkv[:, :h * d] = 0.5
            qkv[:, h * d:(h + kvh) * d] = k.reshape(n, kvh * d)
            qkv[:, (h + kvh) * d:] = v.reshape(n, kvh * d)
            k, v = qkv[:, h * d:(h + kvh) * d], qkv[:, (h + kvh) * d:]
        return dict(k=k, v=v, g=g)
    if case["kind"] == "attn":
        kvh, d = case["kv_heads"], case["dim"]
        kp, vp = _kv_rows(g, case["prefix"], kvh, d)
        ks, vs = _kv_rows(g, sum(_own_lengths(case)), kvh, d)
        q = 1.5 * _normal(g, sum(_counts(case)), case["heads"], d)
        return dict(kp=kp, vp=vp, ks=ks, vs=vs, q=q, g=g)
    n, kk, vocab = case["seqs"], case["drafts"], case["vocab"]
    logits = 2.5 * _normal(g, n, kk + 1, vocab)
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :kk] + 0.7 * _normal(g, n, kk, vocab), -1)
    cut = torch.rand(n, kk, 1, generator=g, device="cuda", dtype=torch.float64)
    drafts = (torch.cumsum(q.double(), -1) > cut).to(torch.uint8).argmax(-1).to(torch.int32)
    u = torch.rand(n, kk + 1, generator=g, device="cuda", dtype=torch.float32)
    return dict(p=p, q=q, drafts=drafts, u=u, g=g)


def _quantise(x):
    """8-bit values and scale of every row (last axis): the integer nearest to
    127 x / max|x| -- in 64 bits, since 32 misplace values next to a border."""
    a = x.abs().amax(-1, keepdim=True)
    scale = a / 127.0
    ad = torch.where(a > 0, a, torch.ones_like(a)).double()
    return torch.round(x.double() * 127.0 / ad).to(torch.int8), scale.squeeze(-1)


def _tables(g, lengths):
    """A page table per sequence over a pool whose pages are in no order."""
    pages = [(n + PAGE - 1) // PAGE for n in lengths]
    width = max(1, max(pages))
    order = torch.randperm(max(1, sum(pages)), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), width, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    return table, max(1, sum(pages))


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def prepare(case, seed):
    x = _inputs(case, seed)
    g = x.pop("g")
    s = dict(case=case, **x)
    if case["kind"] in ("write", "read"):
        counts, kvh, d = _counts(case), case["kv_heads"], case["dim"]
        n = sum(counts)
        s["kout"] = torch.empty(n, kvh, d, device="cuda")
        s["vout"] = torch.empty(n, kvh, d, device="cuda")
        if own:
            from eosllm_b200 import backend as B
            s["B"] = B
            table, n_pages = _tables(g, [case["pos"] + c for c in counts])
            s["table"], s["row0"], s["pos"] = table, _int(_starts(counts)), _int([case["pos"]] * len(counts))
            s["pages"] = torch.zeros(n_pages * B.kv_q8_page_bytes(kvh, d), dtype=torch.uint8, device="cuda")
            s["pool"] = B.kv_q8_pool(s["pages"], n_pages, kvh, d)
            if case["kind"] == "read":
                B.kv_q8_write_dev(s["pool"], s["k"], s["v"], kvh * d, n, s["row0"], table, table.shape[1], s["pos"],
                                  len(counts), stream=torch.cuda.current_stream().cuda_stream)
        elif case["kind"] == "read":
            (s["kq"], s["ksc"]), (s["vq"], s["vsc"]) = _quantise(s["k"]), _quantise(s["v"])
        if case["kind"] == "read":
            del s["k"], s["v"]
        return s
    if case["kind"] == "attn":
        counts, lens, kvh, d = _counts(case), _own_lengths(case), case["kv_heads"], case["dim"]
        s["scale"] = 1.0 / math.sqrt(d)
        s["out"] = torch.empty_like(s["q"])
        if own:
            from eosllm_b200 import backend as B
            s["B"] = B
            stream = torch.cuda.current_stream().cuda_stream
            table, n_pages = _tables(g, [case["prefix"]] + lens)
            s["pages"] = torch.zeros(n_pages * B.kv_q8_page_bytes(kvh, d), dtype=torch.uint8, device="cuda")
            s["pool"] = B.kv_q8_pool(s["pages"], n_pages, kvh, d)
            s["table"] = table[1:].contiguous()
            s["prefix_table"], s["prefix_len"] = table[0].contiguous(), _int([case["prefix"]])
            s["row0"], s["lens"] = _int(_starts(counts)), _int(lens)
            zero = _int([0] * len(lens))
            if case["prefix"]:
                B.kv_q8_write_dev(s["pool"], s["kp"], s["vp"], kvh * d, case["prefix"], _int([0, case["prefix"]]),
                                  s["prefix_table"], table.shape[1], zero, 1, stream=stream)
            B.kv_q8_write_dev(s["pool"], s["ks"], s["vs"], kvh * d, sum(lens), _int(_starts(lens)), s["table"],
                              table.shape[1], zero, len(lens), stream=stream)
            s["batch"] = B.attn_batch(prefix_table=s["prefix_table"], prefix_len=s["prefix_len"],
                                      max_prefix=case["prefix"], table=s["table"], table_stride=table.shape[1],
                                      seq_len=s["lens"], max_len=max(lens), row0=s["row0"], n_seq=len(lens),
                                      n_rows=sum(counts), max_rows=max(counts))
            n = B.kv_q8_attn_scratch_bytes(s["pool"], s["batch"], case["heads"])
            s["scratch"] = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
        else:
            for name in ("kp", "vp"):
                s[name + "_q"], s[name + "_s"] = _quantise(s[name]) if case["prefix"] else (None, None)
            # every sequence's own rows side by side, padded to the longest
            own_max, starts = max(lens), _starts(lens)
            index = torch.zeros(len(lens), own_max, dtype=torch.int64, device="cuda")
            for i, n in enumerate(lens):
                index[i, :n] = torch.arange(starts[i], starts[i + 1], device="cuda")
            for name in ("ks", "vs"):
                qv, sc = _quantise(s[name])
                s[name + "_q"], s[name + "_s"] = qv[index], sc[index]
            r0, rmax = _starts(counts), max(counts)
            pick = torch.zeros(len(counts), rmax, dtype=torch.int64, device="cuda")
            back = torch.zeros(sum(counts), dtype=torch.int64, device="cuda")
            seen = torch.zeros(len(counts), rmax, dtype=torch.int64, device="cuda")
            for i, c in enumerate(counts):
                pick[i, :c] = torch.arange(r0[i], r0[i + 1], device="cuda")
                back[r0[i]:r0[i + 1]] = i * rmax + torch.arange(c, device="cuda")
                seen[i, :c] = lens[i] - c + 1 + torch.arange(c, device="cuda")
            s["pick"], s["back"], s["seen"] = pick, back, seen
        for name in ("kp", "vp", "ks", "vs"):
            del s[name]
        return s
    n, kk = case["seqs"], case["drafts"]
    s["n_draft"] = _int(_draft_counts(case))
    s["tokens"] = torch.empty(n, kk + 1, dtype=torch.int32, device="cuda")
    s["count"] = torch.empty(n, dtype=torch.int32, device="cuda")
    if own:
        from eosllm_b200 import backend as B
        s["B"] = B
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    c, B = s["case"], s["B"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] in ("write", "read"):
        n, kvh, d, n_seq = s["kout"].shape[0], c["kv_heads"], c["dim"], c["seqs"]
        if c["kind"] == "write":
            B.kv_q8_write_dev(s["pool"], s["k"], s["v"], (c["heads"] + 2 * kvh) * d, n, s["row0"], s["table"],
                              s["table"].shape[1], s["pos"], n_seq, stream=stream)
        B.kv_q8_read_dev(s["pool"], s["kout"], s["vout"], kvh * d, n, s["row0"], s["table"], s["table"].shape[1],
                         s["pos"], n_seq, stream=stream)
        return s["kout"], s["vout"]
    if c["kind"] == "attn":
        hd = c["heads"] * c["dim"]
        B.kv_q8_attn_dev(s["pool"], s["batch"], s["q"], hd, s["out"], hd, c["heads"], s["scale"], s["scratch"],
                         s["scratch"].numel(), stream=stream)
        return s["out"]
    B.verify_draft_dev(s["p"], s["q"], c["vocab"], s["drafts"], s["n_draft"], c["drafts"], s["u"], c["seqs"],
                       c["vocab"], s["tokens"], s["count"], stream=stream)
    return s["tokens"], s["count"]


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "write":
        n, kvh, d = s["kout"].shape
        out = []
        for x in (s["k"], s["v"]):
            q, sc = _quantise(x.reshape(n, kvh, d))
            out.append(q.float() * sc[..., None])
        return tuple(out)
    if c["kind"] == "read":
        return s["kq"].float() * s["ksc"][..., None], s["vq"].float() * s["vsc"][..., None]
    return _plain_attention(s) if c["kind"] == "attn" else _plain_verify(s)


def _plain_attention(s):
    c = s["case"]
    kvh, d, group = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    n = s["q"].shape[0]
    b, rmax = s["pick"].shape
    q = s["q"].view(n, kvh, group, d) * s["scale"]
    # each sequence's rows against its own keys
    k = s["ks_q"].float() * s["ks_s"][..., None]                          # [b, len, kvh, d]
    v = s["vs_q"].float() * s["vs_s"][..., None]
    qs = q[s["pick"]].permute(0, 2, 1, 3, 4).reshape(b, kvh, rmax * group, d)
    own_s = torch.matmul(qs, k.permute(0, 2, 3, 1)).view(b, kvh, rmax, group, -1)
    hidden = torch.arange(own_s.shape[-1], device="cuda") >= s["seen"][..., None]      # [b, rmax, len]
    own_s = own_s.masked_fill(hidden[:, None, :, None], -math.inf)
    top = own_s.amax(-1)                                                  # [b, kvh, rmax, group]
    if c["prefix"]:
        # every row against the shared keys
        kp = s["kp_q"].float() * s["kp_s"][..., None]
        vp = s["vp_q"].float() * s["vp_s"][..., None]
        pre_s = torch.matmul(q.permute(1, 0, 2, 3).reshape(kvh, n * group, d), kp.permute(1, 2, 0))
        flat = pre_s.amax(-1).view(kvh, n, group)
        top = torch.maximum(top, flat[:, s["pick"]].permute(1, 0, 2, 3))
    e = torch.exp(own_s - top[..., None])
    total = e.sum(-1)
    o = torch.matmul(e.view(b, kvh, rmax * group, -1), v.permute(0, 2, 1, 3)).view(b, kvh, rmax, group, d)
    total = total.permute(0, 2, 1, 3).reshape(b * rmax, kvh, group)[s["back"]]
    o = o.permute(0, 2, 1, 3, 4).reshape(b * rmax, kvh, group, d)[s["back"]]
    if c["prefix"]:
        row_top = top.permute(0, 2, 1, 3).reshape(b * rmax, kvh, group)[s["back"]].permute(1, 0, 2)
        e = torch.exp(pre_s - row_top.reshape(kvh, n * group, 1))
        total = total + e.sum(-1).view(kvh, n, group).permute(1, 0, 2)
        o = o + torch.matmul(e, vp.permute(1, 0, 2)).view(kvh, n, group, d).permute(1, 0, 2, 3)
    return (o / total[..., None]).view(n, c["heads"], d)


def _plain_verify(s):
    p, q, x, u, k = s["p"], s["q"], s["drafts"].long(), s["u"], s["n_draft"].long()
    n, kk = x.shape
    slots = torch.arange(kk, device="cuda")
    px = torch.gather(p[:, :kk], 2, x[..., None]).squeeze(-1).double()
    qx = torch.gather(q, 2, x[..., None]).squeeze(-1).double()
    good = (u[:, :kk].double() * qx < px) & (slots < k[:, None])
    taken = good.long().cumprod(1).sum(1)
    rows = torch.arange(n, device="cuda")
    target = p[rows, taken].double()
    w = target
    if kk:
        left = (target - q[rows, taken.clamp(max=kk - 1)].double()).clamp(min=0)
        use = (taken < k) & (left.sum(-1) > 0)
        w = torch.where(use[:, None], left, target)
    run_sum = torch.cumsum(w, -1)
    cut = u[:, kk].double() * run_sum[:, -1]
    token = (run_sum > cut[:, None]).to(torch.uint8).argmax(-1).int()
    out = torch.full((n, kk + 1), NO_TOKEN, dtype=torch.int32, device="cuda")
    if kk:
        out[:, :kk] = torch.where(slots < taken[:, None], s["drafts"], out[:, :kk])
    out[rows, taken] = token
    return out, (taken + 1).int()


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _stored(x):
    """What the cache holds for rows x: whole numbers times the 32-bit scale."""
    top = x.abs().max(dim=-1, keepdim=True).values
    step = (top / 127.0).double()
    ratio = (127.0 * x.double()) / top.double().clamp_min(1e-300)
    return ratio.round() * step


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] in ("write", "read"):
        n, kvh, d = sum(_counts(case)), case["kv_heads"], case["dim"]
        return tuple(_stored(x[name].reshape(n, kvh, d)) for name in ("k", "v"))
    if case["kind"] == "attn":
        counts, lens, d = _counts(case), _own_lengths(case), case["dim"]
        group = case["heads"] // case["kv_heads"]
        q = x["q"].double()
        out = torch.zeros_like(q)
        r0, l0 = _starts(counts), _starts(lens)
        seq_k = [_stored(x["ks"][l0[i]:l0[i + 1]]) for i in range(len(lens))]
        seq_v = [_stored(x["vs"][l0[i]:l0[i + 1]]) for i in range(len(lens))]
        for j in range(case["kv_heads"]):
            kp = _stored(x["kp"][:, j]) if case["prefix"] else None
            vp = _stored(x["vp"][:, j]) if case["prefix"] else None
            for i, c in enumerate(counts):
                qi = q[r0[i]:r0[i + 1], j * group:(j + 1) * group].reshape(c * group, d)
                z = qi @ seq_k[i][:, j].T
                at = torch.arange(c, device="cuda").repeat_interleave(group)
                z[torch.arange(lens[i], device="cuda")[None] > (lens[i] - c + at)[:, None]] = -math.inf
                values = seq_v[i][:, j]
                if kp is not None:
                    z, values = torch.cat([qi @ kp.T, z], 1), torch.cat([vp, values], 0)
                prob = torch.softmax(z / math.sqrt(d), dim=1)
                out[r0[i]:r0[i + 1], j * group:(j + 1) * group] = (prob @ values).view(c, group, d)
        return out
    p, q, drafts, u = (x[name].cpu().double() for name in ("p", "q", "drafts", "u"))
    n, kk = drafts.shape
    tokens = torch.full((n, kk + 1), NO_TOKEN, dtype=torch.int32)
    count = torch.zeros(n, dtype=torch.int32)
    for i, k in enumerate(_draft_counts(case)):
        a = 0
        while a < k:
            t = int(drafts[i, a])
            if not u[i, a] * q[i, a, t] < p[i, a, t]:
                break
            tokens[i, a] = t
            a += 1
        w = p[i, a]
        if a < k:
            rest = torch.relu(p[i, a] - q[i, a])
            w = rest if rest.sum() > 0 else w
        sums = w.cumsum(0)
        tokens[i, a] = int(torch.searchsorted(sums, u[i, kk] * sums[-1], right=True).clamp(max=w.numel() - 1))
        count[i] = a + 1
    return tokens.cuda(), count.cuda()
