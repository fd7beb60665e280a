"""Attention with modified scores and masks (ops.attn_mod_fwd / attn_mod_bwd) against the formula in
64 bits, and its refusals (CPU)."""

import math

import pytest
import torch

from hack_fe30cb28_opus_5_5_ultracode_b200 import _lib, ops


def allowed_keys(length, causal=True, window=0, prefix=0, ids=None):
    """bool [length, length]: which key each query sees."""
    i = torch.arange(length)[:, None]
    j = torch.arange(length)[None, :]
    ok = torch.ones(length, length, dtype=torch.bool)
    if causal:
        ok &= (j <= i) | (j < prefix)
    if window:
        ok &= (i - j).abs() < window
    if ids is not None:
        run = torch.cat([torch.zeros(1, dtype=torch.long),
                         (ids[1:] != ids[:-1]).long().cumsum(0)]) if length else ids.long()
        ok &= (run[:, None] == run[None, :]) & (ids >= 0)[:, None]
    return ok


def formula(q, k, v, lengths, scale, dout=None, causal=True, softcap=0.0, slopes=None, window=0,
            doc_ids=None, prefix_len=None):
    """(out, lse[, dq, dk, dv]) in 64 bits on the CPU, by the formula."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    n, HQ, D = q.shape
    group = HQ // k.shape[1]
    out, lse = torch.zeros_like(q), torch.full((HQ, n), -math.inf, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    t0 = 0
    for b, length in enumerate(lengths):
        t1 = t0 + length
        ids = doc_ids[t0:t1].cpu() if doc_ids is not None else None
        pre = int(prefix_len[b]) if prefix_len is not None else 0
        ok = allowed_keys(length, causal, window, pre, ids)
        away = (torch.arange(length)[:, None] - torch.arange(length)[None, :]).abs()
        for h in range(HQ):
            g = h // group
            x = q[t0:t1, h] @ k[t0:t1, g].t() * scale
            bend = torch.ones_like(x)
            if softcap:
                bend = 1 - torch.tanh(x / softcap) ** 2
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * away
            x = x.masked_fill(~ok, -math.inf)
            norm = torch.logsumexp(x, -1)
            p = torch.where(ok, torch.exp(x - norm[:, None]), 0.0)
            vv = torch.where(ok.any(0)[:, None], v[t0:t1, g], 0.0)
            out[t0:t1, h], lse[h, t0:t1] = p @ vv, norm
            if dout is not None:
                go = torch.where(ok.any(1)[:, None], dout[t0:t1, h].double().cpu(), 0.0)
                ds = torch.where(ok, p * (go @ vv.t() - (go * out[t0:t1, h]).sum(-1, keepdim=True)),
                                 0.0) * bend * scale
                dq[t0:t1, h] = ds @ torch.where(ok.any(0)[:, None], k[t0:t1, g], 0.0)
                dk[t0:t1, g] += ds.t() @ torch.where(ok.any(1)[:, None], q[t0:t1, h], 0.0)
                dv[t0:t1, g] += p.t() @ go
        t0 = t1
    return (out, lse) if dout is None else (out, lse, dq, dk, dv)


def rel(x, y):
    x, y = x.double().cpu(), y.double().cpu()
    return ((x - y).norm() / y.norm().clamp(min=1e-30)).item()


def batch(lengths, heads, dtype, seed=0, std=1.0, extra=0):
    HQ, HKV, D = heads
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths) + extra
    q = (torch.randn(n, HQ, D, generator=g) * std).to(dtype).cuda()
    k = (torch.randn(n, HKV, D, generator=g) * std).to(dtype).cuda()
    v = torch.randn(n, HKV, D, generator=g).to(dtype).cuda()
    dout = torch.randn(n, HQ, D, generator=g).to(dtype).cuda()
    cu = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    return q, k, v, dout, cu


def documents(lengths, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    ids = []
    for length in lengths:
        row, at = [], 0
        while len(row) < length:
            row += [at if torch.rand(1, generator=g) < 0.8 else -1] * \
                int(torch.randint(1, max(2, length // 2 + 1), (1,), generator=g))
            at += 1
        ids += row[:length]
    return torch.tensor(ids + [0] * extra, dtype=torch.int32)


# One 16-bit rounding of P and one of the result are off by at most half a step each, u = eps / 2
# relative to each value; their 2-norms add to at most 2 u of the result's. What P's rounding
# does to a row of the output is bounded by u times sum p |v|, up to ~sqrt(keys) above the
# output's own size when p is flat and v has mean zero; errors of independent signs bring that back
# to u |p v| in the 2-norm. 3 u leaves a third for the fp32 arithmetic in between.
TOL = {torch.float16: 3 * 2.0 ** -11, torch.bfloat16: 3 * 2.0 ** -8}

MODES = [dict(), dict(causal=False), dict(window=1), dict(window=70), dict(window=300, causal=False),
         dict(softcap=20.0), dict(softcap=2.0), dict(slopes=True), dict(docs=True),
         dict(prefix=True), dict(docs=True, prefix=True, window=90, softcap=30.0, slopes=True)]


def mode_args(mode, lengths, HQ, seed=0, extra=0):
    m = dict(mode)
    if m.pop("slopes", False):
        m["slopes"] = 2.0 ** (-8.0 * torch.arange(1, HQ + 1) / HQ)
    if m.pop("docs", False):
        m["doc_ids"] = documents(lengths, seed, extra)
    if m.pop("prefix", False):
        m["prefix_len"] = torch.tensor([(7 * b + 3) * length // (9 * b + 5)
                                        for b, length in enumerate(lengths)], dtype=torch.int32)
    return m, {key: x.cuda() if torch.is_tensor(x) else x for key, x in m.items()}


LENGTHS = [[1], [0, 3, 0], [127, 129, 1], [300, 257, 33, 0, 700], [1030], [257, 130, 5] * 40]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: str(x)[:24])
@pytest.mark.parametrize("mode", MODES, ids=str)
@pytest.mark.parametrize("heads,dtype", [((4, 2, 64), torch.float16), ((7, 1, 128), torch.bfloat16)],
                         ids=["h4-2-64-fp16", "h7-1-128-bf16"])
def test_forward_matches_the_formula(lengths, mode, heads, dtype):
    q, k, v, _, cu = batch(lengths, heads, dtype)
    scale = heads[2] ** -0.5
    host, dev = mode_args(mode, lengths, heads[0])
    out, lse = ops.attn_mod_fwd(q, k, v, cu, max(lengths), scale, **dev)
    want_out, want_lse = formula(q, k, v, lengths, scale, **host)
    assert ops.device_status() == 0
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse.cpu()), empty)
    assert not out.cpu()[empty.t()].any()
    assert rel(out, want_out) < TOL[dtype]
    # lse in fp32: scores of a few units, rounded and exponentiated to ~1e-6 relative
    assert (lse.cpu().double()[~empty] - want_lse[~empty]).abs().max().item() < 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: str(x)[:24])
@pytest.mark.parametrize("mode", MODES, ids=str)
@pytest.mark.parametrize("heads,dtype", [((4, 2, 64), torch.bfloat16), ((6, 1, 128), torch.float16)],
                         ids=["h4-2-64-bf16", "h6-1-128-fp16"])
def test_backward_matches_the_formula(lengths, mode, heads, dtype):
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=1)
    scale = heads[2] ** -0.5
    host, dev = mode_args(mode, lengths, heads[0])
    out, lse = ops.attn_mod_fwd(q, k, v, cu, max(lengths), scale, **dev)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, max(lengths), scale, **dev)
    want = formula(q, k, v, lengths, scale, dout=dout, **host)[2:]
    assert ops.device_status() == 0
    for name, x, y in zip(("dq", "dk", "dv"), got, want):
        assert x.dtype == dtype and torch.isfinite(x).all(), name
        # a row whose probabilities are all 0 or 1 has a zero gradient in the formula, here at most
        # the rounding of out inside dout . out: 2^-8 or 2^-11 of |dout| |out| ~ D
        floor = TOL[dtype] * 0.02 * y.numel() ** 0.5
        assert (x.double().cpu() - y).norm().item() < TOL[dtype] * y.norm().item() + floor, name


ALL = dict(docs=True, prefix=True, window=90, softcap=30.0, slopes=True)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4, 4, 64), (2, 1, 128)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_slices_of_a_fused_row_with_nan_in_the_padding(heads, dtype):
    """q, k and v as slices of one buffer; padding tokens and rows behind the last sequence hold NaN and
    infinities, which reach nothing, and the outputs' rows behind the last sequence stay."""
    HQ, HKV, D = heads
    lengths, extra = [200, 0, 333], 61
    n = sum(lengths) + extra
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=2, extra=extra)
    host, dev = mode_args(ALL, lengths, HQ, seed=3, extra=extra)
    for a, b in ((0, 3), (120, 140), (195, 230), (400, 401)):
        host["doc_ids"][a:b] = -1
    dev["doc_ids"].copy_(host["doc_ids"])
    bad = (host["doc_ids"] < 0).cuda()
    bad[n - extra:] = True
    fused = torch.cat([t.flatten(1) for t in (q, k, v)], 1)
    fused[bad] = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype).cuda()[
        torch.arange(int(bad.sum())).cuda() % 3][:, None]
    dout[bad] = math.nan
    s = [fused[:, a:b].unflatten(1, (-1, D)) for a, b in
         ((0, HQ * D), (HQ * D, (HQ + HKV) * D), ((HQ + HKV) * D, (HQ + 2 * HKV) * D))]
    mark = 7.0
    out, lse = torch.full_like(q, mark), torch.full((HQ, n), mark, device="cuda")
    grads = [torch.full_like(t, mark) for t in (q, k, v)]
    ops.attn_mod_fwd(*s, cu, 333, D ** -0.5, out=out, lse=lse, **dev)
    ops.attn_mod_bwd(dout, *s, out, lse, cu, 333, D ** -0.5, dq=grads[0], dk=grads[1], dv=grads[2],
                     **dev)
    assert ops.device_status() == 0
    want = formula(q, k, v, lengths, D ** -0.5,
                   dout=torch.where(bad[:, None, None], 0, dout), **host)
    for x in (out, *grads):
        assert (x[n - extra:] == mark).all()
    assert (lse[:, n - extra:] == mark).all()
    assert not any(x[bad][:-extra].any() for x in (out, *grads))
    assert torch.isneginf(lse[:, bad][:, :-extra]).all()
    for x, y in zip((out, *grads), (want[0], *want[2:])):
        x, y = x.double().cpu()[:n - extra], y[:n - extra]
        floor = TOL[dtype] * 0.02 * y.numel() ** 0.5  # see test_backward_matches_the_formula
        assert (x - y).norm().item() < TOL[dtype] * y.norm().item() + floor


@pytest.mark.gpu
def test_repeats_other_streams_replays_and_two_graphs_agree_to_the_bit():
    lengths, heads, scale = [700, 1, 450], (6, 2, 64), 0.125
    q, k, v, dout, cu = batch(lengths, heads, torch.bfloat16, seed=4)
    _, dev = mode_args(ALL, lengths, heads[0])

    def run():
        out, lse = ops.attn_mod_fwd(q, k, v, cu, 700, scale, **dev)
        return (out, lse, *ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 700, scale, **dev))

    first = run()
    same = lambda got: all(torch.equal(a, b) for a, b in zip(first, got))  # noqa: E731
    assert same(run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    with torch.cuda.stream(side):
        assert same(run())
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                results.append(run())
    both = [torch.cuda.Stream(), torch.cuda.Stream()]
    for t in (t for r in results for t in r):
        t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(both, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(same(r) for r in results)
    # new contents in the captured tensors are read anew
    q.copy_(q.flip(0))
    graphs[0].replay()
    again = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, results[0])) and not same(again)


@pytest.mark.gpu
@pytest.mark.parametrize("max_len", [130, 131, 200, 277])
def test_max_len_may_be_longer_than_the_sequences(max_len):
    lengths, heads = [130, 17, 130], (4, 1, 64)
    q, k, v, dout, cu = batch(lengths, heads, torch.float16, seed=5)
    want = formula(q, k, v, lengths, 0.125, dout=dout)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, max_len, 0.125)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, max_len, 0.125)
    for x, y in zip((out, *got), (want[0], *want[2:])):
        assert rel(x, y) < 1.5 * TOL[torch.float16]


@pytest.mark.gpu
def test_a_window_beyond_every_length_is_none():
    q, k, v, dout, cu = batch([300, 5], (2, 2, 128), torch.bfloat16, seed=6)
    for causal in (True, False):
        want = ops.attn_mod_fwd(q, k, v, cu, 300, 0.1, causal=causal)
        for window in (300, ops.INT_MAX, 1 << 40):
            got = ops.attn_mod_fwd(q, k, v, cu, 300, 0.1, causal=causal, window=window)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            g = ops.attn_mod_bwd(dout, q, k, v, *got, cu, 300, 0.1, causal=causal, window=window)
            assert torch.isfinite(torch.cat([x.flatten() for x in g])).all()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(), dict(softcap=40.0), dict(slopes="negative")], ids=str)
@pytest.mark.parametrize("dtype,std", [(torch.bfloat16, 6.0), (torch.float16, 0.05)], ids=str)
def test_scores_of_hundreds_and_of_nearly_nothing(mode, dtype, std):
    """std 6: scores up to ~150, rows that one key takes almost whole; a distance bias that grows with
    the distance (negative slopes)."""
    lengths, heads = [290, 129], (4, 2, 64)
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=7, std=std)
    mode = dict(mode)
    if mode.get("slopes") == "negative":
        mode["slopes"] = -torch.tensor([0.5, 0.25, 0.01, 0.002])
    dev = {a: b.cuda() if torch.is_tensor(b) else b for a, b in mode.items()}
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 290, 0.125, **dev)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 290, 0.125, **dev)
    want = formula(q, k, v, lengths, 0.125, dout=dout, **mode)
    assert rel(out, want[0]) < TOL[dtype]
    # fp32 sums of 64 products |q k| of up to ~70, off by at most 64 x 2^-24 x their sum (~360)
    assert (lse.double().cpu() - want[1]).abs().max().item() < 64 * 2.0 ** -24 * 360
    for x, y in zip(got, want[2:]):
        floor = TOL[dtype] * 0.02 * max(std, 1) * y.numel() ** 0.5
        assert (x.double().cpu() - y).norm().item() < TOL[dtype] * y.norm().item() + floor


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(), dict(window=5000, softcap=30.0), dict(slopes=True)], ids=str)
def test_long_rows(mode):
    """33,001 tokens, rows of the result checked in 64 bits: one key's score is 10 above the rest, whose
    probabilities near 2^-15 together weigh as much as it."""
    n, heads, dtype = 33001, (2, 1, 64), torch.float16
    q, k, v, dout, cu = batch([n], heads, dtype, seed=8, std=0.5)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[3, 0, 0] = 20.0   # 4 x 20 x 0.125 = 10 above
    host, dev = mode_args(mode, [n], 2)
    rows = torch.tensor([0, 1, 127, 128, 4095, 20000, 32895, 32896, 33000])
    out, lse = ops.attn_mod_fwd(q, k, v, cu, n, 0.125, **dev)
    grads = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, n, 0.125, **dev)
    assert ops.device_status() == 0
    kk, vv = k[:, 0].double().cpu(), v[:, 0].double().cpu()
    want, want_dq = torch.zeros(len(rows), 2, 64).double(), torch.zeros(len(rows), 2, 64).double()
    for h in range(2):
        x = q[rows, h].double().cpu() @ kk.t() * 0.125
        bend = torch.ones_like(x)
        if "softcap" in mode:
            bend = 1 - torch.tanh(x / 30) ** 2
            x = 30 * torch.tanh(x / 30)
        away = rows[:, None] - torch.arange(n)[None]
        if "slopes" in mode:
            x = x - float(host["slopes"][h]) * away.abs()
        ok = (away >= 0) & (away < mode.get("window", n))
        p = torch.softmax(x.masked_fill(~ok, -math.inf), -1)
        want[:, h] = p @ vv
        go = dout[rows, h].double().cpu()
        ds = p * (go @ vv.t() - (go * want[:, h]).sum(-1, keepdim=True)) * bend * 0.125
        want_dq[:, h] = ds @ kk
    assert rel(out[rows], want) < TOL[dtype]
    # fp16 dS of 2^-15 |dP - Dvec| (|dP - Dvec| ~ 8): steps of 2^-24, off by at most 2^-13 of it more
    assert rel(grads[0][rows], want_dq) < TOL[dtype] + 2.0 ** -13
    assert all(torch.isfinite(x).all() for x in grads)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(causal=False), ALL, dict(prefix=True, softcap=3.0)], ids=str)
def test_gradients_against_differences(mode):
    """The derivative along the gradient's own direction is its norm: the formula's output moved both
    ways along it, in 64 bits (the differences' own error is 1e-6 of it)."""
    lengths, heads, dtype = [150, 61], (4, 2, 64), torch.bfloat16
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=9)
    host, dev = mode_args(mode, lengths, 4)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 150, 0.125, **dev)
    grads = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 150, 0.125, **dev)
    for at in range(3):
        step = grads[at].double().cpu()
        size = step.norm()
        step = step / size * 1e-3
        sides = []
        for sign in (1, -1):
            x = [t.double().cpu() for t in (q, k, v)]
            x[at] = x[at] + sign * step
            sides.append((formula(*x, lengths, 0.125, **host)[0] * dout.double().cpu()).sum())
        slope = (sides[0] - sides[1]) / 2e-3
        assert abs(slope - size) < TOL[dtype] * size


@pytest.mark.gpu
def test_no_tokens_and_no_sequences():
    for lengths in ([], [0, 0]):
        q, k, v, dout, cu = batch(lengths, (4, 2, 64), torch.float16)
        cu = torch.zeros(len(lengths) + 1, dtype=torch.int32, device="cuda")
        out, lse = ops.attn_mod_fwd(q, k, v, cu, 0, 0.125)
        got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 0, 0.125)
        assert [t.shape for t in got] == [q.shape, k.shape, v.shape] and lse.shape == (4, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("change", [
    dict(scale=0.0), dict(scale=math.inf), dict(scale=math.nan), dict(softcap=-1.0),
    dict(softcap=math.nan), dict(softcap=1e-6), dict(window=-1), dict(max_len=-1), dict(max_len=11),
    dict(k="heads"), dict(k="dtype"), dict(k="short"), dict(k="order"), dict(k="odd"),
    dict(v="expand"), dict(cu="long"), dict(cu="none"), dict(slopes="short"), dict(slopes="half"),
    dict(doc_ids="short"), dict(prefix_len="short"),
    dict(doc_ids="cpu"), dict(D=96), dict(dtype=torch.float32), dict(out="dtype"),
    dict(lse="shape")], ids=str)
def test_bad_arguments_are_refused(change):
    D, dtype = change.get("D", 64), change.get("dtype", torch.float16)
    q, k, v, dout, cu = batch([10], (4, 2, D), dtype)
    kw = {x: change[x] for x in ("softcap", "window") if x in change}
    kind = change.get("k")
    k = {"heads": k[:, :1].repeat(1, 3, 1), "dtype": k.bfloat16(), "short": k[:9],
         "order": k.transpose(0, 1).contiguous().transpose(0, 1),
         "odd": torch.zeros(10 * 2 * D + 1, device="cuda", dtype=dtype)[1:].view(10, 2, D)}.get(kind, k)
    if "v" in change:
        v = v[:1].expand(10, 2, D)
    cu = {"long": cu.long(), "none": cu[:0]}.get(change.get("cu"), cu)
    extra = {"slopes": {"short": torch.ones(3), "half": torch.ones(4).half()},
             "doc_ids": {"short": torch.zeros(9).int(), "cpu": torch.zeros(10).int()},
             "prefix_len": {"short": torch.zeros(2).int()}}
    for name, kinds in extra.items():
        if name in change:
            t = kinds[change[name]]
            kw[name] = t if change[name] == "cpu" else t.cuda()
    if "out" in change:
        kw["out"] = q.float()
    if "lse" in change:
        kw["lse"] = torch.zeros(10, 4, device="cuda")
    args = (cu, change.get("max_len", 10), change.get("scale", 0.125))
    with pytest.raises(ValueError):
        ops.attn_mod_fwd(q, k, v, *args, **kw)
    out, lse = kw.pop("out", q), kw.pop("lse", torch.zeros(4, 10, device="cuda"))
    with pytest.raises(ValueError):
        ops.attn_mod_bwd(dout, q, k, v, out, lse, *args, **kw)


def test_cpu_tensors_are_refused():
    q, kv = torch.zeros(4, 2, 64).half(), torch.zeros(4, 1, 64).half()
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attn_mod_fwd(q, kv, kv, cu, 4, 0.125)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attn_mod_bwd(q, q, kv, kv, q, torch.zeros(2, 4), cu, 4, 0.125)


def fake_args(**change):
    """Arguments the library checks before it launches anything (made-up, aligned addresses)."""
    f = dict(q=1 << 12, k=2 << 12, v=3 << 12, out=4 << 12, lse=5 << 12, cu_seqlens=6 << 12,
             dout=7 << 12, dq=8 << 12, dk=9 << 12, dv=10 << 12, workspace=11 << 12,
             workspace_floats=1 << 20, ldq=256, ldk=128, ldv=128, scale=0.125, softcap=0.0, n=10,
             B=1, max_len=10, HQ=4, HKV=2, D=64, dtype=0, causal=1, window=0)
    f.update(change)
    return _lib.struct("ql_attn_mod_args", **f)


@pytest.mark.parametrize("change,status", [
    (dict(D=96), 3), (dict(dtype=2), 1), (dict(n=-1), 1), (dict(max_len=11), 1), (dict(HKV=3), 1),
    (dict(HKV=0), 1), (dict(window=-1), 1), (dict(scale=0.0), 1), (dict(scale=math.nan), 1),
    (dict(softcap=-1.0), 1), (dict(softcap=1e-6), 1), (dict(q=None), 1), (dict(k=(2 << 12) + 8), 1),
    (dict(ldk=130), 1), (dict(ldk=64), 1), (dict(cu_seqlens=None), 1), (dict(lse=None), 1),
    (dict(doc_ids=1 << 16), 1), (dict(doc_ids=1 << 16, ranges=(1 << 17) + 4), 1),
    (dict(B=1 << 30), 3), (dict(n=1 << 24, max_len=1 << 24), 3), (dict(n=1 << 30), 1)], ids=str)
def test_the_library_refuses_before_any_launch(change, status):
    for entry in ("ql_attn_mod_fwd", "ql_attn_mod_bwd"):
        args = fake_args(**change)
        with pytest.raises(_lib.QLError) as e:
            _lib.call(entry, ops.ctypes_ref(args), None)
        assert e.value.status == status


@pytest.mark.parametrize("change", [dict(dout=None), dict(dk=None), dict(dv=(10 << 12) + 2),
                                    dict(workspace=None)], ids=str)
def test_the_backward_refuses_before_any_launch(change):
    args = fake_args(**change)
    with pytest.raises(_lib.QLError) as e:
        _lib.call("ql_attn_mod_bwd", ops.ctypes_ref(args), None)
    assert e.value.status == ops.STATUS_BAD_ARG


@pytest.mark.gpu
def test_prefixes_beyond_the_sequence_and_below_zero():
    lengths, heads = [140, 37, 5], (2, 1, 64)
    q, k, v, dout, cu = batch(lengths, heads, torch.float16, seed=14)
    prefix = torch.tensor([1 << 30, -(1 << 30), 5], dtype=torch.int32)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 140, 0.125, prefix_len=prefix.cuda())
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 140, 0.125, prefix_len=prefix.cuda())
    want = formula(q, k, v, lengths, 0.125, dout=dout, prefix_len=prefix)
    for x, y in zip((out, *got), (want[0], *want[2:])):
        assert rel(x, y) < 1.5 * TOL[torch.float16]


@pytest.mark.gpu
def test_tensors_beyond_32_bit_offsets():
    """The last sequence of a batch of 2.3 G elements gives what it gives alone."""
    HQ, HKV, D, length, B, dtype = 128, 2, 128, 2000, 70, torch.bfloat16
    n = length * B
    assert n * HQ * D > 1 << 31
    torch.manual_seed(15)
    q, dout = (torch.empty(n, HQ, D, device="cuda", dtype=dtype) for _ in range(2))
    k, v = (torch.randn(n, HKV, D, device="cuda").to(dtype) for _ in range(2))
    last = slice(n - length, n)
    for t in (q, dout):
        t[:-length].fill_(0.25)
        t[last] = torch.randn(length, HQ, D, device="cuda").to(dtype)
    cu = torch.arange(0, n + 1, length, device="cuda", dtype=torch.int32)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, length, 0.1, window=100)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, length, 0.1, window=100)
    s = [t[last].clone() for t in (q, k, v)]
    one_out, one_lse = ops.attn_mod_fwd(*s, cu[:2], length, 0.1, window=100)
    one = ops.attn_mod_bwd(dout[last].clone(), *s, one_out, one_lse, cu[:2], length, 0.1, window=100)
    assert ops.device_status() == 0
    for x, y in zip((out, *got), (one_out, *one)):
        assert (x[last].double() - y.double()).norm() < TOL[dtype] * y.double().norm()
    assert torch.allclose(lse[:, last], one_lse, atol=2e-5, rtol=0)


@pytest.mark.gpu
def test_a_prefix_without_causal_changes_nothing():
    q, k, v, dout, cu = batch([200, 90], (2, 1, 128), torch.bfloat16, seed=16)
    prefix = torch.tensor([50, 90], dtype=torch.int32).cuda()
    for mods in (dict(), dict(window=40)):
        a = ops.attn_mod_fwd(q, k, v, cu, 200, 0.1, causal=False, **mods)
        b = ops.attn_mod_fwd(q, k, v, cu, 200, 0.1, causal=False, prefix_len=prefix, **mods)
        g = ops.attn_mod_bwd(dout, q, k, v, *a, cu, 200, 0.1, causal=False, **mods)
        h = ops.attn_mod_bwd(dout, q, k, v, *b, cu, 200, 0.1, causal=False, prefix_len=prefix, **mods)
        assert all(torch.equal(x, y) for x, y in zip((*a, *g), (*b, *h)))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[45, 27], [5, 3, 9, 2], [1, 2, 1], [200]], ids=str)
@pytest.mark.parametrize("mode", [dict(), dict(softcap=30.0), dict(slopes=True, causal=False)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_gradients_of_few_tokens_carry_their_own_rounding_only(lengths, mode, dtype):
    """P and dS in two 16-bit parts: what stays is half a step of each result (the parts' own rest is
    below 2^-15 of it, fp32 sums likewise: a tenth of a half-step is left for them)."""
    heads, scale = (6, 2, 64), 0.125
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=17)
    host, dev = mode_args(mode, lengths, heads[0])
    out, lse = ops.attn_mod_fwd(q, k, v, cu, max(lengths), scale, **dev)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, max(lengths), scale, **dev)
    want = formula(q, k, v, lengths, scale, dout=dout, **host)[2:]
    for name, x, y in zip(("dq", "dk", "dv"), got, want):
        assert rel(x, y) < 1.1 * torch.finfo(dtype).eps / 2, name


@pytest.mark.gpu
def test_rows_of_one_key_have_no_gradient_in_q():
    q, k, v, dout, cu = batch([1, 300, 1], (4, 2, 64), torch.bfloat16, seed=18)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 300, 0.125, window=1, softcap=20.0)
    dq, dk, dv = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 300, 0.125, window=1, softcap=20.0)
    assert not dq.any() and torch.equal(out, v.repeat_interleave(2, 1))
    assert rel(dv, dout.double().cpu().unflatten(1, (2, 2)).sum(2)) < 2.0 ** -8


def own_rounding(x, y, dtype):
    """Whether x is as far from y as y's rounding to the type, and a little: the operands' second parts
    leave 2^-16 (bf16) or 2^-22 of each term, fp16 ones below 2^-14 some 2^-25 of terms near 2^-7."""
    spare = 2.0 ** -13 if dtype == torch.bfloat16 else 2.0 ** -16
    return rel(x, y) < 1.02 * rel(y.to(dtype), y) + spare


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(), dict(softcap=30.0), dict(slopes=True, causal=False)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_a_short_sequence_has_the_same_gradients_alone_and_in_a_batch(mode, dtype):
    lengths, heads, scale = [45, 700, 256, 3, 129], (6, 2, 64), 0.125
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=24)
    host, dev = mode_args(mode, lengths, heads[0])
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 700, scale, **dev)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 700, scale, **dev)
    want = formula(q, k, v, lengths, scale, dout=dout, **host)[2:]
    assert ops.device_status() == 0
    at = 0
    for length in lengths:
        s = slice(at, at + length)
        at += length
        if length > 256:
            continue
        one = [t[s].contiguous() for t in (dout, q, k, v, out)] + [lse[:, s].contiguous()]
        alone = ops.attn_mod_bwd(*one, cu.new_tensor([0, length]), length, scale, **dev)
        assert torch.equal(alone[0], got[0][s])  # dk and dv: another split of the heads may sum in another order
        for name, x, y, z in zip(("dq", "dk", "dv"), got, want, alone):
            assert own_rounding(x[s], y[s], dtype) and own_rounding(z, y[s], dtype), (name, length)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(window=4), dict(window=100, causal=False), dict(ids=True)], ids=str)
def test_short_reaches_in_long_rows_carry_their_own_rounding_only(mode):
    """Windows and documents of few keys in 2,100 tokens: as exact as a batch of few tokens."""
    n, heads, dtype = 2100, (4, 1, 128), torch.bfloat16
    q, k, v, dout, cu = batch([n], heads, dtype, seed=25)
    mode = dict(mode)
    if mode.pop("ids", False):
        mode["doc_ids"] = torch.arange(n, dtype=torch.int32) // 30
    dev = {a: b.cuda() if torch.is_tensor(b) else b for a, b in mode.items()}
    out, lse = ops.attn_mod_fwd(q, k, v, cu, n, 0.1, **dev)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, n, 0.1, **dev)
    want = formula(q, k, v, [n], 0.1, dout=dout, **mode)[2:]
    for name, x, y in zip(("dq", "dk", "dv"), got, want):
        assert own_rounding(x, y, dtype), name


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(causal=False), dict(softcap=3.0), dict(slopes=True)], ids=str)
def test_gradients_of_longer_rows_against_differences(mode):
    """test_gradients_against_differences where every tile sees more than two blocks of keys."""
    lengths, heads, dtype = [700, 390], (4, 2, 64), torch.bfloat16
    q, k, v, dout, cu = batch(lengths, heads, dtype, seed=26)
    host, dev = mode_args(mode, lengths, 4)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 700, 0.125, **dev)
    grads = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 700, 0.125, **dev)
    for at in range(3):
        step = grads[at].double().cpu()
        size = step.norm()
        step = step / size * 1e-3
        sides = []
        for sign in (1, -1):
            x = [t.double().cpu() for t in (q, k, v)]
            x[at] = x[at] + sign * step
            sides.append((formula(*x, lengths, 0.125, **host)[0] * dout.double().cpu()).sum())
        slope = (sides[0] - sides[1]) / 2e-3
        assert abs(slope - size) < TOL[dtype] * size


@pytest.mark.gpu
@pytest.mark.parametrize("slope", [-0.4375, -0.8125, -0.7071])
def test_distance_biases_of_thousands(slope):
    """Keys 16,000 tokens away carry the weight (negative slopes, a window), q = 0: row after row the same scores,
    -slope |i - j|, at other places of their blocks. A bias is off by one rounding of its own size,
    and not at all where slope / scale x distance has few bits, so that the rows' lse differ by the
    last step of their logarithm and sum at most."""
    n, window, heads, dtype = 16700, 16000, (2, 1, 64), torch.float16
    q, k, v, dout, cu = batch([n], heads, dtype, seed=27)
    q.zero_()
    dout.fill_(1.0)
    mods = dict(window=window, slopes=torch.tensor([slope, slope / 2]).cuda())
    out, lse = ops.attn_mod_fwd(q, k, v, cu, n, 0.125, **mods)
    dq, dk, dv = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, n, 0.125, **mods)
    assert ops.device_status() == 0
    away, few = torch.arange(window, dtype=torch.float64), 200  # the rest weighs less than 1e-18
    vv, most = v[:, 0].double().cpu(), 0.0
    for h, s in enumerate(mods["slopes"].double().tolist()):
        want = torch.logsumexp(-s * away, 0).item()
        most = max(most, want)
        row = lse[h, window:].double().cpu()
        # roundings of scale log2(e), slope / scale, a bias, the row's maximum and of the two steps to
        # the natural logarithm, each 2^-24 of a number no larger than lse
        assert ((row - want).abs() <= 6 * 2.0 ** -24 * want).all()
        if slope != -0.7071:
            assert (row.max() - row.min()).item() <= 2 * 2.0 ** -23 * want
        p = torch.exp(-s * away[-few:] - want).flip(0)  # of keys i - window + 1, ...
        exact = (vv.unfold(0, few, 1)[1:1 + n - window] * p).sum(-1)
        # the biases' roundings once more, P's and the result's, each of at most sum p |v|
        bound = (3 * 2.0 ** -24 * want + 3 * 2.0 ** -11) * vv.abs().max()
        assert ((out[window:, h].double().cpu() - exact).abs() <= bound).all()
    # with dout = 1 a key's dv is the sum of its probabilities, 1 a head where every row that gives it weight
    # sees a whole window; the forward's lse roundings, as many of the backward's, P's and dv's
    whole = dv[150:600].double().cpu()
    assert ((whole - 2).abs() <= 2 * (2 * 2.0 ** -11 + 12 * 2.0 ** -24 * most)).all()
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all()


def test_slopes_over_a_scale_of_nothing_are_refused():
    for entry in ("ql_attn_mod_fwd", "ql_attn_mod_bwd"):
        args = fake_args(slopes=12 << 12, scale=1e-31)
        with pytest.raises(_lib.QLError) as e:
            _lib.call(entry, ops.ctypes_ref(args), None)
        assert e.value.status == ops.STATUS_BAD_ARG


APART = {f: (i + 1) << 20 for i, f in enumerate(("q", "k", "v", "out", "lse", "cu_seqlens", "dout", "dq",
                                                 "dk", "dv", "workspace", "slopes", "prefix_len",
                                                 "doc_ids", "ranges"))}


@pytest.mark.parametrize("entry,change", [
    *(("ql_attn_mod_fwd", c) for c in (
        dict(out="q", ldq=264), dict(out="k"), dict(out="v"), dict(lse="q"), dict(out="lse"), dict(lse="cu_seqlens"),
        dict(out=APART["k"] - 16), dict(out=APART["q"] + 9 * 512 + 496), dict(ranges="v"),
        dict(ranges="doc_ids"))),
    *(("ql_attn_mod_bwd", c) for c in (
        dict(dq="dout"), dict(dk="dout"), dict(dv="out"), dict(dq="q"), dict(dk="k"), dict(dk="v"),
        dict(dq="dk"), dict(dk="dv"), dict(dv="lse"), dict(workspace="dout"), dict(workspace="dq"),
        dict(ranges="workspace"), dict(dk=APART["dq"] + 10 * 256 * 2 - 16)))], ids=str)
def test_outputs_that_share_memory_are_refused(entry, change):
    f = {**APART, **{x: APART.get(y, y) for x, y in change.items()}}
    args = fake_args(**f)
    with pytest.raises(_lib.QLError) as e:
        _lib.call(entry, ops.ctypes_ref(args), None)
    assert e.value.status == ops.STATUS_BAD_ARG


@pytest.mark.gpu
def test_shared_memory_is_refused_with_a_reason():
    q, k, v, dout, cu = batch([40, 9], (2, 2, 64), torch.float16, seed=28)
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 40, 0.125)
    place = q.clone()  # out in q's place is no harm
    got = ops.attn_mod_fwd(place, k, v, cu, 40, 0.125, out=place)
    assert got[0] is place and torch.equal(place, out) and torch.equal(got[1], lse)
    wide = torch.empty(49, 3, 64, device="cuda", dtype=q.dtype)
    for kw in (dict(out=k), dict(out=v), dict(out=wide.view(-1)[:q.numel()].view_as(q))):
        with pytest.raises(ValueError, match="share memory"):
            ops.attn_mod_fwd(wide[:, :2], k, v, cu, 40, 0.125, **kw)
    for kw in (dict(dq=dout), dict(dk=k), dict(dv=out), dict(dq=q, dk=q)):
        with pytest.raises(ValueError, match="share memory"):
            ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 40, 0.125, **kw)
    # neighbours in one buffer do not share
    want = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 40, 0.125)
    room = torch.empty(3, *q.shape, device="cuda", dtype=q.dtype)
    got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 40, 0.125, dq=room[0], dk=room[1], dv=room[2])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # nor do tensors without elements
    empty = q[:0]
    ops.attn_mod_fwd(empty, empty, empty, cu[:1], 0, 0.125, out=empty)


EXTREME = [dict(softcap=3e38), dict(scale=3e38), dict(scale=1e-30, softcap=1e10), dict(scale=2.0, softcap=2e38)]


@pytest.mark.parametrize("change", EXTREME, ids=str)
def test_scales_and_caps_beyond_fp32_are_refused_by_the_library(change):
    """softcap log2(e) and scale log2(e) have to be finite, scale / softcap a normal number."""
    for entry in ("ql_attn_mod_fwd", "ql_attn_mod_bwd"):
        args = fake_args(**change)
        with pytest.raises(_lib.QLError) as e:
            _lib.call(entry, ops.ctypes_ref(args), None)
        assert e.value.status == ops.STATUS_BAD_ARG


@pytest.mark.gpu
def test_caps_far_above_the_scores_change_nothing_and_larger_ones_are_refused():
    q, k, v, dout, cu = batch([150, 20], (2, 1, 64), torch.float16, seed=30)
    plain = ops.attn_mod_fwd(q, k, v, cu, 150, 0.125)
    for cap in (1e6, 1e20, 1e36):
        out, lse = ops.attn_mod_fwd(q, k, v, cu, 150, 0.125, softcap=cap)
        # the same scores, off by 1.2e-7 of a few units
        assert (lse - plain[1]).abs().max() < 2e-5 and rel(out, plain[0].double().cpu()) < 2.0 ** -11
        got = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, 150, 0.125, softcap=cap)
        assert all(torch.isfinite(x).all() for x in got)
    for change in EXTREME:
        scale, cap = change.get("scale", 0.125), change.get("softcap", 0.0)
        with pytest.raises(ValueError):
            ops.attn_mod_fwd(q, k, v, cu, 150, scale, softcap=cap)
        with pytest.raises(ValueError):
            ops.attn_mod_bwd(dout, q, k, v, *plain, cu, 150, scale, softcap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("cap,scale", [(30.0, 0.125), (50.0, 0.0883883), (1.5, 0.25), (1e4, 1.0)])
def test_the_cap_against_tanh_in_64_bits(cap, scale):
    """A query that sees one key has lse = cap(scale q . k). Scores of one size share a batch, so that each
    of the three forms is used over its whole range."""
    dtype = torch.float16
    for low, high in ((1e-3, 0.1), (0.1, 0.4), (0.4, 0.75), (0.75, 4.0)):  # of the tanh's argument
        n, g = 4000, torch.Generator().manual_seed(29)
        x = torch.linspace(low, high, n, dtype=torch.float64) * cap / scale
        q, k = torch.zeros(n, 1, 64), torch.zeros(n, 1, 64)
        q[:, 0, 0] = x.sqrt()
        k[:, 0, 0] = x.sqrt() * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0)
        q, k = q.to(dtype), k.to(dtype)
        cu = torch.arange(n + 1, dtype=torch.int32).cuda()
        lse = ops.attn_mod_fwd(q.cuda(), k.cuda(), k.cuda(), cu, 1, scale, softcap=cap)[1][0]
        score = q[:, 0, 0].double() * k[:, 0, 0].double() * scale
        want = cap * torch.tanh(score / cap)
        # the fits' 1.2e-7 and 0.7e-7, their evaluation, scale / cap, the two changes of the logarithm's base and the
        # constants of both: at most ten roundings of 2^-24; the 2^7 of fp16 in the row's sum: two of 2^-24 x 7
        bound = want.abs() * (1.2e-7 + 10 * 2.0 ** -24) + 14 * 2.0 ** -24
        assert ((lse.double().cpu() - want).abs() <= bound).all(), (low, high)
    assert ops.device_status() == 0
