"""Attention with modified scores and masks (ops.attn_mod_fwd / attn_mod_bwd) against the formula in
64 bits, and its refusals (CPU)."""

import math

import pytest
import torch

from hack_fe30cb28_opus_5_5_ultracode_b200 import ops


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


LENGTHS = [[1], [0, 3, 0], [127, 129, 1], [300, 257, 33, 0, 700], [1030]]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
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
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
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
