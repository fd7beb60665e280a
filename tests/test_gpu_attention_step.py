"""The operators of a LoRA attention block with several position axes run together, as a training step
would: mrope_fwd, attn_mod_fwd, attn_mod_bwd, mrope_bwd, the LoRA gradients, clip_grads."""

import sys
import threading

import pytest
import torch

from hack_fe30cb28_opus_5_5_ultracode_b200 import ops
from tests.test_gpu_attn_mod import allowed_keys
from tests.test_gpu_mrope import angles, case, rotate

HQ, HKV, D = 6, 2, 64
SECTIONS = (8, 12, 12)
LENGTHS = [150, 1, 83]
CAP, WINDOW, SCALE, LORA = 30.0, 64, 0.125, 2.0


def in_64_bits(c, dout, ids, prefix, interleaved):
    """(out, leaf gradients in the order qkv, Bq, Bv, xq, xv) by autograd in 64 bits."""
    leaf = {x: c[x].double().requires_grad_() for x in ("qkv", "Bq", "Bv", "xq", "xv")}
    n = c["qkv"].shape[0]
    q, k, v = (t.unflatten(1, (-1, D)) for t in
               leaf["qkv"].split([HQ * D, HKV * D, HKV * D], 1))
    q = q + LORA * (leaf["xq"] @ leaf["Bq"].t()).view(n, HQ, D)
    v = v + LORA * (leaf["xv"] @ leaf["Bv"].t()).view(n, HKV, D)
    cos, sin = angles(c["cos"], c["sin"], c["pos"], SECTIONS, interleaved)
    q, k = rotate(q, cos, sin), rotate(k, cos, sin)
    outs, t0 = [], 0
    for b, length in enumerate(LENGTHS):
        at = slice(t0, t0 + length)
        ok = allowed_keys(length, True, WINDOW, int(prefix[b]), ids[at])
        kk, vv = (t[at].repeat_interleave(HQ // HKV, 1) for t in (k, v))
        x = CAP * torch.tanh(torch.einsum("ihd,jhd->hij", q[at], kk) * SCALE / CAP)
        x = x.masked_fill(~ok, -1e30)
        p = torch.softmax(x, -1) * ok
        outs.append(torch.einsum("hij,jhd->ihd", p, vv))
        t0 += length
    out = torch.cat(outs)
    (out * dout.double()).sum().backward()
    return out.detach(), [t.grad for t in leaf.values()]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_a_step_of_them_together(dtype, interleaved):
    n = sum(LENGTHS)
    c = case(n, (HQ, HKV, D), dtype, SECTIONS, seed=11)
    g = torch.Generator().manual_seed(12)
    dout = torch.randn(n, HQ, D, generator=g).to(dtype)
    ids = torch.randint(0, 9, (n,), generator=g).sort().values.int()
    ids[40:47] = -1
    prefix = torch.tensor([30, 1, 0], dtype=torch.int32)
    want_out, want = in_64_bits(c, dout, ids, prefix, interleaved)

    d = {x: t.cuda() for x, t in c.items()}
    cu = torch.tensor([0] + LENGTHS, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    rope = (d["cos"], d["sin"], d["pos"], HQ, HKV, D, SECTIONS)
    mods = dict(softcap=CAP, window=WINDOW, doc_ids=ids.cuda(), prefix_len=prefix.cuda())
    dout = dout.cuda()

    def step(max_norm=1e30):
        q, k, v = ops.mrope_fwd(d["qkv"], *rope, interleaved=interleaved, lora_scale=LORA,
                                xq=d["xq"], Bq=d["Bq"], xv=d["xv"], Bv=d["Bv"])
        out, lse = ops.attn_mod_fwd(q, k, v, cu, max(LENGTHS), SCALE, **mods)
        grads = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, max(LENGTHS), SCALE, **mods)
        dqkv, dxq, dxv = ops.mrope_bwd(*grads, *rope, interleaved=interleaved, dtype=dtype,
                                       Bq=d["Bq"], Bv=d["Bv"], lora_scale=LORA)
        dB = ops.lora_grads([(dqkv[:, :HQ * D], d["xq"], LORA, False),
                             (dqkv[:, (HQ + HKV) * D:], d["xv"], LORA, False)])
        leaves = [dqkv, *dB, dxq, dxv]
        before = [t.clone() for t in leaves]
        return out, before, ops.clip_grads(leaves, max_norm), leaves

    out, got, norm, leaves = step()
    assert ops.device_status() == 0
    # roundings to the type on the way: q, k, v, P and out, then dS, the three gradients and dqkv. Each
    # moves what follows by at most half a step, u, of its own size, and the softmax of scores of a few
    # units passes that on about as it is: 5 u forwards, 9 u in all
    u = torch.finfo(dtype).eps / 2
    rel = lambda x, y: ((x.double().cpu() - y).norm() / y.norm()).item()  # noqa: E731
    assert rel(out, want_out) < 5 * u
    for name, x, y in zip(("qkv", "Bq", "Bv", "xq", "xv"), got, want):
        assert rel(x, y) < 9 * u, name
    total = torch.stack([y.norm() for y in want]).norm()
    assert abs(norm.item() - total.item()) < 9 * u * total.item()
    assert all(torch.equal(a, b) for a, b in zip(got, leaves))  # within the norm: untouched
    _, got, norm, leaves = step(max_norm=1.0)
    for x, y in zip(leaves, got):
        # the factor in fp32, one rounding of the result
        assert rel(x, y.double().cpu() / (norm.item() + 1e-6)) < u + 2.0 ** -21 if x.dtype == dtype else \
            rel(x, y.double().cpu() / (norm.item() + 1e-6)) < 2.0 ** -21


@pytest.mark.gpu
def test_a_captured_step_follows_its_inputs():
    """The whole chain captured once and replayed on new contents, beside the same calls made eagerly."""
    dtype = torch.bfloat16
    n = sum(LENGTHS)
    d = {x: t.cuda() for x, t in case(n, (HQ, HKV, D), dtype, SECTIONS, seed=13).items()}
    cu = torch.tensor([0] + LENGTHS, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    rope = (d["cos"], d["sin"], d["pos"], HQ, HKV, D, SECTIONS)
    dout = torch.randn(n, HQ, D, device="cuda").to(dtype)

    def step():
        q, k, v = ops.mrope_fwd(d["qkv"], *rope)
        out, lse = ops.attn_mod_fwd(q, k, v, cu, max(LENGTHS), SCALE, window=50)
        grads = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, max(LENGTHS), SCALE, window=50)
        dqkv = ops.mrope_bwd(*grads, *rope, dtype=dtype)[0]
        return out, ops.clip_grads([dqkv], 0.5), dqkv

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            replayed = step()
    for _ in range(3):
        d["qkv"].copy_(torch.randn_like(d["qkv"]))
        d["pos"].copy_(torch.randint_like(d["pos"], 500))
        dout.copy_(torch.randn_like(dout))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))
    assert ops.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_a_step_of_longer_rows(dtype, monkeypatch):
    """The chain where tiles see up to six blocks of keys, so that the backward's products run in one part."""
    here = sys.modules[__name__]
    lengths = [750, 1, 290]
    monkeypatch.setattr(here, "LENGTHS", lengths)
    monkeypatch.setattr(here, "WINDOW", 600)
    n = sum(lengths)
    c = case(n, (HQ, HKV, D), dtype, SECTIONS, seed=31)
    g = torch.Generator().manual_seed(32)
    dout = torch.randn(n, HQ, D, generator=g).to(dtype)
    ids, prefix = (torch.arange(n) >= 740).int(), torch.tensor([200, 1, 0], dtype=torch.int32)
    ids[700:720] = -1
    want_out, want = in_64_bits(c, dout, ids, prefix, True)
    d = {x: t.cuda() for x, t in c.items()}
    cu = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    rope = (d["cos"], d["sin"], d["pos"], HQ, HKV, D, SECTIONS)
    mods = dict(softcap=CAP, window=600, doc_ids=ids.cuda(), prefix_len=prefix.cuda())
    q, k, v = ops.mrope_fwd(d["qkv"], *rope, interleaved=True, lora_scale=LORA, xq=d["xq"], Bq=d["Bq"],
                            xv=d["xv"], Bv=d["Bv"])
    out, lse = ops.attn_mod_fwd(q, k, v, cu, 750, SCALE, **mods)
    grads = ops.attn_mod_bwd(dout.cuda(), q, k, v, out, lse, cu, 750, SCALE, **mods)
    dqkv, dxq, dxv = ops.mrope_bwd(*grads, *rope, interleaved=True, dtype=dtype, Bq=d["Bq"], Bv=d["Bv"],
                                   lora_scale=LORA)
    dB = ops.lora_grads([(dqkv[:, :HQ * D], d["xq"], LORA, False),
                         (dqkv[:, (HQ + HKV) * D:], d["xv"], LORA, False)])
    got = [dqkv, *dB, dxq, dxv]
    norm = ops.grad_norm(got)
    assert ops.device_status() == 0
    # as many roundings as in test_a_step_of_them_together
    u = torch.finfo(dtype).eps / 2
    rel = lambda x, y: ((x.double().cpu() - y).norm() / y.norm()).item()  # noqa: E731
    assert rel(out, want_out) < 5 * u
    for name, x, y in zip(("qkv", "Bq", "Bv", "xq", "xv"), got, want):
        assert rel(x, y) < 9 * u, name
    total = torch.stack([y.norm() for y in want]).norm()
    assert abs(norm.item() - total.item()) < 9 * u * total.item()


@pytest.mark.gpu
def test_two_host_threads_at_once():
    """The same calls from two threads, each on a stream of its own, give what one gives, first calls of a
    kernel included."""
    dtype = torch.bfloat16
    n = sum(LENGTHS)
    d = {x: t.cuda() for x, t in case(n, (HQ, HKV, D), dtype, SECTIONS, seed=41).items()}
    cu = torch.tensor([0] + LENGTHS, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    rope = (d["cos"], d["sin"], d["pos"], HQ, HKV, D, SECTIONS)
    dout = torch.randn(n, HQ, D, device="cuda").to(dtype)
    slopes = torch.linspace(0.1, 0.9, HQ).cuda()
    mods = [dict(window=50), dict(softcap=20.0), dict(slopes=slopes), dict(softcap=9.0, slopes=slopes)]

    def step(mod):
        q, k, v = ops.mrope_fwd(d["qkv"], *rope)
        out, lse = ops.attn_mod_fwd(q, k, v, cu, max(LENGTHS), SCALE, **mod)
        grads = ops.attn_mod_bwd(dout, q, k, v, out, lse, cu, max(LENGTHS), SCALE, **mod)
        dqkv = ops.mrope_bwd(*grads, *rope, dtype=dtype)[0]
        return [out, lse, *grads, ops.clip_grads([dqkv], 0.5), dqkv]

    torch.cuda.synchronize()
    start, results, errors = threading.Barrier(2), [None, None], []

    def work(at):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                start.wait()
                results[at] = [step(m) for _ in range(5) for m in mods]
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    want = [step(m) for m in mods]
    for got in results:
        for i, one in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(one, want[i % len(mods)]))
    assert ops.device_status() == 0
