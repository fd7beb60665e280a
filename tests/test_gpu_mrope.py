"""qkv + LoRA + RoPE with several position axes (ops.mrope_fwd / mrope_bwd) against the formula in 64
bits, and its refusals (CPU)."""

import time

import pytest
import torch

from hack_fe30cb28_opus_5_5_ultracode_b200 import _lib, ops


def axes_of(sections, interleaved):
    left, order = list(sections), []
    if not interleaved:
        return [x for x, c in enumerate(sections) for _ in range(c)]
    while any(left):
        for x in range(len(sections)):
            if left[x]:
                left[x] -= 1
                order.append(x)
    return order


def rotate(x, cos, sin, back=False):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    s = -sin if back else sin
    return torch.cat([a * cos - b * s, b * cos + a * s], -1)


def angles(cos, sin, pos, sections, interleaved):
    half = cos.shape[1]
    ax = torch.tensor(axes_of(sections, interleaved))
    row = pos.long()[ax].t()
    f = torch.arange(half)
    return cos.double()[row, f][:, None], sin.double()[row, f][:, None]


def case(n, heads, dtype, sections, seed=0, positions=500):
    HQ, HKV, D = heads
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = torch.outer(torch.arange(positions, dtype=torch.float64),
                    1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    return dict(qkv=r(n, (HQ + 2 * HKV) * D).to(dtype), cos=t.cos().float(), sin=t.sin().float(),
                pos=torch.randint(0, positions, (len(sections), n), generator=g).int(),
                xq=r(n, 16).to(dtype), xv=r(n, 16).to(dtype), Bq=(r(HQ * D, 16) * 0.2).to(dtype),
                Bv=(r(HKV * D, 16) * 0.2).to(dtype), dq=r(n, HQ, D), dk=r(n, HKV, D),
                dv=r(n, HKV, D))


def cuda(c):
    return {k: v.cuda() for k, v in c.items()}


# one rounding of each output to the type: at most half a step, eps / 2, of the value (plus fp32
# arithmetic, some 2^-21); in the 2-norm no more than that either
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rel(x, y):
    return ((x.double().cpu() - y).norm() / y.norm().clamp(min=1e-30)).item()


SHAPES = [((4, 2, 64), (8, 12, 12), False), ((12, 2, 128), (16, 24, 24), True),
          ((28, 4, 128), (64,), False), ((3, 3, 192), (50, 0, 16, 30), True),
          ((5, 1, 256), (1, 127), True)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7, 8, 17, 300, 5001, 19001])
@pytest.mark.parametrize("heads,sections,interleaved", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward_and_backward_match_the_formula(n, heads, sections, interleaved, dtype):
    if n > 5000 and heads[0] > 12:
        n = n // 4
    HQ, HKV, D = heads
    c, s = case(n, heads, dtype, sections), 1.75
    d = cuda(c)
    args = (d["cos"], d["sin"], d["pos"], HQ, HKV, D, sections)
    cos, sin = angles(c["cos"], c["sin"], c["pos"], sections, interleaved)
    x = c["qkv"].double().view(n, HQ + 2 * HKV, D)
    for lora in (True, False):
        kw = {k: d[k] for k in ("xq", "xv", "Bq", "Bv")} if lora else {}
        got = ops.mrope_fwd(d["qkv"], *args, interleaved=interleaved, lora_scale=s, **kw)
        q, k, v = x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]
        if lora:
            q = q + s * (c["xq"].double() @ c["Bq"].double().t()).view(n, HQ, D)
            v = v + s * (c["xv"].double() @ c["Bv"].double().t()).view(n, HKV, D)
        for a, b in zip(got, (rotate(q, cos, sin), rotate(k, cos, sin), v)):
            assert a.dtype == dtype and rel(a, b) < HALF_STEP[dtype] * 1.01 + 1e-6
        for grads in (torch.float32, dtype):
            gs = [c[k].to(grads) for k in ("dq", "dk", "dv")]
            gd = [g.cuda() for g in gs]
            kw = {k: d[k] for k in ("Bq", "Bv")} if lora else {}
            dqkv, dxq, dxv = ops.mrope_bwd(*gd, *args, interleaved=interleaved, dtype=dtype,
                                           lora_scale=s, **kw)
            gq, gk = (rotate(g.double(), cos, sin, back=True) for g in gs[:2])
            gv = gs[2].double()
            want = torch.cat([gq, gk, gv], 1).view(n, -1)
            assert dqkv.dtype == dtype and rel(dqkv, want) < HALF_STEP[dtype] * 1.01 + 1e-6
            if not lora:
                assert dxq is None and dxv is None
                continue
            # g in two 16-bit parts: what is left over is 2^-17 (bf16) of each term at most, and
            # the fp32 sums of a few thousand terms add about as little
            for a, b in ((dxq, s * gq.reshape(n, -1) @ c["Bq"].double()),
                         (dxv, s * gv.reshape(n, -1) @ c["Bv"].double())):
                assert a.dtype == torch.float32 and rel(a, b) < 2.0 ** -17 + 2e-6
    assert ops.device_status() == 0


@pytest.mark.gpu
def test_one_axis_equals_the_single_position_rope():
    heads, n = (12, 2, 128), 700
    c = cuda(case(n, heads, torch.float16, (64,)))
    a = ops.rope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"][0].contiguous(), *heads, 1.0)
    b = ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], *heads, (64,))
    for x, y in zip(a, b):  # the same fp32 formula; contraction may differ by one rounding
        assert rel(x, y.double().cpu()) < 2.0 ** -11


@pytest.mark.gpu
def test_strided_positions_and_given_outputs():
    heads, n, sections = (4, 2, 64), 90, (8, 12, 12)
    c = cuda(case(n, heads, torch.bfloat16, sections))
    wide = torch.full((3, 200), -1, device="cuda", dtype=torch.int32)
    wide[:, 10:10 + n] = c["pos"]
    out = [torch.empty(n, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2)]
    got = ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], wide[:, 10:10 + n], *heads, sections, out=out)
    want = ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], *heads, sections)
    assert all(g is o and torch.equal(g, w) for g, o, w in zip(got, out, want))


@pytest.mark.gpu
def test_positions_off_the_table_are_reported_and_read_nothing():
    heads, sections = (4, 2, 64), (8, 12, 12)
    c = cuda(case(5, heads, torch.float16, sections))
    c["pos"][1, 2], c["pos"][0, 4] = 500, -1
    ops.device_status(clear=True)
    q, _, v = ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], *heads, sections)
    assert ops.device_status(clear=True) == 1  # QL_STATUS_BAD_ARG
    ax = torch.tensor(axes_of(sections, False) * 2)
    assert not q[2, :, (ax == 1).cuda()].any() and not q[4, :, (ax == 0).cuda()].any()
    assert q[2, :, (ax == 0).cuda()].all() and torch.isfinite(v).all()


@pytest.mark.gpu
def test_no_tokens():
    c = cuda(case(0, (4, 2, 64), torch.float16, (8, 12, 12)))
    q, k, v = ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], 4, 2, 64, (8, 12, 12))
    assert q.shape == (0, 4, 64) and k.shape == v.shape == (0, 2, 64)


def test_cpu_tensors_are_refused():
    c = case(3, (4, 2, 64), torch.float16, (8, 12, 12))
    with pytest.raises(ValueError, match="CUDA"):
        ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], 4, 2, 64, (8, 12, 12))
    with pytest.raises(ValueError, match="CUDA"):
        ops.mrope_bwd(c["dq"], c["dk"], c["dv"], c["cos"], c["sin"], c["pos"], 4, 2, 64, (8, 12, 12))


@pytest.mark.gpu
@pytest.mark.parametrize("change", [dict(sections=(8, 12, 11)), dict(sections=(8, 12, 13, -1)),
                                    dict(sections=(4,) * 8), dict(pos="long"), dict(pos="short"),
                                    dict(cos="half"), dict(D=96), dict(qkv="strided"),
                                    dict(xq="alone"), dict(Bq="dtype")], ids=str)
def test_bad_arguments_are_refused(change):
    c = cuda(case(6, (4, 2, 64), torch.float16, (8, 12, 12)))
    kw = {k: c[k] for k in ("xq", "Bq")}
    sections, D = change.get("sections", (8, 12, 12)), change.get("D", 64)
    if change.get("pos") == "long":
        c["pos"] = c["pos"].long()
    if change.get("pos") == "short":
        c["pos"] = c["pos"][:, :5]
    if change.get("cos") == "half":
        c["cos"] = c["cos"].half()
    if change.get("qkv") == "strided":
        c["qkv"] = torch.cat([c["qkv"], c["qkv"]], 1)[:, ::2]
    if change.get("xq") == "alone":
        del kw["Bq"]
    if change.get("Bq") == "dtype":
        kw["Bq"] = kw["Bq"].float()
    with pytest.raises(ValueError):
        ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], 4, 2, D, sections, **kw)


def fake_args(**change):
    """Arguments the library checks before it launches anything (made-up, aligned addresses)."""
    f = dict(qkv=1 << 12, q=2 << 12, k=3 << 12, v=4 << 12, dq=5 << 12, dk=6 << 12, dv=7 << 12,
             dqkv=8 << 12, cos=9 << 12, sin=10 << 12, pos=11 << 12, ld_pos=5, lora_scale=1.0, n=5,
             HQ=4, HKV=2, D=64, dtype=0, grad_dtype=0, positions=9, axes=3, sec0=8, sec1=12,
             sec2=12, interleaved=0)
    f.update(change)
    return _lib.struct("ql_mrope_args", **f)


@pytest.mark.parametrize("change,status", [
    (dict(axes=0), 1), (dict(axes=5), 1), (dict(sec0=9), 1), (dict(sec0=-8, sec1=28), 1),
    (dict(D=32), 3), (dict(D=320), 3), (dict(dtype=2), 1), (dict(n=-1), 1), (dict(ld_pos=4), 1),
    (dict(cos=None), 1), (dict(positions=-1), 1), (dict(HKV=0), 1)], ids=str)
def test_the_library_refuses_before_any_launch(change, status):
    for entry in ("ql_mrope_fwd", "ql_mrope_bwd"):
        args = fake_args(**change)
        with pytest.raises(_lib.QLError) as e:
            _lib.call(entry, ops.ctypes_ref(args), None)
        assert e.value.status == status
    for entry, only in (("ql_mrope_fwd", dict(qkv=None)), ("ql_mrope_fwd", dict(q=8)),
                        ("ql_mrope_fwd", dict(xq=1 << 16)), ("ql_mrope_bwd", dict(dqkv=None)),
                        ("ql_mrope_bwd", dict(dxlo_q=1 << 16)), ("ql_mrope_bwd", dict(grad_dtype=1))):
        args = fake_args(**only)
        with pytest.raises(_lib.QLError) as e:
            _lib.call(entry, ops.ctypes_ref(args), None)
        assert e.value.status == 1


@pytest.mark.gpu
def test_tensors_beyond_32_bit_offsets():
    """The last rows of a batch of 2.2 G elements give what they give alone."""
    heads, sections, n, few = (64, 8, 128), (16, 24, 24), 212000, 100
    HQ, HKV, D = heads
    C = (HQ + 2 * HKV) * D
    assert n * C > 1 << 31
    c = cuda(case(few, heads, torch.bfloat16, sections))
    big = torch.zeros(n, C, device="cuda", dtype=torch.bfloat16)
    big[-few:] = c["qkv"]
    pos = torch.zeros(3, n, device="cuda", dtype=torch.int32)
    pos[:, -few:] = c["pos"]
    tables = (c["cos"], c["sin"])
    one = ops.mrope_fwd(c["qkv"], *tables, c["pos"], *heads, sections)
    many = ops.mrope_fwd(big, *tables, pos, *heads, sections)
    assert all(torch.equal(x[-few:], y) for x, y in zip(many, one))
    back = ops.mrope_bwd(*many, *tables, pos, *heads, sections, dtype=torch.bfloat16, Bq=c["Bq"])
    alone = ops.mrope_bwd(*one, *tables, c["pos"], *heads, sections, dtype=torch.bfloat16, Bq=c["Bq"])
    assert torch.equal(back[0][-few:], alone[0])
    assert rel(back[1][-few:], alone[1].double().cpu()) < 2.0 ** -20


@pytest.mark.gpu
def test_a_bad_position_leaves_the_waits_of_other_calls_alone():
    """The status word keeps the bad argument, and a wait that runs out afterwards lasts as long as its
    limit and is recorded over it; other kernels run as if nothing had been recorded."""
    heads, sections = (4, 2, 64), (8, 12, 12)
    c = cuda(case(5, heads, torch.float16, sections))
    c["pos"][1, 2] = -1
    ops.device_status(clear=True)
    ops.mrope_fwd(c["qkv"], c["cos"], c["sin"], c["pos"], *heads, sections)
    assert ops.device_status(clear=False) == ops.STATUS_BAD_ARG
    a, b = torch.randn(4096, 2048, device="cuda").half(), torch.randn(4096, 2048, device="cuda").half()
    want = a.float() @ b.float().t()
    for _ in range(5):
        assert rel(ops.gemm(a, b), want.double().cpu()) < 1e-3
    assert ops.device_status(clear=False) == ops.STATUS_BAD_ARG
    returned = torch.zeros(1, device="cuda", dtype=torch.int32)
    t0 = time.perf_counter()
    _lib.call("ql_wait_probe", int(50e6), returned.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert returned.item() == 2 and 0.04 < time.perf_counter() - t0 < 1.9
    assert ops.device_status(clear=True) == ops.STATUS_TIMEOUT


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 3e4, 1e6])
@pytest.mark.parametrize("dtype,grads", [(torch.float16, torch.float32), (torch.float16, torch.float16),
                                         (torch.bfloat16, torch.float32)], ids=str)
def test_dx_lo_is_good_to_fp32_for_gradients_of_any_size(size, dtype, grads):
    """One gradient a token, not turned (position 0), beside tokens with gradients of other sizes: dx_lo is
    the product of two numbers. The parts g is split into leave 2^-22 of it at most, their
    products with B are exact in fp32, and their sum, the CTA's and the scaling by 1.5 round
    at most five times, by up to 2^-23 each: below 2^-20 together."""
    HQ, HKV, D = heads = (4, 2, 64)
    if grads == torch.float16 and size > 3e4:
        size = 6e4
    n, sections = 40, (8, 12, 12)
    c = case(n, heads, dtype, sections, seed=21)
    c["pos"].zero_()
    g = torch.Generator().manual_seed(22)
    at = torch.randint(0, HQ * D, (n,), generator=g), torch.randint(0, HKV * D, (n,), generator=g)
    sizes = torch.where(torch.arange(n) % 3 == 0, 1.0, size)  # every third token ordinary
    dq, dv = torch.zeros(n, HQ * D), torch.zeros(n, HKV * D)
    for x, col in ((dq, at[0]), (dv, at[1])):
        x[torch.arange(n), col] = (torch.rand(n, generator=g) + 0.09) * sizes
    dq, dv = dq.to(grads), dv.to(grads)
    d = cuda(c)
    _, dxq, dxv = ops.mrope_bwd(dq.cuda().view(n, HQ, D), torch.zeros(n, HKV, D, device="cuda", dtype=grads),
                                dv.cuda().view(n, HKV, D), d["cos"], d["sin"], d["pos"], *heads, sections,
                                dtype=dtype, Bq=d["Bq"], Bv=d["Bv"], lora_scale=1.5)
    assert ops.device_status() == 0
    for got, x, B in ((dxq, dq, c["Bq"]), (dxv, dv, c["Bv"])):
        want = 1.5 * x.double() @ B.double()
        assert ((got.double().cpu() - want).abs() <= 2.0 ** -20 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [77, 5003])
@pytest.mark.parametrize("size", [1e-5, 1e-3, 1e6])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_dx_lo_of_small_and_large_gradients(size, dtype, n):
    """Dense fp32 gradients whose sizes differ from token to token. Against |g| |B| summed, an fp32 sum of
    256 terms in 16-term steps rounds some 50 times (split parts included) by at most 2^-23."""
    HQ, HKV, D = heads = (4, 2, 64)
    c, sections = case(n, heads, dtype, (8, 12, 12), seed=23), (8, 12, 12)
    by = size * 10.0 ** (torch.arange(n) % 4 - 2.0)[:, None, None]
    for x in ("dq", "dk", "dv"):
        c[x] = c[x] * by
    d = cuda(c)
    got = ops.mrope_bwd(d["dq"], d["dk"], d["dv"], d["cos"], d["sin"], d["pos"], *heads, sections, dtype=dtype,
                        Bq=d["Bq"], Bv=d["Bv"])[1:]
    cos, sin = angles(c["cos"], c["sin"], c["pos"], sections, False)
    gq, gv = rotate(c["dq"].double(), cos, sin, back=True).view(n, -1), c["dv"].double().view(n, -1)
    for a, g, B in zip(got, (gq, gv), (c["Bq"].double(), c["Bv"].double())):
        assert ((a.double().cpu() - g @ B).abs() <= 50 * 2.0 ** -23 * (g.abs() @ B.abs())).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("entry,change", [
    *(("ql_mrope_fwd", c) for c in (dict(q="qkv"), dict(k="qkv"), dict(v="q"), dict(k="v"), dict(q="xq"),
                                    dict(v="Bv"), dict(k="pos"), dict(q=(1 << 20) + 5 * 512 * 2 - 16))),
    *(("ql_mrope_bwd", c) for c in (dict(dqkv="dq"), dict(dqkv="dk"), dict(dqkv="dv"), dict(dxlo_q="dqkv"),
                                    dict(dxlo_v="Bq"), dict(dxlo_q="dxlo_v"), dict(dxlo_v="dv")))],
    ids=str)
def test_outputs_that_share_memory_are_refused(entry, change):
    names = "qkv q k v dq dk dv dqkv cos sin pos xq xv Bq Bv dxlo_q dxlo_v".split()
    apart = {x: (i + 1) << 20 for i, x in enumerate(names)}
    f = {**apart, **{x: apart.get(y, y) for x, y in change.items()}}
    args = fake_args(**f)
    with pytest.raises(_lib.QLError) as e:
        _lib.call(entry, ops.ctypes_ref(args), None)
    assert e.value.status == ops.STATUS_BAD_ARG


@pytest.mark.gpu
def test_shared_memory_is_refused_with_a_reason():
    heads, n, sections = (4, 2, 64), 30, (8, 12, 12)
    c = cuda(case(n, heads, torch.bfloat16, sections))
    tables = (c["cos"], c["sin"], c["pos"], *heads, sections)
    room = torch.empty(n * 8 * 64, device="cuda", dtype=torch.bfloat16)
    q, k, v = (t.view(n, h, 64) for t, h in zip(room.split([n * 256, n * 128, n * 128]), (4, 2, 2)))
    got = ops.mrope_fwd(c["qkv"], *tables, out=(q, k, v))  # neighbours do not share
    assert all(torch.equal(x, y) for x, y in zip(got, ops.mrope_fwd(c["qkv"], *tables)))
    for out in ((q, k, k), (q, q.view(-1)[:n * 128].view(n, 2, 64), c["qkv"].view(-1)[:n * 128].view(n, 2, 64))):
        with pytest.raises(ValueError, match="share memory"):
            ops.mrope_fwd(c["qkv"], *tables, out=out)
    with pytest.raises(ValueError, match="share memory"):
        ops.mrope_bwd(q, k, v, *tables, dtype=torch.bfloat16, out=room.view(n, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,sections", [((4, 1, 128), (24, 20, 20)), ((2, 2, 64), (14, 10, 8))], ids=str)
def test_interleaved_axes_whose_first_keeps_the_remainder(heads, sections):
    n, dtype = 333, torch.bfloat16
    HQ, HKV, D = heads
    c = case(n, heads, dtype, sections, seed=33)
    d = cuda(c)
    got = ops.mrope_fwd(d["qkv"], d["cos"], d["sin"], d["pos"], *heads, sections, interleaved=True)
    back = ops.mrope_bwd(d["dq"], d["dk"], d["dv"], d["cos"], d["sin"], d["pos"], *heads, sections, interleaved=True,
                         dtype=dtype)[0]
    # in turn while an axis has some left: 0 1 2 0 1 2 ..., the first axis alone at the end
    order = [f % 3 if f < 3 * min(sections) else None for f in range(D // 2)]
    left = [s - min(sections) for s in sections]
    rest = [a for r in range(max(left)) for a in range(3) if left[a] > r]
    ax = torch.tensor([a for a in order if a is not None] + rest)
    row, f = c["pos"].long()[ax].t(), torch.arange(D // 2)
    cos, sin = c["cos"].double()[row, f][:, None], c["sin"].double()[row, f][:, None]
    x = c["qkv"].double().view(n, HQ + 2 * HKV, D)
    for a, b in zip(got, (rotate(x[:, :HQ], cos, sin), rotate(x[:, HQ:HQ + HKV], cos, sin), x[:, HQ + HKV:])):
        assert rel(a, b) < HALF_STEP[dtype] * 1.01 + 1e-6
    want = torch.cat([rotate(c["dq"].double(), cos, sin, back=True), rotate(c["dk"].double(), cos, sin, back=True),
                      c["dv"].double()], 1).view(n, -1)
    assert rel(back, want) < HALF_STEP[dtype] * 1.01 + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 4, 60])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_dx_lo_over_many_heads(n, dtype):
    """3,584 terms a sum. A unit of 64 terms takes at most six sums on the tensor core, cut off by up to 2^-23
    each; the units' errors have independent signs, and adding them up rounds by 2^-24."""
    HQ, HKV, D = heads = (28, 4, 128)
    sections = (16, 24, 24)
    c = case(n, heads, dtype, sections, seed=34)
    d = cuda(c)
    got = ops.mrope_bwd(d["dq"], d["dk"], d["dv"], d["cos"], d["sin"], d["pos"], *heads, sections, dtype=dtype,
                        Bq=d["Bq"], Bv=d["Bv"])[1:]
    cos, sin = angles(c["cos"], c["sin"], c["pos"], sections, False)
    gq, gv = rotate(c["dq"].double(), cos, sin, back=True).view(n, -1), c["dv"].double().view(n, -1)
    for a, g, B in zip(got, (gq, gv), (c["Bq"].double(), c["Bv"].double())):
        assert rel(a, g @ B) < 8 * 2.0 ** -23
    assert ops.device_status() == 0
