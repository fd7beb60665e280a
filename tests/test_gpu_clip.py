"""The global gradient norm and clipping (ops.grad_norm / clip_grads) against 64-bit sums, and their
refusals (CPU)."""

import math
import subprocess
import sys
from array import array

import pytest
import torch

from hack_fe30cb28_opus_5_5_ultracode_b200 import _lib, ops

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def grads_of(sizes, dtypes, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).to(dtypes[i % len(dtypes)]).cuda()
            for i, n in enumerate(sizes)]


def norm_of(grads):
    return math.sqrt(sum(float(g.double().pow(2).sum()) for g in grads))


def expected(grads, max_norm, inv_scale=1.0):
    norm = norm_of(grads) * inv_scale
    return norm, min(1.0, max_norm / (norm + 1e-6)) * inv_scale


def check(outs, grads, factor):
    for o, g in zip(outs, grads):
        want = g.double() * factor
        # one rounding of the result: half a step of the value, or of the smallest normal number
        # for those below it; the fp32 factor is off by two roundings
        step = want.abs().clamp(min=torch.finfo(o.dtype).tiny) * (HALF_STEP[o.dtype] + 3 * 2.0 ** -24)
        assert ((o.double() - want).abs() <= step * 1.001).all()


F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
LISTS = [([1], [F32]), ([0, 5, 0], [F16]), ([7, 8, 9, 4096, 8191, 8193, 16385, 1], [F32, BF16, F16]),
         ([24576, 24576, 4096] * 37, [F32]), ([33] * 129, [BF16]), ([3, 50000] * 700, [F32, F16]),
         ([10_000_001], [BF16]), ([3_000_000, 5], [F32])]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,dtypes", LISTS, ids=lambda x: str(x)[:30])
@pytest.mark.parametrize("max_norm,inv_scale", [(1.0, 1.0), (0.5, 2.0 ** -7), (1e9, 1.0), (1e9, 0.5)])
def test_norm_and_clip_match_64_bits(sizes, dtypes, max_norm, inv_scale):
    grads = grads_of(sizes, dtypes)
    norm, factor = expected(grads, max_norm, inv_scale)
    got = ops.grad_norm(grads, inv_scale)
    assert got.dtype == F32 and got.shape == ()
    # squares and partial sums of at most a few thousand in fp32 (independent roundings), the
    # rest in fp64, one rounding of the result
    assert abs(got.item() - norm) <= 1e-6 * norm
    outs = [torch.full_like(g, 7.0, dtype=F32) for g in grads]
    keep = [g.clone() for g in grads]
    assert torch.equal(ops.clip_grads(grads, max_norm, inv_scale, out=outs), got)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    check(outs, keep, factor)
    assert torch.equal(ops.clip_grads(grads, max_norm, inv_scale), got)
    check(grads, keep, factor)
    if factor == 1.0:
        assert all(torch.equal(a, b) for a, b in zip(grads, keep))


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_views_at_any_alignment(offset):
    for dtype in (F16, BF16, F32):
        flat = grads_of([30011], [dtype])[0]
        before = flat.clone()
        views = [flat[offset:9000 + offset], flat[9000 + offset:9001 + offset], flat[12000 + offset:]]
        norm, factor = expected([v.clone() for v in views], 1.0)
        keep = [v.clone() for v in views]
        assert abs(ops.clip_grads(views, 1.0).item() - norm) <= 1e-6 * norm
        check(views, keep, factor)
        assert torch.equal(flat[:offset], before[:offset])  # around and between the views
        assert torch.equal(flat[9001 + offset:12000 + offset], before[9001 + offset:12000 + offset])


@pytest.mark.gpu
def test_the_scale_may_live_on_the_device():
    grads = grads_of([1000, 3], [F32])
    scale = torch.tensor(2.0 ** -5, device="cuda")
    a, b = [g.clone() for g in grads], [g.clone() for g in grads]
    assert torch.equal(ops.clip_grads(a, 0.1, scale), ops.clip_grads(b, 0.1, 2.0 ** -5))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_norm_that_is_not_finite_shows(bad):
    grads = grads_of([1000, 3], [F32])
    grads[1][2] = bad
    want = [g.clone() for g in grads]
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in want]
    for p, g in zip(params, want):
        p.grad = g
    norm = torch.nn.utils.clip_grad_norm_(params, 1.0)
    got = ops.clip_grads(grads, 1.0)
    assert torch.equal(torch.isnan(got), torch.isnan(norm)) and not torch.isfinite(got)
    for a, p in zip(grads, params):
        assert torch.equal(torch.isfinite(a), torch.isfinite(p.grad))


@pytest.mark.gpu
def test_like_torch_on_an_adapter_sized_list():
    grads = grads_of([24576, 4096] * 56, [F32], std=1e-3)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    a = torch.nn.utils.clip_grad_norm_(params, 0.3)
    b = ops.clip_grads(grads, 0.3)
    assert abs(a.item() - b.item()) < 1e-6 * a.item()
    for g, p in zip(grads, params):
        assert torch.allclose(g, p.grad, rtol=1e-6, atol=0)


@pytest.mark.gpu
def test_an_empty_list_has_norm_zero():
    assert ops.clip_grads([], 1.0).item() == 0.0
    assert ops.grad_norm([]).item() == 0.0


@pytest.mark.gpu
def test_repeatable_and_capturable():
    grads = grads_of([50001, 77, 8192] * 9, [BF16, F32])
    outs = [torch.zeros_like(g) for g in grads]
    want = ops.clip_grads(grads, 1.0, out=outs)
    wanted = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            norm = ops.clip_grads(grads, 1.0, out=outs)
    for scale in (1.0, 3.0):
        for g in grads:
            g.mul_(scale)
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        if scale == 1.0:
            assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outs, wanted))
        else:
            n, f = expected(grads, 1.0)
            assert abs(norm.item() - n) < 1e-6 * n
            check(outs, grads, f)


@pytest.mark.gpu
def test_bad_lists_are_refused():
    a, b = grads_of([100, 50], [F32])
    for bad, kw in (([a, a], {}), ([a, a[10:20]], {}), ([a[::2]], {}), ([a.int()], {}),
                    ([a, b], dict(out=[a.clone()])), ([a, b], dict(out=[a.clone(), a.clone()])),
                    ([a, b], dict(out=[b.new_zeros(100), a[:50]])), ([a], dict(out=[a[:].half()[:99]])),
                    ([a], dict(inv_scale=torch.ones(2, device="cuda"))),
                    ([a], dict(inv_scale=torch.ones((), device="cuda", dtype=torch.float64)))):
        with pytest.raises(ValueError):
            ops.clip_grads(bad, 1.0, **kw)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grads([a], bad)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        ops.grad_norm([torch.ones(3)])
    with pytest.raises(ValueError, match="CUDA"):
        ops.clip_grads([torch.ones(3)], 1.0)


def lib_call(entry="ql_clip_grads", **change):
    """A call with made-up addresses, for what the library checks before it launches anything."""
    f = dict(grads=[1 << 20], outs=[2 << 20], n=[10], dtypes=[2], out_dtypes=[2], max_norm=1.0,
             norm=3 << 20, ws=4 << 20, bytes=1 << 20)
    f.update(change)
    held = [array("Q", f["grads"]), array("Q", f["outs"]), array("q", f["n"]),
            array("i", f["dtypes"]), array("i", f["out_dtypes"])]
    at = [a.buffer_info()[0] for a in held]
    tail = (1.0, None, f["norm"], f["ws"], f["bytes"], None)
    if entry == "ql_grad_norm":
        _lib.call(entry, at[0], at[2], at[3], len(held[0]), *tail)
    else:
        _lib.call(entry, *at, len(held[0]), f["max_norm"], *tail)


@pytest.mark.parametrize("change", [dict(dtypes=[3]), dict(n=[-1]), dict(grads=[0]),
                                    dict(grads=[(1 << 20) + 2]), dict(norm=0), dict(ws=0),
                                    dict(ws=(4 << 20) + 4), dict(bytes=8)], ids=str)
def test_both_entries_refuse_before_any_launch(change):
    for entry in ("ql_clip_grads", "ql_grad_norm"):
        with pytest.raises(_lib.QLError) as e:
            lib_call(entry, **change)
        assert e.value.status == ops.STATUS_BAD_ARG


TWO = dict(grads=[1 << 20, 2 << 20], outs=[1 << 20, 2 << 20], n=[100, 100], dtypes=[2, 2],
           out_dtypes=[2, 2])


@pytest.mark.parametrize("change", [
    dict(out_dtypes=[-1]), dict(outs=[0]), dict(outs=[(2 << 20) + 1]), dict(max_norm=-1.0),
    dict(max_norm=math.nan), dict(outs=[1 << 20], out_dtypes=[1]),
    {**TWO, "grads": [1 << 20, 1 << 20], "outs": [1 << 20, 1 << 20]},       # the same tensor twice
    {**TWO, "grads": [1 << 20, (1 << 20) + 396], "outs": [1 << 20, (1 << 20) + 396]},
    {**TWO, "outs": [3 << 20, 3 << 20]},                                   # one output for two
    {**TWO, "outs": [3 << 20, 1 << 20]},                                   # another's gradient
    {**TWO, "dtypes": [1, 2], "outs": [(1 << 20) + 100, 3 << 20]}], ids=str)
def test_clipping_refuses_before_any_launch(change):
    with pytest.raises(_lib.QLError) as e:
        lib_call(**change)
    assert e.value.status == ops.STATUS_BAD_ARG


@pytest.mark.gpu
def test_lists_of_thousands_and_empty_tensors():
    grads = grads_of([0, 5, 0, 129] * 700, [F32, BF16, F16])
    norm, factor = expected(grads, 0.5)
    before = [g.clone() for g in grads]
    got = ops.clip_grads(grads, 0.5)
    assert abs(got.item() - norm) < 1e-6 * norm
    check(grads, before, factor)


@pytest.mark.gpu
def test_a_tensor_beyond_32_bit_offsets():
    n = (1 << 31) + 12345
    g = torch.zeros(n, device="cuda", dtype=BF16)
    g[-1000:] = 3.0
    g[:1000] = 4.0
    norm = ops.clip_grads([g], 50.0)
    assert abs(norm.item() - 25000 ** 0.5) < 1e-3
    want = torch.tensor([4.0, 3.0]) * (50.0 / (25000 ** 0.5 + 1e-6))
    assert torch.equal(torch.stack([g[0], g[-1]]).cpu(), want.to(BF16))
    assert g[1000:-1000].abs().max().item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F32, BF16, F16]], ids=str)
@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e-15, 1e18, 1e25, 1e33])
def test_squares_outside_the_range_of_fp32(size, dtypes):
    """Gradients whose squares overflow or vanish in fp32: the norm and the clipped values stay right (the
    factor is off by a rounding of the norm, of the ratio and of the product: 2^-22)."""
    sizes = [1, 7, 2048, 4099, 40000, 8]
    grads = grads_of(sizes, [F32], seed=5)
    grads = [(g * (1.0 if dtypes[i % len(dtypes)] == F16 else size)).to(dtypes[i % len(dtypes)])
             for i, g in enumerate(grads)]
    grads.append(torch.zeros(5000, device="cuda"))
    views = [*grads, torch.cat([grads[4].float(), grads[4].float()])[3:40003]]  # one that is not aligned
    norm, factor = expected(views, size * 0.01)
    assert abs(ops.grad_norm(views).item() - norm) <= 1e-6 * norm
    outs = [torch.empty_like(g, dtype=F32) for g in views]
    assert abs(ops.clip_grads(views, size * 0.01, out=outs).item() - norm) <= 1e-6 * norm
    if 1e-20 < size < 1e20:  # else 1e-6 or a subnormal ratio decides
        for o, g in zip(outs, views):
            want = g.double() * factor
            assert ((o.double() - want).abs() <= 2.0 ** -21 * want.abs() + torch.finfo(F32).tiny).all()
    assert all(torch.isfinite(o).all() for o in outs)


@pytest.mark.gpu
def test_a_norm_beyond_fp32_is_infinite():
    g = torch.full((100,), 3e38, device="cuda")
    assert ops.grad_norm([g]).item() == math.inf
    assert ops.grad_norm([g], 0.01).item() == pytest.approx(3e37, rel=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("place", [False, True])
def test_what_an_infinite_norm_and_a_nan_do(place):
    """An infinite norm: finite gradients become 0, infinite ones NaN. A NaN: all become NaN."""
    for bad in (math.inf, -math.inf, math.nan):
        grads = grads_of([1000, 3, 50], [F32, BF16], seed=6)
        grads[1][2] = bad
        outs = None if place else [torch.full_like(g, 7.0, dtype=F32) for g in grads]
        norm = ops.clip_grads(grads, 1.0, out=outs)
        got = grads if place else outs
        if math.isnan(bad):
            assert math.isnan(norm.item()) and all(torch.isnan(o).all() for o in got)
            continue
        assert norm.item() == math.inf and math.isnan(got[1][2].item())
        got[1][2] = 0.0
        assert not any(o.any() for o in got)


def test_a_list_too_long_for_the_memory_is_an_error_not_an_abort():
    """The check for shared memory of 4 M tensors wants 128 MB; where the process may have 32 MB more, the entry
    returns a status."""
    code = """
import ctypes, resource, sys
from array import array
lib = ctypes.CDLL(sys.argv[1])
n = 1 << 22
addr, out = array("Q", range(1 << 20, (1 << 20) + 4 * n, 4)), array("Q", range(1 << 30, (1 << 30) + 4 * n, 4))
size, kind = array("q", [1]) * n, array("i", [2]) * n
at = [ctypes.c_void_p(a.buffer_info()[0]) for a in (addr, out, size, kind, kind)]
one = ctypes.c_float(1.0)
def call(count):
    return lib.ql_clip_grads(*at, count, one, one, None, ctypes.c_void_p(16), ctypes.c_void_p(16),
                             ctypes.c_int64(1 << 40), None)
out[0] = out[1]
assert call(2) == 1  # the library runs and refuses shared memory
out[0] = 1 << 30
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (32 << 20),) * 2)
sys.exit(40 + call(n))
"""
    done = subprocess.run([sys.executable, "-c", code, _lib.LIB_PATH], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 40 + 2, (done.returncode, done.stderr[-500:])  # QL_STATUS_CUDA


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("size", [1e-25, 1e-3, 1e22])
def test_few_values_among_zeros(dtype, size):
    """Sparse gradients, zeros of both signs: each value counts, whatever the loads beside it hold."""
    g = torch.Generator().manual_seed(7)
    for n, offset in ((100_003, 0), (40_000, 1), (31, 0), (9, 3)):
        flat = torch.zeros(n + offset)
        flat[::2] = -0.0
        at = torch.randint(offset, n + offset, (max(1, n // 997),), generator=g).unique()
        flat[at] = (torch.rand(len(at), generator=g) + 0.5) * size
        view = flat.to(dtype).cuda()[offset:]
        want = norm_of([view])
        assert want > 0 and abs(ops.grad_norm([view]).item() - want) <= 1e-6 * want
        assert ops.grad_norm([torch.full_like(view, -0.0)]).item() == 0.0
