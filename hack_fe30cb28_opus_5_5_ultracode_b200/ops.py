"""torch-facing wrappers of the C ABI: each takes CUDA tensors, checks layouts, and launches on
the current stream. Names follow the reference's launch wrappers (solution/engine.py:103-109,
947-1045) so the tests read like the reference's own.
"""

from array import array

import torch

from . import _lib
from ._lib import call

_DT = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
INT_MAX = 2147483647
STATUS_BAD_ARG = 1  # QL_STATUS_BAD_ARG of include/qlora_sm100.h: the library refuses the arguments
STATUS_UNSUPPORTED = 3  # QL_STATUS_UNSUPPORTED of include/qlora_sm100.h: no kernel for this request
STATUS_TIMEOUT = 4  # QL_STATUS_TIMEOUT of include/qlora_sm100.h: a kernel gave up a bounded wait


def dtype_code(dtype):
    try:
        return _DT[dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {dtype}") from None


def stream_ptr():
    """The current CUDA stream of the current device, as a raw pointer (called for every
    launch: the raw lookup skips torch.cuda.current_stream()'s Python-level device resolution)."""
    try:
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    except AttributeError:  # pragma: no cover - other torch builds
        return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("CUDA tensors required (the library has no CPU path)")


_INF = float("inf")


def _index_of(first, *others):
    """The CUDA device index the tensors (None: absent) share."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError("CUDA tensors required (the library has no CPU path)")
    for t in others:
        if t is not None and t.get_device() != dev:
            _need_cuda(t)
            raise ValueError("the tensors must be on one device")
    return dev


def _exact(t, name, shape, dtype):
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)}, got {t.dtype} "
                         f"{list(t.shape)}")


def _given(t, name, shape, dtype, dev):
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the inputs' device")
    _exact(t, name, shape, dtype)


def _address(t):
    return 0 if t is None else t.data_ptr()


class _on_device:
    """Makes a CUDA device the current one for a launch (its current stream is launched on); nothing
    to switch in the usual case."""

    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _launch(name, dev, args):
    """Calls an entry point that takes one packed argument struct, on device dev's current stream."""
    with _on_device(dev):
        status = getattr(_lib.lib(), name)(args, stream_ptr())
    if status == STATUS_BAD_ARG:  # what is not checked before the call
        raise ValueError("outputs that share memory with an input or one another, or that do not "
                         "start at a multiple of 16 bytes")
    _lib.check(name, status)


# ---------------------------------------------------------------------------------------------
# NF4
# ---------------------------------------------------------------------------------------------
def nf4_dequant(w, out=None, transpose=False, dtype=torch.float16):
    """Dequantize an NF4 weight (an object with packed, absmax, code, nested, code2, absmax2,
    offsets, bs2, seg1, seg2, shape = (rows, cols)) into out [rows, cols] (or its transpose)."""
    rows, cols = w.shape
    if out is None:
        out = torch.empty((cols, rows) if transpose else (rows, cols), device=w.packed.device,
                          dtype=dtype)
    _need_cuda(w.packed, out)
    assert out.is_contiguous()
    call("ql_nf4_dequant", _ptr(w.packed), _ptr(w.absmax), _ptr(w.code2), _ptr(w.absmax2),
         _ptr(w.offsets), _ptr(w.code), _ptr(out), rows, cols, int(w.nested), int(w.bs2),
         int(getattr(w, "seg1", INT_MAX)), int(getattr(w, "seg2", INT_MAX)),
         dtype_code(out.dtype), int(transpose), stream_ptr())
    return out


def nf4_weight_struct(w):
    """The ql_nf4_weight view of an NF4 weight object (as ops.nf4_dequant reads it)."""
    rows, cols = w.shape
    return _lib.struct("ql_nf4_weight", packed=_ptr(w.packed), absmax=_ptr(w.absmax),
                       code=_ptr(w.code), code2=_ptr(w.code2), absmax2=_ptr(w.absmax2),
                       offsets=_ptr(w.offsets), rows=rows, cols=cols,
                       seg1=int(getattr(w, "seg1", INT_MAX)), seg2=int(getattr(w, "seg2", INT_MAX)),
                       nested=int(w.nested), bs2=int(w.bs2))


def gemm_nf4(a, w, layout=0, out=None, bias=None, accumulate=False, out_dtype=None,
             residual=None):
    """out = a @ W^T (layout 0, W [N, K]) or a @ W (layout 1, W [K, N]) with the NF4 weight w
    dequantised inside the kernel (ql_gemm_nf4)."""
    M, K = a.shape
    rows, cols = w.shape
    N = rows if layout == 0 else cols
    if (cols if layout == 0 else rows) != K:
        raise ValueError(f"inner dimensions differ: {a.shape} x NF4 {w.shape} (layout {layout})")
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=out_dtype or a.dtype)
    ws = nf4_weight_struct(w)
    call("ql_gemm_nf4", _ptr(a), a.stride(0), ctypes_ref(ws), int(layout), _ptr(out),
         out.stride(0), _ptr(bias), M, dtype_code(a.dtype), dtype_code(out.dtype),
         int(accumulate), _ptr(residual), stream_ptr())
    return out


# ---------------------------------------------------------------------------------------------
# GEMM
# ---------------------------------------------------------------------------------------------
def gemm(a, b, out=None, bias=None, accumulate=False, out_dtype=None, residual=None,
         b_kn=False):
    """out[M, N] (+)= a[M, K] @ b[N, K]^T (+ bias) on tcgen05; with b_kn, b is [K, N] and
    out = a @ b (ql_gemm_nn). a and b: fp16 or bf16 with unit column stride; out: fp16 / bf16 /
    fp32 with unit column stride."""
    M, K = a.shape
    N, K2 = (b.shape[1], b.shape[0]) if b_kn else b.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {a.shape} x {b.shape}")
    if a.dtype != b.dtype:
        raise ValueError("a and b must have the same dtype")
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=out_dtype or a.dtype)
    _need_cuda(a, b, out, bias)
    if a.stride(1) != 1 or b.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("gemm needs unit column strides")
    if bias is not None and bias.dtype != a.dtype:
        raise ValueError("bias must have the input dtype")
    if residual is not None and (residual.stride(0) != out.stride(0) or residual.stride(1) != 1):
        raise ValueError("residual must share the output's row stride")
    ws = gemm_workspace(a.device, int(_lib.lib().ql_gemm_workspace_bytes(M, N, K)))
    call("ql_gemm_nn" if b_kn else "ql_gemm_tn", _ptr(a), a.stride(0), _ptr(b), b.stride(0),
         _ptr(out), out.stride(0), _ptr(bias), M, N, K, dtype_code(a.dtype),
         dtype_code(out.dtype), int(accumulate), _ptr(residual), _ptr(ws),
         0 if ws is None else ws.numel(), stream_ptr())
    return out


def gemm_set_mode(mode):
    """Tile kind of the GEMMs (mode & 3): 0 per-shape cost model, 1 single-CTA tiles, 2 2-SM
    pair tiles; + 4: one 64-wide K chunk per pipeline stage (2-D copies) instead of two."""
    call("ql_gemm_set_mode", int(mode))


def attn_set_deterministic(on):
    """The layer backward's attention gradients summed in a fixed order (bit-reproducible run to
    run) or by fp32 bulk reductions (default; ql_attn_set_deterministic)."""
    call("ql_attn_set_deterministic", 1 if on else 0)


def attn_set_impl(impl):
    """Attention kernels for D = 128: 0 default (tcgen05), 1 warp-level mma.sync, 2 tcgen05."""
    call("ql_attn_set_impl", int(impl))


_GEMM_WS = {}


def gemm_workspace(device, nbytes):
    """A zero-initialised, grow-only split-K workspace per device (its counter region is left
    zero by every GEMM, so it is reused as is)."""
    if nbytes <= 0:
        return None
    ws = _GEMM_WS.get(device)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(nbytes, device=device, dtype=torch.uint8)
        _GEMM_WS[device] = ws
    return ws


PROFILE_KINDS = ("gemm", "dequant", "rms_fwd", "rms_bwd", "rope_fwd", "rope_bwd", "attn_fwd",
                 "attn_bwd", "glu_fwd", "glu_bwd", "lora_colsum", "ce", "other")


def profile_start(capacity=200000):
    """Time every library operation with CUDA events (see ql_profile_start)."""
    call("ql_profile_start", int(capacity))


def profile_stop():
    call("ql_profile_stop")


def profile_read():
    """{kind: {"count", "ms", "flops", "bytes"}} of the operations recorded since profile_start."""
    import ctypes

    n = len(PROFILE_KINDS)
    arrs = [(ctypes.c_double * n)() for _ in range(4)]
    call("ql_profile_read", *[ctypes.addressof(a) for a in arrs])
    return {k: {"count": arrs[0][i], "ms": arrs[1][i], "flops": arrs[2][i], "bytes": arrs[3][i]}
            for i, k in enumerate(PROFILE_KINDS) if arrs[0][i]}


def set_pdl(on):
    """Programmatic dependent launch on (default) or off for this library's launches
    (ql_set_pdl)."""
    call("ql_set_pdl", 1 if on else 0)


def launch_count():
    """Kernels launched through the library so far (its own counter)."""
    return int(_lib.lib().ql_launch_count())


def device_status(clear=True):
    """The library's device status word: QL_STATUS_TIMEOUT if a kernel gave up a wait, else
    QL_STATUS_BAD_ARG if an id or position lay outside its table."""
    import ctypes

    v = ctypes.c_int(0)
    call("ql_device_status", ctypes.addressof(v), int(clear))
    return v.value


# ---------------------------------------------------------------------------------------------
# dropout / RMSNorm
# ---------------------------------------------------------------------------------------------
class Drop:
    """The LoRA dropout state of one layer's two masks (TorchDropout.draw, engine.py:787-797):
    tok = packed tokens' indices in the padded batch, seed, Philox counters of the q and v
    calls, the dropout kernel's threads, p, VEC."""

    def __init__(self, tok, seed, ctr_q, ctr_v, threads, p, vec=4, drop_q=True, drop_v=True):
        self.tok, self.seed, self.ctr_q, self.ctr_v = tok, int(seed), int(ctr_q), int(ctr_v)
        self.threads, self.p, self.vec = int(threads), float(p), int(vec)
        self.drop_q, self.drop_v = bool(drop_q), bool(drop_v)

    def fields(self):
        return dict(tok=_ptr(self.tok), seed=self.seed, ctr_q=self.ctr_q, ctr_v=self.ctr_v,
                    threads=self.threads, p_keep=1.0 - self.p, keep_scale=1.0 / (1.0 - self.p),
                    vec=self.vec, drop_q=int(self.drop_q), drop_v=int(self.drop_v))


def dropout_keep(nelem, seed, ctr, threads, p, vec=4, device="cuda"):
    out = torch.empty(nelem, device=device, dtype=torch.int8)
    call("ql_dropout_keep", _ptr(out), nelem, int(seed), int(ctr), int(threads), 1.0 - p,
         int(vec), stream_ptr())
    return out


def rms_fwd(x, w, eps, dtype=torch.float16, delta=None, write_y=True, drop=None, Aq=None,
            Av=None, want_yq=False, out_y=None, out_xsum=None, keep_bits=None):
    """(xsum, y, yq, yv, rstd, xq, xv) of reference _rms_fwd (engine.py:947-966), with the
    LoRA-A products xq / xv when Aq / Av are given. keep_bits: (keep_q, keep_v) int32
    [n, H / 32] tensors (or None) that receive the dropout masks as bits."""
    n, H = x.shape
    dev = x.device
    xsum = (out_xsum if out_xsum is not None else torch.empty_like(x)) if delta is not None else x
    y = (out_y if out_y is not None else torch.empty((n, H), device=dev, dtype=dtype)) \
        if write_y else None
    dq = drop is not None and drop.drop_q
    dv = drop is not None and drop.drop_v
    yq = torch.empty((n, H), device=dev, dtype=dtype) if dq and want_yq else None
    yv = torch.empty((n, H), device=dev, dtype=dtype) if dv and want_yq else None
    xq = torch.empty((n, 16), device=dev, dtype=dtype) if dq and Aq is not None else None
    xv = torch.empty((n, 16), device=dev, dtype=dtype) if dv and Av is not None else None
    rstd = torch.empty((n,), device=dev, dtype=torch.float32)
    fields = dict(x=_ptr(x), delta=_ptr(delta), w=_ptr(w), xsum=_ptr(xsum) if delta is not None
                  else None, y=_ptr(y), yq=_ptr(yq), yv=_ptr(yv), rstd=_ptr(rstd),
                  Aq=_ptr(Aq) if dq else None, Av=_ptr(Av) if dv else None, xq=_ptr(xq),
                  xv=_ptr(xv), n=n, H=H, rank=16, dtype=dtype_code(dtype), eps=float(eps),
                  vec=4)
    if keep_bits is not None:
        fields.update(keep_q=_ptr(keep_bits[0]), keep_v=_ptr(keep_bits[1]))
    if drop is not None:
        fields.update(drop.fields())
    args = _lib.struct("ql_rms_fwd_args", **fields)
    call("ql_rms_fwd", ctypes_ref(args), stream_ptr())
    return xsum, y, yq, yv, rstd, xq, xv


def rms_bwd(dy, x, rstd, w, dtype=torch.float16, dres=None, tq=None, tv=None, dxlo_q=None,
            dxlo_v=None, Aq=None, Av=None, drop=None, grad_scale=1.0, out=None, out16=None,
            keep_bits=None):
    """Reference _rms_bwd (engine.py:969-981); dx fp32 (and its 16-bit copy into out16).
    keep_bits: the forward's (keep_q, keep_v) mask bits, read instead of redrawing the masks."""
    n, H = x.shape
    dx = out if out is not None else torch.empty_like(x)
    fields = dict(dy=_ptr(dy), ld_dy=dy.stride(0), x=_ptr(x), rstd=_ptr(rstd), w=_ptr(w),
                  dres=_ptr(dres), dx=_ptr(dx), dx16=_ptr(out16), tq=_ptr(tq), tv=_ptr(tv),
                  dxlo_q=_ptr(dxlo_q), dxlo_v=_ptr(dxlo_v), Aq=_ptr(Aq), Av=_ptr(Av), n=n, H=H,
                  rank=16, dtype=dtype_code(dtype), grad_scale=float(grad_scale), vec=4)
    if keep_bits is not None:
        fields.update(keep_q=_ptr(keep_bits[0]), keep_v=_ptr(keep_bits[1]))
    if drop is not None:
        fields.update(drop.fields())
    args = _lib.struct("ql_rms_bwd_args", **fields)
    call("ql_rms_bwd", ctypes_ref(args), stream_ptr())
    return dx


def ctypes_ref(s):
    import ctypes

    return ctypes.addressof(s)


# ---------------------------------------------------------------------------------------------
# qkv + RoPE
# ---------------------------------------------------------------------------------------------
def rope_fwd(qkv, cos, sin, pos, HQ, HKV, D, lora_scale, lq=None, lv=None, xq=None, xv=None,
             Bq=None, Bv=None, out=None):
    n = qkv.shape[0]
    dev, dt = qkv.device, qkv.dtype
    if out is None:
        q = torch.empty((n, HQ, D), device=dev, dtype=dt)
        k = torch.empty((n, HKV, D), device=dev, dtype=dt)
        v = torch.empty((n, HKV, D), device=dev, dtype=dt)
    else:
        q, k, v = out
    args = _lib.struct("ql_rope_fwd_args", qkv=_ptr(qkv), lq=_ptr(lq), lv=_ptr(lv), xq=_ptr(xq),
                       xv=_ptr(xv), Bq=_ptr(Bq), Bv=_ptr(Bv), cos=_ptr(cos), sin=_ptr(sin),
                       pos=_ptr(pos), q=_ptr(q), k=_ptr(k), v=_ptr(v),
                       lora_scale=float(lora_scale), n=n, HQ=HQ, HKV=HKV, D=D, rank=16,
                       dtype=dtype_code(dt))
    call("ql_rope_fwd", ctypes_ref(args), stream_ptr())
    return q, k, v


def rope_bwd(dq, dk, dv, cos, sin, pos, HQ, HKV, D, dtype=torch.float16, Bq=None, Bv=None,
             lora_scale=1.0, out=None):
    """(dqkv, dxlo_q, dxlo_v): the pre-rotary qkv gradient and, with Bq / Bv, the LoRA-A
    output gradients s * (g . B) (fp32)."""
    n = dq.shape[0]
    dev = dq.device
    C = (HQ + 2 * HKV) * D
    dqkv = out if out is not None else torch.empty((n, C), device=dev, dtype=dtype)
    dxlo_q = torch.empty((n, 16), device=dev, dtype=torch.float32) if Bq is not None else None
    dxlo_v = torch.empty((n, 16), device=dev, dtype=torch.float32) if Bv is not None else None
    args = _lib.struct("ql_rope_bwd_args", dq=_ptr(dq), dk=_ptr(dk), dv=_ptr(dv), cos=_ptr(cos),
                       sin=_ptr(sin), pos=_ptr(pos), dqkv=_ptr(dqkv), Bq=_ptr(Bq), Bv=_ptr(Bv),
                       dxlo_q=_ptr(dxlo_q), dxlo_v=_ptr(dxlo_v), lora_scale=float(lora_scale),
                       n=n, HQ=HQ, HKV=HKV, D=D, kv_heads_in=dk.shape[1], rank=16,
                       dtype=dtype_code(dtype), grad_dtype=dtype_code(dq.dtype))
    call("ql_rope_bwd", ctypes_ref(args), stream_ptr())
    return dqkv, dxlo_q, dxlo_v


_MROPE = _lib.packer("ql_mrope_args", """qkv xq xv Bq Bv q k v dq dk dv dqkv dxlo_q dxlo_v cos sin
    pos ld_pos lora_scale n HQ HKV D dtype grad_dtype positions axes sec0 sec1 sec2 sec3
    interleaved""")


def _mrope_inputs(cos, sin, pos, n, HQ, HKV, D, sections, dtype):
    """The checked (pos row stride, table rows, axes, four section sizes) both directions of mrope
    share."""
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError(f"unsupported dtype {dtype}")
    if HQ <= 0 or HKV <= 0 or D <= 0 or D % 64 or D > 256:
        raise ValueError(f"heads ({HQ}, {HKV}, {D}): D must be 64, 128, 192 or 256")
    axes = len(sections)
    if not 1 <= axes <= 4 or min(sections) < 0 or sum(sections) != D // 2:
        raise ValueError(f"sections {tuple(sections)} must be 1 to 4 counts that add to {D // 2}")
    if pos.dim() != 2 or pos.shape != (axes, n) or pos.dtype is not torch.int32 \
            or (n > 1 and pos.stride(1) != 1) or (axes > 1 and pos.stride(0) < n):
        raise ValueError(f"pos must be int32 [{axes}, {n}] with unit column stride")
    rows = cos.shape[0]
    _exact(cos, "cos", (rows, D // 2), torch.float32)
    _exact(sin, "sin", (rows, D // 2), torch.float32)
    return pos.stride(0) if axes > 1 else n, rows, axes, (*sections, 0, 0, 0)[:4]


def mrope_fwd(qkv, cos, sin, pos, HQ, HKV, D, sections, interleaved=False, lora_scale=1.0, xq=None,
              xv=None, Bq=None, Bv=None, out=None):
    """(q, k, v) of rope_fwd with several position axes (ql_mrope_fwd): pos int32 [axes, n],
    sections = how many of the D / 2 frequencies each axis has, in blocks or (interleaved) dealt
    to the axes in turn while an axis has some left; cos / sin the rotary table of one axis.
    xq / Bq, xv / Bv: the LoRA-B products q += lora_scale xq Bq^T, added in fp32. A position outside the
    table turns nothing (its frequencies give 0) and is recorded for device_status(). out: (q, k, v) to
    write; they must not share memory with an input or one another."""
    dev = _index_of(qkv, cos, sin, pos, xq, xv, Bq, Bv)
    if qkv.dim() != 2:
        raise ValueError("qkv must be [tokens, (HQ + 2 HKV) D]")
    n, dt = qkv.shape[0], qkv.dtype
    ld, rows, axes, sec = _mrope_inputs(cos, sin, pos, n, HQ, HKV, D, sections, dt)
    _exact(qkv, "qkv", (n, (HQ + 2 * HKV) * D), dt)
    for lo, B, name, heads in ((xq, Bq, "q", HQ), (xv, Bv, "v", HKV)):
        if (lo is None) != (B is None):
            raise ValueError(f"x{name} goes with B{name}")
        if lo is not None:
            _exact(lo, "x" + name, (n, 16), dt)
            _exact(B, "B" + name, (heads * D, 16), dt)
    if out is None:
        q, k, v = qkv.new_empty((n, HQ, D)), qkv.new_empty((n, HKV, D)), qkv.new_empty((n, HKV, D))
    else:
        q, k, v = out
        for name, t, heads in (("q", q, HQ), ("k", k, HKV), ("v", v, HKV)):
            _given(t, name, (n, heads, D), dt, dev)
    args = _MROPE(qkv.data_ptr(), _address(xq), _address(xv), _address(Bq), _address(Bv),
                  q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, 0, 0, 0, 0, 0, cos.data_ptr(),
                  sin.data_ptr(), pos.data_ptr(), ld, lora_scale, n, HQ, HKV, D, _DT[dt], 0, rows,
                  axes, *sec, bool(interleaved))
    _launch("ql_mrope_fwd", dev, args)
    return q, k, v


def mrope_bwd(dq, dk, dv, cos, sin, pos, HQ, HKV, D, sections, interleaved=False,
              dtype=torch.float16, Bq=None, Bv=None, lora_scale=1.0, out=None):
    """(dqkv, dxlo_q, dxlo_v) of mrope_fwd (ql_mrope_bwd): the pre-rotary qkv gradient in `dtype`
    from dq [n, HQ, D], dk / dv [n, HKV, D] (dtype or fp32), and with Bq / Bv the LoRA-A output
    gradients lora_scale * (g . B), fp32 [n, 16]. out: dqkv to write; it must not share memory with an input."""
    dev = _index_of(dq, dk, dv, cos, sin, pos, Bq, Bv)
    if dq.dim() != 3:
        raise ValueError("dq must be [tokens, HQ, D]")
    n, gt = dq.shape[0], dq.dtype
    ld, rows, axes, sec = _mrope_inputs(cos, sin, pos, n, HQ, HKV, D, sections, dtype)
    if gt is not dtype and gt is not torch.float32:
        raise ValueError(f"gradients must be {dtype} or fp32")
    _exact(dq, "dq", (n, HQ, D), gt)
    _exact(dk, "dk", (n, HKV, D), gt)
    _exact(dv, "dv", (n, HKV, D), gt)
    dxlo_q = dxlo_v = None
    if Bq is not None:
        _exact(Bq, "Bq", (HQ * D, 16), dtype)
        dxlo_q = dq.new_empty((n, 16), dtype=torch.float32)
    if Bv is not None:
        _exact(Bv, "Bv", (HKV * D, 16), dtype)
        dxlo_v = dq.new_empty((n, 16), dtype=torch.float32)
    C = (HQ + 2 * HKV) * D
    if out is None:
        out = dq.new_empty((n, C), dtype=dtype)
    else:
        _given(out, "out", (n, C), dtype, dev)
    args = _MROPE(0, 0, 0, _address(Bq), _address(Bv), 0, 0, 0, dq.data_ptr(), dk.data_ptr(),
                  dv.data_ptr(), out.data_ptr(), _address(dxlo_q), _address(dxlo_v),
                  cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), ld, lora_scale, n, HQ, HKV, D,
                  _DT[dtype], _DT[gt], rows, axes, *sec, bool(interleaved))
    _launch("ql_mrope_bwd", dev, args)
    return out, dxlo_q, dxlo_v


# ---------------------------------------------------------------------------------------------
# gradient norm and clipping
# ---------------------------------------------------------------------------------------------
_ADDRESS, _NUMEL = torch.Tensor.data_ptr, torch.Tensor.numel
_CONTIGUOUS, _INDEX = torch.Tensor.is_contiguous, torch.Tensor.get_device


def _grad_list(tensors, name, dev):
    """The tensors' addresses and dtype codes as arrays for the library, after their checks."""
    if dev < 0 or set(map(_INDEX, tensors)) - {dev}:
        _need_cuda(*tensors)
        raise ValueError(f"{name} must be on one device")
    if not all(map(_CONTIGUOUS, tensors)):
        raise ValueError(f"{name} must be contiguous")
    kinds = [t.dtype for t in tensors]
    if len(set(kinds)) == 1:
        codes = array("i", (dtype_code(kinds[0]),)) * len(kinds)
    else:
        codes = array("i", map(dtype_code, kinds))
    return array("Q", map(_ADDRESS, tensors)), codes


def _clip_call(grads, inv_scale, max_norm=None, out=None):
    grads = list(grads)
    count = len(grads)
    dev = grads[0].get_device() if grads else torch.cuda.current_device()
    addr, kind = _grad_list(grads, "gradients", dev)
    size = array("q", map(_NUMEL, grads))
    o_addr, o_kind = addr, kind
    if out is not None:
        out = list(out)
        if array("q", map(_NUMEL, out)) != size:
            raise ValueError("out must hold a tensor of as many elements for each gradient")
        o_addr, o_kind = _grad_list(out, "out", dev)
    scale_dev = 0
    if torch.is_tensor(inv_scale):
        if inv_scale.numel() != 1 or inv_scale.dtype is not torch.float32 \
                or inv_scale.get_device() != dev:
            raise ValueError("inv_scale must be a number or an fp32 scalar on the gradients' device")
        scale_dev, inv_scale = inv_scale.data_ptr(), 1.0
    lib = _lib.lib()
    addresses = [a.buffer_info()[0] for a in (addr, o_addr, size, kind, o_kind)]
    with _on_device(dev):
        norm = torch.empty((), device="cuda", dtype=torch.float32)
        ws = norm.new_empty(lib.ql_grad_norm_workspace(count) // 8, dtype=torch.float64)
        tail = (inv_scale, scale_dev, norm.data_ptr(), ws.data_ptr(), ws.shape[0] * 8, stream_ptr())
        if max_norm is None:
            call("ql_grad_norm", addresses[0], addresses[2], addresses[3], count, *tail)
        else:
            status = lib.ql_clip_grads(*addresses, count, max_norm, *tail)
            if status == STATUS_BAD_ARG:
                raise ValueError("gradients or outputs share memory with one another, or a gradient "
                                 "is its own output in another dtype")
            _lib.check("ql_clip_grads", status)
    return norm


def grad_norm(grads, inv_scale=1.0):
    """The global 2-norm inv_scale * sqrt(sum of squares) of a list of gradient tensors (fp16, bf16
    or fp32, contiguous, one device), as an fp32 scalar on the device (ql_grad_norm). inv_scale: a
    number or a device scalar, e.g. one over a GradScaler's scale."""
    return _clip_call(grads, inv_scale)


def clip_grads(grads, max_norm, inv_scale=1.0, out=None):
    """Rescales the gradients by inv_scale * min(1, max_norm / (norm + 1e-6)), in place or into the
    tensors of `out` (as many elements each, any of the three dtypes, e.g. fp32 master gradients), and returns
    the norm before clipping as a device scalar (ql_clip_grads): torch.nn.utils.clip_grad_norm_ with
    the unscaling folded in, in two kernels and with no host read. As there, a NaN makes the norm and
    every gradient NaN, and an infinite norm makes finite gradients 0 and infinite ones NaN: look at
    the norm, not at the gradients, for an overflow."""
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative")
    return _clip_call(grads, inv_scale, float(max_norm), out)


# ---------------------------------------------------------------------------------------------
# SwiGLU, LoRA weight gradients, embedding
# ---------------------------------------------------------------------------------------------
def glu_fwd(gu, I, out=None):
    n = gu.shape[0]
    m = out if out is not None else torch.empty((n, I), device=gu.device, dtype=gu.dtype)
    call("ql_glu_fwd", _ptr(gu), _ptr(m), n, I, dtype_code(gu.dtype), stream_ptr())
    return m


def glu_bwd(dm, gu, I):
    call("ql_glu_bwd", _ptr(dm), _ptr(gu), gu.shape[0], I, dtype_code(gu.dtype), stream_ptr())
    return gu


def lora_colsum(X, Y, scale=1.0, transpose=False, out=None, workspace=None):
    """scale * X^T Y as [ncols, R] (or [R, ncols] with transpose), fp32; X [n, ncols] may be a
    column slice (unit column stride)."""
    n, ncols = X.shape
    R = Y.shape[1]
    if out is None:
        out = torch.empty((R, ncols) if transpose else (ncols, R), device=X.device,
                          dtype=torch.float32)
    need = int(_lib.lib().ql_lora_colsum_workspace(n, ncols, R))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, device=X.device, dtype=torch.float32)
    call("ql_lora_colsum", _ptr(X), X.stride(0), dtype_code(X.dtype), _ptr(Y),
         dtype_code(Y.dtype), n, ncols, R, float(scale), int(transpose), _ptr(out),
         _ptr(workspace), workspace.numel(), stream_ptr())
    return out


_LG_WS = {}


def lora_grads(jobs):
    """The LoRA weight gradients of a layer in one launch (ql_lora_grads). jobs: up to 4 tuples
    (X [n, ncols] 16-bit with unit column stride, Y [n, 16] 16-bit or fp32, scale, transpose);
    returns the fp32 outputs ([ncols, 16], or [16, ncols] when transposed)."""
    import ctypes

    n = jobs[0][0].shape[0]
    x_dtype = jobs[0][0].dtype
    outs, structs = [], []
    for X, Y, scale, transpose in jobs:
        ncols = X.shape[1]
        out = torch.empty((16, ncols) if transpose else (ncols, 16), device=X.device,
                          dtype=torch.float32)
        outs.append(out)
        structs.append(dict(X=_ptr(X), ldx=X.stride(0), Y=_ptr(Y), out=_ptr(out), ncols=ncols,
                            y_dtype=dtype_code(Y.dtype), transpose=int(transpose),
                            scale=float(scale)))
    arr = (_lib.STRUCTS["ql_lora_grad_job"] * len(jobs))(
        *[_lib.struct("ql_lora_grad_job", **f) for f in structs])
    nc = (ctypes.c_int32 * len(jobs))(*[X.shape[1] for X, _, _, _ in jobs])
    need = int(_lib.lib().ql_lora_grads_workspace(n, ctypes.addressof(nc), len(jobs)))
    ws = _LG_WS.get(jobs[0][0].device)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(need, device=jobs[0][0].device, dtype=torch.uint8)  # counters start at 0
        _LG_WS[jobs[0][0].device] = ws
    call("ql_lora_grads", ctypes.addressof(arr), len(jobs), n, dtype_code(x_dtype), _ptr(ws),
         ws.numel(), stream_ptr())
    return outs


def embed(ids, W, out=None):
    """Rows W[ids] as fp32 [n, H]; W on the GPU, or in page-locked host memory (read over the
    host link by ql_embed_host)."""
    n = ids.numel()
    h = out if out is not None else torch.empty((n, W.shape[1]), device=ids.device,
                                                dtype=torch.float32)
    call("ql_embed" if W.is_cuda else "ql_embed_host", _ptr(ids), _ptr(W), _ptr(h), n,
         W.shape[1], W.shape[0], dtype_code(W.dtype), stream_ptr())
    return h


# ---------------------------------------------------------------------------------------------
# cross-entropy head
# ---------------------------------------------------------------------------------------------
def ce_rows(logits, target, write_grad=True, zero_unsupervised=False, loss=None, entropy=None,
            correct=None):
    rows, V = logits.shape
    dev = logits.device
    loss = loss if loss is not None else torch.empty(rows, device=dev, dtype=torch.float32)
    entropy = entropy if entropy is not None else torch.empty(rows, device=dev,
                                                              dtype=torch.float32)
    correct = correct if correct is not None else torch.empty(rows, device=dev,
                                                              dtype=torch.int32)
    args = _lib.struct("ql_ce_rows_args", logits=_ptr(logits), target=_ptr(target),
                       loss=_ptr(loss), entropy=_ptr(entropy), correct=_ptr(correct), rows=rows,
                       V=V, ld=logits.stride(0), write_grad=int(write_grad),
                       zero_unsupervised=int(zero_unsupervised), dtype=dtype_code(logits.dtype))
    call("ql_ce_rows", ctypes_ref(args), stream_ptr())
    return loss, entropy, correct


def ce_piece(logits, w, target, state, best_idx, xt, alpha, wt, v0, n_sup, acc=None,
             part=None, part_valid=False, H=None):
    """Reference _ce_piece (engine.py:1033-1038) on a vocabulary piece [v0, v0 + width) of the
    logits. acc / part: the fp32 gradient accumulator moved to the new running max in place,
    acc = alpha (acc + part) (part folded in when part_valid)."""
    rows, width = logits.shape
    args = _lib.struct("ql_ce_piece_args", logits=_ptr(logits), w=_ptr(w), target=_ptr(target),
                       state=_ptr(state), best_idx=_ptr(best_idx), xt=_ptr(xt),
                       alpha=_ptr(alpha), wt=_ptr(wt), rows=rows, v0=int(v0), width=width,
                       ld=logits.stride(0), n_sup=int(n_sup),
                       H=int(H) if H is not None else w.shape[1],
                       dtype=dtype_code(logits.dtype), acc=_ptr(acc), part=_ptr(part),
                       part_valid=int(bool(part_valid)))
    call("ql_ce_piece", ctypes_ref(args), stream_ptr())


def ce_finish(state, best_idx, xt, target, loss, entropy, correct, acc, wt, dh, n_sup,
              part=None):
    args = _lib.struct("ql_ce_finish_args", state=_ptr(state), best_idx=_ptr(best_idx),
                       xt=_ptr(xt), target=_ptr(target), loss=_ptr(loss),
                       entropy=_ptr(entropy), correct=_ptr(correct), acc=_ptr(acc),
                       wt=_ptr(wt), dh=_ptr(dh), rows=state.shape[0], n_sup=int(n_sup),
                       H=acc.shape[1], dtype=dtype_code(dh.dtype), part=_ptr(part))
    call("ql_ce_finish", ctypes_ref(args), stream_ptr())


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def attn_fwd(q, k, v, cu_seqlens, max_len, scale, out=None, lse=None):
    n, HQ, D = q.shape
    HKV = k.shape[1]
    out = out if out is not None else torch.empty_like(q)
    lse = lse if lse is not None else torch.empty((HQ, n), device=q.device, dtype=torch.float32)
    args = _lib.struct("ql_attn_fwd_args", q=_ptr(q), k=_ptr(k), v=_ptr(v),
                       cu_seqlens=_ptr(cu_seqlens), out=_ptr(out), lse=_ptr(lse),
                       scale=float(scale), n=n, B=cu_seqlens.numel() - 1, max_len=int(max_len),
                       HQ=HQ, HKV=HKV, D=D, dtype=dtype_code(q.dtype))
    call("ql_attn_fwd", ctypes_ref(args), stream_ptr())
    return out, lse


def attn_bwd(dout, q, k, v, out, lse, cu_seqlens, max_len, scale, dq=None, dk=None, dv=None,
             dvec=None, deterministic=False):
    """Reference _attn_bwd (engine.py:864-869): dq, dk, dv (fp32; dk / dv per KV head). With
    deterministic, each contribution goes to its own slot of a partials workspace and one kernel
    sums them in a fixed order (D = 128)."""
    n, HQ, D = q.shape
    HKV = k.shape[1]
    dev = q.device
    parts = None
    if deterministic:
        floats = int(_lib.lib().ql_attn_bwd_partials_floats(n, int(max_len), HQ, HKV))
        parts = torch.empty(max(floats, 4), device=dev, dtype=torch.float32)
    dq = dq if dq is not None else torch.empty((n, HQ, D), device=dev, dtype=torch.float32)
    dk = dk if dk is not None else torch.empty((n, HKV, D), device=dev, dtype=torch.float32)
    dv = dv if dv is not None else torch.empty((n, HKV, D), device=dev, dtype=torch.float32)
    dvec = dvec if dvec is not None else torch.empty((HQ, n), device=dev, dtype=torch.float32)
    args = _lib.struct("ql_attn_bwd_args", q=_ptr(q), k=_ptr(k), v=_ptr(v), out=_ptr(out),
                       dout=_ptr(dout), lse=_ptr(lse), cu_seqlens=_ptr(cu_seqlens),
                       dvec=_ptr(dvec), dq=_ptr(dq), dk=_ptr(dk), dv=_ptr(dv),
                       scale=float(scale), n=n, B=cu_seqlens.numel() - 1, max_len=int(max_len),
                       HQ=HQ, HKV=HKV, D=D, dtype=dtype_code(q.dtype), partials=_ptr(parts))
    call("ql_attn_bwd", ctypes_ref(args), stream_ptr())
    return dq, dk, dv


_ATTN_MOD = _lib.packer("ql_attn_mod_args", """q k v out lse cu_seqlens slopes prefix_len doc_ids
    ranges dout dq dk dv workspace workspace_floats ldq ldk ldv scale softcap n B max_len HQ HKV D
    dtype causal window""")


def _attn_mod_inputs(q, k, v, cu_seqlens, max_len, scale, softcap, slopes, window, doc_ids,
                     prefix_len):
    """The checked sizes both directions of attn_mod share: (n, HQ, HKV, D, B, row strides of q, k
    and v, dtype code, device index, window as the library takes it)."""
    dev = _index_of(q, k, v, cu_seqlens, slopes, doc_ids, prefix_len)
    dt = q.dtype
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be [tokens, heads, D]")
    n, HQ, D = q.shape
    HKV = k.shape[1]
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise ValueError(f"unsupported dtype {dt}")
    if D != 64 and D != 128:
        raise ValueError(f"head size {D}: 64 or 128 are supported")
    if HKV == 0 or HQ == 0 or HQ % HKV:
        raise ValueError(f"{HQ} query heads over {HKV} key heads")
    kv = (n, HKV, D)
    strides = []
    for name, t, shape, heads in (("q", q, q.shape, HQ), ("k", k, kv, HKV), ("v", v, kv, HKV)):
        if t.shape != shape or t.dtype is not dt:
            raise ValueError(f"{name} must be a {dt} {list(shape)}, got {t.dtype} {list(t.shape)}")
        ld, inner, unit = t.stride()
        if n and (unit != 1 or (inner != D and heads > 1)):
            raise ValueError(f"{name}'s heads must be contiguous within a row")
        if n < 2:
            ld = heads * D
        if ld < heads * D or ld & 7 or t.data_ptr() & 15:
            raise ValueError(f"{name}'s rows must start at multiples of 16 bytes and not overlap")
        strides.append(ld)
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be int32 [sequences + 1]")
    B = cu_seqlens.shape[0] - 1
    _exact(cu_seqlens, "cu_seqlens", (B + 1,), torch.int32)
    if slopes is not None:
        _exact(slopes, "slopes", (HQ,), torch.float32)
    if doc_ids is not None:
        _exact(doc_ids, "doc_ids", (n,), torch.int32)
    if prefix_len is not None:
        _exact(prefix_len, "prefix_len", (B,), torch.int32)
    if not (0 <= max_len <= n and window >= 0 and 0 < scale < _INF and 0 <= softcap < _INF):
        raise ValueError("needs 0 <= max_len <= tokens, window >= 0, 0 < scale < inf and "
                         "0 <= softcap < inf")
    if slopes is not None and scale < 1e-30:
        raise ValueError("slopes with a scale below 1e-30 are not supported")
    if 0 < softcap < 1e-4 * scale:
        raise ValueError("a softcap below 1e-4 scale is not supported")
    if scale > 2.3e38 or softcap > 2.3e38 or 0 < scale < 1.1754944e-38 * softcap:
        raise ValueError("scale and softcap of at most 2.3e38 and scale / softcap of at least 1.2e-38 "
                         "are supported")
    return n, HQ, HKV, D, B, strides, _DT[dt], dev, min(window, INT_MAX)


def attn_mod_fwd(q, k, v, cu_seqlens, max_len, scale, causal=True, softcap=0.0, slopes=None,
                 window=0, doc_ids=None, prefix_len=None, out=None, lse=None):
    """(out, lse) of varlen GQA attention with modified scores and masks (ql_attn_mod_fwd).

    q [n, HQ, D], k / v [n, HKV, D] (fp16 or bf16, D 64 or 128; rows may be strided, e.g. slices of
    a fused qkv), cu_seqlens int32 [B + 1], max_len at least the longest sequence. With positions
    i, j within a sequence: s = cap(scale q_i . k_j) - slopes[h] |i - j|, cap(x) = softcap
    tanh(x / softcap); a query sees key j if j <= i or j < prefix_len[b] (causal;
    without it prefix_len changes nothing), |i - j| < window
    (window > 0), and both are in the same run of equal doc_ids (negative ids: padding). slopes
    fp32 [HQ], doc_ids int32 [n], prefix_len int32 [B]. out as q (contiguous), lse fp32 [HQ, n];
    a query that sees nothing gets out 0 and lse -inf. Rows behind the last sequence are not written. out
    may be a contiguous q itself; otherwise outputs that share memory with an input or one another are
    refused."""
    n, HQ, HKV, D, B, ld, dt, dev, window = _attn_mod_inputs(
        q, k, v, cu_seqlens, max_len, scale, softcap, slopes, window, doc_ids, prefix_len)
    if out is None:
        out = q.new_empty((n, HQ, D))
    else:
        _given(out, "out", (n, HQ, D), q.dtype, dev)
    if lse is None:
        lse = q.new_empty((HQ, n), dtype=torch.float32)
    else:
        _given(lse, "lse", (HQ, n), torch.float32, dev)
    ranges = q.new_empty((n, 2), dtype=torch.int32) if doc_ids is not None else None
    args = _ATTN_MOD(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                     cu_seqlens.data_ptr(), _address(slopes), _address(prefix_len),
                     _address(doc_ids), _address(ranges), 0, 0, 0, 0, 0, 0, *ld, scale, softcap, n,
                     B, max_len, HQ, HKV, D, dt, bool(causal), window)
    _launch("ql_attn_mod_fwd", dev, args)
    return out, lse


def attn_mod_bwd(dout, q, k, v, out, lse, cu_seqlens, max_len, scale, causal=True, softcap=0.0,
                 slopes=None, window=0, doc_ids=None, prefix_len=None, dq=None, dk=None, dv=None):
    """(dq, dk, dv) of attn_mod_fwd, in q's dtype, given its arguments, out and lse
    (ql_attn_mod_bwd); dout [n, HQ, D] contiguous; gradients that share memory with an input or one
    another are refused. Bit-identical from run to run. Rows that see (keys that are seen by) at most 256 others, by tiles
    of 128, get gradients off by their own rounding only; longer sums add one rounding of P and dS. In
    fp16 a loss scale too large for dS = P (dP - Dvec) gives gradients that are not finite."""
    n, HQ, HKV, D, B, ld, dt, dev, window = _attn_mod_inputs(
        q, k, v, cu_seqlens, max_len, scale, softcap, slopes, window, doc_ids, prefix_len)
    dtype, shape, kv = q.dtype, (n, HQ, D), (n, HKV, D)
    _given(dout, "dout", shape, dtype, dev)
    _given(out, "out", shape, dtype, dev)
    _given(lse, "lse", (HQ, n), torch.float32, dev)
    grads = []
    for name, t, want in (("dq", dq, shape), ("dk", dk, kv), ("dv", dv, kv)):
        if t is None:
            t = q.new_empty(want)
        else:
            _given(t, name, want, dtype, dev)
        grads.append(t)
    lib = _lib.lib()
    with _on_device(dev):  # the workspace's size goes by the device's SMs
        floats = lib.ql_attn_mod_bwd_workspace(n, max_len, HQ, HKV, D, bool(causal), window)
    # a multiple of four floats, and behind it the documents' ranges
    ws = q.new_empty(floats + (0 if doc_ids is None else 2 * n) + 4, dtype=torch.float32)
    work = ws.data_ptr()
    args = _ATTN_MOD(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                     cu_seqlens.data_ptr(), _address(slopes), _address(prefix_len),
                     _address(doc_ids), 0 if doc_ids is None else work + 4 * floats,
                     dout.data_ptr(), *(t.data_ptr() for t in grads), work, floats, *ld, scale,
                     softcap, n, B, max_len, HQ, HKV, D, dt, bool(causal), window)
    _launch("ql_attn_mod_bwd", dev, args)
    return tuple(grads)


def gather_rows(src, idx, out=None):
    n, H = idx.numel(), src.shape[1]
    out = out if out is not None else torch.empty((n, H), device=src.device, dtype=torch.float32)
    call("ql_gather_rows", _ptr(src), _ptr(idx), _ptr(out), n, H, stream_ptr())
    return out


def scatter_rows(src, idx, out, scale=None, out16=None):
    n, H = src.shape
    call("ql_scatter_rows", _ptr(src), _ptr(idx), _ptr(scale), _ptr(out), _ptr(out16), n, H,
         dtype_code(out16.dtype) if out16 is not None else 0, stream_ptr())
    return out
