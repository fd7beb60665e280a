"""Operators measured on a GPU: rotary positions with several axes, attention with modified scores
and masks, and the global gradient norm with clipping. Each case runs in its plain form (elementary
torch operations in 32 bits, rounded once) or, with `own`, through this package's entry points.

Shapes are those of the package's model configurations: heads (12, 2, 128), (28, 4, 128) and
(4, 2, 64), LoRA rank 16, batches of packed sequences with int32 cu_seqlens.
"""

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
RANK = 16
LORA_SCALE = 2.0
POSITIONS = 16384
HEADS = ((12, 2, 128), (28, 4, 128), (4, 2, 64))
HIDDEN = {12: 1536, 28: 3584, 4: 256}
SECTIONS = {128: (16, 24, 24), 64: (8, 12, 12)}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _mrope(name, n, heads, dtype, back, lora, interleaved, layout):
    return {"name": name, "op": "mrope", "n": n, "HQ": heads[0], "HKV": heads[1], "D": heads[2],
            "dtype": dtype, "back": back, "lora": lora, "interleaved": interleaved,
            "layout": layout}


def _attn(name, seqs, lo, hi, heads, dtype, back, layout, causal=True, softcap=0.0, slopes=False,
          window=0, docs=0, prefix=False):
    return {"name": name, "op": "attn", "seqs": seqs, "lo": lo, "hi": hi, "HQ": heads[0],
            "HKV": heads[1], "D": heads[2], "dtype": dtype, "back": back, "layout": layout,
            "causal": causal, "softcap": softcap, "slopes": slopes, "window": window,
            "docs": docs, "prefix": prefix}


def _clip(name, tensors, rows, cols, dtype, out, limit, scale):
    return {"name": name, "op": "clip", "tensors": tensors, "rows": rows, "cols": cols,
            "dtype": dtype, "out": out, "limit": limit, "scale": scale}


def listed():
    big, mid, small = HEADS[1], HEADS[0], HEADS[2]
    return [
        # one small picture and its caption, forward only: launch latency
        _mrope("mrope_fwd_one_row", 61, small, "fp16", False, True, False, 1),
        # a training micro-batch of about a thousand tokens, both directions, LoRA products inside
        _mrope("mrope_train_1k", 1090, mid, "fp16", True, True, False, 2),
        # the long-row batch of the larger model, frequencies dealt to the axes in turn
        _mrope("mrope_train_24k", 24411, big, "bf16", True, True, True, 3),
        # evaluation of one short row with a sliding window: the smallest call
        _attn("attn_fwd_short_window", 1, 47, 47, small, "fp16", False, 1, window=16),
        # the ordinary fine-tuning micro-batch, several documents packed in each row, some padding
        _attn("attn_train_documents", 4, 200, 420, mid, "fp16", True, 2, docs=4),
        # scoring long rows with capped scores and a sliding window
        _attn("attn_fwd_cap_window", 8, 2048, 4096, mid, "bf16", False, 3, softcap=30.0,
              window=1024),
        # prompts seen in both directions (prefix mask), the larger model's heads, training
        _attn("attn_train_prefix", 4, 1024, 4096, big, "bf16", True, 4, prefix=True),
        # one long row with a distance bias in place of rotary positions, training
        _attn("attn_train_distance_8k", 1, 8192, 8192, mid, "bf16", True, 5, slopes=True),
        # capped scores at head size 64, rows of very different lengths, training
        _attn("attn_train_cap_ragged", 8, 64, 2048, small, "fp16", True, 6, softcap=50.0),
        # a two-layer adapter's gradients, within the limit: nothing is rescaled
        _clip("clip_few_within", 8, 16, 256, "fp32", False, 100.0, 1.0),
        # every adapter gradient of the 28-layer model, unscaled and clipped into the
        # optimizer's buffers
        _clip("clip_adapters", 112, 16, 1536, "fp32", True, 1.0, 2.0 ** -16),
        # 16-bit gradients of full weight matrices into fp32 master gradients
        _clip("clip_full_weights", 84, 8960, 1536, "bf16", True, 1.0, 1.0),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, evenly over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("mrope", "attn", "attn", "attn", "clip"))
    heads = rng.choice(HEADS)
    dtype = rng.choice(("fp16", "bf16"))
    layout = rng.randrange(1 << 20)
    if op == "mrope":
        case = _mrope("", _between(rng, 1, 24000), heads, dtype, rng.random() < 0.6,
                      rng.random() < 0.7, rng.random() < 0.5, layout)
    elif op == "attn":
        seqs = rng.randint(1, 8)
        hi = _between(rng, 1, 4096)
        while seqs * hi * hi * heads[0] > 8e8:
            hi = hi * 3 // 4
        case = _attn("", seqs, max(1, int(hi * rng.random())), hi, heads, dtype,
                     rng.random() < 0.7, layout, causal=rng.random() < 0.85,
                     softcap=rng.choice((0.0, 0.0, 30.0, 50.0)), slopes=rng.random() < 0.25,
                     window=rng.choice((0, 0, _between(rng, 1, 2048))),
                     docs=rng.choice((0, 0, rng.randint(2, 9))), prefix=rng.random() < 0.3)
    else:
        rows = _between(rng, 1, 4096)
        case = _clip("", _between(rng, 1, 400), rows, _between(rng, 1, max(1, 1_500_000 // rows)),
                     rng.choice(("fp16", "bf16", "fp32")), True, rng.choice((0.1, 1.0, 1e6)),
                     rng.choice((1.0, 2.0 ** -10)))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------
# layouts: what a case's shape and mask are, whatever the values
# ---------------------------------------------------------------------------------------------
def _lengths(case):
    rng = np.random.RandomState(case["layout"])
    return rng.randint(case["lo"], case["hi"] + 1, case["seqs"]).astype(np.int64)


def _documents(case, lengths):
    """Document ids of the packed tokens: up to `docs` runs per row, the last few tokens of about
    every second row padding (-1)."""
    rng = np.random.RandomState(case["layout"] + 1)
    ids = []
    for length in lengths:
        cuts = np.sort(rng.randint(0, length + 1, case["docs"] - 1))
        row = np.searchsorted(cuts, np.arange(length), side="right")
        pad = int(rng.randint(0, 17)) if rng.rand() < 0.5 else 0
        if 0 < pad < length:
            row[length - pad:] = -1
        ids.append(row)
    return np.concatenate(ids).astype(np.int32)


def _prefixes(case, lengths):
    rng = np.random.RandomState(case["layout"] + 2)
    return (lengths * rng.uniform(0.1, 0.6, len(lengths))).astype(np.int32)


def _axis_positions(case):
    """int32 [3, n]: stretches of text (the three positions equal) and pictures (time fixed,
    height and width over a grid), each starting after the largest position before it."""
    rng = np.random.RandomState(case["layout"])
    parts, total, at = [], 0, 0
    while total < case["n"]:
        if rng.rand() < 0.5:
            length = int(rng.randint(1, 200))
            part = np.tile(np.arange(length), (3, 1))
        else:
            h, w = (int(v) for v in rng.randint(2, 33, 2))
            y, x = np.divmod(np.arange(h * w), w)
            part = np.stack([np.zeros_like(y), y, x])
        parts.append(part + at)
        at = (at + int(part.max()) + 1) % (POSITIONS - 300)
        total += part.shape[1]
    return np.concatenate(parts, axis=1)[:, :case["n"]].astype(np.int32)


def _frequency_axes(case):
    """The axis (0, 1, 2) of each of the D / 2 frequencies: blocks of the sections, or dealt to the
    axes in turn while an axis has some left."""
    sections = SECTIONS[case["D"]]
    if not case["interleaved"]:
        return np.repeat(np.arange(3), sections)
    left, axes = list(sections), []
    while len(axes) < sum(sections):
        for axis in range(3):
            if left[axis]:
                left[axis] -= 1
                axes.append(axis)
    return np.array(axes)


def _grad_shapes(case):
    """The tensors' shapes: [rows, cols], every second one transposed, every fourth an eighth."""
    shapes = []
    for i in range(case["tensors"]):
        rows, cols = case["rows"], case["cols"]
        if i % 4 == 3:
            cols = max(1, cols // 8)
        shapes.append((cols, rows) if i % 2 else (rows, cols))
    return shapes


def _pairs(case):
    """How many (query, key) pairs the mask of an attention case allows, per head."""
    lengths = _lengths(case)
    docs = _documents(case, lengths) if case["docs"] else None
    prefix = _prefixes(case, lengths) if case["prefix"] else np.zeros(len(lengths), np.int64)
    total, start = 0, 0
    for length, pre in zip(lengths, prefix):
        i = np.arange(length)
        lo, hi = np.zeros_like(i), np.full_like(i, length)
        if case["causal"]:
            hi = np.maximum(i + 1, pre)
        if case["window"]:
            lo, hi = np.maximum(lo, i - case["window"] + 1), np.minimum(hi, i + case["window"])
        if docs is not None:
            ids = docs[start:start + length]
            edge = np.flatnonzero(np.diff(ids)) + 1
            first = np.concatenate([[0], edge])[np.searchsorted(edge, i, side="right")]
            last = np.concatenate([edge, [length]])[np.searchsorted(edge, i, side="right")]
            lo, hi = np.maximum(lo, first), np.where(ids >= 0, np.minimum(hi, last), 0)
        total += int(np.maximum(hi - lo, 0).sum())
        start += length
    return total


def work(case):
    if case["op"] == "mrope":
        n, c = case["n"], (case["HQ"] + 2 * case["HKV"]) * case["D"]
        qv = (case["HQ"] + case["HKV"]) * case["D"]
        # qkv in, q / k / v out; the gradients in and out; adapter factors and their gradients
        moved = n * c * 2 * 2 + n * 12
        flops = n * c * 4
        if case["lora"]:
            moved += n * RANK * 2 * 2 + qv * RANK * 2
            flops += n * qv * RANK * 2
        if case["back"]:
            moved += n * c * 2 * 2
            flops += n * c * 4
            if case["lora"]:
                moved += n * RANK * 2 * 4
                flops += n * qv * RANK * 2
        return {"bytes": moved, "flops": flops}
    if case["op"] == "attn":
        n, d = int(_lengths(case).sum()), case["D"]
        q, kv = n * case["HQ"] * d * 2, n * case["HKV"] * d * 2
        moved = 2 * q + 2 * kv + n * case["HQ"] * 4
        flops = _pairs(case) * case["HQ"] * d * 4
        if case["back"]:
            moved += 2 * q + 2 * kv  # dout in, dq / dk / dv out
            flops += _pairs(case) * case["HQ"] * d * 10
        return {"bytes": moved, "flops": flops}
    size = sum(r * c for r, c in _grad_shapes(case))
    given = size * (4 if case["dtype"] == "fp32" else 2)
    return {"bytes": given + (size * 4 if case["out"] else 0), "flops": size * 3}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _to_gpu(array):
    return torch.from_numpy(np.ascontiguousarray(array)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "clip":
        shapes, dtype = _grad_shapes(case), DTYPES[case["dtype"]]
        sizes = [r * c for r, c in shapes]
        # one buffer of all gradients, as the training step hands them out, and views of it
        flat = torch.empty(sum(sizes), device="cuda", dtype=dtype)
        step = 1 << 26
        for at in range(0, flat.numel(), step):
            part = flat[at:at + step]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda")
                       .mul_(1e-3 / case["scale"]))
        state["flat"] = flat
        state["grads"] = [v.view(s) for v, s in zip(flat.split(sizes), shapes)]
        if case["out"]:
            state["flat_out"] = torch.zeros(sum(sizes), device="cuda")
            state["outs"] = [v.view(s) for v, s in zip(state["flat_out"].split(sizes), shapes)]
        return state
    dtype, hq, hkv, d = DTYPES[case["dtype"]], case["HQ"], case["HKV"], case["D"]
    if case["op"] == "mrope":
        n = case["n"]
        state["qkv"] = _normal(gen, (n, (hq + 2 * hkv) * d), dtype)
        angles = torch.outer(torch.arange(POSITIONS, dtype=torch.float64),
                             1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
        state["cos"], state["sin"] = angles.cos().float().cuda(), angles.sin().float().cuda()
        state["pos"] = _to_gpu(_axis_positions(case))
        state["axes"] = _to_gpu(_frequency_axes(case))
        if case["lora"]:
            for name, out in (("q", hq * d), ("v", hkv * d)):
                state["x" + name] = _normal(gen, (n, RANK), dtype)
                state["B" + name] = _normal(gen, (out, RANK), dtype, 0.05)
        if case["back"]:
            state["dq"] = _normal(gen, (n, hq, d), dtype)
            state["dk"] = _normal(gen, (n, hkv, d), dtype)
            state["dv"] = _normal(gen, (n, hkv, d), dtype)
        return state
    lengths = _lengths(case)
    n, rows, longest = int(lengths.sum()), len(lengths), int(lengths.max())
    start = np.concatenate([[0], np.cumsum(lengths)])
    state["q"] = _normal(gen, (n, hq, d), dtype, 1.5)
    state["k"] = _normal(gen, (n, hkv, d), dtype, 1.5)
    state["v"] = _normal(gen, (n, hkv, d), dtype)
    if case["back"]:
        state["dout"] = _normal(gen, (n, hq, d), dtype)
    state["cu_seqlens"] = _to_gpu(start.astype(np.int32))
    state["max_len"] = longest
    # the packed tokens' places in the padded batch, which the training step keeps as well
    row = np.repeat(np.arange(rows), lengths)
    state["tok"] = _to_gpu(row * longest + np.arange(n) - start[row])
    state["rows"] = rows
    state["doc_ids"] = _to_gpu(_documents(case, lengths)) if case["docs"] else None
    state["prefix_len"] = _to_gpu(_prefixes(case, lengths)) if case["prefix"] else None
    state["slope_of"] = None
    if case["slopes"]:
        state["slope_of"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if state["op"] == "mrope":
        return _run_mrope(state)
    if state["op"] == "attn":
        return _run_attn(state)
    return _run_clip(state)


def _turn(x, cos, sin, sign):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin * sign, b * cos + a * sin * sign], -1)


def _run_mrope(s):
    hq, hkv, d, dtype = s["HQ"], s["HKV"], s["D"], s["qkv"].dtype
    if own:
        from hack_fe30cb28_opus_5_5_ultracode_b200 import ops

        sections = SECTIONS[d]
        got = ops.mrope_fwd(s["qkv"], s["cos"], s["sin"], s["pos"], hq, hkv, d, sections,
                            interleaved=s["interleaved"], lora_scale=LORA_SCALE,
                            xq=s.get("xq"), xv=s.get("xv"), Bq=s.get("Bq"), Bv=s.get("Bv"))
        if not s["back"]:
            return list(got)
        back = ops.mrope_bwd(s["dq"], s["dk"], s["dv"], s["cos"], s["sin"], s["pos"], hq, hkv, d,
                             sections, interleaved=s["interleaved"], dtype=dtype,
                             lora_scale=LORA_SCALE, Bq=s.get("Bq"), Bv=s.get("Bv"))
        return [*got, *(g for g in back if g is not None)]
    n = s["qkv"].shape[0]
    freq = torch.arange(d // 2, device="cuda")
    place = s["pos"].long()[s["axes"].long()].t()          # [n, D / 2]: each frequency's position
    cos, sin = s["cos"][place, freq][:, None], s["sin"][place, freq][:, None]
    q, k, v = s["qkv"].float().split([hq * d, hkv * d, hkv * d], -1)
    if s["lora"]:
        q = q + LORA_SCALE * (s["xq"].float() @ s["Bq"].float().t())
        v = v + LORA_SCALE * (s["xv"].float() @ s["Bv"].float().t())
    got = [_turn(q.view(n, hq, d), cos, sin, 1.0), _turn(k.reshape(n, hkv, d), cos, sin, 1.0),
           v.reshape(n, hkv, d)]
    got = [g.to(dtype) for g in got]
    if not s["back"]:
        return got
    gq = _turn(s["dq"].float(), cos, sin, -1.0).view(n, -1)
    gk = _turn(s["dk"].float(), cos, sin, -1.0).view(n, -1)
    gv = s["dv"].float().view(n, -1)
    got.append(torch.cat([gq, gk, gv], -1).to(dtype))
    if s["lora"]:
        got += [LORA_SCALE * (gq @ s["Bq"].float()), LORA_SCALE * (gv @ s["Bv"].float())]
    return got


def _allowed(s, longest):
    """bool [rows, longest, longest]: which key each query may see, in the padded batch."""
    at = torch.arange(longest, device="cuda")
    real = torch.zeros(s["rows"] * longest, device="cuda", dtype=torch.bool)
    real[s["tok"]] = True
    real = real.view(s["rows"], longest)
    ahead = at[None, :] - at[:, None]
    ok = real[:, :, None] & real[:, None, :]
    if s["causal"]:
        seen = (ahead <= 0)[None]
        if s["prefix_len"] is not None:
            seen = seen | (at[None, None, :] < s["prefix_len"][:, None, None])
        ok &= seen
    if s["window"]:
        ok &= (ahead.abs() < s["window"])[None]
    if s["doc_ids"] is not None:
        ids = torch.full((s["rows"] * longest,), -1, device="cuda", dtype=torch.int32)
        ids[s["tok"]] = s["doc_ids"]
        ids = ids.view(s["rows"], longest)
        change = torch.zeros_like(ids)
        change[:, 1:] = ids[:, 1:] != ids[:, :-1]
        run_of = change.cumsum(1)                      # a document is a run of equal ids
        ok &= (run_of[:, :, None] == run_of[:, None, :]) & (ids >= 0)[:, :, None]
    return ok[:, None, None]


def _padded(x, s, longest):
    """Packed [n, heads, D] as fp32 [rows, heads, longest, D]."""
    full = torch.zeros((s["rows"] * longest, *x.shape[1:]), device="cuda")
    full[s["tok"]] = x.float()
    return full.view(s["rows"], longest, *x.shape[1:]).transpose(1, 2)


def _packed(x, s, dtype):
    """The inverse of _padded, for [rows, heads, longest, ...]."""
    flat = x.transpose(1, 2).reshape(-1, x.shape[1], *x.shape[3:])
    return flat[s["tok"]].to(dtype)


def _run_attn(s):
    hq, hkv, d, dtype = s["HQ"], s["HKV"], s["D"], s["q"].dtype
    scale = d ** -0.5
    if own:
        from hack_fe30cb28_opus_5_5_ultracode_b200 import ops

        mods = dict(causal=s["causal"], softcap=s["softcap"], slopes=s["slope_of"],
                    window=s["window"], doc_ids=s["doc_ids"], prefix_len=s["prefix_len"])
        out, lse = ops.attn_mod_fwd(s["q"], s["k"], s["v"], s["cu_seqlens"], s["max_len"], scale,
                                    **mods)
        if not s["back"]:
            return [out, lse]
        return [out, lse, *ops.attn_mod_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse,
                                            s["cu_seqlens"], s["max_len"], scale, **mods)]
    rows, longest, group = s["rows"], s["max_len"], hq // hkv
    q = _padded(s["q"], s, longest).view(rows, hkv, group, longest, d)
    k = _padded(s["k"], s, longest)[:, :, None]
    v = _padded(s["v"], s, longest)[:, :, None]
    score = (q @ k.transpose(-1, -2)).mul_(scale)
    bent = None
    if s["softcap"]:
        bent = (score / s["softcap"]).tanh_()
        score = bent * s["softcap"]
    if s["slope_of"] is not None:
        at = torch.arange(longest, device="cuda", dtype=torch.float32)
        away = (at[None, :] - at[:, None]).abs()
        score = score - s["slope_of"].float().view(hkv, group, 1, 1) * away
    score.masked_fill_(~_allowed(s, longest), float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).view(rows, hq, longest)
    p = p.div_(torch.where(total > 0, total, 1.0))
    out = (p @ v).view(rows, hq, longest, d)
    got = [_packed(out, s, dtype), _packed(lse, s, torch.float32).t().contiguous()]
    if not s["back"]:
        return got
    g = _padded(s["dout"], s, longest).view(rows, hkv, group, longest, d)
    dv = (p.transpose(-1, -2) @ g).sum(2)
    dp = g @ v.transpose(-1, -2)
    ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p)
    if bent is not None:
        ds = ds * (1.0 - bent * bent)
    dq = (ds @ k).mul_(scale).view(rows, hq, longest, d)
    dk = (ds.transpose(-1, -2) @ q).mul_(scale).sum(2)
    return got + [_packed(dq, s, dtype), _packed(dk, s, dtype), _packed(dv, s, dtype)]


def _run_clip(s):
    outs = s["outs"] if s["out"] else None
    flat = s["flat_out"] if s["out"] else s["flat"]
    if own:
        from hack_fe30cb28_opus_5_5_ultracode_b200 import ops

        return [ops.clip_grads(s["grads"], s["limit"], inv_scale=s["scale"], out=outs), flat]
    squares = [g.float().square().sum(dtype=torch.float64) for g in s["grads"]]
    norm = (torch.stack(squares).sum().sqrt() * s["scale"]).float()
    factor = (s["limit"] / (norm + 1e-6)).clamp(max=1.0) * s["scale"]
    for o, g in zip(outs or s["grads"], s["grads"]):
        o.copy_(g.float() * factor)
    return [norm, flat]


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "mrope":
        return _exact_mrope(s)
    if case["op"] == "attn":
        return _exact_attn(s)
    return _exact_clip(s)


def _exact_mrope(s):
    n, hq, hkv, d = s["qkv"].shape[0], s["HQ"], s["HKV"], s["D"]
    axes, half = s["axes"].tolist(), d // 2
    pos = s["pos"].long()
    # a head's pair (x[f], x[f + D / 2]) as the complex number that e^(i angle) multiplies
    turn = torch.stack([torch.complex(s["cos"][pos[a], f].double(), s["sin"][pos[a], f].double())
                        for f, a in enumerate(axes)], -1)[:, None]

    def rotate(x, by):
        x = x.double()
        z = torch.complex(x[..., :half], x[..., half:]) * by
        return torch.cat([z.real, z.imag], -1)

    x = s["qkv"].double().view(n, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["lora"]:
        q = q + LORA_SCALE * torch.einsum("nr,or->no", s["xq"].double(),
                                          s["Bq"].double()).view(n, hq, d)
        v = v + LORA_SCALE * torch.einsum("nr,or->no", s["xv"].double(),
                                          s["Bv"].double()).view(n, hkv, d)
    got = [rotate(q, turn), rotate(k, turn), v]
    if not s["back"]:
        return got
    gq, gk = rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())
    gv = s["dv"].double()
    got.append(torch.cat([gq, gk, gv], 1).reshape(n, -1))
    if s["lora"]:
        got.append(LORA_SCALE * torch.einsum("no,or->nr", gq.reshape(n, -1), s["Bq"].double()))
        got.append(LORA_SCALE * torch.einsum("no,or->nr", gv.reshape(n, -1), s["Bv"].double()))
    return got


def _exact_attn(s):
    hq, hkv, d = s["HQ"], s["HKV"], s["D"]
    cu = s["cu_seqlens"].tolist()
    n, group, scale = cu[-1], hq // hkv, d ** -0.5
    new = lambda *shape: torch.zeros(shape, device="cuda", dtype=torch.float64)  # noqa: E731
    out, lse = new(n, hq, d), new(hq, n)
    dq, dk, dv = new(n, hq, d), new(n, hkv, d), new(n, hkv, d)
    for b, (t0, t1) in enumerate(zip(cu[:-1], cu[1:])):
        length = t1 - t0
        i = torch.arange(length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        blocked = torch.zeros(length, length, device="cuda", dtype=torch.bool)
        if s["causal"]:
            reach = int(s["prefix_len"][b]) if s["prefix_len"] is not None else 0
            blocked |= (j > i) & (j >= reach)
        if s["window"]:
            blocked |= (i - j >= s["window"]) | (j - i >= s["window"])
        if s["doc_ids"] is not None:
            ids, label, labels = s["doc_ids"][t0:t1].tolist(), 0, []
            for at, value in enumerate(ids):
                label += at > 0 and value != ids[at - 1]
                labels.append(label if value >= 0 else -1)
            labels = torch.tensor(labels, device="cuda")
            blocked |= (labels[:, None] != labels[None, :]) | (labels < 0)[:, None]
        for h in range(hq):
            q, k, v = s["q"][t0:t1, h].double(), s["k"][t0:t1, h // group].double(), \
                s["v"][t0:t1, h // group].double()
            x = torch.mm(q, k.t()) * scale
            slope = torch.ones_like(x)
            if s["softcap"]:
                slope = torch.cosh(x / s["softcap"]) ** -2
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            if s["slope_of"] is not None:
                x = x - float(s["slope_of"][h]) * (i - j).abs()
            x = torch.where(blocked, float("-inf"), x)
            norm = torch.logsumexp(x, -1)
            p = torch.where(blocked, 0.0, torch.exp(x - norm[:, None]))
            o = torch.mm(p, v)
            out[t0:t1, h], lse[h, t0:t1] = o, norm
            if s["back"]:
                g = s["dout"][t0:t1, h].double()
                ds = p * (torch.mm(g, v.t()) - (g * o).sum(-1, keepdim=True)) * slope * scale
                dq[t0:t1, h] = torch.mm(ds, k)
                dk[t0:t1, h // group] += torch.mm(ds.t(), q)
                dv[t0:t1, h // group] += torch.mm(p.t(), g)
    return [out, lse, dq, dk, dv] if s["back"] else [out, lse]


def _exact_clip(s):
    total = sum(float(g.double().pow(2).sum()) for g in s["grads"])
    norm = total ** 0.5 * s["scale"]
    factor = min(1.0, s["limit"] / (norm + 1e-6)) * s["scale"]
    return [torch.tensor(norm, dtype=torch.float64), s["flat"].double() * factor]
