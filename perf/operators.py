"""The block-scaled 8-bit floating-point operators, as a user's program calls them.

``listed()`` gives the cases, ``draw(rng)`` one more of the same ranges, ``prepare(case, seed)``
what a program has in hand before a call, ``run(state)`` one pass: in elementary torch operations
where ``own`` is false, through the framework's entry points where it is true.  ``exact(case,
seed)`` is the same from the definition in 64 bits, ``work(case)`` what a pass cannot do without.

A block of 128 values x with A = max(max|x|, 2^-100) is held as q = round(x * (F / A)) in e4m3
(F = 448) or e5m2 (F = 57344) with the scale A / F.  Activations have a scale for each row and 128
columns, stored [ceil(k/128)][rows]; weights [m][k] one for each 128 x 128 block, stored
[ceil(m/128)][ceil(k/128)].
"""
import torch

own = False

BLOCK = 128
TINY = 2.0 ** -100
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ---------------------------------------------------------------------------------
def listed():
    return [
        # activations of a small ragged batch, a last block of 104 columns, the wide-range format
        {"name": "quant_ragged", "op": "quant", "rows": 333, "cols": 1000, "type": "f16", "format": "e5m2", "block_rows": 1},
        # activations of a long prompt (the 8192 x 4096 MatMul operand of the benchmark)
        {"name": "quant_prompt", "op": "quant", "rows": 8192, "cols": 4096, "type": "bf16", "format": "e4m3", "block_rows": 1},
        # the benchmark's 4096 x 11008 weight, laid out once from 32-bit values
        {"name": "quant_weight", "op": "quant", "rows": 11008, "cols": 4096, "type": "f32", "format": "e4m3", "block_rows": 128},
        # one token between two layers: latency
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096, "type": "bf16", "format": "e4m3", "resid": True, "plain": False},
        # an odd width, no residual yet (a model's first norm), the plain output kept for a router
        {"name": "norm_ragged", "op": "norm", "rows": 517, "cols": 1001, "type": "f32", "format": "e4m3", "resid": False, "plain": True},
        # a long prompt
        {"name": "norm_prompt", "op": "norm", "rows": 8192, "cols": 4096, "type": "bf16", "format": "e4m3", "resid": True, "plain": False},
        # one token's projection: the weight is read once
        {"name": "matmul_token", "op": "matmul", "n": 1, "k": 4096, "m": 4096, "type": "bf16", "a_format": "e4m3", "b_format": "e4m3"},
        # ragged in every direction (k = 1000 and the classifier's 1000 columns plus 1), 32-bit output
        {"name": "matmul_ragged", "op": "matmul", "n": 300, "k": 1000, "m": 1001, "type": "f32", "a_format": "e5m2", "b_format": "e4m3"},
        # the benchmark's largest MatMul
        {"name": "matmul_prompt", "op": "matmul", "n": 8192, "k": 4096, "m": 11008, "type": "bf16", "a_format": "e4m3", "b_format": "e4m3"},
        # a few tokens over many experts: most of them hold one row or none
        {"name": "experts_token", "op": "experts", "groups": 64, "n": 48, "k": 2048, "m": 1024, "type": "bf16"},
        # a small uneven batch, odd sizes, rows behind the last group
        {"name": "experts_ragged", "op": "experts", "groups": 7, "n": 1003, "k": 1000, "m": 520, "type": "f16"},
        # a long prompt over sixteen experts
        {"name": "experts_prompt", "op": "experts", "groups": 16, "n": 8192, "k": 4096, "m": 4096, "type": "bf16"},
    ]


def _size(rng, low, high):
    """A size from low to high, spread over its logarithm; two of three as they fall, the others multiples of 16."""
    v = int(round(low * (high / low) ** rng.random()))
    return max(low, v if rng.random() < 2 / 3 else (v + 15) // 16 * 16 if v > 16 and (v + 15) // 16 * 16 <= high else v)


def draw(rng):
    op = rng.choice(["quant", "norm", "matmul", "experts"])
    type_ = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quant":
        blocks = rng.choice([1, 1, 128])
        rows = _size(rng, 1, 8192)
        return {"op": op, "rows": rows, "cols": _size(rng, 64, 8192 if rows <= 4096 else 4096), "type": type_,
                "format": rng.choice(["e4m3", "e4m3", "e5m2"]), "block_rows": blocks}
    if op == "norm":
        rows = _size(rng, 1, 8192)
        return {"op": op, "rows": rows, "cols": _size(rng, 64, 8192 if rows <= 2048 else 4096 if rows <= 4096 else 2048), "type": type_,
                "format": rng.choice(["e4m3", "e4m3", "e5m2"]), "resid": rng.random() < 0.7, "plain": rng.random() < 0.3}
    if op == "matmul":
        return {"op": op, "n": _size(rng, 1, 8192), "k": _size(rng, 128, 4096), "m": _size(rng, 64, 8192), "type": type_,
                "a_format": rng.choice(["e4m3", "e4m3", "e5m2"]), "b_format": rng.choice(["e4m3", "e4m3", "e4m3", "e5m2"])}
    return {"op": op, "groups": _size(rng, 1, 64), "n": _size(rng, 1, 8192), "k": _size(rng, 128, 2048), "m": _size(rng, 64, 2048), "type": type_}


def work(case):
    c, up = case, lambda v: -(-v // BLOCK)
    if c["op"] == "quant":
        blocks = (c["rows"] if c["block_rows"] == 1 else up(c["rows"])) * up(c["cols"])
        return {"bytes": c["rows"] * c["cols"] * (SIZES[c["type"]] + 1) + 4 * blocks, "flops": 3 * c["rows"] * c["cols"]}
    if c["op"] == "norm":
        each = SIZES[c["type"]] * (1 + 2 * c["resid"] + c["plain"]) + 1
        return {"bytes": c["rows"] * c["cols"] * each + 4 * c["rows"] * up(c["cols"]) + c["cols"] * SIZES[c["type"]],
                "flops": 7 * c["rows"] * c["cols"]}
    n, k, m = c["n"], c["k"], c["m"]
    if c["op"] == "matmul":
        return {"bytes": n * k + m * k + 4 * up(k) * (n + up(m)) + n * m * SIZES[c["type"]], "flops": 2 * n * k * m}
    sizes = _rows_of(c)
    used, rows = sum(s > 0 for s in sizes), sum(sizes)
    return {"bytes": rows * k + used * m * k + 4 * up(k) * (rows + used * up(m)) + rows * m * SIZES[c["type"]] + 4 * (c["groups"] + 1),
            "flops": 2 * rows * k * m}


def _rows_of(c):
    """Rows of each group: uneven as a router leaves them (weights 1 / (place + 1) in a fixed shuffled order), every
    eighth group empty; where the case has several groups, n // 50 rows lie behind the last one."""
    g = c["groups"]
    share = [0.0 if g > 1 and i % 8 == 5 else 1.0 / (1 + (i * 7919 + 3) % g) for i in range(g)]
    rows, total, at, sizes = c["n"] - (c["n"] // 50 if g > 1 else 0), sum(share), 0.0, []
    for s in share:
        start = int(at / total * rows + 0.5)
        at += s
        sizes.append(int(at / total * rows + 0.5) - start)
    return sizes


# ---- the inputs --------------------------------------------------------------------------------
def _values(gen, *shape):
    """Activations: normal, some channels ten times as large, as hidden states have them."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    return x * (1 + 9 * (torch.rand(shape[-1], generator=gen, device="cuda") < 0.02))


def _blocks_of(x, block_rows):
    """x [..., rows, cols] padded to whole blocks and seen as [..., row blocks, block_rows, column blocks, 128]."""
    rows, cols = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    return x.reshape(*x.shape[:-2], x.shape[-2] // block_rows, block_rows, x.shape[-1] // BLOCK, BLOCK)


def _quantise(x, format_, block_rows):
    """x [..., rows, cols] in 32 bits -> (8-bit values of the same shape, scales [..., row blocks, column blocks])."""
    rows, cols = x.shape[-2:]
    b = _blocks_of(x, block_rows)
    top = b.abs().amax(dim=(-3, -1), keepdim=True).clamp_min(TINY)
    f = LARGEST[format_]
    q = (b * (f / top)).clamp(-f, f).to(FORMATS[format_])
    q = q.reshape(*x.shape[:-2], b.shape[-4] * block_rows, b.shape[-2] * BLOCK)[..., :rows, :cols]
    return q.contiguous(), (top / f).squeeze(-1).squeeze(-2)


def _operand(x, format_):
    """Activations as the quantising operators leave them: 8-bit rows and scales [column blocks][rows]."""
    q, s = _quantise(x, format_, 1)
    return q, s.transpose(-1, -2).contiguous()


def _rows16(q):
    """The same values in rows that lie a multiple of 16 bytes apart, as the framework asks of 8-bit operands that it reads in place."""
    room = torch.zeros(*q.shape[:-1], (q.shape[-1] + 15) // 16 * 16, dtype=torch.uint8, device=q.device)
    room[..., : q.shape[-1]] = q.view(torch.uint8)
    return room.view(q.dtype)[..., : q.shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c, up = case, lambda v: -(-v // BLOCK)
    empty = lambda *shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if c["op"] == "quant":
        x = _values(gen, c["rows"], c["cols"]) * (1.0 if c["block_rows"] == 1 else 0.02)
        shape = (up(c["cols"]), c["rows"]) if c["block_rows"] == 1 else (up(c["rows"]), up(c["cols"]))
        return {"case": c, "x": x.to(TYPES[c["type"]]), "q": empty(c["rows"], c["cols"], dtype=FORMATS[c["format"]]), "scale": empty(*shape, dtype=torch.float32)}
    if c["op"] == "norm":
        t, shape = TYPES[c["type"]], (c["rows"], c["cols"])
        s = {"case": c, "x": _values(gen, *shape).to(t), "weight": (1 + 0.1 * torch.randn(c["cols"], generator=gen, device="cuda")).to(t)}
        s["resid"] = (4 * _values(gen, *shape)).to(t) if c["resid"] else None
        s["resid_out"] = empty(*shape, dtype=t) if c["resid"] else None
        s["y"] = empty(*shape, dtype=t) if c["plain"] else None
        s["q"], s["scale"] = empty(*shape, dtype=FORMATS[c["format"]]), empty(up(c["cols"]), c["rows"], dtype=torch.float32)
        return s
    n, k, m = c["n"], c["k"], c["m"]
    groups = (c["groups"],) if c["op"] == "experts" else ()
    a, a_scale = _operand(_values(gen, n, k), c.get("a_format", "e4m3"))
    b, b_scale = _quantise(torch.randn(*groups, m, k, generator=gen, device="cuda") * 0.02, c.get("b_format", "e4m3"), BLOCK)
    s = {"case": c, "a": _rows16(a), "a_scale": a_scale, "b": _rows16(b), "b_scale": b_scale, "c": torch.zeros(n, m, dtype=TYPES[c["type"]], device="cuda")}
    if groups:
        sizes = _rows_of(c)
        ends = [0]
        for v in sizes:
            ends.append(ends[-1] + v)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["most"] = max(sizes)  # the longest group, which a program that pads its groups knows
    return s


# ---- one pass ----------------------------------------------------------------------------------
def _framework():
    import cormorant_b200 as cm

    if _framework.ready is None:
        cm.init("0")
        _framework.ready = cm
    return cm


_framework.ready = None


def run(state):
    s, c = state, state["case"]
    if own:
        cm, stream = _framework(), torch.cuda.current_stream()
        if c["op"] == "quant":
            cm.QuantKernelFp8(s["x"], s["q"], s["scale"], c["rows"], c["cols"], block_rows=c["block_rows"], stream=stream)
            return {"q": s["q"], "scale": s["scale"]}
        if c["op"] == "norm":
            cm.RmsNormKernelFp8(s["x"], s["weight"], s["q"], s["scale"], c["rows"], c["cols"], eps=1e-5, resid=s["resid"], resid_out=s["resid_out"], y=s["y"], stream=stream)
            return {"q": s["q"], "scale": s["scale"], "resid": s["resid_out"], "y": s["y"]}
        if c["op"] == "matmul":
            cm.MatmulKernelFp8(s["a"], s["a_scale"], s["b"], s["b_scale"], s["c"], c["n"], c["k"], c["m"], stream=stream)
        else:
            cm.MatmulKernelFp8Grouped(s["a"], s["a_scale"], s["b"], s["b_scale"], s["c"], s["offsets"], c["groups"], c["n"], c["k"], c["m"], stream=stream)
        return {"c": s["c"]}
    if c["op"] == "quant":
        return _plain_quant(s["x"].float(), c["format"], c["block_rows"])
    if c["op"] == "norm":
        h = s["x"].float() if s["resid"] is None else s["x"].float() + s["resid"].float()
        y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-5) * s["weight"].float()
        t = TYPES[c["type"]]
        return {**_plain_quant(y, c["format"], 1), "resid": None if s["resid"] is None else h.to(t), "y": y.to(t) if c["plain"] else None}
    rows, blocks = s["a_scale"].shape[1], s["a_scale"].shape[0]
    a = _blocks_of(s["a"].float(), 1) * s["a_scale"].t().reshape(rows, 1, blocks, 1)
    a = a.reshape(rows, blocks * BLOCK)
    b = _blocks_of(s["b"].float(), BLOCK) * s["b_scale"].unsqueeze(-1).unsqueeze(-3)
    b = b.reshape(*b.shape[:-4], b.shape[-4] * BLOCK, blocks * BLOCK)[..., : c["m"], :]
    if c["op"] == "matmul":
        return {"c": (a @ b.t()).to(TYPES[c["type"]])}
    # the groups' rows side by side in a padded batch, one batched product, and back; the rows behind the last group stay as they are
    start, size = s["offsets"][:-1].long(), s["offsets"].diff().long()
    place = torch.arange(s["most"], device="cuda")
    at = (start[:, None] + place).clamp_max(rows - 1)
    inside = place < size[:, None]
    c_ = torch.bmm(a[at] * inside[..., None], b.transpose(1, 2)).to(TYPES[c["type"]])
    out = s["c"].clone()
    out[at[inside]] = c_[inside]
    return {"c": out}


def _plain_quant(x, format_, block_rows):
    q, s = _quantise(x, format_, block_rows)
    return {"q": q, "scale": s.t().contiguous() if block_rows == 1 else s}


# ---- the definition in 64 bits -----------------------------------------------------------------
def _exact_quant(x, format_, block_rows):
    rows, cols = x.shape
    f, cb, rb = LARGEST[format_], -(-cols // BLOCK), -(-rows // block_rows)
    column = torch.arange(cols, device="cuda") // BLOCK
    row = torch.arange(rows, device="cuda") // block_rows
    place = row[:, None] * cb + column[None, :]
    top = torch.full((rb * cb,), TINY, dtype=torch.float64, device="cuda")
    top.scatter_reduce_(0, place.reshape(-1), x.abs().reshape(-1), "amax")
    q = torch.clamp(x * f / top[place], -f, f).to(FORMATS[format_]).double()
    scale = (top / f).reshape(rb, cb)
    return {"q": q, "scale": scale.t().contiguous() if block_rows == 1 else scale}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quant":
        return _exact_quant(s["x"].double(), c["format"], c["block_rows"])
    if c["op"] == "norm":
        h = s["x"].double() + (0 if s["resid"] is None else s["resid"].double())
        y = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / c["cols"] + 1e-5) * s["weight"].double()
        return {**_exact_quant(y, c["format"], 1), "resid": None if s["resid"] is None else h, "y": y if c["plain"] else None}
    block = torch.arange(c["k"], device="cuda") // BLOCK
    row = torch.arange(c["m"], device="cuda") // BLOCK
    a = s["a"].double() * s["a_scale"].double()[block].t()
    if c["op"] == "matmul":
        return {"c": a @ (s["b"].double() * s["b_scale"].double()[row][:, block]).t()}
    out, ends = s["c"].double(), s["offsets"].tolist()
    for g in range(c["groups"]):
        if ends[g + 1] > ends[g]:
            w = s["b"][g].double() * s["b_scale"][g].double()[row][:, block]
            out[ends[g] : ends[g + 1]] = a[ends[g] : ends[g + 1]] @ w.t()
    return {"c": out}
